"""The operators where offsets pass 32 bits, and on two threads at once.  Only the few
rows and pages that a case touches are filled and compared."""

from __future__ import annotations

import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def _int32(a):
    return torch.tensor(np.asarray(a, np.int32), device=DEV)


def _ramp(*shape, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=gen, device=DEV).to(BF16)


def test_pages_past_4_gib():
    from heteroserve.kv import pages

    NB = 70000                                        # 16 x 8 x 128 bf16: 32 KB a page, 4.6 GB
    pool = torch.empty(1, 2, NB, 16, 8, 128, dtype=BF16, device=DEV)
    assert pool[0, 0].numel() * 2 < 2 ** 32 < pool.numel() * 2
    high = [NB - 1, NB - 2, NB - 3]
    pool[:, :, high] = _ramp(1, 2, 3, 16, 8, 128)
    want = pool[:, :, high].clone()
    for ids in ([7, 8, 9], [NB - 5, 10, NB - 6]):     # few ids in arguments, and far away
        pages.copy_blocks(pool, high, ids)
        assert torch.equal(pool[:, :, ids], want)
    many = 500
    pages.copy_blocks(pool, [NB - 1] * many, list(range(20, 20 + many)))
    assert torch.equal(pool[:, :, 20:20 + many], pool[:, :, NB - 1:].expand(-1, -1, many, -1, -1, -1))

    tables = torch.full((4, 3), -1, dtype=torch.int32, device=DEV)
    ctx, refs = _int32([40, 0, 0, 0]), torch.zeros(NB, dtype=torch.int32, device=DEV)
    tables[0] = _int32(high)
    refs[high] = 1
    pool[:, :, NB - 9] = 0
    forked = pages.fork_blocks(pool, tables, ctx, refs, [0], [2], [NB - 9])
    assert forked.tolist() == [1] and tables[2].tolist() == [NB - 1, NB - 2, NB - 9]
    assert torch.equal(pool[:, :, NB - 9, :8], want[:, :, 2, :8]) and not pool[:, :, NB - 9, 8:].any()
    before = pool[:, :, [NB - 1, NB - 2, NB - 3, NB - 9]].clone()
    moved, live = pages.compact_blocks(pool, tables, refs)
    assert live.item() == 4 and tables.tolist()[0] == [0, 1, 2] and tables.tolist()[2] == [0, 1, 3]
    assert torch.equal(pool[:, :, :4], before)
    assert refs[:5].tolist() == [2, 2, 1, 1, 0] and int(refs.sum()) == 6


def test_rotary_into_a_slot_past_4_gib():
    from heteroserve.kv import rotary

    NB = 140000                                       # 32 KB a page: 4.6 GB for the keys alone
    kc = torch.empty(NB, 16, 8, 128, dtype=BF16, device=DEV)
    vc = torch.empty(NB, 16, 8, 128, dtype=BF16, device=DEV)
    assert kc.numel() * 2 > 2 ** 32
    q, k, v = _ramp(2, 32, 128), _ramp(2, 8, 128, seed=1), _ramp(2, 8, 128, seed=2)
    at, freq = _int32([5, 16]), torch.full((64,), 0.5, device=DEV)
    tables = _int32([[NB - 1, -1], [3, NB - 2]])
    turned, kept = rotary.rotate_append_kv(q, k, v, at, freq, kc, vc, tables, at, keep_k=True)
    want = rotary.rotate_qk(q, k, at, freq)
    assert torch.equal(turned, want[0]) and torch.equal(kept, want[1])
    for i, (block, row) in enumerate([(NB - 1, 5), (NB - 2, 0)]):
        assert torch.equal(kc[block, row], kept[i]) and torch.equal(vc[block, row], v[i])


@pytest.mark.parametrize("n", [40, 300])
def test_prompts_past_4_gib(n):
    """Rows of a fused projection and outputs both more than 2^32 bytes from the start."""
    from heteroserve.model.prompt_attn import prompt_attention

    T, H, Hkv, D = 530000, 32, 2, 128
    rows = torch.empty(T, (H + 2 * Hkv) * D, dtype=BF16, device=DEV)
    out = torch.empty(T, H, D, dtype=BF16, device=DEV)
    assert out.numel() * 2 > 2 ** 32
    rows[T - 2 * n:] = _ramp(2 * n, (H + 2 * Hkv) * D)
    q, k, v = rows.split([H * D, Hkv * D, Hkv * D], 1)
    q, k, v = q.view(T, H, D), k.view(T, Hkv, D), v.view(T, Hkv, D)
    out[T - 2 * n - 1] = 3.0
    prompt_attention(q, k, v, _int32([T - 2 * n, T - n, T]), n, 0.1, out=out)
    last = [x[T - 2 * n:].contiguous() for x in (q, k, v)]
    want = prompt_attention(*last, _int32([0, n, 2 * n]), n, 0.1)
    # other workgroups may share the work here, and sums have another order: two roundings
    # of the outputs and probabilities of values below 5
    assert (out[T - 2 * n:].float() - want.float()).abs().max().item() <= 4 * 2.0 ** -8 * 5
    assert (out[T - 2 * n - 1] == 3.0).all()


def test_two_threads():
    """Every operator on two threads, each on a stream of its own with a state of its own:
    as one after the other, bit for bit."""
    from heteroserve.kv import pages, rotary
    from heteroserve.model.prompt_attn import prompt_attention

    def work(seed, out, n=20):
        q, k, v = _ramp(90, 8, 64, seed=seed), _ramp(90, 2, 64, seed=seed + 1), _ramp(90, 2, 64, seed=seed + 2)
        freq = torch.full((32,), 0.25, device=DEV)
        at = _int32(np.arange(90) % 45)
        seq = _int32(np.arange(90) // 45)
        first = _ramp(2, 2, 40, 16, 2, 64, seed=seed + 3)
        for _ in range(n):
            pool, refs = first.clone(), torch.zeros(40, dtype=torch.int32, device=DEV)
            tables = torch.full((6, 4), -1, dtype=torch.int32, device=DEV)
            ctx = _int32([45, 45, 0, 0, 0, 0])
            tables[:2, :3] = pages.find_free_blocks(refs, 9)[3:].view(2, 3)
            refs[3:9] = 1
            a, b = rotary.rotate_append_kv(q, k, v, at, freq, pool[0, 0], pool[0, 1], tables, at, seq,
                                           keep_k=True)
            o = prompt_attention(a, b, v, _int32([0, 45, 90]), 45, 0.125)
            p = prompt_attention(a, b, v, _int32([0, 90]), 90, 0.125)
            pages.fork_blocks(pool, tables, ctx, refs, [0, 1, 1], [2, 3, 4], pages.find_free_blocks(refs, 3))
            pages.free_blocks(tables, ctx, refs, [0, 3])
            pages.compact_blocks(pool, tables, refs)
            pages.copy_blocks(pool, [0, 1], [30, 31])
            out.append([a, b, o, p, pool, tables, ctx, refs])
        torch.cuda.current_stream().synchronize()

    want = [[], []]
    for i in range(2):
        work(10 * i, want[i], 1)
    torch.cuda.synchronize()
    got, errors, start = [[], []], [], threading.Barrier(2)

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream(device=DEV)):
                start.wait()
                work(10 * i, got[i])
        except Exception as e:   # reported by the main thread
            errors.append(repr(e))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 20
        for step in got[i]:
            for x, w in zip(step, want[i][0]):
                assert torch.equal(x, w)
