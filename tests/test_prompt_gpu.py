"""Attention over whole prompts against 64-bit arithmetic.

Tolerances, element by element, with u = 2^-24, P the exact probabilities, V the
largest |v| that a row sees and S its largest sum of |q k| over a head's
elements, scaled:
  scores    D products summed in fp32 and scaled are off by (D + 2) u S at most,
            so is their difference to the maximum, the exponential adds 4 u (its
            argument, in powers of 2, 2 u S more): a probability is off by a
            relative 2 (D + 4) u S + 4 u, and so is their sum; the output by twice
            that times sum P |v|
  sums      n terms in fp32: n u sum P |v|, in the numerator and the denominator
  16 bits   probabilities rounded to the type: eps / 2 sum P |v|, and where they
            fall below fp16's normal range 2^-25 V each; the output rounded to it
"""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import operators as ops  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rows(lens, H, Hkv, D, dtype, seed, extra=0, size=1.0):
    """(q, k, v, cu): slices of fused rows, `extra` rows behind the last sequence."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n = sum(lens) + extra
    rows = (torch.randn(n, (H + 2 * Hkv) * D, generator=gen, device=DEV) * size).to(dtype)
    q, k, v = rows.split([H * D, Hkv * D, Hkv * D], 1)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    return q.view(n, H, D), k.view(n, Hkv, D), v.view(n, Hkv, D), cu


def _np(x):
    return x.double().cpu().numpy()


def _tolerance(q, k, v, cu, scale, want, spread, dtype):
    u, D, g = 2.0 ** -24, q.shape[2], q.shape[1] // k.shape[1]
    q, k, v = np.abs(q), np.abs(k), np.abs(v)
    tol = np.zeros_like(want)
    for a, b in zip(cu[:-1], cu[1:]):
        for h in range(q.shape[1]):
            s = np.tril(q[a:b, h] @ k[a:b, h // g].T * abs(scale))
            if not s.size:
                continue
            S = s.max(1, initial=0.0)[:, None]
            n = np.arange(1, b - a + 1)[:, None]
            V = np.maximum.accumulate(v[a:b, h // g].max(1))[:, None]
            rel = 2 * (2 * (D + 4) * u * S + 4 * u + n * u)
            t = rel * spread[a:b, h]
            if dtype is not F32:
                half = torch.finfo(dtype).eps / 2
                t = t + half * spread[a:b, h] * (1 + rel) + half * (np.abs(want[a:b, h]) + t)
                if dtype is F16:
                    t = t + n * 2.0 ** -25 * V + 2.0 ** -25
            tol[a:b, h] = t
    return tol


def _check(q, k, v, cu, dtype, scale=None, max_len=None):
    from heteroserve.model.prompt_attn import prompt_attention

    scale = q.shape[2] ** -0.5 if scale is None else scale
    longest = int(np.diff(cu).max(initial=0)) if max_len is None else max_len
    got = prompt_attention(q, k, v, torch.tensor(cu, device=DEV), longest, scale)
    assert got.dtype is dtype and got.shape == q.shape
    qn, kn, vn = _np(q), _np(k), _np(v)
    want, spread = ops.prompt(qn, kn, vn, cu, scale)
    tol = _tolerance(qn, kn, vn, cu, scale, want, spread, dtype)
    n = cu[-1]
    err = np.abs(_np(got)[:n] - want[:n])
    assert (err <= tol[:n]).all(), (err.max(), np.unravel_index((err - tol[:n]).argmax(), err.shape))
    return got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("lens,H,Hkv", [([1], 1, 1), ([0, 1, 2, 0], 4, 2), ([17, 0, 64, 33], 4, 4),
                                        ([31, 32, 33, 15, 16], 6, 1), ([130, 5], 8, 2)])
def test_small(dtype, D, lens, H, Hkv):
    _check(*_rows(lens, H, Hkv, D, dtype, sum(lens) + D), dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D,H,Hkv", [(64, 2, 2), (128, 4, 1), (32, 2, 1), (256, 2, 1)])
def test_several_tiles(dtype, D, H, Hkv):
    """Lengths around the tiles of queries and keys."""
    _check(*_rows([255, 300, 64, 257], H, Hkv, D, dtype, D), dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_many_heads_and_sequences(dtype):
    """Head counts that are and are not spread evenly over the dies."""
    for H, Hkv in ((16, 16), (16, 8), (9, 3), (40, 8)):
        _check(*_rows([3, 70, 1, 40] * 3, H, Hkv, 64, dtype, H), dtype)
    _check(*_rows([int(x) for x in np.random.default_rng(0).integers(0, 9, 300)], 2, 1, 64, dtype, 7),
           dtype)


def _dense(q, k, v, cu, scale):
    """float64 on the GPU, for long sequences."""
    out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    g = q.shape[1] // k.shape[1]
    for a, b in zip(cu[:-1], cu[1:]):
        a, b = int(a), int(b)
        later = torch.ones(b - a, b - a, dtype=torch.bool, device=DEV).triu(1)
        for h in range(q.shape[1]):
            s = torch.mm(q[a:b, h].double(), k[a:b, h // g].double().t().contiguous()) * scale
            out[a:b, h] = torch.mm(torch.softmax(s.masked_fill(later, -np.inf), -1),
                                   v[a:b, h // g].double())
    return out


@pytest.mark.parametrize("dtype,D,lens,H,Hkv", [
    (BF16, 128, [2500, 1, 1111], 16, 2), (F16, 64, [1025, 4097], 8, 8), (BF16, 256, [700, 1300], 4, 2),
    (F16, 32, [3001], 8, 1), (F32, 128, [1501, 600], 8, 4), (F32, 64, [2049], 3, 3),
    (BF16, 64, [128] * 40, 16, 16), (F16, 128, [8191], 2, 1)])
def test_long(dtype, D, lens, H, Hkv):
    """Relative to each row's 2-norm.  Probabilities and outputs of N(0, 1) values
    rounded to a type each add up to eps / 2 of the output's 2-norm (the rounding
    errors of the probabilities, weighted with the values, add up as the values
    themselves do); fp32 sums of n terms in any order n u at most, and as random
    errors far below 64 u for every n here."""
    from heteroserve.model.prompt_attn import prompt_attention

    q, k, v, cu = _rows(lens, H, Hkv, D, dtype, D + H)
    got = prompt_attention(q, k, v, torch.tensor(cu, device=DEV), max(lens), D ** -0.5).double()
    want = _dense(q, k, v, cu, D ** -0.5)
    tol = 64 * 2.0 ** -24 + (0 if dtype is F32 else 2 * torch.finfo(dtype).eps / 2)
    rel = ((got - want).norm(dim=-1) / want.norm(dim=-1)).max().item()
    assert rel <= tol, (rel, tol)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 30.0])
def test_scales(dtype, scale):
    """No scale, a negative one, and scores so large that one key takes all."""
    _check(*_rows([40, 70], 2, 1, 64, dtype, 4), dtype, scale=scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("D", [64, 256])
def test_what_lies_behind_a_row_does_not_reach_it(dtype, bad, where, D):
    """Rows in front of a NaN or an infinity, of its own sequence and of others, are
    as without it; rows behind it follow the definition."""
    from heteroserve.model.prompt_attn import prompt_attention

    lens, at = [50, 90, 20], 50 + 37
    q, k, v, cu = _rows(lens, 2, 2, D, dtype, 11)
    q, k, v = q.clone(), k.clone(), v.clone()
    cu_d = torch.tensor(cu, device=DEV)
    clean = prompt_attention(q, k, v, cu_d, 90, D ** -0.5)
    dirty = {"k": k, "v": v}[where]
    dirty[at, 0, 5] = bad
    got = prompt_attention(q, k, v, cu_d, 90, D ** -0.5)
    # one head and the rows from `at` on are touched
    assert torch.equal(got[:, 1], clean[:, 1])
    assert torch.equal(got[140:], clean[140:])
    assert torch.isfinite(got[:at]).all()
    tol = 2.0 ** -16 if dtype is F32 else 4 * torch.finfo(dtype).eps
    assert ((got[:at, 0] - clean[:at, 0]).float().abs() <= tol * clean[:at, 0].float().abs().max()).all()
    want = _dense(q[50:140], k[50:140], v[50:140], [0, 90], D ** -0.5)[37:, 0]
    assert torch.equal(torch.isnan(want), torch.isnan(got[at:140, 0]))
    assert torch.equal(want == np.inf, got[at:140, 0] == np.inf)
    assert torch.equal(want == -np.inf, got[at:140, 0] == -np.inf)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_no_sequence_are_left_as_they_were(dtype):
    from heteroserve.model.prompt_attn import prompt_attention

    q, k, v, cu = _rows([20, 33], 2, 1, 64, dtype, 3, extra=70)
    out = torch.full_like(q, 7.0, memory_format=torch.contiguous_format)
    k[53:], v[53:] = float("nan"), float("nan")
    got = prompt_attention(q, k, v, torch.tensor(cu, device=DEV), 33, 0.125, out=out)
    assert got is out and (out[53:] == 7.0).all() and torch.isfinite(out[:53]).all()
    # sequences with rows between them, and one cut short by max_seqlen
    out.fill_(7.0)
    cut = prompt_attention(q, k, v, torch.tensor([5, 20, 53], dtype=torch.int32), 17, 0.125, out=out)
    assert (cut[:5] == 7.0).all() and (cut[37:] == 7.0).all()
    want, _ = ops.prompt(_np(q), _np(k), _np(v), [5, 20, 37], 0.125)
    assert np.abs(_np(cut)[5:37] - want[5:37]).max() < 0.05


def test_offsets_that_are_no_offsets():
    """Descending, negative and far offsets: rows outside [0, T) are never touched, and
    nothing is read behind the tensors."""
    from heteroserve.model.prompt_attn import prompt_attention

    q, k, v, _ = _rows([40], 2, 1, 64, BF16, 3)
    for cu in ([-5, 20, 2 ** 31 - 1], [30, 10, 40], [50, 60, 70], [-2 ** 31, -1, 0]):
        out = torch.full_like(q, 7.0, memory_format=torch.contiguous_format)
        prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32), 64, 0.125, out=out)
        assert torch.isfinite(out).all()


def test_layouts():
    """Heads apart, heads of one, expanded keys, unaligned slices, transposed tensors."""
    from heteroserve.model.prompt_attn import prompt_attention

    q, k, v, cu = _rows([33, 50], 4, 2, 64, BF16, 8)
    cu = torch.tensor(cu, device=DEV)
    want = prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu, 50, 0.125)
    assert torch.equal(prompt_attention(q, k, v, cu, 50, 0.125), want)
    flipped = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(prompt_attention(*flipped, cu, 50, 0.125), want)
    wide = torch.zeros(83, 4, 3, 64, dtype=BF16, device=DEV)
    wide[:, :, 1] = q
    assert torch.equal(prompt_attention(wide[:, :, 1], k, v, cu, 50, 0.125), want)
    odd = torch.zeros(83, 4 * 64 + 3, dtype=BF16, device=DEV)
    odd[:, 3:] = q.reshape(83, 256)
    assert torch.equal(prompt_attention(odd[:, 3:].view(83, 4, 64), k, v, cu, 50, 0.125), want)
    last = torch.zeros(83, 4, 64, 2, dtype=BF16, device=DEV)
    last[..., 1] = q
    assert torch.equal(prompt_attention(last[..., 1], k, v, cu, 50, 0.125), want)
    one = prompt_attention(q, k[:, :1], v[:, :1], cu, 50, 0.125)
    assert torch.equal(prompt_attention(q, k[:, :1].expand(83, 2, 64), v[:, :1].expand(83, 2, 64), cu,
                                        50, 0.125), one)


def test_two_streams_at_once_and_replayed():
    """Calls share nothing: two at once, and a graph replayed beside eager work."""
    from heteroserve.model.prompt_attn import prompt_attention

    sets = [_rows([700, 80], 8, 2, 128, BF16, s) for s in (1, 2)]
    cu = torch.tensor(sets[0][3], device=DEV)
    want = [prompt_attention(q, k, v, cu, 700, 0.09) for q, k, v, _ in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                q, k, v, _ = sets[i]
                got[i].append(prompt_attention(q, k, v, cu, 700, 0.09))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    graph = torch.cuda.CUDAGraph()
    q, k, v, _ = sets[0]
    with torch.cuda.graph(graph):
        out = prompt_attention(q, k, v, cu, 700, 0.09)
    for _ in range(3):
        out.fill_(float("nan"))
        eager = prompt_attention(*sets[1][:3], cu, 700, 0.09)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(eager, want[1])


def test_same_as_the_paged_prefill():
    """The engine's other way to the same rows: through the cache."""
    from heteroserve.kv import pack
    from heteroserve.model.paged_attn_prefill import paged_attention_prefill_varlen
    from heteroserve.model.prompt_attn import prompt_attention

    lens = [60, 200, 16]
    q, k, v, cu = _rows(lens, 8, 2, 128, F16, 6)
    tables = pack.block_table_tensor([[3, 1, 8, 2], list(range(10, 23)), [0]], device=DEV)
    kc, vc = torch.zeros(2, 24, 16, 2, 128, dtype=F16, device=DEV)
    seq = np.repeat(np.arange(3), lens).astype(np.int32)
    at = np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
    pack.append_kv(kc, vc, tables, torch.tensor(at), k, v, torch.tensor(seq))
    cu = torch.tensor(cu, device=DEV)
    a = prompt_attention(q, k, v, cu, 200, 0.09)
    b = paged_attention_prefill_varlen(q.float(), cu, 200, kc, vc, tables,
                                       torch.tensor(lens, dtype=torch.int32), 0.09)
    assert (a.float() - b).abs().max() <= 2e-3 + 2.0 ** -11 * b.abs().max()


def test_nothing_to_do():
    from heteroserve.model.prompt_attn import prompt_attention

    q = torch.empty(0, 4, 64, device=DEV, dtype=BF16)
    assert prompt_attention(q, q, q, torch.zeros(1, dtype=torch.int32), 0, 1.0).shape == (0, 4, 64)
    q, k, v, cu = _rows([5], 4, 4, 64, BF16, 1)
    out = torch.full_like(q, 3.0, memory_format=torch.contiguous_format)
    prompt_attention(q, k, v, torch.zeros(1, dtype=torch.int32), 5, 1.0, out=out)
    prompt_attention(q, k, v, torch.tensor([0, 5]), 0, 1.0, out=out)
    assert (out == 3.0).all()


def test_refusals():
    from heteroserve.model.prompt_attn import prompt_attention

    q, k, v, cu = _rows([8], 4, 2, 64, BF16, 1)
    cu = torch.tensor(cu, device=DEV)

    def refused(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            prompt_attention(*args, cu, 8, 0.1, **kw)

    refused("on CUDA", q.cpu(), k, v)
    refused("same dtype", q, k.float(), v)
    refused("k and v must be", q, k[:7], v)
    refused("k and v must be", q, k, v[:, :1])
    refused("divisible", q[:, :3], k, v)
    refused("total_tokens", q[0], k, v)
    refused("unsupported head_dim", q[..., :48], k[..., :48], v[..., :48])
    refused("unsupported", q.double(), k.double(), v.double())
    refused("out must be", q, k, v, out=torch.empty(8, 4, 64, device=DEV))
    refused("out must be", q, k, v, out=torch.empty(4, 8, 64, device=DEV, dtype=BF16).transpose(0, 1))
    with pytest.raises(RuntimeError, match="cu_seqlens"):
        prompt_attention(q, k, v, torch.zeros(0, dtype=torch.int32), 8, 0.1)
    with pytest.raises(RuntimeError, match="positive"):
        prompt_attention(q, k, v, cu, -1, 0.1)


def test_out_that_is_an_input_and_lengths_past_32_bits():
    from heteroserve.model.prompt_attn import prompt_attention

    q, k, v, cu = _rows([30, 12], 4, 2, 64, BF16, 1)
    cu = torch.tensor(cu, device=DEV)
    want = prompt_attention(q, k, v, cu, 30, 0.1)
    for longest in (42, 2 ** 32, 2 ** 40 + 1):
        assert torch.equal(prompt_attention(q, k, v, cu, longest, 0.1), want)
    with pytest.raises(RuntimeError, match="positive"):
        prompt_attention(q, k, v, cu, -2 ** 32, 0.1)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    both = torch.empty(2 * 42, 4, 64, dtype=BF16, device=DEV)
    both[42:] = q
    with pytest.raises(RuntimeError, match="overlap"):
        prompt_attention(q, k, v, cu, 30, 0.1, out=q)
    with pytest.raises(RuntimeError, match="overlap"):
        prompt_attention(both[42:], k, v, cu, 30, 0.1, out=both[1:43])
    got = prompt_attention(both[42:], k, v, cu, 30, 0.1, out=both[:42])
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D,H,Hkv", [(32, 4, 4), (64, 6, 2), (128, 8, 2), (256, 4, 1)])
def test_many_short_prompts(dtype, D, H, Hkv):
    """A wave each: odd counts of heads and prompts, none and one token, whole tiles and
    one row more, few and many (fp32 heads of 128 and more differ by their number)."""
    gen = np.random.default_rng(D + H)
    for lens in ([1, 32, 0, 31, 17], [33, 64, 63, 1], [int(x) for x in gen.integers(0, 33, 150)],
                 [int(x) for x in gen.integers(0, 65, 40)]):
        _check(*_rows(lens, H, Hkv, D, dtype, D + len(lens)), dtype)
    q, k, v, cu = _rows([20, 40, 30], H, Hkv, D, dtype, 3, extra=2)
    for scale in (0.0, -0.2, 30.0 / D):
        _check(q[:90], k[:90], v[:90], cu, dtype, scale=scale)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B", [65, 300, 1100, 4200])
def test_many_sequences_by_number_and_searched_for(dtype, B):
    """More sequences than lanes: one length but for one (tiles by their number from a
    thousand on) and lengths of which most are short (searched for, in one or two steps).
    Tolerance as of test_long."""
    from heteroserve.model.prompt_attn import prompt_attention

    gen = np.random.default_rng(B)
    for lens in ([70 if B < 1000 else 66] * B,
                 np.where(gen.random(B) < 40 / B, gen.integers(100, 420, B), gen.integers(0, 9, B)).tolist()):
        lens[B // 2] = 130
        q, k, v, cu = _rows(lens, 2, 1, 32, dtype, B)
        got = prompt_attention(q, k, v, torch.tensor(cu, device=DEV), max(lens), 0.2)
        want = _dense_each(q, k, v, cu, 0.2)
        tol = 64 * 2.0 ** -24 + (0 if dtype is F32 else 2 * torch.finfo(dtype).eps / 2)
        rel = ((got.double() - want).norm(dim=-1) / want.norm(dim=-1)).max().item()
        assert rel <= tol, (rel, tol)


def _dense_each(q, k, v, cu, scale):
    """_dense over padded batches: float64 [T, H, D]."""
    lens = np.diff(cu)
    n, B = int(lens.max()), len(lens)
    at = torch.tensor(cu[:-1].astype(np.int64), device=DEV)[:, None] + torch.arange(n, device=DEV)
    here = torch.arange(n, device=DEV) < torch.tensor(lens, device=DEV)[:, None]
    at = torch.where(here, at, 0)
    out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    g = q.shape[1] // k.shape[1]
    later = torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1)
    for h in range(q.shape[1]):
        for b0 in range(0, B, 256):
            i = at[b0:b0 + 256]
            x, y, z = q[i, h].double(), k[i, h // g].double(), v[i, h // g].double()
            s = torch.bmm(x, y.transpose(1, 2).contiguous()) * scale
            o = torch.bmm(torch.softmax(s.masked_fill(later, -np.inf), -1), z)
            m = here[b0:b0 + 256]
            out[i[m], h] = o[m]
    return out


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("D,B", [(64, 3), (256, 3), (128, 130)])
def test_what_lies_behind_a_short_prompts_row(dtype, bad, D, B):
    from heteroserve.model.prompt_attn import prompt_attention

    lens = [30] * B
    q, k, v, cu = _rows(lens, 4, 2, D, dtype, 11)
    q, k, v = q.clone(), k.clone(), v.clone()
    cu_d = torch.tensor(cu, device=DEV)
    for dirty in (k, v):
        clean = prompt_attention(q, k, v, cu_d, 30, D ** -0.5)
        kept, dirty[47, 0, 5] = dirty[47, 0, 5].clone(), bad
        got = prompt_attention(q, k, v, cu_d, 30, D ** -0.5)
        assert torch.equal(got[:, 2:], clean[:, 2:])
        assert torch.equal(got[60:], clean[60:]) and torch.equal(got[:30], clean[:30])
        assert torch.isfinite(got[:47]).all()
        tol = 2.0 ** -16 if dtype is F32 else 4 * torch.finfo(dtype).eps
        assert ((got[30:47] - clean[30:47]).float().abs() <= tol * clean[30:47].float().abs().max()).all()
        want = _dense(q[30:60], k[30:60], v[30:60], [0, 30], D ** -0.5)[17:, :2]
        assert torch.equal(torch.isnan(want), torch.isnan(got[47:60, :2]))
        assert torch.equal(want == np.inf, got[47:60, :2] == np.inf)
        dirty[47, 0, 5] = kept


def test_short_prompts_replayed_and_laid_out_otherwise():
    """Strided, transposed and expanded rows, rows of no sequence, and a replayed graph."""
    from heteroserve.model.prompt_attn import prompt_attention

    for dtype in (F32, F16):
        q, k, v, cu = _rows([33, 0, 50, 7], 4, 2, 64, dtype, 8, extra=3)
        cu = torch.tensor(cu, device=DEV)
        out = torch.full((93, 4, 64), 5.0, dtype=dtype, device=DEV)
        want = prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu, 50, 0.125, out=out)
        assert (want[90:] == 5.0).all()
        flipped = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
        for x in ((q, k, v), flipped):
            assert torch.equal(prompt_attention(*x, cu, 50, 0.125)[:90], want[:90])
        cut = prompt_attention(q, k, v, cu, 40, 0.125, out=torch.full_like(out, 6.0))
        assert torch.equal(cut[:73], want[:73]) and (cut[73:83] == 6.0).all()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = prompt_attention(q, k, v, cu, 50, 0.125)
        for _ in range(3):
            got.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got[:90], want[:90])


@pytest.mark.parametrize("lens", [[40, 20], [300, 5]])
def test_no_scale_and_scores_of_any_size(lens):
    """A scale of 0 makes every finite score 0, however large: the mean of the values."""
    from heteroserve.model.prompt_attn import prompt_attention

    for dtype in (F32, BF16):
        q, k, v, cu = _rows(lens, 2, 1, 64, dtype, 3)
        cu = torch.tensor(cu, device=DEV)
        big = prompt_attention((q * 2.0 ** 50).to(dtype), (k * 2.0 ** 50).to(dtype), v, cu, max(lens), 0.0)
        # scores of 0: other products, so only the rounding of the sums may differ
        none = prompt_attention(torch.zeros_like(q), k, v, cu, max(lens), 0.0)
        tol = 2 * max(lens) * 2.0 ** -24 * v.abs().max().item()
        tol += 0 if dtype is F32 else 2 * torch.finfo(dtype).eps * v.abs().max().item()
        assert (big.float() - none.float()).abs().max().item() <= tol


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D,H,Hkv", [(32, 16, 8), (64, 12, 4), (128, 16, 2), (256, 8, 8)])
def test_lengths_that_differ_and_are_many(dtype, D, H, Hkv):
    """Many prompts of up to some hundred tokens, most far shorter than the longest, and
    the same with rows behind them; lengths around 64 and none.  Tolerance as of
    test_long."""
    from heteroserve.model.prompt_attn import prompt_attention

    gen = np.random.default_rng(D)
    for lens in ([int(x) for x in gen.integers(0, 150, 60)], [63, 64, 65, 127, 128, 129, 1, 0, 400] * 4,
                 [int(x) for x in gen.integers(1, 640, 9)] + [768] + [3] * 20):
        q, k, v, cu = _rows(lens, H, Hkv, D, dtype, D + H, extra=5)
        out = torch.full((sum(lens) + 5, H, D), 9.0, dtype=dtype, device=DEV)
        got = prompt_attention(q, k, v, torch.tensor(cu, device=DEV), max(lens), D ** -0.5, out=out)
        assert (got[-5:] == 9.0).all()
        want = _dense_each(q, k, v, cu, D ** -0.5)[:-5]
        rel = ((got[:-5].double() - want).norm(dim=-1) / want.norm(dim=-1)).max().item()
        assert rel <= 64 * 2.0 ** -24 + (0 if dtype is F32 else 2 * torch.finfo(dtype).eps / 2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_bad_values_among_lengths_that_differ(dtype, bad):
    from heteroserve.model.prompt_attn import prompt_attention

    lens = [200, 30, 90, 10, 150] * 8
    q, k, v, cu = _rows(lens, 16, 16, 64, dtype, 11)
    q, k, v = q.clone(), k.clone(), v.clone()
    cu_d = torch.tensor(cu, device=DEV)
    clean = prompt_attention(q, k, v, cu_d, 200, 0.125)
    for dirty in (k, v):
        kept, dirty[150, 3, 5] = dirty[150, 3, 5].clone(), bad
        got = prompt_attention(q, k, v, cu_d, 200, 0.125)
        same = torch.ones_like(got, dtype=torch.bool)
        same[150:200, 3] = False
        same[:150, 3] = False          # computed again by another order of sums, if in its tile
        assert torch.equal(got[same], clean[same])
        tol = (2.0 ** -16 if dtype is F32 else 4 * torch.finfo(dtype).eps) * clean[:150, 3].float().abs().max()
        assert ((got[:150, 3] - clean[:150, 3]).float().abs() <= tol).all()
        want = _dense(q[:200], k[:200], v[:200], [0, 200], 0.125)[150:, 3]
        assert torch.equal(torch.isnan(want), torch.isnan(got[150:200, 3]))
        dirty[150, 3, 5] = kept
