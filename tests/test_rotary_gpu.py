"""Rotary positions and their cache write against 64-bit arithmetic.

Tolerance of a turned element a c - b s in fp32: the angle's fraction is rounded
once (2^-25 turns, pi 2^-24 radians), sine and cosine are within 2 units (2^-22),
two products and a sum round (3 * 2^-24): below 2^-20 (|a| + |b|) in all.  An
output of fewer bits is off by half a step more.
"""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import operators as ops  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _close(got, want, size, dtype, what):
    """size: |a| + |b| of each element."""
    got = got.double().cpu().numpy()
    tol = 2.0 ** -20 * size
    if dtype is not F32:
        tol = tol + torch.finfo(dtype).eps / 2 * (np.abs(want) + tol)
        tol = tol + (2.0 ** -25 if dtype is F16 else 0.0)     # half a step of subnormals
    assert got.shape == want.shape, what
    assert (np.abs(got - want) <= tol).all(), (what, np.abs(got - want).max())


def _inputs(n, H, Hkv, D, dtype, seed):
    """q, k, v as slices of fused rows."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rows = torch.randn(n, (H + 2 * Hkv) * D, generator=gen, device=DEV).to(dtype)
    q, k, v = rows.split([H * D, Hkv * D, Hkv * D], 1)
    return q.view(n, H, D), k.view(n, Hkv, D), v.view(n, Hkv, D)


def _np(x):
    return x.double().cpu().numpy()


def _size(x, pairs, interleaved):
    """|a| + |b| of every element (|a| where it passes)."""
    x = np.abs(_np(x))
    out = x.copy()
    a, b = ((slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved
            else (slice(0, pairs), slice(pairs, 2 * pairs)))
    out[..., a] = out[..., b] = x[..., a] + x[..., b]
    return out


def _freq(pairs):
    return torch.tensor((10000.0 ** (-np.arange(pairs) / pairs)).astype(np.float32), device=DEV)


@pytest.mark.parametrize("src", [F32, F16, BF16])
@pytest.mark.parametrize("out", [F32, F16, BF16])
@pytest.mark.parametrize("n,H,Hkv,D,pairs,axes,interleaved", [
    (1, 4, 4, 64, 32, 1, False), (7, 8, 2, 128, 64, 3, False), (33, 6, 1, 32, 8, 2, True),
    (5, 3, 3, 256, 128, 4, True), (9, 2, 1, 80, 20, 2, False), (4, 2, 2, 36, 18, 1, True),
    (3, 1, 1, 7, 2, 2, False), (1100, 2, 1, 64, 16, 3, False), (1030, 3, 1, 48, 24, 2, True)])
def test_rotate(src, out, n, H, Hkv, D, pairs, axes, interleaved):
    """Whole and partial heads, both pairings, sizes that are no 16-byte groups, and
    as many rows as make workgroups take several."""
    from heteroserve.kv import rotary

    q, k, _ = _inputs(n, H, Hkv, D, src, n + D)
    rng = np.random.default_rng(n)
    pos = rng.integers(0, 5000, (axes, n)).astype(np.int32)
    pair_axis = torch.tensor(rng.integers(0, axes, pairs).astype(np.int32))
    freq = _freq(pairs)
    got = rotary.rotate_qk(q, k, torch.tensor(pos), freq, axes=pair_axis, interleaved=interleaved,
                           out_dtype=out)
    for x, y, name in ((q, got[0], "q"), (k, got[1], "k")):
        want = ops.rotate(_np(x), pos, _np(freq), pair_axis.numpy(), interleaved)
        assert y.dtype is out and y.is_contiguous()
        _close(y, want, _size(x, pairs, interleaved), out, name)


def test_far_and_negative_positions():
    """Angles of up to 2^31 radians keep their fraction."""
    from heteroserve.kv import rotary

    pos = np.array([0, 1, -1, 999_983, -70_001, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31], np.int32)
    q, k, _ = _inputs(len(pos), 2, 1, 64, F32, 5)
    freq = _freq(32)
    got, _ = rotary.rotate_qk(q, k, torch.tensor(pos), freq)
    _close(got, ops.rotate(_np(q), pos, _np(freq)), _size(q, 32, False), F32, "q")


def test_axes_that_name_no_axis_count_as_the_first():
    from heteroserve.kv import rotary

    q, k, _ = _inputs(6, 2, 2, 64, F32, 6)
    pos = torch.arange(12, dtype=torch.int32).view(2, 6)
    bad = torch.tensor([-1, 0, 1, 2, 2 ** 31 - 1, -2 ** 31] * 5 + [0, 1], dtype=torch.int32)
    good = torch.where((bad < 0) | (bad > 1), 0, bad)
    a = rotary.rotate_qk(q, k, pos, _freq(32), axes=bad)
    b = rotary.rotate_qk(q, k, pos, _freq(32), axes=good)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    first = rotary.rotate_qk(q, k, pos[0], _freq(32))     # no axes: all on the first
    none = rotary.rotate_qk(q, k, pos, _freq(32), axes=torch.zeros(32, dtype=torch.int32))
    assert torch.equal(first[0], none[0])


@pytest.mark.parametrize("src,cache", [(F32, F16), (F32, BF16), (BF16, BF16), (F16, F32), (BF16, F16),
                                       (F32, F32), (F16, F16)])
@pytest.mark.parametrize("n,H,Hkv,D,pairs,BS", [(5, 8, 2, 128, 64, 16), (1, 4, 4, 64, 16, 8),
                                                (40, 2, 1, 36, 9, 5), (1025, 4, 1, 32, 16, 16)])
def test_append(src, cache, n, H, Hkv, D, pairs, BS):
    """Keys and values in their slots, the rest of the cache as it was; rows that
    append_kv would skip still give their q and k."""
    from heteroserve.kv import pack, rotary

    q, k, v = _inputs(n, H, Hkv, D, src, n + BS)
    rng = np.random.default_rng(n + D)
    B, MB = 4, -(-n // BS) + 2
    nb = B * MB + 3
    tables = torch.tensor(rng.permutation(nb)[:B * MB].reshape(B, MB).astype(np.int32), device=DEV)
    seq = np.sort(rng.integers(0, B, n)).astype(np.int32)
    at = np.zeros(n, np.int32)
    for b in range(B):
        at[seq == b] = np.arange((seq == b).sum()) + 3
    pos = np.stack([at + 100, at // 3, at % 3]).astype(np.int32)
    if n > 4:      # rows that are skipped: no such sequence, behind the table, padding
        seq[0], at[1] = B, MB * BS
        tables[seq[2], at[2] // BS] = -1
    axes = rotary.axes_of([pairs - 2 * (pairs // 3), pairs // 3, pairs // 3])
    freq = _freq(pairs)
    kc = torch.randn(nb, BS, Hkv, D, device=DEV).to(cache)
    vc = torch.randn(nb, BS, Hkv, D, device=DEV).to(cache)
    k0, v0 = kc.clone(), vc.clone()
    q_out, k_out = rotary.rotate_append_kv(q, k, v, torch.tensor(pos), freq, kc, vc, tables,
                                           torch.tensor(at), seq_ids=torch.tensor(seq), axes=axes,
                                           out_dtype=F32, keep_k=True)
    want_q = ops.rotate(_np(q), pos, _np(freq), axes.numpy())
    want_k = ops.rotate(_np(k), pos, _np(freq), axes.numpy())
    _close(q_out, want_q, _size(q, pairs, False), F32, "q")
    _close(k_out, want_k, _size(k, pairs, False), F32, "k")
    # the cache: append_kv of the turned keys, which are rounded once from fp32
    pack.append_kv(k0, v0, tables, torch.tensor(at), k_out, v.float(), torch.tensor(seq))
    assert torch.equal(kc, k0)
    assert torch.equal(vc, v0)


def test_single_tokens_without_sequence_ids_and_without_k():
    from heteroserve.kv import rotary

    q, k, v = _inputs(3, 4, 2, 64, BF16, 9)
    tables = torch.tensor([[2, 0], [1, -1], [3, 4]], dtype=torch.int32, device=DEV)
    at = torch.tensor([17, 4, 31], dtype=torch.int32, device=DEV)
    kc, vc = torch.zeros(2, 5, 16, 2, 64, device=DEV, dtype=BF16)
    got, none = rotary.rotate_append_kv(q, k, v, at, _freq(32), kc, vc, tables, at)
    assert none is None and got.dtype is BF16
    want = ops.rotate(_np(k), at.cpu().numpy(), _np(_freq(32)))
    for i, slot in enumerate((0 * 16 + 1, 1 * 16 + 4, 4 * 16 + 15)):
        _close(kc.view(-1, 2, 64)[slot], want[i], _size(k, 32, False)[i], BF16, i)
        assert torch.equal(vc.view(-1, 2, 64)[slot], v[i])


def test_values_of_the_caches_type_keep_every_bit():
    from heteroserve.kv import rotary

    for D in (64, 36):     # 16-byte groups, and none
        q, k, _ = _inputs(4, 1, 1, D, BF16, 2)
        bits = torch.randint(-2 ** 15, 2 ** 15, (4, 1, D), dtype=torch.int16, device=DEV)
        bits[:, :, 0] = 0x7F81      # a signalling NaN
        kc, vc = torch.zeros(2, 1, 4, 1, D, device=DEV, dtype=BF16)
        at = torch.arange(4, dtype=torch.int32, device=DEV)
        rotary.rotate_append_kv(q, k, bits.view(BF16), at, _freq(8), kc, vc,
                                torch.zeros(1, 1, dtype=torch.int32, device=DEV), at,
                                seq_ids=torch.zeros(4, dtype=torch.int32))
        assert torch.equal(vc.view(torch.int16).view(4, 1, D), bits)


@pytest.mark.parametrize("cut", [1, 3])
def test_unaligned_rows(cut):
    """Slices that start off a 16-byte boundary, and head rows that are no rows of the
    source."""
    from heteroserve.kv import rotary

    gen = torch.Generator(device=DEV).manual_seed(cut)
    wide = torch.randn(6, 2 * 64 + cut, generator=gen, device=DEV).to(BF16)
    q = wide[:, cut:].view(6, 2, 64)
    swapped = torch.randn(2, 6, 64, generator=gen, device=DEV).to(BF16).transpose(0, 1)
    pos = torch.arange(6, dtype=torch.int32)
    a = rotary.rotate_qk(q, swapped, pos, _freq(32))
    b = rotary.rotate_qk(q.contiguous(), swapped.contiguous(), pos, _freq(32))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_rows():
    from heteroserve.kv import rotary

    q = torch.empty(0, 4, 64, device=DEV)
    a, b = rotary.rotate_qk(q, q, torch.empty(1, 0, dtype=torch.int32), _freq(32))
    assert a.shape == b.shape == (0, 4, 64)


def test_on_another_stream_and_replayed():
    from heteroserve.kv import rotary

    q, k, v = _inputs(8, 8, 2, 128, BF16, 3)
    at = torch.arange(8, dtype=torch.int32, device=DEV)
    tables = torch.arange(8, dtype=torch.int32, device=DEV).view(8, 1)
    freq = _freq(64)
    kc, vc = torch.zeros(2, 8, 16, 2, 128, device=DEV, dtype=BF16)

    def step():
        return rotary.rotate_append_kv(q, k, v, at, freq, kc, vc, tables, at, keep_k=True)

    want = step()
    want_k = kc.clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kc.zero_()
        got = step()
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(kc, want_k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        kc.zero_()
        got[0].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(kc, want_k)


def test_refusals():
    from heteroserve.kv import rotary

    q, k, v = _inputs(4, 4, 2, 64, BF16, 1)
    pos = torch.arange(4, dtype=torch.int32)
    kc, vc = torch.zeros(2, 4, 16, 2, 64, device=DEV, dtype=BF16)
    bt = torch.zeros(4, 1, dtype=torch.int32, device=DEV)

    def refused(match, *args, **kw):
        call = rotary.rotate_qk if len(args) == 4 else rotary.rotate_append_kv
        with pytest.raises(RuntimeError, match=match):
            call(*args, **kw)

    f = _freq(32)
    refused("on CUDA", q.cpu(), k, pos, f)
    refused("dtype of q", q, k.float(), pos, f)
    refused("rows, the head_dim", q, k[:3], pos, f)
    refused("positions must be", q, k, pos[:3], f)
    refused("inv_freq", q, k, pos, _freq(33))
    refused("axes for 32", q, k, pos, f, axes=torch.zeros(3, dtype=torch.int32))
    refused("unsupported", q, k, pos, f, out_dtype=torch.float64)
    refused("same count", q, k, v[:3], pos, f, kc, vc, bt, pos)
    refused("same count", q, k, v.float(), pos, f, kc, vc, bt, pos)
    refused("K/V rows", q, k, v, pos, f, kc[..., :32].contiguous(), vc[..., :32].contiguous(), bt, pos)
    refused("written in place", q, k, v, pos, f, kc.transpose(1, 2), vc.transpose(1, 2), bt, pos)
    refused("more rows than tables", q, k, v, pos, f, kc, vc, bt[:3], pos)
    refused("sequence ids", q, k, v, pos, f, kc, vc, bt, pos, seq_ids=pos[:2])
    refused("at least|positions for", q, k, v, pos, f, kc, vc, bt, pos[:2])
    with pytest.raises(RuntimeError, match="sections"):
        rotary.axes_of([-1, 2])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D,pairs,interleaved", [(64, 32, False), (64, 16, True), (80, 20, False),
                                                 (128, 24, False), (7, 3, True)])
@pytest.mark.parametrize("n", [3, 2100])
def test_outputs_that_are_their_sources(dtype, D, pairs, interleaved, n):
    """hs_rotary and hs_rotary_append in place, as the header allows them."""
    from heteroserve import _hip
    from heteroserve.kv import rotary

    lib = _hip.lib()
    H, Hkv = 3, 2
    q, k, v = [x.contiguous() for x in _inputs(n, H, Hkv, D, dtype, 5)]
    at, freq = torch.arange(n, dtype=torch.int32, device=DEV), _freq(pairs)
    want = rotary.rotate_qk(q, k, at, freq, interleaved=interleaved)
    code, stream = _hip.dtype_code(dtype), _hip.stream_of(q.device)
    a, b = q.clone(), k.clone()
    turn = (at.data_ptr(), 1, freq.data_ptr(), None, pairs, int(interleaved), n, H, Hkv, D)
    _hip.check(lib.hs_rotary(a.data_ptr(), b.data_ptr(), code, H * D, Hkv * D, *turn, a.data_ptr(),
                             b.data_ptr(), code, stream))
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    a, b = q.clone(), k.clone()
    kc, vc = torch.zeros(2, -(-n // 16), 16, Hkv, D, dtype=dtype, device=DEV)
    table = torch.arange(-(-n // 16), dtype=torch.int32, device=DEV)
    seq = torch.zeros(n, dtype=torch.int32, device=DEV)
    _hip.check(lib.hs_rotary_append(
        a.data_ptr(), b.data_ptr(), v.data_ptr(), code, H * D, Hkv * D, Hkv * D, *turn, a.data_ptr(),
        b.data_ptr(), code, kc.data_ptr(), vc.data_ptr(), code, kc.shape[0], 16, table.data_ptr(), 1,
        table.numel(), at.data_ptr(), seq.data_ptr(), stream))
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    assert torch.equal(kc.view(-1, Hkv, D)[:n], want[1]) and torch.equal(vc.view(-1, Hkv, D)[:n], v)


def test_expanded_and_overlapping_rows():
    from heteroserve.kv import rotary

    q, k, v = _inputs(1, 4, 2, 64, BF16, 5)
    at, freq = torch.arange(6, dtype=torch.int32, device=DEV), _freq(32)
    wide = [x.expand(6, -1, 64) for x in (q, k, v)]
    want = rotary.rotate_qk(*[x.contiguous() for x in wide[:2]], at, freq)
    got = rotary.rotate_qk(*wide[:2], at, freq)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    kc, vc = torch.zeros(2, 1, 16, 2, 64, dtype=BF16, device=DEV)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    got, none = rotary.rotate_append_kv(*wide, at, freq, kc, vc, table, at, torch.zeros_like(at))
    assert torch.equal(got, want[0]) and none is None
    assert torch.equal(kc[0, :6], want[1]) and torch.equal(vc[0, :6], v.expand(6, 2, 64))
    flat = torch.randn(64 * 9, device=DEV).to(BF16)
    slid = flat.as_strided((6, 2, 64), (64, 64, 1))
    want = rotary.rotate_qk(slid.contiguous(), slid.contiguous(), at, freq)
    assert torch.equal(rotary.rotate_qk(slid, slid, at, freq)[0], want[0])
