"""The 4-bit cache's writes, reads and attention against 64-bit arithmetic.

What is written is the definition's to the bit (the oracle rounds the same exact
quotients), so caches are compared byte for byte.  What is read is n s + lo, exact in
fp32 but for one rounding (n s has 15 bits), then rounded to the output's type.

Attention.  An fp32 dot product of D terms is off by at most (D + 2) 2^-24 of the sum of
its terms' sizes, |q| (n s + |lo|) scale; query and probabilities are carried in two fp16
terms of 22 bits (2^-22), and the base-2 scores round three times more: (D + 64) 2^-23 in
all, and a score's error moves the row by p |v - out| times it.  A sum of n probabilities
or products is off by n 2^-24, the probabilities themselves by 2^-22: (n + 64) 2^-23 of
the sum of p (n s + |lo|).
"""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import long_context as lc  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _np(x):
    return x.double().cpu().numpy()


def _tables(lens, BS, rng, width=None):
    """(block tables [B, MB] int32, number of blocks): pages in no order."""
    held = [-(-int(n) // BS) for n in lens]
    blocks = sum(held) + 3
    bt = np.full((len(lens), width or max(held + [1])), -1, np.int32)
    ids = iter(rng.permutation(blocks))
    for b, k in enumerate(held):
        for j in range(k):
            bt[b, j] = next(ids)
    return bt, blocks


def _pool(blocks, BS, Hkv, D, fill=0):
    from heteroserve.kv import quant

    pool = quant.empty_pool_q4(1, blocks, BS, Hkv, D, device=DEV)
    return pool.fill_(fill)


def _rows(rng, n, Hkv, D, dtype):
    """k, v as slices of fused rows, with an offset for each channel."""
    x = rng.normal(size=(n, 2 * Hkv * D)) + rng.normal(size=2 * Hkv * D) * 2
    x = torch.tensor(x, device=DEV).to(dtype)
    return [y.view(n, Hkv, D) for y in x.split(Hkv * D, 1)]


def _placed(cache, bt, BS, seq, at):
    """Rows (block, offset) of a cache [NB, BS, ...] as an array."""
    return cache.cpu().numpy()[bt[seq, at // BS], at % BS]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,Hkv,D,BS", [(1, 2, 64, 16), (7, 8, 128, 16), (40, 1, 32, 5), (33, 3, 256, 8),
                                        (1030, 2, 32, 16)])
def test_append_and_read(dtype, n, Hkv, D, BS):
    """To the byte, and the rest of the cache as it was; rows that name no slot are not
    written and read as zeros."""
    from heteroserve.kv import quant

    rng = np.random.default_rng(n + D)
    seq = rng.integers(0, 3, n)
    at = np.empty(n, np.int64)
    for b in range(3):
        at[seq == b] = rng.permutation(max(1, int((seq == b).sum()) + 9))[:int((seq == b).sum())]
    bt, blocks = _tables([n + 9] * 3, BS, rng)
    seq, at = seq.astype(np.int32), at.astype(np.int32)
    bad = n > 5
    if bad:
        seq[0], at[1], at[2], seq[3] = 3, -1, bt.shape[1] * BS, -1
        bt[seq[4], at[4] // BS] = -1
    pool = _pool(blocks, BS, Hkv, D, fill=0xA5)
    before = pool.cpu().numpy().copy()
    k, v = _rows(rng, n, Hkv, D, dtype)
    args = (pool[0, 0], pool[0, 1], torch.tensor(bt), torch.tensor(at))
    quant.append_kv_q4(*args, k, v, seq_ids=torch.tensor(seq))
    ok = np.array([0 <= s < 3 and 0 <= p < bt.shape[1] * BS and bt[s, p // BS] >= 0 for s, p in zip(seq, at)])
    assert ok.all() != bad
    want = before.copy()
    for i, x in enumerate((k, v)):
        rec = lc.records(*lc.quantise(_np(x)), keys=i == 0)
        want[0, i][bt[seq[ok], at[ok] // BS], at[ok] % BS] = rec[ok]
    assert np.array_equal(pool.cpu().numpy(), want)
    for out in (F32, F16, BF16):
        got = quant.read_kv_q4(*args, seq_ids=torch.tensor(seq), dtype=out)
        for i, x in enumerate(got):
            assert x.shape == (n, Hkv, D) and x.dtype is out
            exact = np.zeros((n, Hkv, D))
            exact[ok] = lc.values(_placed(pool[0, i], bt, BS, seq[ok], at[ok]), i == 0)
            once = torch.tensor(exact).to(F32)
            assert torch.equal(x.cpu(), once.to(out))


@pytest.mark.parametrize("how", ["odd address", "element strides", "heads apart", "flat", "one row over"])
def test_append_of_rows_of_any_layout(how):
    from heteroserve.kv import quant

    rng = np.random.default_rng(5)
    n, Hkv, D, BS = 6, 2, 64, 16
    k, v = (x.contiguous() for x in _rows(rng, n, Hkv, D, BF16))
    want = _pool(3, BS, Hkv, D)
    at = torch.arange(n, dtype=torch.int32)
    bt = torch.tensor([[1, -1]], dtype=torch.int32)
    seq = torch.zeros(n, dtype=torch.int32)
    quant.append_kv_q4(want[0, 0], want[0, 1], bt, at, k, v, seq_ids=seq)
    if how == "odd address":
        wide = torch.zeros(n, Hkv * D + 3, dtype=BF16, device=DEV)
        wide[:, 1:-2] = k.view(n, -1)
        k = wide[:, 1:-2].view(n, Hkv, D)
    elif how == "element strides":
        k = k.repeat_interleave(2, -1)[..., ::2]
    elif how == "heads apart":
        k = k.transpose(0, 1).contiguous().transpose(0, 1)
    elif how == "flat":
        k = k.view(n, Hkv * D)
    else:
        k, v = k[:1].expand(n, Hkv, D), v[:1].expand(n, Hkv, D)
        want.zero_()
        quant.append_kv_q4(want[0, 0], want[0, 1], bt, at, k.contiguous(), v.contiguous(), seq_ids=seq)
    got = _pool(3, BS, Hkv, D)
    quant.append_kv_q4(got[0, 0], got[0, 1], bt, at, k, v, seq_ids=seq)
    assert torch.equal(got, want)


def test_values_at_borders_and_beyond_fp16():
    """Quotients half way between two numbers, groups of one value, of zeros, of fp16's
    subnormals, infinities, and NaN, which takes its group of 32 and no other."""
    from heteroserve.kv import quant

    rng = np.random.default_rng(1)
    D, x = 128, []
    ties = np.concatenate([np.arange(16), np.arange(15) + 0.5, [7.25]])
    for scale in (1.0, 2.0 ** -7, 3 * 2.0 ** -20, 2.0 ** 11, 0.1):
        for off in (0.0, 1.0, -12.0):
            x.append(np.concatenate([rng.permutation(ties + off) * scale for _ in range(4)]))
    x.append(np.repeat([0.0, 0.1, -65504.0, 1e-6], 32))
    x.append(np.repeat([1e30, -1e30, 65519.0, 2.0 ** -25], 32))
    for odd in (np.inf, -np.inf, np.nan):
        y = rng.normal(size=D)
        y[40] = odd
        x.append(y)
    x.append(rng.normal(size=D) * 1e38)
    x.append(rng.normal(size=D) * 1e-7)
    x = torch.tensor(np.array(x), dtype=F32, device=DEV)[:, None]
    n = x.shape[0]
    pool = _pool(2, 64, 1, D)
    args = (pool[0, 0], pool[0, 1], torch.tensor([[1]]), torch.arange(n))
    seq = torch.zeros(n, dtype=torch.int64)
    quant.append_kv_q4(*args, x, -x, seq_ids=seq)
    got = quant.read_kv_q4(*args, seq_ids=seq, dtype=F32)
    for i, y in enumerate((x, -x)):
        step, s, lo = lc.quantise(_np(y))
        want = torch.tensor((step * s[..., None] + lo[..., None]).reshape(y.shape)).to(F32)
        assert torch.equal(torch.nan_to_num(got[i].cpu(), nan=12345.0), torch.nan_to_num(want, nan=12345.0))
    nan = torch.isnan(got[0][-3]).view(4, 32).all(1).tolist()
    assert nan == [False, True, False, False] and not torch.isnan(got[0][:-3]).any()


def _attend(lens, H, Hkv, D, BS, window, sinks, seed, scale=None, junk=True, width=None, q_size=1.0):
    """(got, want, tolerance): random records in the visible slots, junk (NaN steps among
    it) everywhere else."""
    from heteroserve.model.paged_attn_q4 import paged_attention_q4

    rng = np.random.default_rng(seed)
    scale = D ** -0.5 if scale is None else scale
    bt, blocks = _tables(lens, BS, rng, width)
    shape = (2, blocks, BS, Hkv, 5 * D // 8)
    rec = np.full(shape, 0xff, np.uint8) if junk else np.zeros(shape, np.uint8)   # fp16 NaN
    q = rng.normal(size=(len(lens), H, D)).astype(np.float32) * q_size
    want, tol = np.zeros((2, len(lens), H, D))
    _attend.spread = np.zeros_like(want)
    for b, n in enumerate(lens):
        at = lc.visible(n, window, sinks)
        page, off = bt[b, at // BS], at % BS
        kv = []
        for i in range(2):
            x = rng.normal(size=(len(at), Hkv, D)) + 2 * rng.normal(size=(Hkv, D)) * (i == 0)
            kv.append(lc.records(*lc.quantise(x), keys=i == 0))
            rec[i, page, off] = kv[-1]
        out, spread, weight = lc.decode(q[b], lc.values(kv[0], True), lc.values(kv[1], False), scale,
                                        lc.sizes(kv[0], True), lc.sizes(kv[1], False))
        want[b], _attend.spread[b] = out, spread
        tol[b] = (D + 64) * 2.0 ** -23 * weight + (len(at) + 64) * 2.0 ** -23 * spread
    cache = torch.tensor(rec, device=DEV)
    got = paged_attention_q4(torch.tensor(q, device=DEV), cache[0], cache[1], torch.tensor(bt),
                             torch.tensor(lens), scale, window=window, sinks=sinks)
    assert got.dtype is F32 and got.shape == q.shape
    return _np(got), want, tol


def _check(*args, **how):
    got, want, tol = _attend(*args, **how)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()


@pytest.mark.parametrize("H,Hkv,D,BS", [(4, 4, 64, 16), (8, 2, 128, 16), (6, 2, 32, 8), (8, 1, 256, 16),
                                        (3, 3, 128, 5), (20, 1, 64, 1), (17, 1, 32, 32), (32, 2, 128, 16),
                                        (12, 4, 256, 3), (5, 5, 32, 16)])
def test_attention(H, Hkv, D, BS):
    """Lengths of zero, one, around tiles and parts; groups of every size."""
    _check([0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 130, 200], H, Hkv, D, BS, 0, 0, H + D)


@pytest.mark.parametrize("H,Hkv,D", [(5, 1, 128), (14, 2, 128), (9, 1, 128), (9, 1, 256), (20, 1, 256),
                                     (7, 1, 256), (6, 2, 256), (5, 1, 64), (10, 5, 64), (33, 1, 128)])
def test_groups_of_every_size(H, Hkv, D):
    """Columns of the products by heads and groups in every split, not all of them used."""
    _check([0, 3, 64, 100, 333], H, Hkv, D, 16, 0, 0, H + D)
    _check([0, 3, 64, 100, 333], H, Hkv, D, 16, 90, 2, H + D)


@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 128), (4, 4, 64), (16, 1, 32), (2, 1, 256), (16, 2, 128),
                                     (12, 1, 64), (4, 1, 256)])
def test_rounding_errors_average_out(H, Hkv, D):
    """The bounds above are of the worst case, which lost second terms would pass.  For 300
    keys with errors that do not depend on one another: probabilities off by up to 2^-20 (a
    score of up to 16 is rounded) and products by 2^-22 leave 2^-24 of the sum of their sizes,
    sums of 10 chunks' products rounded to 2^-24 about 2^-23; a second term that is missing
    (2^-12 of each product) leaves 2^-17, one that is wrong once in a thousand 2^-21."""
    got, want, _ = _attend([300] * 24, H, Hkv, D, 16, 0, 0, D)
    spread = _attend.spread
    assert np.sqrt(np.mean((got - want) ** 2)) <= 2.0 ** -22 * np.sqrt(np.mean(spread ** 2))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (63, 1), (64, 0), (65, 64), (100, 7),
                                          (1000, 3), (30, 5000), (2 ** 31, 2 ** 40)])
@pytest.mark.parametrize("H,Hkv,D,BS", [(8, 2, 128, 16), (3, 3, 64, 5)])
def test_attention_through_a_window(H, Hkv, D, BS, window, sinks):
    _check([0, 1, 40, 64, 65, 129, 333], H, Hkv, D, BS, window, sinks, window % 1000 + sinks % 1000 + D)


@pytest.mark.parametrize("H,Hkv,D,window", [(8, 2, 128, 0), (4, 4, 64, 0), (16, 1, 32, 700), (2, 1, 256, 0)])
def test_long_rows_in_parts(H, Hkv, D, window):
    _check([3001, 1, 517, 0, 2048], H, Hkv, D, 16, window, 4 if window else 0, D)


def test_many_rows():
    """More rows than CUs, most of them short."""
    lens = [int(x) for x in np.random.default_rng(0).integers(0, 90, 700)]
    _check(lens, 2, 1, 64, 16, 0, 0, 9)


@pytest.mark.parametrize("scale,q_size", [(0.0, 1.0), (-0.3, 1.0), (1e-30, 1.0), (0.1, 1e-38), (30.0, 1.0),
                                          (1e30, 1e-30), (1e-20, 1e25)])
def test_scales_and_sizes_of_queries(scale, q_size):
    _check([5, 70, 200], 4, 2, 64, 16, 0, 0, 3, scale=scale, q_size=q_size)


@pytest.mark.parametrize("v_size", [1e-6, 1e-3, 1e3, 6e4])
def test_values_of_every_size(v_size):
    """Values whose steps differ by powers of two from token to token, small ones first and
    last: what is lost is relative to the row's own values."""
    from heteroserve.model.paged_attn_q4 import paged_attention_q4

    rng = np.random.default_rng(2)
    n, H, Hkv, D, BS = 300, 4, 2, 128, 16
    size = v_size * 2.0 ** -np.abs(np.arange(n) - n // 2).clip(max=20)[:, None, None]
    k = lc.records(*lc.quantise(rng.normal(size=(n, Hkv, D))), keys=True)
    v = lc.records(*lc.quantise(rng.normal(size=(n, Hkv, D)) * size), keys=False)
    for rows in (np.arange(n), np.arange(n // 2), np.arange(20)):
        m = len(rows)
        cache = np.zeros((2, -(-n // BS), BS, Hkv, 5 * D // 8), np.uint8)
        cache[0].reshape(-1, Hkv, 5 * D // 8)[:m] = k[rows]
        cache[1].reshape(-1, Hkv, 5 * D // 8)[:m] = v[rows]
        q = rng.normal(size=(1, H, D)).astype(np.float32)
        want, spread, weight = lc.decode(q[0], lc.values(k[rows], True), lc.values(v[rows], False), D ** -0.5,
                                         lc.sizes(k[rows], True), lc.sizes(v[rows], False))
        cache = torch.tensor(cache, device=DEV)
        got = paged_attention_q4(torch.tensor(q, device=DEV), cache[0], cache[1],
                                 torch.arange(cache.shape[1])[None], torch.tensor([m]), D ** -0.5)
        # steps of 2^-25 of the probabilities' fp16 terms next to the largest step's: 2^-24 of it
        tol = (D + 64) * 2.0 ** -23 * weight + (m + 64) * 2.0 ** -23 * spread
        assert (np.abs(_np(got)[0] - want) <= tol).all(), (m, (np.abs(_np(got)[0] - want) / tol).max())


def test_a_peaked_row():
    """One key far above the others, first, last or in between: its value comes back."""
    from heteroserve.kv import quant
    from heteroserve.model.paged_attn_q4 import paged_attention_q4

    D, n = 64, 150
    for peak in (0, 70, n - 1):
        k = torch.zeros(n, 1, D, device=DEV)
        k[peak] = 50.0
        v = torch.randn(n, 1, D, generator=torch.Generator(DEV).manual_seed(peak), device=DEV)
        pool = _pool(10, 16, 1, D)
        bt, at = torch.arange(10, dtype=torch.int32)[None], torch.arange(n)
        quant.append_kv_q4(pool[0, 0], pool[0, 1], bt, at, k, v, seq_ids=torch.zeros(n, dtype=torch.int32))
        held = quant.read_kv_q4(pool[0, 0], pool[0, 1], bt, at[peak:peak + 1], seq_ids=torch.tensor([0]),
                                dtype=F32)[1]
        got = paged_attention_q4(torch.ones(1, 2, D, device=DEV), pool[0, 0], pool[0, 1], bt,
                                 torch.tensor([n]), 1.0)
        tol = 2.0 ** -20 * (held.abs() + 8)       # the value's rounding, n s and lo apart
        assert ((got[0] - held[0]).abs() <= tol[0]).all()


def test_a_visible_nan_reaches_its_row_and_group_only():
    from heteroserve.model.paged_attn_q4 import paged_attention_q4

    rng = np.random.default_rng(4)
    H, Hkv, D, n = 4, 2, 128, 100
    x = rng.normal(size=(2, n, Hkv, D))
    x[1, 30, 0, 70] = np.nan                 # a value: elements 64 .. 95 of KV head 0's rows
    rec = [lc.records(*lc.quantise(x[i]), keys=i == 0) for i in range(2)]
    cache = torch.tensor(np.stack(rec).reshape(2, 10, 10, Hkv, -1), device=DEV)
    q = torch.randn(2, H, D, device=DEV)
    bt = torch.arange(10, dtype=torch.int32).repeat(2, 1)
    args = (cache[0], cache[1], bt)
    nan = torch.isnan(paged_attention_q4(q, *args, torch.tensor([100, 30]), 0.1))
    assert not nan[1].any() and not nan[0, 2:].any()
    assert nan[0, :2].view(2, 4, 32).all(-1).tolist() == [[False, False, True, False]] * 2
    assert not nan[0, :2, :64].any() and not nan[0, :2, 96:].any()
    # out of the window, behind the sinks
    assert not torch.isnan(paged_attention_q4(q, *args, torch.tensor([100, 30]), 0.1, window=69,
                                              sinks=30)).any()
    x[0, 30, 0, 3] = np.nan                  # a key: all of its KV head's rows
    cache[0] = torch.tensor(lc.records(*lc.quantise(x[0]), keys=True).reshape(10, 10, Hkv, -1))
    nan = torch.isnan(paged_attention_q4(q, *args, torch.tensor([100, 30]), 0.1))
    assert nan[0, :2].all() and not nan[0, 2:].any() and not nan[1].any()


def test_tables_of_any_content():
    """Entries outside the pool are read as block 0, context lengths past the table end at
    it, negative ones are none."""
    from heteroserve.model.paged_attn_q4 import paged_attention_q4

    rng = np.random.default_rng(6)
    H, Hkv, D, BS = 2, 1, 64, 16
    rec = np.stack([lc.records(*lc.quantise(rng.normal(size=(4, BS, Hkv, D))), keys=i == 0) for i in (0, 1)])
    cache = torch.tensor(rec, device=DEV)
    q = torch.randn(4, H, D, device=DEV)
    bt = np.array([[1, 9, -1], [2 ** 31 - 1, 3, -2 ** 31], [2, 3, 1], [1, 2, 3]], np.int64)
    ctx = np.array([40, 48, 10 ** 6, -5])
    got = _np(paged_attention_q4(q, cache[0], cache[1], torch.tensor(bt), torch.tensor(ctx), 0.2))
    for b in range(4):
        at = np.arange(max(0, min(ctx[b], 48)))
        page = np.where((bt[b] < 0) | (bt[b] >= 4), 0, bt[b])[at // BS]
        k, v = (lc.values(rec[i][page, at % BS], i == 0) for i in (0, 1))
        want, spread, weight = lc.decode(_np(q)[b], k, v, 0.2)
        assert (np.abs(got[b] - want) <= 1e-4 * (spread + weight)).all()
    # far lengths of 64 bits, and no rows at all
    far = paged_attention_q4(q[:1], cache[0], cache[1], torch.tensor(bt[2:3]), torch.tensor([2 ** 40]), 0.2)
    assert torch.equal(far, paged_attention_q4(q[:1], cache[0], cache[1], torch.tensor(bt[2:3]),
                                               torch.tensor([48]), 0.2))
    assert paged_attention_q4(q[:0], cache[0], cache[1], torch.tensor(bt[:0]), torch.tensor(ctx[:0]),
                              0.2).shape == (0, H, D)


def test_refusals():
    from heteroserve.kv import quant
    from heteroserve.model.paged_attn_q4 import paged_attention_q4

    pool = _pool(4, 16, 2, 64)
    kc, vc = pool[0, 0], pool[0, 1]
    q, c = torch.zeros(2, 4, 64, device=DEV), torch.zeros(2, dtype=torch.int32)
    k, t = torch.zeros(2, 2, 64, device=DEV), torch.zeros(2, 2, dtype=torch.int32)

    def no(match, call, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            call(*args, **kw)

    for call, more in ((quant.append_kv_q4, (k, k)), (quant.read_kv_q4, ())):
        no("uint8", call, kc.to(torch.int8), vc.to(torch.int8), t, c, *more)
        no("shape|must be", call, kc, vc[:1], t, c, *more)
        no("records of", call, kc[..., :32], vc[..., :32], t, c, *more)
        no("contiguous", call, kc.transpose(0, 1), vc.transpose(0, 1), t, c, *more)
        no("on CUDA", call, kc.cpu(), vc.cpu(), t, c, *more)
        no("max_blocks", call, kc, vc, t[0], c, *more)
        no("integers", call, kc, vc, t, c.float(), *more)
        no("integers", call, kc, vc, t, c.bool(), *more)
        no("sequence ids", call, kc, vc, t, c, *more, seq_ids=c[:1])
        no("more rows than tables", call, kc, vc, t[:1], c, *more)
    no("positions", quant.append_kv_q4, kc, vc, t, c[:1], k, k)
    no("rows must be", quant.append_kv_q4, kc, vc, t, c, k[:, :1], k)
    no("rows must be", quant.append_kv_q4, kc, vc, t, c, k.view(2, 64, 2), k)
    no("count and dtype", quant.append_kv_q4, kc, vc, t, c, k, k[:1])
    no("count and dtype", quant.append_kv_q4, kc, vc, t, c, k, k.half())
    no("dtype", quant.append_kv_q4, kc, vc, t, c, k.double(), k.double())
    no("dtype", quant.read_kv_q4, kc, vc, t, c, dtype=torch.int32)
    no("same device", quant.append_kv_q4, kc, vc, t, c, k.cpu(), k.cpu())
    no("float32", paged_attention_q4, q.half(), kc, vc, t, c, 0.1)
    no("q must be", paged_attention_q4, q[..., :32], kc, vc, t, c, 0.1)
    no("q must be", paged_attention_q4, q[0], kc, vc, t, c, 0.1)
    no("same device", paged_attention_q4, q.cpu(), kc, vc, t, c, 0.1)
    no("max_blocks", paged_attention_q4, q, kc, vc, t[:1], c, 0.1)
    no("one entry", paged_attention_q4, q, kc, vc, t, c[:1], 0.1)
    no("divisible", paged_attention_q4, q[:, :3].contiguous(), kc, vc, t, c, 0.1)
    no("negative", paged_attention_q4, q, kc, vc, t, c, 0.1, window=-1)
    no("negative", paged_attention_q4, q, kc, vc, t, c, 0.1, sinks=-1)
    no("finite", paged_attention_q4, q, kc, vc, t, c, float("nan"))
    with pytest.raises(TypeError):
        paged_attention_q4(q, kc, vc, t, c, 0.1, window=1.5)


def test_pages_of_the_pool_move_as_bytes():
    """Copies, forks, compaction and the migration payload take the 4-bit pool as it is."""
    from heteroserve.kv import pack, pages, quant
    from heteroserve.model.paged_attn_q4 import paged_attention_q4

    rng = np.random.default_rng(8)
    L, NB, BS, Hkv, D, n = 2, 12, 16, 2, 64, 41
    pool = quant.empty_pool_q4(L, NB, BS, Hkv, D, device=DEV)
    tables = torch.tensor([[9, 4, 11], [-1, -1, -1]], dtype=torch.int32, device=DEV)
    ctx = torch.tensor([n, 0], dtype=torch.int32, device=DEV)
    refs = torch.zeros(NB, dtype=torch.int32, device=DEV)
    refs[[9, 4, 11]] = 1
    for layer in range(L):
        k, v = _rows(rng, n, Hkv, D, F16)
        quant.append_kv_q4(pool[layer, 0], pool[layer, 1], tables, torch.arange(n), k, v,
                           seq_ids=torch.zeros(n, dtype=torch.int32))
    q = torch.randn(1, 4, D, device=DEV)

    def attend(p, t, length):
        return [paged_attention_q4(q, p[layer, 0], p[layer, 1], t, length, 0.1) for layer in range(L)]

    want = attend(pool, tables[:1], ctx[:1])
    fresh = pages.find_free_blocks(refs, 1)
    assert pages.fork_blocks(pool, tables, ctx, refs, [0], [1], fresh).tolist() == [1]
    for a, b in zip(want, attend(pool, tables[1:], ctx[1:])):
        assert torch.equal(a, b)
    pages.compact_blocks(pool, tables, refs)
    for row in (slice(0, 1), slice(1, 2)):
        for a, b in zip(want, attend(pool, tables[row], ctx[row])):
            assert torch.equal(a, b)
    payload = pack.export_blocks_device(pool, tables[0].tolist())
    other = quant.empty_pool_q4(L, NB, BS, Hkv, D, device=DEV)
    pack.write_blocks_device(other, [2, 0, 7], payload)
    for a, b in zip(want, attend(other, torch.tensor([[2, 0, 7]]), ctx[:1])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 64), (8, 2, 128), (16, 2, 128), (6, 3, 256), (3, 1, 32)])
def test_records_of_any_finite_numbers(H, Hkv, D):
    """Steps and lowest values up to fp16's largest, which no append writes together: values
    of up to 16 times that, in some chunks of a row and not in others.

    The sizes that errors are relative to are those of what is added: n s + lo is (n - 8) s and
    lo + 8 s, at most 8 s + |lo + 8 s|, of keys (n - 8) s, lo and 8 s, at most 16 s + |lo|, where the
    tests above, whose elements' n differ from key to key, do with n s + |lo| (an element of 0 in a group
    of large ones is off by 2^-22 of their step, half of which it may be off by itself)."""
    from heteroserve.model.paged_attn_q4 import paged_attention_q4

    rng = np.random.default_rng(D + H)
    n, BS, G = 400, 16, D // 32
    rec = rng.integers(0, 256, (2, 32, BS, Hkv, 5 * D // 8)).astype(np.uint8)
    step = (rng.random((2, 32, BS, Hkv, G)) * 65504).astype(np.float16)
    low = (rng.uniform(-1, 1, step.shape) * 65504).astype(np.float16)
    for x in (step, low):                    # blocks of ordinary sizes between
        x[:, 8:20] = (x[:, 8:20].astype(np.float64) * 1e-4).astype(np.float16)
    rec[..., D // 2:] = np.concatenate([step, low], -1).view(np.uint8)
    lens, bt = [n, 130, 17], np.stack([rng.permutation(32)[:25] for _ in range(3)])
    q = (rng.normal(size=(3, H, D)) * 1e-6).astype(np.float32)
    cache = torch.tensor(rec, device=DEV)
    got = _np(paged_attention_q4(torch.tensor(q, device=DEV), cache[0], cache[1], torch.tensor(bt),
                                 torch.tensor(lens), 0.1))
    for b, m in enumerate(lens):
        at = np.arange(m)
        k, v = (rec[i][bt[b, at // BS], at % BS] for i in (0, 1))
        (ks, kl), (vs, vl) = (np.split(np.repeat(np.ascontiguousarray(x[..., D // 2:]).view(np.float16)
                                                 .astype(np.float64), 32, -1), 2, -1) for x in (k, v))
        want, spread, weight = lc.decode(q[b], lc.values(k, True), lc.values(v, False), 0.1,
                                         16 * ks + np.abs(kl), 8 * vs + np.abs(vl + 8 * vs))
        tol = (D + 64) * 2.0 ** -23 * weight + (m + 64) * 2.0 ** -23 * spread
        assert (np.abs(got[b] - want) <= tol).all(), (b, (np.abs(got[b] - want) / tol).max())
