"""Decode through a window over fp32, fp16 and bf16 caches against 64-bit arithmetic.

Tolerances: a dot product of D fp32 terms is off by at most (D + 2) 2^-24 of the sum of
its terms' sizes, a query carried in 16-bit terms by 2^-22 of them, and the base-2 scores
round three times more: (D + 64) 2^-23; a score's error moves the row by p |v - out| times it.
Sums of n products are off by n 2^-24, the probabilities by 2^-22: (n + 64) 2^-23 of the
sum of p |v|.
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


def _tables(lens, BS, rng):
    held = [-(-int(n) // BS) for n in lens]
    blocks = sum(held) + 3
    bt = np.full((len(lens), max(held + [1])), -1, np.int32)
    ids = iter(rng.permutation(blocks))
    for b, k in enumerate(held):
        for j in range(k):
            bt[b, j] = next(ids)
    return bt, blocks


def _attend(lens, H, Hkv, D, BS, dtype, window, sinks, seed, scale=None, q_size=1.0, hide=True):
    """(got, want, tolerance); slots that no row sees hold NaN, and with `hide` table
    entries whose pages no row sees are -1."""
    from heteroserve.model.paged_attn_window import paged_attention_window

    rng = np.random.default_rng(seed)
    scale = D ** -0.5 if scale is None else scale
    bt, blocks = _tables(lens, BS, rng)
    cache = torch.full((2, blocks, BS, Hkv, D), float("nan"), dtype=dtype)
    q = rng.normal(size=(len(lens), H, D)).astype(np.float32) * q_size
    want, tol = np.zeros((2, len(lens), H, D))
    given = bt.copy()
    for b, n in enumerate(lens):
        at = lc.visible(n, window, sinks)
        page, off = bt[b, at // BS], at % BS
        rows = [torch.tensor(rng.normal(size=(len(at), Hkv, D))).to(dtype) for _ in range(2)]
        for i in range(2):
            cache[i, page, off] = rows[i]
        if hide:
            given[b, ~np.isin(np.arange(bt.shape[1]), at // BS)] = -1
        want[b], spread, weight = lc.decode(q[b], _np(rows[0]), _np(rows[1]), scale)
        tol[b] = (D + 64) * 2.0 ** -23 * weight + (len(at) + 64) * 2.0 ** -23 * spread
    cache = cache.to(DEV)
    got = paged_attention_window(torch.tensor(q, device=DEV), cache[0], cache[1], torch.tensor(given),
                                 torch.tensor(lens), scale, window, sinks)
    assert got.dtype is F32 and got.shape == q.shape
    return _np(got), want, tol


def _check(*args, **how):
    got, want, tol = _attend(*args, **how)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / np.maximum(tol, 1e-300)).max()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (31, 33), (64, 0), (100, 7), (1000, 3),
                                          (30, 5000), (0, 9), (2 ** 31, 2 ** 40)])
@pytest.mark.parametrize("H,Hkv,D,BS", [(8, 2, 128, 16), (3, 3, 64, 5)])
def test_windows(dtype, window, sinks, H, Hkv, D, BS):
    """Windows and sinks of any size, in and across pages; lengths on both sides."""
    _check([0, 1, 2, 40, 64, 65, 129, 333], H, Hkv, D, BS, dtype, window, sinks,
           window % 1000 + sinks % 1000 + D)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hkv,D,BS", [(4, 4, 64, 16), (6, 2, 32, 8), (8, 1, 256, 16), (20, 1, 64, 1),
                                        (17, 1, 32, 32), (32, 2, 128, 16), (12, 4, 256, 3), (5, 5, 32, 7)])
def test_geometries(dtype, H, Hkv, D, BS):
    _check([0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 130, 200], H, Hkv, D, BS, dtype, 120, 3, H + D)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 128), (4, 4, 64), (16, 1, 32), (2, 1, 256)])
def test_long_windows_in_parts(dtype, H, Hkv, D):
    _check([5001, 1, 517, 0, 2048], H, Hkv, D, 16, dtype, 2700, 4, D)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_many_rows(dtype):
    lens = [int(x) for x in np.random.default_rng(0).integers(0, 90, 700)]
    _check(lens, 2, 1, 64, 16, dtype, 40, 2, 9)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale,q_size", [(0.0, 1.0), (-0.3, 1.0), (1e-30, 1.0), (0.1, 1e-38), (30.0, 1.0),
                                          (1e30, 1e-30), (1e-20, 1e25)])
def test_scales_and_sizes_of_queries(dtype, scale, q_size):
    _check([5, 70, 200], 4, 2, 64, 16, dtype, 90, 2, 3, scale=scale, q_size=q_size)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hkv", [(4, 4), (8, 2)])
def test_no_window_is_paged_attention(dtype, H, Hkv):
    """Over the whole context, and with a window as long as it, the call is
    paged_attention's."""
    from heteroserve.model.paged_attn import paged_attention
    from heteroserve.model.paged_attn_window import paged_attention_window

    rng = np.random.default_rng(H)
    lens = [300, 17, 1, 0, 128]
    bt, blocks = _tables(lens, 16, rng)
    gen = torch.Generator(DEV).manual_seed(H)
    cache = torch.randn(2, blocks, 16, Hkv, 64, generator=gen, device=DEV).to(dtype)
    q = torch.randn(5, H, 64, generator=gen, device=DEV)
    args = (q, cache[0], cache[1], torch.tensor(bt), torch.tensor(lens), 0.125)
    want = paged_attention(*args)
    for window, sinks in ((0, 0), (300, 0), (10 ** 9, 4), (100, 200)):
        got = paged_attention_window(*args, window, sinks)
        assert (got - want).abs().max() <= 2e-5      # of values around 1: 2^-16 for split operands


def test_a_visible_nan_or_infinity_reaches_its_head_only():
    from heteroserve.model.paged_attn_window import paged_attention_window

    for dtype in (F32, F16, BF16):
        cache = torch.randn(2, 8, 16, 2, 64, device=DEV).to(dtype)
        cache[1, 2, 3, 0, 5] = float("nan")
        cache[0, 4, 3, 1, 5] = float("inf")
        q = torch.randn(1, 4, 64, device=DEV)
        q[..., 5] = q[..., 5].abs() + 0.1        # a score of +infinity
        bt = torch.arange(8)[None]
        got = paged_attention_window(q, cache[0], cache[1], bt, torch.tensor([128]), 0.1, 0)
        bad = ~torch.isfinite(got)
        assert bad[0, :2, 5].all() and bad[0, :2].sum() == 2 and bad[0, 2:].all()
        # keys 0 .. 34, then 68 ..: the NaN is key 35, the infinity key 67
        got = paged_attention_window(q, cache[0], cache[1], bt, torch.tensor([128]), 0.1, 60, 35)
        assert torch.isfinite(got).all()


def test_rows_near_the_lowest_number():
    """Scores far below zero, all of them: a softmax like any other."""
    from heteroserve.model.paged_attn_window import paged_attention_window

    cache = torch.full((2, 4, 16, 1, 32), 1.0, device=DEV)
    cache[1] = torch.randn(4, 16, 1, 32, device=DEV)
    q = torch.full((1, 1, 32), -2.0 ** 62, device=DEV)
    got = paged_attention_window(q, cache[0], cache[1], torch.arange(4)[None], torch.tensor([64]), 2.0 ** 59,
                                 40, 3)
    want = cache[1].view(64, 32)[lc.visible(64, 40, 3)].mean(0)
    assert (got[0, 0] - want).abs().max() < 1e-5


def test_refusals():
    from heteroserve.model.paged_attn_window import paged_attention_window

    kc = torch.zeros(4, 16, 2, 64, device=DEV)
    q, c = torch.zeros(2, 4, 64, device=DEV), torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(2, 2, dtype=torch.int32)

    def no(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            paged_attention_window(*args, **kw)

    no("float32", q.half(), kc, kc, t, c, 0.1, 4)
    no("head_dim", q[..., :32], kc, kc, t, c, 0.1, 4)
    no("q must be", q[0], kc, kc, t, c, 0.1, 4)
    no("on CUDA", q.cpu(), kc, kc, t, c, 0.1, 4)
    no("on CUDA", q, kc.cpu(), kc.cpu(), t, c, 0.1, 4)
    no("shape", q, kc, kc[:2], t, c, 0.1, 4)
    no("dtype", q, kc, kc.half(), t, c, 0.1, 4)
    no("dtype", q, kc.to(torch.uint8), kc.to(torch.uint8), t, c, 0.1, 4)
    no("max_blocks", q, kc, kc, t[:1], c, 0.1, 4)
    no("integers", q, kc, kc, t.float(), c, 0.1, 4)
    no("one entry", q, kc, kc, t, c[:1], 0.1, 4)
    no("divisible", q[:, :3].contiguous(), kc, kc, t, c, 0.1, 4)
    no("negative", q, kc, kc, t, c, 0.1, -1)
    no("negative", q, kc, kc, t, c, 0.1, 4, sinks=-1)
    no("finite", q, kc, kc, t, c, float("inf"), 4)
    with pytest.raises(TypeError):
        paged_attention_window(q, kc, kc, t, c, 0.1, 1.5)
