"""Rows in which one token's probability, or its values, are far from the others': a first
token that takes most of the weight and has next to no values (what sinks are in earnest),
groups of unlike ranges in one record, a token of huge values that counts for nothing.

Scores are made of one product, so that their own error is small: queries are 1 in one place
and keys are multiples of 2^-4, next to the dominant ones, whole numbers `gap` away.  With scale
ln 2 a score is that element, in log2 units.

What is allowed, of the sum of p times a value's size, root mean square over a row's elements
of one group of 32: scores are off by three roundings of the scale and the query (2^-24 each), a
query's last terms (2^-23) and three of their sums, 2^-21.5 of `gap` log2 units, gap 2^-22 of the
probability; probabilities, their products with a step, the terms that these go to the matrix
cores in (2^-22 each at most) and the rounded sums are within 4 2^-22 together, since the
errors of different keys do not depend on one another.  fp32 arithmetic has the same bound.  Lost
second terms or numbers below fp16's normal ones leave 2^-17 and more."""

from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import long_context as lc  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
BS = 16
SCALE = float(np.float32(math.log(2)))
RISING = [3, 70, 140, 141, 270, 340, 500, 640], [12, 30, 41, 52, 70, 99, 110, 124]   # tokens, gaps
RANGES = np.array([1.0, 2.0 ** -8, 2.0 ** -3, 2.0 ** -11, 1.0, 2.0 ** -6, 2.0, 2.0 ** -1])


def _f16(x):
    return np.clip(x, -65504, 65504).astype(np.float16).astype(np.float64)


def _keys(rng, n, Hkv, D, odd, gap):
    """(n, s, lo): elements of [-1/2, 1/2), and `gap` (one, or one for each) in all elements of the
    tokens `odd`."""
    G = D // 32
    num = rng.integers(0, 16, (n, Hkv, G, 32))
    s, lo = np.full((n, Hkv, G), 2.0 ** -4), np.full((n, Hkv, G), -0.5)
    num[odd], lo[odd] = 0, np.reshape(gap, (-1, 1, 1))
    return num, s, lo


def _values(rng, n, Hkv, D, odd, size):
    """(n, s, lo): steps within a factor of 2 of their group's range, `size` times that of the
    tokens `odd`."""
    G = D // 32
    num = rng.integers(0, 16, (n, Hkv, G, 32))
    s = RANGES[:G] / 16 * rng.uniform(0.5, 1, (n, Hkv, G))
    lo = -s * rng.uniform(6, 9, s.shape)
    s[odd] *= size
    lo[odd] *= size
    return num, _f16(s), _f16(lo)


def _held(x, dtype):
    num, s, lo = x
    v = (num * s[..., None] + lo[..., None]).reshape(*num.shape[:2], -1)
    return torch.tensor(v).to(F32).to(dtype)


def _case(kind, n, H, Hkv, D, odd, gap, size, rows, window, sinks, seed):
    """Every row of a batch sees the same tokens; its queries are its own."""
    from heteroserve.model.paged_attn_q4 import paged_attention_q4
    from heteroserve.model.paged_attn_window import paged_attention_window

    rng = np.random.default_rng(seed)
    keys, vals = _keys(rng, n, Hkv, D, odd, gap), _values(rng, n, Hkv, D, odd, size)
    pages = -(-n // BS)
    order = rng.permutation(pages)
    if kind == "q4":
        held = [lc.records(*x, keys=i == 0) for i, x in enumerate((keys, vals))]
        k, v = (lc.values(x, i == 0) for i, x in enumerate(held))
        sizes = [lc.sizes(x, i == 0) for i, x in enumerate(held)]
        flat = torch.zeros(2, pages * BS, Hkv, 5 * D // 8, dtype=torch.uint8)
        held = [torch.tensor(x) for x in held]
        call = paged_attention_q4
    else:
        held = [_held(x, kind) for x in (keys, vals)]
        k, v = (x.double().numpy() for x in held)
        sizes = [np.abs(k), np.abs(v)]
        flat = torch.zeros(2, pages * BS, Hkv, D, dtype=kind)
        call = paged_attention_window
    for i in range(2):
        flat[i, :n] = held[i]
    cache = torch.empty_like(flat).view(2, pages, BS, Hkv, -1)
    cache[:, torch.tensor(order)] = flat.view(2, pages, BS, Hkv, -1)
    cache = cache.to(DEV)
    q = np.zeros((rows, H, D), np.float32)
    q[np.arange(rows)[:, None], np.arange(H), rng.integers(0, D, (rows, H))] = 1
    bt = torch.tensor(order, dtype=torch.int32, device=DEV).expand(rows, pages)
    got = call(torch.tensor(q, device=DEV), cache[0], cache[1], bt,
               torch.full((rows,), n, dtype=torch.int32, device=DEV), SCALE, window, sinks).double().cpu().numpy()
    at = lc.visible(n, window, sinks)
    for b in {0, rows // 2, rows - 1}:
        want, spread, _ = lc.decode(q[b], k[at], v[at], SCALE, sizes[0][at], sizes[1][at])
        err = np.sqrt(((got[b] - want) ** 2).reshape(H, -1, 32).mean(-1))
        most = (np.abs(gap).max() + 4) * 2.0 ** -22 * np.sqrt((spread ** 2).reshape(H, -1, 32).mean(-1))
        assert (err <= most).all(), (b, (err / most).max(-1))


GEOMETRIES = [(8, 2, 128), (16, 1, 128), (4, 4, 64), (8, 4, 256), (2, 2, 32), (8, 1, 64), (9, 1, 256), (6, 1, 128)]


@pytest.mark.parametrize("gap", [8, 14, 20, 30, 60, 110])
@pytest.mark.parametrize("size", [0.0, 2.0 ** -10, 1.0])
@pytest.mark.parametrize("H,Hkv,D", GEOMETRIES)
def test_a_sink_over_4_bits(H, Hkv, D, size, gap):
    """In rows of one part, of several, and behind a window, where rows are whole."""
    for n, rows, window, sinks in ((300, 2, 0, 0), (2500, 2, 0, 0), (3000, 128, 1020, 4)):
        _case("q4", n, H, Hkv, D, [0], gap, size, rows, window, sinks, gap + D)


@pytest.mark.parametrize("where", [0, 150, 299])
@pytest.mark.parametrize("gap", [-14, -22, -30, -40, -60, -110])
@pytest.mark.parametrize("H,Hkv,D", GEOMETRIES)
def test_huge_values_that_count_for_nothing_over_4_bits(H, Hkv, D, gap, where):
    for size in (2.0 ** 10, 2.0 ** 17):
        _case("q4", 300, H, Hkv, D, [where], gap, size, 2, 0, 0, D - gap)


@pytest.mark.parametrize("H,Hkv,D", GEOMETRIES)
def test_maxima_that_rise_over_4_bits(H, Hkv, D):
    """Tokens 40 log2 units above the others here and there, and tokens that each lie 11 to 30 above
    all before them, without values, with small or huge ones: what came before counts less and less."""
    for size in (0.0, 2.0 ** -8):
        _case("q4", 700, H, Hkv, D, [5, 130, 131, 400], 40, size, 2, 0, 0, D)
    for size in (0.0, 2.0 ** -12, 2.0 ** 14):
        _case("q4", 700, H, Hkv, D, *RISING, size, 2, 0, 0, D)


TYPES = [F16, BF16, F32]


@pytest.mark.parametrize("gap", [8, 14, 20, 30, 60, 110])
@pytest.mark.parametrize("size", [0.0, 2.0 ** -10, 1.0])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", GEOMETRIES)
def test_a_sink_of_an_ordinary_cache(H, Hkv, D, dtype, size, gap):
    for n, rows, window, sinks in ((300, 2, 0, 0), (2500, 2, 0, 0), (3000, 128, 1020, 4)):
        _case(dtype, n, H, Hkv, D, [0], gap, size, rows, window, sinks, gap + D)


@pytest.mark.parametrize("where", [0, 150, 299])
@pytest.mark.parametrize("gap", [-14, -22, -30, -40, -60, -110])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", GEOMETRIES)
def test_huge_values_that_count_for_nothing_in_an_ordinary_cache(H, Hkv, D, dtype, gap, where):
    for size in (2.0 ** 10, 2.0 ** 15):
        _case(dtype, 300, H, Hkv, D, [where], gap, size, 2, 0, 0, D - gap)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", GEOMETRIES)
def test_maxima_that_rise_in_an_ordinary_cache(H, Hkv, D, dtype):
    for size in (0.0, 2.0 ** -8):
        _case(dtype, 700, H, Hkv, D, [5, 130, 131, 400], 40, size, 2, 0, 0, D)
    for size in (0.0, 2.0 ** -12, 2.0 ** 14):
        _case(dtype, 700, H, Hkv, D, *RISING, size, 2, 0, 0, D)


@pytest.mark.parametrize("H,Hkv,D", [x for x in GEOMETRIES if x[2] > 32])
@pytest.mark.parametrize("kind", ["q4", F16, BF16, F32])
@pytest.mark.parametrize("n", [3, 300])
def test_one_large_element_of_a_query(H, Hkv, D, kind, n):
    """2^14 times the others, where the keys are next to nothing: 2^-20, in a group of their own.
    Products are off by 2^-22 and what they add up to by as much, so scores by less than 2^-21 of
    their terms' sizes.  Two fp16 terms that end at 2^-27 of the largest element leave 2^-19."""
    from heteroserve.model.paged_attn_q4 import paged_attention_q4
    from heteroserve.model.paged_attn_window import paged_attention_window

    rng = np.random.default_rng(D + H)
    G = D // 32
    num, vals = rng.integers(0, 16, (n, Hkv, G, 32)), _values(rng, n, Hkv, D, [], 0)
    s = np.full((n, Hkv, G), 2.0 ** -4)
    s[..., 1] = 2.0 ** -20
    keys = num, s, -8 * s
    q = rng.normal(size=(2, H, D)).astype(np.float32)
    q[:, np.arange(H), 32 + rng.integers(0, 32, H)] = 2.0 ** 14
    pages = -(-n // BS)
    flat = np.zeros((2, pages * BS, Hkv, 5 * D // 8 if kind == "q4" else D))
    if kind == "q4":
        held = [lc.records(*x, keys=i == 0) for i, x in enumerate((keys, vals))]
        k, v = (lc.values(x, i == 0) for i, x in enumerate(held))
        sizes, call, kept = [lc.sizes(x, i == 0) for i, x in enumerate(held)], paged_attention_q4, torch.uint8
    else:
        held = [_held(x, kind).double().numpy() for x in (keys, vals)]
        k, v = held
        sizes, call, kept = [np.abs(k), np.abs(v)], paged_attention_window, kind
    flat[:, :n] = held
    cache = torch.tensor(flat).to(kept).view(2, pages, BS, Hkv, -1).to(DEV)
    got = call(torch.tensor(q, device=DEV), cache[0], cache[1], torch.arange(pages).expand(2, pages),
               torch.full((2,), n), 0.25, window=0).double().cpu().numpy()
    for b in range(2):
        want, spread, weight = lc.decode(q[b], k, v, 0.25, *sizes)
        err, most = (np.sqrt((x ** 2).reshape(H, -1, 32).mean(-1)) for x in (got[b] - want, spread + weight))
        assert (err <= 2.0 ** -21 * most).all(), (b, (err / most * 2.0 ** 21).max(-1))
