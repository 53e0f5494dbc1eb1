"""Whole prompts at the ends of the number range: the largest values, scales and scores,
and probabilities far below the largest one.  The helpers' tolerances are those of
test_prompt_gpu.py; what differs is derived at each test."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def _batches():
    """(lens, H, Hkv) that take a wave each, split keys, 64-row and 128-row workgroups."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    many = -(-cus // 16)
    return [([1, 40, 64, 3], 2, 1), ([300, 7], 2, 2), ([130, 20, 70] * many, 16, 2),
            ([200] * (2 * many), 16, 2)]


def _call(q, k, v, cu, lens, scale):
    from heteroserve.model.prompt_attn import prompt_attention

    return prompt_attention(q, k, v, torch.tensor(cu, device=DEV), max(lens), scale)


def _cu(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [0.0, 1e-40, -3e-39, 2e-38])
@pytest.mark.parametrize("which", range(4))
def test_least_scales_and_largest_scores(dtype, scale, which):
    """q . k of up to 1e38 under a scale of 0 or of fp32's subnormals.  Tolerance of
    test_prompt_gpu.py with the sums |q k| themselves, and what a step of subnormals (of
    scale times log2(e), or in the place of 0) makes of a score: 2^-149 S powers of 2."""
    lens, H, Hkv = _batches()[which]
    cu, n, D = _cu(lens), sum(lens), 64
    gen = torch.Generator(device=DEV).manual_seed(which)
    big = 2.0 ** 60
    q = (torch.randn(n, H, D, generator=gen, device=DEV).clamp(-3, 3) * big).to(dtype)
    k = (torch.randn(n, Hkv, D, generator=gen, device=DEV).clamp(-3, 3) * big).to(dtype)
    v = torch.randn(n, Hkv, D, generator=gen, device=DEV).to(dtype)
    got = _call(q, k, v, cu, lens, scale).double()
    held = float(np.float32(scale))
    half = 0.0 if dtype is F32 else torch.finfo(dtype).eps / 2
    worst = 0.0
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        later = torch.ones(b - a, b - a, dtype=torch.bool, device=DEV).triu(1)
        for h in range(H):
            x, y = q[a:b, h].double(), k[a:b, h // (H // Hkv)].double()
            z = v[a:b, h // (H // Hkv)].double()
            s = torch.mm(x, y.t().contiguous()) * held
            S = torch.mm(x.abs(), y.abs().t().contiguous()).max().item()
            assert torch.mm(x, y.t().contiguous()).abs().max().item() < 3.4e38 and S * abs(held) < 60
            p = torch.softmax(s.masked_fill(later, -np.inf), -1)
            want, spread = torch.mm(p, z), torch.mm(p, z.abs())
            rel = 2 * (2 * (D + 4) * U * S * abs(held) + 4 * U + (b - a) * U + 2.0 ** -149 * S)
            tol = rel * spread + half * spread * (1 + rel)
            tol = tol + half * (want.abs() + tol)
            worst = max(worst, ((got[a:b, h] - want).abs() - tol).max().item())
    assert worst <= 0.0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("which", range(4))
def test_lowest_scores(dtype, which):
    """Every score is the same and near fp32's lowest number, in powers of 2: a row's mean.
    (One product a score, and no rounding in the rest: a power of 2 as key.)"""
    lens, H, Hkv = _batches()[which]
    cu, n, D = _cu(lens), sum(lens), 64
    gen = torch.Generator(device=DEV).manual_seed(which)
    at = 1.5 * 2.0 ** 6 if dtype is F16 else 1.5 * 2.0 ** 62
    q, k = (torch.zeros(n, h, D, dtype=dtype, device=DEV) for h in (H, Hkv))
    q[..., 3], k[..., 3] = -at, at
    v = torch.randn(n, Hkv, D, generator=gen, device=DEV).to(dtype)
    scale = 3.2e38 / 1.4426950408889634 / (at * at)
    got = _call(q, k, v, cu, lens, scale).double()
    assert torch.isfinite(got).all()
    half = 0.0 if dtype is F32 else torch.finfo(dtype).eps / 2
    rel = 2 * (max(lens) + 4) * U
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        count = torch.arange(1, b - a + 1, device=DEV, dtype=torch.float64)[:, None, None]
        want = (v[a:b].double().cumsum(0) / count).repeat_interleave(H // Hkv, 1)
        spread = (v[a:b].double().abs().cumsum(0) / count).repeat_interleave(H // Hkv, 1)
        tol = rel * spread + half * spread
        tol = tol + half * (want.abs() + tol) + (2.0 ** -25 if dtype is F16 else 0.0)
        assert ((got[a:b] - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens,H,Hkv", [([60, 33], 2, 1), ([4097, 200], 2, 1), ([40, 700, 1] * 8, 64, 64),
                                        ([2000] * 3, 16, 16)])
@pytest.mark.parametrize("below", [20.0, 24.0, 26.0, 28.0])
def test_many_keys_far_below_one(dtype, lens, H, Hkv, below):
    """One key takes nearly all of a row but has no value; what the row gets is the sum of
    many probabilities of 2^-below.  In fp16 they are held to 2^-32 of the largest one each
    (2^7 times below the type's smallest step), the rest is relative to what they add up to."""
    cu, n, D = _cu(lens), sum(lens), 64
    q, k = (torch.zeros(n, h, D, dtype=dtype, device=DEV) for h in (H, Hkv))
    v = torch.ones(n, Hkv, D, dtype=dtype, device=DEV)
    q[..., 0] = 1
    first = torch.tensor(cu[:-1].astype(np.int64), device=DEV)
    k[first, :, 0] = 16.0
    v[first] = 0
    scale = below / 16 * 0.6931471805599453
    got = _call(q, k, v, cu, lens, scale).double()
    p = 2.0 ** -below
    half = 0.0 if dtype is F32 else torch.finfo(dtype).eps / 2
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        i = torch.arange(b - a, device=DEV, dtype=torch.float64)[:, None, None]
        want = (i * p / (1 + i * p)).expand(b - a, H, D)
        # scores of up to 28 times fp32's u, twice, and the scale's own rounding
        rel = 2 * (4 * U * 28 + 4 * U + (b - a) * U)
        tol = (rel + half) * want
        tol = tol + half * (want + tol)
        if dtype is F16:
            tol = tol + i * 2.0 ** -32 + 2.0 ** -25
        assert ((got[a:b] - want).abs() <= tol).all(), (a, (got[a:b] - want).abs().max())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("which", range(4))
def test_values_up_to_the_types_largest(dtype, D, which):
    """The mean of finite values is finite, whatever their sum.  Queries of 0: every
    probability is 1 / n, a mean of n values; weights and sums in fp32 are each off by a
    relative (n + 4) u, a 16-bit type's by half a step more, and so is the output."""
    lens, H, Hkv = _batches()[which]
    cu, n, top = _cu(lens), sum(lens), torch.finfo(dtype).max
    gen = torch.Generator(device=DEV).manual_seed(D)
    q = torch.zeros(n, H, D, dtype=dtype, device=DEV)
    k = torch.randn(n, Hkv, D, generator=gen, device=DEV).to(dtype)
    v = (torch.rand(n, Hkv, D, generator=gen, device=DEV, dtype=torch.float64) / 2 + 0.5) * top
    v = v.to(dtype)
    v[:, :, 1], v[:, :, 2] = top, -top
    got = _call(q, k, v, cu, lens, D ** -0.5).double()
    assert torch.isfinite(got).all()
    half = 0.0 if dtype is F32 else torch.finfo(dtype).eps / 2
    rel = 2 * (max(lens) + 4) * U + 2 * half + half * half
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        count = torch.arange(1, b - a + 1, device=DEV, dtype=torch.float64)[:, None, None]
        want = (v[a:b].double().cumsum(0) / count).repeat_interleave(H // Hkv, 1)
        assert ((got[a:b] - want).abs() <= rel * want.abs()).all()
