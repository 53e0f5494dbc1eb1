"""Values of overlapping rows, given flat to the rotary cache write."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 36])
def test_flat_values_of_overlapping_rows(dtype, D):
    """[n, Hkv * D] rows that are expanded, slide, or lie apart."""
    from heteroserve.kv import rotary

    gen = torch.Generator(device=DEV).manual_seed(D)
    flat = torch.randn(40 * D, generator=gen, device=DEV).to(dtype)
    q, k = flat[:24 * D].view(6, 4, D), flat[-12 * D:].view(6, 2, D)
    at = torch.arange(6, dtype=torch.int32, device=DEV)
    table, seq = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros_like(at)
    freq = torch.linspace(1, 0.1, 16, device=DEV)
    for v in (flat[:2 * D].expand(6, 2 * D), flat.as_strided((6, 2 * D), (D, 1)),
              flat.as_strided((6, 2 * D), (5 * D, 1)), flat.as_strided((6, 2 * D), (1, 3)),
              flat.as_strided((6, 2 * D), (0, 0))):
        kc, vc = torch.zeros(2, 1, 16, 2, D, dtype=dtype, device=DEV)
        want_k, want_v = torch.zeros(2, 1, 16, 2, D, dtype=dtype, device=DEV)
        rotary.rotate_append_kv(q, k, v.contiguous().view(6, 2, D), at, freq, want_k, want_v, table, at, seq)
        rotary.rotate_append_kv(q, k, v, at, freq, kc, vc, table, at, seq)
        assert torch.equal(vc, want_v) and torch.equal(kc, want_k)
        assert torch.equal(vc[0, :6], v.reshape(6, 2, D)) and not vc[0, 6:].any()
