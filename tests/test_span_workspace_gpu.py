"""Wide tables on the GPU: more rows than parts are fitted for, whose parts grow so that their
states stay in bounds, and fitted ones, whose states lie by number; a workspace holds no more than the query said.

Tolerances are those of arithmetic in fp32, (D + 64) 2^-23 of the scores' sizes and (n + 64) 2^-23 of
sum p |v|."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import long_context as lc  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BS = 16


@pytest.mark.parametrize("kv", ["q4", torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B", [40, 256, 300])
def test_rows_of_wide_tables_and_nothing_behind_the_workspace(kv, B):
    from heteroserve import _hip

    rng = np.random.default_rng(B)
    H, Hkv, D, pages, MB = 16, 2, 128, 200, 8192
    gen = torch.Generator(DEV).manual_seed(B)
    k, v = (torch.randn(pages * BS, Hkv, D, generator=gen, device=DEV) for _ in range(2))
    lens = rng.choice([0, 1, 300, 511, 512, 513, 2048, 4096, 5000, 9001], B)
    lens[B // 3] = 40000
    bt = torch.tensor(rng.integers(0, pages, (B, MB)).astype(np.int32), device=DEV)
    ctx = torch.tensor(lens.astype(np.int32), device=DEV)
    q = torch.randn(B, H, D, generator=gen, device=DEV)
    L = _hip.lib()
    if kv == "q4":
        rec = [lc.records(*lc.quantise(x.double().cpu().numpy()), keys=i == 0) for i, x in enumerate((k, v))]
        k, v = (lc.values(x, i == 0) for i, x in enumerate(rec))
        cache = torch.tensor(np.stack(rec), device=DEV).view(2, pages, BS, Hkv, 5 * D // 8)
        head, query, call = (), L.hs_q4_decode_workspace_bytes, L.hs_q4_decode
    else:
        cache = torch.stack([k, v]).to(kv).view(2, pages, BS, Hkv, D)
        k, v = cache.view(2, pages * BS, Hkv, D).double().cpu().numpy()
        head, query, call = (_hip.dtype_code(kv),), L.hs_window_decode_workspace_bytes, L.hs_window_decode
    need = query(*head, B, H, Hkv, D, BS, MB, 0, 0)
    assert 0 < need < 2 ** 29 and need % 4 == 0
    room = torch.full((need // 4 + 4096,), 123456.0, device=DEV)
    out = torch.full((B, H, D), float("nan"), device=DEV)

    def ptr(x):
        return ctypes.c_void_p(x.data_ptr())

    for _ in range(2):
        rc = call(ptr(q), ptr(cache[0]), ptr(cache[1]), *head, pages, ptr(bt), ptr(ctx), ptr(out), B, H, Hkv, D,
                  BS, MB, D ** -0.5, 0, 0, ptr(room), need, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0, L.hs_last_error()
    torch.cuda.synchronize()
    assert bool((room[need // 4:] == 123456.0).all())
    got, table = out.double().cpu().numpy(), bt.cpu().numpy()
    assert np.isfinite(got).all() and not got[lens == 0].any()
    for b in [B // 3, *rng.choice(B, 12, replace=False)]:
        at = np.arange(lens[b])
        rows = table[b, at // BS].astype(np.int64) * BS + at % BS
        want, spread, weight = lc.decode(q[b].double().cpu().numpy(), k[rows], v[rows], D ** -0.5)
        tol = (D + 64) * 2.0 ** -23 * weight + (len(at) + 64) * 2.0 ** -23 * spread
        assert (np.abs(got[b] - want) <= tol).all(), (b, lens[b])
