"""CPU checks of the long-context oracle, of what the 4-bit cache and the window decode
refuse before any GPU call, and of their Python layer without a library."""

from __future__ import annotations

import ctypes
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

from oracle import long_context as lc

ROOT = Path(__file__).resolve().parents[1]
FAKE = ctypes.c_void_p(0x1000)
M = 2 ** 31 - 1


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("keys", [True, False])
def test_records_hold_what_quantise_gives(D, keys):
    x = np.random.default_rng(D).normal(size=(3, 2, D)) * 3 + 1
    n, s, lo = lc.quantise(x)
    rec = lc.records(n, s, lo, keys)
    assert rec.shape == (3, 2, 5 * D // 8)
    want = (n * s[..., None] + lo[..., None]).reshape(x.shape)
    assert np.array_equal(lc.values(rec, keys), want)
    # half a step, and what the ends lose in fp16
    off = np.abs(want - x).reshape(3, 2, -1, 32).max(-1)
    assert (off <= s / 2 + 2.0 ** -11 * (np.abs(lo) + 15 * s)).all()
    assert np.array_equal(lc.sizes(rec, keys), (n * s[..., None] + np.abs(lo)[..., None]).reshape(x.shape))
    # every word holds 8 neighbours of one group, every element is held once
    at = [[lc._element(w, e, D // 32, keys) for e in range(8)] for w in range(D // 8)]
    assert sorted(sum(at, [])) == list(range(D))
    assert all(a == list(range(a[0], a[0] + 8)) and a[0] % 8 == 0 for a in at)


def test_groups_of_one_value_and_of_none():
    n, s, lo = lc.quantise(np.array([[0.0] * 32 + [2.5] * 32, [1e6] * 32 + [-1e6, 1e6] * 16,
                                     [float("nan")] + [1.0] * 31 + list(range(32))]))
    assert s[0].tolist() == [0, 0] and lo[0].tolist() == [0, 2.5] and not n[0].any()
    assert lo[1].tolist() == [65504, -65504] and s[1, 0] == 0 and set(n[1, 1]) == {0, 15}
    assert np.isnan(lo[2, 0]) and s[2, 0] == 0 and lo[2, 1] == 0


def test_visible():
    assert lc.visible(0, 4, 2).tolist() == [] and lc.visible(-3, 0, 0).tolist() == []
    assert lc.visible(5, 0, 0).tolist() == [0, 1, 2, 3, 4]
    assert lc.visible(10, 3, 2).tolist() == [0, 1, 7, 8, 9]
    assert lc.visible(4, 3, 2).tolist() == [0, 1, 2, 3]
    assert lc.visible(9, 1, 0).tolist() == [8]


def test_decode_of_one_key_and_of_equal_ones():
    rng = np.random.default_rng(0)
    q, k, v = rng.normal(size=(4, 32)), rng.normal(size=(3, 2, 32)), rng.normal(size=(3, 2, 32))
    out, spread, weight = lc.decode(q, k[:1], v[:1], 0.2)
    assert np.allclose(out, v[0].repeat(2, 0)) and np.allclose(weight, 0)
    assert np.allclose(spread, np.abs(v[0]).repeat(2, 0))
    same, _, _ = lc.decode(q, k[:1].repeat(3, 0), v, 0.2)
    assert np.allclose(same, v.mean(0).repeat(2, 0))
    assert not lc.decode(q, k[:0], v[:0], 0.2)[0].any()


# --- refusals ------------------------------------------------------------------


@pytest.fixture(scope="module")
def lib():
    from heteroserve import _hip

    if not _hip.lib_path().exists():
        pytest.fail(f"{_hip.lib_path()} missing: run python hetero-serve_amd/build.py")
    return _hip.open_library()


def _refused(lib, rc, code, needle):
    assert rc == code and needle in lib.hs_last_error(), (rc, lib.hs_last_error())


def _append(lib, cache=FAKE, NB=8, BS=16, Hkv=2, D=64, bt=FAKE, B=2, MB=2, at=FAKE, n=3, k=FAKE, v=FAKE,
            src=2, k_row=128, v_row=128):
    return lib.hs_q4_append(cache, FAKE, NB, BS, Hkv, D, bt, B, MB, at, None, n, k, v, src, k_row, v_row,
                            None)


def _read(lib, cache=FAKE, NB=8, BS=16, Hkv=2, D=64, bt=FAKE, B=2, MB=2, at=FAKE, n=3, k=FAKE, v=FAKE,
          out=2):
    return lib.hs_q4_read(cache, FAKE, NB, BS, Hkv, D, bt, B, MB, at, None, n, k, v, out, None)


def test_row_refusals(lib):
    for call in (_append, _read):
        _refused(lib, call(lib, cache=None), -1, b"null")
        _refused(lib, call(lib, bt=None), -1, b"null")
        _refused(lib, call(lib, at=None), -1, b"null")
        _refused(lib, call(lib, k=None), -1, b"null")
        _refused(lib, call(lib, v=None), -1, b"null")
        _refused(lib, call(lib, cache=ctypes.c_void_p(0x1004)), -1, b"aligned")
        _refused(lib, call(lib, n=-1), -1, b"positive")
        _refused(lib, call(lib, Hkv=0), -1, b"positive")
        _refused(lib, call(lib, NB=0), -1, b"positive")
        _refused(lib, call(lib, MB=0), -1, b"positive")
        _refused(lib, call(lib, D=96), -2, b"head_dim")
        assert call(lib, n=0, cache=None, k=None) == 0
    _refused(lib, _append(lib, src=3), -1, b"dtype")
    _refused(lib, _append(lib, k_row=127), -1, b"stride")
    _refused(lib, _append(lib, v_row=127), -1, b"stride")
    _refused(lib, _append(lib, n=2 ** 62), -2, b"too large")
    _refused(lib, _append(lib, k_row=2 ** 62), -2, b"too large")
    _refused(lib, _append(lib, Hkv=2 ** 27, k_row=2 ** 40, v_row=2 ** 40), -2, b"too large")
    _refused(lib, _read(lib, out=-1), -1, b"dtype")
    _refused(lib, _read(lib, k=ctypes.c_void_p(0x1008)), -1, b"aligned")
    _refused(lib, _read(lib, n=2 ** 40), -2, b"too large")


def _decode(lib, q=FAKE, k=FAKE, kv=2, NB=8, bt=FAKE, ctx=FAKE, out=FAKE, B=2, H=4, Hkv=2, D=64, BS=16,
            MB=2, scale=0.1, window=0, sinks=0, ws=None, have=0):
    if kv == "q4":
        return lib.hs_q4_decode(q, k, FAKE, NB, bt, ctx, out, B, H, Hkv, D, BS, MB, scale, window, sinks,
                                ws, have, None)
    return lib.hs_window_decode(q, k, FAKE, kv, NB, bt, ctx, out, B, H, Hkv, D, BS, MB, scale, window,
                                sinks, ws, have, None)


@pytest.mark.parametrize("kv", ["q4", 0, 1, 2])
def test_decode_refusals(lib, kv):
    for name in ("q", "k", "bt", "ctx", "out"):
        _refused(lib, _decode(lib, kv=kv, **{name: None}), -1, b"null")
    for name in ("q", "out"):
        _refused(lib, _decode(lib, kv=kv, **{name: ctypes.c_void_p(0x1008)}), -1, b"aligned")
    _refused(lib, _decode(lib, kv=kv, k=ctypes.c_void_p(0x1004)), -1, b"aligned")
    _refused(lib, _decode(lib, kv=kv, H=5), -1, b"divisible")
    _refused(lib, _decode(lib, kv=kv, D=96), -2, b"head_dim")
    for name in ("H", "Hkv", "BS", "MB", "NB"):
        _refused(lib, _decode(lib, kv=kv, **{name: 0}), -1, b"positive")
    _refused(lib, _decode(lib, kv=kv, B=-1), -1, b"positive")
    _refused(lib, _decode(lib, kv=kv, window=-1), -1, b"negative")
    _refused(lib, _decode(lib, kv=kv, sinks=-1), -1, b"negative")
    for scale in (float("inf"), float("nan"), 3e38):
        _refused(lib, _decode(lib, kv=kv, scale=scale), -1, b"finite")
    _refused(lib, _decode(lib, kv=kv, MB=2 ** 27), -2, b"too wide")
    _refused(lib, _decode(lib, kv=kv, NB=2 ** 27), -2, b"too long")
    _refused(lib, _decode(lib, kv=kv, MB=2 ** 20, window=0), -4, b"workspace")
    _refused(lib, _decode(lib, kv=kv, MB=2 ** 20, ws=ctypes.c_void_p(0x1008), have=2 ** 62), -1, b"aligned")
    _refused(lib, _decode(lib, kv=kv, B=M, H=2 ** 20, Hkv=2 ** 20, MB=2 ** 26), -2, b"too large")
    assert _decode(lib, kv=kv, B=0, q=None) == 0


def test_workspace_queries(lib):
    def q4(B=2, H=4, Hkv=2, D=64, BS=16, MB=2 ** 12, window=0, sinks=0):
        return lib.hs_q4_decode_workspace_bytes(B, H, Hkv, D, BS, MB, window, sinks)

    assert q4() > 0 and q4(B=0) == q4(D=96) == q4(H=3) == q4(window=-1) == q4(MB=2 ** 28) == 0
    assert q4(window=16, sinks=4) <= q4()
    for kv in (0, 1, 2):
        assert lib.hs_window_decode_workspace_bytes(kv, 2, 4, 2, 64, 16, 2 ** 12, 0, 0) > 0
    for kv in (-1, 3):
        assert lib.hs_window_decode_workspace_bytes(kv, 2, 4, 2, 64, 16, 2 ** 12, 0, 0) == 0


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("window", [0, 1, 256, 5000])
def test_workspace_queries_of_every_kind(lib, D, window):
    """One row to many, tables narrow and wide, every type: sizes that grow with the rows, and 0
    where a row is one part whatever it holds."""
    for MB in (1, 32, 2048, 2 ** 16):
        sizes = []
        for B in (1, 3, 64, 256, 257, 5000):
            kinds = [lib.hs_window_decode_workspace_bytes(kv, B, 12, 6, D, 16, MB, window, 4) for kv in range(3)]
            sizes.append([*kinds, lib.hs_q4_decode_workspace_bytes(B, 12, 6, D, 16, MB, window, 4)])
        if MB == 1 or window == 1:
            assert not np.any(sizes)
        if MB >= 2048 and not window:
            assert np.all(sizes) and all(np.all(np.diff(x[2:5]) > 0) for x in zip(*sizes))


def test_the_unknown_kv_type_is_refused(lib):
    for kv in (-1, 3):
        _refused(lib, _decode(lib, kv=kv), -1, b"dtype")


def test_refusals_under_asan_and_ubsan():
    sys.path.insert(0, str(ROOT / "hetero-serve_amd"))
    import build as hs_build

    if os.environ.get("HETEROSERVE_HIP_LIB") == str(hs_build.SAN_LIB):
        pytest.skip("this is that run")
    if not hs_build.SAN_LIB.exists():
        pytest.fail(f"{hs_build.SAN_LIB} missing: run python hetero-serve_amd/build.py --sanitize")
    env = dict(os.environ)
    env.update(LD_PRELOAD=str(hs_build.asan_runtime()),
               ASAN_OPTIONS="detect_leaks=0:halt_on_error=1",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1",
               HETEROSERVE_HIP_LIB=str(hs_build.SAN_LIB))
    r = subprocess.run([sys.executable, "-m", "pytest", str(Path(__file__)), "-q", "-p",
                        "no:cacheprovider", "-k", "row_refusals or decode_refusals or queries"],
                       capture_output=True, text=True, env=env, cwd=str(ROOT), timeout=600)
    out = r.stdout + r.stderr
    assert r.returncode == 0, out[-4000:]
    assert "runtime error" not in out and "AddressSanitizer" not in out, out[-4000:]


def test_the_python_layer_without_a_library(monkeypatch):
    torch = pytest.importorskip("torch")
    from heteroserve import _hip
    from heteroserve.kv import quant
    from heteroserve.model import paged_attn_q4, paged_attn_window

    monkeypatch.setattr(_hip, "_state", "unavailable")
    monkeypatch.setattr(_hip, "_error", "no HIP device")
    q, c = torch.zeros(2, 4, 64), torch.zeros(2, dtype=torch.int32)
    pool, t = quant.empty_pool_q4(1, 4, 16, 2, 64, device="cpu"), torch.zeros(2, 2, dtype=torch.int32)
    kc = torch.zeros(4, 16, 2, 64)
    assert pool.shape == (1, 2, 4, 16, 2, 40) and pool.dtype is torch.uint8 and not pool.any()
    for call in (lambda: quant.append_kv_q4(pool[0, 0], pool[0, 1], t, c, q, q),
                 lambda: quant.read_kv_q4(pool[0, 0], pool[0, 1], t, c),
                 lambda: paged_attn_q4.paged_attention_q4(q, pool[0, 0], pool[0, 1], t, c, 0.1),
                 lambda: paged_attn_window.paged_attention_window(q, kc, kc, t, c, 0.1, 4)):
        with pytest.raises(RuntimeError, match="unavailable: no HIP device"):
            call()
    for mod in (paged_attn_q4, paged_attn_window):
        assert not mod.is_available() and mod.build_error() == "no HIP device"


def test_record_bytes():
    pytest.importorskip("torch")
    from heteroserve.kv import quant

    assert [quant.record_bytes(d) for d in (32, 64, 128, 256)] == [20, 40, 80, 160]
    for d in (0, 96, 512):
        with pytest.raises(RuntimeError, match="head_dim"):
            quant.record_bytes(d)
