"""CPU checks of include/hsattn_ops.h: declarations, exports, and arguments that are
refused before any GPU call; a C99 host of the header; the same refusals with the
host code under sanitizers."""

from __future__ import annotations

import ctypes
import os
import re
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "hsattn_ops.h"
FAKE = ctypes.c_void_p(0x1000)
M = 2 ** 31 - 1


def _declared():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return sorted(set(re.findall(r"\b(hs_[a-z0-9_]+)\s*\(", text)))


@pytest.fixture(scope="module")
def lib():
    from heteroserve import _hip

    if not _hip.lib_path().exists():
        pytest.fail(f"{_hip.lib_path()} missing: run python hetero-serve_amd/build.py")
    return _hip.open_library()


def test_declarations_are_bound_and_exported(lib):
    from heteroserve import _hip

    assert _declared() == sorted(_hip.OPERATOR_SYMBOLS)
    assert not set(_declared()) & set(_hip.EXPORTED_SYMBOLS)
    for name in _declared():
        assert hasattr(lib, name), name


def _refused(lib, rc, code, needle):
    assert rc == code and needle in lib.hs_last_error(), (rc, lib.hs_last_error())


def _rotary(lib, q=FAKE, src=0, q_row=256, axes=1, freq=FAKE, pairs=32, n=3, H=4, Hkv=2, D=64,
            k_out=FAKE, out=0):
    return lib.hs_rotary(q, FAKE, src, q_row, 128, FAKE, axes, freq, None, pairs, 0, n, H, Hkv, D, FAKE,
                         k_out, out, None)


def _append(lib, v=FAKE, v_row=128, kv=0, NB=8, BS=16, bt=FAKE, B=2, MB=2, n=3, pairs=32, at=FAKE,
            D=64):
    return lib.hs_rotary_append(FAKE, FAKE, v, 0, 4 * D, 2 * D, v_row, FAKE, 1, FAKE, None, pairs, 0, n, 4,
                                2, D, FAKE, None, 0, FAKE, FAKE, kv, NB, BS, bt, B, MB, at, None, None)


def test_rotary_refusals(lib):
    _refused(lib, _rotary(lib, q=None), -1, b"null")
    _refused(lib, _rotary(lib, k_out=None), -1, b"null")
    _refused(lib, _rotary(lib, freq=None), -1, b"null")
    _refused(lib, _rotary(lib, src=3), -1, b"dtype")
    _refused(lib, _rotary(lib, out=-1), -1, b"dtype")
    _refused(lib, _rotary(lib, q_row=255), -1, b"stride")
    _refused(lib, _rotary(lib, axes=0), -1, b"positive")
    _refused(lib, _rotary(lib, pairs=0), -1, b"positive")
    _refused(lib, _rotary(lib, pairs=33), -1, b"head_dim / 2")
    _refused(lib, _rotary(lib, n=-1), -1, b"positive")
    assert _rotary(lib, n=0, q=None, k_out=None) == 0
    _refused(lib, _append(lib, v=None), -1, b"null")
    _refused(lib, _append(lib, bt=None), -1, b"null")
    _refused(lib, _append(lib, at=None), -1, b"null")
    _refused(lib, _append(lib, v_row=127), -1, b"stride")
    _refused(lib, _append(lib, kv=9), -1, b"dtype")
    _refused(lib, _append(lib, BS=0), -1, b"positive")
    _refused(lib, _append(lib, B=0), -1, b"positive")
    # sizes that no launch or offset holds
    _refused(lib, _append(lib, D=4096, pairs=2000, v_row=8192), -2, b"pairs")
    _refused(lib, _rotary(lib, H=M, Hkv=M, D=M, pairs=1000, q_row=2 ** 62), -1, b"stride")
    _refused(lib, _rotary(lib, n=2 ** 62), -2, b"too large")
    _refused(lib, _rotary(lib, H=2 ** 22, q_row=2 ** 28), -2, b"too large")


def _prompt(lib, q=FAKE, dtype=2, strides=(256, 64, 128, 64, 128, 64), cu=FAKE, B=2, T=10, longest=5, H=4,
            Hkv=2, D=64, out=FAKE):
    return lib.hs_prompt_attention(q, FAKE, FAKE, dtype, *strides, cu, B, T, longest, H, Hkv, D, 0.1, out,
                                   None)


def test_prompt_refusals(lib):
    _refused(lib, _prompt(lib, q=None), -1, b"null")
    _refused(lib, _prompt(lib, cu=None), -1, b"null")
    _refused(lib, _prompt(lib, dtype=5), -1, b"dtype")
    _refused(lib, _prompt(lib, H=5), -1, b"divisible")
    _refused(lib, _prompt(lib, D=96), -2, b"head_dim")
    _refused(lib, _prompt(lib, D=0), -1, b"positive")
    _refused(lib, _prompt(lib, T=-1), -1, b"positive")
    _refused(lib, _prompt(lib, longest=-1), -1, b"positive")
    _refused(lib, _prompt(lib, strides=(256, 60, 128, 64, 128, 64)), -1, b"16 bytes")
    _refused(lib, _prompt(lib, strides=(256, 64, -128, 64, 128, 64)), -1, b"negative")
    _refused(lib, _prompt(lib, strides=(2 ** 62, 64, 128, 64, 128, 64)), -2, b"too large")
    _refused(lib, _prompt(lib, out=ctypes.c_void_p(0x1008)), -1, b"aligned")
    _refused(lib, _prompt(lib, T=2 ** 31), -2, b"too many rows")
    _refused(lib, _prompt(lib, H=2 ** 20, Hkv=1), -2, b"too many heads")
    assert _prompt(lib, T=0, q=None) == _prompt(lib, B=0, q=None) == _prompt(lib, longest=0, q=None) == 0


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf")])
def test_prompt_scales_that_are_none(lib, scale):
    one = ctypes.c_void_p(0x1000)
    rc = lib.hs_prompt_attention(one, one, one, 2, 256, 64, 128, 64, 128, 64, one, 1, 8, 8, 4, 2, 64,
                                 scale, one, None)
    _refused(lib, rc, -1, b"finite")


def test_page_refusals(lib):
    _refused(lib, lib.hs_kv_copy(None, 1, 8, 1024, FAKE, FAKE, 3, None), -1, b"null")
    _refused(lib, lib.hs_kv_copy(FAKE, 1, 0, 1024, FAKE, FAKE, 3, None), -1, b"positive")
    _refused(lib, lib.hs_kv_copy(FAKE, M, M, 2 ** 62, FAKE, FAKE, M, None), -2, b"too large")
    assert lib.hs_kv_copy(None, 1, 8, 1024, None, None, 0, None) == 0
    ids = (ctypes.c_int64 * 449)()
    _refused(lib, lib.hs_kv_copy_host_ids(FAKE, 1, 8, 1024, ids, ids, 449, None), -2, b"too many")
    _refused(lib, lib.hs_kv_find_free(None, 8, FAKE, 3, None), -1, b"null")
    _refused(lib, lib.hs_kv_find_free(FAKE, 8, FAKE, -3, None), -1, b"positive")
    _refused(lib, lib.hs_kv_find_free(FAKE, 2 ** 22 + 1, FAKE, 3, None), -2, b"at most")
    assert lib.hs_kv_find_free(None, 8, None, 0, None) == 0

    def fork(pool=FAKE, L=1, NB=8, page=1024, BS=16, MB=2, n=3, done=FAKE):
        return lib.hs_kv_fork(pool, L, NB, page, BS, FAKE, 4, MB, FAKE, FAKE, FAKE, FAKE, FAKE, n, done,
                              None)

    _refused(lib, fork(pool=None), -1, b"null")
    _refused(lib, fork(done=None), -1, b"null")
    _refused(lib, fork(MB=0), -1, b"positive")
    _refused(lib, fork(page=1000), -1, b"multiple of block_size")
    _refused(lib, fork(L=M, NB=M, page=2 ** 60), -2, b"too large")
    _refused(lib, fork(L=2 ** 20), -2, b"too large")
    assert fork(pool=None, n=0) == 0
    _refused(lib, lib.hs_kv_free(FAKE, 4, 2, FAKE, None, 8, FAKE, 1, None), -1, b"null")
    _refused(lib, lib.hs_kv_free(FAKE, 0, 2, FAKE, FAKE, 8, FAKE, 1, None), -1, b"positive")
    _refused(lib, lib.hs_kv_free(FAKE, 4, 2 ** 25, FAKE, FAKE, 8, FAKE, 1, None), -2, b"too wide")
    assert lib.hs_kv_free(None, 4, 2, None, None, 8, None, 0, None) == 0

    def compact(NB=8, page=1024, ws=FAKE, have=2 ** 40, live=FAKE):
        return lib.hs_kv_compact(FAKE, 1, NB, page, FAKE, 4, 2, FAKE, FAKE, live, ws, have, None)

    need = lib.hs_kv_compact_workspace_bytes(8)
    assert need > 0 and lib.hs_kv_compact_workspace_bytes(0) == 0
    assert lib.hs_kv_compact_workspace_bytes(M) >= 4 * M
    _refused(lib, compact(live=None), -1, b"null")
    _refused(lib, compact(page=0), -1, b"positive")
    _refused(lib, compact(ws=None), -4, b"workspace")
    _refused(lib, compact(have=need - 1), -4, b"workspace")
    _refused(lib, compact(NB=2 ** 22 + 1), -2, b"at most")
    _refused(lib, compact(page=2 ** 62), -2, b"too large")


def test_the_python_layer_without_a_library(monkeypatch):
    """No compute fallback: every call raises and names the reason."""
    torch = pytest.importorskip("torch")
    from heteroserve import _hip
    from heteroserve.kv import pages, rotary
    from heteroserve.model import prompt_attn

    monkeypatch.setattr(_hip, "_state", "unavailable")
    monkeypatch.setattr(_hip, "_error", "no HIP device")
    q = torch.zeros(2, 4, 64)
    t, c = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(1, 2, 4, 16, 1, 8)
    calls = [lambda: rotary.rotate_qk(q, q, c, torch.ones(32)),
             lambda: rotary.rotate_append_kv(q, q, q, c, torch.ones(32), q, q, t, c),
             lambda: prompt_attn.prompt_attention(q, q, q, c, 2, 1.0),
             lambda: pages.copy_blocks(pool, [0], [1]),
             lambda: pages.find_free_blocks(c, 1),
             lambda: pages.fork_blocks(pool, t, c, c, [0], [1], [0]),
             lambda: pages.free_blocks(t, c, c, [0]),
             lambda: pages.compact_blocks(pool, t, c)]
    assert not prompt_attn.is_available() and prompt_attn.build_error() == "no HIP device"
    for call in calls:
        with pytest.raises(RuntimeError, match="unavailable: no HIP device"):
            call()


def test_axes_of():
    pytest.importorskip("torch")
    from heteroserve.kv import rotary

    assert rotary.axes_of([2, 0, 3]).tolist() == [0, 0, 2, 2, 2]
    assert rotary.axes_of([3, 1, 2], interleaved=True).tolist() == [0, 1, 2, 0, 2, 0]
    assert rotary.axes_of([]).tolist() == []


def test_header_as_c99(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    from heteroserve import _hip

    lib = _hip.lib_path()
    src = tmp_path / "ops.c"
    src.write_text('#include <stdio.h>\n#include "hsattn_ops.h"\ntypedef void (*any_fn)(void);\n'
                   "static const any_fn fns[] = {"
                   + ", ".join(f"(any_fn){n}" for n in _declared())
                   + "};\nint main(void) { printf(\"%d %d\\n\", (int)(sizeof fns / sizeof fns[0]),\n"
                   "  hs_kv_copy(NULL, 0, 0, 0, NULL, NULL, 1, NULL)); return 0; }\n")
    exe = tmp_path / "ops"
    subprocess.run([gcc, "-std=c99", "-pedantic", "-Wall", "-Wextra", "-Werror",
                    f"-I{ROOT / 'include'}", str(src), f"-L{lib.parent}", f"-l:{lib.name}",
                    f"-Wl,-rpath,{lib.parent}", "-o", str(exe)], check=True, capture_output=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.stdout.split() == [str(len(_declared())), "-1"]


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
                        "no:cacheprovider", "-k", "page_refusals or rotary_refusals or prompt_refusals"],
                       capture_output=True, text=True, env=env, cwd=str(ROOT), timeout=600)
    out = r.stdout + r.stderr
    assert r.returncode == 0, out[-4000:]
    assert "runtime error" not in out and "AddressSanitizer" not in out, out[-4000:]


def test_host_ids():
    """Lists, arrays, tensors and the odd element: as torch indexing takes them."""
    np, torch = pytest.importorskip("numpy"), pytest.importorskip("torch")
    from heteroserve.kv import pages

    for ids, want in (([3, 0, 9], [3, 0, 9]), ([-1, 2], [9, 2]), ([], []), ((4, 5), [4, 5]), ([True], [1]),
                      (np.array([1, -10]), [1, 0]), (torch.tensor([[7], [8]]), [7, 8]), ([np.int32(6)], [6]),
                      ([2.0], [2])):
        assert pages._host_ids(ids, 10).tolist() == want
    for ids in ([10], [0, -11], [2 ** 70], np.array([10])):
        with pytest.raises(IndexError, match="out of bounds"):
            pages._host_ids(ids, 10)
