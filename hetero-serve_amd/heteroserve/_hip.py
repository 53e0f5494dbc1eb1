"""Loader and tensor marshalling for libhsattn.so (the gfx950 C-ABI library).

This module is the only place that touches ctypes.  It keeps the reference's
module-state contract (heteroserve/model/paged_attn.py:197-252): the library is
loaded once, on first use, and a failure is recorded with a reason rather than
raised at import.  Unlike the reference there is no compute fallback: an entry
point called while the library is unavailable raises RuntimeError.

Environment:
  HETEROSERVE_DISABLE_CUDA_KERNEL  treat the library as unavailable (reference flag)
  HETEROSERVE_HIP_LIB              path of libhsattn.so (default: next to this file)
  HETEROSERVE_PREFILL_GRID=1       keep the MFMA prefill on its grid kernel (one workgroup
                                   per query tile) where the persistent one would run;
                                   read at each call, for comparisons

PyTorch provides device memory and the current stream; every kernel launches
on ``torch.cuda.current_stream(device)`` of the input's device.
"""

from __future__ import annotations

import ctypes
import operator
import os
import threading
from pathlib import Path
from typing import Optional

try:
    import torch
except ImportError as _exc:   # reported by _load()
    torch = None
    _torch_error = str(_exc)

ABI_VERSION = 5
DTYPE_F32, DTYPE_F16, DTYPE_BF16 = 0, 1, 2

_lock = threading.Lock()
_lib: Optional[ctypes.CDLL] = None
_state = "unloaded"          # "unloaded" | "ready" | "unavailable"
_error: Optional[str] = None

_c_int, _c_i64, _c_size, _c_float, _c_vp = (
    ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float, ctypes.c_void_p)

# name -> (restype, argtypes); must match include/hsattn.h
_SIGNATURES = {
    "hs_abi_version": (_c_int, []),
    "hs_last_error": (ctypes.c_char_p, []),
    "hs_profile_next_launch": (_c_int, [_c_vp, _c_vp]),
    "hs_device_cu_count": (_c_int, [_c_int]),
    "hs_choose_num_splits": (_c_i64, [_c_i64, _c_i64, _c_i64]),
    "hs_decode_workspace_bytes": (_c_size, [_c_int] * 8),
    "hs_decode": (_c_int, [_c_vp, _c_vp, _c_vp, _c_int, _c_int, _c_vp, _c_vp, _c_vp,
                           _c_int, _c_int, _c_int, _c_int, _c_int, _c_int, _c_float,
                           _c_int, _c_int, _c_vp, _c_size, _c_vp]),
    "hs_decode_noalloc": (_c_int, [_c_vp, _c_vp, _c_vp, _c_int, _c_int, _c_vp, _c_vp, _c_vp,
                                   _c_int, _c_int, _c_int, _c_int, _c_int, _c_int, _c_float,
                                   _c_int, _c_int, _c_vp]),
    "hs_decode_shared_workspace_bytes": (_c_size, [_c_int] * 7),
    "hs_decode_shared": (_c_int, [_c_vp, _c_vp, _c_vp, _c_int, _c_int, _c_vp, _c_vp, _c_vp,
                                  _c_int, _c_int, _c_int, _c_int, _c_int, _c_int, _c_float,
                                  _c_int, _c_vp, _c_size, _c_vp]),
    "hs_prefill_workspace_bytes": (_c_size, [_c_int] * 5),
    "hs_prefill": (_c_int, [_c_vp, _c_vp, _c_vp, _c_int, _c_int, _c_vp, _c_vp, _c_vp,
                            _c_int, _c_int, _c_int, _c_int, _c_int, _c_int, _c_int,
                            _c_float, _c_int, _c_vp, _c_size, _c_vp]),
    "hs_prefill_varlen": (_c_int, [_c_vp, _c_vp, _c_int, _c_vp, _c_vp, _c_int, _c_int,
                                   _c_vp, _c_vp, _c_vp, _c_int, _c_int, _c_int, _c_int,
                                   _c_int, _c_int, _c_float, _c_int, _c_vp, _c_size, _c_vp]),
    "hs_kv_pack": (_c_int, [_c_vp, _c_int, _c_int, _c_i64, _c_vp, _c_int, _c_vp, _c_vp]),
    "hs_kv_unpack": (_c_int, [_c_vp, _c_int, _c_int, _c_i64, _c_vp, _c_int, _c_vp, _c_vp]),
    "hs_kv_gather": (_c_int, [_c_vp, _c_int, _c_int, _c_i64, _c_vp, _c_int, _c_int, _c_int,
                              _c_vp, _c_vp]),
    "hs_block_tables": (_c_int, [_c_vp, _c_int, _c_int, _c_vp, _c_vp]),
    "hs_kv_scatter": (_c_int, [_c_vp, _c_vp, _c_int, _c_i64, _c_int, _c_int, _c_vp, _c_i64,
                               _c_vp, _c_vp, _c_int, _c_i64, _c_vp]),
    "hs_kv_append": (_c_int, [_c_vp, _c_vp, _c_int, _c_int, _c_int, _c_int, _c_int, _c_vp,
                              _c_int, _c_int, _c_vp, _c_vp, _c_i64, _c_vp, _c_vp, _c_int, _c_i64,
                              _c_vp]),
}

EXPORTED_SYMBOLS = tuple(_SIGNATURES)

# must match include/hsattn_ops.h
_OPERATORS = {
    "hs_rotary": (_c_int, [_c_vp, _c_vp, _c_int, _c_i64, _c_i64, _c_vp, _c_int, _c_vp, _c_vp, _c_int,
                           _c_int, _c_i64, _c_int, _c_int, _c_int, _c_vp, _c_vp, _c_int, _c_vp]),
    "hs_rotary_append": (_c_int, [_c_vp, _c_vp, _c_vp, _c_int, _c_i64, _c_i64, _c_i64, _c_vp, _c_int,
                                  _c_vp, _c_vp, _c_int, _c_int, _c_i64, _c_int, _c_int, _c_int,
                                  _c_vp, _c_vp, _c_int, _c_vp, _c_vp, _c_int, _c_int, _c_int, _c_vp,
                                  _c_int, _c_int, _c_vp, _c_vp, _c_vp]),
    "hs_prompt_attention": (_c_int, [_c_vp, _c_vp, _c_vp, _c_int] + [_c_i64] * 6
                            + [_c_vp, _c_int, _c_i64, _c_int, _c_int, _c_int, _c_int, _c_float,
                               _c_vp, _c_vp]),
    "hs_kv_copy": (_c_int, [_c_vp, _c_int, _c_int, _c_i64, _c_vp, _c_vp, _c_int, _c_vp]),
    "hs_kv_find_free": (_c_int, [_c_vp, _c_int, _c_vp, _c_int, _c_vp]),
    "hs_kv_fork": (_c_int, [_c_vp, _c_int, _c_int, _c_i64, _c_int, _c_vp, _c_int, _c_int, _c_vp,
                            _c_vp, _c_vp, _c_vp, _c_vp, _c_int, _c_vp, _c_vp]),
    "hs_kv_free": (_c_int, [_c_vp, _c_int, _c_int, _c_vp, _c_vp, _c_int, _c_vp, _c_int, _c_vp]),
    "hs_kv_compact_workspace_bytes": (_c_size, [_c_int]),
    "hs_kv_compact": (_c_int, [_c_vp, _c_int, _c_int, _c_i64, _c_vp, _c_int, _c_int, _c_vp, _c_vp,
                               _c_vp, _c_vp, _c_size, _c_vp]),
    "hs_q4_append": (_c_int, [_c_vp, _c_vp] + [_c_int] * 4 + [_c_vp, _c_int, _c_int, _c_vp, _c_vp, _c_i64,
                              _c_vp, _c_vp, _c_int, _c_i64, _c_i64, _c_vp]),
    "hs_q4_read": (_c_int, [_c_vp, _c_vp] + [_c_int] * 4 + [_c_vp, _c_int, _c_int, _c_vp, _c_vp, _c_i64,
                            _c_vp, _c_vp, _c_int, _c_vp]),
    "hs_q4_decode_workspace_bytes": (_c_size, [_c_int] * 8),
    "hs_q4_decode": (_c_int, [_c_vp, _c_vp, _c_vp, _c_int, _c_vp, _c_vp, _c_vp] + [_c_int] * 6
                     + [_c_float, _c_int, _c_int, _c_vp, _c_size, _c_vp]),
    "hs_window_decode_workspace_bytes": (_c_size, [_c_int] * 9),
    "hs_window_decode": (_c_int, [_c_vp, _c_vp, _c_vp, _c_int, _c_int, _c_vp, _c_vp, _c_vp] + [_c_int] * 6
                         + [_c_float, _c_int, _c_int, _c_vp, _c_size, _c_vp]),
}

OPERATOR_SYMBOLS = tuple(_OPERATORS)

# entry points of this layer's own; must match csrc/hs_private.h
_PRIVATE = {
    "hs_kv_pack_host_ids": (_c_int, [_c_vp, _c_int, _c_int, _c_i64, _c_vp, _c_int, _c_vp, _c_vp]),
    "hs_kv_unpack_host_ids": (_c_int, [_c_vp, _c_int, _c_int, _c_i64, _c_vp, _c_int, _c_vp, _c_vp]),
    "hs_kv_scatter_layers": (_c_int, [_c_vp, _c_vp, _c_int, _c_i64, _c_int, _c_int, _c_int, _c_i64,
                                      _c_vp, _c_i64, _c_vp, _c_vp, _c_int, _c_i64, _c_i64, _c_i64,
                                      _c_vp]),
    "hs_kv_copy_host_ids": (_c_int, [_c_vp, _c_int, _c_int, _c_i64, _c_vp, _c_vp, _c_int, _c_vp]),
}


def lib_path() -> Path:
    env = os.environ.get("HETEROSERVE_HIP_LIB")
    return Path(env) if env else Path(__file__).resolve().parent / "libhsattn.so"


def open_library(path: Optional[Path] = None) -> ctypes.CDLL:
    """dlopen libhsattn.so and bind its signatures.  Needs no GPU.  OSError when the
    library is of another ABI, or was built without an entry point that this
    layer calls."""
    path = path or lib_path()
    lib = ctypes.CDLL(str(path))

    def bind(name, res, args):
        fn = getattr(lib, name, None)
        if fn is None:
            raise OSError(f"no {name} in {path}: rebuild it")
        fn.restype = res
        fn.argtypes = args
        return fn

    got = bind("hs_abi_version", *_SIGNATURES["hs_abi_version"])()
    if got != ABI_VERSION:
        raise OSError(f"libhsattn ABI version {got}, expected {ABI_VERSION}")
    for name, (res, args) in {**_SIGNATURES, **_PRIVATE, **_OPERATORS}.items():
        bind(name, res, args)
    return lib


def _load() -> None:
    global _lib, _state, _error
    if _state != "unloaded":
        return
    with _lock:
        if _state != "unloaded":
            return
        if os.environ.get("HETEROSERVE_DISABLE_CUDA_KERNEL"):
            _state, _error = "unavailable", "disabled by HETEROSERVE_DISABLE_CUDA_KERNEL"
            return
        if torch is None:
            _state, _error = "unavailable", f"torch unavailable: {_torch_error}"
            return
        if not torch.cuda.is_available():
            _state, _error = "unavailable", "no HIP device"
            return
        arch = getattr(torch.cuda.get_device_properties(0), "gcnArchName", "").split(":")[0]
        if arch != "gfx950":
            _state, _error = "unavailable", (
                f"libhsattn.so is built for gfx950 only; device 0 is {arch or 'unknown'}")
            return
        path = lib_path()
        if not path.exists():
            _state, _error = "unavailable", (
                f"{path} is missing -- build it with python hetero-serve_amd/build.py")
            return
        try:
            _lib = open_library(path)
        except OSError as exc:
            _state, _error = "unavailable", f"OSError: {str(exc)[:200]}"
            return
        _state = "ready"


def ready() -> bool:
    _load()
    return _state == "ready"


def error() -> Optional[str]:
    _load()
    return _error


def lib(what: str = "paged attention HIP kernel") -> ctypes.CDLL:
    """The loaded library, or RuntimeError naming why it is unavailable."""
    if _state == "ready":
        return _lib
    _load()
    if _state != "ready":
        raise RuntimeError(f"{what} unavailable: {_error}")
    return _lib


def check(rc: int) -> None:
    if rc != 0:
        raise RuntimeError(_lib.hs_last_error().decode(errors="replace"))


# ---------------------------------------------------------------------------
# marshalling helpers
#
# A small decode step is a few microseconds on the GPU, so the calls below are
# what such a step costs: they compare device indexes (an int from one C call)
# instead of device objects, convert only what needs converting, ask torch for
# the raw stream, and remember workspace sizes.  A decode call of 8 sequences
# took 16.2 us of host time before.
# ---------------------------------------------------------------------------

_DTYPE_CODES = {} if torch is None else {
    torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}
_raw_stream = getattr(getattr(torch, "_C", None), "_cuda_getCurrentRawStream", None)
_device = getattr(getattr(torch, "_C", None), "_cuda_getDevice", None)   # once HIP is up
_INT32 = getattr(torch, "int32", None)


def dtype_code(dt) -> int:
    code = _DTYPE_CODES.get(dt)
    if code is None:
        raise RuntimeError(f"unsupported KV cache dtype {dt} (float32, float16 or bfloat16)")
    return code


def stream_of(device) -> int:
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device() if device.index is None else device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _stream_at(index: int) -> int:
    """The current stream of device `index`."""
    if _raw_stream is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(index).cuda_stream


def _int32_on(t, device):
    if not torch.is_tensor(t):
        t = torch.as_tensor(t)
    if t.dtype is _INT32 and t.get_device() == device.index and t.is_contiguous():
        return t
    return t.to(device=device, dtype=torch.int32).contiguous()


def _whole_on(what: str, t, device):
    """_int32_on of integers only.  One that 32 bits do not hold becomes the nearest that
    they do, so what named no row or block still names none."""
    if not torch.is_tensor(t):
        t = torch.as_tensor(t)
    dt = t.dtype
    if dt is _INT32:
        if t.get_device() == device.index and t.is_contiguous():
            return t
    elif t.numel():
        if dt.is_floating_point or dt.is_complex or dt is torch.bool:
            raise RuntimeError(f"{what} must be integers, got {dt}")
        if dt is torch.int64 or dt is torch.uint32 or dt is torch.uint64:
            t = t.to(device=device, dtype=torch.int64)
            if dt is torch.uint64:
                t = t.masked_fill(t < 0, 0x7fffffff)
            t = t.clamp(-0x80000000, 0x7fffffff)
    return _int32_on(t, device)


def _check_device(q, k_cache, v_cache) -> int:
    """The device index that all three tensors are on."""
    index = q.get_device()
    if index < 0 or not q.is_cuda:
        raise RuntimeError("q must be on CUDA")
    if k_cache.get_device() != index or v_cache.get_device() != index:
        if not (k_cache.is_cuda and v_cache.is_cuda):
            raise RuntimeError("kv cache must be on CUDA")
        raise RuntimeError("q and the kv cache must be on the same device")
    return index


def _check_q(q):
    if q.dtype is not torch.float32:
        raise RuntimeError(f"q must be float32, got {q.dtype}")
    return q.contiguous()


def _check_kv(k_cache, v_cache, D):
    """(k_cache, v_cache) contiguous, and their shape."""
    shape = k_cache.shape
    if len(shape) != 4:
        raise RuntimeError("k_cache must be [NB, BS, H, D]")
    if v_cache.shape != shape:
        raise RuntimeError("v_cache must have the shape of k_cache")
    if k_cache.dtype is not v_cache.dtype:
        raise RuntimeError("k_cache and v_cache must have the same dtype")
    if shape[3] != D:
        raise RuntimeError(f"head_dim mismatch: q has {D}, cache has {shape[3]}")
    return k_cache.contiguous(), v_cache.contiguous(), shape


class _DeviceGuard:
    """Make device `index` current for the duration of a library call."""

    __slots__ = ("_index", "_prev")

    def __init__(self, index: int):
        self._index = index
        self._prev = None

    def __enter__(self):
        cur = _device() if _device is not None else torch.cuda.current_device()
        if cur != self._index:
            self._prev = cur
            torch.cuda.set_device(self._index)

    def __exit__(self, *exc):
        if self._prev is not None:
            torch.cuda.set_device(self._prev)


# Workspace sizes of decode calls by their arguments and device.  The sizes are
# fixed for a device and a library; the table is emptied when it grows past
# what a server's batch sizes and table widths make.
_WS_SIZES: dict = {}
_WS_SIZES_MAX = 4096


def _decode_workspace(query, index: int, *sizes: int) -> int:
    """query(*sizes), with device `index` current (only sizes above 0 are kept:
    0 may also be a failed query)."""
    key = (query.__name__, index, sizes)
    n = _WS_SIZES.get(key)
    if n is None:
        n = query(*sizes)
        if n:
            if len(_WS_SIZES) >= _WS_SIZES_MAX:
                _WS_SIZES.clear()
            _WS_SIZES[key] = n
    return n


def decode(q, k_cache, v_cache, block_tables, context_lens, scale: float,
           num_splits: int, partition_tokens: int = 0, shared_pages: bool = False):
    """out[B, H, D] fp32 = paged decode attention via hs_decode.

    shared_pages=True (fixed partitions only, num_splits == 0) runs
    hs_decode_shared: partitions whose block ids several sequences share are
    read once for all of them."""
    L = lib()
    index = _check_device(q, k_cache, v_cache)
    if q.dim() != 3:
        raise RuntimeError("q must be [B, H, D]")
    q = _check_q(q)
    B, H, D = q.shape
    k_cache, v_cache, (NB, BS, Hkv, _) = _check_kv(k_cache, v_cache, D)
    dev = q.device
    bt = _int32_on(block_tables, dev)
    ctx = _int32_on(context_lens, dev)
    if bt.dim() != 2 or bt.shape[0] != B:
        raise RuntimeError("block_tables must be [B, max_blocks]")
    if ctx.numel() != B:
        raise RuntimeError("context_lens must have one entry per sequence")
    MB = bt.shape[1]
    out = q.new_empty(q.shape)
    if B == 0:
        return out
    scale, num_splits, partition_tokens = float(scale), int(num_splits), int(partition_tokens)
    if shared_pages and num_splits != 0:
        raise RuntimeError("shared_pages needs fixed partitions (num_splits == 0)")
    with _DeviceGuard(index):
        if shared_pages:
            ws_bytes = _decode_workspace(L.hs_decode_shared_workspace_bytes, index, B, H, Hkv, D,
                                         BS, max(MB, 1), partition_tokens)
        else:
            ws_bytes = _decode_workspace(L.hs_decode_workspace_bytes, index, B, H, Hkv, D, BS,
                                         max(MB, 1), num_splits, partition_tokens)
        ws = q.new_empty((ws_bytes + 3) // 4) if ws_bytes else None
        wsp = ws.data_ptr() if ws is not None else None
        if shared_pages:
            rc = L.hs_decode_shared(
                q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), dtype_code(k_cache.dtype),
                NB, bt.data_ptr(), ctx.data_ptr(), out.data_ptr(), B, H, Hkv, D, BS, MB,
                scale, partition_tokens, wsp, ws_bytes, _stream_at(index))
        else:
            rc = L.hs_decode(
                q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), dtype_code(k_cache.dtype),
                NB, bt.data_ptr(), ctx.data_ptr(), out.data_ptr(), B, H, Hkv, D, BS, MB,
                scale, num_splits, partition_tokens, wsp, ws_bytes, _stream_at(index))
        check(rc)
    return out


def _prefill_workspace(L, B: int, rows: int, H: int, D: int, use_mfma: bool, split: bool,
                       device):
    """(tensor or None, bytes): the key-range split's scratch, when it applies."""
    nbytes = L.hs_prefill_workspace_bytes(B, rows, H, D, int(bool(use_mfma))) if split else 0
    if not nbytes:
        return None, 0
    return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes


def prefill(q, k_cache, v_cache, block_tables, context_lens, scale: float, use_mfma: bool,
            split: bool = True):
    """out[B, S, H, D] fp32 = causal chunked prefill via hs_prefill.

    split=False passes no workspace, so the matrix-core kernel runs without
    the key-range split (for tests of that launch shape)."""
    L = lib()
    index = _check_device(q, k_cache, v_cache)
    if q.dim() != 4:
        raise RuntimeError("q must be [B, S, H, D]")
    q = _check_q(q)
    B, S, H, D = q.shape
    k_cache, v_cache, (NB, BS, Hkv, _) = _check_kv(k_cache, v_cache, D)
    bt = _int32_on(block_tables, q.device)
    ctx = _int32_on(context_lens, q.device)
    if bt.dim() != 2 or bt.shape[0] != B:
        raise RuntimeError("block_tables must be [B, max_blocks]")
    if ctx.numel() != B:
        raise RuntimeError("context_lens must have one entry per sequence")
    out = q.new_empty(q.shape)
    if B == 0 or S == 0:
        return out
    with _DeviceGuard(index):
        ws, ws_bytes = _prefill_workspace(L, B, S, H, D, use_mfma, split, q.device)
        check(L.hs_prefill(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), dtype_code(k_cache.dtype),
            NB, bt.data_ptr(), ctx.data_ptr(), out.data_ptr(), B, S, H, Hkv, D, BS,
            bt.shape[1], float(scale), int(bool(use_mfma)),
            ws.data_ptr() if ws is not None else None, ws_bytes, _stream_at(index)))
    return out


def prefill_varlen(q, cu_seqlens_q, max_seqlen_q: int, k_cache, v_cache, block_tables,
                   context_lens, scale: float, use_mfma: bool, split: bool = True):
    """out[T, H, D] fp32 for ragged chunks via hs_prefill_varlen (split as for
    prefill)."""
    L = lib()
    index = _check_device(q, k_cache, v_cache)
    if q.dim() != 3:
        raise RuntimeError("q must be [total_tokens, H, D]")
    q = _check_q(q)
    T, H, D = q.shape
    k_cache, v_cache, (NB, BS, Hkv, _) = _check_kv(k_cache, v_cache, D)
    bt = _int32_on(block_tables, q.device)
    ctx = _int32_on(context_lens, q.device)
    cu = _int32_on(cu_seqlens_q, q.device)
    B = bt.shape[0]
    if cu.numel() != B + 1 or ctx.numel() != B:
        raise RuntimeError("cu_seqlens_q must be [B + 1] and context_lens [B]")
    out = q.new_empty(q.shape)
    if B == 0 or T == 0:
        return out
    with _DeviceGuard(index):
        ws, ws_bytes = _prefill_workspace(L, B, int(max_seqlen_q), H, D, use_mfma, split,
                                          q.device)
        check(L.hs_prefill_varlen(
            q.data_ptr(), cu.data_ptr(), int(max_seqlen_q), k_cache.data_ptr(),
            v_cache.data_ptr(), dtype_code(k_cache.dtype), NB, bt.data_ptr(), ctx.data_ptr(),
            out.data_ptr(), B, H, Hkv, D, BS, bt.shape[1], float(scale),
            int(bool(use_mfma)), ws.data_ptr() if ws is not None else None, ws_bytes,
            _stream_at(index)))
    return out


def choose_num_splits(num_seqs: int, num_heads: int, max_context: int) -> int:
    L = lib("v3 kernel")
    s = L.hs_choose_num_splits(int(num_seqs), int(num_heads), int(max_context))
    if s < 0:
        raise RuntimeError(L.hs_last_error().decode(errors="replace"))
    return int(s)


HOST_IDS = 896   # most block ids that fit a kernel's arguments (csrc/hs_private.h)


def _pages(pool):
    """(layers, blocks, bytes of one page) of pool [L, 2, NB, BS, Hkv, D]."""
    Ls, _, NB, BS, H, D = pool.shape
    return Ls, NB, BS * H * D * pool.element_size()


def kv_pack(pool, ids_dev, out) -> None:
    """out[n, L, 2, page] = pool[L, 2, NB, page][:, :, ids]  (bitwise)."""
    L = lib("KV pack HIP kernel")
    index = pool.get_device()
    with _DeviceGuard(index):
        check(L.hs_kv_pack(pool.data_ptr(), *_pages(pool), ids_dev.data_ptr(), ids_dev.numel(),
                           out.data_ptr(), _stream_at(index)))


def kv_unpack(pool, ids_dev, src) -> None:
    """pool[:, :, ids[i]] = src[i]  (bitwise; ids must not repeat)."""
    L = lib("KV unpack HIP kernel")
    index = pool.get_device()
    with _DeviceGuard(index):
        check(L.hs_kv_unpack(pool.data_ptr(), *_pages(pool), ids_dev.data_ptr(),
                             ids_dev.numel(), src.data_ptr(), _stream_at(index)))


def kv_pack_host_ids(pool, ids, out) -> None:
    """kv_pack with at most HOST_IDS ids in a contiguous int64 numpy array."""
    L = lib("KV pack HIP kernel")
    index = pool.get_device()
    with _DeviceGuard(index):
        check(L.hs_kv_pack_host_ids(pool.data_ptr(), *_pages(pool), ids.ctypes.data, ids.size,
                                    out.data_ptr(), _stream_at(index)))


def kv_unpack_host_ids(pool, ids, src) -> None:
    """kv_unpack with at most HOST_IDS ids in a contiguous int64 numpy array."""
    L = lib("KV unpack HIP kernel")
    index = pool.get_device()
    with _DeviceGuard(index):
        check(L.hs_kv_unpack_host_ids(pool.data_ptr(), *_pages(pool), ids.ctypes.data, ids.size,
                                      src.data_ptr(), _stream_at(index)))


def kv_gather(cache, block_tables_dev, length: int, out) -> None:
    """out[B, length, Hkv, D] = cache[NB, BS, Hkv, D] gathered through the tables."""
    L = lib("KV gather HIP kernel")
    NB, BS = cache.shape[:2]
    row = cache[0, 0].numel() * cache.element_size()
    B, MB = block_tables_dev.shape
    with _DeviceGuard(cache.get_device()):
        check(L.hs_kv_gather(cache.data_ptr(), NB, BS, row, block_tables_dev.data_ptr(), MB,
                             B, int(length), out.data_ptr(), _stream_at(cache.get_device())))


def _rows(x, Hkv: int, D: int):
    """(tensor, row stride in elements) of new K or V rows [n, Hkv, D].

    Accepts [n, Hkv, D] or [n, Hkv * D]; the rows may be strided (a slice of
    the fused QKV output) but each row's Hkv * D elements must be contiguous.
    """
    if x.dim() == 3:
        if tuple(x.shape[1:]) != (Hkv, D):
            raise RuntimeError(f"K/V rows must be [n, {Hkv}, {D}], got {tuple(x.shape)}")
        row_ok = x.stride(2) == 1 and x.stride(1) == D
    elif x.dim() == 2:
        if x.shape[1] != Hkv * D:
            raise RuntimeError(f"K/V rows must be [n, {Hkv * D}], got {tuple(x.shape)}")
        row_ok = x.stride(1) == 1
    else:
        raise RuntimeError(f"K/V rows must be [n, Hkv, D], got {tuple(x.shape)}")
    if not row_ok:
        x = x.contiguous()
    stride = x.stride(0) if x.shape[0] > 1 else Hkv * D
    return x, stride


def _check_write(k_cache, v_cache, k, v):
    """The caches are written in place: CUDA, contiguous, same shape/dtype.
    Returns their shape and device index."""
    shape = k_cache.shape
    if len(shape) != 4:
        raise RuntimeError("k_cache must be [NB, BS, Hkv, D]")
    if v_cache.shape != shape or v_cache.dtype is not k_cache.dtype:
        raise RuntimeError("k_cache and v_cache must have the same shape and dtype")
    index = k_cache.get_device()
    if (index < 0 or v_cache.get_device() != index or k.get_device() != index
            or v.get_device() != index):
        if not (k_cache.is_cuda and v_cache.is_cuda and k.is_cuda and v.is_cuda):
            raise RuntimeError("kv cache and new rows must be on CUDA")
        raise RuntimeError("kv cache and new rows must be on the same device")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise RuntimeError("kv cache must be contiguous (it is written in place)")
    return shape, index


def _same_rows(k, v, Hkv: int, D: int):
    k, ks = _rows(k, Hkv, D)
    v, vs = _rows(v, Hkv, D)
    if k.shape[0] != v.shape[0] or k.dtype != v.dtype:
        raise RuntimeError("k and v rows must have the same count and dtype")
    if ks != vs:
        k, v = k.contiguous(), v.contiguous()
        ks = vs = Hkv * D
    return k, v, ks


def kv_scatter(k_cache, v_cache, slots, k, v, wrap: bool = False) -> None:
    """k_cache.view(-1, Hkv, D)[slots] = k.to(cache dtype); same for v.  wrap:
    negative slots count from the end (otherwise they are skipped)."""
    L = lib("KV scatter HIP kernel")
    (NB, BS, Hkv, D), index = _check_write(k_cache, v_cache, k, v)
    k, v, stride = _same_rows(k, v, Hkv, D)
    n = k.shape[0]
    if slots.numel() != n:
        raise RuntimeError(f"{slots.numel()} slots for {n} rows")
    slots = torch.as_tensor(slots).to(device=k_cache.device, dtype=torch.int64).contiguous()
    with _DeviceGuard(index):
        head = (k_cache.data_ptr(), v_cache.data_ptr(), dtype_code(k_cache.dtype), NB * BS, Hkv, D)
        rows = (slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), dtype_code(k.dtype))
        if wrap:
            check(L.hs_kv_scatter_layers(*head, 1, 0, *rows, 0, D, stride, _stream_at(index)))
        else:
            check(L.hs_kv_scatter(*head, *rows, stride, _stream_at(index)))


def kv_scatter_layers(pool, slots, k, v) -> None:
    """pool[l, 0].view(-1, Hkv, D)[slots] = k[l].transpose(0, 1) for every layer of
    pool [L, 2, NB, BS, Hkv, D] and k, v [>= L, Hkv, T, D], in one launch;
    negative slots count from the end."""
    lib_ = lib("KV scatter HIP kernel")
    L, _, NB, BS, Hkv, D = pool.shape
    if L == 0:
        return
    (_, _, _, _), index = _check_write(pool[0, 0], pool[0, 1], k, v)
    T = slots.numel()
    for x in (k, v):
        if x.shape[0] < L:
            raise IndexError(f"index {x.shape[0]} is out of bounds for dimension 0 with size "
                             f"{x.shape[0]}")
        if tuple(x.shape[1:]) != (Hkv, T, D):
            raise RuntimeError(f"K/V must be [{L}, {Hkv}, {T}, {D}], got {tuple(x.shape)}")
    if k.dtype != v.dtype:
        raise RuntimeError("k and v rows must have the same count and dtype")
    if k.stride() != v.stride() or k.stride(3) != 1:
        k, v = k.contiguous(), v.contiguous()
    # a dim of one index has no stride of its own
    sl, sh, st = (k.stride(i) if k.shape[i] > 1 else n for i, n in
                  enumerate((Hkv * T * D, T * D, D)))
    slots = slots.to(device=pool.device, dtype=torch.int64).contiguous()
    with _DeviceGuard(index):
        check(lib_.hs_kv_scatter_layers(
            pool.data_ptr(), pool[0, 1].data_ptr(), dtype_code(pool.dtype), NB * BS, Hkv, D, L,
            2 * NB * BS * Hkv * D, slots.data_ptr(), T, k.data_ptr(), v.data_ptr(),
            dtype_code(k.dtype), sl, sh, st, _stream_at(index)))


def kv_append(k_cache, v_cache, block_tables, positions, k, v, seq_ids=None) -> None:
    """Row i -> slot block_tables[s][pos // BS] * BS + pos % BS of sequence
    s = seq_ids[i] (or i), pos = positions[i]; cast as kv_scatter."""
    L = lib("KV append HIP kernel")
    (NB, BS, Hkv, D), index = _check_write(k_cache, v_cache, k, v)
    k, v, stride = _same_rows(k, v, Hkv, D)
    n = k.shape[0]
    dev = k_cache.device
    bt = _int32_on(block_tables, dev)
    pos = _int32_on(positions, dev)
    if pos.numel() != n:
        raise RuntimeError(f"{pos.numel()} positions for {n} rows")
    sid = None if seq_ids is None else _int32_on(seq_ids, dev)
    if sid is not None and sid.numel() != n:
        raise RuntimeError(f"{sid.numel()} sequence ids for {n} rows")
    if sid is None and n > bt.shape[0]:
        raise RuntimeError("without seq_ids, row i uses table row i: more rows than tables")
    with _DeviceGuard(index):
        check(L.hs_kv_append(k_cache.data_ptr(), v_cache.data_ptr(), dtype_code(k_cache.dtype), NB,
                             BS, Hkv, D, bt.data_ptr(), bt.shape[0], bt.shape[1], pos.data_ptr(),
                             None if sid is None else sid.data_ptr(), n, k.data_ptr(),
                             v.data_ptr(), dtype_code(k.dtype), stride, _stream_at(index)))


def block_tables(packed_dev, B: int, width: int, out) -> None:
    """out[B, width] int32 from the packed [off[0..B], ids...] device buffer."""
    L = lib("block table HIP kernel")
    with _DeviceGuard(out.get_device()):
        check(L.hs_block_tables(packed_dev.data_ptr(), B, width, out.data_ptr(),
                                _stream_at(out.get_device())))


# ---------------------------------------------------------------------------
# rotary positions, whole prompts, pages in place
# ---------------------------------------------------------------------------


def _head_rows(x, heads: int, D: int):
    """_rows of [n, heads, D] or [n, heads * D], a copy of rows that overlap."""
    s = x.stride()
    if len(s) == 3 and s[2] == 1 and (s[1] == D or heads == 1) and s[0] >= heads * D:
        return x, s[0]
    x, row = _rows(x, heads, D)
    if row < heads * D:      # rows that overlap, such as an expanded one's
        return x.contiguous(), heads * D
    return x, row


def _contiguous_like(x, dtype):
    return torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format)


def _rotary_head(q, k, positions, inv_freq, axes, interleaved):
    """What both rotary calls pass first: (q, k, their row strides, the device index,
    the arguments from positions to D, and the tensors those point to)."""
    if q.dim() != 3 or k.dim() != 3:
        raise RuntimeError("q must be [n, H, D] and k [n, Hkv, D]")
    n, H, D = q.shape
    k_rows, Hkv, k_dim = k.shape
    index = q.get_device()
    if index < 0 or k.get_device() != index:
        raise RuntimeError("q and k must be on CUDA, on the same device")
    if k_rows != n or k_dim != D or k.dtype is not q.dtype:
        raise RuntimeError("k must have the rows, the head_dim and the dtype of q")
    dev = q.device
    pos = _whole_on("positions", positions, dev)
    n_axes = 1 if pos.dim() <= 1 else pos.shape[0]
    if pos.dim() > 2 or pos.numel() != n_axes * n:
        raise RuntimeError(f"positions must be [axes, {n}] or [{n}], got {tuple(pos.shape)}")
    freq = inv_freq
    if freq.dtype is not torch.float32 or freq.get_device() != index or not freq.is_contiguous():
        freq = freq.to(device=dev, dtype=torch.float32).contiguous()
    pairs = freq.numel()
    if not 0 < pairs <= D // 2:
        raise RuntimeError(f"inv_freq must have 1 to head_dim / 2 = {D // 2} entries, got {pairs}")
    pa = None if axes is None else _whole_on("axes", axes, dev)
    if pa is not None and pa.numel() != pairs:
        raise RuntimeError(f"{pa.numel()} axes for {pairs} rotary pairs")
    q, q_row = _head_rows(q, H, D)
    k, k_row = _head_rows(k, Hkv, D)
    middle = (pos.data_ptr(), n_axes, freq.data_ptr(), None if pa is None else pa.data_ptr(), pairs,
              1 if interleaved else 0, n, H, Hkv, D)
    return q, k, (q_row, k_row), index, middle, (pos, freq, pa)


def rotary(q, k, positions, inv_freq, axes, interleaved, out_dtype):
    """(q, k) turned by hs_rotary, contiguous, of out_dtype (q's when None)."""
    L = lib("rotary HIP kernel")
    out_dtype = out_dtype or q.dtype
    out_code = dtype_code(out_dtype)
    q, k, strides, index, middle, keep = _rotary_head(q, k, positions, inv_freq, axes, interleaved)
    q_out = _contiguous_like(q, out_dtype)
    k_out = _contiguous_like(k, out_dtype)
    with _DeviceGuard(index):
        check(L.hs_rotary(q.data_ptr(), k.data_ptr(), dtype_code(q.dtype), *strides, *middle,
                          q_out.data_ptr(), k_out.data_ptr(), out_code, _stream_at(index)))
    return q_out, k_out


def rotary_append(q, k, v, positions, inv_freq, k_cache, v_cache, block_tables, cache_positions,
                  seq_ids, axes, interleaved, out_dtype, keep_k):
    """(q, k or None) turned by hs_rotary_append, which writes k and v into the caches."""
    L = lib("rotary HIP kernel")
    out_dtype = out_dtype or q.dtype
    out_code = dtype_code(out_dtype)
    q, k, strides, index, middle, keep = _rotary_head(q, k, positions, inv_freq, axes, interleaved)
    n, Hkv, D = k.shape
    (NB, BS, cache_heads, cache_dim), cache_index = _check_write(k_cache, v_cache, k, v)
    if cache_index != index:
        raise RuntimeError("kv cache and new rows must be on the same device")
    if cache_heads != Hkv or cache_dim != D:
        raise RuntimeError(f"K/V rows must be [n, {cache_heads}, {cache_dim}], got {tuple(k.shape)}")
    if v.dtype is not k.dtype or v.shape[0] != n:
        raise RuntimeError("k and v rows must have the same count and dtype")
    if v.dim() == 3 and v.shape != k.shape:
        raise RuntimeError(f"K/V rows must be [n, {Hkv}, {D}], got {tuple(v.shape)}")
    v, v_row = _head_rows(v, Hkv, D)
    dev = q.device
    bt = _whole_on("block_tables", block_tables, dev)
    at = _whole_on("cache_positions", cache_positions, dev)
    sid = None if seq_ids is None else _whole_on("seq_ids", seq_ids, dev)
    if bt.dim() != 2:
        raise RuntimeError("block_tables must be [B, max_blocks]")
    B, MB = bt.shape
    if at.numel() != n:
        raise RuntimeError(f"{at.numel()} positions for {n} rows")
    if sid is not None and sid.numel() != n:
        raise RuntimeError(f"{sid.numel()} sequence ids for {n} rows")
    if sid is None and n > B:
        raise RuntimeError("without seq_ids, row i uses table row i: more rows than tables")
    q_out = _contiguous_like(q, out_dtype)
    k_out = _contiguous_like(k, out_dtype) if keep_k else None
    with _DeviceGuard(index):
        check(L.hs_rotary_append(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), dtype_code(q.dtype), *strides, v_row, *middle,
            q_out.data_ptr(), None if k_out is None else k_out.data_ptr(), out_code,
            k_cache.data_ptr(), v_cache.data_ptr(), dtype_code(k_cache.dtype), NB, BS, bt.data_ptr(),
            B, MB, at.data_ptr(), None if sid is None else sid.data_ptr(), _stream_at(index)))
    return q_out, k_out


def _heads(x):
    """(tensor, pointer, row stride, head stride): rows and heads any multiple of 16
    bytes apart, D elements of a head contiguous; a contiguous copy of anything else."""
    s0, s1, s2 = x.stride()
    ptr = x.data_ptr()
    unit = 15 // x.element_size()      # a mask: 3 or 7
    if (s2 != 1 or ptr & 15 or (s0 | s1) & unit or not 0 <= s0 <= 1 << 22
            or not 0 <= s1 <= 1 << 22):
        x = x.contiguous()
        if x.data_ptr() & 15:
            x = x.clone(memory_format=torch.contiguous_format)
        # (a dim of one index may still have any stride of its own)
        ptr, s0, s1 = x.data_ptr(), x.shape[1] * x.shape[2], x.shape[2]
    return x, ptr, s0, s1


def _overlap(out, x) -> bool:
    """Whether contiguous `out` and the range from x's first to its last element share
    a byte."""
    if not x.numel():
        return False
    p, size = x.data_ptr(), x.element_size()
    end = p + size * (1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride())))
    return p < out.data_ptr() + size * out.numel() and out.data_ptr() < end


def prompt_attention(q, k, v, cu_seqlens, max_seqlen: int, scale: float, out=None):
    """out[T, H, D] of q's dtype via hs_prompt_attention."""
    L = lib("prompt attention kernel")
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise RuntimeError("q must be [total_tokens, H, D], k and v [total_tokens, Hkv, D]")
    index = q.get_device()
    if index < 0 or k.get_device() != index or v.get_device() != index:
        raise RuntimeError("q, k and v must be on CUDA, on the same device")
    shape, kv_shape, dtype = q.shape, k.shape, q.dtype
    T, H, D = shape
    Hkv = kv_shape[1]
    if kv_shape != (T, Hkv, D) or v.shape != kv_shape:
        raise RuntimeError(f"k and v must be [{T}, Hkv, {D}], got {tuple(k.shape)}, {tuple(v.shape)}")
    if k.dtype is not dtype or v.dtype is not dtype:
        raise RuntimeError("q, k and v must have the same dtype")
    code = dtype_code(dtype)
    cu = _whole_on("cu_seqlens", cu_seqlens, q.device)
    B = cu.numel() - 1
    if cu.dim() != 1 or B < 0:
        raise RuntimeError("cu_seqlens must be [B + 1]")
    if out is None:
        out = _contiguous_like(q, dtype)
    elif (out.shape != shape or out.dtype is not dtype or out.get_device() != index
          or not out.is_contiguous() or out.data_ptr() % 16):
        raise RuntimeError("out must be a contiguous, 16-byte aligned tensor like q")
    elif _overlap(out, q) or _overlap(out, k) or _overlap(out, v):
        raise RuntimeError("out must not overlap q, k or v")
    max_len = int(max_seqlen)
    if max_len > T:        # (the library takes 32 bits)
        max_len = T
    elif max_len < 0:
        raise RuntimeError("max_seqlen must be positive or 0")
    q, qp, qr, qh = _heads(q)
    k, kp, kr, kh = _heads(k)
    v, vp, vr, vh = _heads(v)
    with _DeviceGuard(index):
        check(L.hs_prompt_attention(qp, kp, vp, code, qr, qh, kr, kh, vr, vh, cu.data_ptr(), B, T,
                                    max_len, H, Hkv, D, float(scale), out.data_ptr(),
                                    _stream_at(index)))
    return out


def _check_state(name: str, t, dim: int, index: int):
    """A tensor that a page operation changes in place."""
    if t.dtype is torch.int32 and t.dim() == dim and t.get_device() == index >= 0 and t.is_contiguous():
        return
    if t.dtype is not torch.int32 or t.dim() != dim or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous int32 tensor of {dim} dim(s): it is "
                           "written in place")
    raise RuntimeError(f"{name} must be on CUDA, on the device of the others")


def kv_copy(pool, src_dev, dst_dev) -> None:
    """pool[:, :, dst] = pool[:, :, src]  (bitwise, device int64 ids)."""
    L = lib("KV copy HIP kernel")
    index = pool.get_device()
    with _DeviceGuard(index):
        check(L.hs_kv_copy(pool.data_ptr(), *_pages(pool), src_dev.data_ptr(), dst_dev.data_ptr(),
                           src_dev.numel(), _stream_at(index)))


def kv_copy_host_ids(pool, src, dst) -> None:
    """kv_copy with at most HOST_IDS / 2 pairs in array("q")s."""
    L = lib("KV copy HIP kernel")
    index = pool.get_device()
    with _DeviceGuard(index):
        check(L.hs_kv_copy_host_ids(pool.data_ptr(), *_pages(pool), src.buffer_info()[0],
                                    dst.buffer_info()[0], len(src), _stream_at(index)))


def kv_find_free(ref_counts, n: int):
    """int32 [n]: the lowest free blocks, -1 past the last."""
    L = lib("free block search HIP kernel")
    index = ref_counts.get_device()
    _check_state("ref_counts", ref_counts, 1, index)
    out = ref_counts.new_empty(n)
    with _DeviceGuard(index):
        check(L.hs_kv_find_free(ref_counts.data_ptr(), ref_counts.numel(), out.data_ptr(), n,
                                _stream_at(index)))
    return out


def kv_fork(pool, block_tables, context_lens, ref_counts, parents, children, fresh):
    """int32 [n], 1 where row children[i] became a fork of row parents[i]."""
    L = lib("KV fork HIP kernel")
    index = pool.get_device()
    _check_state("block_tables", block_tables, 2, index)
    _check_state("context_lens", context_lens, 1, index)
    _check_state("ref_counts", ref_counts, 1, index)
    B, MB = block_tables.shape
    n = parents.numel()
    if context_lens.numel() != B or ref_counts.numel() != pool.shape[2]:
        raise RuntimeError("context_lens must have one entry per table row, ref_counts one per block")
    if children.numel() != n or fresh.numel() != n:
        raise RuntimeError("parents, children and fresh must have the same length")
    forked = torch.empty_like(parents)
    with _DeviceGuard(index):
        check(L.hs_kv_fork(pool.data_ptr(), *_pages(pool), pool.shape[3], block_tables.data_ptr(), B, MB,
                           context_lens.data_ptr(), ref_counts.data_ptr(), parents.data_ptr(),
                           children.data_ptr(), fresh.data_ptr(), n, forked.data_ptr(),
                           _stream_at(index)))
    return forked


def kv_free(block_tables, context_lens, ref_counts, rows) -> None:
    L = lib("KV free HIP kernel")
    index = ref_counts.get_device()
    _check_state("block_tables", block_tables, 2, index)
    _check_state("context_lens", context_lens, 1, index)
    _check_state("ref_counts", ref_counts, 1, index)
    B, MB = block_tables.shape
    if context_lens.numel() != B:
        raise RuntimeError("context_lens must have one entry per table row")
    with _DeviceGuard(index):
        check(L.hs_kv_free(block_tables.data_ptr(), B, MB, context_lens.data_ptr(), ref_counts.data_ptr(),
                           ref_counts.numel(), rows.data_ptr(), rows.numel(), _stream_at(index)))


def kv_compact(pool, block_tables, ref_counts):
    """(moved_to int32 [NB], live int32 [1])."""
    L = lib("KV compaction HIP kernel")
    index = pool.get_device()
    _check_state("block_tables", block_tables, 2, index)
    _check_state("ref_counts", ref_counts, 1, index)
    NB = pool.shape[2]
    if ref_counts.numel() != NB:
        raise RuntimeError("ref_counts must have one entry per block")
    need = L.hs_kv_compact_workspace_bytes(NB)
    made = ref_counts.new_empty(NB + 1 + (need + 3) // 4)
    moved_to, live, ws = made[:NB], made[NB:NB + 1], made[NB + 1:]
    with _DeviceGuard(index):
        check(L.hs_kv_compact(pool.data_ptr(), *_pages(pool), block_tables.data_ptr(),
                              *block_tables.shape, ref_counts.data_ptr(), moved_to.data_ptr(),
                              live.data_ptr(), ws.data_ptr(), need, _stream_at(index)))
    return moved_to, live

# ---------------------------------------------------------------------------
# the 4-bit cache, and decode through a window
# ---------------------------------------------------------------------------

_Q4_DIMS = {20: 32, 40: 64, 80: 128, 160: 256}   # record bytes -> head_dim


def _q4_shape(k_cache, v_cache):
    """(NB, BS, Hkv, D) of a pair of 4-bit caches, and their device index."""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise RuntimeError("k_cache and v_cache must be [NB, BS, Hkv, record_bytes(D)]")
    if k_cache.dtype is not torch.uint8 or v_cache.dtype is not torch.uint8:
        raise RuntimeError("a 4-bit cache must be uint8")
    D = _Q4_DIMS.get(shape[3])
    if D is None:
        raise RuntimeError(f"a 4-bit cache has records of {sorted(_Q4_DIMS)} bytes, got {shape[3]}")
    index = k_cache.get_device()
    if index < 0 or v_cache.get_device() != index:
        raise RuntimeError("kv cache must be on CUDA, on one device")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise RuntimeError("a 4-bit cache must be contiguous")
    return (shape[0], shape[1], shape[2], D), index


def _q4_rows(block_tables, positions, seq_ids, n, device):
    """(tables, positions, sequence ids or None) of n rows, int32 on the device."""
    bt = _whole_on("block_tables", block_tables, device)
    at = _whole_on("positions", positions, device)
    sid = None if seq_ids is None else _whole_on("seq_ids", seq_ids, device)
    if bt.dim() != 2:
        raise RuntimeError("block_tables must be [B, max_blocks]")
    if n is None:
        n = at.numel()
    if at.numel() != n:
        raise RuntimeError(f"{at.numel()} positions for {n} rows")
    if sid is not None and sid.numel() != n:
        raise RuntimeError(f"{sid.numel()} sequence ids for {n} rows")
    if sid is None and n > bt.shape[0]:
        raise RuntimeError("without seq_ids, row i uses table row i: more rows than tables")
    return bt, at, sid


def q4_append(k_cache, v_cache, block_tables, positions, k, v, seq_ids) -> None:
    """Rows of k and v into a 4-bit cache via hs_q4_append."""
    L = lib("4-bit KV append HIP kernel")
    (NB, BS, Hkv, D), index = _q4_shape(k_cache, v_cache)
    if k.get_device() != index or v.get_device() != index:
        raise RuntimeError("kv cache and new rows must be on the same device")
    code = dtype_code(k.dtype)
    for x in (k, v):
        if x.dim() == 3 and x.shape[1:] != (Hkv, D):
            raise RuntimeError(f"K/V rows must be [n, {Hkv}, {D}], got {tuple(x.shape)}")
    k, k_row = _head_rows(k, Hkv, D)
    v, v_row = _head_rows(v, Hkv, D)
    n = k.shape[0]
    if v.shape[0] != n or v.dtype is not k.dtype:
        raise RuntimeError("k and v rows must have the same count and dtype")
    bt, at, sid = _q4_rows(block_tables, positions, seq_ids, n, k_cache.device)
    with _DeviceGuard(index):
        check(L.hs_q4_append(k_cache.data_ptr(), v_cache.data_ptr(), NB, BS, Hkv, D, bt.data_ptr(),
                             bt.shape[0], bt.shape[1], at.data_ptr(),
                             None if sid is None else sid.data_ptr(), n, k.data_ptr(), v.data_ptr(),
                             code, k_row, v_row, _stream_at(index)))


def q4_read(k_cache, v_cache, block_tables, positions, seq_ids, dtype):
    """(k, v) [n, Hkv, D] out of a 4-bit cache via hs_q4_read."""
    L = lib("4-bit KV read HIP kernel")
    (NB, BS, Hkv, D), index = _q4_shape(k_cache, v_cache)
    dtype = dtype or torch.float16
    code = dtype_code(dtype)
    dev = k_cache.device
    bt, at, sid = _q4_rows(block_tables, positions, seq_ids, None, dev)
    n = at.numel()
    k = torch.empty((n, Hkv, D), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    with _DeviceGuard(index):
        check(L.hs_q4_read(k_cache.data_ptr(), v_cache.data_ptr(), NB, BS, Hkv, D, bt.data_ptr(),
                           bt.shape[0], bt.shape[1], at.data_ptr(),
                           None if sid is None else sid.data_ptr(), n, k.data_ptr(), v.data_ptr(), code,
                           _stream_at(index)))
    return k, v


def _whole_number(what: str, x) -> int:
    """A size that the library takes as 32 bits: sizes past that see no more than those."""
    x = operator.index(x)
    if x < 0:
        raise RuntimeError(f"{what} must not be negative, got {x}")
    return min(x, 0x7fffffff)


def _span_decode(L, query, call, head, q, k_cache, v_cache, NB, BS, Hkv, block_tables, context_lens,
                 scale, window, sinks, index):
    """hs_q4_decode or hs_window_decode; head: what the query takes first."""
    B, H, D = q.shape
    dev = q.device
    bt = _whole_on("block_tables", block_tables, dev)
    ctx = _whole_on("context_lens", context_lens, dev)
    if bt.dim() != 2 or bt.shape[0] != B:
        raise RuntimeError("block_tables must be [B, max_blocks]")
    if ctx.numel() != B:
        raise RuntimeError("context_lens must have one entry per sequence")
    window, sinks = _whole_number("window", window), _whole_number("sinks", sinks)
    if q.data_ptr() & 15:
        q = q.clone()
    out = q.new_empty(q.shape)
    if B == 0:
        return out
    MB = bt.shape[1]
    sizes = (*head, B, H, Hkv, D, BS, MB, window, sinks)
    key = (query.__name__, index, sizes)
    ws_bytes = known = _WS_SIZES.get(key)
    with _DeviceGuard(index):
        if known is None:
            ws_bytes = query(*sizes)
        ws = q.new_empty((ws_bytes + 3) // 4) if ws_bytes else None
        check(call(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), *head, NB, bt.data_ptr(),
                   ctx.data_ptr(), out.data_ptr(), B, H, Hkv, D, BS, MB, float(scale), window, sinks,
                   None if ws is None else ws.data_ptr(), ws_bytes, _stream_at(index)))
    if known is None:   # a size of 0 too, now that the call has not refused it
        if len(_WS_SIZES) >= _WS_SIZES_MAX:
            _WS_SIZES.clear()
        _WS_SIZES[key] = ws_bytes
    return out


def q4_decode(q, k_cache, v_cache, block_tables, context_lens, scale: float, window: int, sinks: int):
    """out[B, H, D] fp32: decode over a 4-bit cache via hs_q4_decode."""
    L = lib("4-bit attention HIP kernel")
    (NB, BS, Hkv, D), index = _q4_shape(k_cache, v_cache)
    if q.dim() != 3 or q.shape[2] != D:
        raise RuntimeError(f"q must be [B, H, {D}], got {tuple(q.shape)}")
    if q.get_device() != index:
        raise RuntimeError("q and the kv cache must be on the same device")
    return _span_decode(L, L.hs_q4_decode_workspace_bytes, L.hs_q4_decode, (), _check_q(q), k_cache,
                        v_cache, NB, BS, Hkv, block_tables, context_lens, scale, window, sinks, index)


def window_decode(q, k_cache, v_cache, block_tables, context_lens, scale: float, window: int, sinks: int):
    """out[B, H, D] fp32: decode through a window via hs_window_decode."""
    L = lib("window attention HIP kernel")
    index = _check_device(q, k_cache, v_cache)
    if q.dim() != 3:
        raise RuntimeError("q must be [B, H, D]")
    q = _check_q(q)
    k_cache, v_cache, (NB, BS, Hkv, _) = _check_kv(k_cache, v_cache, q.shape[2])
    return _span_decode(L, L.hs_window_decode_workspace_bytes, L.hs_window_decode,
                        (dtype_code(k_cache.dtype),), q, k_cache, v_cache, NB, BS, Hkv, block_tables,
                        context_lens, scale, window, sinks, index)
