"""Fused decode ops backed by libdecodebench_hip.so (HIP, gfx950).

Each op takes torch tensors on the GPU, allocates its output with
``torch.empty`` and launches one kernel (two where K is split over workgroups
or an F4 merge takes a launch of its own, up to three for paged attention) on
``torch.cuda.current_stream()``
through the C ABI declared in ``include/decodebench_hip.h``.  No op allocates
inside the library, synchronises, or reads device memory on the host, so the
ops work as ``Sequence`` stages, inside a ``profile(fused=...)`` callable, and
under ``torch.cuda.graph`` capture.

This follows the plug-in pattern of the reference's custom-kernel example
(examples/custom_kernel/bindings.cpp:13-30: output from ``empty_like``, launch
on the current stream) with ctypes over a C ABI instead of a torch extension.

There is no fallback: if the HIP library is missing or cannot be loaded the
ops raise ``RuntimeError`` naming the build command.

A call that needs nothing but its checks, an output and the launch goes
through ``_fastcall`` (csrc/fastcall.cpp), which does the same in native code;
it answers None for everything else, and without it (built for another torch)
the Python steps below do all of it.
"""

from __future__ import annotations

import ctypes as C
import math
import sys
import threading
from contextlib import nullcontext
from pathlib import Path
from typing import NamedTuple

LIB_PATH = Path(__file__).resolve().parent / "lib" / "libdecodebench_hip.so"
FAST_PATH = Path(__file__).resolve().parent / "lib" / "_fastcall.so"

DB_OK = 0
DB_ERR_INVALID = -1
DB_ERR_UNSUPPORTED = -2
DTYPE_F16 = 0
DTYPE_FP8_E4M3 = 1
DTYPE_BF16 = 2

_lock = threading.Lock()
_lib = None
_fast = None  # the _fastcall module, once the library is loaded
_cu_cache: dict[int, int] = {}
_ws_cache: dict[tuple, object] = {}
_captured_ws: dict[tuple, object] = {}  # workspaces made under graph capture (kept alive)

_p = C.c_void_p
_i = C.c_int
_ll = C.c_longlong


class _PagedCache(C.Structure):
    """``db_paged_cache`` of the C ABI."""

    _fields_ = [("k", _p), ("v", _p), ("k_scale", _p), ("v_scale", _p),
                ("k_page_stride", _ll), ("k_head_stride", _ll), ("k_token_stride", _ll),
                ("v_page_stride", _ll), ("v_head_stride", _ll), ("v_token_stride", _ll),
                ("pages", _i), ("page_size", _i), ("Hkv", _i), ("D", _i), ("dtype", _i)]


class _Moe(C.Structure):
    """``db_moe`` of the C ABI."""

    _fields_ = [("wg", _p), ("wu", _p), ("wd", _p), ("sg", _p), ("su", _p), ("sd", _p),
                ("E", _i), ("H", _i), ("I", _i), ("dtype", _i), ("w_dtype", _i)]


def load_library():
    """Load the HIP library (after torch, so both share one HIP runtime)."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        import torch  # noqa: F401  -- torch's libamdhip64 must be loaded first

        if not LIB_PATH.exists():
            raise RuntimeError(
                f"HIP library {LIB_PATH} is not built; run "
                "`python -m decodebench_amd.build` (hipcc, gfx950)")
        lib = C.CDLL(str(LIB_PATH))
        protos = {
            "db_abi_version": (_i, []),
            "db_last_error": (C.c_char_p, []),
            "db_device_cu_count": (_i, [C.POINTER(_i)]),
            "db_f1_rmsnorm_gemv": (_i, [_p, _p, _p, _p, _p, _i, _i, _i, C.c_float, _i, _p]),
            "db_f2_gateup_swiglu": (_i, [_p, _p, _p, _p, _p, _p, _i, _i, _i, _i, _p]),
            "db_f2_rmsnorm_gateup_swiglu": (_i, [_p, _p, _p, _p, _p, _p, _p, _i, _i, _i,
                                                 C.c_float, _i, _p]),
            "db_gemv": (_i, [_p, _p, _p, _p, _i, _i, _i, _i, _p]),
            "db_gemv_workspace_bytes": (C.c_size_t, [_i, _i, _i, _i, _i, _i]),
            "db_gemv_ws": (_i, [_p, _p, _p, _p, _p, _p, _p, _p, C.c_size_t, _i, _i, _i, C.c_float,
                                _i, _p]),
            "db_f4_default_splits": (_i, [_i, _i, _i, _i]),
            "db_f4_workspace_bytes": (C.c_size_t, [_i, _i, _i, _i, _i, _i]),
            "db_f4_splitkv": (_i, [_p, _p, _p, _p, _p, C.c_size_t, _i, _i, _i, _i, _i, _i,
                                   C.c_float, _p]),
            "db_f4_splitkv_noalloc": (_i, [_p, _p, _p, _p, _i, _i, _i, _i, _i, _i, C.c_float,
                                           _p]),
            "db_paged_plan": (_i, [_p, _p, _p, _ll, _i, _p, _i, _p, _i, _i, _i, _p, _p, _p, _p,
                                   _p, _p]),
            "db_rope_append": (_i, [_p, _ll, _p, _i, _p, _p, _p, _i, _i, C.POINTER(_PagedCache),
                                    _p, _i, _i, _i, _p]),
            "db_paged_attention_workspace_bytes": (C.c_size_t, [_i, _i, _i, _i, _i, _i,
                                                               C.POINTER(C.c_size_t)]),
            "db_paged_attention": (_i, [_p, _ll, _ll, _p, C.POINTER(_PagedCache), _p, _ll, _i, _p,
                                        _p, _i, _i, _i, _i, C.c_float, _i, _i, _i, _p,
                                        C.c_size_t, _p]),
            "db_quantize_blocks": (_i, [_p, _ll, _p, _p, _ll, _ll, _i, _i, _i, _p]),
            "db_gemm_blocks_workspace_bytes": (C.c_size_t, [_i, _i, _i, _i]),
            "db_gemm_blocks": (_i, [_p, _ll, _p, _ll, _ll, _p, _p, _p, _i, _i, _i, _i, _i, _p,
                                    C.c_size_t, _p]),
            "db_moe_route_workspace_bytes": (C.c_size_t, [_i, _i, _i]),
            "db_moe_route": (_i, [_p, _ll, _p, _p, _p, _i, _i, _i, _i, _i, _i, _p, C.c_size_t,
                                  _p]),
            "db_moe_experts_workspace_bytes": (C.c_size_t, [C.POINTER(_Moe), _i, _i]),
            "db_moe_experts": (_i, [_p, _ll, _p, _p, C.POINTER(_Moe), _p, _i, _i, _p, C.c_size_t,
                                    _p]),
            "db_moe_layer_workspace_bytes": (C.c_size_t, [C.POINTER(_Moe), _i, _i]),
            "db_moe_layer": (_i, [_p, _ll, _p, C.POINTER(_Moe), _p, _i, _i, _i, _p, C.c_size_t,
                                  _p]),
            "db_stream_read": (_i, [_p, C.c_size_t, _i, C.c_uint, _p, _p]),
            "db_stream_capture_id": (_i, [_p, C.POINTER(C.c_ulonglong)]),
            "db_tune": (_i, [C.c_char_p, _i]),
            "db_tune_get": (_i, [C.c_char_p, C.POINTER(_i)]),
            "db_f4_launch_info": (_i, [_i, _i, _i, _i, _i, C.POINTER(_i), C.POINTER(_i)]),
            "db_null_kernel": (_i, [_p]),
        }
        for name, (res, args) in protos.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        if lib.db_abi_version() != 1:
            raise RuntimeError("libdecodebench_hip.so ABI version mismatch")
        _load_fast(lib)
        _lib = lib
        return lib


def fast_built_for() -> str:
    """The torch and the Python that a ``_fastcall`` module has to be built for
    to be used: it holds their object layouts, which an import does not check."""
    torch = _torch or _torch_mod()
    return f"torch {torch.__version__}, {sys.implementation.cache_tag}"


def _load_fast(lib) -> None:
    """Load the native call path and hand it the library's entry points."""
    global _fast
    import importlib.machinery
    import importlib.util

    torch = _torch or _torch_mod()
    get_device = getattr(torch._C, "_cuda_getDevice", None)
    if get_device is None or not FAST_PATH.exists():
        return
    loader = importlib.machinery.ExtensionFileLoader("_fastcall", str(FAST_PATH))
    spec = importlib.util.spec_from_file_location("_fastcall", str(FAST_PATH), loader=loader)
    try:
        mod = importlib.util.module_from_spec(spec)
        loader.exec_module(mod)
    except ImportError:  # built against another torch whose symbols differ
        return
    if getattr(mod, "built_for", None) != fast_built_for():
        return
    entry = tuple(C.cast(getattr(lib, name), C.c_void_p).value for name in (
        "db_f1_rmsnorm_gemv", "db_f2_gateup_swiglu", "db_f2_rmsnorm_gateup_swiglu", "db_gemv",
        "db_f4_default_splits", "db_f4_workspace_bytes", "db_f4_splitkv",
        "db_stream_capture_id", "db_gemv_workspace_bytes", "db_gemv_ws", "db_paged_plan",
        "db_rope_append", "db_paged_attention_workspace_bytes", "db_paged_attention",
        "db_quantize_blocks", "db_gemm_blocks_workspace_bytes", "db_gemm_blocks",
        "db_moe_route_workspace_bytes", "db_moe_route", "db_moe_experts_workspace_bytes",
        "db_moe_experts", "db_moe_layer_workspace_bytes", "db_moe_layer"))
    mod.init(entry, _raw_stream, get_device, _ws_cache, _cu_cache)
    _fast = mod


def _check(rc: int, what: str) -> None:
    if rc == DB_OK:
        return
    msg = load_library().db_last_error().decode(errors="replace")
    if rc == DB_ERR_INVALID:
        raise ValueError(f"{what}: {msg}")
    if rc == DB_ERR_UNSUPPORTED:
        raise NotImplementedError(f"{what}: {msg}")
    raise RuntimeError(f"{what} failed (HIP error {rc}): {msg}")


def _same_device(*named) -> None:
    """All tensors of one call must live on one GPU."""
    dev = named[0][0].device
    for t, name in named[1:]:
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, expected {dev} like {named[0][1]}")


_torch = None
_raw_stream = None


def _torch_mod():
    """torch, imported once, and the fastest handle to the current stream."""
    global _torch, _raw_stream
    if _torch is None:
        import torch

        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        _raw_stream = raw if raw is not None else (
            lambda idx: torch.cuda.current_stream(idx).cuda_stream)
        _torch = torch
    return _torch


def _gpu_tensors(*items) -> int:
    """Check ``(tensor, name, dtype or None)`` items in one pass: a torch
    tensor on a GPU, of that dtype, contiguous, all on one GPU.  Returns the
    GPU's index.  Every check is a C-level attribute read, so the hot call
    stays cheap."""
    torch = _torch or _torch_mod()
    idx, first = -1, None
    for t, name, dt in items:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not t.is_cuda:
            raise ValueError(f"{name} must be on a GPU device (got {t.device})")
        if dt is not None and t.dtype != dt:
            raise TypeError(f"{name} must be {dt} (got {t.dtype})")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        d = t.get_device()
        if first is None:
            idx, first = d, name
        elif d != idx:
            raise ValueError(f"{name} is on cuda:{d}, expected cuda:{idx} like {first}")
    return idx


def _on_device(idx: int):
    """Makes GPU ``idx`` current where it is not."""
    torch = _torch
    return nullcontext() if torch.cuda.current_device() == idx else torch.cuda.device(idx)


def _launch(fn, idx: int, what: str, *args) -> None:
    """``fn(*args, stream)`` on GPU ``idx`` (made current if it is not) and
    its current stream; a non-zero status raises."""
    torch = _torch
    if torch.cuda.current_device() == idx:
        rc = fn(*args, _raw_stream(idx))
    else:
        with torch.cuda.device(idx):
            rc = fn(*args, _raw_stream(idx))
    if rc:
        _check(rc, what)


def _output(shape, idx: int, out, name: str = "out"):
    """A new fp16 tensor of ``shape`` on GPU ``idx``, or ``out`` checked."""
    torch = _torch
    if out is None:
        return torch.empty(shape, dtype=torch.float16, device=torch.device("cuda", idx))
    _gpu_tensors((out, name, torch.float16))
    if out.get_device() != idx:
        raise ValueError(f"{name} is on cuda:{out.get_device()}, expected cuda:{idx}")
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)} (got {tuple(out.shape)})")
    return out


def _apart(out, *named) -> None:
    """Refuse an ``out`` that shares memory with an input, from its first element
    to its last: some workgroups write it while others still read."""
    if out.numel() == 0:
        return
    begin = out.data_ptr()
    end = begin + out.numel() * out.element_size()
    for t, name in named:
        if t is None or t.numel() == 0:
            continue
        first = t.data_ptr()
        last = sum((n - 1) * step for n, step in zip(t.shape, t.stride()))
        if first < end and begin < first + (last + 1) * t.element_size():
            raise ValueError(f"out must not share memory with {name}")


def cu_count(device=None) -> int:
    """Compute units of a GPU (index, torch.device or None for the current one)."""
    if isinstance(device, int) and device in _cu_cache:
        return _cu_cache[device]
    torch = _torch or _torch_mod()
    if isinstance(device, int):
        idx = device
    else:
        dev = torch.device("cuda" if device is None else device)
        idx = dev.index if dev.index is not None else torch.cuda.current_device()
    if idx not in _cu_cache:
        _cu_cache[idx] = torch.cuda.get_device_properties(idx).multi_processor_count
    return _cu_cache[idx]


def null_kernel(device=None) -> None:
    """Launch the library's empty kernel on the current stream (the
    launch-overhead probe of ``decodebench_amd.calibrate``)."""
    import torch

    dev = torch.device("cuda" if device is None else device)
    with torch.cuda.device(dev):
        rc = load_library().db_null_kernel(torch.cuda.current_stream(dev).cuda_stream)
    _check(rc, "db_null_kernel")


def stream_read(src, kb_per_wave: int = 8, sink=None) -> None:
    """Launch the read-only streaming probe over all of ``src`` (a contiguous
    GPU tensor of a whole number of ``kb_per_wave`` KB) on the current stream.

    ``src`` should hold zeros: the probe stores to ``sink`` only when the
    folded data equals its (non-zero) magic value, so it then writes
    nothing.  ``sink`` (int32, >= nbytes/16 elements) is allocated when not
    given; pass one to keep the call allocation-free (graph capture)."""
    import torch

    idx = _gpu_tensors((src, "src", None))
    nbytes = src.numel() * src.element_size()
    if sink is None:
        sink = _torch.empty(max(1, nbytes // 16), dtype=_torch.int32, device=src.device)
    _launch((_lib or load_library()).db_stream_read, idx, "db_stream_read", src.data_ptr(),
            nbytes, int(kb_per_wave), 0x9E3779B9, sink.data_ptr())


def tune(key: str, value: int) -> None:
    """Set a launch-geometry knob of the library (for tuning sweeps).  The
    library keeps one set of knobs per host thread: the value applies to
    the launches this thread makes."""
    _check(load_library().db_tune(key.encode(), int(value)), "db_tune")


def f4_launch_info(B: int, Hq: int, Hkv: int, L: int, S: int) -> tuple[int, int]:
    """(splits, launches) of an F4 call of this shape on the current device:
    launches is 1 when the split merge runs in the same launch (or there is
    one split), 2 when it takes a second launch."""
    s, n = C.c_int(0), C.c_int(0)
    _check(load_library().db_f4_launch_info(B, Hq, Hkv, L, S, C.byref(s), C.byref(n)),
           "db_f4_launch_info")
    return s.value, n.value


def tuned(key: str) -> int:
    """This thread's current value of a launch-geometry knob."""
    v = C.c_int(0)
    _check(load_library().db_tune_get(key.encode(), C.byref(v)), "db_tune_get")
    return v.value


def _weights(W, w_scale, name: str, N: int, K: int):
    """(dtype code, scale pointer, items to check) for an fp16 or e4m3 weight
    matrix."""
    torch = _torch or _torch_mod()
    if W.dtype == torch.float16:
        if w_scale is not None:
            raise ValueError(f"{name}: fp16 weights take no scale")
        return DTYPE_F16, None, ()
    if W.dtype in (torch.float8_e4m3fn, torch.uint8):
        if w_scale is None:
            raise ValueError(f"{name}: fp8 weights need a per-row fp32 scale")
        if not isinstance(w_scale, torch.Tensor) or tuple(w_scale.shape) != (N,):
            raise ValueError(f"{name} scale must be a tensor of shape ({N},)")
        return DTYPE_FP8_E4M3, w_scale.data_ptr(), ((w_scale, f"{name} scale", torch.float32),)
    raise TypeError(f"{name}: unsupported weight dtype {W.dtype}")


def _as_2d(x, name: str):
    if x.dim() == 1:
        return x.unsqueeze(0), True
    if x.dim() != 2:
        raise ValueError(f"{name} must be [K] or [B, K] (got {tuple(x.shape)})")
    return x, False


def _split_launch(out, x, g, W, W2, s, s2, y, B: int, K: int, N: int, eps: float, dt: int,
                  idx: int) -> bool:
    """Launch a GEMV op with K split over workgroups, in a workspace from
    torch's allocator, where the library would (``db_gemv_workspace_bytes``).
    Returns whether it did; a call with its own ``out`` allocates nothing, and
    one that is refused or has no room for the workspace is left to the entry
    point without one."""
    torch, lib = _torch, _lib or load_library()
    if out is not None or B < 9 or torch.cuda.current_device() != idx:
        return False
    nbytes = lib.db_gemv_workspace_bytes(g is not None, W2 is not None, B, K, N, dt)
    if nbytes == 0:
        return False
    try:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=y.device)
    except torch.cuda.OutOfMemoryError:
        return False
    return lib.db_gemv_ws(x, g, W, W2, s, s2, y.data_ptr(), ws.data_ptr(), nbytes, B, K, N, eps,
                          dt, _raw_stream(idx)) == DB_OK


def f1_rmsnorm_gemv(x, g, W, eps: float = 1e-6, w_scale=None, out=None):
    """F1: ``F.linear(rmsnorm(x, g, eps), W)`` in one kernel.

    x [B,K] (or [K]) fp16, g [K] fp16, W [N,K] fp16 (or e4m3 + w_scale [N]).
    Returns [B,N] fp16 (or [N] for a 1-D x), written to ``out`` if given."""
    if out is None and _fast is not None:
        y = _fast.f1(x, g, W, eps, w_scale)
        if y is not None:
            return y
    torch = _torch or _torch_mod()
    x2, squeeze = _as_2d(x, "x")
    B, K = x2.shape
    if W.dim() != 2 or W.shape[1] != K or g.shape != (K,):
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, g {tuple(g.shape)}, "
                         f"W {tuple(W.shape)}")
    N = W.shape[0]
    dt, sp, sc = _weights(W, w_scale, "W", N, K)
    idx = _gpu_tensors((x, "x", torch.float16), (g, "g", torch.float16), (W, "W", None), *sc)
    y = _output((B, N), idx, out)
    if out is not None:
        _apart(out, (x2, "x"))
    if not _split_launch(out, x2.data_ptr(), g.data_ptr(), W.data_ptr(), None, sp, None, y, B, K,
                         N, float(eps), dt, idx):
        _launch((_lib or load_library()).db_f1_rmsnorm_gemv, idx, "db_f1_rmsnorm_gemv",
                x2.data_ptr(), g.data_ptr(), W.data_ptr(), sp, y.data_ptr(), B, K, N,
                float(eps), dt)
    return y[0] if squeeze else y


def f2_gateup_swiglu(x, Wg, Wu, sg=None, su=None, out=None):
    """F2: ``silu(F.linear(x, Wg)) * F.linear(x, Wu)`` in one kernel.

    x [B,K] (or [K]) fp16, Wg/Wu [N,K] fp16 (or e4m3 + per-row scales)."""
    if out is None and _fast is not None:
        y = _fast.f2(x, Wg, Wu, sg, su)
        if y is not None:
            return y
    torch = _torch or _torch_mod()
    x2, squeeze = _as_2d(x, "x")
    B, K = x2.shape
    if Wg.dim() != 2 or Wg.shape != Wu.shape or Wg.shape[1] != K or Wg.dtype != Wu.dtype:
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, Wg {tuple(Wg.shape)}, "
                         f"Wu {tuple(Wu.shape)}")
    N = Wg.shape[0]
    dt, sgp, sgc = _weights(Wg, sg, "Wg", N, K)
    _, sup, suc = _weights(Wu, su, "Wu", N, K)
    idx = _gpu_tensors((x, "x", torch.float16), (Wg, "Wg", None), (Wu, "Wu", None), *sgc, *suc)
    y = _output((B, N), idx, out)
    if out is not None:
        _apart(out, (x2, "x"))
    if not _split_launch(out, x2.data_ptr(), None, Wg.data_ptr(), Wu.data_ptr(), sgp, sup, y, B,
                         K, N, 0.0, dt, idx):
        _launch((_lib or load_library()).db_f2_gateup_swiglu, idx, "db_f2_gateup_swiglu",
                x2.data_ptr(), Wg.data_ptr(), Wu.data_ptr(), sgp, sup, y.data_ptr(), B, K, N, dt)
    return y[0] if squeeze else y


def f2_rmsnorm_gateup_swiglu(x, g, Wg, Wu, eps: float = 1e-6, sg=None, su=None, out=None):
    """RMSNorm -> F2 in one kernel: ``f2_gateup_swiglu(rmsnorm(x, g, eps), Wg, Wu)``
    with the normalised activations kept on chip (the post-attention half
    of the decode-layer chain).

    x [B,K] (or [K]) fp16, g [K] fp16, Wg/Wu [N,K] fp16 (or e4m3 + per-row
    scales).  Returns [B,N] fp16 (or [N])."""
    if out is None and _fast is not None:
        y = _fast.f2n(x, g, Wg, Wu, eps, sg, su)
        if y is not None:
            return y
    torch = _torch or _torch_mod()
    x2, squeeze = _as_2d(x, "x")
    B, K = x2.shape
    if (Wg.dim() != 2 or Wg.shape != Wu.shape or Wg.shape[1] != K or Wg.dtype != Wu.dtype
            or g.shape != (K,)):
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, g {tuple(g.shape)}, "
                         f"Wg {tuple(Wg.shape)}, Wu {tuple(Wu.shape)}")
    N = Wg.shape[0]
    dt, sgp, sgc = _weights(Wg, sg, "Wg", N, K)
    _, sup, suc = _weights(Wu, su, "Wu", N, K)
    idx = _gpu_tensors((x, "x", torch.float16), (g, "g", torch.float16), (Wg, "Wg", None),
                       (Wu, "Wu", None), *sgc, *suc)
    y = _output((B, N), idx, out)
    if out is not None:
        _apart(out, (x2, "x"))
    if not _split_launch(out, x2.data_ptr(), g.data_ptr(), Wg.data_ptr(), Wu.data_ptr(), sgp, sup,
                         y, B, K, N, float(eps), dt, idx):
        _launch((_lib or load_library()).db_f2_rmsnorm_gateup_swiglu, idx,
                "db_f2_rmsnorm_gateup_swiglu", x2.data_ptr(), g.data_ptr(), Wg.data_ptr(),
                Wu.data_ptr(), sgp, sup, y.data_ptr(), B, K, N, float(eps), dt)
    return y[0] if squeeze else y


def gemv(x, W, w_scale=None, out=None):
    """Plain projection ``F.linear(x, W)`` (fp16 out, fp32 accumulation)."""
    if out is None and _fast is not None:
        y = _fast.gemv(x, W, w_scale)
        if y is not None:
            return y
    torch = _torch or _torch_mod()
    x2, squeeze = _as_2d(x, "x")
    B, K = x2.shape
    if W.dim() != 2 or W.shape[1] != K:
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, W {tuple(W.shape)}")
    N = W.shape[0]
    dt, sp, sc = _weights(W, w_scale, "W", N, K)
    idx = _gpu_tensors((x, "x", torch.float16), (W, "W", None), *sc)
    y = _output((B, N), idx, out)
    if out is not None:
        _apart(out, (x2, "x"))
    if not _split_launch(out, x2.data_ptr(), None, W.data_ptr(), None, sp, None, y, B, K, N, 0.0,
                         dt, idx):
        _launch((_lib or load_library()).db_gemv, idx, "db_gemv",
                x2.data_ptr(), W.data_ptr(), sp, y.data_ptr(), B, K, N, dt)
    return y[0] if squeeze else y


def f4_default_splits(B: int, Hkv: int, L: int, device=None) -> int:
    return int(load_library().db_f4_default_splits(B, Hkv, L, cu_count(device)))


def f4_workspace(B: int, Hq: int, Hkv: int, L: int, D: int, S: int, device):
    """Workspace for db_f4_splitkv (None when S = 1), zero-filled when it is
    made: the split tickets of the in-launch merge must start at zero, and
    every call leaves them at zero again.

    Outside graph capture it is cached per size, device and current stream,
    so one buffer serves every later call of that size on that stream, whose
    calls run in order.  Calls on different streams get different buffers,
    so they may overlap.  torch draws streams from a fixed pool per device,
    so the cache stays bounded.

    Under graph capture each capture (each hipGraph being recorded) gets a
    workspace of its own from the graph's memory pool, shared by the calls
    of that size it records (they run in stream order on replay), never the
    cached one: graphs captured on torch's one capture stream would
    otherwise share it, and replaying two of them at once on different
    streams would mix their partial records.  Its zero fill is recorded
    into the graph ahead of the first F4 call of the capture, so a graph
    replays one small fill kernel besides its F4 launches.  Those
    workspaces stay referenced until :func:`release_captured_workspaces`,
    so the pool never hands their memory to another graph while one that
    uses it can still be replayed."""
    import torch

    nbytes = int(load_library().db_f4_workspace_bytes(B, Hq, Hkv, L, D, S))
    if nbytes == 0:
        return None
    return _kept_workspace((), nbytes, nbytes, device)


def _kept_workspace(kind: tuple, nbytes: int, zeroed: int, device):
    """A workspace whose first ``zeroed`` bytes were zero when it was made, kept
    as :func:`f4_workspace` says; ``kind`` tells those of other ops apart."""
    import torch

    dev = torch.device(device)
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    stream = torch.cuda.current_stream(idx).cuda_stream
    if torch.cuda.is_current_stream_capturing():
        cid = C.c_ulonglong(0)
        _check(load_library().db_stream_capture_id(stream, C.byref(cid)),
               "db_stream_capture_id")
        key = (*kind, idx, stream, cid.value, nbytes)
        cache = _captured_ws
    else:
        key = (*kind, idx, stream, nbytes)
        cache = _ws_cache
    ws = cache.get(key)
    if ws is None:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        ws[:zeroed].zero_()
        cache[key] = ws
    return ws


def release_captured_workspaces() -> int:
    """Drop the references to the workspaces of F4 and paged attention made
    under graph capture; call it once every graph that recorded such calls has
    been destroyed.
    Returns how many were released."""
    n = len(_captured_ws)
    _captured_ws.clear()
    return n


def _splits_for(workspace, B: int, Hq: int, Hkv: int, L: int, D: int, S: int, idx: int) -> int:
    """The default split count ``S`` where the caller's workspace holds its
    records, else that of a workgroup per CU and at least 8 tiles per split
    (a caller may have sized the workspace for it)."""
    held = workspace.numel() * workspace.element_size()
    if held >= load_library().db_f4_workspace_bytes(B, Hq, Hkv, L, D, S):
        return S
    pairs, tiles = max(1, B * Hkv), -(-L // 16)
    return max(1, min(S, -(-cu_count(idx) // pairs), max(1, tiles // 8), 256))


def f4_flashdecode(q, K, V, scale: float | None = None, n_splits: int | None = None,
                   workspace=None, out=None):
    """F4: split-KV GQA decode attention with the log-sum-exp merge.

    q [B,Hq,D], K/V [B,Hkv,L,D] fp16 (D = 128); query head h reads KV head
    h // (Hq // Hkv).  ``scale`` defaults to 1/sqrt(D); ``n_splits`` defaults
    to the library's CU-count-based choice.  Returns [B,Hq,D] fp16."""
    if out is None and workspace is None and _fast is not None:
        o = _fast.f4(q, K, V, scale, n_splits)
        if o is not None:
            return o
    torch = _torch or _torch_mod()
    if q.dim() != 3 or K.dim() != 4 or K.shape != V.shape:
        raise ValueError(f"expected q [B,Hq,D] and K, V [B,Hkv,L,D]; got q {tuple(q.shape)}, "
                         f"K {tuple(K.shape)}, V {tuple(V.shape)}")
    B, Hq, D = q.shape
    Bk, Hkv, L, Dk = K.shape
    if Bk != B or Dk != D:
        raise ValueError(f"q {tuple(q.shape)} and K {tuple(K.shape)} disagree on B or D")
    f16 = torch.float16
    idx = _gpu_tensors((q, "q", f16), (K, "K", f16), (V, "V", f16),
                       *(((workspace, "workspace", None),) if workspace is not None else ()))
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    lib = _lib or load_library()
    S = int(lib.db_f4_default_splits(B, Hkv, L, cu_count(idx))) if n_splits is None \
        else int(n_splits)
    if workspace is not None and n_splits is None:
        S = _splits_for(workspace, B, Hq, Hkv, L, D, S, idx)
    if workspace is None:
        workspace = f4_workspace(B, Hq, Hkv, L, D, S, idx)
    ws_ptr = workspace.data_ptr() if workspace is not None else None
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    o = _output((B, Hq, D), idx, out)
    _launch(lib.db_f4_splitkv, idx, "db_f4_splitkv", q.data_ptr(), K.data_ptr(), V.data_ptr(),
            o.data_ptr(), ws_ptr, ws_bytes, B, Hq, Hkv, L, D, S, scale)
    return o


def f4_flashdecode_noalloc(q, K, V, scale: float | None = None, n_splits: int | None = None,
                           out=None):
    """F4 through ``db_f4_splitkv_noalloc``: the same kernels as
    :func:`f4_flashdecode`, with the split partials in a library-owned
    device array (``DB_F4_SCRATCH_BYTES`` per GPU) instead of a workspace,
    so the library allocates nothing.  Pass ``out`` ([B,Hq,D] fp16,
    contiguous) to allocate nothing on the Python side either.

    Every call on one GPU shares that array: calls that overlap in time on
    one GPU (concurrent streams or concurrently replayed graphs) race.  Make
    the first call on a device outside graph capture (it looks up the
    array's device address)."""
    torch = _torch or _torch_mod()
    if q.dim() != 3 or K.dim() != 4 or K.shape != V.shape:
        raise ValueError(f"expected q [B,Hq,D] and K, V [B,Hkv,L,D]; got q {tuple(q.shape)}, "
                         f"K {tuple(K.shape)}, V {tuple(V.shape)}")
    B, Hq, D = q.shape
    Bk, Hkv, L, Dk = K.shape
    if Bk != B or Dk != D:
        raise ValueError(f"q {tuple(q.shape)} and K {tuple(K.shape)} disagree on B or D")
    f16 = torch.float16
    idx = _gpu_tensors((q, "q", f16), (K, "K", f16), (V, "V", f16))
    out = _output((B, Hq, D), idx, out)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    lib = _lib or load_library()
    S = int(lib.db_f4_default_splits(B, Hkv, L, cu_count(idx))) if n_splits is None \
        else int(n_splits)
    _launch(lib.db_f4_splitkv_noalloc, idx, "db_f4_splitkv_noalloc", q.data_ptr(), K.data_ptr(),
            V.data_ptr(), out.data_ptr(), B, Hq, Hkv, L, D, S, scale)
    return out


# ------------------------------------------------ a step over a paged KV cache
class PagedPlan(NamedTuple):
    """What :func:`paged_plan` lays out for a step of T token rows and R requests."""

    q_start: object    # int32 [R + 1]: request r has the rows q_start[r] .. q_start[r + 1] - 1
    kv_len: object     # int32 [R]: tokens in the cache once the step's are appended
    position: object   # int32 [T]
    slot: object       # int64 [T]: page number * page_size + place in the page, -1: none
    free_next: object  # int32 [1]: where in free_pages the next step's pages begin


_INT_MAX = 2 ** 31 - 1  # the C ABI's sizes are ints


def _strided(t, name: str, dt, dim: int):
    """Check a GPU tensor of ``dim`` dimensions whose last one is contiguous;
    returns its GPU's index."""
    torch = _torch or _torch_mod()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU device (got {t.device})")
    if dt is not None and t.dtype != dt:
        raise TypeError(f"{name} must be {dt} (got {t.dtype})")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions (got {tuple(t.shape)})")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    if max(t.shape) > _INT_MAX:
        raise ValueError(f"{name} {tuple(t.shape)} has a dimension of 2^31 or more")
    return t.get_device()


def _one_gpu(idx: int, *named) -> None:
    for other, name in named:
        if other != idx:
            raise ValueError(f"{name} is on cuda:{other}, expected cuda:{idx}")


def _strides(t, n: int):
    """The first n strides, 0 where there is one element and none counts."""
    return [st if size > 1 else 0 for st, size in zip(t.stride()[:n], t.shape)]


def _activation(t, name: str) -> int:
    torch = _torch
    if t.dtype == torch.float16:
        return DTYPE_F16
    if t.dtype == torch.bfloat16:
        return DTYPE_BF16
    raise TypeError(f"{name} must be torch.float16 or torch.bfloat16 (got {t.dtype})")


def _paged_cache(K, V, k_scale, v_scale, act, idx: int):
    """The cache [pages, Hkv, page_size, D] as the C ABI takes it: strided, of the
    activations' type or e4m3 with one fp32 scale per KV head."""
    torch = _torch
    _one_gpu(idx, (_strided(K, "K", None, 4), "K"), (_strided(V, "V", None, 4), "V"))
    if K.shape != V.shape or K.dtype != V.dtype:
        raise ValueError(f"K {tuple(K.shape)} {K.dtype} and V {tuple(V.shape)} {V.dtype} must "
                         "agree")
    pages, Hkv, page, D = K.shape
    c = _PagedCache(K.data_ptr(), V.data_ptr(), None, None, *_strides(K, 3), *_strides(V, 3),
                    pages, page, Hkv, D, DTYPE_FP8_E4M3)
    if K.dtype == torch.float8_e4m3fn:
        for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if t is None:
                raise ValueError(f"an e4m3 cache needs {name}, an fp32 tensor of shape ({Hkv},)")
            _one_gpu(idx, (_gpu_tensors((t, name, torch.float32)), name))
            if tuple(t.shape) != (Hkv,):
                raise ValueError(f"{name} must have shape ({Hkv},) (got {tuple(t.shape)})")
        c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        return c
    if K.dtype != act:
        raise TypeError(f"the cache must be {act} or torch.float8_e4m3fn (got {K.dtype})")
    if k_scale is not None or v_scale is not None:
        raise ValueError("a 16-bit cache takes no scales")
    c.dtype = _activation(K, "K")
    return c


def _row_output(shape, dtype, idx: int, out):
    torch = _torch
    if out is None:
        return torch.empty(shape, dtype=dtype, device=torch.device("cuda", idx))
    _one_gpu(idx, (_gpu_tensors((out, "out", dtype)), "out"))
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"out must have shape {tuple(shape)} (got {tuple(out.shape)})")
    return out


def paged_plan(past_len, new_len, block_table, free_pages, page_size: int, n_tokens: int,
               free_start=None) -> PagedPlan:
    """Lay out a step's tokens over a paged cache, on the GPU: rows, lengths,
    positions and cache slots, and the pages that the requests need.

    past_len [R] int32 tokens of each request in the cache, new_len [R] int32
    tokens of this step, block_table [R, width] int32 (rows may be strided).
    Pages are taken from ``free_pages`` [F] int32 from ``free_start`` on (an
    int32 tensor [1]; None: 0), requests in order, and entered in
    ``block_table`` in place.  ``n_tokens`` is T, the rows that the step has
    room for: rows behind the last token get slot -1, tokens beyond them are
    left out of ``kv_len``.  Where pages run out (``free_next`` > F) or a
    request outgrows its table row, the tokens concerned get slot -1."""
    if _fast is not None:
        p = _fast.plan(past_len, new_len, block_table, free_pages, page_size, n_tokens, free_start)
        if p is not None:
            return PagedPlan(*p)
    torch = _torch or _torch_mod()
    i32 = torch.int32
    idx = _gpu_tensors((past_len, "past_len", i32), (new_len, "new_len", i32),
                       (free_pages, "free_pages", i32),
                       *(((free_start, "free_start", i32),) if free_start is not None else ()))
    _one_gpu(idx, (_strided(block_table, "block_table", i32, 2), "block_table"))
    R, width = block_table.shape
    if past_len.shape != (R,) or new_len.shape != (R,):
        raise ValueError(f"past_len {tuple(past_len.shape)} and new_len {tuple(new_len.shape)} "
                         f"must have one entry for each of the {R} rows of block_table")
    if free_pages.dim() != 1:
        raise ValueError(f"free_pages must be [F] (got {tuple(free_pages.shape)})")
    if free_start is not None and free_start.numel() != 1:
        raise ValueError("free_start must have one element")
    if R > 1 and block_table.stride(0) < width:
        raise ValueError("block_table rows must not overlap")
    T, page = int(n_tokens), int(page_size)
    if not 0 <= T <= _INT_MAX:
        raise ValueError(f"n_tokens must be >= 0 and below 2^31 (got {T})")
    if not 1 <= page <= _INT_MAX:
        raise ValueError(f"page_size must be >= 1 and below 2^31 (got {page})")
    if free_pages.numel() > _INT_MAX:
        raise ValueError(f"free_pages has {free_pages.numel()} entries, 2^31 or more")
    dev = past_len.device
    q_start = torch.empty(R + 1, dtype=i32, device=dev)
    kv_len = torch.empty(R, dtype=i32, device=dev)
    position = torch.empty(T, dtype=i32, device=dev)
    slot = torch.empty(T, dtype=torch.int64, device=dev)
    free_next = torch.empty(1, dtype=i32, device=dev)
    _launch((_lib or load_library()).db_paged_plan, idx, "db_paged_plan", past_len.data_ptr(),
            new_len.data_ptr(), block_table.data_ptr(), max(block_table.stride(0), width), width,
            free_pages.data_ptr(), free_pages.numel(),
            None if free_start is None else free_start.data_ptr(), page, R, T,
            q_start.data_ptr(), kv_len.data_ptr(), position.data_ptr(), slot.data_ptr(),
            free_next.data_ptr())
    return PagedPlan(q_start, kv_len, position, slot, free_next)


def rope_append(qkv, position, slot, K, V, inv_freq, axes=None, interleaved: bool = False,
                k_scale=None, v_scale=None, out=None):
    """Rotary positions on the queries and keys of a projection, keys and
    values into the pages of the cache.  Returns the turned queries [T,Hq,D].

    qkv [T, (Hq + 2 Hkv) D] fp16 or bf16 (rows may be strided), query, key and
    value heads side by side; K/V [pages, Hkv, page_size, D] of that type, or
    float8_e4m3fn with fp32 ``k_scale``/``v_scale`` [Hkv] (any strides with
    contiguous rows of D, so a [pages, page_size, Hkv, D] cache is passed as its
    ``permute(0, 2, 1, 3)``); slot [T] int64 as :func:`paged_plan` gives it (a
    slot outside the cache writes nothing; slots must differ).  D is a multiple of
    16 up to 256 (:func:`paged_attention` reads caches of D 64 and 128).

    Pair i of a head turns by ``position * inv_freq[i]`` (inv_freq fp32, rot/2
    entries, rot <= D; elements past rot stay): elements i and i + rot/2, or
    2i and 2i+1 where ``interleaved``.  position is int32 [T], or [A, T] for
    tokens with A axes (time, height, width): ``axes`` then names the axis of
    each pair, e.g. ``[0] * 16 + [1] * 24 + [2] * 24``."""
    axis_map = None if axes is None else bytes(axes)
    if out is None and _fast is not None:
        q = _fast.rope(qkv, position, slot, K, V, inv_freq, axis_map, interleaved, k_scale,
                       v_scale)
        if q is not None:
            return q
    torch = _torch or _torch_mod()
    idx = _strided(qkv, "qkv", None, 2)
    dt = _activation(qkv, "qkv")
    cache = _paged_cache(K, V, k_scale, v_scale, qkv.dtype, idx)
    T, Hkv, D = qkv.shape[0], cache.Hkv, cache.D
    Hq = qkv.shape[1] // D - 2 * Hkv if D else 0
    if Hq < 1 or (Hq + 2 * Hkv) * D != qkv.shape[1]:
        raise ValueError(f"qkv rows of {qkv.shape[1]} elements are not (Hq + 2 * {Hkv}) * {D}")
    _one_gpu(idx, (_gpu_tensors((position, "position", torch.int32), (slot, "slot", torch.int64),
                                (inv_freq, "inv_freq", torch.float32)), "position"))
    n_axes = 1 if position.dim() == 1 else position.shape[0]
    if position.dim() not in (1, 2) or position.shape[-1] != T or slot.shape != (T,):
        raise ValueError(f"position {tuple(position.shape)} and slot {tuple(slot.shape)} must "
                         f"have one entry for each of the {T} rows of qkv")
    if inv_freq.dim() != 1:
        raise ValueError(f"inv_freq must be [rot / 2] (got {tuple(inv_freq.shape)})")
    if axis_map is not None:
        if len(axis_map) != inv_freq.numel():
            raise ValueError(f"axes has {len(axis_map)} entries for {inv_freq.numel()} pairs")
    elif n_axes != 1:
        raise ValueError("positions of several axes need axes, the axis of each pair")
    q = _row_output((T, Hq, D), qkv.dtype, idx, out)
    _launch((_lib or load_library()).db_rope_append, idx, "db_rope_append", qkv.data_ptr(),
            qkv.stride(0) if T > 1 else qkv.shape[1], position.data_ptr(), n_axes, axis_map,
            slot.data_ptr(), inv_freq.data_ptr(), 2 * inv_freq.numel(), bool(interleaved),
            C.byref(cache), q.data_ptr(), T, Hq, dt)
    return q


def paged_attention(q, K, V, block_table, q_start, kv_len, scale: float | None = None,
                    causal: bool = True, window: int | None = None, max_new: int | None = None,
                    k_scale=None, v_scale=None, out=None):
    """Attention of each request's new tokens over its pages of the cache:
    single tokens, drafts and chunks of a prompt alike.  Returns [T,Hq,D].

    q [T,Hq,D] fp16 or bf16 (token and head strides free); K/V and their scales
    as in :func:`rope_append`, D 64 or 128, Hq a multiple of Hkv; block_table
    [R, width], q_start [R+1] and kv_len [R] int32 on the GPU.  Request r has
    the rows q_start[r] .. q_start[r+1]-1, the last of its kv_len[r] tokens,
    whose keys and values are in the cache already.  A token sees the keys up
    to its own position (``causal``; all of its request otherwise), with
    ``window`` only the last that many; a token that sees nothing gets zeros,
    and what hidden keys and values hold never counts.  Rows that belong to no
    request are not written; q_start ascends, and where it does not, a row is the
    first request's that names it.

    ``max_new`` is the most new tokens a request has, where the caller knows it
    (1 in a plain decode step): it spares the kernels that such a call does not
    need (256 requests of one token and 500 keys: 71 us instead of 102), and
    nothing else."""
    if out is None and _fast is not None:
        o = _fast.paged(q, K, V, block_table, q_start, kv_len, scale, causal, window, max_new,
                        k_scale, v_scale)
        if o is not None:
            return o
    torch = _torch or _torch_mod()
    idx = _strided(q, "q", None, 3)
    dt = _activation(q, "q")
    cache = _paged_cache(K, V, k_scale, v_scale, q.dtype, idx)
    T, Hq, D = q.shape
    if D != cache.D:
        raise ValueError(f"q {tuple(q.shape)} and K {tuple(K.shape)} disagree on D")
    i32 = torch.int32
    _one_gpu(idx, (_strided(block_table, "block_table", i32, 2), "block_table"),
             (_gpu_tensors((q_start, "q_start", i32), (kv_len, "kv_len", i32)), "q_start"))
    R, width = block_table.shape
    if q_start.shape != (R + 1,) or kv_len.shape != (R,):
        raise ValueError(f"q_start {tuple(q_start.shape)} and kv_len {tuple(kv_len.shape)} must "
                         f"have R + 1 and R entries for the {R} rows of block_table")
    if window is not None and window < 1:
        raise ValueError(f"window must be >= 1 (got {window})")
    if max_new is not None and max_new < 1:
        raise ValueError(f"max_new must be >= 1 (got {max_new})")
    scale = 1.0 / math.sqrt(D) if scale is None and D else float(scale or 0.0)
    o = _row_output((T, Hq, D), q.dtype, idx, out)
    lib = _lib or load_library()
    most = min(int(max_new or T), T)
    with _on_device(idx):
        zeroed = C.c_size_t(0)
        nbytes = lib.db_paged_attention_workspace_bytes(T, Hq, cache.Hkv, D, R, most,
                                                        C.byref(zeroed))
        # Tickets that start at zero are kept as F4's are; otherwise nothing in the
        # workspace outlives the call, and torch's allocator hands it out anew.
        if zeroed.value:
            ws = _kept_workspace(("paged", zeroed.value), nbytes, zeroed.value, idx)
        else:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    _launch(lib.db_paged_attention, idx, "db_paged_attention", q.data_ptr(), *_strides(q, 2),
            o.data_ptr(), C.byref(cache), block_table.data_ptr(), *_strides(block_table, 1), width,
            q_start.data_ptr(), kv_len.data_ptr(), T, R, Hq, most, scale, bool(causal),
            min(int(window or 0), _INT_MAX), dt, ws.data_ptr(), nbytes)
    return o


# ------------------------------------- block-scaled e4m3, mixture of experts
def _workspace(nbytes: int, device):
    """Memory of one call from torch's allocator, which takes it back in stream
    order; nothing in it outlives the call."""
    return _torch.empty(nbytes, dtype=_torch.uint8, device=device) if nbytes else None


def _blocks(n: int) -> int:
    return -(-n // 128)


def _row_stride(t) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def quantize_blocks(x):
    """e4m3 with one fp32 scale for each 128 elements of a row: ``(q, scale)``,
    q float8_e4m3fn [T, K] and scale [T, ceil(K / 128)] (a block's tokens side by
    side in memory, as :func:`gemm_blocks` reads them best).

    x [T, K] fp16 or bf16 (rows may be strided), K a multiple of 16.
    ``scale[t, b] = max |x[t, 128 b ..]| * (1 / 448)`` in fp32 (1 where that is 0) and
    ``q = e4m3(clamp(x / scale, -448, 448))``, rounded to nearest even; an Inf or
    NaN makes its block's scale one."""
    if _fast is not None:
        r = _fast.quantize_blocks(x)
        if r is not None:
            return r
    torch = _torch or _torch_mod()
    idx = _strided(x, "x", None, 2)
    dt = _activation(x, "x")
    T, K = x.shape
    q = torch.empty((T, K), dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty((_blocks(K), T), dtype=torch.float32, device=x.device).t()
    _launch((_lib or load_library()).db_quantize_blocks, idx, "db_quantize_blocks", x.data_ptr(),
            _row_stride(x), q.data_ptr(), scale.data_ptr(), 1, T, T, K, dt)
    return q, scale


def _block_scale(s, name: str, shape, idx: int):
    """The fp32 scales of e4m3 weights, one for each block of 128 x 128."""
    if s is None:
        raise ValueError(f"e4m3 weights need {name}, an fp32 tensor of shape {shape}")
    _one_gpu(idx, (_gpu_tensors((s, name, _torch.float32)), name))
    if tuple(s.shape) != shape:
        raise ValueError(f"{name} must have shape {shape} (got {tuple(s.shape)})")
    return s.data_ptr()


def gemm_blocks(x, W, w_scale, x_scale=None, dtype=None, out=None):
    """Projection ``y = x W^T`` on e4m3 weights with one fp32 scale for each
    block of 128 x 128, by 8-bit matrix instructions; fp32 sums, rounded once.

    W [N, K] float8_e4m3fn (or its bytes), w_scale [ceil(N/128), ceil(K/128)]
    (``quant.quantize_e4m3_blocks``), K a multiple of 16.  x [T, K] (or [K]) fp16
    or bf16 is quantised on the way, as :func:`quantize_blocks` does, and
    y [T, N] has its type; or x is float8_e4m3fn with x_scale [T, ceil(K/128)],
    and y is ``dtype`` (torch.float16 if not given).  Rows of x may be strided,
    and x_scale anyhow; ``out`` shares no memory with an input."""
    if out is None and _fast is not None:
        y = _fast.gemm_blocks(x, W, w_scale, x_scale, dtype)
        if y is not None:
            return y
    torch = _torch or _torch_mod()
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a torch.Tensor")
    x2, squeeze = _as_2d(x, "x")
    idx = _strided(x2, "x", None, 2)
    T, K = x2.shape
    if x2.dtype == torch.float8_e4m3fn:
        xdt, dtype = DTYPE_FP8_E4M3, dtype or torch.float16
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"dtype must be torch.float16 or torch.bfloat16 (got {dtype})")
        ydt = DTYPE_F16 if dtype == torch.float16 else DTYPE_BF16
        if x_scale is None:
            raise ValueError(f"e4m3 activations need x_scale, an fp32 tensor of shape "
                             f"{(T, _blocks(K))}")
        if not isinstance(x_scale, torch.Tensor):
            raise TypeError("x_scale must be a torch.Tensor")
        xs = x_scale.unsqueeze(0) if squeeze and x_scale.dim() == 1 else x_scale
        if not xs.is_cuda or xs.dtype != torch.float32 or tuple(xs.shape) != (T, _blocks(K)):
            raise ValueError(f"x_scale must be an fp32 GPU tensor of shape {(T, _blocks(K))} "
                             f"(got {xs.dtype} {tuple(xs.shape)} on {xs.device})")
        _one_gpu(idx, (xs.get_device(), "x_scale"))
        xsp, (xs_t, xs_b) = xs.data_ptr(), _strides(xs, 2)
    else:
        xdt = ydt = _activation(x2, "x")
        if x_scale is not None:
            raise ValueError("16-bit activations take no x_scale")
        if dtype is not None and dtype != x2.dtype:
            raise TypeError(f"dtype must be {x2.dtype} like x (got {dtype})")
        dtype, xsp, xs_t, xs_b = x2.dtype, None, 0, 0
    if not isinstance(W, torch.Tensor) or W.dim() != 2 or W.shape[1] != K:
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, "
                         f"W {tuple(getattr(W, 'shape', ()))}")
    if W.dtype not in (torch.float8_e4m3fn, torch.uint8):
        raise TypeError(f"W must be torch.float8_e4m3fn (got {W.dtype})")
    _one_gpu(idx, (_gpu_tensors((W, "W", None)), "W"))
    N = W.shape[0]
    sp = _block_scale(w_scale, "w_scale", (_blocks(N), _blocks(K)), idx)
    y = _row_output((T, N), dtype, idx, out)
    if out is not None:
        _apart(out, (x2, "x"), (W, "W"), (w_scale, "w_scale"), (x_scale, "x_scale"))
    lib = _lib or load_library()
    with _on_device(idx):
        nbytes = lib.db_gemm_blocks_workspace_bytes(T, K, N, xdt)
    ws = _workspace(nbytes, x.device)
    _launch(lib.db_gemm_blocks, idx, "db_gemm_blocks", x2.data_ptr(), _row_stride(x2), xsp, xs_t,
            xs_b, W.data_ptr(), sp, y.data_ptr(), T, K, N, xdt, ydt,
            None if ws is None else ws.data_ptr(), nbytes)
    return y[0] if squeeze else y


def _router(x, Wr, top_k):
    torch = _torch or _torch_mod()
    idx = _strided(x, "x", None, 2)
    dt = _activation(x, "x")
    _one_gpu(idx, (_gpu_tensors((Wr, "Wr", x.dtype)), "Wr"))
    if Wr.dim() != 2 or Wr.shape[1] != x.shape[1]:
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, Wr {tuple(Wr.shape)}")
    k = int(top_k)
    if not 1 <= k <= min(Wr.shape[0], 64):
        raise ValueError(f"top_k must be between 1 and the {Wr.shape[0]} experts, at most 64 "
                         f"(got {k})")
    return idx, dt, k


def moe_route(x, Wr, top_k: int, renormalize: bool = True):
    """The experts of each token and their weights: ``(experts, weights)``,
    int32 and fp32 [T, top_k], the largest first.

    x [T, H] fp16 or bf16 (rows may be strided), Wr [E, H] of that type, H a
    multiple of 8, E <= 1024, top_k <= 64.  The logits ``x Wr^T`` are summed in
    64 bits; equal ones go to the lower index, NaN counts above all numbers.
    Weights are the softmax over the chosen experts (``renormalize``) or
    over all of them."""
    if _fast is not None:
        r = _fast.moe_route(x, Wr, top_k, renormalize)
        if r is not None:
            return r
    idx, dt, k = _router(x, Wr, top_k)
    torch = _torch
    T, H = x.shape
    E = Wr.shape[0]
    experts = torch.empty((T, k), dtype=torch.int32, device=x.device)
    weights = torch.empty((T, k), dtype=torch.float32, device=x.device)
    lib = _lib or load_library()
    with _on_device(idx):
        nbytes = lib.db_moe_route_workspace_bytes(T, H, E)
    ws = _workspace(nbytes, x.device)
    _launch(lib.db_moe_route, idx, "db_moe_route", x.data_ptr(), _row_stride(x), Wr.data_ptr(),
            experts.data_ptr(), weights.data_ptr(), T, H, E, k, bool(renormalize), dt,
            None if ws is None else ws.data_ptr(), nbytes)
    return experts, weights


def _experts(x, Wg, Wu, Wd, sg, su, sd, idx: int, dt: int):
    """The experts' weights as the C ABI takes them: of x's type, or e4m3 with
    fp32 scales of blocks of 128 x 128."""
    torch = _torch
    H = x.shape[1]
    _one_gpu(idx, (_gpu_tensors((Wg, "Wg", None), (Wu, "Wu", None), (Wd, "Wd", None)), "Wg"))
    if Wg.dim() != 3 or Wg.shape[2] != H or Wu.shape != Wg.shape or \
            tuple(Wd.shape) != (Wg.shape[0], H, Wg.shape[1]):
        raise ValueError(f"expected Wg, Wu [E, I, {H}] and Wd [E, {H}, I]; got "
                         f"{tuple(Wg.shape)}, {tuple(Wu.shape)}, {tuple(Wd.shape)}")
    if Wu.dtype != Wg.dtype or Wd.dtype != Wg.dtype:
        raise TypeError(f"Wg, Wu and Wd must have one type (got {Wg.dtype}, {Wu.dtype}, "
                        f"{Wd.dtype})")
    E, I = Wg.shape[:2]
    m = _Moe(Wg.data_ptr(), Wu.data_ptr(), Wd.data_ptr(), None, None, None, E, H, I, dt, dt)
    if Wg.dtype in (torch.float8_e4m3fn, torch.uint8):
        m.w_dtype = DTYPE_FP8_E4M3
        m.sg = _block_scale(sg, "sg", (E, _blocks(I), _blocks(H)), idx)
        m.su = _block_scale(su, "su", (E, _blocks(I), _blocks(H)), idx)
        m.sd = _block_scale(sd, "sd", (E, _blocks(H), _blocks(I)), idx)
    elif Wg.dtype != x.dtype:
        raise TypeError(f"the experts' weights must be {x.dtype} like x or "
                        f"torch.float8_e4m3fn (got {Wg.dtype})")
    elif sg is not None or su is not None or sd is not None:
        raise ValueError("16-bit weights take no scales")
    return m


def moe_experts(x, experts, weights, Wg, Wu, Wd, sg=None, su=None, sd=None, out=None):
    """The experts of a mixture-of-experts layer on tokens that are routed:
    ``y[t] = sum_j weights[t, j] Wd[e] (silu(Wg[e] x[t]) * (Wu[e] x[t]))``,
    e = experts[t, j].  Returns [T, H] of x's type.

    x [T, H] fp16 or bf16 (rows may be strided); experts int32 and weights fp32
    [T, k], as :func:`moe_route` gives them; Wg, Wu [E, I, H] and Wd [E, H, I] of
    x's type, or float8_e4m3fn (or its bytes) with fp32 scales of blocks of
    128 x 128 (sg, su [E, ceil(I/128), ceil(H/128)], sd [E, ceil(H/128),
    ceil(I/128)]).  H and I are multiples of 8, of 16 for e4m3.

    An expert outside [0, E) adds nothing; a token without any gets zeros; an
    expert named twice counts twice.  Sums are fp32, the result is rounded once.
    What the gate gives stays in fp32 for a token or a few; beyond that it is rounded
    to x's type before the down product (in fp16, above 65504 it becomes Inf).  Made for
    the few tokens of a decode step: the weights bound the call.  ``out`` may be x
    itself and shares no memory with another input."""
    if out is None and _fast is not None:
        y = _fast.moe_experts(x, experts, weights, Wg, Wu, Wd, sg, su, sd)
        if y is not None:
            return y
    torch = _torch or _torch_mod()
    idx = _strided(x, "x", None, 2)
    dt = _activation(x, "x")
    _one_gpu(idx, (_gpu_tensors((experts, "experts", torch.int32),
                                (weights, "weights", torch.float32)), "experts"))
    T, H = x.shape
    if experts.dim() != 2 or experts.shape[0] != T or experts.shape != weights.shape:
        raise ValueError(f"experts {tuple(experts.shape)} and weights {tuple(weights.shape)} "
                         f"must be [{T}, k]")
    k = experts.shape[1]
    m = _experts(x, Wg, Wu, Wd, sg, su, sd, idx, dt)
    y = _row_output((T, H), x.dtype, idx, out)
    if out is not None:
        _apart(out, (experts, "experts"), (weights, "weights"), (Wg, "Wg"), (Wu, "Wu"),
               (Wd, "Wd"), (sg, "sg"), (su, "su"), (sd, "sd"))
    lib = _lib or load_library()
    with _on_device(idx):
        nbytes = lib.db_moe_experts_workspace_bytes(C.byref(m), T, k)
    ws = _workspace(nbytes, x.device)
    _launch(lib.db_moe_experts, idx, "db_moe_experts", x.data_ptr(), _row_stride(x),
            experts.data_ptr(), weights.data_ptr(), C.byref(m), y.data_ptr(), T, k,
            None if ws is None else ws.data_ptr(), nbytes)
    return y


def moe_layer(x, Wr, Wg, Wu, Wd, top_k: int, renormalize: bool = True, sg=None, su=None, sd=None,
              out=None):
    """A whole mixture-of-experts layer: :func:`moe_route` and
    :func:`moe_experts` in one call, with their arguments.  Returns [T, H]."""
    if out is None and _fast is not None:
        y = _fast.moe_layer(x, Wr, Wg, Wu, Wd, top_k, renormalize, sg, su, sd)
        if y is not None:
            return y
    idx, dt, k = _router(x, Wr, top_k)
    m = _experts(x, Wg, Wu, Wd, sg, su, sd, idx, dt)
    if Wr.shape[0] != m.E:
        raise ValueError(f"Wr has {Wr.shape[0]} rows for {m.E} experts")
    T, H = x.shape
    y = _row_output((T, H), x.dtype, idx, out)
    if out is not None:
        _apart(out, (Wr, "Wr"), (Wg, "Wg"), (Wu, "Wu"), (Wd, "Wd"), (sg, "sg"), (su, "su"),
               (sd, "sd"))
    lib = _lib or load_library()
    with _on_device(idx):
        nbytes = lib.db_moe_layer_workspace_bytes(C.byref(m), T, k)
    ws = _workspace(nbytes, x.device)
    _launch(lib.db_moe_layer, idx, "db_moe_layer", x.data_ptr(), _row_stride(x), Wr.data_ptr(),
            C.byref(m), y.data_ptr(), T, k, bool(renormalize),
            None if ws is None else ws.data_ptr(), nbytes)
    return y
