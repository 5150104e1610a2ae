"""ctypes binding of libsimsd_b200.so (the C ABI in include/simsd_b200.h).

This module is the only place that touches the shared library.  It has no CPU
fallback: if the library is missing, every operator raises.  Workspaces are
cached per device and reused serially, like the reference's split-K staging
buffer (kernels/thin_linear_fused.py:173-190); `reset_workspace()` drops them
(call it before re-capturing graphs into a new memory pool).
"""
from __future__ import annotations

import contextlib
import ctypes
import sys
import warnings
from pathlib import Path

import torch

LIB_PATH = Path(__file__).resolve().with_name("libsimsd_b200.so")

SIMSD_OK = 0
SIMSD_ERR_SHAPE = -1
SIMSD_ERR_DTYPE = -2
SIMSD_ERR_WORKSPACE = -3
SIMSD_ERR_LAUNCH = -4
SIMSD_ERR_ALIGN = -5
SIMSD_ERR_DEVICE = -6
SIMSD_ERR_UNSUPPORTED = -7
SIMSD_ERR_SCRATCH_LIMIT = -8

SIMSD_BF16, SIMSD_F16, SIMSD_F32 = 0, 1, 2
EPI_NONE, EPI_SILU_MUL = 0, 1
PATH_AUTO, PATH_TC, PATH_SIMT = 0, 1, 2

LAUNCH_PDL = 1
LAUNCH_INKERNEL_REDUCE = 2
LAUNCH_GROUPED_FIXUP = 4
LAUNCH_MOE_SIZE_CLASSES = 8
IPC_HANDLE_BYTES = 64
SIGNAL_BYTES = 256

HEADER_BYTES = 256 * 1024          # simsd_workspace_header_bytes()
PAGED_COUNTER_BYTES = 4096

DEV_ERR_TIMEOUT = 1
DEV_ERR_BAD_INDEX = 2
DEV_ERR_CAPACITY = 4

_DTYPE = {torch.bfloat16: SIMSD_BF16, torch.float16: SIMSD_F16, torch.float32: SIMSD_F32}

# name -> (restype, argtypes); every symbol include/simsd_b200.h declares
_P, _I, _L, _S, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float
SIGNATURES: dict[str, tuple] = {
    "simsd_version": (ctypes.c_char_p, []),
    "simsd_status_string": (ctypes.c_char_p, [_I]),
    "simsd_device_sm_count": (_I, []),
    "simsd_set_launch_flags": (_I, [_I]),
    "simsd_get_launch_flags": (_I, []),
    "simsd_debug_cluster_plan": (_I, [_I, _I, _I, _I, _P, _P, _P]),
    "simsd_debug_set_trace": (_I, [_P, _S]),
    "simsd_workspace_header_bytes": (_S, []),
    "simsd_workspace_init": (_I, [_P, _S, _P]),
    "simsd_workspace_error": (_I, [_P, _P, ctypes.POINTER(_I)]),
    "simsd_thin_linear_workspace_size": (_S, [_I, _I, _I, _I, _I, _I]),
    "simsd_thin_linear": (_I, [_P, _L, _L, _P, _L, _L, _P, _P, _P, _L, _I, _I, _I, _I, _I, _I, _I,
                               _P, _S, _P]),
    "simsd_thin_linear_noalloc": (_I, [_P, _L, _L, _P, _L, _L, _P, _P, _P, _L, _I, _I, _I, _I, _I, _P]),
    "simsd_thin_linear_noalloc_error": (_I, [_P, ctypes.POINTER(_I)]),
    "simsd_moe_route_ex": (_I, [_P, _L, _I, _P, _L, _I, _P, _I, _I, _I, _I, _I, _F, _P, _P, _L, _I, _P, _P]),
    "simsd_moe_route": (_I, [_P, _L, _I, _P, _L, _I, _P, _I, _I, _I, _I, _I, _F, _P, _P, _P, _P]),
    "simsd_moe_align": (_I, [_P, _I, _I, _P, _P, _P, _P, _I, _I, _P, _P, _P, _P]),
    "simsd_moe_workspace_size": (_S, [_I, _I, _I, _I, _I, _I]),
    "simsd_moe_dispatch_shared_last": (_I, [_P, _L, _P, _P, _P, _P, _L, _L, _P, _L, _L, _P, _L, _I, _I, _I, _I, _I, _I, _P, _S, _P]),
    "simsd_moe_dispatch": (_I, [_P, _L, _P, _P, _P, _P, _L, _L, _P, _L, _L, _P, _L, _P, _L, _I, _I,
                                _I, _I, _I, _I, _P, _S, _P]),
    "simsd_ipc_alloc": (_I, [_S, ctypes.POINTER(_P)]),
    "simsd_ipc_free": (_I, [_P]),
    "simsd_ipc_handle": (_I, [_P, _P]),
    "simsd_ipc_open": (_I, [_P, ctypes.POINTER(_P)]),
    "simsd_ipc_close": (_I, [_P]),
    "simsd_thin_linear_argmax": (_I, [_P, _L, _L, _P, _L, _L, _P, _P, _I, _I, _I, _I, _P, _S, _P]),
    "simsd_thin_linear_cat": (_I, [_P, _L, _L, _I, _P, _P, _P, _P, _L, _I, _I, _I, _P, _S, _P]),
    "simsd_rmsnorm": (_I, [_P, _L, _P, _L, _P, _L, _P, _P, _L, _I, _I, _F, _I, _P]),
    "simsd_qk_norm_rope": (_I, [_P, _L, _I, _I, _I, _I, _P, _P, _P, _P, _F, _P, _P, _P, _L, _I, _I, _P]),
    "simsd_verify_attention_workspace_size": (_S, [_I, _I, _I, _I]),
    "simsd_verify_attention": (_I, [_P, _P, _P, _L, _I, _I, _I, _I, _P, _L, _F, _P, _I, _P, _S, _P]),
    "simsd_paged_append": (_I, [_P, _L, _I, _I, _I, _I, _I, _P, _P, _F, _P, _P, _L, _P, _P, _P, _P, _P, _I, _I, _L, _L,
                                _L, _I, _P, _P]),
    "simsd_paged_attention_workspace_size": (_S, [_I, _I, _I, _I]),
    "simsd_paged_attention": (_I, [_P, _P, _P, _I, _I, _L, _L, _L, _P, _L, _I, _P, _P, _L, _L, _I, _I, _I, _I, _I, _F,
                                   _P, _P, _I, _P, _S, _P, _P]),
    "simsd_paged_attention_window": (_I, [_P, _P, _P, _I, _I, _L, _L, _L, _P, _L, _I, _P, _P, _L, _L, _I, _I, _I, _I, _I,
                                          _F, _I, _I, _P, _P, _I, _P, _S, _P, _P]),
    "simsd_paged_append8": (_I, [_P, _L, _L, _I, _I, _I, _I, _I, _I, _P, _P, _F, _P, _P, _L, _P, _L, _I, _P, _P, _P, _P, _P,
                                 _P, _P, _I, _I, _I, _L, _L, _L, _L, _L, _L, _I, _P, _P]),
    "simsd_paged_attention8_workspace_size": (_S, [_I, _I, _I, _I]),
    "simsd_paged_attention8": (_I, [_P, _P, _P, _P, _P, _I, _I, _I, _L, _L, _L, _L, _L, _L, _P, _L, _I, _P, _P, _L, _L, _I,
                                    _I, _I, _I, _I, _F, _I, _I, _P, _P, _I, _P, _S, _P, _P]),
    "simsd_paged_reserve": (_I, [_P, _L, _I, _P, _P, _P, _P, _I, _P, _I, _I, _I, _P, _P, _P, _P, _S, _P, _P]),
    "simsd_paged_release": (_I, [_P, _L, _I, _P, _P, _I, _P, _P, _I, _I, _P, _S, _P, _P]),
    "simsd_adjust_logits": (_I, [_P, _L, _L, _P, _L, _L, _I, _I, _I, _I, _P, _L, _P, _L, _P, _L, _P, _P, _P, _P, _L, _P, _L,
                                 _I, _P, _L, _L, _P, _P]),
    "simsd_count_tokens": (_I, [_P, _L, _P, _L, _I, _I, _I, _P, _P]),
    "simsd_speculative_verify_workspace_size": (_S, [_I, _I, _I]),
    "simsd_speculative_verify": (_I, [_P, _L, _L, _P, _L, _L, _P, _L, _P, _L, _P, _L, _P, _P, _I, _I, _I, _I, _P, _P,
                                      _P, _P, _S, _P, _P]),
    "simsd_allgather_wait": (_I, [_P, _I, _I, _P, _S, _P]),
    "simsd_thin_linear_allgather": (_I, [_P, _L, _L, _P, _L, _L, _P, _P, _P, _L, _I, _I, _I, _I, _I, _I, _I, _I,
                                         _I, _P, _S, _P]),
    "simsd_moe_ep_plan": (_I, [_P, _I, _I, _I, _I, _P, _P, _P, _P, _P, _P]),
    "simsd_moe_gather_rows": (_I, [_P, _L, _P, _I, _I, _I, _I, _P, _L, _P]),
    "simsd_moe_combine": (_I, [_P, _L, _P, _P, _P, _L, _P, _L, _I, _I, _I, _I, _P]),
    "simsd_moe_ep_send": (_I, [_P, _L, _P, _P, _I, _I, _I, _I, _I, _P, _P, _I, _P]),
    "simsd_moe_ep_return": (_I, [_P, _L, _P, _I, _I, _I, _I, _P, _I, _P]),
}

_lib = None


def lib() -> ctypes.CDLL:
    """Load libsimsd_b200.so once; raise if it has not been built."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH.name} is not built; run `python simsd-release_b200/build.py` "
                "(nvcc, sm_100a). There is no CPU fallback.")
        L = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        # Over the streams' scratch, the GIL orders one thread's calls with another's (the
        # native binding holds it too): a verification is two launches on the same bytes.
        held = ctypes.PyDLL(str(LIB_PATH))
        for name in ("simsd_paged_attention", "simsd_paged_attention_window", "simsd_paged_attention8", "simsd_paged_reserve",
                     "simsd_paged_release", "simsd_speculative_verify"):
            fn = getattr(held, name)
            fn.restype, fn.argtypes = SIGNATURES[name]
            setattr(L, name, fn)
        _lib = L
    return _lib


_BOUND = ("simsd_paged_append", "simsd_paged_attention_window", "simsd_paged_attention_workspace_size",
          "simsd_speculative_verify", "simsd_speculative_verify_workspace_size", "simsd_paged_append8",
          "simsd_paged_attention8", "simsd_paged_attention8_workspace_size", "simsd_paged_reserve", "simsd_paged_release",
          "simsd_adjust_logits", "simsd_count_tokens")
_binding = None


class _CtypesOnly:
    """Stands in for the native binding where there is none: every request takes the Python way."""

    @staticmethod
    def paged_append(*_):
        return None

    paged_attention = speculative_verify = paged_append
    paged_append8 = paged_attention8 = paged_reserve = paged_release = adjust_logits = count_tokens = paged_append

    @staticmethod
    def forget():
        pass


def binding():
    """The native short way to the serving operators (csrc/binding.cpp), bound to this library.

    Where it has not been built, or was built for another torch or Python, the operators are
    called through ctypes (some 8 us a call more), with one warning."""
    global _binding
    if _binding is None:
        L = lib()
        wanted = "torch %s, Python %d.%d" % (torch.__version__, *sys.version_info[:2])
        try:
            from . import _binding as native
            found = getattr(native, "built_for", "another version")
            why = None if found == wanted else f"it was built for {found}"
        except ImportError as e:
            why = str(e)
        if why is None:
            native.bind({n: ctypes.cast(getattr(L, n), ctypes.c_void_p).value for n in _BOUND}, error_ptr, stream_scratch)
            _binding = native
        else:
            warnings.warn(f"kernels/_binding.so is not used with {wanted} ({why}): the serving operators go through "
                          "ctypes. `python simsd-release_b200/build.py` builds it.", RuntimeWarning, stacklevel=3)
            _binding = _CtypesOnly()
    return _binding


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DTYPE[dt]
    except KeyError:
        raise TypeError(f"unsupported dtype {dt}; expected bfloat16, float16 or float32") from None


def check(rc: int, what: str) -> None:
    if rc == SIMSD_OK:
        return
    msg = f"{what}: {lib().simsd_status_string(rc).decode()} (status {rc})"
    if rc == SIMSD_ERR_SHAPE:
        raise ValueError(msg)
    if rc == SIMSD_ERR_DTYPE:
        raise TypeError(msg)
    raise RuntimeError(msg)


def stream_ptr(dev: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if dev.index is None else dev.index)


_SIDE_STREAMS: dict[torch.device, torch.cuda.Stream] = {}


def side_stream(dev: torch.device) -> torch.cuda.Stream:
    """A second stream per device for work that overlaps the caller's stream
    (callers order it with wait_stream on both sides)."""
    s = _SIDE_STREAMS.get(dev)
    if s is None:
        s = _SIDE_STREAMS[dev] = torch.cuda.Stream(device=dev)
    return s


def device_guard(dev: torch.device):
    """`torch.cuda.device(dev)` when `dev` is not the current device (tensors of a
    sharded model may live elsewhere); a no-op context otherwise, which keeps the
    common call cheap."""
    if dev.index is None or dev.index == torch.cuda.current_device():
        return _NO_GUARD
    return torch.cuda.device(dev)


_NO_GUARD = contextlib.nullcontext()


_WS_SIZES: dict[tuple, int] = {}


def thin_workspace_size(dev_index: int, M: int, N: int, K: int, code: int, epilogue: int, split: int) -> int:
    """simsd_thin_linear_workspace_size, memoised (pure arithmetic for a device)."""
    key = (dev_index, M, N, K, code, epilogue, split)
    v = _WS_SIZES.get(key)
    if v is None:
        v = _WS_SIZES[key] = lib().simsd_thin_linear_workspace_size(M, N, K, code, epilogue, split)
    return v


def require_cuda(*tensors: torch.Tensor) -> torch.device:
    dev = tensors[0].device
    if dev.type != "cuda":
        raise RuntimeError(
            "the simsd_b200 operators run on CUDA tensors only (no CPU fallback); "
            f"got a tensor on {dev}")
    for t in tensors[1:]:
        if t is not None and t.device != dev:
            raise RuntimeError(f"all tensors must be on {dev}; got one on {t.device}")
    return dev


# ------------------------------------------------------------------ workspaces
_WORKSPACES: dict[torch.device, torch.Tensor] = {}
# Outgrown workspaces stay alive until reset_workspace(): a CUDA graph captured
# earlier may still hold their addresses.
_RETIRED: list[torch.Tensor] = []


def workspace(dev: torch.device, nbytes: int) -> torch.Tensor:
    """Per-device scratch of at least `nbytes`, header zeroed (grows, never shrinks)."""
    buf = _WORKSPACES.get(dev)
    if buf is None or buf.numel() < nbytes:
        size = max(nbytes, 0 if buf is None else buf.numel())
        size = (size + (1 << 20) - 1) & ~((1 << 20) - 1)
        if buf is not None:
            _RETIRED.append(buf)
        buf = torch.zeros(size, dtype=torch.uint8, device=dev)
        _WORKSPACES[dev] = buf
        _ERROR_PTRS.pop(dev.index, None)
        if _binding is not None:
            _binding.forget()
    return buf


# Device index -> address of the error word in that device's workspace header.
_ERROR_PTRS: dict[int, int] = {}


def error_ptr(index: int) -> int:
    """Device address of the error word in the workspace header of CUDA device `index` (`device_error` reads it)."""
    ptr = _ERROR_PTRS.get(index)
    if ptr is None:
        ptr = _ERROR_PTRS[index] = workspace(torch.device("cuda", index), HEADER_BYTES).data_ptr() + HEADER_BYTES - 64
    return ptr


_STREAM_SCRATCH: dict[tuple[int, int], tuple[int, int, torch.Tensor]] = {}


def stream_scratch(index: int, stream: int, nbytes: int, zeroed: int):
    """(address, bytes, owner) of scratch of at least `nbytes` for `stream` of CUDA device
    `index` (both current), its first `zeroed` bytes zero when new (the operators leave
    them zero).  Each stream has its own, so calls on several streams share none; a call
    under graph capture gets one of the graph's memory, zeroed by the graph on every
    replay.  Keep the owner until the call has been issued."""
    if torch._C._cuda_isCurrentStreamCapturing():
        buf = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", index))
        buf[:zeroed].zero_()
        return buf.data_ptr(), nbytes, buf
    held = _STREAM_SCRATCH.get((index, stream))
    if held is None or held[1] < nbytes:
        # an outgrown one goes back to torch's allocator, which hands it out again
        # only to later work of the stream it was allocated on: this one
        buf = torch.zeros(nbytes, dtype=torch.uint8, device=torch.device("cuda", index))
        held = _STREAM_SCRATCH[(index, stream)] = (buf.data_ptr(), nbytes, buf)
    return held


def reset_workspace() -> None:
    """Drop the cached workspaces (call before re-capturing graphs in a new pool)."""
    _WORKSPACES.clear()
    _RETIRED.clear()
    _ERROR_PTRS.clear()
    _STREAM_SCRATCH.clear()
    if _binding is not None:
        _binding.forget()


def device_error(dev: torch.device | None = None) -> int:
    """OR of the device error bits recorded in `dev`'s workspace (synchronises)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if dev is None else dev
    buf = _WORKSPACES.get(dev)
    if buf is None:
        return 0
    out = ctypes.c_int(0)
    with torch.cuda.device(dev):
        check(lib().simsd_workspace_error(buf.data_ptr(), stream_ptr(dev), ctypes.byref(out)),
              "simsd_workspace_error")
    return out.value


def clear_device_error(dev: torch.device | None = None) -> None:
    """Zero `dev`'s workspace header (error word and tile counters), stream-ordered.  The
    streams' scratch is dropped: a launch that gave up may have left counters in it."""
    dev = torch.device("cuda", torch.cuda.current_device()) if dev is None else dev
    for key in [k for k in _STREAM_SCRATCH if dev.index in (None, k[0])]:
        del _STREAM_SCRATCH[key]
    if _binding is not None:
        _binding.forget()
    buf = _WORKSPACES.get(dev)
    if buf is None:
        return
    with torch.cuda.device(dev):
        check(lib().simsd_workspace_init(buf.data_ptr(), buf.numel(), stream_ptr(dev)),
              "simsd_workspace_init")


def _set_flag(bit: int, enable: bool) -> bool:
    L = lib()
    old = L.simsd_get_launch_flags()
    L.simsd_set_launch_flags((old | bit) if enable else (old & ~bit))
    return bool(old & bit)


def set_pdl(enable: bool) -> bool:
    """Launch kernels as programmatic dependents (weights must not be written by the
    kernel right before each call on the same stream).  Returns the previous setting."""
    return _set_flag(LAUNCH_PDL, enable)


def set_grouped_fixup(enable: bool) -> bool:
    """MoE grouped GEMMs: sum split tiles in a separate reduction kernel instead of
    inside the GEMM (the default); same bits.  Returns the previous setting."""
    return _set_flag(LAUNCH_GROUPED_FIXUP, enable)


def set_inkernel_reduce(enable: bool) -> bool:
    """Sum split-K tiles inside the GEMM (last contributor) instead of in a separate
    reduction kernel; the bits are the same either way.  Returns the previous setting."""
    return _set_flag(LAUNCH_INKERNEL_REDUCE, enable)


class moe_size_classes:
    """Context manager: MoE dispatches issued (or captured) in its body split
    each grouped GEMM by expert size (SIMSD_LAUNCH_MOE_SIZE_CLASSES)."""

    def __init__(self, enable: bool = True):
        self.enable = enable

    def __enter__(self):
        self.prev = _set_flag(LAUNCH_MOE_SIZE_CLASSES, self.enable)
        return self

    def __exit__(self, *exc):
        _set_flag(LAUNCH_MOE_SIZE_CLASSES, self.prev)
        return False


class weights_static:
    """Context manager enabling programmatic dependent launch for its body."""

    def __init__(self, enable: bool = True):
        self.enable = enable

    def __enter__(self):
        self.prev = set_pdl(self.enable)
        return self

    def __exit__(self, *exc):
        set_pdl(self.prev)
        return False
