"""ctypes binding of libtreemoe_amd.so (declared in include/treemoe_amd.h).

The library is loaded once per process.  A missing library is an error: the
product path has no CPU fallback.
"""

from __future__ import annotations

import ctypes
import functools
import os
from pathlib import Path

_LIB_PATH = Path(os.environ.get(
    "TREEMOE_AMD_LIB", Path(__file__).resolve().parent / "libtreemoe_amd.so"))

P = ctypes.c_void_p
I64 = ctypes.c_int64
I32 = ctypes.c_int
F32 = ctypes.c_float
F64 = ctypes.c_double

# name -> argtypes; every entry point returns int (0 = ok)
SIGNATURES: dict[str, list] = {
    "tm_op1_router_gates": [P, P, I64, I64, I64, P, I32, P],
    "tm_op1_route_bucket": [P, P, I64, I64, I64, F32, I32, I64, I64, I64] + [P] * 10 + [P],
    "tm_op1_route": [P, P, P, I64, I64, I64, I64, F32, I32, I64, I64, I64] + [P] * 11 + [I32, P],
    "tm_op1_gemm1": [P, P, P, P, P, P, I64, I64, I64, I64, I64, I32, P],
    "tm_op1_gemm2": [P, P, P, P, P, P, I64, I64, I64, I64, I64, I64, I32, P],
    "tm_op1_combine": [P, P, P, I64, I64, I64, I32, P],
    "tm_op1_prefill_gemm1": [P, P, P, P, P, P, P, I64, I64, I64, I64, I64, I32, P],
    "tm_op1_prefill_gemm2": [P, P, P, P, P, P, P, I64, I64, I64, I64, I64, I64, I32, P],
    "tm_op1_prefill_tiles": [I64] * 6 + [P, P],
    "tm_op1_prefill_gemm1_routed": [P] * 6 + [I64] * 5 + [F32, I32, I64, I64, I64] + [P] * 10
                                   + [I32, P],
    "tm_op4_argmax_walk": [P, I32, I64, I64, I64, P, P, P, P, I64, I64, I32, P, P, P, P, P, P],
    "tm_op4_kv_commit": [P, P, I64, I64, I64, I64, I64, I64, I64, P, P, P, I64, P, I64, I64,
                         I64, P, P],
    "tm_host_device_pointer": [P, P],
    "tm_stream_capture_id": [P, P],
    "tm_op4_argmax_walk_noalloc": [P, I32, I64, I64, I64, P, P, P, P, I64, I64, I32, P, P, P,
                                   P, P],
    "tm_op4_rep_penalty": [P, I32, I64, I64, I64, P, I64, F32, P, I64, P],
    "tm_op4_sample_walk": [P, I32, I64, I64, I64, P, I64, P, P, P, P, I64, P, P, F32, P, P, P,
                           P, P],
    "tm_tree_attention": [P, I64, P, P, I64, P, P, I64, I64, I64, P, I64, I64, P, I64, I32, P,
                          I64, I64, I64, I64, F32, P, I64, I64, P, I64, P],
    "tm_tree_attention_plan": [I64, I64, I64, I64, I64, I64, I64, P, P],
    "tm_tree_mask_pack": [P, I64, I64, P, P],
    "tm_rms_norm": [P, I64, P, I64, I32, P, I32, I64, I64, F32, I32, P, I64, P, I64, P],
    "tm_rms_norm_fp8": [P, I64, P, I64, I32, P, I32, I64, I64, F32, I32, P, I64, P, I64, I64, P,
                        I64, P],
    "tm_rotary": [P, I64] * 4 + [P, I32, P, F32] + [I64] * 5 + [I32, I32, P],
    "tm_rotary_append": [P, I64] * 4 + [P, P, I64, I64, I64, I64, P, I64, I64, P, F32]
                        + [I64] * 5 + [I32, I32, P],
    "tm_sample_tokens": [P, I32, I64, I64, I64, P, P, F64, P, I64, P, F64, P, F64, P, P, I64, P],
    "tm_prompt_plan": [P, P, I64, I64, I64, P, I64, P, I64, P],
    "tm_prompt_attention": [P, I64] * 3 + [P, I64, P] + [I64] * 6 + [F32, I32, P, I64, P, I64, P],
    "tm_prompt_cached_workspace": [I64] * 5 + [P],
    "tm_prompt_attention_cached": [P, I64, I64, P, P, I64, I64, I64, I64, P, I64, I64, I64, I64,
                                   I64, F32, I32, P, I64, P, I64, P],
}

TM_OBJECTIVE = {"mass": 0, "critical_path": 1}
TM_DTYPE_F32 = 0
TM_DTYPE_BF16 = 1
TM_DTYPE_F16 = 2
TM_GEMM_TILE_M = 64
TM_OP4_MAX_PARTS = 64
TM_OP4_NOALLOC_MAX_NODES = 2048
TM_MAX_NORM_HIDDEN = 65536
TM_MAX_SAMPLE_VOCAB = 262144
TM_MAX_PROMPT_KEYS = 1 << 24
TM_MAX_ROWS = 1 << 21

_lib = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not _LIB_PATH.exists():
            raise RuntimeError(
                f"treemoe_spec_amd: native library {_LIB_PATH} is missing; build it with "
                "`python -m treemoe_spec_amd._build` (there is no CPU fallback)")
        handle = ctypes.CDLL(str(_LIB_PATH))
        for name, argtypes in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.argtypes = argtypes
            fn.restype = ctypes.c_int
        handle.tm_version.argtypes = []
        handle.tm_version.restype = ctypes.c_int
        handle.tm_status_string.argtypes = [ctypes.c_int]
        handle.tm_status_string.restype = ctypes.c_char_p
        _lib = handle
    return _lib


def fast_binding():
    """The CPython binding of the per-step entry points, or None where it is not
    built or TREEMOE_AMD_LIB names a library other than the one it is linked to."""
    if _LIB_PATH.resolve() != Path(__file__).resolve().parent / "libtreemoe_amd.so":
        return None
    try:
        from treemoe_spec_amd import _tmfast
    except ImportError:
        return None
    return _tmfast


@functools.cache
def layer_binding():
    """The CPython binding _tmlayer, or None where it is not built or
    TREEMOE_AMD_LIB names a library other than the one it is linked to."""
    if _LIB_PATH.resolve() != Path(__file__).resolve().parent / "libtreemoe_amd.so":
        return None
    try:
        from treemoe_spec_amd import _tmlayer
    except ImportError:
        return None
    return _tmlayer


@functools.cache
def entry(name: str):
    """An entry point as a callable that returns its status: that of the CPython
    binding where there is one, else ctypes."""
    return getattr(layer_binding() or lib(), name)


def launch(name: str, index: int, *args) -> None:
    """An entry point on torch's current stream of device ``index``, with that device
    current during the call."""
    import torch

    if index == torch._C._cuda_getDevice():
        rc = entry(name)(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = entry(name)(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, name)


def stream_made_on(device) -> int | None:
    """torch's current raw stream of ``device``, None for one that has none."""
    import torch

    return torch._C._cuda_getCurrentRawStream(device.index) if device.type == "cuda" else None


def used_by(index: int, made_on: int | None, *tensors) -> None:
    """A call on torch's current stream of device ``index`` reads ``tensors``, which a plan
    allocated on the raw stream ``made_on``: where the streams differ their memory is not
    given away, once the plan is gone, before that call has ended."""
    import torch

    if made_on is not None and torch._C._cuda_getCurrentRawStream(index) != made_on:
        stream = torch.cuda.current_stream(index)
        for t in tensors:
            t.record_stream(stream)


@functools.cache
def dtype_code(dtype) -> int | None:
    """TM_DTYPE_* of a torch dtype, None for one that the kernels do not take."""
    import torch

    return {torch.float32: TM_DTYPE_F32, torch.bfloat16: TM_DTYPE_BF16,
            torch.float16: TM_DTYPE_F16}.get(dtype)


def require(what: str, device, **tensors) -> None:
    """All given tensors on ``device``, a ROCm device, and none that a gradient is
    asked of or that carries a forward-mode tangent: these operators have no
    derivatives.  (Callers look for the common case themselves and come here for the
    error: host time is what bounds their smallest calls.)"""
    import torch
    from torch.autograd import forward_ad

    if device.type != "cuda":
        raise RuntimeError(f"treemoe_spec_amd {what} runs on ROCm devices only; "
                           f"got a tensor on {device}")
    grad = torch.is_grad_enabled()
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")
        if grad and t.requires_grad:
            raise RuntimeError(f"{what} has no backward pass, but {name} requires a gradient; "
                               "call it under torch.no_grad()")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no forward derivative, but {name} carries a tangent; "
                               "call it on the primal")


def check(rc: int, what: str) -> None:
    if rc != 0:
        msg = lib().tm_status_string(rc).decode()
        raise RuntimeError(f"{what} failed with status {rc}: {msg}")


def call(name: str, *args) -> None:
    check(getattr(lib(), name)(*args), name)


def ptr(t) -> int:
    """Device address of a torch tensor (None -> NULL)."""
    return 0 if t is None else t.data_ptr()


def stream_of(device) -> int:
    """Raw handle of torch's current stream on ``device`` (a torch.device,
    'cuda[:N]' or an index)."""
    import torch

    if isinstance(device, int):
        idx = device
    else:
        idx = (device if isinstance(device, torch.device) else torch.device(device)).index
    if idx is None:
        idx = torch.cuda.current_device()
    return torch._C._cuda_getCurrentRawStream(idx)
