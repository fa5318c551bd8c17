"""Root-mean-square norm with the residual's addition, and its 8-bit form.

The reference's decoder layer (treemoe/model/mixtral.py:268-340) adds the
attention's or the experts' output to the residual stream and norms the sum, as
separate torch operations; here both are one launch of ``tm_rms_norm``.  The
8-bit form writes the normed rows as OCP e4m3 with float32 scales, the operands of
an 8-bit product.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from treemoe_spec_amd import _capi
from treemoe_spec_amd._capi import dtype_code

_SCALE_GROUPS = (32, 64, 128, 256, 512)
_ROWS = torch.contiguous_format


def _checked(what, x, weight, eps, residual, residual_out):
    """(device index, T, H, x's row stride, dtype codes of x, weight and residual)."""
    shape, wshape = x.shape, weight.shape
    if len(shape) != 2 or len(wshape) != 1 or wshape[0] != shape[1]:
        raise ValueError("x must be [T, H] and weight [H]")
    t, h = shape
    dt, wdt = dtype_code(x.dtype), dtype_code(weight.dtype)
    if dt is None:
        raise ValueError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    if wdt != dt and wdt != _capi.TM_DTYPE_F32:
        raise ValueError("weight must have x's dtype or float32")
    if h < 1 or h > _capi.TM_MAX_NORM_HIDDEN:
        raise ValueError(f"H must be 1..{_capi.TM_MAX_NORM_HIDDEN}, got {h}")
    if t > _capi.TM_MAX_ROWS:
        raise ValueError(f"T must be at most {_capi.TM_MAX_ROWS}, got {t}")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    index = x.get_device()
    if index < 0 or weight.get_device() != index or residual_out is not None \
            or (residual is not None and (residual.get_device() != index
                                          or residual.requires_grad)) \
            or x.requires_grad or weight.requires_grad or forward_ad._current_level >= 0:
        _capi.require(what, x.device, x=x, weight=weight, residual=residual,
                      residual_out=residual_out)
    xs, step = x.stride()
    if step != 1 or weight.stride(0) != 1:
        raise ValueError("x and weight must have unit stride along H")
    rdt = 0
    if residual is not None:
        rdt = dtype_code(residual.dtype)
        if residual.shape != shape or residual.stride(1) != 1:
            raise ValueError("residual must be [T, H] like x, with unit stride along H")
        if rdt != dt and rdt != _capi.TM_DTYPE_F32:
            raise ValueError("residual must have x's dtype or float32")
        if residual_out is not None and (residual_out.shape != shape
                                         or residual_out.dtype != residual.dtype
                                         or residual_out.stride(1) != 1):
            raise ValueError("residual_out must be [T, H] of the residual's dtype")
    elif residual_out is not None:
        raise ValueError("residual_out without a residual")
    return index, t, h, xs, dt, wdt, rdt


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, *,
             residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
             residual_out: torch.Tensor | None = None):
    """``s = x (+ residual)``; returns ``s / sqrt(mean(s ** 2) + eps) * weight`` in
    x's dtype, and with a residual the pair of that and ``s`` in the residual's
    dtype.  x [T, H] float32, bfloat16 or float16, rows at any stride; weight [H] and
    residual [T, H] in x's dtype or float32.  The norm takes ``s`` before it is
    rounded.  ``out`` may be ``x`` and ``residual_out`` may be ``residual``;
    otherwise outputs share no memory with inputs or each other."""
    index, t, h, xs, dt, wdt, rdt = _checked("rms_norm", x, weight, eps, residual, residual_out)
    if out is None:
        out = torch.empty_like(x, memory_format=_ROWS)
        ost = h
    else:
        if out.shape != x.shape or out.dtype != x.dtype or out.stride(1) != 1 \
                or out.get_device() != index:
            raise ValueError("out must be [T, H] of x's dtype, on x's device")
        ost = out.stride(0)
        _capi.require("rms_norm", x.device, out=out)
    if residual is None:
        _capi.launch("tm_rms_norm", index, x.data_ptr(), xs, 0, 0, dt, weight.data_ptr(), wdt,
                     t, h, eps, dt, out.data_ptr(), ost, 0, 0)
        return out
    if residual_out is None:
        residual_out = torch.empty_like(residual, memory_format=_ROWS)
        ros = h
    else:
        ros = residual_out.stride(0)
    _capi.launch("tm_rms_norm", index, x.data_ptr(), xs, residual.data_ptr(), residual.stride(0),
                 rdt, weight.data_ptr(), wdt, t, h, eps, dt, out.data_ptr(), ost,
                 residual_out.data_ptr(), ros)
    return out, residual_out


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, *,
                 residual: torch.Tensor | None = None, scale_group: int | None = None,
                 residual_out: torch.Tensor | None = None):
    """The norm as ``float8_e4m3fn`` [T, H] and float32 scales: one for every row
    ([T], the default) or for every ``scale_group`` columns (32, 64, 128, 256 or
    512; [T, H / scale_group]).  A scale is the largest magnitude over 448 (1 where
    that is 0), a value the norm over its scale, rounded to the nearest e4m3.  Returns
    (values, scales), with a residual (values, scales, sum)."""
    if scale_group is not None and (scale_group not in _SCALE_GROUPS
                                    or x.shape[-1] % scale_group != 0):
        raise ValueError(f"scale_group must be one of {_SCALE_GROUPS} and divide H")
    index, t, h, xs, dt, wdt, rdt = _checked("rms_norm_fp8", x, weight, eps, residual,
                                             residual_out)
    dev = x.device
    out = torch.empty((t, h), dtype=torch.float8_e4m3fn, device=dev)
    groups = 1 if scale_group is None else h // scale_group
    scales = torch.empty((t,) if scale_group is None else (t, groups), dtype=torch.float32,
                         device=dev)
    if residual is None:
        _capi.launch("tm_rms_norm_fp8", index, x.data_ptr(), xs, 0, 0, dt, weight.data_ptr(),
                     wdt, t, h, eps, dt, out.data_ptr(), h, scales.data_ptr(), groups,
                     scale_group or 0, 0, 0)
        return out, scales
    if residual_out is None:
        residual_out = torch.empty_like(residual, memory_format=_ROWS)
    _capi.launch("tm_rms_norm_fp8", index, x.data_ptr(), xs, residual.data_ptr(),
                 residual.stride(0), rdt, weight.data_ptr(), wdt, t, h, eps, dt, out.data_ptr(),
                 h, scales.data_ptr(), groups, scale_group or 0, residual_out.data_ptr(),
                 residual_out.stride(0))
    return out, scales, residual_out
