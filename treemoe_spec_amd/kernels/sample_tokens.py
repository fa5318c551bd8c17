"""Sampling of tokens from given random numbers: temperature, top-k, top-p, min-p.

The reference samples its draft's children and the first token after a prompt in
torch; the sampling mode's verification (``fused_verify_commit`` with
``temperature > 0``, treemoe/ref/verify_ref.py:60-89) then takes the distribution
of every node as ``draft_probs``.  ``sample_tokens`` makes both, token and
distribution, in one launch.
"""

from __future__ import annotations

import math
import operator
import sys

import torch
from torch.autograd import forward_ad

from treemoe_spec_amd import _capi
from treemoe_spec_amd._capi import dtype_code, ptr


def _per_row(name, value, n, dtype, lo, hi):
    """(device tensor or None, scalar) of a parameter given as a number or [N]."""
    if isinstance(value, torch.Tensor) and value.dim() > 0:
        if value.dim() != 1 or value.shape[0] != n or value.dtype != dtype \
                or (n > 1 and value.stride(0) != 1):
            raise ValueError(f"{name} must be a number or a contiguous {dtype} tensor of N entries")
        return value, lo
    value = operator.index(value) if dtype is torch.int32 else float(value)
    if not lo <= value <= hi:
        raise ValueError(f"{name} must be {lo}..{hi}, got {value}")
    return None, value


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, *,
                  temperature: float | torch.Tensor = 1.0, top_k: int | torch.Tensor = 0,
                  top_p: float | torch.Tensor = 1.0, min_p: float | torch.Tensor = 0.0,
                  return_probs: bool = False, probs_out: torch.Tensor | None = None):
    """One token for every row of ``logits`` [N, V] (float32, bfloat16 or float16, rows
    at any stride) from ``uniforms`` [N] (float32 in [0, 1)); int64 [N].

    With w = exp((logit - max) / temperature) and tokens ordered by logit, the lower
    index first among equals: ``top_k`` keeps the first k (0: all), ``top_p`` the
    shortest prefix of those that holds top_p of their weight (at least one),
    ``min_p`` what weighs at least min_p.  The token is the first index at which
    the running sum of the kept weights exceeds uniform * their sum.  Temperature 0
    takes the largest logit.  NaN logits are never taken; a row without any logit
    above -inf gives -1.

    The parameters are numbers, or tensors [N] (float32; int32 for top_k) on the
    logits' device, whose values are clamped to their ranges.  With
    ``return_probs`` returns (tokens, probs): the distribution of every row, float32
    [N, V], in ``probs_out`` where given: the rows that ``fused_verify_commit`` takes
    as ``draft_probs``."""
    shape = logits.shape
    if len(shape) != 2:
        raise ValueError("logits must be [N, V]")
    n, v = shape
    dt = dtype_code(logits.dtype)
    if dt is None:
        raise ValueError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if not 1 <= v <= _capi.TM_MAX_SAMPLE_VOCAB:
        raise ValueError(f"V must be 1..{_capi.TM_MAX_SAMPLE_VOCAB}, got {v}")
    if n > _capi.TM_MAX_ROWS:
        raise ValueError(f"N must be at most {_capi.TM_MAX_ROWS}, got {n}")
    if uniforms.shape != (n,) or uniforms.dtype != torch.float32 \
            or (n > 1 and uniforms.stride(0) != 1):
        raise ValueError("uniforms must be a contiguous float32 tensor of N entries")
    ls = logits.stride()
    if v > 1 and ls[1] != 1:
        raise ValueError("logits must have unit stride along V")
    temps, temp = _per_row("temperature", temperature, n, torch.float32, 0.0, sys.float_info.max)
    ks, k = _per_row("top_k", top_k, n, torch.int32, 0, math.inf)
    ps, p = _per_row("top_p", top_p, n, torch.float32, 0.0, 1.0)
    ms, m = _per_row("min_p", min_p, n, torch.float32, 0.0, 1.0)
    index = logits.get_device()
    if index < 0 or uniforms.get_device() != index or logits.requires_grad \
            or uniforms.requires_grad or probs_out is not None \
            or forward_ad._current_level >= 0 \
            or not (temps is ks is ps is ms is None):
        _capi.require("sample_tokens", logits.device, logits=logits, uniforms=uniforms,
                      temperature=temps, top_k=ks, top_p=ps, min_p=ms, probs_out=probs_out)
    probs, pp, pst = None, 0, 0
    if return_probs:
        probs = probs_out
        if probs is None:
            probs = torch.empty((n, v), dtype=torch.float32, device=logits.device)
        elif probs.shape != shape or probs.dtype != torch.float32 \
                or (v > 1 and probs.stride(1) != 1):
            raise ValueError("probs_out must be float32 [N, V] with unit stride along V")
        elif probs.data_ptr() == logits.data_ptr() and n:
            raise ValueError("probs_out must lie apart from the logits")
        pp, pst = probs.data_ptr(), probs.stride(0)
    elif probs_out is not None:
        raise ValueError("probs_out without return_probs")
    tokens = torch.empty(n, dtype=torch.int64, device=logits.device)
    _capi.launch("tm_sample_tokens", index, logits.data_ptr(), dt, n, v, ls[0],
                 uniforms.data_ptr(), ptr(temps), temp, ptr(ks), min(k, v), ptr(ps), p, ptr(ms),
                 m, tokens.data_ptr(), pp, pst)
    return (tokens, probs) if return_probs else tokens
