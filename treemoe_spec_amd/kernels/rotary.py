"""Rotary positions on queries and keys, and on a prompt's way into the cache.

The reference rotates q and k in torch before ``kv.append`` or ``write_tree``
(treemoe/model/mixtral.py:172-206, kv_cache.py:62-78); here ``rotary_embed`` is one
launch for both, and ``rotary_append`` one launch for the rotation of a prompt's
chunk or of a decoded token and the cache's rows.

A ``RotaryPlan`` holds the frequencies of a model, made once: fixed-point
fractions of a turn (2^-64), so that the kernel reduces any position exactly.
"""

from __future__ import annotations

import math
import operator
from fractions import Fraction

import torch
from torch.autograd import forward_ad

from treemoe_spec_amd import _capi
from treemoe_spec_amd._capi import dtype_code
from treemoe_spec_amd.kv_cache import device_tables_of

# 2 pi to 36 digits, as a fraction: more than the 64 bits of a turn
_TWO_PI = Fraction(6283185307179586476925286766559005768, 10 ** 36)


def _check_factor(scaling: dict) -> float:
    factor = float(scaling["factor"])
    if not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError("the scaling's factor must be at least 1")
    return factor


def rotary_frequencies(dim: int, theta: float, scaling: dict | None = None):
    """(radians a position of the dim / 2 pairs, magnitude) in double precision.

    scaling: None, or a dict with "type" and "factor" s:
      linear  every frequency over s
      ntk     the base becomes theta * s ** (dim / (dim - 2))
      yarn    pairs that turn over "beta_fast" (32) times in
              "original_max_position" positions keep their frequency, those under
              "beta_slow" (1) have it over s, a linear ramp over the pair index
              between; magnitude 0.1 ln s + 1, or "attention_factor"
    """
    if scaling is None:
        return [theta ** (-2.0 * i / dim) for i in range(dim // 2)], 1.0
    kind = scaling.get("type")
    if kind not in ("linear", "ntk", "yarn"):
        raise ValueError(f"unknown rotary scaling {kind!r}")
    s = _check_factor(scaling)
    if kind == "linear":
        return [theta ** (-2.0 * i / dim) / s for i in range(dim // 2)], 1.0
    if kind == "ntk":
        if dim < 4:
            raise ValueError("ntk scaling needs at least 4 rotated elements")
        base = theta * s ** (dim / (dim - 2))
        return [base ** (-2.0 * i / dim) for i in range(dim // 2)], 1.0
    span = float(scaling["original_max_position"]) / (2.0 * math.pi)
    fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
    if not (span > 0 and fast > slow > 0):
        raise ValueError("yarn needs original_max_position > 0 and beta_fast > beta_slow > 0")

    def pair_of(turns):  # the pair that turns so often over the original length
        return dim * math.log(span / turns) / (2.0 * math.log(theta))

    lo = max(math.floor(pair_of(fast)), 0)
    hi = min(math.ceil(pair_of(slow)), dim - 1)
    out = []
    for i in range(dim // 2):
        ramp = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
        f = theta ** (-2.0 * i / dim)
        out.append(f * (1.0 - ramp) + f / s * ramp)
    return out, float(scaling.get("attention_factor", 0.1 * math.log(s) + 1.0))


class RotaryPlan:
    """Frequencies of the rotated part of a head, on one device.

    head_dim and rotary_dim (default: the whole head) are multiples of 16.
    ``interleaved``: pairs are elements (2i, 2i+1), else (i, i + rotary_dim / 2).
    ``inv_freq``: radians a position of the rotary_dim / 2 pairs in place of
    theta's and the scaling's.  Keep the plan as long as a graph that captured a call
    with it."""

    def __init__(self, head_dim: int, theta: float = 1e6, *, rotary_dim: int | None = None,
                 interleaved: bool = False, scaling: dict | None = None, inv_freq=None,
                 device="cuda"):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim % 16 or not 16 <= head_dim <= 1024:
            raise ValueError("head_dim must be a multiple of 16, 16..1024")
        if rotary_dim % 16 or not 16 <= rotary_dim <= head_dim:
            raise ValueError("rotary_dim must be a multiple of 16, at most head_dim")
        if inv_freq is None:
            if not (theta > 1.0 and math.isfinite(theta)):
                raise ValueError("theta must be above 1")
            freq, self.magnitude = rotary_frequencies(rotary_dim, float(theta), scaling)
        else:
            if scaling is not None:
                raise ValueError("give inv_freq or scaling, not both")
            freq, self.magnitude = [float(f) for f in inv_freq], 1.0
            if len(freq) != rotary_dim // 2 or not all(math.isfinite(f) for f in freq):
                raise ValueError("inv_freq must hold rotary_dim / 2 finite values")
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, rotary_dim, int(interleaved)
        self.inv_freq = freq
        turns = []
        for f in freq:
            u = round(Fraction(f) / _TWO_PI * 2 ** 64) % 2 ** 64
            turns.append(u - 2 ** 64 if u >= 2 ** 63 else u)  # the same 64 bits, signed
        self.turns = torch.tensor(turns, dtype=torch.int64).to(device)
        self.device = self.turns.device
        self.made_on = _capi.stream_made_on(self.device)


def _heads_of(name: str, t: torch.Tensor, hd: int, dtype, tokens: int) -> tuple[int, int]:
    """(heads, token stride) of a [T, heads, hd] tensor."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != tokens or shape[2] != hd:
        raise ValueError(f"{name} must be [T, heads, {hd}] with {tokens} tokens")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}")
    st = t.stride()
    if st[2] != 1 or (st[1] != hd and shape[1] > 1):
        raise ValueError(f"{name} must have contiguous heads")
    return shape[1], st[0]


def _output(name: str, out: torch.Tensor | None, x: torch.Tensor, heads: int, hd: int,
            index: int) -> tuple[torch.Tensor, int]:
    """(output like ``x``, its token stride)."""
    if out is None:
        return torch.empty_like(x, memory_format=torch.contiguous_format), heads * hd
    n, stride = _heads_of(name, out, hd, x.dtype, x.shape[0])
    if n != heads or out.get_device() != index:
        raise ValueError(f"{name} must have the shape of its input, on the same device")
    _capi.require(name, x.device, **{name: out})
    return out, stride


def rotary_embed(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                 plan: RotaryPlan, *, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None):
    """q [T, Hq, hd] and k [T, kvh, hd] (or None) rotated by ``positions`` [T] (int32
    or int64); returns (q', k').  float32, bfloat16 or float16, heads contiguous,
    tokens at any 16-byte aligned stride.  ``q_out`` may be ``q``, ``k_out`` may be
    ``k``; otherwise outputs share no memory with inputs or each other."""
    dtype, hd = q.dtype, plan.head_dim
    dt = dtype_code(dtype)
    if dt is None:
        raise ValueError(f"q must be float32, bfloat16 or float16, got {dtype}")
    index = q.get_device()
    turns = plan.turns
    if index < 0 or positions.get_device() != index or turns.get_device() != index \
            or q.requires_grad or (k is not None and (k.get_device() != index
                                                      or k.requires_grad)) \
            or forward_ad._current_level >= 0:
        _capi.require("rotary_embed", q.device, q=q, k=k, positions=positions, plan=turns)
    t = q.shape[0]
    if t > _capi.TM_MAX_ROWS:
        raise ValueError(f"T must be at most {_capi.TM_MAX_ROWS}, got {t}")
    heads, qs = _heads_of("q", q, hd, dtype, t)
    wide = positions.dtype == torch.int64
    if positions.shape != (t,) or not (wide or positions.dtype == torch.int32) \
            or (t > 1 and positions.stride(0) != 1):
        raise ValueError("positions must be a contiguous int32 or int64 tensor of T entries")
    q_out, qos = _output("q_out", q_out, q, heads, hd, index)
    kp = ks = kop = kos = kvh = 0
    if k is not None:
        kvh, ks = _heads_of("k", k, hd, dtype, t)
        k_out, kos = _output("k_out", k_out, k, kvh, hd, index)
        kp, kop = k.data_ptr(), k_out.data_ptr()
    elif k_out is not None:
        raise ValueError("k_out without k")
    _capi.launch("tm_rotary", index, q.data_ptr(), qs, kp, ks, q_out.data_ptr(), qos, kop, kos,
                 positions.data_ptr(), 1 if wide else 0, turns.data_ptr(), plan.magnitude, t,
                 heads, kvh, hd, plan.rotary_dim, plan.interleaved, dt)
    _capi.used_by(index, plan.made_on, turns)
    return q_out, k_out


def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: RotaryPlan, kv,
                  layer: int, start_pos: int, *, q_out: torch.Tensor | None = None):
    """Tokens at positions start_pos .. start_pos + T - 1: returns q [T, Hq, hd]
    rotated, and stores the rotated k and v [T, kvh, hd] at those positions of the
    paged cache ``kv``, mapping pages as ``append`` does (treemoe/model/kv_cache.py:
    62-78); ``kv.seq_len`` grows to cover them.  A call that maps a page copies the block
    table to the device and waits for it, so a capture needs its pages mapped by an
    eager call before; a replay repeats the positions of the capture, in the pages that
    the device table then holds."""
    dtype, hd = q.dtype, plan.head_dim
    dt = dtype_code(dtype)
    if dt is None:
        raise ValueError(f"q must be float32, bfloat16 or float16, got {dtype}")
    kc, vc, turns = kv.k, kv.v, plan.turns
    index = q.get_device()
    if index < 0 or k.get_device() != index or v.get_device() != index \
            or turns.get_device() != index or kc.get_device() != index \
            or vc.get_device() != index or q.requires_grad or k.requires_grad \
            or v.requires_grad or kc.requires_grad or vc.requires_grad \
            or forward_ad._current_level >= 0:
        _capi.require("rotary_append", q.device, q=q, k=k, v=v, plan=turns, k_cache=kc,
                      v_cache=vc)
    t = q.shape[0]
    if t > _capi.TM_MAX_ROWS:
        raise ValueError(f"T must be at most {_capi.TM_MAX_ROWS}, got {t}")
    heads, qs = _heads_of("q", q, hd, dtype, t)
    kvh, ks = _heads_of("k", k, hd, dtype, t)
    vh, vs = _heads_of("v", v, hd, dtype, t)
    if vh != kvh:
        raise ValueError("k and v must have the same shape")
    cshape, cst = kc.shape, kc.stride()
    if kc.dtype != dtype or vc.dtype != dtype or vc.shape != cshape or vc.stride() != cst \
            or len(cshape) != 5 or cshape[3] != kvh or cshape[4] != hd or cst[4] != 1 \
            or (cst[3] != hd and kvh > 1) or cshape[2] != kv.block_size:
        raise ValueError("cache layout must be [L, pages, page, kv_heads, head_dim] of q's dtype")
    layer, start_pos = operator.index(layer), operator.index(start_pos)
    layers = cshape[0]
    if not -layers <= layer < layers:
        raise IndexError(f"layer {layer} is out of range for a cache of {layers} layers")
    if start_pos < 0:
        raise ValueError("start_pos must not be negative")
    q_out, qos = _output("q_out", q_out, q, heads, hd, index)
    if t == 0:
        return q_out
    end = start_pos + t
    kv._ensure_capacity(end)
    table, _ = device_tables_of(kv, q.device)
    off = kc.element_size() * cst[0] * (layer % layers)
    _capi.launch("tm_rotary_append", index, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
                 q_out.data_ptr(), qos, kc.data_ptr() + off, vc.data_ptr() + off, cst[1], cst[2],
                 cshape[2], cshape[1], table.data_ptr(), len(kv.block_table), start_pos,
                 turns.data_ptr(), plan.magnitude, t, heads, kvh, hd, plan.rotary_dim,
                 plan.interleaved, dt)
    _capi.used_by(index, plan.made_on, turns)
    kv.seq_len = max(kv.seq_len, end)
    return q_out
