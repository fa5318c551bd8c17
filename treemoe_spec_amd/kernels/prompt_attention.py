"""Causal attention of prompts, packed or over the paged cache, down to one token.

The reference's prompt branch (treemoe/model/mixtral.py:208-250) appends the prompt's
keys to the cache, gathers the whole sequence and calls
``F.scaled_dot_product_attention`` with a causal mask, one sequence at a time.
``prompt_attention`` takes many sequences packed one after the other,
``prompt_attention_cached`` reads one sequence's pages in place: a prompt, a later
chunk of one, or a decoded token.  The context comes back as [T, Hq * hd], the layout
``o_proj`` takes.
"""

from __future__ import annotations

import ctypes
import operator

import torch
from torch.autograd import forward_ad

from treemoe_spec_amd import _capi
from treemoe_spec_amd._capi import dtype_code, ptr
from treemoe_spec_amd.kv_cache import device_tables_of


class PromptPlan:
    """The work list of ``prompt_attention`` for one batch, made once and used by
    every layer.  ``q_lens``: each sequence's queries; ``k_lens`` (default: the same):
    its keys, of which the queries are the last.  A graph that captured a call reads the
    plan's lists on every replay: keep the plan as long as the graph."""

    def __init__(self, q_lens, k_lens=None, *, num_heads: int, num_kv_heads: int,
                 device="cuda"):
        q_lens = [operator.index(n) for n in q_lens]
        k_lens = q_lens if k_lens is None else [operator.index(n) for n in k_lens]
        if len(k_lens) != len(q_lens):
            raise ValueError("q_lens and k_lens must have the same length")
        for nq, nk in zip(q_lens, k_lens):
            if not 0 <= nq <= nk <= _capi.TM_MAX_PROMPT_KEYS:
                raise ValueError("every sequence needs 0 <= queries <= keys <= "
                                 f"{_capi.TM_MAX_PROMPT_KEYS}, got {nq} and {nk}")
        if num_kv_heads < 1 or num_heads < num_kv_heads or num_heads % num_kv_heads:
            raise ValueError("num_heads must be a multiple of num_kv_heads")
        n = len(q_lens)
        ql, kl = (ctypes.c_int64 * n)(*q_lens), (ctypes.c_int64 * n)(*k_lens)
        sizes = (ctypes.c_int64 * 7)()
        _capi.call("tm_prompt_plan", ql, kl, n, num_heads, num_kv_heads, None, 0, None, 0, sizes)
        items = torch.zeros(max(1, sizes[0]), 8, dtype=torch.int32)
        joins = torch.zeros(max(1, sizes[1]), 8, dtype=torch.int32)
        _capi.call("tm_prompt_plan", ql, kl, n, num_heads, num_kv_heads, items.data_ptr(),
                   sizes[0], joins.data_ptr(), sizes[1], sizes)
        self.num_items, self.num_joins, self.num_slots, self.tiling, self.q_rows, \
            self.k_rows, self.tile_rows = list(sizes)
        self.num_heads, self.num_kv_heads = num_heads, num_kv_heads
        self.items, self.joins = items.to(device), joins.to(device)
        self.device = self.items.device
        self.made_on = _capi.stream_made_on(self.device)


def _check_q(q: torch.Tensor, out: torch.Tensor | None):
    """(dtype code, T, Hq, hd, token stride of q, of out) of q; checks ``out``."""
    dt = dtype_code(q.dtype)
    if dt is None or dt == _capi.TM_DTYPE_F32:
        raise ValueError(f"q must be bfloat16 or float16, got {q.dtype}")
    shape = q.shape
    if len(shape) != 3:
        raise ValueError("q must be [T, heads, head_dim]")
    t, hq, hd = shape
    st = q.stride()
    if hd != 128 and hd != 64:
        raise ValueError(f"head_dim must be 64 or 128, got {hd}")
    if st[2] != 1 or (st[1] != hd and hq > 1):
        raise ValueError("q must have contiguous heads")
    width = hq * hd
    ost = width
    if out is not None:
        if out.shape != (t, width) or out.dtype != q.dtype or out.stride(1) != 1:
            raise ValueError("out must be [T, Hq * hd] of q's dtype")
        ost = out.stride(0) if t > 1 else width
        if out.data_ptr() == q.data_ptr() and t:
            raise ValueError("out must lie apart from q, k and v")
    # (the stride of one token says nothing)
    return dt, t, hq, hd, st[0] if t > 1 else width, ost


def _check_scale(scale: float | None, hd: int) -> float:
    if scale is None:
        return hd ** -0.5
    scale = float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError("scale must be positive")
    return scale


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PromptPlan, *,
                     scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """q [T, Hq, hd], k and v [S, kvh, hd] (bfloat16 or float16, head_dim 64 or 128,
    heads contiguous): ``plan``'s sequences one after the other.  A query attends to
    its sequence's keys up to its own position.  Returns [T, Hq * hd]; T and S may
    exceed the plan's rows (a padded batch): in a new result the rows behind the last
    sequence are 0 (a fill by torch), in ``out`` they stay as they were.  ``out``
    shares no memory with q, k and v."""
    dt, t, hq, hd, qs, ost = _check_q(q, out)
    index = q.get_device()
    if index < 0 or k.get_device() != index or v.get_device() != index \
            or plan.items.get_device() != index or out is not None or q.requires_grad \
            or k.requires_grad or v.requires_grad or forward_ad._current_level >= 0:
        _capi.require("prompt_attention", q.device, q=q, k=k, v=v, plan=plan.items, out=out)
    for name, x in (("k", k), ("v", v)):
        if x.dim() != 3 or x.shape[2] != hd or x.dtype != q.dtype or x.shape != k.shape:
            raise ValueError("k and v must be [S, kv_heads, head_dim] of q's dtype")
        if x.stride(2) != 1 or (x.stride(1) != hd and x.shape[1] > 1):
            raise ValueError(f"{name} must have contiguous heads")
    s, kvh, _ = k.shape
    if hq != plan.num_heads or kvh != plan.num_kv_heads:
        raise ValueError(f"the plan is for {plan.num_heads} heads over {plan.num_kv_heads}, "
                         f"got {hq} over {kvh}")
    if t < plan.q_rows or s < plan.k_rows:
        raise ValueError(f"the plan's sequences need {plan.q_rows} queries and {plan.k_rows} "
                         f"keys, got {t} and {s}")
    scale = _check_scale(scale, hd)
    if out is None:
        out = torch.empty((t, hq * hd), dtype=q.dtype, device=q.device)
        if t > plan.q_rows:
            out[plan.q_rows:].zero_()
    nbytes = plan.num_slots * kvh * plan.tile_rows * (hd + 2) * 4
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _capi.launch("tm_prompt_attention", index, q.data_ptr(), qs, k.data_ptr(),
                 k.stride(0) if s > 1 else kvh * hd, v.data_ptr(),
                 v.stride(0) if s > 1 else kvh * hd, plan.items.data_ptr(), plan.num_items,
                 plan.joins.data_ptr(), plan.num_joins, plan.num_slots, plan.tiling, hq, kvh,
                 hd, scale, dt, out.data_ptr(), ost, ptr(ws), nbytes)
    _capi.used_by(index, plan.made_on, plan.items, plan.joins)
    return out


def _workspace_bytes(*sizes) -> int:
    """tm_prompt_cached_workspace(T, seq_len, Hq, kvh, hd)."""
    fast = _capi.layer_binding()
    if fast is not None:
        rc, nbytes = fast.prompt_cached_workspace(*sizes)
        if rc:
            _capi.check(rc, "tm_prompt_cached_workspace")
        return nbytes
    size = ctypes.c_int64()
    _capi.call("tm_prompt_cached_workspace", *sizes, ctypes.byref(size))
    return size.value


def prompt_attention_cached(q: torch.Tensor, kv, layer: int, *, scale: float | None = None,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """q [T, Hq, hd]: the last T of ``kv``'s ``seq_len`` positions, whose keys and values
    the cache holds already (``rotary_append``, ``append``).  Query t attends to
    positions 0 .. seq_len - T + t of ``layer``, read in place through the block table.
    The cache is [L, pages, page, kv_heads, head_dim] of q's dtype, page size a power of
    two.  Returns [T, Hq * hd].  A replay of a captured call repeats the length of the
    capture, in the pages that the cache's device table then holds."""
    dt, t, hq, hd, qs, ost = _check_q(q, out)
    kc, vc = kv.k, kv.v
    index = q.get_device()
    if index < 0 or kc.get_device() != index or vc.get_device() != index or out is not None \
            or q.requires_grad or kc.requires_grad or vc.requires_grad \
            or forward_ad._current_level >= 0:
        _capi.require("prompt_attention_cached", q.device, q=q, k_cache=kc, v_cache=vc, out=out)
    cshape, cst = kc.shape, kc.stride()
    if kc.dtype != q.dtype or vc.dtype != q.dtype or vc.shape != cshape or vc.stride() != cst \
            or len(cshape) != 5 or cshape[4] != hd or cst[4] != 1 \
            or (cst[3] != hd and cshape[3] > 1) or cshape[2] != kv.block_size:
        raise ValueError("cache layout must be [L, pages, page, kv_heads, head_dim] of q's dtype")
    layers, pages, page, kvh, _ = cshape
    if hq % kvh:
        raise ValueError("num_heads must be a multiple of num_kv_heads")
    if page & (page - 1):
        raise ValueError(f"page size must be a power of two, got {page}")
    layer = operator.index(layer)
    if not -layers <= layer < layers:
        raise IndexError(f"layer {layer} is out of range for a cache of {layers} layers")
    seq_len = kv.seq_len
    if t > seq_len:
        raise ValueError(f"{t} queries over a cache of {seq_len} positions")
    scale = _check_scale(scale, hd)
    dev = q.device
    if out is None:
        out = torch.empty((t, hq * hd), dtype=q.dtype, device=dev)
    if t == 0:
        return out
    table, _ = device_tables_of(kv, dev)
    nbytes = _workspace_bytes(t, seq_len, hq, kvh, hd)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    off = kc.element_size() * cst[0] * (layer % layers)
    _capi.launch("tm_prompt_attention_cached", index, q.data_ptr(), qs, t, kc.data_ptr() + off,
                 vc.data_ptr() + off, cst[1], cst[2], page, pages, table.data_ptr(),
                 len(kv.block_table), seq_len, hq, kvh, hd, scale, dt, out.data_ptr(), ost,
                 ptr(ws), nbytes)
    return out
