"""Attention of many branches of one sequence: requests behind a shared prompt, beams,
drafted chains.

The reference continues one sequence at a time (treemoe/model/mixtral.py:208-250).  Here
the tokens of all branches go through a layer together: ``branch_attention`` reads the
shared sequence's pages (once for all branches, where each adds few tokens), each branch's
own keys from a ``BranchCache``, and stores the new keys and values there.  The context comes back as
[T, Hq * hd], the layout ``o_proj`` takes.
"""

from __future__ import annotations

import ctypes
import operator

import torch

from treemoe_spec_amd import _capi
from treemoe_spec_amd._capi import ptr
from treemoe_spec_amd.kernels.prompt_attention import _check_q, _check_scale
from treemoe_spec_amd.kv_cache import device_tables_of


class BranchPlan:
    """Lists of a step in which the branches add different numbers of tokens
    (``counts``, 0 for a branch that takes no part), made once and used by every
    layer.  A graph that captured a call reads them on every replay: keep the plan as
    long as the graph."""

    def __init__(self, counts, *, num_heads: int, num_kv_heads: int, device="cuda"):
        counts = [operator.index(n) for n in counts]
        if any(not 0 <= n <= _capi.TM_MAX_PROMPT_KEYS for n in counts):
            raise ValueError(f"counts must be 0..{_capi.TM_MAX_PROMPT_KEYS}")
        if num_kv_heads < 1 or num_heads < num_kv_heads or num_heads % num_kv_heads:
            raise ValueError("num_heads must be a multiple of num_kv_heads")
        n = len(counts)
        host = (ctypes.c_int64 * n)(*counts)
        sizes = (ctypes.c_int64 * 3)()
        _capi.call("tm_branch_plan", host, n, num_heads, num_kv_heads, None, 0, None, 0, sizes)
        self.num_units, self.total, self.max_count = list(sizes)
        lists = torch.zeros(max(1, self.num_units + self.total), 4, dtype=torch.int32)
        tokens = lists[self.num_units:]
        _capi.call("tm_branch_plan", host, n, num_heads, num_kv_heads, lists.data_ptr(),
                   self.num_units, tokens.data_ptr() if self.total else None, self.total, sizes)
        self.counts, self.num_heads, self.num_kv_heads = counts, num_heads, num_kv_heads
        self.lists = lists.to(device)
        self.device_counts = torch.tensor(counts, dtype=torch.int32).to(device)
        self.device = self.lists.device
        self.made_on = _capi.stream_made_on(self.device)


def branch_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv, branches, layer: int,
                     plan: BranchPlan | None = None, *, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """q [T, Hq, hd], k and v [T, kvh, hd] (bfloat16 or float16, head_dim 64 or 128,
    heads contiguous, q and k rotated): the new tokens of every branch, branch after
    branch; without a ``plan`` the same number of each.  A token sees ``kv``'s
    ``seq_len`` positions, what its branch holds, and the branch's new tokens up to
    itself.  k and v are stored behind what the branches hold in ``layer`` of
    ``branches``, which hold them from ``branches.advance`` on, after the last layer.

    ``kv``: [L, pages, page, kv_heads, head_dim], page size a power of two; its
    ``seq_len`` may be 0.  With a plan, T may exceed its tokens (a padded batch): in a new
    result those rows are 0 (a fill by torch), in ``out`` they stay as they were.
    Returns [T, Hq * hd]; ``out`` shares no memory with the other tensors.  A replay of a
    captured call takes the sequence's length from the capture and the branches' from the
    device."""
    dt, t, hq, hd, qs, ost = _check_q(q, out)
    kc, vc, bk, bv = kv.k, kv.v, branches.k, branches.v
    lengths, origin = branches.lengths, branches.origin
    dtype = q.dtype
    index = q.get_device()
    if not _capi.ready(index, q, k, v, kc, vc, bk, bv, lengths, origin, out,
                       plan and plan.lists):
        _capi.require("branch_attention", q.device, q=q, k=k, v=v, k_cache=kc, v_cache=vc,
                      branch_k=bk, branch_v=bv, lengths=lengths, origin=origin,
                      plan=plan and plan.lists, out=out)
    kshape, ks, vs = k.shape, k.stride(), v.stride()
    if len(kshape) != 3 or kshape[0] != t or kshape[2] != hd or v.shape != kshape \
            or k.dtype != dtype or v.dtype != dtype:
        raise ValueError("k and v must be [T, kv_heads, head_dim] of q's dtype")
    kvh = kshape[1]
    if ks[2] != 1 or vs[2] != 1 or (kvh > 1 and (ks[1] != hd or vs[1] != hd)):
        raise ValueError("k and v must have contiguous heads")
    if kvh < 1 or hq % kvh:
        raise ValueError("num_heads must be a multiple of num_kv_heads")
    cshape, cst = kc.shape, kc.stride()
    if kc.dtype != dtype or vc.dtype != dtype or vc.shape != cshape or vc.stride() != cst \
            or len(cshape) != 5 or cshape[3] != kvh or cshape[4] != hd or cst[4] != 1 \
            or (cst[3] != hd and kvh > 1) or cshape[2] != kv.block_size:
        raise ValueError("cache layout must be [L, pages, page, kv_heads, head_dim] of q's dtype")
    layers, pages, page = cshape[0], cshape[1], cshape[2]
    if page & (page - 1):
        raise ValueError(f"page size must be a power of two, got {page}")
    bshape, bst = bk.shape, bk.stride()
    if bk.dtype != dtype or bv.dtype != dtype or bv.shape != bshape or bv.stride() != bst \
            or len(bshape) != 5 or bshape[3] != kvh or bshape[4] != hd or bst[4] != 1 \
            or (bst[3] != hd and kvh > 1):
        raise ValueError("branches must be [L, rows, capacity, kv_heads, head_dim] of q's dtype")
    rows, capacity = bshape[1], bshape[2]
    if lengths.dtype != torch.int32 or lengths.shape != (rows,) or not lengths.is_contiguous():
        raise ValueError("the branches' lengths must be contiguous int32 [rows]")
    if origin is not None and (origin.dtype != torch.int32 or origin.stride(1) != 1
                               or origin.shape != (rows, capacity)):
        raise ValueError("the branches' origin must be int32 [rows, capacity]")
    layer = operator.index(layer)
    if not (-layers <= layer < layers and -bshape[0] <= layer < bshape[0]):
        raise IndexError(f"layer {layer} is out of range for caches of {layers} and {bshape[0]} "
                         "layers")
    group = hq // kvh
    if plan is None:
        if t % rows:
            raise ValueError(f"{t} tokens of {rows} branches: give a plan where they differ")
        total, count = t, t // rows
        tile = 32 if count * group <= 32 else 128
        units, tokens, num_units = 0, 0, rows * -(-count * group // tile)
    else:
        if plan.num_heads != hq or plan.num_kv_heads != kvh or len(plan.counts) != rows:
            raise ValueError(f"the plan is for {plan.num_heads} heads over {plan.num_kv_heads} and "
                             f"{len(plan.counts)} branches, got {hq} over {kvh} and {rows}")
        total, count, num_units = plan.total, plan.max_count, plan.num_units
        if t < total:
            raise ValueError(f"the plan needs {total} tokens, got {t}")
        units = plan.lists.data_ptr()
        tokens = units + 16 * num_units
    longest = branches.longest
    most = longest + count
    if most > capacity and plan is not None and hasattr(branches, "host_lengths"):
        most = max(a + b for a, b in zip(branches.host_lengths, plan.counts))
    if most > capacity:
        raise ValueError(f"a branch would hold {most} keys, over the capacity of {capacity}")
    scale = _check_scale(scale, hd)
    if out is None:
        out = q.new_empty(t, hq * hd)
        if t > total:
            out[total:].zero_()
    if total == 0:
        return out
    seq_len = kv.seq_len
    table = mapped = 0
    if seq_len:
        table, mapped = device_tables_of(kv, q.device)[0].data_ptr(), len(kv.block_table)
    nbytes = _capi.workspace_bytes("branch_workspace", total, num_units, count, seq_len, longest,
                                   hq, kvh, hd)
    ws = q.new_empty(nbytes // 2) if nbytes else None
    size = kc.element_size()
    at, bat = size * cst[0] * (layer % layers), size * bst[0] * (layer % bshape[0])
    _capi.launch("tm_branch_attention", index, q.data_ptr(), qs, k.data_ptr(),
                 ks[0] if t > 1 else kvh * hd, v.data_ptr(), vs[0] if t > 1 else kvh * hd, total,
                 kc.data_ptr() + at, vc.data_ptr() + at, cst[1], cst[2], page, pages, table,
                 mapped, seq_len, bk.data_ptr() + bat, bv.data_ptr() + bat, bst[1], bst[2], rows,
                 capacity, ptr(origin), 0 if origin is None else origin.stride(0),
                 lengths.data_ptr(), longest, units, num_units, tokens, count, hq, kvh, hd, scale,
                 dt, out.data_ptr(), ost, ptr(ws), nbytes)
    if plan is not None:
        _capi.used_by(index, plan.made_on, plan.lists)
    return out
