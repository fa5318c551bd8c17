"""A cache that stays bounded: the weight that every cached key gets from the queries,
and the eviction of the keys that get least.

The reference's cache (treemoe/model/kv_cache.py) only grows.  Here ``attention_mass``
sums, for every key, the attention weights of the tokens that see it, and ``evict`` cuts the
cache to the keys of the largest sums, beside the first and the most recent ones.
"""

from __future__ import annotations

import operator

import torch

from treemoe_spec_amd import _capi
from treemoe_spec_amd._capi import ptr
from treemoe_spec_amd.kernels.prompt_attention import _check_q, _check_scale
from treemoe_spec_amd.kv_cache import device_tables_of


def _cache_layout(kv, kc, vc):
    """(layers, pages, page, kv_heads, head_dim) and strides of a paged cache."""
    shape, st = kc.shape, kc.stride()
    if vc.dtype != kc.dtype or vc.shape != shape or vc.stride() != st or len(shape) != 5 \
            or st[4] != 1 or (st[3] != shape[4] and shape[3] > 1) or shape[2] != kv.block_size:
        raise ValueError("cache layout must be [L, pages, page, kv_heads, head_dim]")
    page = shape[2]
    if page & (page - 1):
        raise ValueError(f"page size must be a power of two, got {page}")
    return shape, st


def attention_mass(q: torch.Tensor, kv, layer: int, mass: torch.Tensor | None = None, *,
                   scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """q [T, Hq, hd] (bfloat16 or float16, head_dim 64 or 128, rotated): the last T of
    ``kv``'s ``seq_len`` positions, whose keys ``layer`` holds already.  Returns float32
    [kv_heads, seq_len]: for every key the softmax weights that it gets, summed over the
    tokens that see it and the query heads of its KV head, added to ``mass`` [kv_heads, >=
    seq_len] where given.  A row whose scores are all -inf gives nothing.  ``out``
    [kv_heads, >= seq_len] takes the first seq_len columns of the result; it may be
    ``mass``, or shares no memory with it.  A replay of a captured call repeats the length of
    the capture."""
    dt, t, hq, hd, qs, _ = _check_q(q, None)
    kc, vc = kv.k, kv.v
    index = q.get_device()
    if not _capi.ready(index, q, kc, mass, out):
        _capi.require("attention_mass", q.device, q=q, k_cache=kc, mass=mass, out=out)
    shape, cst = _cache_layout(kv, kc, vc)
    layers, pages, page, kvh, chd = shape
    if kc.dtype != q.dtype or chd != hd:
        raise ValueError("the cache must have q's dtype and head_dim")
    if kvh < 1 or hq % kvh:
        raise ValueError("num_heads must be a multiple of num_kv_heads")
    layer = operator.index(layer)
    if not -layers <= layer < layers:
        raise IndexError(f"layer {layer} is out of range for a cache of {layers} layers")
    n = kv.seq_len
    if t > n:
        raise ValueError(f"{t} queries over a cache of {n} positions")
    scale = _check_scale(scale, hd)
    if out is None:
        out = q.new_empty((kvh, n), dtype=torch.float32)
    for name, x in (("mass", mass), ("out", out)):
        if x is not None and (x.dtype != torch.float32 or x.dim() != 2 or x.shape[0] != kvh
                              or x.shape[1] < n or (x.stride(1) != 1 and x.shape[1] > 1)
                              or (kvh > 1 and x.stride(0) < n)):
            raise ValueError(f"{name} must be float32 [kv_heads, >= seq_len] with unit stride "
                             "along the keys")
    if mass is not None and mass.data_ptr() == out.data_ptr() and kvh > 1 \
            and mass.stride(0) != out.stride(0):
        raise ValueError("out must be mass, or lie apart from it")
    if n == 0:
        return out
    table, _ = device_tables_of(kv, q.device)
    nbytes = _capi.workspace_bytes("mass_workspace", t, n, hq, kvh, hd)
    ws = out.new_empty(nbytes // 4) if nbytes else None
    _capi.launch("tm_attention_mass", index, q.data_ptr(), qs, t,
                 kc.data_ptr() + kc.element_size() * cst[0] * (layer % layers), cst[1], cst[2],
                 page, pages, table.data_ptr(), len(kv.block_table), n, hq, kvh, hd, scale, dt,
                 ptr(mass), 0 if mass is None else mass.stride(0), out.data_ptr(), out.stride(0),
                 ptr(ws), nbytes)
    return out


def evict(kv, mass: torch.Tensor, keep: int, *, positions: torch.Tensor | None = None,
          next_position: int | None = None, recent: int = 0, sinks: int = 0):
    """Cuts the paged cache ``kv`` from ``seq_len`` to ``keep`` keys, in every layer's KV heads
    those with the largest ``mass`` (float32 [L, kv_heads, >= seq_len]; the lower slot first
    among equals, NaN last) beside the first ``sinks`` and the last ``recent`` positions,
    which stay in any case (sinks + recent <= keep).  Kept keys in slots from ``keep`` on
    move, with their values, into the slots that have become free below, in order;
    ``kv.seq_len`` becomes ``keep``, the pages stay mapped.  A cache of ``keep`` keys or
    fewer stays as it is.

    Returns (mass, positions): of what the slots then hold, the mass like ``mass``, 0 from
    ``keep`` on, and the positions int32 [L, kv_heads, keep].  Give both to the next call, with
    what ``attention_mass`` has added since: ``positions`` covers the first slots, those
    behind it are the last ones before ``next_position`` (default, without ``positions``:
    ``seq_len``).  ``next_position`` is also the position to rotate the next token by: tokens
    go on in slot ``kv.seq_len``, so rotate with ``rotary_embed`` and store with ``kv.append``.
    Every attention over the whole cache goes on as before, since it does not depend on
    the order of the slots.  A replay of a captured call repeats the lengths of the capture."""
    kc, vc = kv.k, kv.v
    index = kc.get_device()
    if not _capi.ready(index, kc, vc, mass, positions):
        _capi.require("evict", kc.device, k_cache=kc, v_cache=vc, mass=mass, positions=positions)
    shape, cst = _cache_layout(kv, kc, vc)
    layers, pages, page, kvh, hd = shape
    size, n = kc.element_size(), kv.seq_len
    if size not in (1, 2, 4) or hd * size % 16:
        raise ValueError("a key must be a multiple of 16 bytes, of elements of 1, 2 or 4")
    keep, recent, sinks = (operator.index(x) for x in (keep, recent, sinks))
    if keep < 0 or recent < 0 or sinks < 0 or recent + sinks > keep:
        raise ValueError(f"need 0 <= recent + sinks <= keep, got {recent}, {sinks} and {keep}")
    keep = min(keep, n)
    if mass.dtype != torch.float32 or mass.dim() != 3 or mass.shape[:2] != (layers, kvh) \
            or mass.shape[2] < n or (mass.shape[2] > 1 and mass.stride(2) != 1):
        raise ValueError("mass must be float32 [L, kv_heads, >= seq_len] with unit stride along "
                         "the keys")
    recorded = pl = ph = 0
    if positions is not None:
        if positions.dtype != torch.int32 or positions.dim() != 3 \
                or positions.shape[:2] != (layers, kvh) or positions.shape[2] > n \
                or (positions.shape[2] > 1 and positions.stride(2) != 1):
            raise ValueError("positions must be int32 [L, kv_heads, <= seq_len] with unit stride "
                             "along the keys")
        if next_position is None:
            raise ValueError("positions without next_position")
        recorded, pl, ph = positions.shape[2], positions.stride(0), positions.stride(1)
    next_position = n if next_position is None else operator.index(next_position)
    if not n <= next_position < 2 ** 31:
        raise ValueError(f"next_position must be seq_len .. 2^31 - 1, got {next_position}")
    columns = mass.shape[2]
    new_mass = mass.new_empty(layers, kvh, columns)
    new_positions = mass.new_empty((layers, kvh, keep), dtype=torch.int32)
    if columns == 0:
        return new_mass, new_positions
    table, _ = device_tables_of(kv, kc.device)
    nbytes = _capi.workspace_bytes("evict_workspace", layers, kvh, n, keep)
    ws = mass.new_empty(nbytes // 4)
    _capi.launch("tm_evict", index, kc.data_ptr(), vc.data_ptr(), size, layers, cst[0], cst[1],
                 cst[2], kvh, hd, page, pages, table.data_ptr(), len(kv.block_table), n, keep,
                 mass.data_ptr(), mass.stride(0), mass.stride(1), columns,
                 ptr(positions) if recorded else 0, pl, ph, recorded, next_position, recent, sinks,
                 new_mass.data_ptr(), new_positions.data_ptr(), ws.data_ptr(), nbytes)
    kv.seq_len = keep
    return new_mass, new_positions
