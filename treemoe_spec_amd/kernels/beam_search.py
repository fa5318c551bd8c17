"""Beam search's step: the selection over beams and vocabulary, and the reordering of
what the beams hold.

The reference decodes one continuation, greedy or sampled; beams go through a forward
together by ``branch_attention``, and ``beam_select`` picks their candidates from its
logits in two launches.  What goes with a beam (its tokens, its table of origins in a
``BranchCache``, states of its own) follows by ``reorder_rows``.
"""

from __future__ import annotations

import operator

import torch

from treemoe_spec_amd import _capi
from treemoe_spec_amd._capi import dtype_code, ptr


def beam_select(logits: torch.Tensor, scores: torch.Tensor, *, num: int | None = None,
                finished: torch.Tensor | None = None, pad_token: int = 0):
    """The ``num`` best continuations (default: as many as beams) of each group of beams.

    ``logits`` [G * K, V] (float32, bfloat16 or float16, rows at any stride), the rows of
    a group's K beams one after the other; ``scores`` [G, K] float32, the beams' summed
    log-probabilities.  A beam's candidates are every token with ``scores + log
    softmax(logits)``, formed in 64 bits (exponentials good to 2e-13); one that has
    ``finished`` [G, K] (bool) has a single candidate, ``pad_token`` with its score
    unchanged.  Returns (scores float32, parents int32, tokens int64), each [G, num], the
    larger score first, of equal ones the lower beam, then the larger logit, then the lower
    token; parents are beams within the group.

    NaN logits count as -inf; a score of -inf or NaN, or a row with no logit above -inf,
    gives no candidates; where fewer than ``num`` are left, the rest are -inf, -1 and -1.
    K and num are at most 64.  At the first step, where all beams are alike, give all but
    the first a score of -inf."""
    shape = logits.shape
    if len(shape) != 2 or scores.dim() != 2:
        raise ValueError("logits must be [G * K, V] and scores [G, K]")
    groups, beams = scores.shape
    rows, v = shape
    dt = dtype_code(logits.dtype)
    if dt is None:
        raise ValueError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if rows != groups * beams:
        raise ValueError(f"{rows} rows of logits for {groups} groups of {beams} beams")
    num = beams if num is None else operator.index(num)
    if not (1 <= beams <= _capi.TM_MAX_BEAMS and 1 <= num <= _capi.TM_MAX_BEAMS):
        raise ValueError(f"beams and num must be 1..{_capi.TM_MAX_BEAMS}, got {beams} and {num}")
    if not 1 <= v <= _capi.TM_MAX_SAMPLE_VOCAB:
        raise ValueError(f"V must be 1..{_capi.TM_MAX_SAMPLE_VOCAB}, got {v}")
    if rows > _capi.TM_MAX_ROWS:
        raise ValueError(f"G * K must be at most {_capi.TM_MAX_ROWS}, got {rows}")
    pad_token = operator.index(pad_token)
    if not 0 <= pad_token < v:
        raise ValueError(f"pad_token must be a token, 0..{v - 1}")
    if scores.dtype != torch.float32 or not scores.is_contiguous():
        raise ValueError("scores must be contiguous float32 [G, K]")
    if finished is not None and (finished.shape != scores.shape or finished.dtype != torch.bool
                                 or not finished.is_contiguous()):
        raise ValueError("finished must be contiguous bool [G, K]")
    stride, step = logits.stride()
    if step != 1 and v > 1:
        raise ValueError("logits must have unit stride along V")
    index = logits.get_device()
    if not _capi.ready(index, logits, scores, finished):
        _capi.require("beam_select", logits.device, logits=logits, scores=scores,
                      finished=finished)
    best = scores.new_empty(groups, num)
    parents = scores.new_empty((groups, num), dtype=torch.int32)
    tokens = scores.new_empty((groups, num), dtype=torch.int64)
    nbytes = _capi.workspace_bytes("beam_workspace", groups, beams, v, num)
    ws = scores.new_empty(nbytes // 4)
    _capi.launch("tm_beam_select", index, logits.data_ptr(), dt, groups, beams, v,
                 stride if rows > 1 else v, scores.data_ptr(), ptr(finished), pad_token, num,
                 best.data_ptr(), parents.data_ptr(), tokens.data_ptr(), ws.data_ptr(), nbytes)
    return best, parents, tokens


def reorder_rows(x: torch.Tensor, parents: torch.Tensor, *, out: torch.Tensor | None = None,
                 columns: int | None = None) -> torch.Tensor:
    """Row g * K + i of the result is row g * K + parents[g, i] of ``x`` [G * K, ...] (any
    type, each row contiguous); ``parents`` int32 [G, K], the first K columns of
    ``beam_select``'s for example.  A parent outside 0..K-1 stands for the beam itself.
    ``out`` may be ``x``, or shares no memory with it; ``columns`` (with ``out``): only
    so many leading elements of each row, the others of ``out`` stay as they were."""
    if parents.dim() != 2 or parents.dtype != torch.int32:
        raise ValueError("parents must be int32 [G, K]")
    groups, beams = parents.shape
    if not 1 <= beams <= _capi.TM_MAX_BEAMS or groups > 65535:
        raise ValueError(f"parents must be [G, K] with K 1..{_capi.TM_MAX_BEAMS} and G up to "
                         f"65535, got {groups} and {beams}")
    pstride = parents.stride(0)
    if (beams > 1 and parents.stride(1) != 1) or (groups > 1 and pstride < beams):
        raise ValueError("parents must have unit stride along K and rows of their own")
    if x.dim() < 1 or x.shape[0] != groups * beams:
        raise ValueError(f"x must have a row for each of {groups * beams} beams")
    rows = x.shape[0]
    index = x.get_device()
    if not _capi.ready(index, x, parents, out):
        _capi.require("reorder_rows", x.device, x=x, parents=parents, out=out)
    if out is None:
        if columns is not None:
            raise ValueError("columns without out")
        out = x.new_empty(*x.shape)
    elif out.shape != x.shape or out.dtype != x.dtype:
        raise ValueError("out must have x's shape and type")
    size, width = x.element_size(), 1
    for d in range(x.dim() - 1, 0, -1):   # rows contiguous in both
        n = x.shape[d]
        if n > 1 and (x.stride(d) != width or out.stride(d) != width):
            raise ValueError("each row of x and out must be contiguous")
        width *= n
    # (bytes move: a conjugation or negation that torch has put off would be lost)
    if x.is_conj() or x.is_neg() or out.is_conj() or out.is_neg():
        raise ValueError("x and out must be materialised: no pending conjugation or negation")
    if rows == 0 or width == 0:
        return out
    xs, outs = (x.stride(0), out.stride(0)) if rows > 1 else (width, width)
    if xs < width or outs < width:
        raise ValueError("the rows of x and out must lie apart")
    if out.data_ptr() == x.data_ptr() and xs != outs:
        raise ValueError("out must be x, or lie apart from it")
    if columns is not None:
        columns = operator.index(columns)
        if not 0 <= columns <= width:
            raise ValueError(f"columns must be 0..{width}, got {columns}")
        width = columns
        if width == 0:
            return out
    _capi.launch("tm_reorder_rows", index, x.data_ptr(), xs * size, out.data_ptr(), outs * size,
                 width * size, parents.data_ptr(), pstride, groups, beams)
    return out
