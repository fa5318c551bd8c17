"""CPU: calls of the branch, beam and eviction operators at the edges of what they take."""

from __future__ import annotations

import pytest
import torch

from treemoe_spec_amd import _capi
from treemoe_spec_amd.kernels import beam_search as bs
from treemoe_spec_amd.kernels import branch_attention as ba
from treemoe_spec_amd.kv_cache import BranchCache
from tests.test_branch_args import CFG, _branch_args, calls  # noqa: F401  (a fixture)


@pytest.mark.parametrize("heads", [128, 144, 256, 1024])
def test_plan_of_more_heads_than_a_tile_has_rows(heads):
    """A token of a plan may take several tiles.  (The address of k, checked behind the sizes,
    ends the call before a launch.)"""
    plan = ba.BranchPlan([1, 2, 0], num_heads=heads, num_kv_heads=1, device="cpu")
    assert plan.num_units == -(-heads // 128) + -(-2 * heads // 128)
    args = dict(q_stride=64 * heads, out_stride=64 * heads, k=8, T=3, rows=3, units=16, tokens=16,
                num_units=plan.num_units, max_count=2, Hq=heads, kvh=1)
    lib = _capi.lib()
    assert lib.tm_branch_attention(*_branch_args(**args)) == 1002
    most = 3 * -(-heads // 128)
    assert lib.tm_branch_attention(*_branch_args(**args | dict(num_units=most))) == 1002
    assert lib.tm_branch_attention(*_branch_args(**args | dict(num_units=most + 1))) == 1001


def test_reorder_of_views_that_torch_has_not_computed(calls):  # noqa: F811
    """Bytes are moved, so a conjugation or negation put off by torch is refused, not lost."""
    x = torch.zeros(6, 4, dtype=torch.complex64)
    parents = torch.zeros(2, 3, dtype=torch.int32)
    for bad in (x.conj(), torch._neg_view(torch.zeros(6, 4))):
        with pytest.raises(ValueError, match="materialised"):
            bs.reorder_rows(bad, parents)
        with pytest.raises(ValueError, match="materialised"):
            bs.reorder_rows(torch.zeros(6, 4, dtype=bad.dtype), parents, out=bad)
    assert not calls
    bs.reorder_rows(x, parents)
    assert calls[0][0] == "tm_reorder_rows"


def test_lengths_are_whole_numbers(calls):  # noqa: F811
    br = BranchCache(CFG, 2, 10, device="cpu")
    br.advance(5)
    for bad in ([1.9, 2], [2, "3"], torch.tensor([1.0, 2.0])):
        with pytest.raises(TypeError):
            br.set_lengths(bad)
    assert br.host_lengths == [5, 5]
    br.set_lengths(torch.tensor([3, 0]))
    assert br.host_lengths == [3, 0] and br.longest == 3 and br.lengths.tolist() == [3, 0]
