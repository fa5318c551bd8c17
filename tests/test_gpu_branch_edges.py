"""Branch attention and attention mass at the edges of their value ranges and head shapes.
Tolerances: test_gpu_prompt_attention and test_gpu_cache_eviction."""

from __future__ import annotations

import pytest
import torch

from tests import test_gpu_branch_attention as t_branch
from tests import test_gpu_cache_eviction as t_evict
from tests import test_gpu_prompt_attention as t_attn

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")
U = 2.0 ** -24


def _say(msg):
    print(msg, flush=True)


@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("t,past", [(2, 0), (2, 300), (8, 1), (10, 70), (16, 500), (17, 500)])
def test_mass_of_a_row_that_is_not_a_number(t, past, bad):
    """Of few rows and of more: it reaches the keys that it sees, of its KV head, and no others."""
    from treemoe_spec_amd.kernels.cache_eviction import attention_mass

    _say(f"mass with a query of {bad}, {t} tokens behind {past}")
    n, at = t + past, t // 2
    q, k, v = t_attn._qkv(t, n, 4, 2, 64, BF, t + past)
    k[:, 1, 7] = k[:, 1, 7].abs() + 0.5        # (an infinite query scores +infinity there)
    kv = t_attn._cache(n, 2, 64, BF, 16, t)
    kv.append(0, k.cuda(), v.cuda(), 0)
    q[at, 3, 7] = bad
    got = attention_mass(q.cuda(), kv, 0).cpu().double()
    assert bool(got[1, :past + at + 1].isnan().all())
    q[at, 3] = 0.0                             # (what it gives lies before the keys compared)
    want = t_evict._want(q, k, 64 ** -0.5)
    ds = 130 * U * 64 ** -0.5 * float(q.abs().max()) * float(k.abs().max()) * 64
    bound = (2 * ds + 736 * U) * want + 2.0 ** -90
    off = (got - want).abs()
    assert bool((off[0] <= bound[0]).all())
    assert bool((off[1, past + at + 1:] <= bound[1, past + at + 1:]).all())


@pytest.mark.parametrize("lengths,count,why", [
    ([3, 5], 1, "ranges by workgroups"), ([200] + [1] * 69, 1, "ranges by waves"),
    ([9, 4], 20, "tiles of 128 rows")])
def test_infinity_behind_a_weight_that_vanishes(lengths, count, why):
    """An infinite value whose weight is below what fp32 holds: its element is not finite, as in a
    sum of products, however the keys are split; the other elements are the value that
    has all the weight."""
    from treemoe_spec_amd.kernels.branch_attention import branch_attention

    _say(f"branches: infinity behind a vanishing weight, {why}")
    s = t_branch.Setup(300, lengths, 8, 2, 128, BF, seed=20)
    q, k, v = s.new(len(lengths) * count)
    q.fill_(4.0)
    k.fill_(4.0)                # 181 above all others: 2^-261 of the weight is left to them
    v[1:] = v[0]                # (also where a branch's new keys share it)
    s.kv.k.zero_()
    s.br.k[:, :, :max(lengths)] = 0.0
    page, off = s.kv.slot_of(290)
    s.kv.v[1, page, off, 1, 5] = INF
    out = branch_attention(q.cuda(), k.cuda(), v.cuda(), s.kv, s.br, 1).cpu()
    out = out.view(len(q), 2, 4, 128)
    hit = torch.zeros(out.shape, dtype=torch.bool)
    hit[:, 1, :, 5] = True
    assert not bool(out[hit].isfinite().any())
    # (equal keys' weights are rounded alike and summed as rounded: what is left are fp32 sums of 20
    # terms and the result's rounding, 2^-8)
    want = v.view(len(q), 2, 1, 128).expand(out.shape)
    assert bool(((out - want).abs()[~hit] <= 2.0 ** -7 * want.abs()[~hit]).all())


def test_ranges_without_keys_leave_nothing():
    """Workspace that held NaN before: ranges of short branches have no keys, and no part."""
    from treemoe_spec_amd import _capi
    from treemoe_spec_amd.kernels.branch_attention import branch_attention

    _say("branches: ranges without keys over old NaN")
    lengths = [600] + [i % 7 for i in range(69)]
    s = t_branch.Setup(200, lengths, 32, 8, 128, BF, seed=21)
    q, k, v = s.new(70)
    nbytes = _capi.workspace_bytes("branch_workspace", 70, 70, 1, 200, 600, 32, 8, 128)
    args = [x.cuda() for x in (q, k, v)]
    out = torch.empty(70, 32 * 128, dtype=BF, device="cuda")
    old = torch.full((nbytes // 2,), NAN, dtype=BF, device="cuda")
    where = old.data_ptr()
    del old                     # what the call's workspace is made of
    branch_attention(*args, s.kv, s.br, 1, out=out)
    assert torch.empty(nbytes // 2, dtype=BF, device="cuda").data_ptr() == where
    s.check(out.cpu(), q, k, v, 1, [1] * 70)


@pytest.mark.parametrize("hq,hd,dtype", [(144, 64, BF), (256, 128, F16)])
@pytest.mark.parametrize("counts,prefix", [([1, 1], 0), ([2, 0, 1], 70), ([1, 3, 1, 0], 1000),
                                           ([2, 2], 300)])
def test_more_heads_than_a_tile_has_rows(counts, prefix, hq, hd, dtype):
    """A token's heads fill several tiles, with a plan and without."""
    from treemoe_spec_amd.kernels.branch_attention import BranchPlan

    _say(f"branches: {hq} heads over one, {counts} behind {prefix}")
    s = t_branch.Setup(prefix, [(7 * i + 3) % 90 for i in range(len(counts))], hq, 1, hd, dtype,
                       seed=22)
    t_branch._run(s, counts, plan=BranchPlan(counts, num_heads=hq, num_kv_heads=1))
    if len(set(counts)) == 1:
        t_branch._run(s, counts, layer=0)
