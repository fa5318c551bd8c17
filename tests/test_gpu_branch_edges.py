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


@pytest.mark.parametrize("hq", [144, 1024])
@pytest.mark.parametrize("t,past", [(1, 0), (2, 65), (5, 700)])
def test_mass_of_more_heads_than_a_tile_has_rows(t, past, hq):
    _say(f"mass of {hq} heads over one, {t} tokens behind {past}")
    t_evict._mass(t, t + past, hq, 1, 64, BF, 16, t, add=past > 0)


def test_mass_of_rows_beyond_a_few_stages():
    """The bound of the sum over a key's rows, all positive, from the rows: an accumulator takes 8
    of each 64, each addition half a step of what is there; then 3 joins of accumulators and
    lanes, up to 8 parts of the rows, and `before`.  The other shares are
    test_gpu_cache_eviction's: 600 u for the sum over the keys has, a lane and stage of 64 keys
    one addition, one product and a factor of two roundings where the maximum grew, 4 * 128, and
    11 within a stage, 35 ranges joined."""
    from treemoe_spec_amd.kernels.cache_eviction import attention_mass

    t, hq, kvh, hd = 4096, 16, 8, 64
    _say(f"mass of {t} tokens over themselves")
    q, k, v = t_attn._qkv(t, t, hq, kvh, hd, BF, 31, 2.0)
    kv = t_attn._cache(t, kvh, hd, BF, 64, 31)
    kv.append(1, k.cuda(), v.cuda(), 0)
    got = attention_mass(q.cuda(), kv, 1).double().cpu()
    want = t_evict._want(q, k, hd ** -0.5)
    ds = 130 * U * hd ** -0.5 * float(q.abs().max()) * float(k.abs().max()) * hd
    terms = 8 * (t * hq // kvh // 64) + 3 + 8 + 1
    off = (got - want).abs()
    assert bool((off <= (2 * ds + (8 + 64 + 600 + terms) * U) * want + 2.0 ** -90).all())


@pytest.mark.parametrize("hd,page", [(16, 16), (64, 1), (80, 64), (128, 16)])
@pytest.mark.parametrize("n,keep", [(100, 60), (1100, 1030), (2500, 300)])
def test_evict_of_one_byte_elements(n, keep, hd, page):
    _say(f"evict {n} -> {keep} of one byte, hd={hd}")
    g = torch.Generator().manual_seed(n + hd)
    kv = t_evict._cache_of(2, n, 3, hd, torch.int8, page, g)
    for x in (kv.k, kv.v):
        x.copy_(torch.randint(-128, 128, x.shape, generator=g, dtype=torch.int8))
    mass = torch.exp(2 * torch.randn(2, 3, n, generator=g))
    t_evict._check_evict(kv, mass, keep, recent=16, sinks=4)


def test_evict_of_float8():
    """The bytes of 8-bit floats move as they are, NaN among them."""
    from treemoe_spec_amd.kernels.cache_eviction import evict
    from treemoe_spec_amd.kv_cache import MixtralConfig, PagedKVCache

    _say("evict float8")
    g = torch.Generator().manual_seed(32)
    kv = PagedKVCache(MixtralConfig(num_layers=2, num_kv_heads=2, head_dim=64), 10,
                      dtype=torch.float8_e4m3fn, page_size=16, tree_size=1)
    same = PagedKVCache(kv.config, 10, dtype=torch.int8, page_size=16, tree_size=1)
    for x, y in ((kv.k, same.k), (kv.v, same.v)):
        y.copy_(torch.randint(-128, 128, y.shape, generator=g, dtype=torch.int8))
        x.view(torch.int8).copy_(y)
    mass = torch.rand(2, 2, 130, generator=g).cuda()
    got = []
    for c in (kv, same):
        c._ensure_capacity(130)
        c.seq_len = 130
        got.append(evict(c, mass, 70, recent=8))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert torch.equal(kv.k.view(torch.int8), same.k) and torch.equal(kv.v.view(torch.int8), same.v)
