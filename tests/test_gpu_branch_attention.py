"""branch_attention on the GPU against attention in 64 bits, branch by branch (tolerances:
test_gpu_prompt_attention), and what it leaves in the branch cache.

Every place that no branch holds is NaN: pages behind the sequence, places behind a
branch's length, rows behind the plan's tokens."""

from __future__ import annotations

import pytest
import torch

from tests import test_gpu_prompt_attention as t_attn

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16
NAN = float("nan")


def _say(msg):
    print(msg, flush=True)


class Setup:
    """A sequence of `prefix` positions in pages of `page`, and branches that hold
    `lengths` keys; beams > 1: keys lie in any row of a group."""

    def __init__(self, prefix, lengths, hq, kvh, hd, dtype, page=16, beams=1, seed=0, layers=2,
                 capacity=None, spare=20):
        from treemoe_spec_amd.kv_cache import BranchCache, MixtralConfig

        g = torch.Generator().manual_seed(seed)
        self.g, self.hq, self.kvh, self.hd, self.dtype = g, hq, kvh, hd, dtype
        self.kv = t_attn._cache(prefix, kvh, hd, dtype, page, seed, layers)
        for layer in range(layers if prefix else 0):
            k, v = (torch.randn(prefix, kvh, hd, generator=g).to(dtype) for _ in range(2))
            self.kv.append(layer, k.cuda(), v.cuda(), 0)
        cfg = MixtralConfig(num_layers=layers, num_kv_heads=kvh, head_dim=hd)
        rows = len(lengths)
        cap = capacity or max(lengths) + spare
        self.br = BranchCache(cfg, rows, cap, dtype=dtype, beams=beams)
        k, v = (torch.full((layers, rows, cap, kvh, hd), NAN, dtype=dtype) for _ in range(2))
        self.origin = torch.arange(rows)[:, None].repeat(1, cap)
        for b, n in enumerate(lengths):
            if beams > 1:
                pick = torch.randint(0, beams, (n,), generator=g)
                self.origin[b, :n] = b // beams * beams + pick
            k[:, b, :n] = torch.randn(layers, n, kvh, hd, generator=g).to(dtype)
            v[:, b, :n] = torch.randn(layers, n, kvh, hd, generator=g).to(dtype)
        self.br.k.copy_(k)
        self.br.v.copy_(v)
        if beams > 1:
            self.br.origin.copy_(self.origin)
        self.br.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        self.br.host_lengths, self.br.longest = list(lengths), max(lengths)
        self.k, self.v, self.lengths = k, v, list(lengths)

    def new(self, total, pad=0, scale=2.0):
        q = (torch.randn(total, self.hq, self.hd, generator=self.g) * scale).to(self.dtype)
        k, v = (torch.randn(total, self.kvh, self.hd, generator=self.g).to(self.dtype)
                for _ in range(2))
        if pad:
            q, k, v = (torch.cat([x, torch.full((pad, *x.shape[1:]), NAN, dtype=self.dtype)])
                       for x in (q, k, v))
        return q, k, v

    def check(self, out, q, k, v, layer, counts, scale=None):
        """The context of every branch, and the caches after the call."""
        shared = [x.cpu() for x in self.kv.gather(layer)] if self.kv.seq_len else None
        first = 0
        for b, n in enumerate(counts):
            m = self.lengths[b]
            if n:
                rows = self.origin[b, :m]
                held = [x[layer, rows, torch.arange(m)] for x in (self.k, self.v)]
                keys, values = (torch.cat(([] if shared is None else [shared[i]])
                                          + [held[i], (k, v)[i][first:first + n]])
                                for i in (0, 1))
                t_attn._check(out[first:first + n], q[first:first + n], keys, values,
                              self.kv.seq_len + m, scale)
            self.k[layer, b, m:m + n] = k[first:first + n]
            self.v[layer, b, m:m + n] = v[first:first + n]
            first += n
        for got, want in ((self.br.k, self.k), (self.br.v, self.v)):
            assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))


def _run(s, counts, layer=1, pad=0, scale=None, plan=None, **kw):
    from treemoe_spec_amd.kernels.branch_attention import BranchPlan, branch_attention

    q, k, v = s.new(sum(counts), pad, kw.pop("q_scale", 2.0))
    if plan is None and (len(set(counts)) > 1 or pad):
        plan = BranchPlan(counts, num_heads=s.hq, num_kv_heads=s.kvh)
    out = branch_attention(q.cuda(), k.cuda(), v.cuda(), s.kv, s.br, layer, plan, scale=scale, **kw)
    torch.cuda.synchronize()
    s.check(out.cpu(), q, k, v, layer, counts, scale)
    return out


HEADS = [(32, 8, 128), (8, 2, 64), (4, 4, 128), (3, 1, 64), (16, 2, 128), (7, 1, 128),
         (64, 1, 64)]


@pytest.mark.parametrize("hq,kvh,hd", HEADS)
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("prefix,page", [(0, 16), (1, 16), (65, 64), (517, 16)])
def test_one_token_each(prefix, page, hq, kvh, hd, dtype):
    _say(f"branches: one token each, prefix {prefix} heads={hq}/{kvh} hd={hd} {dtype}")
    s = Setup(prefix, [0, 1, 63, 64, 65, 200, 7], hq, kvh, hd, dtype, page, seed=prefix + hd)
    _run(s, [1] * 7)


@pytest.mark.parametrize("branches", [1, 2, 8, 9, 33, 70])
@pytest.mark.parametrize("prefix", [0, 300, 4100])
@pytest.mark.parametrize("hq,kvh,hd", [(32, 8, 128), (4, 4, 64)])
def test_batches(branches, prefix, hq, kvh, hd):
    _say(f"branches: {branches} over {prefix} heads={hq}/{kvh} hd={hd}")
    s = Setup(prefix, [(i * 37) % 150 for i in range(branches)], hq, kvh, hd, BF, 64,
              seed=branches)
    _run(s, [1] * branches)


@pytest.mark.parametrize("count", [2, 5, 8, 9, 33, 150])
@pytest.mark.parametrize("prefix", [0, 130])
@pytest.mark.parametrize("hq,kvh,hd,dtype", [(8, 2, 128, BF), (16, 4, 64, F16)])
def test_several_tokens_each(count, prefix, hq, kvh, hd, dtype):
    _say(f"branches: {count} tokens each over {prefix} heads={hq}/{kvh} hd={hd} {dtype}")
    _run(Setup(prefix, [0, 70, 3], hq, kvh, hd, dtype, seed=count, spare=160), [count] * 3)


@pytest.mark.parametrize("counts", [[3, 0, 1], [0, 0, 9, 0, 2], [1, 200, 0, 33, 8], [0, 1]])
@pytest.mark.parametrize("prefix,page", [(0, 16), (700, 16), (64, 64)])
@pytest.mark.parametrize("pad", [0, 5])
def test_ragged(counts, prefix, page, pad):
    _say(f"branches: ragged {counts} over {prefix} pad {pad}")
    s = Setup(prefix, [(11 * i) % 40 for i in range(len(counts))], 8, 2, 128, BF, page,
              seed=prefix, capacity=260)
    out = _run(s, counts, pad=pad)
    if pad:
        assert not bool(out[sum(counts):].any())


@pytest.mark.parametrize("prefix,page", [(0, 16), (63, 16), (64, 16), (65, 1), (300, 64),
                                         (1000, 16), (2500, 64)])
@pytest.mark.parametrize("counts", [[64], [32, 96, 31], [30, 0, 62, 128], [200, 150]])
@pytest.mark.parametrize("hq,kvh,hd,dtype", [(8, 2, 128, BF), (32, 8, 64, F16)])
def test_branches_that_fill_tiles(counts, prefix, page, hq, kvh, hd, dtype):
    """Shared and own keys as one sequence, in one range or several."""
    _say(f"branches: {counts} that fill tiles over {prefix} page {page} {hq}/{kvh} hd={hd}")
    s = Setup(prefix, [(37 * i) % 150 for i in range(len(counts))], hq, kvh, hd, dtype, page,
              seed=prefix + 1, capacity=400)
    _run(s, counts)


@pytest.mark.parametrize("counts,prefix,hq,kvh,hd,dtype", [
    ([33] * 24, 1700, 16, 16, 64, F16),
    ([9] * 30, 3900, 16, 4, 128, BF),
    ([9, 0, 8, 1, 12, 10] * 7, 3333, 16, 4, 64, BF),
])
def test_branches_that_leave_tiles_empty(counts, prefix, hq, kvh, hd, dtype):
    """Many rows short of whole tiles behind many shared keys: those once for all branches."""
    _say(f"branches: {len(counts)} short of tiles over {prefix} heads={hq}/{kvh} hd={hd} {dtype}")
    s = Setup(prefix, [(i * 29) % 200 for i in range(len(counts))], hq, kvh, hd, dtype, 64,
              seed=prefix, layers=2, spare=40)
    _run(s, counts)


@pytest.mark.parametrize("counts,prefix,hq,kvh,hd,dtype", [
    ([230] * 8 + [225, 0, 1], 600, 32, 8, 64, F16),
    ([240] * 22, 150, 12, 3, 128, BF),
])
def test_tiles_of_more_than_a_round(counts, prefix, hq, kvh, hd, dtype):
    """The first tiles whole, those of the last round in ranges, joined."""
    _say(f"branches: {len(counts)} of {counts[0]} over {prefix} heads={hq}/{kvh} hd={hd} {dtype}")
    s = Setup(prefix, [(i * 53) % 170 for i in range(len(counts))], hq, kvh, hd, dtype, 16,
              seed=prefix, layers=2, capacity=420)
    _run(s, counts)


@pytest.mark.parametrize("beams,groups", [(2, 3), (4, 1), (5, 2), (8, 9)])
@pytest.mark.parametrize("count", [1, 3, 20, 32])
@pytest.mark.parametrize("hd", [64, 128])
def test_beams_share_rows(beams, groups, count, hd):
    _say(f"branches: {groups} x {beams} beams, {count} tokens, hd={hd}")
    lengths = [n for g in range(groups) for n in [(29 * g) % 190 + 1] * beams]
    s = Setup(133, lengths, 8, 2, hd, BF, beams=beams, seed=beams, spare=40)
    _run(s, [count] * (beams * groups))


def test_many_rows():
    """Prompts behind a shared one: the tall and the paired tiles of the shared keys."""
    _say("branches: many rows")
    _run(Setup(2100, [0] * 9, 32, 8, 128, BF, 64, seed=1, capacity=420),
         [400, 1, 333, 57, 0, 290, 128, 77, 31])
    _run(Setup(700, [5, 0, 0], 8, 2, 64, F16, 16, seed=2, capacity=700), [600, 333, 650])


def test_long_own_keys():
    """Own keys over several ranges."""
    _say("branches: long own keys")
    _run(Setup(40, [3000, 1, 2049], 8, 2, 128, BF, seed=3, spare=5), [1, 1, 1])
    _run(Setup(40, [20000, 9000], 8, 2, 128, BF, seed=3, spare=5), [1, 1])
    _run(Setup(0, [9000], 8, 2, 64, F16, seed=3, spare=5), [3])
    _run(Setup(0, [3000, 700], 8, 2, 128, BF, seed=4, spare=60), [50, 50])


def test_longest_may_be_too_small():
    """The split goes by the host's lengths, the keys by the device's: a replay's may have
    grown."""
    _say("branches: device lengths beyond the host's")
    for host in (0, 3):
        for counts in ([1, 1, 1], [40, 64, 1]):
            s = Setup(100, [900, 3, 333], 8, 2, 128, BF, seed=host, spare=70)
            s.br.longest = host
            s.br.host_lengths = [host] * 3
            _run(s, counts)


def test_strides_scale_and_out():
    from treemoe_spec_amd.kernels.branch_attention import branch_attention

    _say("branches: views of one projection, scale, out")
    s = Setup(77, [5, 0, 61], 8, 2, 128, BF, seed=6)
    qkv = torch.randn(6, 12 * 128 + 64, generator=s.g).to(BF)
    q, k, v = qkv[:, :12 * 128].view(6, 12, 128).split([8, 2, 2], 1)
    dev = qkv.cuda()
    dq, dk, dv = dev[:, :12 * 128].view(6, 12, 128).split([8, 2, 2], 1)
    big = torch.full((6, 8 * 128 + 16), 7.0, dtype=BF, device="cuda")
    out = big[:, :8 * 128]
    got = branch_attention(dq, dk, dv, s.kv, s.br, -1, scale=0.3, out=out)
    torch.cuda.synchronize()
    assert got is out and bool((big[:, 8 * 128:] == 7.0).all())
    s.check(out.cpu(), q, k, v, 1, [2, 2, 2], 0.3)


def test_rows_behind_the_plan_stay():
    from treemoe_spec_amd.kernels.branch_attention import BranchPlan, branch_attention

    _say("branches: out's rows behind the plan's")
    s = Setup(30, [4, 4], 8, 2, 64, BF, seed=8)
    q, k, v = s.new(5, 3)
    out = torch.full((8, 512), 3.0, dtype=BF, device="cuda")
    plan = BranchPlan([4, 1], num_heads=8, num_kv_heads=2)
    branch_attention(q.cuda(), k.cuda(), v.cuda(), s.kv, s.br, 1, plan, out=out)
    torch.cuda.synchronize()
    assert bool((out[5:] == 3.0).all())
    s.check(out.cpu(), q, k, v, 1, [4, 1])
    none = BranchPlan([0, 0], num_heads=8, num_kv_heads=2)
    out.fill_(5.0)
    branch_attention(q.cuda(), k.cuda(), v.cuda(), s.kv, s.br, 1, none, out=out)
    assert bool((out == 5.0).all())


@pytest.mark.parametrize("where", ["shared", "own", "new"])
@pytest.mark.parametrize("n", [3, 64])
def test_not_finite(where, n):
    """Infinities in a value that is seen reach the output of those that see it, alone."""
    from treemoe_spec_amd.kernels.branch_attention import branch_attention

    _say(f"branches: not finite, {where}, {n} tokens each")
    s = Setup(90, [20, 70], 8, 2, 128, BF, seed=9, spare=70)
    q, k, v = s.new(2 * n, scale=1.0)
    if where == "shared":
        page, off = s.kv.slot_of(80)
        s.kv.v[1, page, off, 1, 5] = float("inf")
    elif where == "own":
        s.br.v[1, 1, 69, 1, 5] = float("inf")
    else:
        v[n + 1, 1, 5] = float("inf")      # the second branch's second token
    out = branch_attention(q.cuda(), k.cuda(), v.cuda(), s.kv, s.br, 1)
    torch.cuda.synchronize()
    hit = torch.zeros(2 * n, 8, 128, dtype=torch.bool)
    hit[{"shared": 0, "own": n, "new": n + 1}[where]:, 4:, 5] = True
    assert bool((out.view(2 * n, 8, 128).cpu().isinf() == hit).all())
    assert bool(out.view(2 * n, 8, 128).cpu()[~hit].isfinite().all())


def test_hidden_scores():
    """Keys whose scores are all -inf (an infinite key against the query's sign) give 0."""
    from treemoe_spec_amd.kernels.branch_attention import branch_attention

    _say("branches: scores of -inf")
    s = Setup(0, [3], 4, 1, 64, BF, seed=10)
    q, k, v = s.new(1)
    q.fill_(1.0)
    for x in (s.br.k[:, :, :3], k):
        x.fill_(0.0)
        x[..., 0] = float("-inf")
    out = branch_attention(q.cuda(), k.cuda(), v.cuda(), s.kv, s.br, 1)
    assert not bool(out.any())


def test_advance_reorder_and_cut():
    """A few steps of one group of beams against a plain list of keys a beam."""
    from treemoe_spec_amd.kernels.branch_attention import BranchPlan, branch_attention

    _say("branches: steps, reordered")
    s = Setup(50, [0] * 6, 8, 2, 128, BF, beams=3, seed=11, capacity=40)
    held = [[] for _ in range(6)]
    shared = [x.cpu() for x in s.kv.gather(1)]
    for step in range(9):
        n = 1 + step % 3
        q, k, v = s.new(6 * n)
        plan = BranchPlan([n] * 6, num_heads=8, num_kv_heads=2) if step % 2 else None
        out = branch_attention(q.cuda(), k.cuda(), v.cuda(), s.kv, s.br, 1, plan)
        for b in range(6):
            rows = slice(b * n, b * n + n)
            keys = torch.cat([shared[0]] + [x for x, _ in held[b]] + [k[rows]])
            values = torch.cat([shared[1]] + [x for _, x in held[b]] + [v[rows]])
            t_attn._check(out[rows].cpu(), q[rows], keys, values, keys.shape[0] - n)
            held[b] = held[b] + [(k[i:i + 1], v[i:i + 1]) for i in range(b * n, b * n + n)]
        s.br.advance(plan if plan is not None else n)
        parents = torch.randint(0, 3, (2, 3), generator=s.g, dtype=torch.int32)
        if step == 4:
            parents[0, 1] = -1     # stays
        s.br.reorder(parents.cuda())
        held = [list(held[b // 3 * 3 + (int(parents[b // 3, b % 3]) if int(parents[b // 3, b % 3])
                                        >= 0 else b % 3)]) for b in range(6)]
        if step == 6:
            s.br.set_lengths([7] * 3 + [9] * 3)
            held = [h[:7 if b < 3 else 9] for b, h in enumerate(held)]
    assert s.br.host_lengths == [len(h) for h in held]
    assert s.br.lengths.tolist() == s.br.host_lengths
    s.br.read_lengths()
    assert s.br.longest == max(len(h) for h in held)
    s.br.reset()
    assert s.br.lengths.tolist() == [0] * 6 and s.br.longest == 0


def test_repeated_calls_are_equal():
    _say("branches: the same bits again")
    from treemoe_spec_amd.kernels.branch_attention import branch_attention

    s = Setup(1500, [(i * 53) % 400 for i in range(20)], 32, 8, 128, BF, seed=12)
    q, k, v = (x.cuda() for x in s.new(20))
    first = branch_attention(q, k, v, s.kv, s.br, 0)
    for _ in range(5):
        assert torch.equal(first, branch_attention(q, k, v, s.kv, s.br, 0))
