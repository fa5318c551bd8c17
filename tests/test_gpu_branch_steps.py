"""Branch attention, beam search, attention mass and eviction together: a prompt, its cache
cut by the weights that its last tokens give, and a beam search behind it; the search's step
under graph capture; calls on two streams and from two threads; offsets past 32 bits.

The steps' numbers are held against 64-bit formulas of each operator's own inputs
(tolerances: those operators' tests); replays, streams and threads against the same
call's bits on one stream."""

from __future__ import annotations

import functools
import threading

import pytest
import torch

from tests import test_gpu_beam_search as t_beam
from tests import test_gpu_cache_eviction as t_evict
from tests import test_gpu_prompt_attention as t_attn

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
LAYERS, HQ, KVH, HD, VOCAB = 2, 8, 2, 64, 700


def _say(msg):
    print(msg, flush=True)


@functools.cache
def _streams():
    """Four at once: streams go over the card's four hardware queues in turn, one of which is the
    default stream's, so tests that come later get theirs as if these were not there."""
    return [torch.cuda.Stream() for _ in range(4)]


class Search:
    """Beams behind a prompt whose cache has been cut, through `LAYERS` layers of attention
    alone; `next` is the position of the next token."""

    def __init__(self, beams=3, groups=2, prompt=300, keep=96, seed=0, capacity=40):
        from treemoe_spec_amd.kernels.cache_eviction import attention_mass, evict
        from treemoe_spec_amd.kernels.prompt_attention import prompt_attention_cached
        from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_append
        from treemoe_spec_amd.kv_cache import BranchCache, MixtralConfig

        g = torch.Generator().manual_seed(seed)
        cfg = MixtralConfig(num_layers=LAYERS, num_kv_heads=KVH, head_dim=HD)
        self.rows, self.beams, self.groups = beams * groups, beams, groups
        self.plan = RotaryPlan(HD, 1e4)
        self.embed = torch.randn(VOCAB, 1, HQ + 2 * KVH, HD, generator=g).to(BF).cuda()
        self.head = (torch.randn(HQ * HD, VOCAB, generator=g) * 0.3).to(BF).cuda()
        self.kv = kv = t_attn._cache(prompt, KVH, HD, BF, 16, seed, LAYERS)
        tokens = torch.randint(0, VOCAB, (prompt,), generator=g)
        mass = torch.empty(LAYERS, KVH, prompt, device="cuda")
        for layer in range(LAYERS):
            q, k, v = self.qkv(tokens.cuda(), layer)
            # in two chunks; the last 32 tokens judge the keys
            for lo, hi in ((0, 200), (200, prompt)):
                qr = rotary_append(q[lo:hi], k[lo:hi], v[lo:hi], self.plan, kv, layer, lo)
                prompt_attention_cached(qr, kv, layer)
            attention_mass(qr[-32:], kv, layer, out=mass[layer])
            keys = kv.gather(layer)[0].cpu()
            t_evict._check(mass[layer], qr[-32:].cpu(), keys)
        self.mass, self.positions = evict(kv, mass, keep, recent=16, sinks=4)
        self.next = prompt
        assert kv.seq_len == keep and int(self.positions.max()) == prompt - 1
        self.br = BranchCache(cfg, self.rows, capacity, beams=beams)
        self.scores = torch.full((groups, beams), -float("inf"), device="cuda")
        self.scores[:, 0] = 0.0
        self.held = torch.zeros(self.rows, capacity, dtype=torch.int64, device="cuda")
        self.tokens = torch.randint(0, VOCAB, (groups, 1), generator=g).expand(groups, beams)
        self.tokens = self.tokens.contiguous().cuda()
        self.position = torch.full((self.rows,), self.next, dtype=torch.int32, device="cuda")
        self.logits = torch.empty(self.rows, VOCAB, dtype=BF, device="cuda")

    def qkv(self, tokens, layer):
        x = self.embed[(tokens + 31 * layer) % VOCAB][:, 0]
        return x.split([HQ, KVH, KVH], 1)

    def step(self, seen=None):
        """One token of every beam; `seen(layer, q, k, v, out)` and `seen(None, logits, scores,
        best)` are told what went in and came out."""
        from treemoe_spec_amd.kernels.beam_search import beam_select, reorder_rows
        from treemoe_spec_amd.kernels.branch_attention import branch_attention
        from treemoe_spec_amd.kernels.rotary import rotary_embed

        for layer in range(LAYERS):
            q, k, v = self.qkv(self.tokens.flatten(), layer)
            qr, kr = rotary_embed(q, k, self.position, self.plan)
            out = branch_attention(qr, kr, v, self.kv, self.br, layer)
            if seen:
                seen(layer, qr, kr, v, out)
        torch.mm(out, self.head, out=self.logits)
        best = beam_select(self.logits, self.scores, num=self.beams)
        if seen:
            seen(None, self.logits, self.scores, best)
        self.br.advance()
        scores, parents, tokens = best
        self.br.reorder(parents)
        reorder_rows(self.held, parents, out=self.held)
        self.held.copy_(torch.cat([tokens.flatten()[:, None], self.held[:, :-1]], 1))
        self.scores.copy_(scores)
        self.tokens.copy_(tokens)
        self.position.add_(1)
        return out

    def state(self):
        self.br.read_lengths()
        return [x.clone() for x in (self.br.k, self.br.v, self.br.lengths, self.br.origin,
                                    self.held, self.scores, self.tokens, self.position,
                                    self.logits)]


def test_search_behind_a_cut_cache():
    _say("prompt, mass, eviction, beam search")
    s = Search()
    held = [[[] for _ in range(s.rows)] for _ in range(LAYERS)]     # keys and values of a beam
    names = [[] for _ in range(s.rows)]                             # its tokens
    shared = [[x.cpu() for x in s.kv.gather(layer)] for layer in range(LAYERS)]
    moves = []

    def seen(layer, *what):
        if layer is None:
            logits, scores, best = what
            want = t_beam._want(logits.cpu(), scores.cpu(), s.beams)
            assert torch.equal(best[1].cpu(), want[1]) and torch.equal(best[2].cpu(), want[2])
            moves.append((best[1].cpu(), best[2].cpu()))
            return
        q, k, v, out = (x.cpu() for x in what)
        for b in range(s.rows):
            old = held[layer][b]
            keys, values = (torch.cat([shared[layer][i]] + [x[i] for x in old]
                                      + [(k, v)[i][b:b + 1]]) for i in (0, 1))
            t_attn._check(out[b:b + 1], q[b:b + 1], keys, values, keys.shape[0] - 1)
            held[layer][b] = old + [(k[b:b + 1], v[b:b + 1])]

    for _ in range(8):
        s.step(seen)
        parents, tokens = moves[-1]
        at = [b // s.beams * s.beams + int(parents.flatten()[b]) for b in range(s.rows)]
        held = [[list(layer[a]) for a in at] for layer in held]
        names = [[int(tokens.flatten()[b])] + names[a] for b, a in enumerate(at)]
    assert [row[:8].tolist() for row in s.held.cpu()] == names
    assert s.br.host_lengths == [8] * s.rows == s.br.lengths.tolist()


def test_captured_step():
    """A step captured once and replayed as the beams grow, with eager calls between."""
    _say("captured search step")
    eager, replayed = Search(seed=3), Search(seed=3)
    other = Search(seed=4)
    stream = _streams()[0]
    with torch.cuda.stream(stream):
        for s in (eager, replayed):
            s.step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        replayed.step()
    for _ in range(6):
        graph.replay()
        eager.step()
        other.step()
        torch.cuda.synchronize()
        for a, b in zip(eager.state(), replayed.state()):
            assert torch.equal(a, b)
    assert replayed.br.host_lengths == [7] * replayed.rows


def test_captured_selection_eviction_and_mass():
    """Graphs whose workspaces live side by side, each replayed several times on inputs that
    change."""
    from treemoe_spec_amd.kernels.beam_search import beam_select
    from treemoe_spec_amd.kernels.branch_attention import BranchPlan, branch_attention
    from treemoe_spec_amd.kernels.cache_eviction import attention_mass, evict
    from treemoe_spec_amd.kv_cache import BranchCache, MixtralConfig

    _say("captured calls of every operator")
    g = torch.Generator(device="cuda").manual_seed(5)
    cfg = MixtralConfig(num_layers=2, num_kv_heads=2, head_dim=128)
    kv = t_attn._cache(900, 2, 128, BF, 16, 5)
    for layer in range(2):
        kv.append(layer, *(torch.randn(900, 2, 128, generator=g, device="cuda").to(BF)
                           for _ in range(2)), 0)
    br = BranchCache(cfg, 4, 300, dtype=BF)
    br.k.normal_(generator=g)
    br.v.normal_(generator=g)
    br.set_lengths([0] * 4)
    br.lengths.copy_(torch.tensor([30, 200, 0, 77], dtype=torch.int32))
    br.read_lengths()
    plan = BranchPlan([60, 0, 3, 33], num_heads=8, num_kv_heads=2)
    q = torch.empty(96, 8, 128, dtype=BF, device="cuda")
    k, v = (torch.empty(96, 2, 128, dtype=BF, device="cuda") for _ in range(2))
    few = [torch.empty(4, n, 128, dtype=BF, device="cuda") for n in (8, 2, 2)]
    logits = torch.empty(6, 5000, device="cuda")
    scores = torch.empty(2, 3, device="cuda")
    mass = torch.empty(2, 2, 900, device="cuda")

    def cut():
        kv.seq_len = 900
        got = evict(kv, mass, 700, recent=50, sinks=2)
        kv.seq_len = 900
        return list(got) + [kv.k.clone(), kv.v.clone()]

    calls = [lambda: [branch_attention(q, k, v, kv, br, 0, plan)],
             lambda: [branch_attention(*few, kv, br, 1)],
             lambda: list(beam_select(logits, scores, num=6)),
             lambda: [attention_mass(few[0][:1], kv, 0), attention_mass(q, kv, 1, mass[1])],
             lambda: [attention_mass(torch.cat([q] * 4), kv, 0)],
             cut]

    def fill():
        for x in (q, k, v, *few, logits):
            x.normal_(generator=g)
        scores.uniform_(-3, 0, generator=g)
        mass.uniform_(0, 5, generator=g)
        kv.k.normal_(generator=g)
        kv.v.normal_(generator=g)

    fill()
    for f in calls:
        f()
    torch.cuda.synchronize()
    graphs = []
    for f in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        graphs.append((f, graph, out))
    for _ in range(4):
        for f, graph, out in graphs:
            fill()
            state = [x.clone() for x in (kv.k, kv.v)]
            want = [x.clone() for x in f()]
            for x, y in zip((kv.k, kv.v), state):
                x.copy_(y)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_streams_and_two_threads():
    _say("two streams, two threads")
    want = []
    for seed in (6, 7):
        s = Search(seed=seed)
        for _ in range(5):
            s.step()
        want.append(s.state())
    pair = [Search(seed=seed) for seed in (6, 7)]
    streams = _streams()[:2]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, stream in zip(pair, streams):
            with torch.cuda.stream(stream):
                s.step()
    torch.cuda.synchronize()
    for s, w in zip(pair, want):
        assert all(torch.equal(a, b) for a, b in zip(s.state(), w))

    pair = [Search(seed=seed) for seed in (6, 7)]
    torch.cuda.synchronize()
    errors = []

    def work(s, stream):
        try:
            with torch.cuda.stream(stream):
                for _ in range(5):
                    s.step()
                stream.synchronize()
        except Exception as e:  # told below, in the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(pair, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    for s, w in zip(pair, want):
        assert all(torch.equal(a, b) for a, b in zip(s.state(), w))


# ------------------------------------------------------------ past 32 bits --

def test_far_branch_rows():
    """A branch cache of more than 2^32 bytes: its last rows."""
    from treemoe_spec_amd.kernels.branch_attention import BranchPlan, branch_attention
    from treemoe_spec_amd.kv_cache import BranchCache, MixtralConfig

    _say("branch rows past 2^32 bytes")
    g = torch.Generator().manual_seed(8)
    kv = t_attn._cache(70, 8, 128, BF, 16, 8, layers=1)
    shared = [torch.randn(70, 8, 128, generator=g).to(BF) for _ in range(2)]
    kv.append(0, *(x.cuda() for x in shared), 0)
    br = BranchCache(MixtralConfig(num_layers=1, num_kv_heads=8, head_dim=128), 40, 60000,
                     beams=20)
    assert br.k.numel() * 2 > 2 ** 32
    old = [torch.randn(2, 90, 8, 128, generator=g).to(BF) for _ in range(2)]
    br.k[0, 38:, :90] = old[0].cuda()
    br.v[0, 38:, :90] = old[1].cuda()
    br.lengths[20:] = 90
    br.read_lengths()
    br.origin[39, :40] = 38                              # an ancestor's
    plan = [BranchPlan([0] * 38 + [1, n], num_heads=8, num_kv_heads=8) for n in (1, 130)]
    for p, n in zip(plan, (1, 130)):
        q, k, v = (torch.randn(n + 1, 8, 128, generator=g).to(BF) for _ in range(3))
        out = branch_attention(q.cuda(), k.cuda(), v.cuda(), kv, br, 0, p).cpu()
        rows = torch.where(torch.arange(90) < 40, 0, 1)
        keys, values = (torch.cat([shared[i], old[i][rows, torch.arange(90)], (k, v)[i][1:]])
                        for i in (0, 1))
        t_attn._check(out[1:], q[1:], keys, values, 160)
        assert torch.equal(br.k[0, 39, 90:90 + n].cpu(), k[1:])
        assert torch.equal(br.v[0, 39, 90:90 + n].cpu(), v[1:])
    assert not bool(br.k[0, :38].any())


def test_far_pages_and_layers():
    """A cache of more than 2^32 bytes: mass and eviction in its last layer and pages."""
    from treemoe_spec_amd.kernels.cache_eviction import attention_mass
    from treemoe_spec_amd.kv_cache import MixtralConfig, PagedKVCache

    _say("pages past 2^32 bytes")
    g = torch.Generator().manual_seed(9)
    cfg = MixtralConfig(num_layers=3, num_kv_heads=8, head_dim=128)
    kv = PagedKVCache(cfg, 20000, page_size=64, tree_size=1)
    assert kv.k.numel() * 2 > 2 ** 32
    kv._free = kv._free[::-1]                            # the last pages first
    n = 700
    kv._ensure_capacity(n)
    kv.seq_len = n
    assert min(kv.block_table) > 19000
    q, k, v = t_attn._qkv(2, n, 32, 8, 128, BF, 10)
    kv.append(2, k.cuda(), v.cuda(), 0)
    got = attention_mass(q.cuda(), kv, 2)
    t_evict._check(got, q, k)
    for layer in range(2):
        kv.append(layer, *(torch.randn(n, 8, 128, generator=g).to(BF).cuda() for _ in range(2)), 0)
    mass = torch.rand(3, 8, n, generator=g)
    small = PagedKVCache(cfg, 14, page_size=64, tree_size=1)   # the same evicted nearby
    small._ensure_capacity(n)
    small.seq_len = n
    for layer in range(3):
        small.append(layer, *kv.gather(layer), 0)
    from treemoe_spec_amd.kernels.cache_eviction import evict

    a = evict(kv, mass.cuda(), 400, recent=30)
    b = evict(small, mass.cuda(), 400, recent=30)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    for layer in range(3):
        assert all(torch.equal(x, y) for x, y in zip(kv.gather(layer), small.gather(layer)))


def test_far_rows_of_beams():
    """Logits and states of more than 2^32 bytes."""
    from treemoe_spec_amd.kernels.beam_search import beam_select, reorder_rows

    _say("beams' rows past 2^32 bytes")
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.zeros(8, 700_000_000, dtype=torch.uint8, device="cuda")
    x[:, -5:] = torch.arange(8, dtype=torch.uint8, device="cuda")[:, None] + 1
    parents = torch.tensor([[3, 1, 0, 0], [2, 2, 1, 0]], dtype=torch.int32, device="cuda")
    reorder_rows(x, parents, out=x)
    assert x[:, -1].tolist() == [4, 2, 1, 1, 7, 7, 6, 5] and not bool(x[:, :1000].any())
    del x
    logits = torch.empty(72000, 32000, dtype=BF, device="cuda")
    for part in logits.split(8000):
        part.normal_(generator=g)
    scores = -torch.rand(18000, 4, generator=g, device="cuda")
    got = [y[-2:].cpu() for y in beam_select(logits, scores, num=8)]
    want = t_beam._want(logits[-8:].cpu(), scores[-2:].cpu(), 8)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
