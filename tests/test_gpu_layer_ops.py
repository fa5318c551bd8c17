"""Norm, rotary, prompt attention and sampling together: a decoder's prompt, a
speculative step and the decoded token after it; and each under graph capture, on two
streams and from two threads.

The steps' numbers are held against 64-bit formulas of each operator's own inputs
(tolerances: those operators' tests); replays, streams and threads against the same
call's bits on one stream."""

from __future__ import annotations

import threading

import pytest
import torch

from tests import test_gpu_prompt_attention as t_attn
from tests import test_gpu_rms_norm as t_norm
from tests import test_gpu_rotary as t_rot
from tests import test_gpu_sample_tokens as t_samp
from tests.engine_harness import TinyConfig, random_model

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _say(msg):
    print(msg, flush=True)


class Decoder:
    """A decoder of bfloat16 operators and a float32 residual stream.  Every result of
    the four operators is checked on the way."""

    def __init__(self, cfg: TinyConfig, seed: int):
        from treemoe_spec_amd.kernels.rotary import RotaryPlan
        from treemoe_spec_amd.moe_adapter import make_moe_fn

        self.cfg = cfg
        self.layers, embed, lm_head = random_model(cfg, seed)
        self.embed, self.lm_head = embed.to(BF), lm_head.to(BF)
        self.plan = RotaryPlan(cfg.head_dim, cfg.rope_theta)
        self.moe_fn = make_moe_fn(expert_budget=cfg.num_experts, tree_size=cfg.tree_size,
                                  device="cuda")

    def cache(self, pages=40):
        from treemoe_spec_amd.kv_cache import MixtralConfig, PagedKVCache

        c = self.cfg
        return PagedKVCache(MixtralConfig(num_layers=c.num_layers, num_kv_heads=c.num_kv_heads,
                                          head_dim=c.head_dim, num_heads=c.num_heads),
                            pages, device="cuda", page_size=c.page_size, tree_size=c.tree_size)

    def norm(self, x, w, residual=None):
        from treemoe_spec_amd.kernels.rms_norm import rms_norm

        w = w.to(x.dtype)
        got = rms_norm(x, w, self.cfg.rms_eps, residual=residual)
        y, total = got if residual is not None else (got, None)
        args = x.cpu(), w.cpu(), None if residual is None else residual.cpu()
        want, s = t_norm._want(*args, self.cfg.rms_eps)
        if total is not None:
            assert float((total.double().cpu() - s).abs().max()) <= float(s.abs().max()) * 2 * t_norm.U
            want, _ = t_norm._want(total.cpu(), args[1], None, self.cfg.rms_eps)
        # the float32 sum is off by one rounding of itself: one more u of the output, or
        # less, for the element and for the root
        t_norm._near(y, want, 52 * t_norm.U)
        return y, total

    def qkv(self, y, lw):
        c = self.cfg
        w = torch.cat([lw.wq, lw.wk, lw.wv]).to(BF)
        full = (y @ w.T).view(y.shape[0], c.num_heads + 2 * c.num_kv_heads, c.head_dim)
        return full.split([c.num_heads, c.num_kv_heads, c.num_kv_heads], 1)

    def rotated(self, got, x, pos):
        want, mag = t_rot._rotate(x.cpu(), pos, self.plan.inv_freq, self.plan.magnitude,
                                  self.cfg.head_dim, False)
        t_rot._near(got, want, mag)

    def run(self, tokens, attention):
        """``attention(layer, q, k, v)`` -> context [T, Hq * hd]; float32 logits."""
        x = self.embed[tokens]
        y, total = self.norm(x, self.layers[0].ln1)[0], x.float()
        for li, lw in enumerate(self.layers):
            o = attention(li, *self.qkv(y, lw))
            y, total = self.norm(o.flatten(1) @ lw.wo.to(BF).T, lw.ln2, total)
            y = self.moe_fn(y, lw, li)
            last = li + 1 == len(self.layers)
            y, total = self.norm(y, lw.ln1 if last else self.layers[li + 1].ln1, total)
        return (y @ self.lm_head.T).float()

    def append(self, kv, start):
        """Attention of positions start.. of one sequence through its cache."""
        from treemoe_spec_amd.kernels.prompt_attention import prompt_attention_cached
        from treemoe_spec_amd.kernels.rotary import rotary_append

        def attention(li, q, k, v):
            qr = rotary_append(q, k, v, self.plan, kv, li, start)
            t = q.shape[0]
            self.rotated(qr, q, torch.arange(start, start + t))
            out = prompt_attention_cached(qr, kv, li)
            kk, vv = kv.gather(li)
            self.rotated(kk[start:], k, torch.arange(start, start + t))
            assert torch.equal(vv[start:], v)
            t_attn._check(out, qr.cpu(), kk.cpu(), vv.cpu(), start)
            return out
        return attention

    def tree(self, kv, depth, mask):
        from treemoe_spec_amd.kernels.rotary import rotary_embed
        from treemoe_spec_amd.kernels.tree_attention import tree_attention

        def attention(li, q, k, v):
            pos = torch.tensor([kv.seq_len + d for d in depth])
            qr, kr = rotary_embed(q, k, pos.cuda(), self.plan)
            self.rotated(qr, q, pos)
            self.rotated(kr, k, pos)
            v = v.clone(memory_format=torch.contiguous_format)  # kr's strides
            return tree_attention(qr, kr, v, kv, li, mask)
        return attention


def _sample(logits, u, **kw):
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    tokens, probs = sample_tokens(logits, u, return_probs=True, **kw)
    t_samp._check(logits.cpu(), u.cpu(), tokens, probs, **kw)
    return tokens, probs


@pytest.mark.parametrize("seed", [3, 8])
def test_prompt_speculative_step_and_decode(seed):
    from oracle.attn_ref import ancestor_mask
    from treemoe_spec_amd.kernels.op4_commit import fused_verify_commit

    _say(f"prompt, draft, verification, decode: seed {seed}")
    cfg = TinyConfig()
    model, g = Decoder(cfg, seed), torch.Generator().manual_seed(seed)
    kv = model.cache()
    prompt = torch.randint(0, cfg.vocab_size, (83,), generator=g).cuda()
    # the prompt in two chunks
    model.run(prompt[:50], model.append(kv, 0))
    logits = model.run(prompt[50:], model.append(kv, 50))
    assert kv.seq_len == 83
    root, _ = _sample(logits[-1:], torch.rand(1, generator=g).cuda(), temperature=0.8, top_p=0.9)

    # a draft of three children of the root, two of the first child
    one = torch.ones(1, 1, dtype=torch.bool, device="cuda")
    head = model.run(root, model.tree(kv, [0], one))
    kids, probs0 = _sample(head.expand(3, -1), torch.rand(3, generator=g).cuda(), temperature=0.7)
    parent = [-1, 0, 0, 0, 1, 1]
    depth = [0, 1, 1, 1, 2, 2]
    mask = ancestor_mask(parent).cuda()
    tokens = torch.cat([root, kids, kids[:2]])
    heads = model.run(tokens[:4], model.tree(kv, depth[:4], mask[:4, :4].contiguous()))
    grand, probs1 = _sample(heads[1:2].expand(2, -1), torch.rand(2, generator=g).cuda(),
                            temperature=0.7)
    tokens = torch.cat([root, kids, grand])
    draft = torch.cat([probs0[:1], probs0, probs1])  # a node's: what it was drawn from
    target = model.run(tokens, model.tree(kv, depth, mask))
    children = [[1, 2, 3], [4, 5], [], [], [], []]
    res = fused_verify_commit(target, draft, tokens, None, children, kv=kv, temperature=0.7,
                              max_depth=2, generator=torch.Generator("cuda").manual_seed(seed))
    n = int(res.num_accepted)
    path = res.accepted_slots[:n].tolist()
    assert 0 <= n <= 2 and kv.seq_len == 83 + 1 + n
    assert all(path[i] in children[path[i - 1] if i else 0] for i in range(n))
    assert res.accepted_tokens[:n].tolist() == tokens[path].tolist()
    bonus = int(res.bonus_token)
    assert 0 <= bonus < cfg.vocab_size

    # the decoded token behind the committed path reads what the commit moved
    start = kv.seq_len
    logits = model.run(torch.tensor([bonus], device="cuda"), model.append(kv, start))
    assert kv.seq_len == start + 1
    last, _ = _sample(logits, torch.rand(1, generator=g).cuda(), temperature=0.0)
    assert int(last) == int(logits.argmax())


def test_packed_prompts_match_their_caches():
    """Two prompts packed into one batch, padded, and each through a cache of its own:
    the same context within the operator's tolerance, from the same inputs."""
    from treemoe_spec_amd.kernels.prompt_attention import PromptPlan, prompt_attention
    from treemoe_spec_amd.kernels.rotary import rotary_embed

    _say("packed prompts and their caches")
    cfg = TinyConfig()
    model, g = Decoder(cfg, 4), torch.Generator().manual_seed(4)
    lens = [70, 21]
    tokens = torch.randint(0, cfg.vocab_size, (sum(lens) + 5,), generator=g).cuda()
    pos = torch.cat([torch.arange(n) for n in lens] + [torch.zeros(5, dtype=torch.int64)])
    plan = PromptPlan(lens, num_heads=cfg.num_heads, num_kv_heads=cfg.num_kv_heads)
    caches = [model.cache() for _ in lens]

    def attention(li, q, k, v):
        qr, kr = rotary_embed(q, k, pos.cuda(), model.plan)
        out = prompt_attention(qr, kr, v, plan)
        at = 0
        for n, kv in zip(lens, caches):
            s = slice(at, at + n)
            t_attn._check(out[s], qr[s].cpu(), kr[s].cpu(), v[s].cpu(), 0)
            model.append(kv, 0)(li, q[s], k[s], v[s])
            assert torch.equal(kv.gather(li)[0], kr[s])
            at += n
        assert not bool(out[at:].any())
        return out

    logits = model.run(tokens, attention)
    ends = logits[torch.tensor(lens).cumsum(0).cuda() - 1]
    _sample(ends, torch.rand(2, generator=g).cuda(), temperature=0.9, top_k=20, min_p=0.01)


# ------------------------------------------------- capture, streams, threads --

def _calls():
    """name -> call of one operator on fixed inputs; each returns a tensor list."""
    from treemoe_spec_amd.kernels.prompt_attention import (PromptPlan, prompt_attention,
                                                           prompt_attention_cached)
    from treemoe_spec_amd.kernels.rms_norm import rms_norm, rms_norm_fp8
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_append, rotary_embed
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    x, w, r = (t.cuda() for t in t_norm._inputs(70, 1024, BF, 1))
    plan = RotaryPlan(128, 1e6)
    q, k, v = (t.cuda() for t in t_rot._qkv(70, 8, 2, 128, BF, 2))
    pos = torch.arange(70).cuda() * 3
    kv, wkv = t_rot._cache(2, 128, BF, 16, 200), t_rot._cache(2, 128, BF, 16, 20)
    kv._ensure_capacity(3000)
    kv.seq_len = 3000
    kv.device_tables("cuda")
    wkv._ensure_capacity(100)
    wkv.device_tables("cuda")
    split = PromptPlan([1, 40], [2500, 2900], num_heads=8, num_kv_heads=2)
    few = PromptPlan([1, 3], [2500, 2900], num_heads=8, num_kv_heads=2)
    assert split.num_joins and few.num_joins and few.tiling == 0
    kk, vv = (torch.randn(5400, 2, 128, dtype=BF, device="cuda") for _ in range(2))
    logits, u = (t.cuda() for t in t_samp._logits(6, 40000, torch.float32, 5))
    return {
        "rms_norm": lambda: list(rms_norm(x, w, residual=r)),
        "rms_norm_fp8": lambda: [t.float() for t in rms_norm_fp8(x, w, residual=r, scale_group=128)],
        "rotary_embed": lambda: list(rotary_embed(q, k, pos, plan)),
        "rotary_append": lambda: [rotary_append(q, k, v, plan, wkv, 1, 7),
                                  wkv.k[1].clone(), wkv.v[1].clone()],
        "prompt_attention": lambda: [prompt_attention(q[:41], kk, vv, split),
                                     prompt_attention(q[:4], kk, vv, few)],
        "prompt_attention_cached": lambda: [prompt_attention_cached(q, kv, 0),
                                            prompt_attention_cached(q[:1], kv, 1)],
        "sample_tokens": lambda: list(sample_tokens(logits, u, top_p=0.9, return_probs=True)),
    }


def _same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_and_replayed():
    """Each operator in a graph of its own; the graphs replayed one after the other and
    on two streams at once, with eager calls and synchronisations between."""
    calls = _calls()
    torch.cuda.synchronize()
    graphs, outs, want = {}, {}, {}
    for name, call in calls.items():
        _say(f"capture {name}")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call()
        torch.cuda.current_stream().wait_stream(s)
        want[name] = call()
        torch.cuda.synchronize()
        graphs[name] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[name]):
            outs[name] = call()
    for r in range(4):
        for name, g in graphs.items():
            _say(f"replay {r} {name}")
            for t in outs[name]:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert _same(outs[name], want[name]), (name, r)
            assert _same(calls[name](), want[name]), (name, r)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    _say("two graphs with workspaces at once")
    for r in range(4):
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            graphs["prompt_attention"].replay()
        with torch.cuda.stream(b):
            graphs["prompt_attention_cached"].replay()
        torch.cuda.synchronize()
        for name in ("prompt_attention", "prompt_attention_cached"):
            assert _same(outs[name], want[name]), (name, r)


def test_two_streams_and_two_threads():
    calls = _calls()
    torch.cuda.synchronize()
    want = {name: call() for name, call in calls.items()}
    torch.cuda.synchronize()
    _say("two streams")
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for r in range(3):
        for name, call in calls.items():
            for s in streams[:1 if name == "rotary_append" else 2]:
                with torch.cuda.stream(s):
                    got.append((name, call()))
    torch.cuda.synchronize()
    assert all(_same(g, want[n]) for n, g in got)

    _say("two threads")
    results, errors = [], []

    def work(skip):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    for name, call in calls.items():
                        if name != skip:
                            results.append((name, call()))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in (None, "rotary_append")]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors and all(_same(g, want[n]) for n, g in results)


def test_a_cache_of_the_reference_layout():
    """rotary_append and prompt_attention_cached on a cache without device tables: the
    same bits as on this package's."""
    from tests.ref_layout_cache import RefLayoutKVCache
    from treemoe_spec_amd.kernels.prompt_attention import prompt_attention_cached
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_append

    _say("cache of the reference layout")
    plan = RotaryPlan(128, 1e6)
    ours, ref = t_rot._cache(2, 128, BF, 64, 20), RefLayoutKVCache(2, 2, 128, 20)
    start = 0
    for t in (100, 30, 1):
        q, k, v = (x.cuda() for x in t_rot._qkv(t, 8, 2, 128, BF, t))
        outs = []
        for kv in (ours, ref):
            for layer in (0, 1):
                qr = rotary_append(q, k, v, plan, kv, layer, start)
                outs.append(prompt_attention_cached(qr, kv, layer))
        start += t
        assert ref.seq_len == ours.seq_len == start
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
