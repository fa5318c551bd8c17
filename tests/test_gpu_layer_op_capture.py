"""Captured rotary_append and prompt_attention_cached after the cache's pages have changed:
a replay works on the positions of the capture, in the pages of the cache's device table."""

from __future__ import annotations

import pytest
import torch

from tests import test_gpu_prompt_attention as t_attn
from tests import test_gpu_rotary as t_rot

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _say(msg):
    print(msg, flush=True)


def _reference_layout():
    from tests.ref_layout_cache import RefLayoutKVCache

    return RefLayoutKVCache(2, 2, 128, 40)


def _own_layout():
    return t_rot._cache(2, 128, BF, 64, 40)


@pytest.mark.parametrize("make", [_own_layout, _reference_layout])
def test_replay_follows_the_table(make):
    from treemoe_spec_amd.kernels.prompt_attention import prompt_attention_cached
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_append

    _say(f"replay after the pages changed {make.__name__}")
    plan, kv, t, s = RotaryPlan(128, 1e6), make(), 3, 200
    q, k, v = (x.cuda() for x in t_attn._qkv(s, s, 8, 2, 128, BF, 1))

    def fill(lo, hi):
        qr = rotary_append(q[lo:hi], k[lo:hi], v[lo:hi], plan, kv, 1, lo)
        return prompt_attention_cached(qr, kv, 1)

    fill(0, s - t)
    want = fill(s - t, s)        # the pages are mapped and on the device
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fill(s - t, s)
    for _ in range(4):
        # the same sequence again, in other pages
        old = list(kv.block_table)
        kv.block_table.clear()
        kv.seq_len = 0
        if hasattr(kv, "reset"):
            kv.reset()
        fill(0, s - t)
        kv._ensure_capacity(s)
        assert not set(old) & set(kv.block_table)
        eager = fill(s - t, s)
        assert torch.equal(eager, want)
        kv.k[1, old], kv.v[1, old] = float("nan"), float("nan")
        for c in (kv.k, kv.v):
            c[1, kv.block_table[-1], (s - t) % 64:].fill_(float("nan"))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_a_plan_dropped_behind_a_call_on_another_stream():
    """The lists of a plan stay its own until the calls that read them have ended."""
    from treemoe_spec_amd.kernels.prompt_attention import PromptPlan, prompt_attention
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_embed

    _say("plans dropped early")
    q, k, v = (x.cuda() for x in t_attn._qkv(70, 900, 8, 2, 128, BF, 3))
    pos = torch.arange(70, device="cuda")

    def plans():
        return PromptPlan([70], [900], num_heads=8, num_kv_heads=2), RotaryPlan(128, 1e6)

    plan, rope = plans()
    want = prompt_attention(q, k, v, plan), rotary_embed(q, None, pos, rope)[0]
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(60):
            busy = busy @ busy * 1e-3     # the calls wait behind it
        got = prompt_attention(q, k, v, plan), rotary_embed(q, None, pos, rope)[0]
        ended = torch.cuda.Event()
        ended.record()
    held = {t.data_ptr() for t in (plan.items, plan.joins, rope.turns)}
    del plan, rope
    others = [plans() for _ in range(3)]
    assert not ended.query()
    assert not held & {t.data_ptr() for a, b in others for t in (a.items, a.joins, b.turns)}
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
