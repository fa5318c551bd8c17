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
