"""CPU: a plan that is used on another stream than it was made on tells the allocator, since
its lists may be read after the caller has dropped it."""

from __future__ import annotations

import pytest
import torch

from treemoe_spec_amd import _capi
from treemoe_spec_amd.kernels import prompt_attention as pa
from treemoe_spec_amd.kernels import rotary as ro

BF = torch.bfloat16


@pytest.fixture()
def device(monkeypatch):
    """Launches recorded instead of made; ``now[0]`` stands for the current stream and
    ``marked`` holds what was marked as used by which."""
    now, marked = [0], []
    monkeypatch.setattr(_capi, "require", lambda *a, **k: None)
    monkeypatch.setattr(_capi, "launch", lambda *a: None)
    monkeypatch.setattr(_capi, "stream_made_on", lambda device: now[0])
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: now[0],
                        raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index=None: now[0])
    monkeypatch.setattr(torch.Tensor, "record_stream",
                        lambda t, s: marked.append((t.data_ptr(), s)))
    return now, marked


def test_prompt_plan(device):
    now, marked = device
    plan = pa.PromptPlan([2], [3000], num_heads=2, num_kv_heads=1, device="cpu")
    q, k = torch.zeros(2, 2, 64, dtype=BF), torch.zeros(3000, 1, 64, dtype=BF)
    pa.prompt_attention(q, k, k, plan)
    assert not marked
    now[0] = 7
    pa.prompt_attention(q, k, k, plan)
    assert marked == [(plan.items.data_ptr(), 7), (plan.joins.data_ptr(), 7)]


def test_rotary_plan(device):
    from treemoe_spec_amd.kv_cache import MixtralConfig, PagedKVCache

    now, marked = device
    plan = ro.RotaryPlan(16, 1e4, device="cpu")
    kv = PagedKVCache(MixtralConfig(num_layers=1, num_kv_heads=1, head_dim=16), 6, device="cpu",
                      dtype=torch.float32, page_size=4, tree_size=4)
    q = torch.zeros(2, 1, 16)
    for _ in range(2):
        ro.rotary_embed(q, None, torch.arange(2), plan)
        ro.rotary_append(q, q, q, plan, kv, 0, 0)
        assert marked == [(plan.turns.data_ptr(), 7)] * (2 if now[0] else 0)
        now[0] = 7
