"""The inference operators refuse tensors that carry a forward-mode tangent, which they
would lose; the same tensors' primals are taken."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from tests import test_gpu_rotary as t_rot

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _calls():
    """name -> (call of a tensor list, the tensors)."""
    from treemoe_spec_amd.kernels.prompt_attention import (PromptPlan, prompt_attention,
                                                           prompt_attention_cached)
    from treemoe_spec_amd.kernels.rms_norm import rms_norm, rms_norm_fp8
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_append, rotary_embed
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    x, r, w = (torch.randn(*s, dtype=BF, device="cuda") for s in ((4, 64), (4, 64), (64,)))
    q, k, v = (t.cuda() for t in t_rot._qkv(4, 4, 2, 64, BF, 1))
    rope, pos = RotaryPlan(64, 1e4), torch.arange(4, device="cuda")
    kv = t_rot._cache(2, 64, BF, 16, 4)
    plan = PromptPlan([4], num_heads=4, num_kv_heads=2)
    logits, u = torch.randn(4, 100, device="cuda"), torch.rand(4, device="cuda")

    def append(q, k, v, kc, vc):
        kv.k, kv.v = kc, vc
        return rotary_append(q, k, v, rope, kv, 0, 0)

    def cached(q, kc, vc):
        kv.k, kv.v = kc, vc
        return prompt_attention_cached(q, kv, 0)

    return {
        "rms_norm": (lambda x, w, r: rms_norm(x, w, residual=r), [x, w, r]),
        "rms_norm_fp8": (lambda x, w, r: rms_norm_fp8(x, w, residual=r), [x, w, r]),
        "rotary_embed": (lambda q, k: rotary_embed(q, k, pos, rope), [q, k]),
        "rotary_append": (append, [q, k, v, kv.k, kv.v]),
        "prompt_attention": (lambda q, k, v: prompt_attention(q, k, v, plan), [q, k, v]),
        "prompt_attention_cached": (cached, [q, kv.k, kv.v]),
        "sample_tokens": (lambda l, u: sample_tokens(l, u, return_probs=True), [logits, u]),
        "sample_tokens temperature": (lambda l, t: sample_tokens(l, u, temperature=t),
                                      [logits, u + 0.5]),
    }


def test_tangents_are_refused():
    for name, (call, tensors) in _calls().items():
        print(name, flush=True)
        call(*tensors)
        for i, t in enumerate(tensors):
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError, match="tangent"):
                    call(*tensors[:i], dual, *tensors[i + 1:])
                call(*tensors)  # without one it is an ordinary call
        torch.cuda.synchronize()
