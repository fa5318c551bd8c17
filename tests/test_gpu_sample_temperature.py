"""sample_tokens at temperatures up to the largest, against the definition in 64 bits
(the oracle and the tolerances of the sampling tests)."""

from __future__ import annotations

import pytest
import torch

from tests import test_gpu_sample_tokens as t_samp

pytestmark = pytest.mark.gpu

F32_MAX = torch.finfo(torch.float32).max


def _say(msg):
    print(msg, flush=True)


@pytest.mark.parametrize("v", [1000, 5001, 32000, 100001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [{}, {"top_p": 0.77}, {"top_p": 0.77, "min_p": 0.5},
                                {"top_k": 700, "top_p": 0.33}])
def test_infinite_and_largest(v, dtype, kw):
    """A row's infinite temperature acts as the largest finite one, and a number near
    the largest double is a temperature: every logit above -inf weighs the same."""
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    _say(f"sample infinite temperature v={v} {dtype} {kw}")
    logits, u = t_samp._logits(4, v, dtype, v)
    g = torch.Generator().manual_seed(v)
    logits[:, torch.randperm(v, generator=g)[:v // 5]] = -float("inf")  # masked, all over the row
    temps = torch.tensor([float("inf"), F32_MAX, 1e30, float("inf")])
    got, probs = sample_tokens(logits.cuda(), u.cuda(), temperature=temps.cuda(),
                               return_probs=True, **kw)
    torch.cuda.synchronize()
    t_samp._check(logits, u, got, probs, temperature=temps.clamp(max=F32_MAX), **kw)
    for temp in (1e307, 1.7e308):
        got, probs = sample_tokens(logits.cuda(), u.cuda(), temperature=temp, return_probs=True,
                                   **kw)
        torch.cuda.synchronize()
        t_samp._check(logits, u, got, probs, temperature=temp, **kw)


@pytest.mark.parametrize("v", [3000, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [{}, {"top_k": 50}, {"top_k": 2000}, {"top_p": 0.9},
                                {"min_p": 0.05}])
def test_logits_further_apart_than_the_largest_float(v, dtype, kw):
    """Logits whose difference passes the type's range, at temperatures that leave them
    a weight."""
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    _say(f"sample far logits v={v} {dtype} {kw}")
    g = torch.Generator().manual_seed(v)
    logits = ((torch.rand(4, v, generator=g) * 2 - 1) * 3.2e38).to(dtype)
    u = torch.rand(4, generator=g)
    temps = torch.tensor([F32_MAX, 1e38, 3e37, 1e38])
    got, probs = sample_tokens(logits.cuda(), u.cuda(), temperature=temps.cuda(),
                               return_probs=True, **kw)
    torch.cuda.synchronize()
    t_samp._check(logits, u, got, probs, temperature=temps, **kw)
