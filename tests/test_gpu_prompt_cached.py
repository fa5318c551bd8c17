"""prompt_attention_cached in each of its tilings, up to a whole long prompt, over pages
from one slot on: against attention in 64 bits, with the bounds of the packed form's tests.
The oracle runs on the GPU, head by head."""

from __future__ import annotations

import pytest
import torch

from tests import test_gpu_prompt_attention as t_attn

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
FEW, SHORT, PAIR, TALL = range(4)


def _say(msg):
    print(msg, flush=True)


def _check(got, q, k, v, past):
    t, hq, hd = q.shape
    s, kvh, _ = k.shape
    scale = hd ** -0.5
    info = torch.finfo(q.dtype)
    e = info.eps / 2
    ds = 130 * t_attn.U * scale * float(q.abs().max()) * float(k.abs().max()) * hd
    hidden = torch.ones(t, s, dtype=torch.bool, device="cuda").triu(past + 1)
    got = got.view(t, hq, hd)
    for h in range(hq):
        kk = k[:, h * kvh // hq].double()
        vv = v[:, h * kvh // hq].double()
        w = torch.softmax((q[:, h].double() @ kk.T.contiguous() * scale)
                          .masked_fill_(hidden, -float("inf")), 1)
        want, mag = w @ vv, w @ vv.abs()
        bound = e * want.abs() + (2 * e + 2 * ds + 640 * t_attn.U) * mag \
            + info.smallest_normal * info.eps
        off = (got[:, h].double() - want).abs()
        assert bool((off <= bound).all()), (h, float((off - bound).max()))


@pytest.mark.parametrize("t,s,hq,kvh,hd,dtype,page,tiling", [
    (1, 700, 32, 8, 128, BF, 2, FEW),
    (8, 1501, 8, 2, 64, FP, 4, FEW),
    (40, 300, 8, 2, 128, BF, 4, SHORT),
    (60, 200, 8, 2, 64, FP, 1, SHORT),
    (300, 1500, 8, 2, 128, BF, 4, PAIR),     # its keys in several ranges
    (301, 1503, 8, 2, 64, FP, 1, PAIR),
    (2000, 2000, 32, 8, 128, BF, 2, PAIR),
    (2001, 2003, 32, 8, 64, BF, 64, PAIR),
    (3600, 3600, 32, 8, 128, BF, 16, TALL),
    (3700, 4001, 32, 8, 64, FP, 64, TALL),
    (1800, 2600, 64, 16, 128, FP, 8, TALL),
    (1800, 2600, 64, 16, 64, BF, 8, TALL),
    (1801, 2603, 64, 8, 128, BF, 4, TALL),
    (1801, 2603, 64, 8, 64, FP, 1, TALL),
    (8192, 8192, 32, 8, 128, BF, 16, TALL),
])
def test_every_tiling(t, s, hq, kvh, hd, dtype, page, tiling):
    """What was never written holds NaN, the slots behind the sequence too."""
    from treemoe_spec_amd.kernels.prompt_attention import PromptPlan, prompt_attention_cached

    _say(f"cached tiling {tiling} t={t} s={s} heads={hq}/{kvh} hd={hd} {dtype} page={page}")
    # the rule is that of packed sequences, by the mean of a tile's keys
    assert PromptPlan([t], [s], num_heads=hq, num_kv_heads=kvh).tiling == tiling
    q, k, v = (x.cuda() for x in t_attn._qkv(t, s, hq, kvh, hd, dtype, t + s))
    kv = t_attn._cache(s, kvh, hd, dtype, page, s)
    kv.append(1, k, v, 0)
    out = prompt_attention_cached(q, kv, 1)
    torch.cuda.synchronize()
    _check(out, q, k, v, s - t)


@pytest.mark.parametrize("page", [4, 16])
def test_thirds(page):
    """Tiles that leave many CUs idle: their keys in three ranges."""
    from treemoe_spec_amd.kernels.prompt_attention import _workspace_bytes, prompt_attention_cached

    t, s, hq, kvh, hd = 520, 3601, 32, 8, 128
    _say(f"cached thirds page={page}")
    assert _workspace_bytes(t, s, hq, kvh, hd) == 3 * 17 * kvh * 128 * (hd + 2) * 4
    q, k, v = (x.cuda() for x in t_attn._qkv(t, s, hq, kvh, hd, BF, 1))
    kv = t_attn._cache(s, kvh, hd, BF, page, s)
    kv.append(0, k, v, 0)
    out = prompt_attention_cached(q, kv, 0)
    torch.cuda.synchronize()
    _check(out, q, k, v, s - t)


def test_a_whole_prompt_in_one_call_and_in_chunks():
    """rotary_append and prompt_attention_cached of a prompt of 4000 tokens, whole and in two
    chunks: the same keys, and the same context within the operator's bounds."""
    from treemoe_spec_amd.kernels.prompt_attention import prompt_attention_cached
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_append

    _say("whole prompt and chunks")
    t, plan = 4000, RotaryPlan(128, 1e6)
    q, k, v = (x.cuda() for x in t_attn._qkv(t, t, 32, 8, 128, BF, 5, scale=1.0))
    one, two = (t_attn._cache(t, 8, 128, BF, 16, t) for _ in range(2))
    qr = rotary_append(q, k, v, plan, one, 0, 0)
    whole = prompt_attention_cached(qr, one, 0)
    parts = []
    for lo, hi in ((0, 2500), (2500, t)):
        qp = rotary_append(q[lo:hi], k[lo:hi], v[lo:hi], plan, two, 0, lo)
        assert torch.equal(qp, qr[lo:hi])
        parts.append(prompt_attention_cached(qp, two, 0))
    kk, vv = one.gather(0)
    assert torch.equal(kk, two.gather(0)[0]) and torch.equal(vv, v)
    _check(whole, qr, kk, vv, 0)
    _check(torch.cat(parts), qr, kk, vv, 0)
