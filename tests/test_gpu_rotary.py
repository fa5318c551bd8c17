"""rotary_embed and rotary_append on the GPU against the rotation in 64 bits.

Tolerances.  With u = 2^-24: the angle is known to 2^-34 turn (4e-10 rad), sine and
cosine to 2^-23 absolutely (argument, polynomial and Horner roundings of about u
each), the magnitude's product to u, and the two products and their difference
to 1.5 u of |a| + |b| each.  |got - want| <= 8 u m (|a| + |b|) + half a step of the
type of the result."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _say(msg):
    print(msg, flush=True)


def _rotate(x, positions, freq, m, part, inter):
    """64-bit rotation, and |a| + |b| of every element's pair."""
    x = x.double()
    ang = positions.double()[:, None] * torch.tensor(freq, dtype=torch.float64)[None]
    cos, sin = (ang.cos() * m)[:, None], (ang.sin() * m)[:, None]
    out, mag = x.clone(), torch.zeros_like(x)
    lo = slice(0, part, 2) if inter else slice(0, part // 2)
    hi = slice(1, part, 2) if inter else slice(part // 2, part)
    a, b = x[..., lo], x[..., hi]
    out[..., lo], out[..., hi] = a * cos - b * sin, b * cos + a * sin
    mag[..., lo] = mag[..., hi] = m * (a.abs() + b.abs())
    return out, mag


def _near(got, want, mag):
    info = torch.finfo(got.dtype)
    bound = want.abs() * info.eps / 2 * (1 + 8 * U) + 8 * U * mag \
        + info.smallest_normal * info.eps
    bad = (got.double().cpu() - want).abs() > bound
    assert not bool(bad.any()), (got.double().cpu() - want)[bad][:4]


def _qkv(t, hq, kvh, hd, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(t, h, hd, generator=g).to(dtype) for h in (hq, kvh, kvh)]


SCALINGS = [None, {"type": "linear", "factor": 3.0}, {"type": "ntk", "factor": 4.0},
            {"type": "yarn", "factor": 8.0, "original_max_position": 4096}]


@pytest.mark.parametrize("t,hq,kvh,hd,part", [(1, 32, 8, 128, 128), (5, 4, 2, 64, 64),
                                              (64, 8, 2, 128, 64), (3, 3, 1, 80, 32),
                                              (1100, 4, 4, 16, 16), (33, 2, 2, 256, 256)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_embed(t, hq, kvh, hd, part, inter, dtype):
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_embed

    _say(f"rotary t={t} heads={hq}/{kvh} hd={hd} part={part} inter={inter} {dtype}")
    scaling = SCALINGS[(t + hd) % 4]
    plan = RotaryPlan(hd, 1e6, rotary_dim=part, interleaved=inter, scaling=scaling)
    q, k, _ = _qkv(t, hq, kvh, hd, dtype, t + hd)
    g = torch.Generator().manual_seed(t)
    pos = torch.randint(0, 1 << 22, (t,), generator=g)
    pos[0] = 0
    for ptype in (torch.int64, torch.int32):
        qo, ko = rotary_embed(q.cuda(), k.cuda(), pos.to(ptype).cuda(), plan)
        torch.cuda.synchronize()
        for got, x in ((qo, q), (ko, k)):
            want, mag = _rotate(x, pos, plan.inv_freq, plan.magnitude, part, inter)
            _near(got, want, mag)
            assert torch.equal(got[..., part:].cpu(), x[..., part:])
    # position 0 turns nothing: the magnitude alone
    assert torch.equal(qo[0].cpu(), _rotate(q, pos, plan.inv_freq, plan.magnitude, part,
                                            inter)[0][0].to(dtype)) or plan.magnitude != 1.0


@pytest.mark.parametrize("pos", [0, 1, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 40 + 12345, -1, -77777])
def test_far_positions(pos):
    """The angle is exact mod a turn at any 64-bit position: against the same product
    in integers (Python's, of unlimited size)."""
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_embed

    _say(f"rotary far position {pos}")
    plan = RotaryPlan(64, 1e4)
    q, _, _ = _qkv(1, 2, 1, 64, torch.float32, 3)
    got, _ = rotary_embed(q.cuda(), None, torch.tensor([pos]).cuda(), plan)
    turns = [(pos * int(f)) % 2 ** 64 for f in plan.turns.tolist()]
    ang = torch.tensor([2 * math.pi * u / 2 ** 64 for u in turns], dtype=torch.float64)
    x = q[0].double()
    a, b = x[:, :32], x[:, 32:]
    want = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], 1)
    mag = torch.cat([a.abs() + b.abs()] * 2, 1)
    _near(got[0], want, mag)


def test_turns_of_the_frequencies():
    """F 2^-64 turns is the frequency to 2^-64 turn and double's own rounding."""
    from treemoe_spec_amd.kernels.rotary import RotaryPlan

    plan = RotaryPlan(128, 1e6)
    for f, u in zip(plan.inv_freq, plan.turns.tolist()):
        assert abs((u % 2 ** 64) / 2 ** 64 * 2 * math.pi - f) <= 1e-15 * f + 2 ** -60


def test_in_place_and_fused_projection_views():
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_embed

    _say("rotary in place")
    plan = RotaryPlan(128, 1e6)
    qkv = torch.randn(9, 12 * 128, device="cuda").to(torch.bfloat16)
    keep = qkv.clone()
    q, k = qkv[:, :8 * 128].view(9, 8, 128), qkv[:, 8 * 128:10 * 128].view(9, 2, 128)
    pos = torch.arange(9, device="cuda") * 100
    want = rotary_embed(q, k, pos, plan)
    got = rotary_embed(q, k, pos, plan, q_out=q, k_out=k)
    torch.cuda.synchronize()
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(qkv[:, 10 * 128:], keep[:, 10 * 128:])


def _cache(kvh, hd, dtype, page, pages, layers=2):
    from treemoe_spec_amd.kv_cache import MixtralConfig, PagedKVCache

    cfg = MixtralConfig(num_layers=layers, num_kv_heads=kvh, head_dim=hd)
    kv = PagedKVCache(cfg, pages, device="cuda", dtype=dtype, page_size=page, tree_size=page)
    kv.k.normal_()
    kv.v.normal_()
    return kv


@pytest.mark.parametrize("t,start,page", [(1, 0, 16), (1, 31, 16), (40, 5, 16), (7, 60, 64),
                                          (1300, 100, 16), (5, 3, 24)])
@pytest.mark.parametrize("dtype,inter,part", [(torch.bfloat16, False, 128),
                                              (torch.float16, True, 64)])
def test_append(t, start, page, dtype, inter, part):
    """The same bits as rotary_embed and the cache's own append; nothing else in
    the cache changes."""
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_append, rotary_embed

    _say(f"rotary_append t={t} start={start} page={page} {dtype}")
    plan = RotaryPlan(128, 1e6, rotary_dim=part, interleaved=inter)
    a = _cache(2, 128, dtype, page, (start + t) // page + 6)
    b = _cache(2, 128, dtype, page, (start + t) // page + 6)
    b.k.copy_(a.k)
    b.v.copy_(a.v)
    q, k, v = (x.cuda() for x in _qkv(t, 8, 2, 128, dtype, t))
    if start:  # what the cache held before
        for kv in (a, b):
            kv._ensure_capacity(start)
            kv.seq_len = start
    pos = torch.arange(t, device="cuda") + start
    want_q, want_k = rotary_embed(q, k, pos, plan)
    a.append(1, want_k, v, start)
    got = rotary_append(q, k, v, plan, b, 1, start)
    torch.cuda.synchronize()
    assert torch.equal(got, want_q)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    assert a.seq_len == b.seq_len == start + t and a.block_table == b.block_table


def test_append_skips_pages_out_of_range():
    """A block table entry outside the cache stores nothing."""
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_append

    _say("rotary_append bad pages")
    plan = RotaryPlan(128, 1e6)
    kv = _cache(2, 128, torch.bfloat16, 16, 6)
    kv.block_table = [3, 6, -1, 4]
    k0, v0 = kv.k.clone(), kv.v.clone()
    q, k, v = (x.cuda() for x in _qkv(64, 4, 2, 128, torch.bfloat16, 2))
    rotary_append(q, k, v, plan, kv, 0, 0)
    torch.cuda.synchronize()
    changed = (kv.v != v0).flatten(2).any(2)
    assert changed[0].tolist() == [False, False, False, True, True, False]
    assert not bool(changed[1].any())
    assert torch.equal(kv.v[0, 3], v[:16]) and torch.equal(kv.v[0, 4], v[48:])
    assert torch.equal(kv.k[1], k0[1])
