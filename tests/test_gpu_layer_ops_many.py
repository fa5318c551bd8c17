"""Norm and rotary positions above 1024 rows, where their kernels take several chunks or
heads a thread, against the 64-bit formulas (oracles and bounds of those operators'
tests)."""

from __future__ import annotations

import pytest
import torch

from tests import test_gpu_rms_norm as t_norm
from tests import test_gpu_rotary as t_rot

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _say(msg):
    print(msg, flush=True)


def _placed(x, aligned):
    """x on the GPU, as rows of a wider buffer that start on 2 or 4 bytes only, or whole."""
    if aligned:
        return x.cuda()
    buf = torch.zeros(x.shape[0], x.shape[1] + 5, dtype=x.dtype, device="cuda")
    view = buf[:, 3:3 + x.shape[1]]
    view.copy_(x)
    return view


@pytest.mark.parametrize("t,h", [(1025, 513), (1025, 520), (1027, 1024), (1025, 1032),
                                 (1026, 4096), (1025, 4104), (1030, 16392)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("aligned", [True, False])
def test_norm(t, h, dtype, aligned):
    from treemoe_spec_amd.kernels.rms_norm import rms_norm

    _say(f"rms_norm t={t} h={h} {dtype} aligned={aligned}")
    x, w, r = t_norm._inputs(t, h, dtype, t + h)
    xd, wd, rd = _placed(x, aligned), w.cuda(), _placed(r, aligned)
    y = rms_norm(xd, wd, 1e-5)
    torch.cuda.synchronize()
    t_norm._near(y, t_norm._want(x, w, None, 1e-5)[0])
    y, s = rms_norm(xd, wd, 1e-6, residual=rd)
    torch.cuda.synchronize()
    want, total = t_norm._want(x, w, r, 1e-6)
    # the sum itself is rounded to fp32 before it is squared or stored
    info = torch.finfo(dtype)
    scale = (x.abs().double() + r.abs().double()) * U
    assert bool(((s.double().cpu() - total).abs() <= total.abs() * info.eps / 2 + scale).all())
    inv = (want / total.where(total != 0, torch.ones_like(total))).abs().amax(1, keepdim=True)
    bound = want.abs() * (info.eps / 2 + 50 * U) + scale * inv + info.smallest_normal * info.eps
    assert bool(((y.double().cpu() - want).abs() <= bound).all())


@pytest.mark.parametrize("t,h,group", [(1030, 1024, None), (1030, 1024, 32), (1030, 1024, 512),
                                       (1029, 4096, None), (1029, 4096, 32), (1029, 4096, 128),
                                       (1029, 4096, 512), (1027, 999, None)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_fp8(t, h, group, dtype):
    from treemoe_spec_amd.kernels.rms_norm import rms_norm_fp8

    _say(f"rms_norm_fp8 t={t} h={h} group={group} {dtype}")
    x, w, r = t_norm._inputs(t, h, dtype, t + h, rdtype=torch.float32)
    q, sc, s = rms_norm_fp8(x.cuda(), w.cuda(), residual=r.cuda(), scale_group=group)
    torch.cuda.synchronize()
    want, _ = t_norm._want(x, w, r, 1e-5)
    assert torch.equal(s.cpu(), x.float() + r)
    parts = want.view(t, -1, group or h)
    scale = parts.abs().amax(2) / 448
    sc = sc.cpu().double().view(t, -1)
    assert bool(((sc - scale).abs() <= scale * 60 * U + 1e-9).all())
    quot = parts / sc[:, :, None]
    got = q.cpu().float().double().view(parts.shape)
    assert bool(((got - quot).abs() <= quot.abs() * (2.0 ** -4 + 120 * U) + 2.0 ** -10 + 2e-4).all())
    assert bool((got.abs().amax(2) == 448).all())


@pytest.mark.parametrize("t", [1024, 1300])
@pytest.mark.parametrize("hq,kvh,hd,part", [(32, 8, 128, 128), (17, 3, 64, 64), (32, 8, 128, 64),
                                            (40, 1, 80, 32)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotary_embed(t, hq, kvh, hd, part, inter, dtype):
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_embed

    _say(f"rotary t={t} heads={hq}/{kvh} hd={hd} part={part} inter={inter} {dtype}")
    plan = RotaryPlan(hd, 1e6, rotary_dim=part, interleaved=inter,
                      scaling={"type": "yarn", "factor": 8.0, "original_max_position": 4096})
    q, k, _ = t_rot._qkv(t, hq, kvh, hd, dtype, t + hq)
    pos = torch.randint(0, 1 << 20, (t,), generator=torch.Generator().manual_seed(t))
    got = rotary_embed(q.cuda(), k.cuda(), pos.cuda(), plan)
    torch.cuda.synchronize()
    for y, x in zip(got, (q, k)):
        want, mag = t_rot._rotate(x, pos, plan.inv_freq, plan.magnitude, part, inter)
        t_rot._near(y, want, mag)
        assert torch.equal(y[..., part:].cpu(), x[..., part:])


@pytest.mark.parametrize("t,start", [(1024, 0), (1300, 37)])
@pytest.mark.parametrize("hq,kvh", [(32, 8), (17, 3)])
@pytest.mark.parametrize("inter,part", [(False, 128), (True, 64)])
def test_rotary_append(t, start, hq, kvh, inter, part):
    """A thread's heads run over q, rotated k and copied v: the bits of rotary_embed and of
    the cache's own append, also around a page that lies outside the cache."""
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_append, rotary_embed

    _say(f"rotary_append t={t} start={start} heads={hq}/{kvh} inter={inter} part={part}")
    page = 16
    plan = RotaryPlan(128, 1e6, rotary_dim=part, interleaved=inter)
    a, b = (t_rot._cache(kvh, 128, torch.bfloat16, page, (start + t) // page + 6) for _ in range(2))
    b.k.copy_(a.k)
    b.v.copy_(a.v)
    k0, v0 = a.k.clone(), a.v.clone()
    q, k, v = (x.cuda() for x in t_rot._qkv(t, hq, kvh, 128, torch.bfloat16, t))
    want_q, want_k = rotary_embed(q, k, torch.arange(t, device="cuda") + start, plan)
    for kv in (a, b):
        kv._ensure_capacity(start + t)
    a.append(1, want_k, v, start)
    bad = 5
    gone, b.block_table[bad] = b.block_table[bad], b.k.shape[1]
    got = rotary_append(q, k, v, plan, b, 1, start)
    torch.cuda.synchronize()
    assert torch.equal(got, want_q)
    a.k[1, gone], a.v[1, gone] = k0[1, gone], v0[1, gone]
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    assert b.seq_len == start + t
