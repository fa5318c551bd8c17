"""rms_norm and rms_norm_fp8 on the GPU against the formula in 64 bits.

Tolerances.  With u = 2^-24 (half a step of float32): the sum of H squares in fp32
by a tree of depth at most 64 + 16 (8 chunks of 8 per thread in sequence, then
folds) is off by 80 u relative, the mean and square root by u each on top
(halved by the root), rsqrt by one unit in the last place (2 u), the three
products by u each: under 50 u.  Then the output's own rounding, half a step of its
type.  The sum's rounding is half a step.  |got - want| <= (eps / 2 + 50 u) |want|,
plus the type's smallest subnormal."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _say(msg):
    print(msg, flush=True)


def _near(got, want, slack=50 * U):
    info = torch.finfo(got.dtype)
    bound = want.abs() * (info.eps / 2 + slack) + info.smallest_normal * info.eps
    bad = (got.double().cpu() - want).abs() > bound
    assert not bool(bad.any()), (got.double().cpu() - want)[bad][:4]


def _want(x, w, r, eps):
    s = x.double() + (0 if r is None else r.double())
    return s / (s.square().mean(1, keepdim=True) + eps).sqrt() * w.double(), s


def _inputs(t, h, dtype, seed, rdtype=None, wdtype=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, h, generator=g).to(dtype)
    w = (1 + 0.2 * torch.randn(h, generator=g)).to(wdtype or dtype)
    r = (torch.randn(t, h, generator=g) * 2).to(rdtype or dtype)
    return x, w, r


@pytest.mark.parametrize("t,h", [(1, 1), (3, 7), (1, 8), (2, 64), (5, 511), (5, 512), (4, 520),
                                 (7, 1024), (2, 1032), (3, 4096), (1, 4097), (2, 8192),
                                 (1, 16384), (2, 16392), (1, 65536), (600, 4096)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norm_and_residual(t, h, dtype):
    from treemoe_spec_amd.kernels.rms_norm import rms_norm

    _say(f"rms_norm t={t} h={h} {dtype}")
    x, w, r = _inputs(t, h, dtype, t * 131 + h)
    y = rms_norm(x.cuda(), w.cuda(), 1e-5)
    torch.cuda.synchronize()
    _near(y, _want(x, w, None, 1e-5)[0])
    y, s = rms_norm(x.cuda(), w.cuda(), 1e-6, residual=r.cuda())
    torch.cuda.synchronize()
    want, total = _want(x, w, r, 1e-6)
    # the sum itself is rounded to fp32 before it is squared or stored
    scale = (x.abs().double() + r.abs().double()) * U
    assert bool(((s.double().cpu() - total).abs()
                 <= total.abs() * torch.finfo(dtype).eps / 2 + scale).all())
    inv = (want / total.where(total != 0, torch.ones_like(total))).abs().amax(1, keepdim=True)
    got = y.double().cpu()
    bound = want.abs() * (torch.finfo(dtype).eps / 2 + 50 * U) + scale * inv \
        + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert bool(((got - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_float32_residual_and_weight(dtype):
    from treemoe_spec_amd.kernels.rms_norm import rms_norm

    _say(f"rms_norm fp32 residual {dtype}")
    x, w, r = _inputs(9, 1000, dtype, 5, torch.float32, torch.float32)
    y, s = rms_norm(x.cuda(), w.cuda(), residual=r.cuda())
    assert s.dtype == torch.float32 and y.dtype == dtype
    want, total = _want(x, w, r, 1e-5)
    assert torch.equal(s.cpu(), x.float() + r)
    assert bool(((y.double().cpu() - want).abs()
                 <= want.abs() * (torch.finfo(dtype).eps / 2 + 50 * U) + 4e-6).all())


def test_strides_and_in_place():
    """Rows of a wider buffer at an odd offset, a row stride of no multiple of 8,
    and outputs in the inputs' memory; nothing around the rows changes."""
    from treemoe_spec_amd.kernels.rms_norm import rms_norm

    for off, width in ((0, 1040), (8, 1040), (3, 1041)):
        _say(f"rms_norm strides off={off} width={width}")
        x, w, r = _inputs(6, 1024, torch.bfloat16, 11)
        plain_y, plain_s = rms_norm(x.cuda(), w.cuda(), residual=r.cuda())
        xb = torch.full((6, width), 7.0, dtype=torch.bfloat16, device="cuda")
        rb = torch.full((6, width), -3.0, dtype=torch.bfloat16, device="cuda")
        xs, rs = xb[:, off:off + 1024], rb[:, off:off + 1024]
        xs.copy_(x)
        rs.copy_(r)
        y, s = rms_norm(xs, w.cuda(), residual=rs, out=xs, residual_out=rs)
        torch.cuda.synchronize()
        assert y is xs and s is rs
        assert torch.equal(xs, plain_y) and torch.equal(rs, plain_s)
        keep = torch.ones(width, dtype=torch.bool)
        keep[off:off + 1024] = False
        assert bool((xb[:, keep.cuda()] == 7.0).all()) and bool((rb[:, keep.cuda()] == -3.0).all())


def test_zero_rows_and_no_rows():
    from treemoe_spec_amd.kernels.rms_norm import rms_norm, rms_norm_fp8

    _say("rms_norm zero rows")
    w = torch.ones(256, device="cuda", dtype=torch.bfloat16)
    z = torch.zeros(2, 256, device="cuda", dtype=torch.bfloat16)
    assert bool((rms_norm(z, w) == 0).all())
    q, sc = rms_norm_fp8(z, w, scale_group=64)
    assert bool((q.float() == 0).all()) and bool((sc == 1).all())
    assert rms_norm(z[:0], w).shape == (0, 256)
    q, sc = rms_norm_fp8(z[:0], w)
    assert q.shape == (0, 256) and sc.shape == (0,)


@pytest.mark.parametrize("t,h,group", [(1, 32, 32), (3, 4096, 128), (5, 4096, None), (2, 1000, None),
                                       (7, 77, None), (4, 512, 512), (3, 8192, 256), (2, 96, 32),
                                       (3, 16384, 64), (2, 20480, None)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_fp8(t, h, group, dtype):
    """Scales within 60 u of the formula's; every value within half an e4m3 step of
    the quotient by that scale (2^-4 of it, or half the subnormal step 2^-9),
    the quotient itself known to 120 u."""
    from treemoe_spec_amd.kernels.rms_norm import rms_norm_fp8

    _say(f"rms_norm_fp8 t={t} h={h} group={group} {dtype}")
    x, w, r = _inputs(t, h, dtype, t + h, rdtype=torch.float32)
    x[0, 0] = 30.0
    q, sc, s = rms_norm_fp8(x.cuda(), w.cuda(), residual=r.cuda(), scale_group=group)
    torch.cuda.synchronize()
    want, total = _want(x, w, r, 1e-5)
    assert torch.equal(s.cpu(), x.float() + r)
    step = group or h
    parts = want.view(t, -1, step)
    scale = parts.abs().amax(2) / 448
    sc = sc.cpu().double().view(t, -1)
    assert bool(((sc - scale).abs() <= scale * 60 * U + 1e-9).all())
    quot = parts / sc[:, :, None]
    got = q.cpu().float().double().view(t, -1, step)
    assert bool(((got - quot).abs() <= quot.abs() * (2.0 ** -4 + 120 * U) + 2.0 ** -10 + 2e-4).all())
    # the largest of every part is the type's largest value
    assert bool((got.abs().amax(2) == 448).all())


def test_non_finite_rows_stay_apart():
    """A NaN or an infinity spoils its own row (and its scale), no other."""
    from treemoe_spec_amd.kernels.rms_norm import rms_norm, rms_norm_fp8

    _say("rms_norm non-finite")
    x, w, _ = _inputs(6, 512, torch.float32, 3)
    clean = rms_norm(x.cuda(), w.cuda())
    x[1, 5], x[4, 100] = float("nan"), float("inf")
    y = rms_norm(x.cuda(), w.cuda())
    keep = torch.tensor([0, 2, 3, 5])
    assert torch.equal(y[keep], clean[keep]) and bool(y[1].isnan().all())
    q, sc = rms_norm_fp8(x.cuda(), w.cuda())
    assert bool(sc[1].isnan()) and bool(q[1].float().isnan().all())
    assert not bool(q[keep].float().isnan().any())


def test_another_stream_and_determinism():
    from treemoe_spec_amd.kernels.rms_norm import rms_norm

    _say("rms_norm stream")
    x, w, r = (t.cuda() for t in _inputs(2000, 4096, torch.bfloat16, 8))
    want = rms_norm(x, w, residual=r)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = rms_norm(x, w, residual=r)
    st.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
