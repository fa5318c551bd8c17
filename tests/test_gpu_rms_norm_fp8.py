"""rms_norm_fp8 where the normed rows are known in every bit: elements of +-1 have a mean
square of 1, so with eps = 0 a row's norm is the weight, and scales and values are the
float32 quotients, rounded to e4m3 once."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _say(msg):
    print(msg, flush=True)


def _signs(t, h, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 2, (t, h), generator=g) * 2 - 1).float()


def _want(y, step):
    parts = y.view(y.shape[0], -1, step)
    scale = parts.abs().amax(2) / 448
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    q = (parts / scale[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.view(y.shape).float(), scale


@pytest.mark.parametrize("t,h,group", [(3, 4096, 32), (1030, 1024, 128), (2, 512, None)])
def test_values_at_the_border_of_two_steps(t, h, group):
    """Quotients next to the middle between two e4m3 values."""
    from treemoe_spec_amd.kernels.rms_norm import rms_norm_fp8

    _say(f"rms_norm_fp8 borders t={t} h={h} group={group}")
    step = group or h
    grid = torch.arange(8, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    middle = (grid[:-1] + grid[1:]) / 2
    x = _signs(t, h, 1)
    for seed in range(6):
        g = torch.Generator().manual_seed(h + seed)
        w = middle[torch.randint(0, len(middle), (h // step, step), generator=g)]
        w[:, 0] = 448.0
        # times a scale of each group's own, rounded: the quotient is the middle or next to it
        w = (w * (1 + torch.rand(h // step, 1, generator=g))).view(h)
        want, scale = _want(x * w, step)
        q, sc = rms_norm_fp8(x.cuda(), w.cuda(), 0.0, scale_group=group)
        torch.cuda.synchronize()
        assert torch.equal(sc.cpu().view(t, -1), scale)
        assert torch.equal(q.float().cpu(), want)


@pytest.mark.parametrize("group", [32, None])
def test_magnitudes_whose_scale_underflows(group):
    """A largest magnitude that leaves 0 when divided by 448 has scale 1, like 0."""
    from treemoe_spec_amd.kernels.rms_norm import rms_norm_fp8

    _say(f"rms_norm_fp8 underflow group={group}")
    x = _signs(3, 256, 2)
    for top in (1.4e-45, 1e-43, 2.8e-43, 7e-43, 1e-40):
        w = torch.zeros(256)
        w[::7] = top
        want, scale = _want(x * w, group or 256)
        q, sc = rms_norm_fp8(x.cuda(), w.cuda(), 0.0, scale_group=group)
        torch.cuda.synchronize()
        assert torch.equal(sc.cpu().view(3, -1), scale)
        assert torch.equal(q.float().cpu(), want), top
