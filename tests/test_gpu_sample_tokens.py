"""sample_tokens on the GPU against the definition in 64 bits (Python and numpy,
row by row).  Tokens are equal wherever the uniform number lies further than 1e-9
of the total from the border of two tokens (the kernel's weights are multiples of
2^-44, V / 2 of them off at most 2^18 2^-45 = 7.5e-9 of the largest in sum;
measured against sums of at least 1); probabilities within 2^-23 of their value
plus 2^-44."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _say(msg):
    print(msg, flush=True)


def _oracle(logits, u, temperature, top_k, top_p, min_p):
    """(token, probs, distance of u's target to the nearest border) of one row."""
    l = logits.astype(np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    v = len(l)
    if l.max() == -np.inf:
        return -1, np.zeros(v), 1.0
    if temperature == 0:
        p = np.zeros(v)
        p[int(l.argmax())] = 1
        return int(l.argmax()), p, 1.0
    with np.errstate(invalid="ignore"):
        z = np.where(l == l.max(), 0.0, (l - l.max()) / temperature)
    w = np.exp(z)
    order = np.lexsort((np.arange(v), -l))
    if 0 < top_k < v:
        order = order[:top_k]
    if top_p < 1:
        c = np.cumsum(w[order])
        n = int(np.searchsorted(c, top_p * c[-1], side="left")) + 1
        order = order[:max(1, min(n, len(order)))]
    order = order[w[order] >= min_p]
    kept = np.zeros(v)
    kept[order] = w[order]
    run = np.cumsum(kept)
    token = int(np.searchsorted(run, u * run[-1], side="right"))
    gap = np.abs(run - u * run[-1]).min() / run[-1]
    return token, kept / run[-1], gap


def _check(logits, u, got, probs=None, **kw):
    per = lambda x, r: x[r].item() if isinstance(x, torch.Tensor) else x  # noqa: E731
    for r in range(logits.shape[0]):
        args = [per(kw.get(n, d), r) for n, d in (("temperature", 1.0), ("top_k", 0),
                                                  ("top_p", 1.0), ("min_p", 0.0))]
        token, p, gap = _oracle(logits[r].float().numpy(), float(u[r]), *args)
        if probs is not None:
            off = np.abs(probs[r].double().cpu().numpy() - p)
            assert (off <= p * 2.0 ** -23 + 2.0 ** -44).all(), (r, off.max())
        assert int(got[r]) == token or gap < 1e-8, (r, int(got[r]), token, gap)


def _logits(n, v, dtype, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, v, generator=g) * scale).to(dtype), torch.rand(n, generator=g)


@pytest.mark.parametrize("n,v", [(1, 1), (3, 2), (2, 63), (5, 1000), (4, 4096), (3, 4099),
                                 (4, 32000), (2, 32768), (2, 32769), (2, 131072), (1, 262144)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", [{}, {"top_k": 50}, {"top_p": 0.9}, {"min_p": 0.05},
                                {"temperature": 0.6, "top_k": 200, "top_p": 0.8, "min_p": 0.01},
                                {"temperature": 0.0}])
def test_against_the_definition(n, v, dtype, kw):
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    _say(f"sample n={n} v={v} {dtype} {kw}")
    logits, u = _logits(n, v, dtype, n * 7 + v)
    got, probs = sample_tokens(logits.cuda(), u.cuda(), return_probs=True, **kw)
    torch.cuda.synchronize()
    _check(logits, u, got, probs, **kw)
    assert torch.equal(sample_tokens(logits.cuda(), u.cuda(), **kw), got)


@pytest.mark.parametrize("kw", [{"top_k": 1}, {"top_k": 7}, {"top_k": 999}, {"top_k": 5000},
                                {"top_p": 0.0}, {"top_p": 1e-6}, {"top_p": 0.5}, {"min_p": 1.0},
                                {"top_k": 300, "top_p": 0.31}])
def test_ties_go_to_the_lowest_index(kw):
    """Few distinct values: the cut falls inside groups of equal logits."""
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    _say(f"sample ties {kw}")
    g = torch.Generator().manual_seed(4)
    rows = [torch.zeros(3001), torch.randint(0, 3, (3001,), generator=g).float(),
            torch.randint(-2, 3, (3001,), generator=g).float() * 1e-3,
            torch.where(torch.rand(3001, generator=g) < 0.5, 0.0, -0.0)]
    logits, u = torch.stack(rows), torch.tensor([0.0, 0.999, 0.5, 0.3])
    got, probs = sample_tokens(logits.cuda(), u.cuda(), return_probs=True, **kw)
    _check(logits, u, got, probs, **kw)


def test_one_parameter_a_row():
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    _say("sample per-row parameters")
    logits, u = _logits(6, 5000, torch.float32, 9)
    kw = {"temperature": torch.tensor([0.0, 0.25, 1.0, 2.0, 1.0, 0.7]),
          "top_k": torch.tensor([0, 10, 0, 5000, 9999, 1], dtype=torch.int32),
          "top_p": torch.tensor([0.5, 1.0, 0.25, 0.75, 0.0, 0.5]),
          "min_p": torch.tensor([0.0, 0.125, 0.0, 0.0, 0.25, 1.0])}
    got, probs = sample_tokens(logits.cuda(), u.cuda(), return_probs=True,
                               **{k: x.cuda() for k, x in kw.items()})
    _check(logits, u, got, probs, **kw)


def test_row_values_out_of_range_act_as_the_nearest():
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    _say("sample clamped parameters")
    logits, u = _logits(4, 2000, torch.float32, 10)
    nan = float("nan")
    bad = {"temperature": [-1.0, 1.0, 1.0, 1.0], "top_k": [0, -5, 0, 0],
           "top_p": [1.0, 7.0, -1.0, nan], "min_p": [0.0, -2.0, 5.0, nan]}
    good = {"temperature": [0.0, 1.0, 1.0, 1.0], "top_k": [0, 0, 0, 0],
            "top_p": [1.0, 1.0, 0.0, 1.0], "min_p": [0.0, 0.0, 1.0, 0.0]}
    out = []
    for kw in (bad, good):
        kw = {k: torch.tensor(x, dtype=torch.int32 if k == "top_k" else torch.float32).cuda()
              for k, x in kw.items()}
        out.append(sample_tokens(logits.cuda(), u.cuda(), return_probs=True, **kw))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


@pytest.mark.parametrize("v", [3000, 40000])
def test_non_finite_logits(v):
    """-inf and NaN are never taken; +inf takes everything; nothing left is -1."""
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    _say(f"sample non-finite v={v}")
    logits, _ = _logits(6, v, torch.float32, 12)
    inf, nan = float("inf"), float("nan")
    logits[0, ::2] = nan
    logits[1, 1:] = -inf
    logits[2] = -inf
    logits[3, [5, 17]] = inf
    logits[4] = nan
    logits[5, :] = torch.finfo(torch.float32).min
    logits[5, 9] = -1e38
    u = torch.tensor([0.3, 0.9, 0.5, 0.6, 0.2, 0.99])
    for kw in ({}, {"top_k": 3}, {"top_p": 0.9}):
        got, probs = sample_tokens(logits.cuda(), u.cuda(), return_probs=True, **kw)
        _check(logits, u, got, probs, **kw)
        assert got.tolist()[1:] == [0, -1, 17, -1, 9]
        assert bool((probs[2] == 0).all()) and not bool(probs.isnan().any())


def test_uniforms_at_the_ends():
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    _say("sample uniforms at the ends")
    logits = torch.zeros(6, 100)
    logits[:, :3] = -float("inf")
    logits[:, 97:] = -float("inf")
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan")])
    got = sample_tokens(logits.cuda(), u.cuda())
    assert got.tolist() == [3, 96, 96, 96, 3, 3]


def test_strides_and_rows_of_a_buffer():
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    _say("sample strides")
    logits, u = _logits(5, 4001, torch.bfloat16, 13)
    want = sample_tokens(logits.cuda(), u.cuda(), top_p=0.9, return_probs=True)
    buf = torch.zeros(5, 4100, dtype=torch.bfloat16, device="cuda")
    view = buf[:, 33:33 + 4001]
    view.copy_(logits)
    out = torch.full((5, 4010), 5.0, device="cuda")
    got = sample_tokens(view, u.cuda(), top_p=0.9, return_probs=True, probs_out=out[:, 3:4004])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert bool((out[:, :3] == 5).all()) and bool((out[:, 4004:] == 5).all())
    # one row of logits for every uniform number
    same = sample_tokens(logits[:1].cuda().expand(5, -1), u.cuda())
    each = sample_tokens(logits[:1].repeat(5, 1).cuda(), u.cuda())
    assert torch.equal(same, each)
    assert sample_tokens(logits[:0].cuda(), u[:0].cuda()).shape == (0,)


def test_frequencies():
    """20000 draws of a 5-token row: every share within 5 standard deviations."""
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    _say("sample frequencies")
    row = torch.tensor([0.5, -1.0, 2.0, 0.0, 1.0])
    n = 20000
    u = torch.rand(n, generator=torch.Generator().manual_seed(1))
    got = sample_tokens(row.cuda().expand(n, -1), u.cuda())
    p = torch.softmax(row.double(), 0)
    share = torch.bincount(got.cpu(), minlength=5) / n
    assert bool(((share - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all())


@pytest.mark.parametrize("v", [32000, 100001])
@pytest.mark.parametrize("kw", [{"top_k": 2000}, {"top_k": 30000, "top_p": 0.7}, {"top_p": 0.5},
                                {"top_p": 0.97, "min_p": 0.3}])
def test_flat_rows(v, kw):
    """Cuts through thousands of equal or nearly equal logits, more than a list holds,
    and through rows that a list of the cut's step serves."""
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    _say(f"sample flat v={v} {kw}")
    g = torch.Generator().manual_seed(v)
    rows = [torch.zeros(v), torch.randint(0, 3, (v,), generator=g).float(),
            torch.randn(v, generator=g) * 0.01, torch.randn(v, generator=g),
            torch.randn(v, generator=g) * 2]
    logits, u = torch.stack(rows), torch.rand(len(rows), generator=g)
    got, probs = sample_tokens(logits.cuda(), u.cuda(), return_probs=True, **kw)
    torch.cuda.synchronize()
    _check(logits, u, got, probs, **kw)
