"""beam_select and reorder_rows on the GPU against their definition in 64 bits on the CPU.

Scores are sums of 64-bit terms: those here and there are off by a few 2^-53 of the largest
term, far below the distance of candidates of unlike logits, so parents and tokens have to be
equal.  The written score is rounded once to fp32: off by 2^-24 of itself, and 2^-40
covers the 64-bit terms (|score| < 2^10)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")


def _say(msg):
    print(msg, flush=True)


def _want(logits, scores, num, finished=None, pad=0):
    """(scores in 64 bits, parents, tokens), candidate by candidate."""
    groups, beams = scores.shape
    rows = logits.double().view(groups, beams, -1)
    out_s = torch.full((groups, num), -INF, dtype=torch.float64)
    out_p = torch.full((groups, num), -1, dtype=torch.int32)
    out_t = torch.full((groups, num), -1, dtype=torch.int64)
    for g in range(groups):
        found = []
        for b in range(beams):
            s = float(scores[g, b])
            if not s > -INF:
                continue
            if finished is not None and bool(finished[g, b]):
                found.append((s, b, 0.0, pad))
                continue
            x = rows[g, b].clone()
            x[x.isnan()] = -INF
            top = float(x.max())
            if top == -INF:
                continue
            if top == INF:
                x = torch.where(x == INF, 0.0, -INF).double()
            z = x - x.max()
            z = z - z.exp().sum().log()
            order = torch.sort(z, descending=True, stable=True).indices[:num].tolist()
            found += [(s + float(z[v]), b, float(x[v]), v) for v in order if z[v] > -INF]
        found.sort(key=lambda c: (-c[0], c[1], -c[2], c[3]))
        for i, (s, b, _, v) in enumerate(found[:num]):
            out_s[g, i], out_p[g, i], out_t[g, i] = s, b, v
    return out_s, out_p, out_t


def _check(logits, scores, num=None, finished=None, pad=0, dev_logits=None):
    from treemoe_spec_amd.kernels.beam_search import beam_select

    n = scores.shape[1] if num is None else num
    got = beam_select(logits.cuda() if dev_logits is None else dev_logits, scores.cuda(), num=num,
                      finished=None if finished is None else finished.cuda(), pad_token=pad)
    torch.cuda.synchronize()
    want = _want(logits, scores, n, finished, pad)
    s, p, t = (x.cpu() for x in got)
    assert s.dtype == F32 and p.dtype == torch.int32 and t.dtype == torch.int64
    assert torch.equal(p, want[1]), (p, want[1])
    assert torch.equal(t, want[2]), (t, want[2])
    live = want[0] > -INF
    off = (s.double() - want[0])[live].abs()
    assert bool((off <= want[0][live].abs() * 2.0 ** -24 + 2.0 ** -40).all())
    assert bool((s[~live] == -INF).all())
    return got


def _inputs(groups, beams, v, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(groups * beams, v, generator=g) * spread).to(dtype)
    return logits, -5.0 * torch.rand(groups, beams, generator=g)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("groups,beams,num", [(1, 1, 1), (1, 4, 8), (3, 2, 4), (2, 5, 5),
                                              (1, 64, 64), (5, 7, 14)])
@pytest.mark.parametrize("v", [1, 3, 63, 1000, 1024, 1025, 4096, 32000])
def test_select(groups, beams, num, v, dtype):
    _say(f"beam_select {groups}x{beams} num {num} of {v} {dtype}")
    _check(*_inputs(groups, beams, v, dtype, v + beams), num)


@pytest.mark.parametrize("v", [131072, 131073, 262144])
@pytest.mark.parametrize("beams,num", [(8, 16), (40, 64)])
def test_large_vocabularies(v, beams, num):
    """More lists than the group's workgroup has threads."""
    _say(f"beam_select {beams} num {num} of {v}")
    _check(*_inputs(1, beams, v, BF, v), num)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("groups,beams,v", [(64, 8, 300), (33, 8, 8193), (130, 4, 4096)])
@pytest.mark.parametrize("num", [1, 16, 17, 64])
def test_many_rows(groups, beams, v, num, dtype):
    """Rows that fill the chip; few lists for many to come out; logits of few values, and in
    order, so that a few threads have all of the largest."""
    _say(f"beam_select {groups}x{beams} num {num} of {v} {dtype}")
    logits, scores = _inputs(groups, beams, v, dtype, num)
    logits[1::5] = (logits[1::5] / 4).round()
    logits[2::5] = logits[2::5].sort(descending=True).values
    logits[3::5] = logits[3::5].sort().values
    logits[4, 7:] = -INF
    _check(logits, scores, num)


@pytest.mark.parametrize("num", [1, 8, 64])
def test_flat_and_tied_rows(num):
    """All logits equal, or of few values: the lower beam and the lower token first."""
    _say(f"beam_select ties num {num}")
    _check(torch.zeros(8, 5000, dtype=BF), torch.zeros(2, 4), num)
    _check(torch.zeros(64, 2048, dtype=F32), torch.zeros(1, 64), num)
    g = torch.Generator().manual_seed(num)
    few = torch.randint(0, 3, (4, 9000), generator=g).to(F16)
    _check(few, torch.zeros(1, 4), num)
    _check(few[:1].repeat(4, 1), torch.tensor([[-1.0, -1.0, 0.0, 0.0]]), num)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_rows_with_little_in_them(dtype):
    """-inf but for a few, all -inf, NaN, infinities, dead beams."""
    _say(f"beam_select masked rows {dtype}")
    logits, scores = _inputs(4, 3, 3000, dtype, 5)
    logits[0, :] = -INF                  # a beam without candidates
    logits[1, 5:] = -INF
    logits[3:6, :] = -INF                # a group without any
    logits[6, 100] = NAN
    logits[7, 2999] = INF
    logits[7, 7] = INF                   # two that share the weight
    logits[8, 1] = torch.finfo(dtype).min
    logits[9, :] = torch.finfo(dtype).min
    logits[10, :] = NAN
    scores[2, 0] = -INF
    scores[3, 2] = NAN
    for num in (1, 4, 64):
        _check(logits, scores, num)


def test_first_step():
    """All beams alike, all but one without a score."""
    _say("beam_select first step")
    logits, _ = _inputs(1, 1, 32000, F32, 6)
    scores = torch.full((1, 5), -INF)
    scores[0, 0] = 0.0
    _check(logits.repeat(5, 1), scores, 10)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_finished(dtype):
    _say(f"beam_select finished {dtype}")
    logits, scores = _inputs(4, 4, 2500, dtype, 7)
    finished = torch.tensor([[1, 0, 0, 1], [1, 1, 1, 1], [0, 0, 0, 0], [0, 1, 0, 0]]).bool()
    scores[3, 1] = -INF
    scores[0, 0] = scores[0, 3]
    logits[finished.view(-1)] = NAN      # of finished beams nothing is read
    for num in (1, 3, 4, 8):
        _check(logits, scores, num, finished, pad=17)


def test_strides():
    """Rows at other strides, that do not start on 16 bytes."""
    _say("beam_select strides")
    for dtype, width, lo in ((F32, 2051, 1), (BF, 2057, 3), (BF, 2064, 8), (F16, 4097, 0)):
        logits, scores = _inputs(2, 3, width, dtype, width)
        _check(logits[:, lo:lo + 2000], scores, 6, dev_logits=logits.cuda()[:, lo:lo + 2000])


def test_close_scores_across_beams():
    """Candidates of two beams 2^-33 apart, which fp32 would not tell."""
    _say("beam_select close scores")
    logits = torch.zeros(2, 4096, dtype=F32)
    logits[:, 1234] = 12.0
    logits[0, 77] = 2.0 ** -20           # beam 0's sum is larger by 2^-20 of some 166850
    _check(logits, torch.zeros(1, 2), 4)


def test_repeated_calls_are_equal():
    from treemoe_spec_amd.kernels.beam_search import beam_select

    _say("beam_select again")
    logits, scores = (x.cuda() for x in _inputs(6, 8, 32000, BF, 9))
    first = beam_select(logits, scores, num=16)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, beam_select(logits, scores, num=16)))


# ------------------------------------------------------------ reorder_rows --

def _moved(x, parents):
    groups, beams = parents.shape
    own = torch.arange(beams).expand(groups, beams)
    at = torch.where((parents >= 0) & (parents < beams), parents.long(), own)
    return x[(at + beams * torch.arange(groups)[:, None]).flatten()]


@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 2), (3, 4), (2, 7), (1, 64), (9, 16)])
@pytest.mark.parametrize("shape,dtype", [((1,), torch.int64), ((300,), torch.int32),
                                         ((5, 7), torch.bool), ((1000, 3), BF), ((4099,), F32),
                                         ((), torch.int64), ((2, 8, 64), F16)])
@pytest.mark.parametrize("same", [False, True])
def test_reorder(groups, beams, shape, dtype, same):
    from treemoe_spec_amd.kernels.beam_search import reorder_rows

    _say(f"reorder {groups}x{beams} of {shape} {dtype} same={same}")
    g = torch.Generator().manual_seed(beams)
    x = torch.randint(0, 100, (groups * beams, *shape), generator=g).to(dtype)
    for lo, hi in ((0, beams), (-1, beams + 1), (0, 1)):
        parents = torch.randint(lo, hi, (groups, beams), generator=g, dtype=torch.int32)
        dev = x.cuda()
        got = reorder_rows(dev, parents.cuda(), out=dev if same else None)
        assert (got is dev) == same
        assert torch.equal(got.cpu(), _moved(x, parents))
        if not same:
            assert torch.equal(dev.cpu(), x)


def test_reorder_columns_and_strides():
    from treemoe_spec_amd.kernels.beam_search import reorder_rows

    _say("reorder columns, strided rows and parents")
    g = torch.Generator().manual_seed(3)
    x = torch.randint(0, 1000, (12, 64), generator=g, dtype=torch.int32)
    parents = torch.randint(0, 4, (3, 9), generator=g, dtype=torch.int32)
    dev, far = x.cuda(), parents.cuda()[:, :4]
    for cols in (0, 1, 17, 64):
        out = torch.full_like(dev, -7)
        assert reorder_rows(dev, far, out=out, columns=cols) is out
        assert torch.equal(out[:, :cols].cpu(), _moved(x, parents[:, :4])[:, :cols])
        assert bool((out[:, cols:] == -7).all())
    view = dev[:, 3:40]
    want = x.clone()
    want[:, 3:40] = _moved(x, parents[:, :4])[:, 3:40]
    reorder_rows(view, far, out=view)
    assert torch.equal(dev.cpu(), want)
    assert reorder_rows(dev[:0], far[:0]).shape == (0, 64)
