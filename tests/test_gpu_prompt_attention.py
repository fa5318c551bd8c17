"""prompt_attention and prompt_attention_cached on the GPU against attention in 64 bits.

Tolerances, for weights w_j summing to 1 over values v_j.  With e = half a step of
the 16-bit type (bf16 2^-8, fp16 2^-11) and u = 2^-24:
  scores    hd products summed in fp32: off by at most (hd + 2) u sum |q_i k_i| scale,
            bounded below by ds = 130 u scale max|q| max|k| hd: a relative error
            of every weight of 2 ds;
  weights   rounded to the type once, e each, above and below the division alike;
            exp2 and its argument: 4 u and 32 u (a base-2 argument up to 2^5 in
            size; smaller weights do not count);
  sums      in fp32: (keys / 16 + 64) u at most, taken as 600 u;
  output    e of itself.
|got - want| <= e |want| + (2 e + 2 ds + 640 u) sum_j w_j |v_j| (numerator and
denominator rounded apart) + the type's smallest subnormal."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _say(msg):
    print(msg, flush=True)


def _want(q, k, v, past, scale):
    """Context and sum_j w_j |v_j| [T, Hq * hd] in 64 bits."""
    t, hq, hd = q.shape
    s, kvh, _ = k.shape
    seen = torch.arange(s)[None] <= torch.arange(t)[:, None] + past
    outs, mags = [], []
    for h in range(hq):
        a = q[:, h].double() @ k[:, h * kvh // hq].double().T * scale
        w = torch.softmax(a.masked_fill(~seen, -float("inf")), 1)
        vv = v[:, h * kvh // hq].double()
        outs.append(w @ vv)
        mags.append(w @ vv.abs())
    return torch.stack(outs, 1).flatten(1), torch.stack(mags, 1).flatten(1)


def _check(got, q, k, v, past, scale=None):
    hd = q.shape[2]
    scale = hd ** -0.5 if scale is None else scale
    want, mag = _want(q, k, v, past, scale)
    info = torch.finfo(q.dtype)
    e = info.eps / 2
    ds = 130 * U * scale * float(q.abs().max()) * float(k.abs().max()) * hd
    bound = e * want.abs() + (2 * e + 2 * ds + 640 * U) * mag + info.smallest_normal * info.eps
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (off[bad][:4], bound[bad][:4], bad.nonzero()[:4])


def _qkv(t, s, hq, kvh, hd, dtype, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn(t, hq, hd, generator=g) * scale).to(dtype),
            torch.randn(s, kvh, hd, generator=g).to(dtype),
            torch.randn(s, kvh, hd, generator=g).to(dtype))


def _packed(q_lens, k_lens, hq, kvh, hd, dtype, seed, chunk=None):
    from treemoe_spec_amd.kernels.prompt_attention import PromptPlan, prompt_attention

    q, k, v = _qkv(sum(q_lens), sum(k_lens), hq, kvh, hd, dtype, seed)
    plan = PromptPlan(q_lens, k_lens, num_heads=hq, num_kv_heads=kvh)
    out = prompt_attention(q.cuda(), k.cuda(), v.cuda(), plan)
    torch.cuda.synchronize()
    q0 = k0 = 0
    for nq, nk in zip(q_lens, k_lens):
        if nq:
            _check(out[q0:q0 + nq], q[q0:q0 + nq], k[k0:k0 + nk], v[k0:k0 + nk], nk - nq)
        q0, k0 = q0 + nq, k0 + nk
    return out


@pytest.mark.parametrize("hq,kvh,hd", [(32, 8, 128), (8, 2, 64), (4, 4, 128), (3, 1, 64),
                                       (16, 2, 128), (7, 1, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t", [1, 2, 31, 32, 33, 63, 64, 65, 129, 257])
def test_one_prompt(t, hq, kvh, hd, dtype):
    _say(f"prompt t={t} heads={hq}/{kvh} hd={hd} {dtype}")
    _packed([t], [t], hq, kvh, hd, dtype, t * 7 + hd)


@pytest.mark.parametrize("q_lens,k_lens", [
    ([5, 1, 0, 130, 64], [5, 1, 0, 130, 64]),
    ([1, 1, 1, 1], [1, 64, 65, 1000]),
    ([17, 40, 3], [300, 40, 67]),
    ([0, 0], [0, 9]),
    ([1] * 40, list(range(1, 41))),
    ([200], [3000]),
])
@pytest.mark.parametrize("hq,kvh,hd", [(8, 2, 128), (4, 4, 64)])
def test_packed(q_lens, k_lens, hq, kvh, hd):
    _say(f"packed {q_lens[:6]} over {k_lens[:6]} heads={hq}/{kvh} hd={hd}")
    _packed(q_lens, k_lens, hq, kvh, hd, torch.bfloat16, len(q_lens) + hd)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_tiles(dtype):
    """Large batches: several tiles a compute unit."""
    _say(f"large tiles {dtype}")
    lens = [1900, 2300, 777]
    _packed(lens, lens, 64, 16, 64, dtype, 5)
    lens = [900, 2, 4000, 0, 3400]
    _packed(lens, lens, 32, 8, 128, dtype, 6)


@pytest.mark.parametrize("q_lens,k_lens,hq,kvh,tiling", [
    ([7, 1, 0], [100, 1, 0], 8, 2, 0),
    ([8] * 3, [3000, 8, 8], 8, 2, 0),
    ([9, 300], [9, 300], 8, 2, 1),
    ([60] * 100, [60] * 100, 8, 2, 1),
    ([700, 3], [1300, 900], 8, 2, 2),
    ([3500, 4000, 1], [3500, 4100, 4000], 32, 8, 3),
    ([60] * 100 + [1], [60] * 100 + [50000], 8, 2, 1),   # short and tall tiles with joins
    ([4000, 1], [4000, 100000], 32, 8, 3),
])
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_every_tiling(q_lens, k_lens, hq, kvh, tiling, dtype, hd):
    """Few rows, short, pair and tall tiles, each with a sequence that leaves parts of
    its tiles without rows."""
    from treemoe_spec_amd.kernels.prompt_attention import PromptPlan

    _say(f"tiling {tiling} {dtype} hd={hd}")
    assert PromptPlan(q_lens, k_lens, num_heads=hq, num_kv_heads=kvh).tiling == tiling
    _packed(q_lens, k_lens, hq, kvh, hd, dtype, tiling + hd)


def _cache(s, kvh, hd, dtype, page, seed, layers=2):
    from treemoe_spec_amd.kv_cache import MixtralConfig, PagedKVCache

    g = torch.Generator().manual_seed(seed)
    cfg = MixtralConfig(num_layers=layers, num_kv_heads=kvh, head_dim=hd)
    kv = PagedKVCache(cfg, (s + page - 1) // page + 5, device="cuda", dtype=dtype,
                      page_size=page, tree_size=1)
    kv.k.fill_(float("nan"))   # what was never written
    kv.v.fill_(float("nan"))
    perm = torch.randperm(len(kv._free), generator=g).tolist()
    kv._free = [kv._free[i] for i in perm]
    return kv


@pytest.mark.parametrize("t,s,page", [(1, 1, 16), (1, 5, 16), (1, 64, 16), (1, 65, 64),
                                      (1, 7777, 16), (2, 1000, 64), (63, 64, 16), (64, 64, 1),
                                      (100, 2500, 16), (517, 1100, 64), (700, 700, 256), (520, 3600, 16)])
@pytest.mark.parametrize("hq,kvh,hd,dtype", [(32, 8, 128, torch.bfloat16),
                                             (8, 2, 64, torch.float16)])
def test_cached(t, s, page, hq, kvh, hd, dtype):
    """Keys read through the block table; slots behind the sequence hold NaN."""
    from treemoe_spec_amd.kernels.prompt_attention import prompt_attention_cached

    _say(f"cached t={t} s={s} page={page} heads={hq}/{kvh} hd={hd} {dtype}")
    q, k, v = _qkv(t, s, hq, kvh, hd, dtype, t + s)
    kv = _cache(s, kvh, hd, dtype, page, s)
    kv.append(1, k.cuda(), v.cuda(), 0)
    out = prompt_attention_cached(q.cuda(), kv, 1)
    torch.cuda.synchronize()
    _check(out, q, k, v, s - t)
    kv2 = _cache(s, kvh, hd, dtype, page, s)
    kv2.append(0, k.cuda(), v.cuda(), 0)
    assert torch.equal(prompt_attention_cached(q.cuda(), kv2, -2), out)


def test_bad_pages_read_inside_the_cache():
    """Block table entries outside the cache read some page of it, no other memory."""
    from treemoe_spec_amd.kernels.prompt_attention import prompt_attention_cached

    _say("cached bad pages")
    q, k, v = _qkv(20, 40, 8, 2, 128, torch.bfloat16, 3)
    kv = _cache(40, 2, 128, torch.bfloat16, 16, 3)
    kv.k.fill_(1.0)
    kv.v.fill_(1.0)
    kv.block_table, kv.seq_len = [-5, 1 << 30, 2], 40
    out = prompt_attention_cached(q.cuda(), kv, 0)
    assert bool((out == 1.0).all())


def test_strides_scale_and_rows_behind():
    """q, k, v as views of one projection, a scale of one's own, and a padded batch."""
    from treemoe_spec_amd.kernels.prompt_attention import PromptPlan, prompt_attention

    _say("prompt strides")
    lens = [50, 0, 80]
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(140, 12 * 64, generator=g).to(torch.bfloat16)
    dev = qkv.cuda()
    q, k, v = (x.unflatten(1, (-1, 64)) for x in dev.split([8 * 64, 2 * 64, 2 * 64], 1))
    plan = PromptPlan(lens, num_heads=8, num_kv_heads=2)
    buf = torch.full((140, 600), 3.0, dtype=torch.bfloat16, device="cuda")
    out = prompt_attention(q, k, v, plan, scale=0.3, out=buf[:, 8:520])
    torch.cuda.synchronize()
    cq, ck, cv = (x.cpu() for x in (q, k, v))
    _check(out[:50], cq[:50], ck[:50], cv[:50], 0, 0.3)
    _check(out[50:130], cq[50:130], ck[50:130], cv[50:130], 0, 0.3)
    assert bool((buf[130:] == 3).all()) and bool((buf[:, :8] == 3).all()) \
        and bool((buf[:, 520:] == 3).all())
    assert bool((prompt_attention(q, k, v, plan, scale=0.3)[130:] == 0).all())
    assert prompt_attention(q, k, v, PromptPlan([], num_heads=8, num_kv_heads=2)).shape == (140, 512)


def test_large_scores():
    """Scores of hundreds: the running reference moves many times."""
    _say("prompt large scores")
    from treemoe_spec_amd.kernels.prompt_attention import PromptPlan, prompt_attention

    q, k, v = _qkv(300, 300, 4, 2, 128, torch.float16, 8, scale=1.0)
    k = (k.float() * torch.linspace(0.1, 30.0, 300)[:, None, None]).to(torch.float16)
    plan = PromptPlan([300], num_heads=4, num_kv_heads=2)
    out = prompt_attention(q.cuda(), k.cuda(), v.cuda(), plan)
    _check(out, q, k, v, 0)


def test_same_on_every_run_and_another_stream():
    from treemoe_spec_amd.kernels.prompt_attention import (PromptPlan, prompt_attention,
                                                           prompt_attention_cached)

    _say("prompt determinism")
    q, k, v = (x.cuda() for x in _qkv(600, 3000, 32, 8, 128, torch.bfloat16, 9))
    plan = PromptPlan([600], [3000], num_heads=32, num_kv_heads=8)
    kv = _cache(3000, 8, 128, torch.bfloat16, 16, 9)
    kv.append(0, k, v, 0)
    want, wantc = prompt_attention(q, k, v, plan), prompt_attention_cached(q, kv, 0)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(st):
            a, b = prompt_attention(q, k, v, plan), prompt_attention_cached(q, kv, 0)
        st.synchronize()
        assert torch.equal(a, want) and torch.equal(b, wantc)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("t,past,hd", [(70, 0, 128), (3, 900, 128), (300, 200, 64)])
def test_what_a_row_does_not_see_does_not_reach_it(bad, t, past, hd):
    """NaN and infinities in the keys and values of later tokens, and of the next
    sequence: the rows before them are what they are without, rows that see one
    are what the formula gives."""
    from treemoe_spec_amd.kernels.prompt_attention import (PromptPlan, prompt_attention,
                                                           prompt_attention_cached)

    _say(f"prompt non-finite {bad} t={t} past={past}")
    s, n = t + past, 40
    q, k, v = _qkv(t + n, s + n, 4, 2, hd, torch.bfloat16, t)
    plan = PromptPlan([t, n], [s, n], num_heads=4, num_kv_heads=2)
    clean = prompt_attention(q.cuda(), k.cuda(), v.cuda(), plan)
    hit = s - max(1, t // 3)            # a key that the last third sees
    first = hit - past                  # and its query
    for where in (k, v):
        kk, vv = k.clone(), v.clone()
        (kk if where is k else vv)[hit, :, 5] = bad
        (kk if where is k else vv)[s + 7] = bad
        out = prompt_attention(q.cuda(), kk.cuda(), vv.cuda(), plan)
        kv = _cache(s, 2, hd, torch.bfloat16, 16, s)
        kv.append(0, kk[:s].cuda(), vv[:s].cuda(), 0)
        outc = prompt_attention_cached(q[:t].cuda(), kv, 0)
        torch.cuda.synchronize()
        for got in (out[:t], outc):
            _check(got[:first], q[:first], k, v, past)
            if where is v:
                # column 5 of every head is the bad value, the others as without it
                g = got[first:].view(-1, 4, hd).cpu().float()
                c = clean[first:t].view(-1, 4, hd).cpu().float()
                assert bool((g[..., 5] == bad).all()) if bad == bad else bool(g[..., 5].isnan().all())
                rest = torch.arange(hd) != 5
                assert float((g - c)[..., rest].norm()) <= 8e-3 * float(c[..., rest].norm())
        _check(out[t:t + 7], q[t:t + 7], k[s:s + 7], v[s:s + 7], 0)


def test_overflowing_scores_and_rows_of_nan():
    """A query of NaN spoils its own row; others of its tile stay."""
    from treemoe_spec_amd.kernels.prompt_attention import PromptPlan, prompt_attention

    _say("prompt NaN query")
    q, k, v = _qkv(90, 90, 4, 2, 128, torch.float16, 4)
    q[33] = float("nan")
    plan = PromptPlan([90], num_heads=4, num_kv_heads=2)
    out = prompt_attention(q.cuda(), k.cuda(), v.cuda(), plan)
    assert bool(out[33].isnan().all())
    q[33] = 0
    keep = [i for i in range(90) if i != 33]
    want, mag = _want(q, k, v, 0, 128 ** -0.5)
    assert not bool(out[keep].isnan().any())
    assert float((out[keep].double().cpu() - want[keep]).norm()) <= 2e-3 * float(want[keep].norm())
