"""attention_mass and evict on the GPU against their definitions in 64 bits on the CPU.

Tolerance of the mass, with u = 2^-24: a score is a sum of hd products in fp32, off by ds =
(hd + 2) u scale max|q| max|k| hd at most (as in test_gpu_prompt_attention), a relative error
of 2 ds of a weight, for the score and for the row's sum; exp2, its argument (up to 2^6 in
size), the sum over the keys of a lane and the quotient: 8 + 64 + 600 u; the sum over a
key's rows, all positive: 64 u for what a lane adds, the waves and `before`.  Weights below
2^-100 may be lost: 2^-90 covers 2^10 of them.

Evictions move bytes: keys, values, masses and positions are equal."""

from __future__ import annotations

import pytest
import torch

from tests import test_gpu_prompt_attention as t_attn

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")
U = 2.0 ** -24


def _say(msg):
    print(msg, flush=True)


def _want(q, k, scale):
    t, hq, hd = q.shape
    n, kvh, _ = k.shape
    seen = torch.arange(n)[None] <= torch.arange(t)[:, None] + n - t
    got = torch.zeros(kvh, n, dtype=torch.float64)
    for h in range(hq):
        a = q[:, h].double() @ k[:, h * kvh // hq].double().T * scale
        w = torch.softmax(a.masked_fill(~seen, -INF), 1)
        got[h * kvh // hq] += torch.where((a.masked_fill(~seen, -INF) == -INF).all(1, True), 0.0,
                                          w).sum(0)
    return got


def _check(got, q, k, before=None, scale=None):
    hd = q.shape[2]
    scale = hd ** -0.5 if scale is None else scale
    want = _want(q, k, scale)
    ds = 130 * U * scale * float(q.abs().max()) * float(k.abs().max()) * hd
    bound = (2 * ds + 736 * U) * want + 2.0 ** -90
    if before is not None:
        want = want + before.double()
        bound = bound + U * want.abs()
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), (off.max(), (off / bound).max())


def _mass(t, n, hq, kvh, hd, dtype, page, seed, scale=None, add=False, q_scale=2.0):
    from treemoe_spec_amd.kernels.cache_eviction import attention_mass

    q, k, v = t_attn._qkv(t, n, hq, kvh, hd, dtype, seed, q_scale)
    kv = t_attn._cache(n, kvh, hd, dtype, page, seed)
    kv.append(1, k.cuda(), v.cuda(), 0)
    g = torch.Generator().manual_seed(seed)
    before = 3.0 * torch.rand(kvh, n, generator=g) if add else None
    got = attention_mass(q.cuda(), kv, 1, None if before is None else before.cuda(), scale=scale)
    torch.cuda.synchronize()
    assert got.shape == (kvh, n) and got.dtype == torch.float32
    _check(got, q, k, before, scale)
    return got


@pytest.mark.parametrize("hq,kvh,hd", [(32, 8, 128), (8, 2, 64), (4, 4, 128), (3, 1, 64),
                                       (16, 2, 128), (7, 1, 128), (64, 1, 64)])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("t,n,page", [(1, 1, 16), (1, 64, 16), (1, 65, 64), (1, 1000, 16),
                                      (2, 2, 16), (8, 300, 64), (9, 9, 1), (33, 200, 16),
                                      (65, 65, 16), (130, 700, 64)])
def test_mass(t, n, page, hq, kvh, hd, dtype):
    _say(f"mass t={t} n={n} page={page} heads={hq}/{kvh} hd={hd} {dtype}")
    _mass(t, n, hq, kvh, hd, dtype, page, t + n + hd, add=n % 2 == 0)


@pytest.mark.parametrize("t,n", [(1, 7777), (64, 7464), (1000, 1000), (700, 3000)])
@pytest.mark.parametrize("dtype,hd", [(BF, 128), (F16, 64)])
def test_mass_long(t, n, dtype, hd):
    _say(f"mass long t={t} n={n} {dtype} hd={hd}")
    _mass(t, n, 8, 2, hd, dtype, 16, t, add=True)


@pytest.mark.parametrize("t,n,hq,kvh,hd,dtype", [(300, 2100, 64, 16, 128, BF),
                                                 (350, 2050, 48, 16, 64, F16),
                                                 (3000, 3000, 16, 16, 64, BF)])
def test_mass_many_heads(t, n, hq, kvh, hd, dtype):
    """Tiles of keys that fill the chip."""
    _say(f"mass t={t} n={n} heads={hq}/{kvh} hd={hd} {dtype}")
    _mass(t, n, hq, kvh, hd, dtype, 64, t, add=True)


def test_mass_scale_strides_and_out():
    from treemoe_spec_amd.kernels.cache_eviction import attention_mass

    _say("mass scale, strides, out")
    _mass(5, 100, 8, 2, 64, BF, 16, 3, scale=0.4)
    q, k, v = t_attn._qkv(6, 90, 8, 2, 128, BF, 4)
    kv = t_attn._cache(90, 2, 128, BF, 16, 4)
    kv.append(0, k.cuda(), v.cuda(), 0)
    wide = torch.full((6, 10 * 128), NAN, dtype=BF, device="cuda")
    wide[:, 128:9 * 128] = q.flatten(1).cuda()
    view = wide[:, 128:9 * 128].unflatten(1, (8, 128))
    mass = torch.rand(2, 120, device="cuda")
    before = mass.cpu()
    assert attention_mass(view, kv, -2, mass, out=mass) is mass     # in place
    _check(mass[:, :90], q, k, before[:, :90])
    assert torch.equal(mass[:, 90:].cpu(), before[:, 90:])
    none = attention_mass(view[:0], kv, 0, mass)                    # no queries: what there was
    assert torch.equal(none, mass[:, :90])
    assert not bool(attention_mass(view[:0], kv, 0).any())


def test_mass_of_hidden_rows():
    """Scores of -inf give nothing; a NaN reaches the keys of the rows that see it."""
    from treemoe_spec_amd.kernels.cache_eviction import attention_mass

    _say("mass of rows without weight")
    q, k, v = t_attn._qkv(40, 200, 4, 1, 64, BF, 5)
    q[3] = 1.0
    kv = t_attn._cache(200, 1, 64, BF, 16, 5)
    k[:, 0, 0] = -INF
    k[:, 0, 1:] = 0.0
    q = q.abs()
    kv.append(0, k.cuda(), v.cuda(), 0)
    assert not bool(attention_mass(q.cuda(), kv, 0).any())
    q, k, v = t_attn._qkv(3, 200, 4, 2, 64, BF, 6)
    k[199, 1, 7] = NAN              # seen by the last token alone
    kv = t_attn._cache(200, 2, 64, BF, 16, 6)
    kv.append(0, k.cuda(), v.cuda(), 0)
    got = attention_mass(q.cuda(), kv, 0).cpu()
    assert bool(got[0].isfinite().all()) and bool(got[1].isnan().all())
    got = attention_mass(q[:2].cuda(), _shorter(kv, 199), 0).cpu()
    _check(got, q[:2], k[:199])


def _shorter(kv, n):
    kv.seq_len = n
    return kv


@pytest.mark.parametrize("t", [40, 300, 1100])
def test_a_row_that_is_not_a_number(t):
    """A NaN in a query reaches the keys that it sees, of its KV head, and no others."""
    from treemoe_spec_amd.kernels.cache_eviction import attention_mass

    _say(f"mass with a NaN query, {t} tokens")
    q, k, v = t_attn._qkv(t, t, 4, 2, 64, BF, t)
    q[t // 3, 3, 7] = NAN
    kv = t_attn._cache(t, 2, 64, BF, 16, t)
    kv.append(0, k.cuda(), v.cuda(), 0)
    got = attention_mass(q.cuda(), kv, 0).cpu()
    assert bool(got[1, :t // 3 + 1].isnan().all())
    q[t // 3, 3] = 0.0
    want = _want(q, k, 64 ** -0.5)
    assert bool(((got[0] - want[0]).abs() <= 1e-4 * want[0] + 2.0 ** -90).all())
    late = got[1, t // 3 + 1:]
    assert bool(((late - want[1, t // 3 + 1:]).abs() <= 1e-4 * late + 2.0 ** -90).all())


def test_mass_is_the_same_again():
    from treemoe_spec_amd.kernels.cache_eviction import attention_mass

    _say("mass again")
    q, k, v = t_attn._qkv(100, 3000, 32, 8, 128, BF, 7)
    kv = t_attn._cache(3000, 8, 128, BF, 64, 7)
    kv.append(0, k.cuda(), v.cuda(), 0)
    first = attention_mass(q.cuda(), kv, 0)
    for _ in range(4):
        assert torch.equal(first, attention_mass(q.cuda(), kv, 0))


# ------------------------------------------------------------------- evict --

def _cache_of(layers, n, kvh, hd, dtype, page, g):
    from treemoe_spec_amd.kv_cache import MixtralConfig, PagedKVCache

    kv = PagedKVCache(MixtralConfig(num_layers=layers, num_kv_heads=kvh, head_dim=hd),
                      -(-n // page) + 4, dtype=dtype, page_size=page, tree_size=1)
    for x in (kv.k, kv.v):
        x.copy_(torch.randn(x.shape, generator=g))
    kv._free = [kv._free[i] for i in torch.randperm(len(kv._free), generator=g).tolist()]
    kv._ensure_capacity(n)
    kv.seq_len = n
    return kv


def _evicted(rows, mass, position, keep, recent, sinks, nxt):
    """Slot lists of one head: which slot each of the first `keep` is filled from."""
    n = len(position)
    order = sorted(range(n), key=lambda s: (
        not (position[s] < sinks or position[s] >= nxt - recent),
        mass[s] != mass[s], -mass[s] if mass[s] == mass[s] else 0.0, s))
    safe = [s for s in range(n) if position[s] < sinks or position[s] >= nxt - recent]
    others = [s for s in order if s not in set(safe)]
    kept = set((safe + others)[:keep])
    movers = iter(sorted(s for s in kept if s >= keep))
    return [s if s in kept else next(movers) for s in range(keep)]


def _check_evict(kv, mass, keep, positions=None, nxt=None, recent=0, sinks=0):
    from treemoe_spec_amd.kernels.cache_eviction import evict

    layers, kvh = mass.shape[:2]
    n = kv.seq_len
    before = [x.cpu().clone() for x in (kv.k, kv.v)]
    want = [x.clone() for x in before]
    next_position = n if nxt is None else nxt
    count = min(keep, n)
    want_mass = torch.zeros(mass.shape)
    want_pos = torch.zeros(layers, kvh, count, dtype=torch.int32)
    recorded = 0 if positions is None else positions.shape[2]
    slots = [kv.slot_of(s) for s in range(n)]
    for layer in range(layers):
        for h in range(kvh):
            pos = list(range(next_position - n, next_position))
            if recorded:
                pos[:recorded] = positions[layer, h].tolist()
            m = mass[layer, h, :n].tolist()
            src = _evicted(None, m, pos, count, recent, sinks, next_position)
            for to, s in enumerate(src):
                want_mass[layer, h, to] = mass[layer, h, s]
                want_pos[layer, h, to] = pos[s]
                if to != s:
                    (tp, to_off), (fp, from_off) = slots[to], slots[s]
                    for w, b in zip(want, before):
                        w[layer, tp, to_off, h] = b[layer, fp, from_off, h]
    got = evict(kv, mass.cuda(), keep, positions=None if positions is None else positions.cuda(),
                next_position=nxt, recent=recent, sinks=sinks)
    torch.cuda.synchronize()
    assert kv.seq_len == count
    assert torch.equal(got[1].cpu(), want_pos)
    assert torch.equal(torch.nan_to_num(got[0].cpu(), nan=-7.0),
                       torch.nan_to_num(want_mass, nan=-7.0))
    for x, w in zip((kv.k, kv.v), want):
        assert torch.equal(x.cpu(), w)
    return got


@pytest.mark.parametrize("layers,kvh,hd,dtype,page", [(1, 1, 128, BF, 16), (3, 2, 64, F16, 64),
                                                      (2, 8, 128, BF, 1),
                                                      (2, 2, 16, torch.float32, 16)])
@pytest.mark.parametrize("n,keep,recent,sinks", [
    (1, 1, 0, 0), (2, 1, 0, 0), (100, 50, 0, 0), (100, 99, 10, 4), (130, 20, 16, 4),
    (65, 64, 64, 0),
    (64, 1, 0, 1), (200, 199, 0, 0), (1100, 1030, 64, 4), (2100, 100, 32, 4), (50, 50, 3, 0),
    (50, 90, 3, 0), (30, 0, 0, 0), (2048, 2000, 100, 4), (2049, 700, 64, 0)])
def test_evict(n, keep, recent, sinks, layers, kvh, hd, dtype, page):
    _say(f"evict {n} -> {keep} recent {recent} sinks {sinks} {layers}x{kvh} hd={hd} {dtype}")
    g = torch.Generator().manual_seed(n + keep)
    kv = _cache_of(layers, n, kvh, hd, dtype, page, g)
    mass = torch.exp(2 * torch.randn(layers, kvh, n + 7, generator=g))
    _check_evict(kv, mass, keep, recent=recent, sinks=sinks)


@pytest.mark.parametrize("layers,n,keep", [(1, 8192, 4000), (1, 8193, 8100), (1, 16384, 8192),
                                           (1, 16385, 9000), (1, 20000, 130), (40, 600, 580),
                                           (40, 600, 300)])
def test_evict_long_and_many(layers, n, keep):
    """Keys of a head beyond what a workgroup holds; heads that fill the chip."""
    _say(f"evict {layers} layers {n} -> {keep}")
    g = torch.Generator().manual_seed(n)
    kv = _cache_of(layers, n, 4, 16, BF, 64, g)
    mass = torch.exp(2 * torch.randn(layers, 4, n, generator=g))
    mass[0, 1] = mass[0, 1].round()
    _check_evict(kv, mass, keep, recent=64, sinks=4)


def test_evict_ties_and_odd_masses():
    _say("evict ties, zeros, infinities, NaN")
    g = torch.Generator().manual_seed(2)
    for mass in (torch.zeros(2, 2, 1500), torch.full((2, 2, 1500), -1.0),
                 torch.randint(0, 3, (2, 2, 1500), generator=g).float()):
        _check_evict(_cache_of(2, 1500, 2, 64, BF, 16, g), mass, 700, recent=33, sinks=2)
    mass = torch.randn(2, 2, 1500, generator=g)
    mass[0, 0, ::3] = NAN
    mass[0, 1, ::4] = INF
    mass[1, 0, ::5] = -INF
    mass[1, 1, ::2] = -0.0
    mass[1, 1, 1::2] = 0.0
    _check_evict(_cache_of(2, 1500, 2, 64, BF, 16, g), mass, 1201)
    _check_evict(_cache_of(2, 1500, 2, 64, BF, 16, g), torch.full((2, 2, 1500), NAN), 3)


def test_evict_again_and_again():
    """A cache that grows by a few tokens and is cut back, its positions handed on."""
    _say("evict again")
    g = torch.Generator().manual_seed(3)
    kv = _cache_of(2, 150, 2, 64, BF, 16, g)
    mass = torch.rand(2, 2, 300, generator=g)
    positions, nxt = None, 150
    for step in range(6):
        new_mass, new_pos = _check_evict(kv, mass, 100, positions, nxt, recent=20, sinks=4)
        positions, mass = new_pos.cpu(), new_mass.cpu()
        assert set(range(4)) <= set(positions[1, 0].tolist())
        assert set(range(nxt - 20, nxt)) <= set(positions[0, 1].tolist())
        grow = 7 + 13 * step
        kv._ensure_capacity(100 + grow)
        kv.seq_len, nxt = 100 + grow, nxt + grow
        mass[:, :, :100 + grow] += torch.rand(2, 2, 100 + grow, generator=g)


def test_evict_strided_inputs():
    _say("evict strided masses and positions")
    g = torch.Generator().manual_seed(4)
    n, keep = 300, 200
    mass = torch.rand(3, 4, 500, generator=g)
    pos = torch.rand(3, 4, 900, generator=g).argsort(2).to(torch.int32)[:, :, :250]
    _check_evict(_cache_of(3, n, 2, 64, BF, 16, g), mass[:, 1:3, 60:400], keep,
                 pos[:, 2:, :120], 1000, recent=30, sinks=2)


def test_attention_after_eviction():
    """Attention over the cut cache is attention over the kept keys, head by head."""
    from treemoe_spec_amd.kernels.cache_eviction import attention_mass, evict
    from treemoe_spec_amd.kernels.prompt_attention import prompt_attention_cached

    _say("evict, then attention")
    n, hq, kvh, hd = 500, 8, 2, 128
    q, k, v = t_attn._qkv(20, n, hq, kvh, hd, BF, 8)
    kv = t_attn._cache(n + 10, kvh, hd, BF, 16, 8, layers=1)
    kv.append(0, k.cuda(), v.cuda(), 0)
    mass = attention_mass(q.cuda(), kv, 0)
    _, positions = evict(kv, mass[None], 128, recent=16, sinks=4)
    q1, k1, v1 = t_attn._qkv(1, 1, hq, kvh, hd, BF, 9)
    kv.append(0, k1.cuda(), v1.cuda(), kv.seq_len)
    assert kv.seq_len == 129
    out = prompt_attention_cached(q1.cuda(), kv, 0).view(1, kvh, hq // kvh, hd)
    for h in range(kvh):
        at = positions[0, h].long().cpu()
        keys, values = (torch.cat([x[at, h:h + 1], y[:, h:h + 1]])
                        for x, y in ((k, k1), (v, v1)))
        t_attn._check(out[:, h].flatten(1), q1[:, h * 4:h * 4 + 4], keys, values, 128)
