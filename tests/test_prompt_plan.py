"""CPU: the work lists of prompt attention, and what its calls refuse."""

from __future__ import annotations

import ctypes
import math
import random

import pytest
import torch

from treemoe_spec_amd import _capi
from treemoe_spec_amd.kernels import prompt_attention as pa

BF = torch.bfloat16
ROWS = (32, 128, 128, 256)


def _plan(q_lens, k_lens=None, hq=8, kvh=2):
    return pa.PromptPlan(q_lens, k_lens, num_heads=hq, num_kv_heads=kvh, device="cpu")


def _check_plan(q_lens, k_lens, hq, kvh):
    """Every tile's keys are covered once, in stages of 64, by items of its own; a split
    tile has one join of its slots; items come longest first."""
    plan = _plan(q_lens, k_lens, hq, kvh)
    group, rows = hq // kvh, plan.tile_rows
    assert rows == ROWS[plan.tiling]
    items, joins = plan.items.tolist(), plan.joins.tolist()
    cover, slots = {}, {}
    for q0, ql, k0, kl, tile, begin, end, slot in items[:plan.num_items]:
        cover.setdefault((q0, ql, k0, kl, tile), []).append((begin, end, slot))
    lengths = [i[6] - i[5] for i in items[:plan.num_items]]
    assert lengths == sorted(lengths, reverse=True)
    q0 = k0 = 0
    seen = 0
    for ql, kl in zip(q_lens, k_lens):
        for tile in range(-(-ql * group // rows)):
            parts = sorted(cover.pop((q0, ql, k0, kl, tile)))
            last = min(ql - 1, (tile * rows + rows - 1) // group)
            assert parts[0][0] == 0 and parts[-1][1] == kl - ql + last + 1
            for (b0, e0, s0), (b1, _, s1) in zip(parts, parts[1:]):
                assert e0 == b1 and e0 % 64 == 0 and s1 == s0 + 1
            assert all(e > b for b, e, _ in parts)
            if len(parts) == 1:
                assert parts[0][2] == -1
            else:
                slots[parts[0][2]] = (q0, ql, tile, parts[0][2], len(parts))
            seen += len(parts)
        q0, k0 = q0 + ql, k0 + kl
    assert not cover and seen == plan.num_items
    assert (plan.q_rows, plan.k_rows) == (sum(q_lens), sum(k_lens))
    assert {j[3]: tuple(j[:5]) for j in joins[:plan.num_joins]} == slots
    assert plan.num_slots == sum(s[4] for s in slots.values())
    assert all(s[4] <= 512 for s in slots.values())
    return plan


@pytest.mark.parametrize("q_lens,k_lens,hq,kvh,tiling", [
    ([1], [1], 8, 2, 0), ([8], [5000], 8, 2, 0), ([9], [9], 8, 2, 1), ([1], [100000], 33, 1, 2),
    ([8192], [8192], 32, 8, 3), ([600], [5000], 32, 8, 2), ([100] * 50, [100] * 50, 32, 8, 1),
    ([0, 0, 5], [0, 4, 5], 4, 4, 0), ([1] * 300, [4000] * 300, 32, 8, 0),
    ([1], [1 << 24], 1, 1, 0), ([60] * 100 + [1], [60] * 100 + [50000], 8, 2, 1),
    ([4000, 1], [4000, 100000], 32, 8, 3),
])
def test_plans(q_lens, k_lens, hq, kvh, tiling):
    assert _check_plan(q_lens, k_lens, hq, kvh).tiling == tiling


def test_random_plans():
    rng = random.Random(5)
    for _ in range(60):
        n = rng.randint(1, 20)
        q = [rng.choice([0, 1, 1, rng.randint(1, 80), rng.randint(1, 1500)]) for _ in range(n)]
        k = [x + rng.choice([0, 0, rng.randint(0, 3000)]) for x in q]
        hq, kvh = rng.choice([(32, 8), (8, 2), (4, 4), (7, 1)])
        _check_plan(q, k, hq, kvh)


def test_empty_plan():
    plan = _plan([])
    assert plan.num_items == plan.num_joins == plan.q_rows == 0


@pytest.mark.parametrize("q_lens,k_lens,hq,kvh", [
    ([3], [2], 8, 2), ([-1], [2], 8, 2), ([3], [1 << 25], 8, 2), ([3], [3, 3], 8, 2),
    ([3], [3], 7, 2), ([3], [3], 1, 2), ([3], [3], 4, 0),
])
def test_plan_refuses(q_lens, k_lens, hq, kvh):
    with pytest.raises(ValueError):
        _plan(q_lens, k_lens, hq, kvh)


@pytest.fixture()
def calls(monkeypatch):
    done = []
    monkeypatch.setattr(_capi, "require", lambda *a, **k: None)
    monkeypatch.setattr(_capi, "launch", lambda *a: done.append(a))
    return done


@pytest.mark.parametrize("kw", [
    {"q": torch.zeros(5, 8, 96, dtype=BF)}, {"q": torch.zeros(5, 8, 64)},
    {"q": torch.zeros(5, 512, dtype=BF)}, {"q": torch.zeros(5, 16, 64, dtype=BF)[:, ::2]},
    {"q": torch.zeros(4, 8, 64, dtype=BF)}, {"q": torch.zeros(5, 4, 64, dtype=BF)},
    {"k": torch.zeros(6, 2, 64, dtype=BF)}, {"k": torch.zeros(7, 2, 64, dtype=torch.float16)},
    {"k": torch.zeros(7, 1, 64, dtype=BF)}, {"v": torch.zeros(8, 2, 64, dtype=BF)},
    {"v": torch.zeros(7, 4, 64, dtype=BF)[:, ::2]}, {"scale": 0.0}, {"scale": -1.0},
    {"scale": math.inf}, {"scale": math.nan}, {"out": torch.zeros(5, 500, dtype=BF)},
    {"out": torch.zeros(5, 512)}, {"out": torch.zeros(512, 5, dtype=BF).T},
])
def test_prompt_attention_refuses(calls, kw):
    a = {"q": torch.zeros(5, 8, 64, dtype=BF), "k": torch.zeros(7, 2, 64, dtype=BF),
         "v": torch.zeros(7, 2, 64, dtype=BF), **kw}
    with pytest.raises(ValueError):
        pa.prompt_attention(a.pop("q"), a.pop("k"), a.pop("v"), _plan([3, 2], [4, 3]), **a)
    assert not calls


def test_out_over_the_queries_is_refused(calls):
    q = torch.zeros(5, 8, 64, dtype=BF)
    k = torch.zeros(7, 2, 64, dtype=BF)
    with pytest.raises(ValueError, match="apart"):
        pa.prompt_attention(q, k, k, _plan([3, 2], [4, 3]), out=q.view(5, 512))
    assert not calls


def test_prompt_attention_arguments(calls):
    plan = _plan([3, 2], [4, 3])
    q = torch.zeros(6, 12, 64, dtype=BF)[:, :8]
    k = torch.zeros(9, 2, 64, dtype=BF)
    out = pa.prompt_attention(q, k, k, plan)
    name, _, *a = calls.pop()
    assert name == "tm_prompt_attention" and a[1] == 768 and a[3] == a[5] == 128
    assert a[7] == plan.num_items and a[11:15] == [0, 8, 2, 64] and a[15] == 0.125
    assert out.shape == (6, 512) and bool((out[5:] == 0).all())


def _kv(page=4, dtype=BF, hd=64):
    from treemoe_spec_amd.kv_cache import MixtralConfig, PagedKVCache

    kv = PagedKVCache(MixtralConfig(num_layers=2, num_kv_heads=2, head_dim=hd), 8, device="cpu",
                      dtype=dtype, page_size=page, tree_size=4)
    kv._ensure_capacity(10)
    kv.seq_len = 10
    return kv


def test_cached_arguments(calls):
    kv = _kv()
    q = torch.zeros(3, 8, 64, dtype=BF)
    pa.prompt_attention_cached(q, kv, -1)
    name, _, *a = calls.pop()
    assert name == "tm_prompt_attention_cached" and a[1:3] == [512, 3]
    assert a[3] == kv.k.data_ptr() + kv.k[0].numel() * 2 and a[5:9] == [512, 128, 4, 8]
    assert a[10:15] == [3, 10, 8, 2, 64]
    assert pa.prompt_attention_cached(q[:0], kv, 0).shape == (0, 512) and not calls
    for err, args in ((IndexError, (q, kv, 2)), (IndexError, (q, kv, -3)),
                      (ValueError, (torch.zeros(11, 8, 64, dtype=BF), kv, 0)),
                      (ValueError, (torch.zeros(3, 7, 64, dtype=BF), kv, 0)),
                      (ValueError, (q, _kv(page=6), 0)), (ValueError, (q, _kv(hd=128), 0)),
                      (ValueError, (q, _kv(dtype=torch.float16), 0))):
        with pytest.raises(err):
            pa.prompt_attention_cached(*args)
    assert not calls


def test_cpu_tensors_raise():
    q = torch.zeros(3, 8, 64, dtype=BF)
    with pytest.raises(RuntimeError, match="ROCm"):
        pa.prompt_attention_cached(q, _kv(), 0)
    with pytest.raises(RuntimeError, match="ROCm"):
        pa.prompt_attention(q, q[:, :2], q[:, :2], _plan([3]))


# -------------------------------------------------------------- C entry points --

def _c(name, defaults, kw):
    return getattr(_capi.lib(), name)(*{**defaults, **kw}.values())


PACKED = dict(q=0, qs=512, k=0, ks=128, v=0, vs=128, items=0, n=1, joins=0, nj=0, slots=0, tiling=1,
              hq=8, kvh=2, hd=64, scale=0.1, dt=1, out=0, os=512, ws=0, wsb=0, stream=0)


@pytest.mark.parametrize("kw,expect", [
    ({"hq": 7}, 1001), ({"kvh": 0}, 1001), ({"hd": 96}, 1001), ({"dt": 0}, 1003),
    ({"scale": 0.0}, 1003), ({"scale": math.nan}, 1003), ({"scale": math.inf}, 1003),
    ({"tiling": 4}, 1003), ({"tiling": -1}, 1003), ({"n": -1}, 1001), ({"n": 1 << 31}, 1001),
    ({"qs": 500}, 1001), ({"ks": 120}, 1001), ({"vs": 1 << 25}, 1001), ({"os": 8}, 1001),
    ({"slots": 2}, 1001), ({"n": 0}, 0),
    ({"n": 1 << 23, "kvh": 8}, 1001), ({"n": 1 << 23, "hq": 1, "kvh": 1, "tiling": 3}, 1001),
    ({"nj": 2}, 1001), ({}, 1003), ({"items": 32, "n": 1, "nj": 1}, 1003), ({"q": 8}, 1002), ({"ks": 132}, 1002), ({"items": 16}, 1002),
    ({"ws": 8}, 1002),
])
def test_prompt_attention_entry_point(kw, expect):
    assert _c("tm_prompt_attention", PACKED, kw) == expect


def test_plan_entry_point():
    plan = _capi.lib().tm_prompt_plan
    one = (ctypes.c_int64 * 1)(8)
    long = (ctypes.c_int64 * 1)(50000)
    sizes = (ctypes.c_int64 * 7)()
    items, joins = (ctypes.c_int32 * 4096)(), (ctypes.c_int32 * 4096)()
    assert plan(one, long, 1, 8, 2, None, 0, None, 0, sizes) == 0
    assert sizes[0] > 1 and sizes[1] > 0
    assert plan(one, long, 1, 8, 2, items, 512, joins, 512, sizes) == 0
    assert plan(one, long, 1, 8, 2, None, 512, joins, 512, sizes) == 1003
    assert plan(one, long, 1, 8, 2, items, 512, None, 512, sizes) == 1003
    assert plan(one, long, 1, 8, 2, items, sizes[0] - 1, joins, 512, sizes) == 1001
    assert plan(one, long, 1, 8, 2, items, 512, joins, 0, sizes) == 1001
    assert plan(one, one, 1, 8, 2, items, 1, None, 0, sizes) == 0 and sizes[1] == 0
    assert plan(long, one, 1, 8, 2, items, 1, None, 0, sizes) == 1001
    assert plan(None, None, 1, 8, 2, items, 1, None, 0, sizes) == 1003
    assert plan(None, None, 0, 8, 2, items, 1, None, 0, sizes) == 0 and sizes[0] == 0
    assert plan(one, one, 1, 8, 2, None, 0, None, 0, None) == 1003


CACHED = dict(q=0, qs=512, T=4, k=0, v=0, sp=16 * 128, ss=128, page=16, pages=4, table=0, n_table=4,
              seq=64, hq=8, kvh=2, hd=64, scale=0.1, dt=2, out=0, os=512, ws=0, wsb=1 << 30, stream=0)


@pytest.mark.parametrize("kw,expect", [
    ({"hd": 32}, 1001), ({"dt": 3}, 1003), ({"scale": -1.0}, 1003), ({"T": 65}, 1001),
    ({"T": -1}, 1001), ({"seq": (1 << 24) + 1}, 1001), ({"page": 24}, 1001), ({"page": 0}, 1001),
    ({"seq": 65}, 1001), ({"n_table": 3}, 1001), ({"pages": 0}, 1001), ({"qs": 8}, 1001),
    ({"ss": 64}, 1001), ({"sp": 128}, 1001), ({"ss": 132, "sp": 16 * 132}, 1002), ({"q": 8}, 1002),
    ({"table": 2}, 1002), ({"T": 0}, 0),
    ({"seq": 4000, "n_table": 250, "pages": 250, "wsb": 100}, 1001),
])
def test_cached_entry_point(kw, expect):
    assert _c("tm_prompt_attention_cached", CACHED, kw) == expect


def test_cached_workspace():
    size = ctypes.c_int64()
    ws = _capi.lib().tm_prompt_cached_workspace
    assert ws(1, 100, 32, 8, 128, ctypes.byref(size)) == 0 and size.value == 0
    # one token over 7777 keys: 31 ranges of 256 keys, 8 KV heads, tiles of 32 rows
    assert ws(1, 7777, 32, 8, 128, ctypes.byref(size)) == 0
    assert size.value == 31 * 8 * 32 * 130 * 4
    assert ws(5, 4, 32, 8, 128, ctypes.byref(size)) == 1001
    assert ws(1, 4, 32, 8, 96, ctypes.byref(size)) == 1001
    fast = _capi.layer_binding()
    assert fast.prompt_cached_workspace(1, 7777, 32, 8, 128) == (0, 31 * 8 * 32 * 130 * 4)
    assert fast.prompt_cached_workspace(5, 4, 32, 8, 128)[0] == 1001
    with pytest.raises(TypeError):
        fast.prompt_cached_workspace(1)


def test_fast_calls_match_ctypes():
    for name, args in (("tm_prompt_attention", PACKED), ("tm_prompt_attention_cached", CACHED)):
        fast = _capi.entry(name)
        assert type(fast).__name__ == "builtin_function_or_method"
        assert fast(*{**args, "hd": 32}.values()) == 1001
        with pytest.raises(TypeError):
            fast(1)
