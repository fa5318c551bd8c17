"""CPU: what the norm, rotary and sampling operators refuse, in Python and at the C
entry points (which check before any launch), and the arguments they pass on."""

from __future__ import annotations

import math

import pytest
import torch

from treemoe_spec_amd import _capi
from treemoe_spec_amd.kernels import rms_norm as rn
from treemoe_spec_amd.kernels import rotary as ro
from treemoe_spec_amd.kernels import sample_tokens as st

BF = torch.bfloat16


@pytest.fixture()
def calls(monkeypatch):
    """Launches recorded instead of made, on CPU tensors."""
    done = []
    monkeypatch.setattr(_capi, "require", lambda *a, **k: None)
    monkeypatch.setattr(_capi, "launch", lambda *a: done.append(a))
    return done


# ------------------------------------------------------------------- Python --

def test_rows_are_bounded(calls):
    n = _capi.TM_MAX_ROWS + 1
    with pytest.raises(ValueError, match="at most"):
        rn.rms_norm(torch.zeros(1, 8).expand(n, 8), torch.zeros(8))
    plan = ro.RotaryPlan(16, 1e4, device="cpu")
    q = torch.zeros(1, 1, 16).expand(n, 1, 16)
    with pytest.raises(ValueError, match="at most"):
        ro.rotary_embed(q, None, torch.zeros(1, dtype=torch.int32).expand(n), plan)
    with pytest.raises(ValueError, match="at most"):
        st.sample_tokens(torch.zeros(1, 8).expand(n, 8), torch.zeros(1).expand(n))
    assert not calls


def test_probs_over_the_logits_are_refused(calls):
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="apart"):
        st.sample_tokens(x, torch.zeros(2), return_probs=True, probs_out=x)
    assert not calls


def test_cpu_tensors_raise():
    x, w = torch.zeros(2, 8), torch.zeros(8)
    with pytest.raises(RuntimeError, match="ROCm"):
        rn.rms_norm(x, w)
    with pytest.raises(RuntimeError, match="ROCm"):
        rn.rms_norm_fp8(x, w)
    plan = ro.RotaryPlan(16, 1e4, device="cpu")
    with pytest.raises(RuntimeError, match="ROCm"):
        ro.rotary_embed(torch.zeros(2, 1, 16), None, torch.arange(2), plan)
    with pytest.raises(RuntimeError, match="ROCm"):
        st.sample_tokens(x, torch.zeros(2))


def test_gradients_are_refused():
    dev = torch.device("cpu")
    with pytest.raises(RuntimeError, match="ROCm"):
        _capi.require("op", dev)
    fake = type("T", (), {"device": torch.device("cuda", 0), "requires_grad": True})()
    with pytest.raises(RuntimeError, match="no backward"):
        _capi.require("op", torch.device("cuda", 0), x=fake)
    with torch.no_grad():
        _capi.require("op", torch.device("cuda", 0), x=fake, y=None)
    with pytest.raises(ValueError, match="is on"):
        _capi.require("op", torch.device("cuda", 1), x=fake)


@pytest.mark.parametrize("kw", [
    {"x": torch.zeros(8)}, {"weight": torch.zeros(7)}, {"x": torch.zeros(2, 8, dtype=torch.int32)},
    {"weight": torch.zeros(8, dtype=BF)}, {"x": torch.zeros(8, 2).T}, {"eps": -1.0},
    {"eps": math.nan}, {"residual": torch.zeros(3, 8)}, {"residual": torch.zeros(2, 8, dtype=BF)},
    {"residual": torch.zeros(8, 2).T}, {"residual_out": torch.zeros(2, 8)},
    {"residual": torch.zeros(2, 8), "residual_out": torch.zeros(2, 8, dtype=BF)},
    {"out": torch.zeros(2, 9)}, {"out": torch.zeros(2, 8, dtype=BF)},
    {"x": torch.zeros(1, 65537), "weight": torch.zeros(65537)},
])
def test_norm_refuses(calls, kw):
    args = {"x": torch.zeros(2, 8), "weight": torch.zeros(8), "eps": 1e-5, **kw}
    with pytest.raises(ValueError):
        rn.rms_norm(args.pop("x"), args.pop("weight"), args.pop("eps"), **args)
    assert not calls


@pytest.mark.parametrize("group", [0, 16, 48, 1024, 64])
def test_norm_refuses_scale_groups(calls, group):
    with pytest.raises(ValueError):
        rn.rms_norm_fp8(torch.zeros(2, 96), torch.zeros(96), scale_group=group)


def test_norm_passes_strides(calls):
    x, r = torch.zeros(3, 20)[:, 2:10], torch.zeros(3, 9)[:, :8]
    y, s = rn.rms_norm(x, torch.zeros(8), 1e-6, residual=r)
    name, _, *a = calls[0]
    assert name == "tm_rms_norm" and a[1] == 20 and a[3] == 9 and a[7:11] == [3, 8, 1e-6, 0]
    assert y.is_contiguous() and s.is_contiguous() and a[12] == 8 and a[14] == 8


@pytest.mark.parametrize("kw", [
    {"head_dim": 24}, {"head_dim": 0}, {"head_dim": 1040}, {"rotary_dim": 8}, {"rotary_dim": 80},
    {"rotary_dim": 24}, {"theta": 1.0}, {"theta": math.inf}, {"scaling": {"type": "other"}},
    {"scaling": {"type": "linear", "factor": 0.5}}, {"scaling": {"type": "ntk", "factor": math.nan}},
    {"scaling": {"type": "yarn", "factor": 2.0, "original_max_position": 0}},
    {"scaling": {"type": "yarn", "factor": 2.0, "original_max_position": 64, "beta_fast": 1.0,
                 "beta_slow": 2.0}},
    {"inv_freq": [1.0]}, {"inv_freq": [math.inf] * 32},
    {"inv_freq": [1.0] * 32, "scaling": {"type": "linear", "factor": 2.0}},
])
def test_rotary_plan_refuses(kw):
    args = {"head_dim": 64, "theta": 1e4, "device": "cpu", **kw}
    with pytest.raises(ValueError):
        ro.RotaryPlan(args.pop("head_dim"), args.pop("theta"), **args)


def test_rotary_frequencies():
    f, m = ro.rotary_frequencies(8, 1e4)
    assert m == 1.0 and f == [1e4 ** (-i / 4) for i in range(4)]
    g, m = ro.rotary_frequencies(8, 1e4, {"type": "linear", "factor": 2.0})
    assert m == 1.0 and g == [x / 2 for x in f]
    g, _ = ro.rotary_frequencies(8, 1e4, {"type": "ntk", "factor": 4.0})
    assert g[0] == 1.0 and g[3] == pytest.approx(f[3] / 4, rel=1e-12)  # the last pair is stretched
    y = {"type": "yarn", "factor": 4.0, "original_max_position": 4096}
    g, m = ro.rotary_frequencies(128, 1e4, y)
    f, _ = ro.rotary_frequencies(128, 1e4)
    assert m == 0.1 * math.log(4.0) + 1.0
    assert g[0] == f[0] and g[63] == f[63] / 4 and all(a >= b for a, b in zip(g, g[1:]))
    assert ro.rotary_frequencies(128, 1e4, {**y, "attention_factor": 1.5})[1] == 1.5


@pytest.mark.parametrize("kw", [
    {"q": torch.zeros(2, 16)}, {"q": torch.zeros(2, 1, 32)},
    {"q": torch.zeros(2, 1, 16, dtype=torch.float64)}, {"q": torch.zeros(2, 4, 16)[:, ::2]},
    {"k": torch.zeros(3, 1, 16)}, {"k": torch.zeros(2, 1, 16, dtype=BF)},
    {"positions": torch.zeros(3, dtype=torch.int64)}, {"positions": torch.zeros(2)},
    {"positions": torch.zeros(4, dtype=torch.int64)[::2]}, {"q_out": torch.zeros(2, 2, 16)},
    {"k": None, "k_out": torch.zeros(2, 1, 16)}, {"k_out": torch.zeros(2, 2, 16)},
])
def test_rotary_refuses(calls, kw):
    plan = ro.RotaryPlan(16, 1e4, device="cpu")
    a = {"q": torch.zeros(2, 1, 16), "k": torch.zeros(2, 1, 16), "positions": torch.arange(2), **kw}
    with pytest.raises(ValueError):
        ro.rotary_embed(a.pop("q"), a.pop("k"), a.pop("positions"), plan, **a)
    assert not calls


def _kv(**kw):
    from treemoe_spec_amd.kv_cache import MixtralConfig, PagedKVCache

    a = {"dtype": torch.float32, "page_size": 4, "tree_size": 4, **kw}
    cfg = MixtralConfig(num_layers=2, num_kv_heads=1, head_dim=16)
    return PagedKVCache(cfg, 6, device="cpu", **a)


def test_rotary_append_arguments(calls):
    plan = ro.RotaryPlan(16, 1e4, device="cpu")
    q, k = torch.zeros(5, 2, 16), torch.zeros(5, 1, 16)
    kv = _kv()
    out = ro.rotary_append(q, k, k, plan, kv, -1, 3)
    name, _, *a = calls.pop()
    assert name == "tm_rotary_append" and out.shape == q.shape
    assert kv.seq_len == 8 and len(kv.block_table) == 2
    assert a[8] == kv.k.data_ptr() + kv.k[0].numel() * 4 and a[10:14] == [64, 16, 4, 6]
    assert a[15:17] == [2, 3]
    ro.rotary_append(q[:0], k[:0], k[:0], plan, kv, 0, 3)
    assert not calls
    for bad in ((_kv(dtype=BF), q, k, 0, 0, ValueError), (kv, q, k, 2, 0, IndexError),
                (kv, q, k, 0, -1, ValueError), (kv, q, torch.zeros(5, 2, 16), 0, 0, ValueError),
                (kv, q[:4], k, 0, 0, ValueError), (kv, q, k, 0, 100, RuntimeError)):
        with pytest.raises(bad[5]):
            ro.rotary_append(bad[1], bad[2], bad[2], plan, bad[0], bad[3], bad[4])
    assert not calls and kv.seq_len == 8


@pytest.mark.parametrize("kw", [
    {"logits": torch.zeros(4)}, {"logits": torch.zeros(2, 4, dtype=torch.int32)},
    {"logits": torch.zeros(4, 2).T}, {"logits": torch.zeros(2, 0)},
    {"uniforms": torch.zeros(3)}, {"uniforms": torch.zeros(2, dtype=torch.float64)},
    {"uniforms": torch.zeros(4)[::2]}, {"temperature": -1.0}, {"temperature": math.nan},
    {"temperature": math.inf}, {"top_k": -1}, {"top_p": 1.5}, {"top_p": -0.1}, {"min_p": 2.0},
    {"top_k": torch.zeros(2, dtype=torch.int64)}, {"top_p": torch.zeros(3)},
    {"min_p": torch.zeros(4)[::2]}, {"probs_out": torch.zeros(2, 4)},
    {"probs_out": torch.zeros(2, 5), "return_probs": True},
])
def test_sample_refuses(calls, kw):
    a = {"logits": torch.zeros(2, 4), "uniforms": torch.zeros(2), **kw}
    with pytest.raises(ValueError):
        st.sample_tokens(a.pop("logits"), a.pop("uniforms"), **a)
    assert not calls


def test_sample_passes_numbers_and_rows(calls):
    logits, u = torch.zeros(2, 10)[:, :8], torch.zeros(2)
    k = torch.zeros(2, dtype=torch.int32)
    st.sample_tokens(logits, u, temperature=0.3, top_k=k, top_p=torch.tensor(0.5), min_p=0.1)
    name, _, *a = calls[0]
    assert name == "tm_sample_tokens" and a[1:5] == [0, 2, 8, 10]
    assert a[6:14] == [0, 0.3, k.data_ptr(), 0, 0, 0.5, 0, 0.1] and a[15:] == [0, 0]
    tokens, probs = st.sample_tokens(logits, u, top_k=10 ** 12, return_probs=True)
    assert tokens.dtype == torch.int64 and probs.shape == (2, 8) and calls[1][2 + 9] == 8


# -------------------------------------------------------------- C entry points --

def _c(name, defaults, kw):
    return getattr(_capi.lib(), name)(*{**defaults, **kw}.values())


NORM = dict(x=0, xs=64, r=0, rs=0, rdt=1, w=0, wdt=1, T=4, H=64, eps=1e-5, dt=1, out=0, os=64,
            ro=0, ros=0, stream=0)


@pytest.mark.parametrize("kw,expect", [
    ({"dt": 3}, 1003), ({"wdt": 2}, 1003), ({"eps": -1.0}, 1003), ({"eps": math.nan}, 1003),
    ({"r": 16, "rdt": 2}, 1003), ({"H": 0}, 1001), ({"H": 65537}, 1001), ({"T": -1}, 1001),
    ({"xs": 63}, 1001), ({"os": 63}, 1001), ({"r": 16, "rs": 64}, 1001),
    ({"r": 16, "rs": 64, "ro": 16, "ros": 63}, 1001), ({"x": 1}, 1002), ({"out": 1}, 1002),
    ({"w": 2, "wdt": 0}, 1002), ({"r": 17, "rs": 64, "ro": 16, "ros": 64}, 1002), ({"T": 0}, 0),
])
def test_norm_entry_point(kw, expect):
    assert _c("tm_rms_norm", NORM, kw) == expect


FP8 = dict(x=0, xs=128, r=0, rs=0, rdt=1, w=0, wdt=1, T=4, H=128, eps=1e-5, dt=1, out=0, os=128,
           scales=0, ss=1, group=128, ro=0, ros=0, stream=0)


@pytest.mark.parametrize("kw,expect", [
    ({"group": 48}, 1001), ({"group": 16}, 1001), ({"group": 1024}, 1001), ({"group": -32}, 1001),
    ({"H": 96, "group": 64}, 1001), ({"group": 32, "ss": 3}, 1001), ({"scales": 2}, 1002),
    ({"T": 0}, 0),
])
def test_norm_fp8_entry_point(kw, expect):
    assert _c("tm_rms_norm_fp8", FP8, kw) == expect


ROT = dict(q=0, qs=4096, k=0, ks=1024, qo=0, qos=4096, ko=0, kos=1024, pos=0, long=1, turns=0,
           mag=1.0, T=4, hq=32, kvh=8, hd=128, part=128, inter=0, dt=1, stream=0)


@pytest.mark.parametrize("kw,expect", [
    ({"dt": 4}, 1003), ({"hd": 120}, 1001), ({"hd": 0}, 1001), ({"part": 144}, 1001),
    ({"part": 0}, 1001), ({"part": 72}, 1001), ({"T": -1}, 1001), ({"T": 1 << 25}, 1001),
    ({"hq": -1}, 1001), ({"kvh": 2000}, 1001), ({"qs": 4000}, 1001), ({"kos": 1000}, 1001),
    ({"q": 8}, 1002), ({"qs": 4100}, 1002), ({"pos": 4}, 1002), ({"turns": 4}, 1002),
    ({"T": 0}, 0), ({"hq": 0, "kvh": 0}, 0),
])
def test_rotary_entry_point(kw, expect):
    assert _c("tm_rotary", ROT, kw) == expect


APP = dict(q=0, qs=4096, k=0, ks=1024, v=0, vs=1024, qo=0, qos=4096, kc=0, vc=0, sp=16 * 1024,
           ss=1024, page=16, pages=10, table=0, n_table=4, start=60, turns=0, mag=1.0, T=4, hq=32,
           kvh=8, hd=128, part=128, inter=0, dt=1, stream=0)


@pytest.mark.parametrize("kw,expect", [
    ({"T": 5}, 1001), ({"start": 61}, 1001), ({"start": -1}, 1001), ({"start": 1 << 31}, 1001),
    ({"page": 0}, 1001), ({"kvh": 0}, 1001), ({"ss": 1000}, 1001), ({"sp": 15 * 1024}, 1001),
    ({"vs": 8}, 1001), ({"pages": -1}, 1001), ({"n_table": 1 << 32}, 1001), ({"v": 8}, 1002),
    ({"vs": 1028}, 1002), ({"kc": 8}, 1002), ({"ss": 1028, "sp": 16 * 1028}, 1002),
    ({"table": 2}, 1002), ({"T": 0}, 0),
])
def test_rotary_append_entry_point(kw, expect):
    assert _c("tm_rotary_append", APP, kw) == expect


SAMPLE = dict(logits=0, dt=0, N=2, V=100, rs=100, u=0, ts=0, t=1.0, ks=0, k=0, ps=0, p=1.0, ms=0,
              m=0.0, tokens=0, probs=0, prs=0, stream=0)


@pytest.mark.parametrize("kw,expect", [
    ({"dt": 3}, 1003), ({"t": -1.0}, 1003), ({"t": math.inf}, 1003), ({"t": math.nan}, 1003),
    ({"k": -1}, 1003), ({"p": 1.5}, 1003), ({"p": math.nan}, 1003), ({"m": -0.5}, 1003),
    ({"N": -1}, 1001), ({"V": 0}, 1001), ({"V": 262145, "rs": 262145}, 1001), ({"rs": -1}, 1001),
    ({"probs": 4, "prs": 99}, 1001), ({"logits": 2}, 1002), ({"u": 2}, 1002), ({"tokens": 4}, 1002),
    ({"probs": 2, "prs": 100}, 1002), ({"ks": 2}, 1002), ({"N": 0}, 0),
])
def test_sample_entry_point(kw, expect):
    assert _c("tm_sample_tokens", SAMPLE, kw) == expect


def test_fast_calls_match_ctypes():
    """The CPython binding takes the same arguments and gives the same status."""
    for name, args in (("tm_rms_norm", NORM), ("tm_rms_norm_fp8", FP8), ("tm_rotary", ROT),
                       ("tm_rotary_append", APP), ("tm_sample_tokens", SAMPLE)):
        fast = _capi.entry(name)
        assert type(fast).__name__ == "builtin_function_or_method"
        bad = {**args, "T" if "T" in args else "N": -1}
        assert fast(*bad.values()) == 1001
        with pytest.raises(TypeError):
            fast(1, 2)
        with pytest.raises(TypeError):
            fast(*["x"] * len(args))
