"""CPU: what branch attention, beam selection, attention mass and eviction refuse, in Python
and at the C entry points (which check before any launch), the lists of a branch plan, and
the host's side of a branch cache."""

from __future__ import annotations

import ctypes

import pytest
import torch

from treemoe_spec_amd import _capi
from treemoe_spec_amd.kernels import beam_search as bs
from treemoe_spec_amd.kernels import branch_attention as ba
from treemoe_spec_amd.kernels import cache_eviction as ce
from treemoe_spec_amd.kv_cache import BranchCache, MixtralConfig, PagedKVCache

BF = torch.bfloat16
CFG = MixtralConfig(num_layers=2, num_kv_heads=2, head_dim=64)


@pytest.fixture()
def calls(monkeypatch):
    """Launches recorded instead of made, on CPU tensors."""
    done = []
    monkeypatch.setattr(_capi, "require", lambda *a, **k: None)
    monkeypatch.setattr(_capi, "launch", lambda *a: done.append(a))
    monkeypatch.setattr(_capi, "used_by", lambda *a: None)
    return done


def _setup(rows=3, capacity=20, seq_len=40, beams=1, dtype=BF):
    kv = PagedKVCache(CFG, 8, device="cpu", dtype=dtype, page_size=16, tree_size=1)
    kv._ensure_capacity(seq_len)
    kv.seq_len = seq_len
    br = BranchCache(CFG, rows, capacity, device="cpu", dtype=dtype, beams=beams)
    return kv, br


def _qkv(t, dtype=BF, heads=8):
    return (torch.zeros(t, heads, 64, dtype=dtype), torch.zeros(t, 2, 64, dtype=dtype),
            torch.zeros(t, 2, 64, dtype=dtype))


# ------------------------------------------------------------------- plans --

def test_plan_lists():
    p = ba.BranchPlan([3, 0, 20, 1], num_heads=8, num_kv_heads=2, device="cpu")
    assert (p.num_units, p.total, p.max_count) == (3, 24, 20)   # 80 rows: tiles of 128
    assert p.lists[:3].tolist() == [[0, 0, 0, 3], [2, 0, 3, 20], [3, 0, 23, 1]]
    tokens = p.lists[3:].tolist()
    assert len(tokens) == 24 and tokens[3:5] == [[2, 0, 1, 0], [2, 1, 1, 0]]
    assert tokens[23] == [3, 0, 2, 0] and p.device_counts.tolist() == [3, 0, 20, 1]
    p = ba.BranchPlan([100, 8], num_heads=8, num_kv_heads=2, device="cpu")   # several tiles
    assert p.lists[:5].tolist() == [[0, i, 0, 100] for i in range(4)] + [[1, 0, 100, 8]]
    p = ba.BranchPlan([], num_heads=8, num_kv_heads=2, device="cpu")
    assert (p.num_units, p.total, p.max_count) == (0, 0, 0)


@pytest.mark.parametrize("counts,heads", [([-1], (8, 2)), ([1.5], (8, 2)), ([1], (8, 3)),
                                          ([1], (1, 2)), ([1 << 25], (8, 2))])
def test_plan_refusals(counts, heads):
    with pytest.raises((ValueError, TypeError)):
        ba.BranchPlan(counts, num_heads=heads[0], num_kv_heads=heads[1], device="cpu")


def test_plan_that_32_bits_cannot_hold():
    with pytest.raises(RuntimeError, match="size"):
        ba.BranchPlan([1 << 24] * 40, num_heads=1024, num_kv_heads=1, device="cpu")


# ------------------------------------------------------------ branch cache --

def test_branch_cache_lengths(calls):
    _, br = _setup(rows=4, capacity=10)
    assert br.rows == 4 and br.capacity == 10 and br.origin is None
    br.advance(3)
    br.advance(ba.BranchPlan([1, 0, 7, 2], num_heads=8, num_kv_heads=2, device="cpu"))
    assert br.host_lengths == [4, 3, 10, 5] and br.longest == 10 and len(calls) == 2
    with pytest.raises(ValueError, match="capacity"):
        br.advance()
    with pytest.raises(ValueError, match="plan for 4"):
        br.advance(ba.BranchPlan([1], num_heads=8, num_kv_heads=2, device="cpu"))
    with pytest.raises(ValueError):
        br.advance(-1)
    with pytest.raises(TypeError):
        br.advance(1.0)
    br.set_lengths([4, 0, 2, 5])
    assert br.longest == 5 and br.lengths.tolist() == [4, 0, 2, 5]
    for bad in ([5, 0, 2, 5], [4, 0, 2], [-1, 0, 2, 5]):
        with pytest.raises(ValueError):
            br.set_lengths(bad)
    br.reset()
    assert br.host_lengths == [0] * 4 == br.lengths.tolist()


def test_beams_are_cut_alike(calls):
    _, br = _setup(rows=6, capacity=8, beams=3)
    assert br.origin.tolist() == [[b] * 8 for b in range(6)]
    br.advance(5)
    br.set_lengths([3, 3, 3, 5, 5, 5])
    with pytest.raises(ValueError, match="same number"):
        br.set_lengths([3, 2, 3, 5, 5, 5])
    with pytest.raises(ValueError, match="parents"):
        br.reorder(torch.zeros(3, 2, dtype=torch.int32))
    br.host_lengths[0] = 1
    with pytest.raises(ValueError, match="same number"):
        br.reorder(torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="beams > 1"):
        _setup()[1].reorder(torch.zeros(3, 1, dtype=torch.int32))


@pytest.mark.parametrize("kw", [{"rows": 0}, {"capacity": 0}, {"beams": 0},
                                {"rows": 5, "beams": 2}])
def test_branch_cache_refusals(kw):
    with pytest.raises(ValueError):
        BranchCache(CFG, **{"rows": 2, "capacity": 4, **kw}, device="cpu")


# -------------------------------------------------------- branch attention --

def test_cpu_tensors_and_gradients_raise():
    kv, br = _setup()
    q, k, v = _qkv(3)
    with pytest.raises(RuntimeError, match="ROCm"):
        ba.branch_attention(q, k, v, kv, br, 0)
    with pytest.raises(RuntimeError, match="ROCm"):
        bs.beam_select(torch.zeros(2, 8), torch.zeros(1, 2))
    with pytest.raises(RuntimeError, match="ROCm"):
        bs.reorder_rows(torch.zeros(2, 8), torch.zeros(1, 2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="ROCm"):
        ce.attention_mass(q, kv, 0)
    with pytest.raises(RuntimeError, match="ROCm"):
        ce.evict(kv, torch.zeros(2, 2, 40), 10)
    with pytest.raises(RuntimeError, match="ROCm"):
        br.advance()
    fake = type("T", (), {"get_device": lambda s: 0, "requires_grad": True})()
    assert not _capi.ready(0, None, fake) and not _capi.ready(-1)


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(3, 8, 64)), ValueError),                       # float32
    (dict(q=torch.zeros(3, 8, 96, dtype=BF)), ValueError),
    (dict(q=torch.zeros(8, 3, 64, dtype=BF).transpose(0, 1)), ValueError),
    (dict(k=torch.zeros(2, 2, 64, dtype=BF)), ValueError),
    (dict(k=torch.zeros(3, 2, 64, dtype=torch.float16)), ValueError),
    (dict(v=torch.zeros(3, 1, 64, dtype=BF)), ValueError),
    (dict(k=torch.zeros(3, 3, 64, dtype=BF), v=torch.zeros(3, 3, 64, dtype=BF)), ValueError),
    (dict(layer=2), IndexError),
    (dict(layer=-3), IndexError),
    (dict(scale=0.0), ValueError),
    (dict(scale=float("nan")), ValueError),
    (dict(out=torch.zeros(3, 511, dtype=BF)), ValueError),
    (dict(plan=ba.BranchPlan([1, 1], num_heads=8, num_kv_heads=2, device="cpu")), ValueError),
    (dict(plan=ba.BranchPlan([1, 1, 1], num_heads=4, num_kv_heads=2, device="cpu")), ValueError),
    (dict(plan=ba.BranchPlan([1, 1, 2], num_heads=8, num_kv_heads=2, device="cpu")), ValueError),
])
def test_branch_attention_refusals(calls, change, error):
    kv, br = _setup()
    q, k, v = _qkv(3)
    a = dict(q=q, k=k, v=v, kv=kv, branches=br, layer=0, plan=None) | change
    with pytest.raises(error):
        ba.branch_attention(**a)
    assert not calls


def test_branch_attention_refuses_what_does_not_fit(calls):
    kv, br = _setup(rows=3, capacity=5)
    with pytest.raises(ValueError, match="give a plan"):
        ba.branch_attention(*_qkv(4), kv, br, 0)
    with pytest.raises(ValueError, match="capacity"):
        ba.branch_attention(*_qkv(18), kv, br, 0)
    br.host_lengths, br.longest = [5, 0, 0], 5
    with pytest.raises(ValueError, match="capacity"):
        ba.branch_attention(*_qkv(3), kv, br, 0)
    plan = ba.BranchPlan([0, 2, 5], num_heads=8, num_kv_heads=2, device="cpu")
    ba.branch_attention(*_qkv(7), kv, br, 0, plan)      # the full branch takes no part
    assert len(calls) == 1
    kv.block_size = 8
    with pytest.raises(ValueError, match="cache layout"):
        ba.branch_attention(*_qkv(7), kv, br, 0, plan)
    kv.block_size = 16
    br.lengths = br.lengths.long()
    with pytest.raises(ValueError, match="lengths"):
        ba.branch_attention(*_qkv(7), kv, br, 0, plan)
    for name in "kv":
        kv2, br2 = _setup()
        setattr(br2, name, torch.zeros(2, 3, 20, 2, 128, dtype=BF))
        with pytest.raises(ValueError, match="branches must be"):
            ba.branch_attention(*_qkv(3), kv2, br2, 0)


def test_no_tokens_launch_nothing(calls):
    kv, br = _setup()
    assert ba.branch_attention(*_qkv(0), kv, br, 0).shape == (0, 512)
    none = ba.BranchPlan([0, 0, 0], num_heads=8, num_kv_heads=2, device="cpu")
    assert not bool(ba.branch_attention(*_qkv(2), kv, br, 0, none).any()) and not calls


# ------------------------------------------------------------ beam search --

@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(2, 3, 8)), dict(logits=torch.zeros(5, 8)),
    dict(logits=torch.zeros(6, 8, dtype=torch.float64)), dict(logits=torch.zeros(8, 6).T),
    dict(logits=torch.zeros(6, 0)), dict(scores=torch.zeros(6)),
    dict(scores=torch.zeros(2, 3, dtype=BF)), dict(scores=torch.zeros(3, 2).T), dict(num=0),
    dict(num=65), dict(pad_token=8), dict(pad_token=-1), dict(finished=torch.zeros(2, 3)),
    dict(finished=torch.zeros(3, 2).bool()), dict(finished=torch.zeros(3, 2).bool().T),
    dict(logits=torch.zeros(65, 8), scores=torch.zeros(1, 65)),
    dict(logits=torch.zeros(1, 1).expand(6, (1 << 18) + 1)),
])
def test_beam_select_refusals(calls, change):
    a = dict(logits=torch.zeros(6, 8), scores=torch.zeros(2, 3)) | change
    with pytest.raises(ValueError):
        bs.beam_select(a.pop("logits"), a.pop("scores"), **a)
    assert not calls


@pytest.mark.parametrize("x,parents,kw", [
    (torch.zeros(6, 8), torch.zeros(2, 3), {}),
    (torch.zeros(6, 8), torch.zeros(6, dtype=torch.int32), {}),
    (torch.zeros(5, 8), torch.zeros(2, 3, dtype=torch.int32), {}),
    (torch.zeros(65, 8), torch.zeros(1, 65, dtype=torch.int32), {}),
    (torch.zeros(8, 6).T, torch.zeros(2, 3, dtype=torch.int32), {}),
    (torch.zeros(6, 8), torch.zeros(3, 2, dtype=torch.int32).T, {}),
    (torch.zeros(1, 8).expand(6, 8), torch.zeros(2, 3, dtype=torch.int32), {}),
    (torch.zeros(6, 8), torch.zeros(2, 3, dtype=torch.int32), {"columns": 2}),
    (torch.zeros(6, 8), torch.zeros(2, 3, dtype=torch.int32), {"out": torch.zeros(6, 7)}),
    (torch.zeros(6, 8), torch.zeros(2, 3, dtype=torch.int32), {"out": torch.zeros(6, 8).int()}),
    (torch.zeros(6, 8), torch.zeros(2, 3, dtype=torch.int32),
     {"out": torch.zeros(6, 8), "columns": 9}),
])
def test_reorder_refusals(calls, x, parents, kw):
    with pytest.raises(ValueError):
        bs.reorder_rows(x, parents, **kw)
    assert not calls


def test_reorder_over_itself_shifted(calls):
    x = torch.zeros(6, 16)
    parents = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="lie apart"):
        bs.reorder_rows(x[:3, :8], parents[:1], out=x.flatten()[:24].view(3, 8))
    bs.reorder_rows(x, parents, out=x, columns=5)
    name, _, src, stride, dst, _, width, *_ = calls[0]
    assert name == "tm_reorder_rows" and src == dst and stride == 64 and width == 20


# --------------------------------------------------------------- eviction --

@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(41, 8, 64, dtype=BF)), ValueError),
    (dict(q=torch.zeros(3, 7, 64, dtype=BF)), ValueError),
    (dict(q=torch.zeros(3, 8, 128, dtype=BF)), ValueError),
    (dict(q=torch.zeros(3, 8, 64, dtype=torch.float16)), ValueError),
    (dict(layer=2), IndexError),
    (dict(scale=-1.0), ValueError),
    (dict(mass=torch.zeros(2, 39)), ValueError),
    (dict(mass=torch.zeros(3, 40)), ValueError),
    (dict(mass=torch.zeros(2, 40, dtype=BF)), ValueError),
    (dict(mass=torch.zeros(40, 2).T), ValueError),
    (dict(mass=torch.zeros(1, 40).expand(2, 40)), ValueError),
    (dict(out=torch.zeros(2, 39)), ValueError),
])
def test_mass_refusals(calls, change, error):
    kv, _ = _setup()
    a = dict(q=torch.zeros(3, 8, 64, dtype=BF), kv=kv, layer=0) | change
    with pytest.raises(error):
        ce.attention_mass(**a)
    assert not calls


@pytest.mark.parametrize("change", [
    dict(keep=-1), dict(keep=10, recent=8, sinks=3), dict(recent=-1), dict(sinks=-1),
    dict(mass=torch.zeros(2, 2, 39)), dict(mass=torch.zeros(1, 2, 40)),
    dict(mass=torch.zeros(2, 2, 40, dtype=torch.float64)),
    dict(mass=torch.zeros(2, 40, 2).transpose(1, 2)),
    dict(positions=torch.zeros(2, 2, 10, dtype=torch.int32)),
    dict(positions=torch.zeros(2, 2, 41, dtype=torch.int32), next_position=100),
    dict(positions=torch.zeros(2, 2, 10, dtype=torch.int64), next_position=100),
    dict(next_position=39), dict(next_position=2 ** 31),
])
def test_evict_refusals(calls, change):
    kv, _ = _setup()
    a = dict(kv=kv, mass=torch.zeros(2, 2, 40), keep=20) | change
    with pytest.raises(ValueError):
        ce.evict(**a)
    assert not calls and kv.seq_len == 40


def test_evict_sets_the_length(calls):
    kv, _ = _setup()
    mass, pos = ce.evict(kv, torch.zeros(2, 2, 64), 20, recent=3)
    assert kv.seq_len == 20 and mass.shape == (2, 2, 64) and pos.shape == (2, 2, 20)
    assert len(kv.block_table) == 3                      # the pages stay mapped
    mass, pos = ce.evict(kv, mass, 30, recent=3)
    assert kv.seq_len == 20 and pos.shape == (2, 2, 20)
    kv.page = kv.k[:, :, :, :, :7]
    kv.k = kv.v = torch.zeros(2, 8, 16, 2, 7, dtype=BF)
    with pytest.raises(ValueError, match="16 bytes"):
        ce.evict(kv, torch.zeros(2, 2, 64), 10)


# ----------------------------------------------------------------- C ABI --

BIG = 1 << 40


def _branch_args(**kw):
    a = dict(q=0, q_stride=512, k=0, k_stride=128, v=0, v_stride=128, T=3, k_cache=0, v_cache=0,
             stride_page=16 * 128, stride_slot=128, page_size=16, cache_pages=8, block_table=0,
             num_table_pages=3, seq_len=40, k_rows=0, v_rows=0, stride_row=20 * 128,
             stride_pos=128, rows=3, capacity=20, origin=0, origin_stride=0, lengths=0, longest=5,
             units=0, num_units=3, tokens=0, max_count=1, Hq=8, kvh=2, hd=64, scale=0.125,
             dtype=1, out=0, out_stride=512, workspace=0, workspace_bytes=BIG, stream=0)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(T=0), 0), (dict(hd=96), 1001), (dict(Hq=7), 1001), (dict(dtype=0), 1003),
    (dict(scale=0.0), 1003), (dict(scale=float("inf")), 1003), (dict(workspace_bytes=0), 1001),
    (dict(T=4), 1001), (dict(num_units=2), 1001), (dict(max_count=0), 1001),
    (dict(longest=21), 1001), (dict(longest=-1), 1001), (dict(seq_len=49), 1001),
    (dict(seq_len=-1), 1001), (dict(page_size=24), 1001), (dict(cache_pages=0), 1001),
    (dict(stride_slot=64), 1001), (dict(stride_page=100), 1001), (dict(stride_row=100), 1001),
    (dict(stride_pos=64), 1001), (dict(q_stride=100), 1001), (dict(out_stride=100), 1001),
    (dict(k_stride=64), 1001), (dict(v_stride=64), 1001), (dict(capacity=-1), 1001),
    (dict(origin=16, origin_stride=19), 1001), (dict(units=16), 1003), (dict(tokens=16), 1003),
    (dict(units=16, tokens=16, num_units=0), 1001), (dict(units=16, tokens=16, num_units=4), 1001),
    (dict(q=8), 1002), (dict(k=8), 1002), (dict(v=2), 1002), (dict(out=8), 1002),
    (dict(k_cache=8), 1002), (dict(v_rows=8), 1002), (dict(q_stride=516), 1002),
    (dict(lengths=2), 1002), (dict(workspace=8), 1002), (dict(origin=2, origin_stride=20), 1002),
    (dict(units=8, tokens=16, num_units=1), 1002),
])
def test_branch_attention_statuses(kw, status):
    assert _capi.lib().tm_branch_attention(*_branch_args(**kw)) == status


def test_workspaces_and_other_statuses():
    lib = _capi.lib()
    n = ctypes.c_int64()
    # 3 branches of one token over 40 keys: one range of shared keys with 12 rows, and one of own
    # keys with 4 rows a branch; 66 floats a row
    assert lib.tm_branch_workspace(3, 3, 1, 40, 5, 8, 2, 64, ctypes.byref(n)) == 0
    assert n.value == 4 * 2 * 66 * (12 + 3 * 4)
    assert lib.tm_branch_workspace(3, 3, 1, 0, 5, 8, 2, 64, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.tm_branch_workspace(3, 3, 4, 0, 5, 8, 2, 64, ctypes.byref(n)) == 1001
    assert lib.tm_branch_workspace(3, 3, 1, 40, 5, 8, 2, 64, None) == 1003
    assert lib.tm_branch_advance(None, None, -1, 3, 20, None, 0, None) == 1001
    assert lib.tm_branch_advance(None, None, 1, 3, 20, 16, 19, None) == 1001
    assert lib.tm_branch_advance(None, None, 1, 0, 20, None, 0, None) == 0
    assert lib.tm_branch_advance(2, None, 1, 3, 20, None, 0, None) == 1002
    assert lib.tm_branch_plan(None, 1, 8, 2, None, 0, None, 0, None) == 1003
    sizes = (ctypes.c_int64 * 3)()
    one = (ctypes.c_int64 * 1)(5)
    assert lib.tm_branch_plan(one, 1, 8, 2, ctypes.addressof(sizes), 0, None, 0, sizes) == 1001

    assert lib.tm_beam_workspace(2, 4, 5000, 8, ctypes.byref(n)) == 0
    assert n.value == 2 * 4 * 2 * (8 * 8 + 12)
    for bad in ((-1, 4, 10, 1), (2, 0, 10, 1), (2, 65, 10, 1), (2, 4, 0, 1), (2, 4, 10, 65),
                (2, 4, (1 << 18) + 1, 1), (1 << 20, 4, 10, 1)):
        assert lib.tm_beam_workspace(*bad, ctypes.byref(n)) == 1001
    assert lib.tm_beam_workspace(2, 4, 10, 1, None) == 1003

    def select(logits=0, dtype=1, stride=10, pad=0, ws=0, nbytes=BIG, tokens=0, groups=2):
        return lib.tm_beam_select(logits, dtype, groups, 4, 10, stride, 0, 0, pad, 3, 0, 0, tokens,
                                  ws, nbytes, None)

    assert select(dtype=7) == 1003 and select(pad=10) == 1001 and select(stride=-1) == 1001
    assert select(nbytes=0) == 1001 and select(logits=1) == 1002 and select(ws=4) == 1002
    assert select(tokens=4) == 1002 and select(groups=0) == 0

    def reorder(x=0, xs=64, out=4096, outs=64, width=64, parents=0, ps=4, groups=2, beams=4):
        return lib.tm_reorder_rows(x, xs, out, outs, width, parents, ps, groups, beams, None)

    assert reorder(beams=65) == 1001 and reorder(groups=65536) == 1001
    assert reorder(xs=60) == 1001 and reorder(outs=60) == 1001 and reorder(ps=3) == 1001
    assert reorder(parents=2) == 1002 and reorder(x=4096, xs=80) == 1003
    assert reorder(width=0) == 0 and reorder(groups=0) == 0
    assert reorder(width=1 << 39, xs=1 << 39, outs=1 << 39) == 1001    # more than a grid

    assert lib.tm_mass_workspace(1, 7777, 32, 8, 128, ctypes.byref(n)) == 0
    assert n.value == 31 * 8 * 4 * 8 + 8 * 4 * 7808 * 4      # statistics, and the scores
    assert lib.tm_mass_workspace(5, 4, 32, 8, 128, ctypes.byref(n)) == 1001
    assert lib.tm_mass_workspace(1, 4, 32, 8, 128, None) == 1003

    def mass(q=0, qs=512, t=3, page=16, pages=8, table=0, mapped=3, seq=40, slot=128, hd=64,
             scale=0.1, dtype=1, before=0, bs_=40, out=0, ms=40, ws=0, nbytes=BIG):
        return lib.tm_attention_mass(q, qs, t, 0, page * slot, slot, page, pages, table, mapped,
                                     seq, 8, 2, hd, scale, dtype, before, bs_, out, ms, ws,
                                     nbytes, None)

    assert mass(dtype=0) == 1003 and mass(scale=-1.0) == 1003 and mass(hd=32) == 1001
    assert mass(seq=49) == 1001 and mass(page=10) == 1001 and mass(pages=0) == 1001
    assert mass(slot=64) == 1001 and mass(qs=100) == 1001 and mass(ms=39) == 1001
    assert mass(before=16, bs_=39) == 1001 and mass(nbytes=0) == 1001 and mass(q=8) == 1002
    assert mass(out=2) == 1002 and mass(ws=4) == 1002 and mass(seq=0, t=0) == 0

    assert lib.tm_evict_workspace(2, 2, 40, 30, ctypes.byref(n)) == 0
    assert n.value == 4 * (4 + 2 * 4 * 10)
    for bad in ((-1, 2, 40, 30), (2, 0, 40, 30), (2, 2, 40, 41), (2, 2, 40, -1),
                (65536, 1, 40, 30), (2, 2, 1 << 25, 30)):
        assert lib.tm_evict_workspace(*bad, ctypes.byref(n)) == 1001

    def evict(k=0, elem=2, layer=8 * 16 * 128, slot=128, hd=64, page=16, pages=8, mapped=3, seq=40,
              keep=20, columns=40, pos=0, recorded=0, nxt=40, recent=0, sinks=0, mass_out=0,
              nbytes=BIG, layers=2):
        return lib.tm_evict(k, 0, elem, layers, layer, page * slot, slot, 2, hd, page, pages, 0,
                            mapped, seq, keep, 0, 80, 40, columns, pos, 0, 0, recorded, nxt,
                            recent, sinks, mass_out, 0, 0, nbytes, None)

    assert evict(elem=3) == 1003 and evict(keep=41) == 1001 and evict(columns=39) == 1001
    assert evict(recorded=41) == 1001 and evict(recorded=5) == 1001 and evict(nxt=39) == 1001
    assert evict(nxt=1 << 31) == 1001 and evict(recent=-1) == 1001 and evict(sinks=-1) == 1001
    assert evict(nbytes=0) == 1001 and evict(mapped=2) == 1001 and evict(page=10) == 1001
    assert evict(slot=64) == 1001 and evict(layer=100) == 1001 and evict(hd=4, slot=8) == 1002
    assert evict(k=8) == 1002 and evict(mass_out=2) == 1002 and evict(layers=0) == 0


def test_binding_agrees_with_ctypes():
    fast = _capi.layer_binding()
    assert fast is not None
    n = ctypes.c_int64()
    for name, sizes in (("branch_workspace", (64, 64, 1, 4096, 700, 32, 8, 128)),
                        ("beam_workspace", (32, 8, 131072, 16)),
                        ("mass_workspace", (4096, 4096, 32, 8, 128)),
                        ("evict_workspace", (32, 8, 8192, 1024)),
                        ("prompt_cached_workspace", (1, 7777, 32, 8, 128))):
        assert getattr(_capi.lib(), "tm_" + name)(*sizes, ctypes.byref(n)) == 0
        assert getattr(fast, name)(*sizes) == (0, n.value) and n.value > 0
        assert _capi.workspace_bytes(name, *sizes) == n.value
        with pytest.raises(TypeError):
            getattr(fast, name)(1)
    with pytest.raises(RuntimeError, match="status 1001"):
        _capi.workspace_bytes("evict_workspace", 1, 1, 5, 6)
