"""Norm, rotary, prompt attention and sampling where element offsets pass 31 and 32 bits:
the same bits as on compact tensors."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
STEP = 2 ** 31 + 2 ** 12  # elements from row to row: the third row lies past 2^32


def _say(msg):
    print(msg, flush=True)


@pytest.fixture(scope="module")
def buffers():
    """Two buffers of three far rows each."""
    got = [torch.empty(2 * STEP + 2 ** 21, dtype=BF, device="cuda") for _ in range(2)]
    yield got
    got.clear()
    torch.cuda.empty_cache()


def _far(buf, like):
    """A copy of ``like`` [3, ...] in ``buf`` with its rows STEP elements apart."""
    view = buf.as_strided(like.shape, (STEP,) + like.stride()[1:])
    view.copy_(like)
    return view


def _rand(*shape, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(BF).cuda()


def test_norm(buffers):
    from treemoe_spec_amd.kernels.rms_norm import rms_norm

    _say("far norm")
    x, w = _rand(3, 4096), _rand(4096, seed=2)
    want = rms_norm(x, w)
    out = _far(buffers[1], torch.zeros_like(x))
    rms_norm(_far(buffers[0], x), w, out=out)
    assert torch.equal(out, want)


def test_rotary(buffers):
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_embed

    _say("far rotary")
    plan = RotaryPlan(128, 1e6)
    q, pos = _rand(3, 8, 128), torch.tensor([5, 2 ** 40, 7]).cuda()
    want = rotary_embed(q, None, pos, plan)[0]
    out = _far(buffers[1], torch.zeros_like(q))
    rotary_embed(_far(buffers[0], q), None, pos, plan, q_out=out)
    assert torch.equal(out, want)


def test_sample(buffers):
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens

    _say("far sampling")
    for v in (32000, 100000):
        logits, u = _rand(3, v) * 3, torch.tensor([0.2, 0.9, 0.6]).cuda()
        want = sample_tokens(logits, u, top_p=0.9)
        assert torch.equal(sample_tokens(_far(buffers[0], logits), u, top_p=0.9), want)


@pytest.mark.parametrize("hq,kvh", [(8, 2), (128, 1)])
def test_queries(buffers, hq, kvh):
    """Query and output rows far apart: few rows, and tiles."""
    from treemoe_spec_amd.kernels.prompt_attention import PromptPlan, prompt_attention

    _say(f"far queries heads={hq}/{kvh}")
    plan = PromptPlan([3], [900], num_heads=hq, num_kv_heads=kvh)
    q, k, v = _rand(3, hq, 128), _rand(900, kvh, 128, seed=2), _rand(900, kvh, 128, seed=3)
    want = prompt_attention(q, k, v, plan)
    out = _far(buffers[1], torch.zeros_like(want))
    prompt_attention(_far(buffers[0], q), k, v, plan, out=out)
    assert torch.equal(out, want)


@pytest.mark.parametrize("t", [3, 40, 600])
def test_keys(buffers, t):
    """A sequence behind 2^32 elements of keys."""
    from treemoe_spec_amd.kernels.prompt_attention import PromptPlan, prompt_attention

    _say(f"far keys t={t}")
    before = 2 ** 32 // 256
    k, v = (b[:(before + 700) * 256].view(-1, 2, 128) for b in buffers)
    k[before:], v[before:] = _rand(700, 2, 128, seed=2), _rand(700, 2, 128, seed=3)
    q = _rand(t, 8, 128)
    lens = dict(num_heads=8, num_kv_heads=2)
    want = prompt_attention(q, k[before:].clone(), v[before:].clone(),
                            PromptPlan([t], [700], **lens))
    skipped = [0, 0]  # sequences of keys that no query asks for
    got = prompt_attention(q, k, v, PromptPlan(skipped + [t], [before // 2] * 2 + [700], **lens))
    assert torch.equal(got, want)


@pytest.mark.parametrize("page", [16, 64])
def test_pages(buffers, page):
    """Pages at the end of a cache of more than 2^32 elements: appended to and read."""
    from treemoe_spec_amd.kernels.prompt_attention import prompt_attention_cached
    from treemoe_spec_amd.kernels.rotary import RotaryPlan, rotary_append
    from treemoe_spec_amd.kv_cache import MixtralConfig, PagedKVCache

    _say(f"far pages of {page}")
    pages = 2 ** 32 // (page * 256) + 100
    cfg = MixtralConfig(num_layers=1, num_kv_heads=2, head_dim=128)
    small = PagedKVCache(cfg, 60 if page == 16 else 16, page_size=page, tree_size=1)
    large = PagedKVCache(cfg, 2, page_size=page, tree_size=1)
    large.k, large.v = (b[:pages * page * 256].view(1, pages, page, 2, 128) for b in buffers)
    large._free = list(range(pages - 60, pages))
    plan = RotaryPlan(128, 1e6)
    for start, t in ((0, 650), (650, 40), (690, 1)):
        q, k, v = _rand(t, 8, 128, seed=t), _rand(t, 2, 128, seed=t + 1), _rand(t, 2, 128, seed=t + 2)
        outs = []
        for kv in (small, large):
            qr = rotary_append(q, k, v, plan, kv, 0, start)
            outs.append(prompt_attention_cached(qr, kv, 0))
        assert torch.equal(outs[0], outs[1])
    assert min(large.block_table) * page * 256 > 2 ** 32
    for kv in (small, large):
        kv.seq_len = 691
    assert all(torch.equal(a, b) for a, b in zip(small.gather(0), large.gather(0)))
