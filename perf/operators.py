"""Cases of the operators around the verification path: what a prompt goes through
before the first tree, and the sampling of the tokens that a tree is drafted from.

Four kinds:

  norm    ``rms_norm`` (with the residual's addition) and ``rms_norm_fp8``
  rotary  ``rotary_embed`` of queries and keys, and ``rotary_append``, which
          also stores the keys and values in the paged cache
  attn    ``prompt_attention`` over packed sequences, and
          ``prompt_attention_cached`` over the paged cache, down to one token
  sample  ``sample_tokens``, with the filtered distribution or without

With ``own`` false ``run`` computes the same outputs in elementary torch
operations, in 32 bits (64 for rotary angles and for sampling's sums).
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5
GROUP = 128            # columns of one 8-bit scale
MAX_TOKENS = 8192
MAX_VOCAB = 131072


def _norm(name, tokens, hidden, dtype="bf16", residual=True, out="same"):
    """out: "same" type as x, or 8 bits with a scale for each "row" or "group"."""
    c = {"kind": "norm", "tokens": tokens, "hidden": hidden, "dtype": dtype,
         "residual": residual, "out": out}
    return {"name": name, **c} if name else c


def _rotary(name, tokens, heads=32, kv_heads=8, hd=128, dtype="bf16", layout="half", part=128,
            scaling="none", first=0, page=0):
    """page: 0 for rotary_embed, else the page size of the cache appended to.
    first: the position of the first token; part: the head's rotated elements."""
    c = {"kind": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "hd": hd,
         "dtype": dtype, "layout": layout, "part": part, "scaling": scaling, "first": first,
         "page": page}
    return {"name": name, **c} if name else c


def _attn(name, lengths, past="0", heads=32, kv_heads=8, hd=128, dtype="bf16", page=0):
    """lengths: each sequence's queries, comma-separated; past: each sequence's
    keys before its first query.  page: 0 for packed keys, else the page size of
    the cache that one sequence's keys lie in."""
    c = {"kind": "attn", "lengths": lengths, "past": past, "heads": heads, "kv_heads": kv_heads,
         "hd": hd, "dtype": dtype, "page": page}
    return {"name": name, **c} if name else c


def _sample(name, rows, vocab=32000, dtype="fp32", temperature=1.0, top_k=0, top_p=1.0,
            min_p=0.0, probs=False):
    c = {"kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype,
         "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
         "probs": probs}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the norm between attention and experts for one decoded token
        _norm("norm_1_token", 1, 4096),
        # the same for a long prompt of odd length
        _norm("norm_6011_prompt", 6011, 4096),
        # a norm whose output feeds an 8-bit product, a scale for every 128 columns
        _norm("norm_2048_fp8_groups", 2048, 4096, out="group"),
        # queries and keys of a 64-node tree, positions by depth
        _rotary("rotary_64_tree", 64, first=4096),
        # a prompt's chunk on its way into the cache, positions stretched for a long context
        _rotary("rotary_append_5003", 5003, scaling="yarn", first=3000, page=16),
        # the longest prompt of the configuration
        _attn("attn_8192_prompt", "8192"),
        # prompts of many users packed together, odd lengths down to one token
        _attn("attn_packed_fp16", "1,17,64,333,517,1000,2048,129,63,700,1,255", past="0",
              dtype="fp16"),
        # the second chunk of a prompt over what the cache holds already
        _attn("attn_517_over_4096_cached", "517", past="4096", page=16),
        # one decoded token over a long cache of odd length
        _attn("attn_1_token_cached", "1", past="7776", page=64),
        # the first token after a prompt
        _sample("sample_1_row", 1, temperature=0.8, top_k=50, top_p=0.9),
        # a tree's draft tokens and the distributions that their verification takes
        _sample("sample_64_draft_probs", 64, dtype="bf16", top_p=0.95, min_p=0.02, probs=True),
        # a large batch over a large vocabulary
        _sample("sample_256_large_vocab", 256, vocab=131072, temperature=0.7, top_p=0.9),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _lengths(rng, total):
    """Random lengths of a batch with at most `total` tokens."""
    out, left = [], total
    while left > 0 and len(out) < 24:
        out.append(min(left, _log_int(rng, 1, max(1, total))))
        left -= out[-1]
    return out


def draw(rng):
    kind = rng.choice(["norm", "rotary", "attn", "attn", "sample"])
    if kind == "norm":
        hidden = rng.choice([4096, 4096, 1024, 512, GROUP * rng.randint(1, 64)])
        out = rng.choice(["same", "same", "row", "group"])
        if out == "same":
            hidden = rng.choice([hidden, _log_int(rng, 65, 8192)])
        return _norm(None, _log_int(rng, 1, MAX_TOKENS), hidden,
                     dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                     residual=rng.choice([True, True, False]), out=out)
    if kind == "rotary":
        heads, kv_heads = rng.choice([(32, 8), (8, 2), (4, 4), (16, 2)])
        hd = rng.choice([128, 128, 64])
        return _rotary(None, _log_int(rng, 1, MAX_TOKENS - 200), heads, kv_heads, hd,
                       dtype=rng.choice(["bf16", "bf16", "fp16"]),
                       layout=rng.choice(["half", "interleaved"]),
                       part=rng.choice([hd, hd, hd // 2]),
                       scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                       first=_log_int(rng, 1, 200000), page=rng.choice([0, 16, 64]))
    if kind == "attn":
        heads, kv_heads = rng.choice([(32, 8), (32, 8), (8, 2), (4, 4), (16, 2)])
        hd, dtype = rng.choice([128, 128, 64]), rng.choice(["bf16", "bf16", "fp16"])
        if rng.random() < 0.5:
            tokens = rng.choice([1, _log_int(rng, 1, 2000)])
            return _attn(None, str(tokens), str(_log_int(rng, 1, 8000 - tokens)), heads, kv_heads,
                         hd, dtype, page=rng.choice([16, 64]))
        lengths = _lengths(rng, _log_int(rng, 1, 6000))
        past = [rng.choice([0, 0, _log_int(rng, 1, 200)]) for _ in lengths]
        return _attn(None, ",".join(map(str, lengths)), ",".join(map(str, past)), heads, kv_heads,
                     hd, dtype)
    vocab = rng.choice([32000, _log_int(rng, 1000, MAX_VOCAB)])
    return _sample(None, _log_int(rng, 1, 128), vocab, dtype=rng.choice(["fp32", "bf16", "fp16"]),
                   temperature=rng.choice([1.0, round(rng.uniform(0.3, 1.5), 3)]),
                   top_k=rng.choice([0, 0, 40, _log_int(rng, 1, 2000)]),
                   top_p=rng.choice([1.0, 0.9, round(rng.uniform(0.3, 0.99), 3)]),
                   min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 4)]),
                   probs=rng.choice([False, True]))


# ------------------------------------------------------------------ inputs --

class _Cache:
    """A paged cache with the attributes that the operators use: pages in a
    random order, page 0 kept for a tree."""

    def __init__(self, positions, page, kv_heads, hd, dtype, g):
        count = -(-positions // page)
        pages = count + 3
        shape = (1, pages, page, kv_heads, hd)
        self.k = torch.randn(shape, generator=g, device=DEV).to(dtype)
        self.v = torch.randn(shape, generator=g, device=DEV).to(dtype)
        order = (torch.randperm(pages - 1, generator=g, device=DEV) + 1).tolist()
        self.block_size, self.tree_block = page, 0
        self.block_table, self._free = order[:count], order[count:]
        self.seq_len = positions
        # the block table on the device and the flat slot of every position
        self.table = torch.tensor(self.block_table, device=DEV)
        at = torch.arange(positions, device=DEV)
        self.slots = self.table[at // page] * page + at % page

    def _ensure_capacity(self, positions):
        while len(self.block_table) * self.block_size < positions:
            self.block_table.append(self._free.pop())


def _ints(text, count=None):
    v = [int(x) for x in text.split(",")]
    return v * (count // len(v)) if count else v


SCALINGS = {
    "none": None,
    "linear": {"type": "linear", "factor": 4.0},
    "ntk": {"type": "ntk", "factor": 4.0},
    "yarn": {"type": "yarn", "factor": 8.0, "original_max_position": 8192, "beta_fast": 32.0,
             "beta_slow": 1.0},
}
THETA = 1e6


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = SimpleNamespace(**case)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    s = {"case": c}
    if c.kind == "norm":
        dt = DTYPES[c.dtype]
        s["x"] = (rnd(c.tokens, c.hidden) * 0.7).to(dt)
        s["weight"] = (1.0 + 0.1 * rnd(c.hidden)).to(dt)
        s["residual"] = (rnd(c.tokens, c.hidden) * 2.0).to(dt) if c.residual else None
    elif c.kind == "rotary":
        dt = DTYPES[c.dtype]
        # one projection's output holds q, k and v side by side
        width = (c.heads + 2 * c.kv_heads) * c.hd
        qkv = rnd(c.tokens, width).to(dt)
        q, k, v = qkv.split([c.heads * c.hd, c.kv_heads * c.hd, c.kv_heads * c.hd], 1)
        s["q"] = q.unflatten(1, (c.heads, c.hd))
        s["k"] = k.unflatten(1, (c.kv_heads, c.hd))
        s["v"] = v.unflatten(1, (c.kv_heads, c.hd))
        if c.page:
            s["positions"] = torch.arange(c.tokens, device=DEV) + c.first
            s["kv"] = _Cache(c.first + c.tokens, c.page, c.kv_heads, c.hd, dt, g)
        else:
            # a tree's nodes: the position goes by the depth
            depth = torch.randint(0, 9, (c.tokens,), generator=g, device=DEV)
            s["positions"] = c.first + depth
        if own:
            from treemoe_spec_amd.kernels.rotary import RotaryPlan
            s["plan"] = RotaryPlan(c.hd, THETA, rotary_dim=c.part,
                                   interleaved=c.layout == "interleaved",
                                   scaling=SCALINGS[c.scaling], device=DEV)
    elif c.kind == "attn":
        dt = DTYPES[c.dtype]
        lens = _ints(c.lengths)
        past = _ints(c.past, len(lens) if "," not in c.past else None)
        total = sum(lens)
        s["q"] = (rnd(total, c.heads, c.hd) * 2.0).to(dt)
        ln, pa = torch.tensor(lens, device=DEV), torch.tensor(past, device=DEV)
        ids = torch.arange(len(lens), device=DEV)
        s["q_seq"] = ids.repeat_interleave(ln)
        s["q_pos"] = torch.arange(total, device=DEV) - (ln.cumsum(0) - ln)[s["q_seq"]] \
            + pa[s["q_seq"]]
        keys = sum(lens) + sum(past)
        s["k_seq"] = ids.repeat_interleave(ln + pa)
        s["k_pos"] = torch.arange(keys, device=DEV) - ((ln + pa).cumsum(0) - ln - pa)[s["k_seq"]]
        if c.page:
            s["kv"] = _Cache(keys, c.page, c.kv_heads, c.hd, dt, g)
        else:
            s["k"] = rnd(keys, c.kv_heads, c.hd).to(dt)
            s["v"] = rnd(keys, c.kv_heads, c.hd).to(dt)
            if own:
                from treemoe_spec_amd.kernels.prompt_attention import PromptPlan
                s["plan"] = PromptPlan(lens, [a + b for a, b in zip(lens, past)],
                                       num_heads=c.heads, num_kv_heads=c.kv_heads, device=DEV)
    else:
        # most tokens far below a few likely ones
        s["logits"] = (rnd(c.rows, c.vocab) * 3.0).to(DTYPES[c.dtype])
        s["uniforms"] = torch.rand(c.rows, generator=g, device=DEV)
    return s


# ------------------------------------------------------------- plain forms --

def _plain_norm(x, weight, residual, out):
    s = x.float() if residual is None else x.float() + residual.float()
    y = s * torch.rsqrt((s * s).mean(1, keepdim=True) + EPS) * weight.float()
    new = [] if residual is None else [s.to(residual.dtype)]
    if out == "same":
        return [y.to(x.dtype)] + new
    parts = y.view(y.shape[0], -1, GROUP if out == "group" else y.shape[1])
    amax = parts.abs().amax(2)
    scale = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
    y8 = (parts / scale[:, :, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return [y8.view(y.shape), scale if out == "group" else scale[:, 0]] + new


def _frequencies(dim, scaling, device):
    """Radians a position of the dim / 2 pairs, in 64 bits, and the magnitude."""
    i = torch.arange(0, dim, 2, device=device, dtype=torch.float64)
    kind = "none" if scaling is None else scaling["type"]
    if kind == "ntk":
        return (THETA * scaling["factor"] ** (dim / (dim - 2))) ** (-i / dim), 1.0
    f = THETA ** (-i / dim)
    if kind == "linear":
        return f / scaling["factor"], 1.0
    if kind == "yarn":
        # pairs that turn more than beta_fast times over the original length keep
        # their frequency, those under beta_slow are stretched, a ramp between
        span = scaling["original_max_position"] / (2 * math.pi)
        edge = lambda turns: dim * math.log(span / turns) / (2 * math.log(THETA))  # noqa: E731
        lo = max(math.floor(edge(scaling["beta_fast"])), 0)
        hi = min(math.ceil(edge(scaling["beta_slow"])), dim - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return (f * (1 - ramp) + f / scaling["factor"] * ramp,
                0.1 * math.log(scaling["factor"]) + 1.0)
    return f, 1.0


def _plain_rotate(x, cos, sin, part, interleaved):
    a = x.float()
    if interleaved:
        lo, hi = a[..., 0:part:2], a[..., 1:part:2]
    else:
        lo, hi = a[..., : part // 2], a[..., part // 2: part]
    u, w = lo * cos - hi * sin, hi * cos + lo * sin
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([turned, a[..., part:]], -1).to(x.dtype)


def _plain_rotary(s, c):
    f, m = _frequencies(c.part, SCALINGS[c.scaling], DEV)
    angle = s["positions"].double()[:, None] * f[None, :]
    cos, sin = ((t(angle) * m).float()[:, None, :] for t in (torch.cos, torch.sin))
    inter = c.layout == "interleaved"
    q = _plain_rotate(s["q"], cos, sin, c.part, inter)
    k = _plain_rotate(s["k"], cos, sin, c.part, inter)
    if not c.page:
        return [q, k]
    kv = s["kv"]
    slots = kv.slots[c.first: c.first + c.tokens]
    kv.k[0].flatten(0, 1)[slots] = k
    kv.v[0].flatten(0, 1)[slots] = s["v"]
    return [q, kv.k[0], kv.v[0]]


def _plain_attention(q, k, v, q_seq, q_pos, k_seq, k_pos):
    group = q.shape[1] // k.shape[1]
    qh = q.float().transpose(0, 1).contiguous()
    kh = k.float().repeat_interleave(group, 1).permute(1, 2, 0).contiguous()
    vh = v.float().repeat_interleave(group, 1).transpose(0, 1).contiguous()
    seen = (q_seq[:, None] == k_seq[None, :]) & (k_pos[None, :] <= q_pos[:, None])
    w = torch.matmul(qh * q.shape[2] ** -0.5, kh).masked_fill_(~seen, -math.inf)
    w = w.sub_(w.amax(2, keepdim=True)).exp_()
    o = torch.matmul(w, vh) / w.sum(2, keepdim=True)
    return o.transpose(0, 1).flatten(1).to(q.dtype)


def _plain_sample(logits, uniforms, c):
    z = logits.double()
    z = (z - z.amax(1, keepdim=True)) / c.temperature
    # by value, the lowest index first among equals
    z, index = torch.sort(z, dim=1, descending=True, stable=True)
    w = z.exp()
    if 0 < c.top_k < c.vocab:
        w[:, c.top_k:] = 0.0
    if c.top_p < 1.0:
        before = w.cumsum(1) - w
        w = torch.where(before < c.top_p * w.sum(1, keepdim=True), w, torch.zeros_like(w))
    if c.min_p > 0.0:
        w = torch.where(w >= c.min_p, w, torch.zeros_like(w))
    kept = torch.zeros_like(w).scatter_(1, index, w)
    run_sum = kept.cumsum(1)
    total = run_sum[:, -1:]
    token = (run_sum <= uniforms.double()[:, None] * total).sum(1)
    return [token, (kept / total).float()] if c.probs else [token]


# --------------------------------------------------------------------- run --

def run(s):
    c = s["case"]
    if c.kind == "norm":
        if not own:
            return _plain_norm(s["x"], s["weight"], s["residual"], c.out)
        from treemoe_spec_amd.kernels.rms_norm import rms_norm, rms_norm_fp8
        if c.out == "same":
            got = rms_norm(s["x"], s["weight"], EPS, residual=s["residual"])
        else:
            got = rms_norm_fp8(s["x"], s["weight"], EPS, residual=s["residual"],
                               scale_group=GROUP if c.out == "group" else None)
        return list(got) if isinstance(got, tuple) else [got]
    if c.kind == "rotary":
        if not own:
            return _plain_rotary(s, c)
        from treemoe_spec_amd.kernels.rotary import rotary_append, rotary_embed
        if not c.page:
            return list(rotary_embed(s["q"], s["k"], s["positions"], s["plan"]))
        kv = s["kv"]
        q = rotary_append(s["q"], s["k"], s["v"], s["plan"], kv, 0, c.first)
        return [q, kv.k[0], kv.v[0]]
    if c.kind == "attn":
        if not own:
            if c.page:
                kv = s["kv"]
                k, v = (t[0].flatten(0, 1)[kv.slots] for t in (kv.k, kv.v))
            else:
                k, v = s["k"], s["v"]
            return [_plain_attention(s["q"], k, v, s["q_seq"], s["q_pos"], s["k_seq"],
                                     s["k_pos"])]
        from treemoe_spec_amd.kernels.prompt_attention import (prompt_attention,
                                                               prompt_attention_cached)
        if c.page:
            return [prompt_attention_cached(s["q"], s["kv"], 0)]
        return [prompt_attention(s["q"], s["k"], s["v"], s["plan"])]
    if not own:
        return _plain_sample(s["logits"], s["uniforms"], c)
    from treemoe_spec_amd.kernels.sample_tokens import sample_tokens
    got = sample_tokens(s["logits"], s["uniforms"], temperature=c.temperature, top_k=c.top_k,
                        top_p=c.top_p, min_p=c.min_p, return_probs=c.probs)
    return list(got) if c.probs else [got]


# -------------------------------------------------------------------- work --

def work(case):
    c = SimpleNamespace(**case)
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[c.dtype]
    if c.kind == "norm":
        n = c.tokens * c.hidden
        out = {"same": size * n, "row": n + 4 * c.tokens, "group": n + 4 * n // GROUP}[c.out]
        return {"bytes": n * size * (3 if c.residual else 1) + c.hidden * size + out,
                "flops": 4 * n}
    if c.kind == "rotary":
        n = c.tokens * (c.heads + (2 if c.page else 1) * c.kv_heads) * c.hd
        pairs = c.tokens * (c.heads + c.kv_heads) * c.part // 2
        return {"bytes": 2 * n * size + (0 if c.page else 8 * c.tokens), "flops": 6 * pairs}
    if c.kind == "attn":
        lens = _ints(c.lengths)
        past = _ints(c.past, len(lens) if "," not in c.past else None)
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(lens, past))
        rows = 2 * sum(lens) * c.heads + 2 * (sum(lens) + sum(past)) * c.kv_heads
        return {"bytes": rows * c.hd * size, "flops": 4 * pairs * c.heads * c.hd}
    n = c.rows * c.vocab
    return {"bytes": n * size + 12 * c.rows + (4 * n if c.probs else 0), "flops": 4 * n}


# ------------------------------------------------------------------- exact --

def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c.kind == "norm":
        v = s["x"].to(torch.float64)
        if s["residual"] is not None:
            v = v + s["residual"].to(torch.float64)
        norm = torch.linalg.vector_norm(v, dim=1).square() / c.hidden + EPS
        y = v / norm.sqrt().unsqueeze(1) * s["weight"].to(torch.float64)
        tail = [] if s["residual"] is None else [v]
        if c.out == "same":
            return [y] + tail
        step = GROUP if c.out == "group" else c.hidden
        scale = torch.stack([t.abs().max(1).values for t in y.split(step, 1)], 1) / 448
        q = y / scale.repeat_interleave(step, 1)
        return [q, scale if c.out == "group" else scale.squeeze(1)] + tail
    if c.kind == "rotary":
        # as the product with e^(i angle), pair by pair
        freq, m = [], 1.0
        way = SCALINGS[c.scaling] or {"type": "none"}
        for i in range(c.part // 2):
            f = THETA ** (-2.0 * i / c.part)
            if way["type"] == "linear":
                f /= way["factor"]
            elif way["type"] == "ntk":
                f = (THETA * way["factor"] ** (c.part / (c.part - 2.0))) ** (-2.0 * i / c.part)
            elif way["type"] == "yarn":
                m = 1.0 + 0.1 * math.log(way["factor"])
                at = [c.part * math.log(way["original_max_position"] / (2 * math.pi * b))
                      / (2 * math.log(THETA)) for b in (way["beta_fast"], way["beta_slow"])]
                lo, hi = max(0, math.floor(at[0])), min(c.part - 1, math.ceil(at[1]))
                mix = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
                f = mix * f / way["factor"] + (1.0 - mix) * f
            freq.append(f)
        f = torch.tensor(freq, dtype=torch.float64, device=DEV)
        angle = torch.outer(s["positions"].to(torch.float64), f)
        turn = torch.polar(torch.full_like(angle, m), angle).unsqueeze(1)
        got = []
        for x in (s["q"], s["k"]):
            x = x.to(torch.float64)
            r, h = x[:, :, : c.part], c.part // 2
            if c.layout == "interleaved":
                y = torch.view_as_real(torch.view_as_complex(
                    r.unflatten(2, (h, 2)).contiguous()) * turn).flatten(2)
            else:
                z = torch.complex(r[:, :, :h].contiguous(), r[:, :, h:].contiguous()) * turn
                y = torch.cat([z.real, z.imag], 2)
            got.append(torch.cat([y, x[:, :, c.part:]], 2))
        if not c.page:
            return got
        kv = s["kv"]
        pages = []
        for cache, rows in ((kv.k, got[1]), (kv.v, s["v"].to(torch.float64))):
            flat = cache[0].to(torch.float64).flatten(0, 1)
            pages.append(flat.index_copy(0, kv.slots[c.first:], rows).view(cache[0].shape))
        return [got[0]] + pages
    if c.kind == "attn":
        if c.page:
            kv = s["kv"]
            at = torch.arange(kv.seq_len, device=DEV)
            k, v = (t[0][kv.table[at // c.page], at % c.page] for t in (kv.k, kv.v))
        else:
            k, v = s["k"], s["v"]
        lens = _ints(c.lengths)
        past = _ints(c.past, len(lens) if "," not in c.past else None)
        out = torch.empty(sum(lens), c.heads, c.hd, dtype=torch.float64, device=DEV)
        q0 = k0 = 0
        for n, p in zip(lens, past):
            after = torch.ones(n, n + p, dtype=torch.bool, device=DEV).triu(p + 1)
            for h in range(c.heads):
                kk = k[k0:k0 + n + p, h * c.kv_heads // c.heads].to(torch.float64)
                vv = v[k0:k0 + n + p, h * c.kv_heads // c.heads].to(torch.float64)
                a = s["q"][q0:q0 + n, h].to(torch.float64) @ kk.T.contiguous() / math.sqrt(c.hd)
                a = torch.softmax(a.masked_fill(after, -math.inf), 1)
                out[q0:q0 + n, h] = a @ vv
            q0, k0 = q0 + n, k0 + n + p
        return [out.view(sum(lens), -1)]
    # the distribution; the tokens are whole numbers
    if not c.probs:
        return None
    got = torch.zeros(c.rows, c.vocab, dtype=torch.float64, device=DEV)
    for r in range(c.rows):
        p = torch.softmax(s["logits"][r].to(torch.float64) / c.temperature, 0)
        order = torch.argsort(-s["logits"][r].to(torch.float64), stable=True)
        if 0 < c.top_k < c.vocab:
            order = order[: c.top_k]
        p = p[order] / p[order].sum()
        n = int((p.cumsum(0) < c.top_p).sum()) + 1 if c.top_p < 1.0 else len(order)
        p, order = p[:n], order[:n]
        keep = p >= c.min_p * p[0]
        got[r, order[keep]] = p[keep] / p[keep].sum()
    return [None, got]
