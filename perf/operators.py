"""Workloads of the paged key/value cache: the plan of a step, the append to the cache, one new token's attention over it.

Every case has a plain form (elementary torch operations in fp32) and, where `own` is true, the
framework's operators.  A serving step runs the three in turn: paged_plan gives every new token its
place in the cache, qk_norm_rope_append normalises and rotates queries and keys and writes keys and
values to those places, paged_attention answers each request's new token.  Inputs are synthetic:
projections ~ N(0, 1), norm weights ~ N(1, 0.1), cached keys and values ~ N(0, 1) quantised to the
cache's type, queries ~ N(0, 2) so that the probabilities are not flat.
"""
import math
import os
import sys

import torch

own = False

E4M3, E5M2, BF16, F32, F64 = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float32, torch.float64
DTYPE = {"bf16": BF16, "f32": F32, "e4m3": E4M3, "e5m2": E5M2}
FP8_MAX = {E4M3: 448.0, E5M2: 57344.0}
CACHE_SCALE = 448.0 / 6.0  # of the fp8 caches: six standard deviations reach the end of e4m3
EPS = 1e-6
MAX_POSITION = 32768
MOST_CACHE_BYTES = 6e8  # keys and values of a drawn case


def listed():
    return [
        # one decode step of 64 requests with contexts up to 8192 tokens: latency alone
        {"name": "plan_decode", "kind": "plan", "requests": 64, "context": 8192, "new": 1, "page": 16, "padded": 0},
        # a large prefill batch: 32 prompts of ragged lengths up to 4096, some behind a cached prefix, tokens padded for a graph
        {"name": "plan_prefill", "kind": "plan", "requests": 32, "context": 512, "new": 4096, "page": 64, "padded": 1000},
        # one decode step of 16 requests, eight query heads to a key/value head, e4m3 cache
        {"name": "append_decode", "kind": "append", "tokens": 16, "heads": 64, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False,
         "norm": True, "src": "bf16", "cache": "e4m3", "q": "bf16", "page": 16, "padded": 0},
        # a prompt batch of 8192 tokens into the e4m3 cache
        {"name": "append_prefill", "kind": "append", "tokens": 8192, "heads": 64, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False,
         "norm": True, "src": "bf16", "cache": "e4m3", "q": "bf16", "page": 64, "padded": 0},
        # a ragged prompt, heads of 64 with half of each rotated in neighbouring pairs, bf16 cache, padded tokens behind it
        {"name": "append_ragged", "kind": "append", "tokens": 2731, "heads": 32, "kv_heads": 32, "dim": 64, "rotary": 32, "interleaved": True,
         "norm": False, "src": "bf16", "cache": "bf16", "q": "bf16", "page": 16, "padded": 85},
        # queries quantised too, for the FP8 attention over the prompt; fp32 projections
        {"name": "append_fp8_queries", "kind": "append", "tokens": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False,
         "norm": True, "src": "f32", "cache": "e4m3", "q": "e4m3", "page": 128, "padded": 0},
        # one request with a short context on one of eight ranks: one key/value head, latency alone
        {"name": "attend_one", "kind": "attend", "requests": 1, "context": 200, "heads": 8, "kv_heads": 1, "dim": 128, "cache": "e4m3", "page": 16, "window": 0},
        # a decode batch of 16 ragged requests up to 4096 tokens
        {"name": "attend_batch", "kind": "attend", "requests": 16, "context": 4096, "heads": 64, "kv_heads": 8, "dim": 128, "cache": "e4m3", "page": 16, "window": 0},
        # a full decode batch: 64 requests of up to 8192 tokens
        {"name": "attend_large", "kind": "attend", "requests": 64, "context": 8192, "heads": 64, "kv_heads": 8, "dim": 128, "cache": "e4m3", "page": 64, "window": 0},
        # one request with a very long context
        {"name": "attend_long", "kind": "attend", "requests": 1, "context": 131072, "heads": 64, "kv_heads": 8, "dim": 128, "cache": "e4m3", "page": 64, "window": 0},
        # a bf16 cache with a key/value head for every query head
        {"name": "attend_bf16", "kind": "attend", "requests": 29, "context": 2000, "heads": 32, "kv_heads": 32, "dim": 64, "cache": "bf16", "page": 32, "window": 0},
        # wide heads, a sliding window
        {"name": "attend_window", "kind": "attend", "requests": 40, "context": 6000, "heads": 16, "kv_heads": 2, "dim": 256, "cache": "bf16", "page": 16, "window": 4096},
    ]


def _log_int(rng, lo, hi, multiple=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return min(hi, max(multiple, int(v) // multiple * multiple))


def draw(rng):
    kind = rng.choice([c["kind"] for c in listed()])  # as often as it is listed
    page = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        requests = _log_int(rng, 1, 1024)
        decode = rng.random() < 0.4
        new = 1 if decode else _log_int(rng, 2, max(2, min(16384, 131072 // requests)))
        return {"kind": kind, "requests": requests, "context": _log_int(rng, 1, 16384), "new": new, "page": page, "padded": rng.randint(0, 64)}
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    group = rng.choice([1, 2, 4, 7, 8, 16]) if kv_heads <= 4 else rng.choice([1, 2, 4, 8])
    cache = rng.choice(["e4m3", "e4m3", "bf16", "bf16", "e5m2"])
    if kind == "append":
        cache = "e4m3" if cache == "e5m2" else cache  # caches of range rather than precision come from elsewhere
        heads = kv_heads * group
        most = max(1, min(16384, (8192 * 80 * 128) // ((heads + 2 * kv_heads) * dim)))
        return {"kind": kind, "tokens": _log_int(rng, 1, most), "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rng.choice([dim, dim, dim // 2]),
                "interleaved": rng.random() < 0.3, "norm": rng.random() < 0.7, "src": rng.choice(["bf16", "bf16", "f32"]), "cache": cache,
                "q": rng.choice(["bf16", "bf16", "e4m3"]), "page": page, "padded": rng.choice([0, rng.randint(1, 100)])}
    token = 2 * kv_heads * dim * (2 if cache == "bf16" else 1)  # bytes of keys and values
    requests = _log_int(rng, 1, 256)
    context = _log_int(rng, 1, max(1, int(min(131072, MOST_CACHE_BYTES / token / requests, 16e6 / requests / kv_heads))))
    return {"kind": kind, "requests": requests, "context": context, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "cache": cache, "page": page,
            "window": rng.choice([0, 0, _log_int(rng, 1, context)])}  # (a window may be as long as the context, or one token)


# ----------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape, std=1.0, mean=0.0, dtype=BF16):
    """In blocks of its first dimension, so that the largest cache needs no fp32 copy of itself."""
    out = torch.empty(*shape, device="cuda", dtype=dtype)
    rows = max(1, (1 << 26) // max(1, out[0].numel())) if out.numel() else 1
    for lo in range(0, shape[0], rows):
        block = out[lo:lo + rows]
        x = torch.randn(block.shape, device="cuda", generator=gen, dtype=F32) * std + mean
        block.copy_(x.clamp(-FP8_MAX[dtype], FP8_MAX[dtype]) if dtype in FP8_MAX else x)
    return out


def _scalar(v):
    return torch.tensor(float(v), device="cuda", dtype=F32)


def _ragged(n, most):
    """Ragged lengths from a quarter of `most` tokens to all of it; among many there is a short and an empty one."""
    lo = max(1, most // 4)
    x = [lo + int((most - lo + 1) * (i * 0.6180339887498949 % 1.0)) for i in range(n)]
    x[0] = most
    if n > 3:
        x[1], x[2] = 1, 0
    return x


def _lengths(seed, n, most):
    """The same lengths in an order of the seed's."""
    order = torch.randperm(n, generator=torch.Generator().manual_seed(int(seed)))
    return torch.tensor(_ragged(n, most), dtype=torch.int32)[order].cuda()


def _pages(lens, page):
    return (lens + page - 1) // page


def _tables(gen, lens, page, spare=1):
    """Block tables over a shuffled pool: [requests, most pages], and the number of pages in the pool."""
    n = _pages(lens.long(), page)
    width, total = int(n.max()) + spare, int(n.sum()) + spare
    order = torch.randperm(total, device="cuda", generator=gen)
    start = torch.cumsum(n, 0) - n
    col = torch.arange(width, device="cuda")
    table = order[(start[:, None] + col).clamp(max=total - 1)]
    return torch.where(col < n[:, None], table, -1).to(torch.int32), total


def _cos_sin(rotary):
    """Cosines and sines of every position, as a model computes them once: [MAX_POSITION, rotary], angles in fp64."""
    inv = 10000.0 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=F64) / rotary)
    angle = torch.arange(MAX_POSITION, device="cuda", dtype=F64)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).to(F32)


def prepare(case, seed):
    if own:
        package = os.path.join(os.getcwd(), "gaudi-pytorch-bridge_b200")  # the repository's root is the working folder
        if package not in sys.path:
            sys.path.insert(0, package)
        import b200_hpu_ops  # noqa: F401
    gen, c, s = _generator(seed), case, {"case": case}
    if c["kind"] == "plan":
        n, page = c["requests"], c["page"]
        s["context"] = _lengths(seed, n, c["context"])
        s["new"] = _lengths(seed + 1, n, c["new"]) if c["new"] > 1 else torch.ones(n, device="cuda", dtype=torch.int32)
        total = (s["context"] + s["new"]).long()
        have, need = int(_pages(s["context"].long(), page).sum()), int(_pages(total, page).sum())
        order = torch.randperm(need + 64, device="cuda", generator=gen).to(torch.int32)
        width = _pages(c["context"] + c["new"], page) + 2
        start = torch.cumsum(_pages(s["context"].long(), page), 0) - _pages(s["context"].long(), page)
        col = torch.arange(width, device="cuda")
        held = order[(start[:, None] + col).clamp(max=need + 63)]
        s["table"] = torch.where(col < _pages(s["context"].long(), page)[:, None], held, -1).to(torch.int32)
        s["free"] = order[have:].contiguous()
        s["tokens"] = int(s["new"].long().sum()) + c["padded"]
    elif c["kind"] == "append":
        t, h, g, d, page = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["page"]
        qkv = _randn(gen, t + c["padded"], h + 2 * g, d, dtype=DTYPE[c["src"]])  # the output of one projection
        s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + g], qkv[:, h + g:]
        s["q_weight"] = _randn(gen, d, std=0.1, mean=1.0) if c["norm"] else None
        s["k_weight"] = _randn(gen, d, std=0.1, mean=1.0) if c["norm"] else None
        s["cos_sin"] = _cos_sin(c["rotary"])
        slots = -(-t // page) * page
        pages = torch.randperm(slots // page + 3, device="cuda", generator=gen)
        at = torch.arange(t, device="cuda")
        first = int(torch.randint(0, MAX_POSITION - t, (1,), device="cuda", generator=gen))
        pad = torch.zeros(c["padded"], device="cuda", dtype=torch.int64)
        s["positions"] = torch.cat([first + at, pad])
        s["slots"] = torch.cat([pages[at // page] * page + at % page, pad - 1])
        fp8 = c["cache"] != "bf16"
        std = CACHE_SCALE if fp8 else 1.0
        s["k_cache"] = _randn(gen, pages.numel(), page, g, d, std=std, dtype=DTYPE[c["cache"]])
        s["v_cache"] = _randn(gen, pages.numel(), page, g, d, std=std, dtype=DTYPE[c["cache"]])
        s["k_scale"] = s["v_scale"] = _scalar(CACHE_SCALE) if fp8 else None
        s["q_scale"] = _scalar(CACHE_SCALE) if c["q"] != "bf16" else None
    else:
        b, g, d, page = c["requests"], c["kv_heads"], c["dim"], c["page"]
        s["lens"] = _lengths(seed, b, c["context"])
        s["table"], pages = _tables(gen, s["lens"], page)
        fp8 = c["cache"] != "bf16"
        std = CACHE_SCALE if fp8 else 1.0
        s["k_cache"] = _randn(gen, pages, page, g, d, std=std, dtype=DTYPE[c["cache"]])
        s["v_cache"] = _randn(gen, pages, page, g, d, std=std, dtype=DTYPE[c["cache"]])
        s["scale_inv"] = _scalar(1.0 / CACHE_SCALE) if fp8 else None
        s["q"] = _randn(gen, b, c["heads"], d, std=2.0)
    return s


# ----------------------------------------------------------------------------- plain forms
def _plain_plan(s, c):
    page, tokens, table = c["page"], s["tokens"], s["table"]
    width = table.shape[1]
    ctx, new = s["context"].long().clamp(min=0), s["new"].long().clamp(min=0)
    have, need = _pages(ctx, page).clamp(max=width), _pages(ctx + new, page).clamp(max=width)
    end, taken = torch.cumsum(new, 0), torch.cumsum(need - have, 0)
    base = taken - (need - have)
    col = torch.arange(width, device=table.device)
    at = base[:, None] + col - have[:, None]
    free = s["free"]
    page_of = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where((col >= have[:, None]) & (col < need[:, None]), page_of, table))
    t = torch.arange(tokens, device=table.device)
    b = torch.searchsorted(end, t, right=True).clamp(max=ctx.numel() - 1)
    real = t < end[-1]
    pos = torch.where(real, ctx[b] + t - (end - new)[b], 0)
    p = table[b, (pos // page).clamp(max=width - 1)].long()
    slot = torch.where(real & (pos // page < width) & (p >= 0), p * page + pos % page, -1)
    start = torch.cat([end.new_zeros(1), end]).to(torch.int32)
    return slot, pos, start, (ctx + new).to(torch.int32), taken[-1:].to(torch.int32), table


def _round(x, dtype, scale):
    x = x if scale is None else x * scale
    return x.clamp(-FP8_MAX[dtype], FP8_MAX[dtype]).to(dtype) if dtype in FP8_MAX else x.to(dtype)


def _plain_norm_rope(x, weight, table, positions, rotary, interleaved):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    row = table[positions]
    cos, sin = row[:, None, :rotary // 2], row[:, None, rotary // 2:]
    r, rest = x[..., :rotary], x[..., rotary:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rotary // 2], r[..., rotary // 2:])
    u, v = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([r, rest], -1)


def _bytes(t):
    """A view of 8-bit values that indexing takes."""
    return t.view(torch.uint8) if t.dtype in FP8_MAX else t


def _plain_append(s, c):
    q = _plain_norm_rope(s["q"], s["q_weight"], s["cos_sin"], s["positions"], c["rotary"], c["interleaved"])
    k = _plain_norm_rope(s["k"], s["k_weight"], s["cos_sin"], s["positions"], c["rotary"], c["interleaved"])
    n = c["tokens"]  # the tokens behind these have no slot
    for cache, x, scale in ((s["k_cache"], k, s["k_scale"]), (s["v_cache"], s["v"].float(), s["v_scale"])):
        _bytes(cache).view(-1, c["kv_heads"], c["dim"])[s["slots"][:n]] = _bytes(_round(x[:n], cache.dtype, scale))
    return _round(q, DTYPE[c["q"]], s["q_scale"]), s["k_cache"], s["v_cache"]


def _plain_attend(s, c):
    b, g, d, r = c["requests"], c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    table = s["table"].long().clamp(min=0)
    n = table.shape[1] * c["page"]

    def gathered(cache):
        x = _bytes(cache)[table].view(cache.dtype).float()
        return (x if s["scale_inv"] is None else x * s["scale_inv"]).reshape(b, n, g, d).transpose(1, 2)

    pos = torch.arange(n, device="cuda")
    lens = s["lens"].long()[:, None]
    seen = (pos < lens) & (pos >= lens - c["window"]) if c["window"] else pos < lens
    scores = (s["q"].float().reshape(b, g, r, d) * (1.0 / math.sqrt(d))) @ gathered(s["k_cache"]).transpose(-1, -2)
    scores = torch.where(seen[:, None, None, :], scores, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ gathered(s["v_cache"])) / total.clamp(min=1e-30)
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)
    return out.reshape(b, g * r, d).to(BF16), lse.reshape(b, g * r)


# ----------------------------------------------------------------------------- one pass
def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        with torch.no_grad():
            return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend}[kind](s, c)
    ops = torch.ops.b200q
    if kind == "plan":
        out = ops.paged_plan(s["context"], s["new"], s["table"], s["free"], None, c["page"], s["tokens"])
        return (*out, s["table"])
    if kind == "append":
        q = ops.qk_norm_rope_append(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], EPS, s["cos_sin"], s["positions"], c["interleaved"],
                                    s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["q_scale"], DTYPE[c["q"]])
        return q, s["k_cache"], s["v_cache"]
    return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], 1.0 / math.sqrt(c["dim"]), s["scale_inv"], s["scale_inv"],
                               c["window"])


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "plan":
        n = c["requests"]
        tokens = sum(_ragged(n, c["new"])) if c["new"] > 1 else n
        pages = tokens / c["page"]  # taken from the pool, and written into the tables
        return {"bytes": 16 * (tokens + c["padded"]) + 8 * pages + 16 * n, "flops": 0}
    size = {"bf16": 2, "f32": 4, "e4m3": 1, "e5m2": 1}
    if c["kind"] == "append":
        t, h, g, d = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        read = (t + c["padded"]) * (h * d * size[c["src"]] + 8 + 8) + t * (2 * g * d * size[c["src"]] + 4 * c["rotary"])
        return {"bytes": read + (t + c["padded"]) * h * d * size[c["q"]] + 2 * t * g * d * size[c["cache"]], "flops": 0}
    b, h, g, d = c["requests"], c["heads"], c["kv_heads"], c["dim"]
    tokens = sum(min(x, c["window"] or x) for x in _ragged(b, c["context"]))
    return {"bytes": 2 * tokens * g * d * size[c["cache"]] + 4 * b * h * d + 4 * b * h + 4 * tokens / c["page"] + 4 * b, "flops": 4 * tokens * h * d}


# ----------------------------------------------------------------------------- the definitions, in 64 bits
def _exact_head(x, weight, angle_cos, angle_sin, interleaved):
    """One tensor [tokens, heads, dim]: RMS norm of each head, then the rotation, each pair on its own."""
    y = x.to(F64)
    if weight is not None:
        y = y / torch.sqrt(torch.sum(y ** 2, -1, keepdim=True) / y.shape[-1] + EPS) * weight.to(F64)
    half = angle_cos.shape[1]
    i = torch.arange(half, device=y.device)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    turned = y.clone()
    turned[..., lo] = y[..., lo] * angle_cos[:, None] - y[..., hi] * angle_sin[:, None]
    turned[..., hi] = y[..., lo] * angle_sin[:, None] + y[..., hi] * angle_cos[:, None]
    return turned


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    s, c = prepare(case, seed), case
    if c["kind"] == "append":
        half = c["rotary"] // 2
        cos, sin = (s["cos_sin"].to(F64)[s["positions"]][:, i * half:(i + 1) * half] for i in (0, 1))
        limit = FP8_MAX.get(DTYPE[c["cache"]], math.inf)
        q = _exact_head(s["q"], s["q_weight"], cos, sin, c["interleaved"]) * (1.0 if s["q_scale"] is None else s["q_scale"].to(F64))
        q = q.clamp(-FP8_MAX.get(DTYPE[c["q"]], math.inf), FP8_MAX.get(DTYPE[c["q"]], math.inf))
        out = [q]
        for cache, x in ((s["k_cache"], _exact_head(s["k"], s["k_weight"], cos, sin, c["interleaved"])), (s["v_cache"], s["v"].to(F64))):
            whole = cache.to(F64)
            x = x * (1.0 if s["k_scale"] is None else s["k_scale"].to(F64))
            page, offset = s["slots"] // c["page"], s["slots"] % c["page"]
            used = s["slots"] >= 0
            whole[page[used], offset[used]] = x[used].clamp(-limit, limit)
            out.append(whole)
        return tuple(out)
    group, scale = c["heads"] // c["kv_heads"], 1.0 if s["scale_inv"] is None else float(s["scale_inv"])
    out = torch.zeros(c["requests"], c["heads"], c["dim"], device="cuda", dtype=F64)
    lse = torch.full((c["requests"], c["heads"]), -math.inf, device="cuda", dtype=F64)
    for b, length in enumerate(s["lens"].tolist()):
        if not length:
            continue
        first = max(0, length - c["window"]) if c["window"] else 0
        at = torch.arange(first, length, device="cuda")
        page = s["table"][b].long()[at // c["page"]]
        k, v = (x[page, at % c["page"]].to(F64) * scale if x.dtype == BF16 else x.view(torch.uint8)[page, at % c["page"]].view(x.dtype).to(F64) * scale
                for x in (s["k_cache"], s["v_cache"]))
        for h in range(c["heads"]):
            w = (k[:, h // group] @ s["q"][b, h].to(F64)) / math.sqrt(c["dim"])
            lse[b, h] = torch.logsumexp(w, 0)
            out[b, h] = torch.exp(w - lse[b, h]) @ v[:, h // group]
    return out, lse
