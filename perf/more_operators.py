"""Workloads of what stands around the FP8 products of a decoder layer: the norm before them, the adapters beside them, the experts in their place.

Every case has a plain form (elementary torch operations in fp32, the choice of experts in fp64) and,
where `own` is true, the framework's operators.  A serving step runs them in turn: add_rms_norm_cast adds
a layer's output to the residual stream, normalises it and hands it to fp8_gemm_v2 in 8 bits with scales;
lora_add_ adds each request's own low-rank adapter to that product; moe_layer routes the tokens of the
next norm to their experts and runs those.  Inputs are synthetic: activations ~ N(0, 1), norm weights
~ N(1, 0.1), projections of variance 1 / fan-in, expert weights quantised per output channel.
"""
import math
import os
import sys

import torch

own = False

E4M3, E5M2, BF16, F32, F64 = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float32, torch.float64
DTYPE = {"bf16": BF16, "f32": F32, "e4m3": E4M3, "e5m2": E5M2}
SIZE = {"bf16": 2, "f32": 4, "e4m3": 1, "e5m2": 1}
FP8_MAX = {E4M3: 448.0, E5M2: 57344.0}
STATIC_SCALE = 448.0 / 6.0  # of the outputs with a given scale: six standard deviations reach the end of e4m3
WEIGHT_STD = 64.0           # of the 8-bit expert weights
EPS = 1e-6
MOST_NORM = 8192 * 8192              # values of a drawn norm
MOST_LORA_BYTES = 5e8                # of a drawn adapter case
MOST_EXPERT_BYTES = 2.3e9            # all experts of a drawn layer


def listed():
    return [
        # one token of a decode step, 8 bits with a scale of its own: latency alone
        {"name": "norm_one", "kind": "norm", "tokens": 1, "dim": 8192, "src": "bf16", "residual": True, "out": "e4m3", "dynamic": True, "keep": False},
        # a decode batch, the bf16 values kept for adapters or a router
        {"name": "norm_decode", "kind": "norm", "tokens": 64, "dim": 4096, "src": "bf16", "residual": True, "out": "e4m3", "dynamic": True, "keep": True},
        # a prompt batch of the FP8 MLP, one scale for the tensor
        {"name": "norm_prefill", "kind": "norm", "tokens": 8192, "dim": 8192, "src": "bf16", "residual": True, "out": "e4m3", "dynamic": False, "keep": False},
        # a ragged batch of fp32 activations without a residual, rows of an odd size
        {"name": "norm_ragged", "kind": "norm", "tokens": 2731, "dim": 2056, "src": "f32", "residual": False, "out": "e4m3", "dynamic": True, "keep": False},
        # one token with one adapter beside a square projection: latency alone
        {"name": "lora_one", "kind": "lora", "tokens": 1, "k": 4096, "n": 4096, "rank": 16, "adapters": 4, "run": 1, "y": "bf16"},
        # a decode batch in which every request has an adapter of its own
        {"name": "lora_decode", "kind": "lora", "tokens": 64, "k": 8192, "n": 8192, "rank": 32, "adapters": 64, "run": 1, "y": "bf16"},
        # a prompt batch: requests of about 512 tokens, eight adapters
        {"name": "lora_prefill", "kind": "lora", "tokens": 4096, "k": 4096, "n": 14336, "rank": 64, "adapters": 8, "run": 512, "y": "bf16"},
        # a ragged step of short prompts and single tokens, fp32 sums, sizes off the tiles
        {"name": "lora_ragged", "kind": "lora", "tokens": 777, "k": 2056, "n": 1416, "rank": 24, "adapters": 37, "run": 9, "y": "f32"},
        # one token through eight of 128 experts
        {"name": "moe_one", "kind": "moe", "tokens": 1, "hidden": 4096, "inner": 1792, "experts": 128, "top_k": 8, "weights": "e4m3", "padded": 0},
        # a decode batch over the same experts, padded for a captured step
        {"name": "moe_batch", "kind": "moe", "tokens": 29, "hidden": 4096, "inner": 1792, "experts": 128, "top_k": 8, "weights": "e4m3", "padded": 3},
        # a few large experts in bf16
        {"name": "moe_bf16", "kind": "moe", "tokens": 5, "hidden": 4096, "inner": 4096, "experts": 8, "top_k": 2, "weights": "bf16", "padded": 0},
        # small experts with sizes off the tiles, a larger batch
        {"name": "moe_small", "kind": "moe", "tokens": 64, "hidden": 2048, "inner": 688, "experts": 32, "top_k": 4, "weights": "e4m3", "padded": 0},
    ]


def _log_int(rng, lo, hi, multiple=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return min(hi // multiple * multiple, max(multiple, int(v) // multiple * multiple))


def draw(rng):
    kind = rng.choice([c["kind"] for c in listed()])  # as often as it is listed
    if kind == "norm":
        dim = _log_int(rng, 256, 16384, rng.choice([8, 8, 64, 1]))
        return {"kind": kind, "tokens": _log_int(rng, 1, max(1, min(16384, MOST_NORM // dim))), "dim": dim, "src": rng.choice(["bf16", "bf16", "f32"]),
                "residual": rng.random() < 0.7, "out": rng.choice(["e4m3", "e4m3", "bf16"]), "dynamic": rng.random() < 0.6, "keep": rng.random() < 0.3}
    if kind == "lora":
        k, n = _log_int(rng, 256, 8192, 8), _log_int(rng, 256, 16384, 8)
        rank = rng.choice([8, 16, 16, 24, 32, 64, 128])
        adapters = _log_int(rng, 1, max(1, min(64, int(MOST_LORA_BYTES / 4 / (2 * rank * (k + n))))))
        tokens = _log_int(rng, 1, max(1, min(8192, int(MOST_LORA_BYTES / 2 / (2 * k + 4 * n)))))
        return {"kind": kind, "tokens": tokens, "k": k, "n": n, "rank": rank, "adapters": adapters, "run": rng.choice([1, _log_int(rng, 1, tokens)]),
                "y": rng.choice(["bf16", "bf16", "f32"])}
    weights = rng.choice(["e4m3", "e4m3", "bf16"])
    hidden, inner = _log_int(rng, 512, 8192, 16), _log_int(rng, 256, 4096, 16)
    most = int(MOST_EXPERT_BYTES / (3 * hidden * inner * SIZE[weights]))
    experts = _log_int(rng, 2, max(2, min(256, most)))
    return {"kind": kind, "tokens": _log_int(rng, 1, 64), "hidden": hidden, "inner": inner, "experts": experts, "top_k": rng.randint(1, min(8, experts)),
            "weights": weights, "padded": rng.choice([0, 0, rng.randint(1, 9)])}


# ----------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape, std=1.0, mean=0.0, dtype=BF16):
    """In blocks of its first dimension, so that large weights need no fp32 copy of themselves."""
    out = torch.empty(*shape, device="cuda", dtype=dtype)
    rows = max(1, (1 << 26) // max(1, out[0].numel())) if out.numel() else 1
    for lo in range(0, shape[0], rows):
        block = out[lo:lo + rows]
        x = torch.randn(block.shape, device="cuda", generator=gen, dtype=F32) * std + mean
        block.copy_(x.clamp(-FP8_MAX[dtype], FP8_MAX[dtype]) if dtype in FP8_MAX else x)
    return out


def _channel_scales(gen, *shape, std):
    """Inverse scales per output channel of weights of about `std`, as a quantiser leaves them: a factor of two apart at most."""
    return std / WEIGHT_STD * (0.75 + 0.75 * torch.rand(*shape, device="cuda", generator=gen, dtype=F32))


def _adapter_rows(gen, c):
    """An adapter for every run of tokens; one run in eight has none."""
    runs = -(-c["tokens"] // c["run"])
    which = torch.randint(0, c["adapters"], (runs,), device="cuda", generator=gen)
    if c["run"] == 1 and c["adapters"] >= runs:
        which = torch.randperm(c["adapters"], device="cuda", generator=gen)[:runs]
    none = torch.rand(runs, device="cuda", generator=gen) < 0.125
    none[0] = False
    return torch.where(none, -1, which).repeat_interleave(c["run"])[:c["tokens"]].to(torch.int32)


def prepare(case, seed):
    if own:
        package = os.path.join(os.getcwd(), "gaudi-pytorch-bridge_b200")  # the repository's root is the working folder
        if package not in sys.path:
            sys.path.insert(0, package)
        import b200_hpu_ops  # noqa: F401
    gen, c, s = _generator(seed), case, {"case": case}
    if c["kind"] == "norm":
        t, d = c["tokens"], c["dim"]
        s["x"] = _randn(gen, t, d, dtype=DTYPE[c["src"]])
        s["residual"] = _randn(gen, t, d, std=2.0, dtype=DTYPE[c["src"]]) if c["residual"] else None
        s["weight"] = _randn(gen, d, std=0.1, mean=1.0)
        fixed = c["out"] != "bf16" and not c["dynamic"]
        s["scale"] = torch.tensor(STATIC_SCALE, device="cuda", dtype=F32) if fixed else None
    elif c["kind"] == "lora":
        s["x"] = _randn(gen, c["tokens"], c["k"])
        s["y"] = _randn(gen, c["tokens"], c["n"], dtype=DTYPE[c["y"]])
        s["a"] = _randn(gen, c["adapters"], c["rank"], c["k"], std=c["k"] ** -0.5)
        s["b"] = _randn(gen, c["adapters"], c["n"], c["rank"], std=c["rank"] ** -0.5)
        s["adapter"] = _adapter_rows(gen, c)
        s["scales"] = 0.5 + torch.rand(c["adapters"], device="cuda", generator=gen, dtype=F32)
    else:
        e, h, f = c["experts"], c["hidden"], c["inner"]
        s["x"] = _randn(gen, c["tokens"] + c["padded"], h)
        s["router"] = _randn(gen, e, h, std=1.5 * h ** -0.5)
        fp8 = c["weights"] in ("e4m3", "e5m2")
        s["gate_up"] = _randn(gen, e, 2 * f, h, std=WEIGHT_STD if fp8 else h ** -0.5, dtype=DTYPE[c["weights"]])
        s["down"] = _randn(gen, e, h, f, std=WEIGHT_STD if fp8 else f ** -0.5, dtype=DTYPE[c["weights"]])
        s["gate_up_scale"] = _channel_scales(gen, e, 2 * f, std=h ** -0.5) if fp8 else None
        s["down_scale"] = _channel_scales(gen, e, h, std=f ** -0.5) if fp8 else None
        s["count"] = torch.tensor([c["tokens"]], device="cuda", dtype=torch.int32) if c["padded"] else None
    return s


# ----------------------------------------------------------------------------- plain forms
def _plain_norm(s, c):
    x = s["x"].float()
    if c["residual"]:
        s["residual"].copy_(s["residual"].float() + x)  # rounded to the stream's type, and that is what is normalised
        x = s["residual"].float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    out_dtype, scale_inv = DTYPE[c["out"]], None
    if out_dtype in FP8_MAX:
        most = FP8_MAX[out_dtype]
        if c["dynamic"]:
            top = y.abs().amax(-1, keepdim=True)
            scale_inv = torch.where(top > 0, top / most, 1.0)
            scaled = y * torch.where(top > 0, most / top, 1.0)
        else:
            scaled = y * s["scale"]
        out = scaled.clamp(-most, most).to(out_dtype)
    else:
        out = y.to(out_dtype)
    return _norm_outputs(s, c, out, scale_inv, y.to(BF16) if c["keep"] else None)


def _norm_outputs(s, c, out, scale_inv, kept):
    result = {"out": out}
    if c["residual"]:
        result["residual"] = s["residual"]
    if DTYPE[c["out"]] in FP8_MAX and c["dynamic"]:
        result["scale_inv"] = scale_inv
    if c["keep"]:
        result["kept"] = kept
    return result


def _plain_lora(s, c):
    x, y = s["x"].float(), s["y"].float()
    for i in range(c["adapters"]):
        part = (x @ s["a"][i].float().t()) @ s["b"][i].float().t()
        y = torch.where((s["adapter"] == i)[:, None], y + s["scales"][i] * part, y)
    s["y"].copy_(y)
    return s["y"]


def _bytes(t):
    """A view of 8-bit values that indexing takes."""
    return t.view(torch.uint8) if t.dtype in FP8_MAX else t


def _weight(w, scale, i):
    """Expert i (an index tensor of one entry) of quantised or bf16 weights, in fp32."""
    x = _bytes(w).index_select(0, i)[0].view(w.dtype).float()
    return x if scale is None else x * scale.index_select(0, i)[0][:, None]


def _plain_moe(s, c):
    x, t, k, e, f = s["x"], s["x"].shape[0], c["top_k"], c["experts"], c["inner"]
    logits = x.double() @ s["router"].double().t()  # fp64: neighbours in the order of the experts are close
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    ids, top = order.indices[:, :k], order.values[:, :k]
    weights = torch.softmax(top, -1).float()
    live = torch.arange(t, device=x.device) < c["tokens"]
    x = x.float()
    out = torch.zeros(t, c["hidden"], device=x.device, dtype=F32)

    def expert(i, rows):
        gu = rows @ _weight(s["gate_up"], s["gate_up_scale"], i).t()
        g, u = gu[:, :f], gu[:, f:]
        return (g / (1.0 + torch.exp(-g)) * u) @ _weight(s["down"], s["down_scale"], i).t()

    if c["tokens"] * k <= e:  # few: token by token
        for row in range(c["tokens"]):
            for j in range(k):
                out[row] += weights[row, j] * expert(ids[row, j:j + 1], x[row:row + 1])[0]
    else:  # many: expert by expert, each over all tokens
        for i in range(e):
            share = torch.where(ids == i, weights, 0.0).sum(-1, keepdim=True)
            part = expert(torch.full((1,), i, device=x.device), x)
            out += torch.where(share > 0, share * part, 0.0)
    out = torch.where(live[:, None], out, 0.0)
    ids = torch.where(live[:, None], ids, -1).to(torch.int32)
    return out.to(BF16), torch.where(live[:, None], weights, 0.0), ids


# ----------------------------------------------------------------------------- one pass
def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        with torch.no_grad():
            return {"norm": _plain_norm, "lora": _plain_lora, "moe": _plain_moe}[kind](s, c)
    ops = torch.ops.b200q
    if kind == "norm":
        return _norm_outputs(s, c, *ops.add_rms_norm_cast(s["x"], s["residual"], s["weight"], EPS, DTYPE[c["out"]], s["scale"], c["keep"]))
    if kind == "lora":
        return ops.lora_add_(s["y"], s["x"], s["a"], s["b"], s["adapter"], s["scales"])
    return ops.moe_layer(s["x"], s["router"], s["gate_up"], s["down"], s["gate_up_scale"], s["down_scale"], c["top_k"], True, s["count"])


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "norm":
        row = c["dim"] * (SIZE[c["src"]] * (3 if c["residual"] else 1) + SIZE[c["out"]] + (2 if c["keep"] else 0))
        scales = 4 * c["tokens"] if c["dynamic"] and c["out"] != "bf16" else 0
        return {"bytes": c["tokens"] * row + 2 * c["dim"] + scales, "flops": 0}
    if c["kind"] == "lora":
        runs = -(-c["tokens"] // c["run"])
        chosen = 0.875 * runs if c["run"] == 1 and c["adapters"] >= runs else c["adapters"] * (1 - (1 - 1 / c["adapters"]) ** (0.875 * runs))
        chosen = max(1.0, chosen)
        live = max(1.0, 0.875 * runs) / runs * c["tokens"]  # tokens with an adapter
        size = 2 * live * c["k"] + 2 * SIZE[c["y"]] * live * c["n"] + 4 * c["tokens"] + chosen * 2 * c["rank"] * (c["k"] + c["n"])
        return {"bytes": size, "flops": 2 * live * c["rank"] * (c["k"] + c["n"])}
    t, h, f, e, k = c["tokens"], c["hidden"], c["inner"], c["experts"], c["top_k"]
    chosen = e * (1 - (1 - k / e) ** t)  # experts that some token goes to, were all as likely
    scales = 4 * (2 * f + h) if c["weights"] != "bf16" else 0
    size = chosen * (3 * f * h * SIZE[c["weights"]] + scales) + 2 * e * h + 4 * (t + c["padded"]) * h + 8 * t * k
    return {"bytes": size, "flops": 6 * t * k * h * f + 2 * t * e * h}


# ----------------------------------------------------------------------------- the definitions, in 64 bits
def _exact_norm(s, c):
    z = s["x"].to(F64)
    result = {}
    if c["residual"]:
        stored = (s["residual"].to(F64) + z).to(DTYPE[c["src"]])
        result["residual"], z = s["residual"].to(F64) + z, stored.to(F64)
    y = z / torch.sqrt(torch.sum(z ** 2, 1, keepdim=True) / z.shape[1] + EPS) * s["weight"].to(F64)[None]
    dtype = DTYPE[c["out"]]
    out = y
    if dtype in FP8_MAX:
        if c["dynamic"]:
            factor = y.abs().max(1, keepdim=True).values / FP8_MAX[dtype]
            factor = factor.masked_fill(factor == 0, 1.0)
            result["scale_inv"], out = factor, y / factor
        else:
            out = (y * s["scale"].to(F64)).clamp(-FP8_MAX[dtype], FP8_MAX[dtype])
    result["out"] = out
    if c["keep"]:
        result["kept"] = y
    return {name: result[name] for name in ("out", "residual", "scale_inv", "kept") if name in result}


def _exact_lora(s, c):
    y = s["y"].to(F64)
    for i in s["adapter"].unique().tolist():
        if i >= 0:
            rows = (s["adapter"] == i).nonzero()[:, 0]
            down = torch.einsum("tk,rk->tr", s["x"][rows].to(F64), s["a"][i].to(F64))
            y[rows] += s["scales"][i].to(F64) * torch.einsum("tr,nr->tn", down, s["b"][i].to(F64))
    return y


def _exact_moe(s, c):
    n, f = c["tokens"], c["inner"]
    x = s["x"].to(F64)
    out, shares = torch.zeros_like(x), torch.zeros(x.shape[0], c["top_k"], device="cuda", dtype=F64)
    chosen = torch.full((x.shape[0], c["top_k"]), -1, device="cuda")
    scores = torch.einsum("th,eh->te", x[:n], s["router"].to(F64))
    shares[:n], chosen[:n] = scores.topk(c["top_k"], dim=1)
    shares[:n] = torch.exp(shares[:n] - torch.logsumexp(shares[:n], 1, keepdim=True))
    for i in chosen[:n].unique().tolist():
        rows, place = (chosen == i).nonzero(as_tuple=True)
        first, second = (w[i].to(F64) if scale is None else w[i].to(F64) * scale[i].to(F64)[:, None]
                         for w, scale in ((s["gate_up"], s["gate_up_scale"]), (s["down"], s["down_scale"])))
        gate, up = x[rows] @ first[:f].t(), x[rows] @ first[f:].t()
        out[rows] += shares[rows, place][:, None] * ((gate * torch.sigmoid(gate) * up) @ second.t())
    return out, shares, None


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "lora": _exact_lora, "moe": _exact_moe}[case["kind"]](s, case)
