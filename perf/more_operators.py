"""What is timed of the feed-forward half of a decoder layer: the residual's addition with the norm behind it, and the whole
sparse expert layer for a few tokens.

Four operators, reached as a user's program reaches them:

* ``add_rms_norm``        s = x + residual rounded to the type of the tensors, y = s / sqrt(mean(s^2) + eps) * weight; forward,
                          and backward from the gradients of both results;
* ``add_rms_norm_fp8``    the same with y as e4m3 rows (what ``quantize_fp8_rows`` makes of y as rounded to its type: one
                          power-of-two scale per row and 128 elements);
* ``moe_fused_layer``     router, softmax and top-k, the gated experts and the weighted sum over a token's experts, for up to
                          16 tokens; with a norm's weight also the addition and the norm in front and the addition of the
                          stream behind: out = s + experts(norm(s));
* ``moe_fused_layer_fp8`` the same on expert weights held as e4m3 values with one scale per 128 x 128 block; the rows in front
                          of the products and the gated unit's result are quantised row by row.

Logits are rounded once to the type of the hidden states, experts are chosen from the rounded ones, and equal ones go to the
lowest index.  Unless a case says otherwise the sizes are those of this repository's benchmark: 128 experts, 8 per token,
hidden 2048, intermediate 768, bf16.

A case is a dict of plain values:

* ``kind``   "norm" (forward), "norm_train" (forward and backward), "norm_fp8", "layer", "layer_fp8";
* ``rows``   rows of the norm, or tokens of the layer; ``hidden``; ``experts``, ``top_k``, ``inter`` (layer only, else 0);
* ``dtype``  "bf16", "fp16" or "fp32": the type of the activations, and of the weights that are not in 8 bits;
* ``added``  norm: whether there is a residual to add; layer: whether addition and norm are part of the call;
* ``renorm`` whether the chosen experts' weights are brought to a sum of one;
* ``zipf``   exponent of the experts' popularity (0: near-uniform).
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
BLOCK = 128
TOP = 448.0  # the largest e4m3 value
EPS = 1e-6
WEIGHT_STD = 0.02
# skewed routing: the hidden states' first channel is a constant of this size, and the router's first column the experts'
# log-popularity over what it is after the norm
MASSIVE = 8.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(name, kind, rows, experts=128, top_k=8, hidden=2048, inter=768, dtype="bf16", added=True, renorm=True, zipf=0.0):
    if kind.startswith("norm"):
        experts = top_k = inter = 0
    return {"name": name, "kind": kind, "rows": rows, "experts": experts, "top_k": top_k, "hidden": hidden, "inter": inter,
            "dtype": dtype, "added": added, "renorm": renorm, "zipf": zipf}


def listed():
    return [
        # the norm in front of the experts for one token: the smallest call, latency
        _case("norm_1", "norm", 1),
        # a long prompt
        _case("norm_16384", "norm", 16384),
        # a training step of 4096 tokens
        _case("norm_train_4096", "norm_train", 4096),
        # rows that no 16-byte access fits
        _case("norm_train_odd_fp16", "norm_train", 1999, hidden=1001, dtype="fp16"),
        # 8-bit experts: a decode batch of 32 users
        _case("norm_fp8_32", "norm_fp8", 32),
        # and a long prompt
        _case("norm_fp8_16384", "norm_fp8", 16384),
        # one user, one token at a time
        _case("layer_1", "layer", 1, added=False),
        # a decode batch, with addition and norm: the largest call
        _case("layer_added_16", "layer", 16),
        # the benchmark's toy configuration 1 in float32
        _case("layer_added_toy_fp32", "layer", 4, experts=8, top_k=2, hidden=64, inter=128, dtype="fp32"),
        # sizes that are a multiple of nothing
        _case("layer_odd_fp16", "layer", 5, experts=60, top_k=4, hidden=1001, inter=333, dtype="fp16", added=False, renorm=False),
        # one user on 8-bit experts, with addition and norm
        _case("layer_fp8_added_1", "layer_fp8", 1),
        # a decode batch on 8-bit experts, skewed routing
        _case("layer_fp8_13_zipf", "layer_fp8", 13, added=False, zipf=1.0),
    ]


def draw(rng):
    """Norms: 1 to 32768 rows, half of them 2048 wide, the others 64 to 8192 in steps of 32, or of any width from 32 to 4096.
    Layers: 1 to 16 tokens, half at the benchmark's sizes, the others with 8 to 160 experts, hidden 256 to 4096 and
    intermediate 128 to 1536 in steps of 32, or of any size from 32 to 1024; some with skewed routing.  8-bit experts in 16-bit
    types only: their gated unit is quantised from 32-bit sums, whose last bits put a value next to a border of the 8-bit grid
    on either side."""

    def log_between(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("norm", "norm_train", "norm_fp8", "layer", "layer", "layer_fp8", "layer_fp8"))
        c = _case("", kind, 1, dtype=rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32")), added=rng.random() < 0.7,
                  renorm=rng.random() < 0.7)
        del c["name"]
        if c["dtype"] == "fp32" and kind == "layer_fp8":
            c["dtype"] = "bf16"
        sizes = rng.choice(("benchmark", "benchmark", "other", "odd"))
        if kind.startswith("norm"):
            c["rows"] = log_between(1, 32768)
            if sizes != "benchmark":
                c["hidden"] = 32 * log_between(2, 256) if sizes == "other" else log_between(32, 4096)
        else:
            c["rows"] = log_between(1, 16)
            if sizes != "benchmark":
                c["experts"], c["top_k"] = rng.choice((8, 16, 60, 64, 96, 128, 160)), rng.choice((1, 2, 4, 6, 8))
                c["hidden"], c["inter"] = 32 * log_between(8, 128), 32 * log_between(4, 48)
            if sizes == "odd":
                c["hidden"], c["inter"] = log_between(32, 1024), log_between(32, 1024)
            if rng.random() < 0.3:
                c["zipf"] = round(rng.uniform(0.5, 1.3), 2)
        if _cost(c) <= most:
            return c


def _cost(c):
    w = work(c)
    return w["bytes"] / 5e12 + w["flops"] / 1e15


def _popularity(c):
    p = [(i + 1.0) ** -c["zipf"] for i in range(c["experts"])]
    total = sum(p)
    return [v / total for v in p]


def work(case):
    """Every input read and every output written once, the weights of the experts that are expected to be chosen."""
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    t, h, i = c["rows"], c["hidden"], c["inter"]
    if c["kind"].startswith("norm"):
        tensors = 4 if c["added"] else 2  # x, residual, stream, y
        # (backward: the two gradients that arrive, and that of x, which is the residual's too)
        row = size * h * (tensors + (tensors - 1 if c["kind"] == "norm_train" else 0))
        return {"bytes": t * row + size * h * (2 if c["kind"] == "norm_train" else 1),
                "flops": (12.0 if c["kind"] == "norm_train" else 5.0) * t * h}
    hit = sum(1.0 - (1.0 - v) ** (t * c["top_k"]) for v in _popularity(c))
    expert = 3.0 * h * i * size if c["kind"] == "layer" else 3.0 * (h * i + 4.0 * math.ceil(h / BLOCK) * math.ceil(i / BLOCK))
    return {"bytes": hit * expert + size * (c["experts"] * (h + t) + t * h * (3 if c["added"] else 2)),
            "flops": 2.0 * t * h * (c["experts"] + 3.0 * c["top_k"] * i)}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _normal(g, shape, dtype, std=1.0):
    return torch.empty(shape, device=DEV, dtype=torch.float32).normal_(0.0, std, generator=g).to(dtype)


def _hidden_states(g, rows, width, dtype):
    """Hidden states: unit variance, with one channel in 64 eight times as large, as real ones have some."""
    x = _normal(g, (rows, width), torch.float32)
    x[:, torch.randint(0, width, (max(1, width // 64),), device=DEV, generator=g)] *= 8.0
    return x.to(dtype)


def _weight8(g, experts, out_features, in_features):
    """An expert matrix as block-quantised checkpoints hold it: e4m3 values, and per 128 x 128 block the fp32 scale
    amax / 448."""
    nb, kb = -(-out_features // BLOCK), -(-in_features // BLOCK)
    w = torch.zeros((experts, nb * BLOCK, kb * BLOCK), device=DEV)
    w[:, :out_features, :in_features] = _normal(g, (experts, out_features, in_features), torch.float32, WEIGHT_STD)
    w = w.view(experts, nb, BLOCK, kb, BLOCK)
    scale = w.abs().amax(dim=(2, 4)) / TOP
    q = (w / scale[:, :, None, :, None]).clamp_(-TOP, TOP).view(experts, nb * BLOCK, kb * BLOCK)
    return q[:, :out_features, :in_features].to(torch.float8_e4m3fn).contiguous(), scale.contiguous()


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype, t, h, i, n = DTYPES[c["dtype"]], c["rows"], c["hidden"], c["inter"], c["experts"]
    s = {"kind": c["kind"], "k": c["top_k"], "renorm": c["renorm"], "residual": None, "norm": None}
    if c["kind"].startswith("norm") or c["added"]:
        s["norm"] = (1.0 + _normal(g, (h,), torch.float32, 0.1)).to(dtype)
    s["x"] = _hidden_states(g, t, h, dtype)
    if c["added"]:
        s["residual"] = _normal(g, (t, h), dtype, 0.5)
    if c["kind"] == "norm_train":
        s["dy"] = _normal(g, (t, h), dtype)
        # (the gradient that comes along the stream; without a residual the input is the stream, and autograd adds it itself)
        s["ds"] = _normal(g, (t, h), dtype) if c["added"] else None
        for name in ("x", "residual", "norm"):
            if s[name] is not None:
                s[name].requires_grad_()
    if not c["kind"].startswith("layer"):
        return s
    router = _normal(g, (n, h), torch.float32, h ** -0.5)
    if c["zipf"]:
        s["x"][:, 0] = MASSIVE
        rows = s["x"].float() if s["residual"] is None else s["x"].float() + s["residual"].float()
        size = MASSIVE / rows.square().mean().sqrt() if c["added"] else MASSIVE
        router[:, 0] = torch.tensor(_popularity(c), device=DEV).log()[torch.randperm(n, device=DEV, generator=g)] / size
    s["router"] = router.to(dtype)
    for name, shape in (("gate", (n, i, h)), ("up", (n, i, h)), ("down", (n, h, i))):
        if c["kind"] == "layer":
            s[name] = _normal(g, shape, dtype, WEIGHT_STD)
        else:
            s[name], s[name + "_scale"] = _weight8(g, *shape)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    package = os.path.join(os.getcwd(), "transformers-qwen3-moe-fused_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from qwen3_moe_fused.fused_mlp import moe_fused_layer, moe_fused_layer_fp8
    from qwen3_moe_fused.kernels.norm import add_rms_norm, add_rms_norm_fp8
    from qwen3_moe_fused.quantize.fp8 import dequantize_fp8_rows

    kind = s["kind"]
    if kind == "norm_train":
        y, stream = add_rms_norm(s["x"], s["residual"], s["norm"], EPS)
        if s["residual"] is None:
            return (y.detach(), *torch.autograd.grad(y, (s["x"], s["norm"]), s["dy"]))
        grads = torch.autograd.grad((y, stream), (s["x"], s["residual"], s["norm"]), (s["dy"], s["ds"]))
        return (y.detach(), stream.detach(), *grads)
    with torch.no_grad():
        if kind == "norm":
            return add_rms_norm(s["x"], s["residual"], s["norm"], EPS)
        if kind == "norm_fp8":
            values, scales, stream = add_rms_norm_fp8(s["x"], s["residual"], s["norm"], EPS)
            return dequantize_fp8_rows(values, scales, s["x"].dtype), stream
        added = {"residual": s["residual"], "norm_weight": s["norm"], "eps": EPS}
        if kind == "layer":
            return moe_fused_layer(s["x"], s["router"], s["gate"], s["up"], s["down"], s["k"], s["renorm"], **added)
        return moe_fused_layer_fp8(s["x"], s["router"], s["gate"], s["gate_scale"], s["up"], s["up_scale"], s["down"],
                                   s["down_scale"], s["k"], s["renorm"], **added)


def _stream(s):
    x = s["x"].detach()
    return x if s["residual"] is None else (x.float() + s["residual"].detach().float()).to(x.dtype)


def _normed(stream, weight, dtype):
    """In 64 bits: what is rounded here is rounded again behind it, or decides which experts are chosen."""
    v = stream.double()
    return (v * torch.rsqrt(v.square().mean(dim=1, keepdim=True) + EPS) * weight.detach().double()).to(dtype)


def _quantized(x):
    """The values that the e4m3 blocks of x (float32) stand for: per row and 128 elements the exponent e is the smallest
    integer, -117 at least, with amax <= 448 * 2^e."""
    rows, width = x.shape
    blocks = -(-width // BLOCK)
    padded = torch.zeros((rows, blocks * BLOCK), device=x.device)
    padded[:, :width] = x
    padded = padded.view(rows, blocks, BLOCK)
    mantissa, exponent = torch.frexp(padded.abs().amax(dim=2))  # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp_(min=-117)
    scale = ((e + 127) << 23).view(torch.float32)[:, :, None]
    inverse = ((127 - e) << 23).view(torch.float32)[:, :, None]
    q = (padded * inverse).to(torch.float8_e4m3fn).float()
    return (q * scale).view(rows, -1)[:, :width]


def _matrix(s, name, expert):
    w = s[name][expert].float()
    if name + "_scale" not in s:
        return w
    scale = s[name + "_scale"][expert]
    return w * scale.repeat_interleave(BLOCK, dim=0)[:w.shape[0]].repeat_interleave(BLOCK, dim=1)[:, :w.shape[1]]


def _chosen(s, logits):
    """Every token's experts and their weights, from the logits as rounded."""
    order = torch.sort(logits.double(), dim=1, descending=True, stable=True)
    p = torch.exp(order.values - order.values[:, :1])
    p = p / p.sum(dim=1, keepdim=True)
    p, chosen = p[:, :s["k"]], order.indices[:, :s["k"]]
    return chosen, p / p.sum(dim=1, keepdim=True) if s["renorm"] else p


def _run_plain(s):
    with torch.no_grad():
        kind, dtype = s["kind"], s["x"].dtype
        stream = _stream(s)
        if kind == "norm":
            return _normed(stream, s["norm"], dtype), stream
        if kind == "norm_fp8":
            return _quantized(_normed(stream, s["norm"], dtype).float()).to(dtype), stream
        if kind == "norm_train":
            return _plain_train(s, stream)
        eight = kind == "layer_fp8"
        rows = stream if s["norm"] is None else _normed(stream, s["norm"], dtype)
        logits = (rows.double() @ s["router"].double().t()).to(dtype)
        chosen, weight = _chosen(s, logits)
        x = _quantized(rows.float()) if eight else rows.float()
        out = torch.zeros(rows.shape, device=rows.device)
        for e in chosen.unique().tolist():
            token, place = (chosen == e).nonzero(as_tuple=True)
            a = x[token]
            u, v = a @ _matrix(s, "gate", e).t(), a @ _matrix(s, "up", e).t()
            hidden = u / (1.0 + torch.exp(-u)) * v
            y = (_quantized(hidden) if eight else hidden) @ _matrix(s, "down", e).t()
            out[token] += weight[token, place].float()[:, None] * y
        return (out if s["norm"] is None else stream.float() + out).to(dtype), logits


def _plain_train(s, stream):
    dtype, v, w, dy = s["x"].dtype, stream.float(), s["norm"].detach().float(), s["dy"].float()
    r = torch.rsqrt(v.square().mean(dim=1, keepdim=True) + EPS)
    unit = v * r
    y = unit * w
    g = dy * w
    dx = r * (g - unit * (g * unit).mean(dim=1, keepdim=True))
    dw = (dy * unit).sum(dim=0)
    if s["residual"] is None:
        return y.to(dtype), dx.to(dtype), dw.to(dtype)
    dx = (dx + s["ds"].float()).to(dtype)
    return y.to(dtype), stream, dx, dx, dw.to(dtype)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact(s)


def _grid64(x):
    """x (float64) on the e4m3 grid of its blocks: 2^e times a multiple of 2^(max(floor(log2 |v|), -6) - 3), ties to even."""
    out = torch.empty_like(x)
    for lo in range(0, x.shape[1], BLOCK):
        v = x[:, lo:lo + BLOCK]
        amax = v.abs().amax(dim=1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.ones_like(amax)) / TOP))
        e = torch.where(amax <= TOP * torch.exp2(e - 1), e - 1, e)  # (log2 may be off by a rounding)
        e = torch.where(amax > TOP * torch.exp2(e), e + 1, e).clamp_(min=-117)
        v = v / torch.exp2(e)
        step = torch.exp2(torch.frexp(v).exponent.double().sub_(1).clamp_(min=-6) - 3)
        out[:, lo:lo + BLOCK] = torch.round(v / step) * step * torch.exp2(e)
    return out


def _matrix64(s, name, expert):
    w = s[name][expert].double()
    if s["kind"] == "layer":
        return w
    rows, cols = (torch.arange(size, device=w.device) // BLOCK for size in w.shape)
    return w * s[name + "_scale"][expert].double()[rows][:, cols]


def _exact(s):
    kind, dtype = s["kind"], s["x"].dtype
    stream = s["x"].detach().double()
    if s["residual"] is not None:
        stream = (stream + s["residual"].detach().double()).to(dtype).double()
    if s["norm"] is not None:
        weight = s["norm"].detach().double()
        length = torch.sqrt(stream.pow(2).sum(dim=1, keepdim=True) / stream.shape[1] + EPS)
        unit = stream / length
        rows = unit * weight
    if kind == "norm":
        return rows, stream
    if kind == "norm_fp8":
        return _grid64(rows.to(dtype).double()), stream
    if kind == "norm_train":
        dy = s["dy"].double()
        along = (dy * weight * unit).sum(dim=1, keepdim=True) / stream.shape[1]
        dx, dw = (dy * weight - unit * along) / length, (dy * unit).sum(dim=0)
        if s["residual"] is None:
            return rows, dx, dw
        return rows, stream, dx + s["ds"].double(), dx + s["ds"].double(), dw
    rows = stream if s["norm"] is None else rows.to(dtype).double()
    logits = torch.mm(rows, s["router"].double().t().contiguous())
    scores = torch.softmax(logits.to(dtype).double(), dim=1)
    x = _grid64(rows) if kind == "layer_fp8" else rows
    out = torch.zeros_like(rows) if s["norm"] is None else stream.clone()
    table = scores.tolist()
    for token, row in enumerate(table):
        best = sorted(range(len(row)), key=lambda e: (-row[e], e))[:s["k"]]
        total = sum(row[e] for e in best) if s["renorm"] else 1.0
        for e in best:
            a = x[token:token + 1]
            u, v = (torch.mm(a, _matrix64(s, name, e).t().contiguous()) for name in ("gate", "up"))
            hidden = u * torch.sigmoid(u) * v
            hidden = _grid64(hidden) if kind == "layer_fp8" else hidden
            out[token] += row[e] / total * torch.mm(hidden, _matrix64(s, "down", e).t().contiguous())[0]
    return out, logits
