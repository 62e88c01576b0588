"""What is timed of the expert products in 8-bit floating point: what a user has the package do with expert weights held
as e4m3 values with one scale per 128 x 128 block.

Three operators: ``moe_fused_linear_fp8`` (one expert projection, forward and input gradient), the gated unit
(gate and up projection, SiLU, product; forward and backward) and the expert MLP (gated unit, then the down projection).
The left operand of every product is quantised to e4m3 too, with one power-of-two scale per row and 128 elements of the
reduction; the sums are taken over the quantised values.  Unless a case says otherwise the sizes are those of this
repository's benchmark: 128 experts, 8 per token, hidden 2048, intermediate 768, bf16.

A case is a dict of plain values:

* ``kind``   "linear" (forward), "linear_train" (forward and input gradient), "glu" (gated unit, forward),
             "glu_products" (the same, which also returns the two projections, as a training step keeps them),
             "glu_backward" (from the unit's gradient and the two projections to the gradient of its input rows),
             "mlp" (gated unit and down projection);
* ``tokens``, ``experts``, ``top_k``, ``hidden``, ``inter``: the products have tokens * top_k rows; ``top_k`` is 1 for the
             projections, whose operand is (tokens, hidden) and weight (experts, inter, hidden);
* ``dtype``  "bf16", "fp16" or "fp32": the type of the activations;
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
WEIGHT_STD = 0.02
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
KINDS = ("linear", "linear_train", "glu", "glu_products", "glu_backward", "mlp")


def _case(name, kind, tokens, experts=128, top_k=8, hidden=2048, inter=768, dtype="bf16", zipf=0.0):
    return {"name": name, "kind": kind, "tokens": tokens, "experts": experts,
            "top_k": 1 if kind.startswith("linear") else top_k, "hidden": hidden, "inter": inter, "dtype": dtype, "zipf": zipf}


def listed():
    return [
        # one projection of one token's eight expert rows: the smallest call, latency
        _case("linear_decode_8", "linear", 8),
        # one projection of a prompt or training batch of 4096 tokens (benchmark configuration 2)
        _case("linear_32768", "linear", 32768),
        # the down projection in a fine-tuning step with frozen weights: forward and input gradient (configuration 3)
        _case("linear_train_32768", "linear_train", 32768, hidden=768, inter=2048),
        # the benchmark's toy configuration 1 in float32
        _case("linear_train_toy_fp32", "linear_train", 512, experts=8, hidden=64, inter=128, dtype="fp32"),
        # sizes that are a multiple of nothing, in fp16: rows that no 16-byte access fits
        _case("linear_train_odd_fp16", "linear_train", 1999, experts=60, hidden=1001, inter=333, dtype="fp16"),
        # the front half of the block for a decode batch of 32 users
        _case("glu_decode_32", "glu", 32),
        # the front half in a fine-tuning step, which keeps the two projections for its backward pass
        _case("glu_products_4096", "glu_products", 4096),
        # and that backward pass
        _case("glu_backward_4096", "glu_backward", 4096),
        # the backward pass of a short batch on a model of other sizes, skewed routing
        _case("glu_backward_333", "glu_backward", 333, experts=60, top_k=4, hidden=1056, inter=352, zipf=1.0),
        # the three projections for one user, one token at a time
        _case("mlp_decode_1", "mlp", 1),
        # a prompt of no round length, skewed routing
        _case("mlp_3001_zipf", "mlp", 3001, zipf=1.0),
        # a long prompt (benchmark configuration 5's): the largest call
        _case("mlp_16384", "mlp", 16384),
    ]


def draw(rng):
    """1 to 16384 tokens (1 to 32768 rows of a single projection); half of the cases at the benchmark's sizes, the others
    with 8 to 160 experts, hidden 256 to 4096 and intermediate 128 to 1536 in steps of 32, or, with up to 2048 rows, of
    any size from 32 to 1024; some with skewed routing.  float32 activations only where it is the inputs that are
    quantised: what is quantised in the middle (the gated unit's result, its gradients) comes out of 32-bit sums, whose last
    bits put a value next to a border of the 8-bit grid on either side."""

    def log_between(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(KINDS)
        single = kind.startswith("linear")
        c = {"kind": kind, "tokens": log_between(1, 32768 if single else 16384), "experts": 128, "top_k": 1 if single else 8,
             "hidden": 2048, "inter": 768, "dtype": rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32")), "zipf": 0.0}
        if c["dtype"] == "fp32" and kind in ("glu_backward", "mlp"):
            c["dtype"] = "bf16"
        sizes = rng.choice(("benchmark", "benchmark", "other", "odd"))
        if sizes != "benchmark":
            c["experts"] = rng.choice((8, 16, 60, 64, 96, 128, 160))
            c["top_k"] = 1 if single else rng.choice((1, 2, 4, 6, 8))
            c["hidden"], c["inter"] = 32 * log_between(8, 128), 32 * log_between(4, 48)
        if sizes == "odd":
            c["tokens"] = max(1, log_between(1, 2048) // c["top_k"])
            c["hidden"], c["inter"] = log_between(32, 1024), log_between(32, 1024)
        if single and rng.random() < 0.5:
            c["hidden"], c["inter"] = c["inter"], c["hidden"]
        if rng.random() < 0.3:
            c["zipf"] = round(rng.uniform(0.5, 1.3), 2)
        if _cost(c) <= most:
            return c


def _cost(c):
    w = work(c)
    return w["bytes"] / 5e12 + w["flops"] / 2e15


def _popularity(c):
    p = [(i + 1.0) ** -c["zipf"] for i in range(c["experts"])]
    total = sum(p)
    return [v / total for v in p]


def work(case):
    """Every input read and every output written once, the weights of the experts that are expected to get rows."""
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    t, h, i = c["tokens"], c["hidden"], c["inter"]
    rows = t * c["top_k"]
    hit = sum(1.0 - (1.0 - v) ** rows for v in _popularity(c))
    weight = hit * (h * i + 4.0 * math.ceil(h / BLOCK) * math.ceil(i / BLOCK))
    product = 2.0 * rows * h * i
    if c["kind"] == "linear":
        return {"bytes": size * rows * (h + i) + weight, "flops": product}
    if c["kind"] == "linear_train":
        return {"bytes": 2 * size * rows * (h + i) + weight, "flops": 2 * product}
    if c["kind"] == "glu":
        return {"bytes": size * (t * h + rows * i) + 2 * weight, "flops": 2 * product}
    if c["kind"] == "glu_products":
        return {"bytes": size * (t * h + 3 * rows * i) + 2 * weight, "flops": 2 * product}
    if c["kind"] == "glu_backward":
        return {"bytes": size * rows * (h + 3 * i) + 2 * weight, "flops": 2 * product}
    return {"bytes": size * (t * h + rows * h) + 3 * weight, "flops": 3 * product}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _normal(g, shape, dtype, std=1.0):
    return torch.empty(shape, device=DEV, dtype=torch.float32).normal_(0.0, std, generator=g).to(dtype)


def _hidden_states(g, rows, width, dtype):
    """Hidden states: unit variance, with one channel in 64 eight times as large, as real ones have some."""
    x = _normal(g, (rows, width), torch.float32)
    x[:, torch.randint(0, width, (max(1, width // 64),), device=DEV, generator=g)] *= 8.0
    return x.to(dtype)


def _weight(g, experts, out_features, in_features):
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
    dtype, t, k, h, i, n = DTYPES[c["dtype"]], c["tokens"], c["top_k"], c["hidden"], c["inter"], c["experts"]
    # every token's experts: the k largest of its logits, which are the experts' log-popularity plus Gumbel noise
    logits = -torch.log(-torch.log(torch.rand((t, n), device=DEV, generator=g).clamp_(1e-6, 1.0 - 1e-6)))
    popularity = torch.tensor(_popularity(c), device=DEV)
    logits += popularity.log()[torch.randperm(n, device=DEV, generator=g)]
    chosen = logits.topk(k, dim=1).indices.reshape(-1)
    sort_idx = torch.argsort(chosen, stable=True)
    counts = torch.bincount(chosen, minlength=n)
    s = {"kind": c["kind"], "m_sizes": counts.to(torch.int32), "sort_idx": sort_idx.to(torch.int32),
         "inv_sort_idx": torch.argsort(sort_idx).to(torch.int32), "k": k,
         "counts": counts.tolist()}  # (on the host, for the plain form's loop over the experts)
    if c["kind"].startswith("linear"):
        s["x"] = _hidden_states(g, t, h, dtype)
        s["w"], s["w_scale"] = _weight(g, n, i, h)
        if c["kind"] == "linear_train":
            s["x"].requires_grad_()
            s["dy"] = _normal(g, (t, i), dtype)
        return s
    s["gate"], s["gate_scale"] = _weight(g, n, i, h)
    s["up"], s["up_scale"] = _weight(g, n, i, h)
    if c["kind"] == "glu_backward":
        for name in ("dh", "e", "g"):
            s[name] = _normal(g, (t * k, i), dtype)
        return s
    s["tokens"] = _hidden_states(g, t, h, dtype)
    if c["kind"] == "mlp":
        s["down"], s["down_scale"] = _weight(g, n, h, i)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    package = os.path.join(os.getcwd(), "transformers-qwen3-moe-fused_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from qwen3_moe_fused.fused_mlp import moe_fused_mlp_fp8
    from qwen3_moe_fused.grouped_gemm.fused import grouped_glu_backward_fp8, grouped_glu_forward_fp8
    from qwen3_moe_fused.quantize.layer_fp8 import moe_fused_linear_fp8

    kind, m_sizes = s["kind"], s["m_sizes"]
    if kind == "linear":
        with torch.no_grad():
            return moe_fused_linear_fp8(s["x"], s["w"], s["w_scale"], m_sizes)
    if kind == "linear_train":
        s["x"].grad = None
        y = moe_fused_linear_fp8(s["x"], s["w"], s["w_scale"], m_sizes)
        y.backward(s["dy"])
        return y.detach(), s["x"].grad
    pair = (s["gate"], s["gate_scale"], s["up"], s["up_scale"])
    if kind == "glu_backward":
        return grouped_glu_backward_fp8(s["dh"], s["e"], s["g"], *pair, m_sizes)
    with torch.no_grad():
        if kind == "mlp":
            return moe_fused_mlp_fp8(s["tokens"], *pair, s["down"], s["down_scale"], m_sizes, s["sort_idx"],
                                     s["inv_sort_idx"], s["k"])
        return grouped_glu_forward_fp8(s["tokens"], *pair, m_sizes, s["sort_idx"], s["k"],
                                       return_products=kind == "glu_products")


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


def _dequantized(w, scale):
    """Matrices in float32: (experts, out, in) with their scales (experts, blocks, blocks)."""
    full = scale.repeat_interleave(BLOCK, dim=1)[:, :w.shape[1]].repeat_interleave(BLOCK, dim=2)[:, :, :w.shape[2]]
    return w.float() * full


def _per_expert(x, w, scale, counts, transposed=False):
    out = torch.empty((x.shape[0], w.shape[2] if transposed else w.shape[1]), device=x.device)
    # all matrices at once where many experts have rows (fewer launches), else one by one
    matrices = _dequantized(w, scale) if 4 * sum(m > 0 for m in counts) > len(counts) else None
    lo = 0
    for e, m in enumerate(counts):
        if m:
            matrix = matrices[e] if matrices is not None else _dequantized(w[e:e + 1], scale[e:e + 1])[0]
            out[lo:lo + m] = x[lo:lo + m] @ (matrix if transposed else matrix.t())
            lo += m
    return out


def _run_plain(s):
    kind, counts = s["kind"], s["counts"]

    def product(x, name, transposed=False):
        return _per_expert(x, s[name], s[name + "_scale"], counts, transposed)

    with torch.no_grad():
        if kind.startswith("linear"):
            x = s["x"]
            y = product(_quantized(x.float()), "w").to(x.dtype)
            return y if kind == "linear" else (y, product(_quantized(s["dy"].float()), "w", True).to(x.dtype))
        if kind == "glu_backward":
            dh, e, g = s["dh"].float(), s["e"].float(), s["g"].float()
            sig = 1.0 / (1.0 + torch.exp(-e))
            de, dg = dh * g * sig * (1.0 + e * (1.0 - sig)), dh * e * sig
            return (product(_quantized(de), "gate", True) + product(_quantized(dg), "up", True)).to(s["dh"].dtype)
        tokens = s["tokens"]
        x = _quantized(tokens.float())[s["sort_idx"].long() // s["k"]]
        e, g = product(x, "gate"), product(x, "up")
        h = e / (1.0 + torch.exp(-e)) * g
        if kind == "glu":
            return h.to(tokens.dtype)
        if kind == "glu_products":
            return h.to(tokens.dtype), e.to(tokens.dtype), g.to(tokens.dtype)
        return product(_quantized(h), "down").to(tokens.dtype)


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


def _matrix64(w, scale, expert):
    n, k = w.shape[1:]
    rows, cols = torch.arange(n, device=w.device) // BLOCK, torch.arange(k, device=w.device) // BLOCK
    return w[expert].double() * scale[expert].double()[rows][:, cols]


def _grouped64(x, m_sizes, matrix):
    parts, lo = [], 0
    for expert, m in enumerate(m_sizes.tolist()):
        if m:
            parts.append(torch.mm(x[lo:lo + m], matrix(expert)))
            lo += m
    return torch.cat(parts)


def _exact(s):
    kind, ms = s["kind"], s["m_sizes"]

    def forward(x, name):
        return _grouped64(x, ms, lambda e: _matrix64(s[name], s[name + "_scale"], e).t().contiguous())

    def backward(x, name):
        return _grouped64(x, ms, lambda e: _matrix64(s[name], s[name + "_scale"], e))

    if kind == "linear":
        return forward(_grid64(s["x"].double()), "w")
    if kind == "linear_train":
        return forward(_grid64(s["x"].detach().double()), "w"), backward(_grid64(s["dy"].double()), "w")
    if kind == "glu_backward":
        dh, e, g = s["dh"].double(), s["e"].double(), s["g"].double()
        sig = torch.sigmoid(e)
        return (backward(_grid64(dh * g * (sig + e * sig * (1.0 - sig))), "gate")
                + backward(_grid64(dh * (e * sig)), "up"))
    x = _grid64(s["tokens"].double())[torch.div(s["sort_idx"].long(), s["k"], rounding_mode="floor")]
    e, g = forward(x, "gate"), forward(x, "up")
    h = e * torch.sigmoid(e) * g
    if kind == "glu":
        return h
    if kind == "glu_products":
        return h, e, g
    return forward(_grid64(h), "down")
