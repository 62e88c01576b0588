"""The norm and the whole expert layer in 64 bits on the CPU, with bounds of what 32-bit arithmetic may differ by.

A rounding to a type t is off by ``finfo(t).eps / 2`` of the value at most (and by half the least subnormal); a sum of n products in 32
bits, in whatever order, by n 2^-24 of the sum of their magnitudes."""
import torch

BLOCK, TOP = 128, 448.0
U32 = 2.0 ** -24


def half_step(value, dtype):
    """What one rounding of ``value`` (float64) to ``dtype`` may be off by, one to 32 bits in front of it included."""
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2 + U32) + info.smallest_normal * info.eps / 2


def stream(x, residual):
    return x.double() if residual is None else (x.double() + residual.double()).to(x.dtype).double()


def norm(s, weight, eps):
    """(y, unit, length) of the stream's rows, float64."""
    length = torch.sqrt(s.square().mean(dim=-1, keepdim=True) + eps)
    unit = s / length
    return unit * weight.double(), unit, length


def norm_gradients(dy, ds, s, weight, eps):
    _, unit, length = norm(s, weight, eps)
    g = dy.double() * weight.double()
    dx = (g - unit * (g * unit).mean(dim=-1, keepdim=True)) / length
    return dx + (0 if ds is None else ds.double()), (dy.double() * unit).reshape(-1, s.shape[-1]).sum(dim=0)


def norm_gradient_bounds(dy, ds, s, weight, eps, dtype, weight_dtype):
    """Of dx: g and its product with s, 40 additions in a row's sum, the products behind it.  Of dw: a sum over all rows."""
    dx, dw = norm_gradients(dy, ds, s, weight, eps)
    _, unit, length = norm(s, weight, eps)
    g = (dy.double() * weight.double()).abs()
    along = (g * unit.abs()).mean(dim=-1, keepdim=True)
    extra = 0 if ds is None else ds.double().abs()
    terms = (g + unit.abs() * along) / length
    rows = s.numel() // s.shape[-1]
    spread = (dy.double() * unit).abs().reshape(-1, s.shape[-1]).sum(dim=0)
    return (half_step(dx, dtype) + U32 * (64 * terms + 4 * (extra + dx.abs())),
            half_step(dw, weight_dtype) + U32 * (rows + 64) * spread)


def grid(x):
    """x (float64) on the e4m3 grid of its rows' blocks of 128 with a power-of-two scale; what is not finite becomes NaN and leaves the
    scale to the others."""
    out = torch.empty_like(x)
    for lo in range(0, x.shape[1], BLOCK):
        v = x[:, lo:lo + BLOCK]
        v = torch.where(v.isfinite(), v, torch.full_like(v, float("nan")))
        amax = torch.nan_to_num(v, nan=0.0).abs().amax(dim=1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.ones_like(amax)) / TOP))
        e = torch.where(amax <= TOP * torch.exp2(e - 1), e - 1, e)
        e = torch.where(amax > TOP * torch.exp2(e), e + 1, e).clamp_(min=-117)
        v = v / torch.exp2(e)
        step = torch.exp2(torch.frexp(v).exponent.double().sub_(1).clamp_(min=-6) - 3)
        out[:, lo:lo + BLOCK] = torch.round(v / step) * step * torch.exp2(e)
    return out


def widened(w, scale):
    """Expert weights in float64, (E, out, in), with their block scales or None."""
    if scale is None:
        return w.double()
    full = scale.double().repeat_interleave(BLOCK, 1)[:, :w.shape[1]].repeat_interleave(BLOCK, 2)[:, :, :w.shape[2]]
    return w.float().double() * full


def choose(logits, k, renorm):
    """[(expert, weight), ...] of every token from its logits as rounded; None for a token that chooses none."""
    picked = []
    for row in logits.double().tolist():
        if any(v != v for v in row) or max(row) in (float("inf"), float("-inf")):
            picked.append(None)
            continue
        p = torch.softmax(torch.tensor(row, dtype=torch.float64), 0).tolist()
        best = sorted(range(len(row)), key=lambda e: (-row[e], e))[:k]
        total = sum(p[e] for e in best) if renorm else 1.0
        picked.append([(e, p[e] / total) for e in best])
    return picked


def layer(rows, s, logits, gate, up, down, k, renorm, dtype, scales=None):
    """(out, bound) in float64 from the rows that the experts get (float64, as rounded to the type), the stream to be added (or None)
    and the logits as rounded.  A token without experts: NaN."""
    eight = scales is not None
    gate, up, down = (widened(w, sc) for w, sc in zip((gate, up, down), scales or (None,) * 3))
    x = grid(rows) if eight else rows
    inner, outer = x.shape[1] + 16, gate.shape[1] + 64
    out = torch.zeros_like(x) if s is None else s.clone()
    bound = out.abs() * U32
    for t, picked in enumerate(choose(logits, k, renorm)):
        if picked is None:
            out[t], bound[t] = float("nan"), 0.0
            continue
        a = x[t:t + 1]
        for e, weight in picked:
            u, v = a @ gate[e].t(), a @ up[e].t()
            du, dv = (U32 * inner * (a.abs() @ w[e].abs().t()) for w in (gate, up))
            sig = torch.sigmoid(u)
            h = u * sig * v
            # |d silu| <= 1.1; the sigmoid's two approximate instructions and the products: 16 roundings
            dh = 1.1 * du * v.abs() + (u * sig).abs() * dv + 1.1 * du * dv + 16 * U32 * h.abs()
            if eight:
                q = grid(h)
                dh = torch.maximum((grid(h + dh) - q).abs(), (grid(h - dh) - q).abs())
                h = q
            elif dtype == torch.bfloat16:
                dh = dh + h.abs() * 2.0 ** -16  # two bf16 values for one of 32 bits
            y = h @ down[e].t()
            dy = dh @ down[e].abs().t() + U32 * outer * (h.abs() @ down[e].abs().t())
            out[t] += weight * y[0]
            # (the weight: exponential, sum over the experts, two divisions)
            bound[t] += weight * (dy[0] + 1.5e-6 * y[0].abs()) + 32 * U32 * (weight * y[0].abs() + out[t].abs())
    return out, bound + half_step(torch.nan_to_num(out), dtype)
