"""The expert products in 8-bit floating point in 64 bits, with the distance that 32-bit sums may keep from them.

A sum of fp32 products is off by at most ``GAMMA`` per addition, relative to the sum of magnitudes (a truncating adder's step,
twice the rounding one's); an output is rounded once, by half a step of its type.  Where something computed is quantised
(the gated unit's result, its gradients), a value whose error reaches a border of the 8-bit grid may land on either side: the
reference returns the grid's step there as slack, and products carry it on with the weights' magnitudes.

Outputs of 16 bits may come from the 8-bit matrix instruction, which adds its products in groups of eight and cuts them off
2^-13 below the group's largest: each is off by less than u = 2^-13 max, with the sign of a product, so a sum's error has a
variance below sum over groups of 8 u^2 / 3 <= 2^-26 (8 / 3) sum of squared products.  ``CUT`` is eight standard deviations
of that, relative to the root of the sum of squares (8 * sqrt(8 / 3) = 13.07)."""
import torch

BLOCK = 128
GAMMA = 2.0 ** -23
CUT = 13.07 * 2.0 ** -13


def blocks_of(n):
    return -(-n // BLOCK)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def scale_exponent(amax):
    """Smallest e >= -117 with amax <= 448 * 2^e (amax float64)."""
    m, p = torch.frexp(amax)  # amax = m 2^p, 0.5 <= m < 1;  448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, p - 9, p - 8)
    return torch.where(amax > 0, e, torch.full_like(e, -117)).clamp(min=-117).double()


def quantize(x, err=None):
    """x (rows, K) float64 -> (values on the grid, exponents (rows, blocks), slack).  err: how far the x of the code under
    test may be off, elementwise."""
    rows, k = x.shape
    nb = blocks_of(k)
    pad = torch.zeros((rows, nb * BLOCK), dtype=torch.float64, device=x.device)
    pad[:, :k] = x
    pad = pad.view(rows, nb, BLOCK)
    finite = pad.isfinite()
    amax = torch.where(finite, pad.abs(), torch.zeros_like(pad)).amax(dim=2)
    e = scale_exponent(amax)
    s = torch.exp2(e)[:, :, None]
    v = torch.where(finite, pad / s, torch.zeros_like(pad))
    step = torch.exp2((torch.frexp(v).exponent - 1).clamp(min=-6).double() - 3)
    q = torch.where(finite, torch.round(v / step) * step * s, torch.full_like(pad, float("nan")))
    slack = torch.zeros_like(q)
    if err is not None:
        ep = torch.zeros_like(pad).view(rows, -1)
        ep[:, :k] = err
        ep = ep.view(rows, nb, BLOCK)
        to_border = (0.5 - (v / step - torch.round(v / step)).abs()) * step * s
        slack = torch.where(to_border <= ep, step * s, slack)
        # a block whose largest value may fall on the other side of its scale's border: every value by a step
        margin = torch.minimum((448 * s[:, :, 0] - amax).abs(), (amax - 224 * s[:, :, 0]).abs())
        near = margin <= ep.amax(dim=2)
        slack = torch.where(near[:, :, None], 2 * step * s, slack)
    return q.view(rows, -1)[:, :k], e, slack.view(rows, -1)[:, :k]


def expand(scale, n, k):
    return scale.double().repeat_interleave(BLOCK, 1)[:, :n].repeat_interleave(BLOCK, 2)[:, :, :k]


def dense(weight, scale):
    return weight.double() * expand(scale, *weight.shape[1:])


def grouped(x, w, counts, transposed=False):
    """Rows past the last expert's come out as NaN (they are not compared)."""
    out = torch.full((x.shape[0], w.shape[2 if transposed else 1]), float("nan"), dtype=torch.float64, device=x.device)
    lo = 0
    for e, m in enumerate(counts):
        hi = min(lo + m, x.shape[0])
        if hi > lo:
            out[lo:hi] = x[lo:hi] @ (w[e] if transposed else w[e].t().contiguous())
        lo = hi
    return out


def product(q, slack, w, counts, transposed=False, cut=False):
    """(sum, bound on the error of the fp32 sum of possibly different neighbours)."""
    red = w.shape[1] if transposed else w.shape[2]
    y = grouped(q, w, counts, transposed)
    bound = (red + blocks_of(red) + 2) * GAMMA * grouped(q.abs(), w.abs(), counts, transposed)
    if cut:
        bound = bound + CUT * grouped(q * q, w * w, counts, transposed).sqrt()
    if bool((slack != 0).any()):
        bound = bound + grouped(slack, w.abs(), counts, transposed) * (1 + 2.0 ** -10)
    return y, bound


def gated(e, de, g, dg):
    """silu(e) g and its bound; the sigmoid's exponent and reciprocal are good to a few steps, relative to |e| too."""
    s = torch.sigmoid(e)
    h = e * s * g
    return h, 1.1 * de * (g.abs() + dg) + (e * s).abs() * dg + (e.abs() + 8) * GAMMA * h.abs() + 2.0 ** -126


def gated_backward(dh, e, g):
    s = torch.sigmoid(e)
    grow = (2 * e.abs() + 16) * GAMMA
    de, dg = dh * g * s * (1 + e * (1 - s)), dh * e * s
    # (1 + e (1 - s) cancels for negative e: its error is relative to its terms)
    return de, grow * (dh * g * s).abs() * (1 + (e * (1 - s)).abs()) + 2.0 ** -126, dg, grow * dg.abs() + 2.0 ** -126


def assert_within(actual, expect, bound, what=""):
    """|actual - expect| <= bound + the rounding of expect to actual's type."""
    dtype = actual.dtype
    a = actual.double()
    # (a value below the type's normal range is rounded in absolute steps)
    limit = bound + half_step(dtype) * (expect.abs() + bound) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bad = ~((a - expect).abs() <= limit) & ~(a.isnan() & expect.isnan())
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at {bad.nonzero()[0].tolist()}: "
                                 f"{a[bad][0]:.9g} for {expect[bad][0]:.9g}, allowed {limit[bad][0]:.3g}")
