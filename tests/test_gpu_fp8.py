"""Expert products in 8-bit floating point against their definition in 64 bits: quantisation bit for bit, the grouped product
and its input gradient, the gated unit and its backward pass, the expert MLP, the module and the block."""
from types import SimpleNamespace

import pytest
import torch

from fp8_reference import (GAMMA, assert_within, blocks_of, dense, gated, gated_backward, grouped, product, quantize,
                           scale_exponent)

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn


def cut_in(out):
    return out.dtype != torch.float32


def make_rows(rows, k, dtype, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, k), generator=g)
    if spread:  # blocks of very different size
        x *= torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g).float())
    return x.to(dtype).to(DEV)


def make_weight(experts, n, k, seed):
    """Any bytes but NaN, any fp32 scales."""
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn((experts, n, k), generator=g) * 40).clamp_(-448, 448).to(FP8)
    scale = torch.rand((experts, blocks_of(n), blocks_of(k)), generator=g) * 1e-3 + 1e-4
    return w.to(DEV), scale.to(DEV)


def counts_of(rows, experts, kind, seed=0):
    if kind == "one":  # all rows with the last expert
        return [0] * (experts - 1) + [rows]
    if kind == "few":  # fewer rows than the operand has
        c = [0] * experts
        c[experts // 2] = rows // 2
        return c
    g = torch.Generator().manual_seed(seed)
    return torch.bincount(torch.randint(0, experts, (rows,), generator=g), minlength=experts).tolist()


def sizes(counts, dtype=torch.int32):
    return torch.tensor(counts, dtype=dtype, device=DEV)


def routed(tokens, k, experts, seed):
    from qwen3_moe_fused.kernels.indexing import get_expert_counts_and_idx

    g = torch.Generator().manual_seed(seed)
    sel = torch.rand((tokens, experts), generator=g).topk(k, dim=1).indices.reshape(-1).to(DEV)
    m_sizes, sort_idx, inv = get_expert_counts_and_idx(sel, experts)
    return m_sizes, sort_idx, inv, m_sizes.tolist()


# ---- quantisation ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 127), (5, 128), (2, 129), (67, 640), (33, 1001), (1, 5000), (300, 264)])
def test_rows_are_quantised_bit_for_bit(dtype, rows, k):
    from qwen3_moe_fused.quantize.fp8 import dequantize_fp8_rows, quantize_fp8_rows

    x = make_rows(rows, k, dtype, rows + k)
    x[0] = 0
    if rows > 2:
        x[1] *= 2.0 ** -14
        x[2, k // 2] = torch.finfo(dtype).max
    q, s = quantize_fp8_rows(x)
    ref, e, _ = quantize(x.double())
    assert q.shape == (rows, k) and q.dtype == FP8 and s.shape == (rows, blocks_of(k)) and s.dtype == torch.float8_e8m0fnu
    assert torch.equal(s.view(torch.uint8).double() - 127, e)
    values = q.double() * torch.exp2(e).repeat_interleave(128, 1)[:, :k]
    assert torch.equal(values, ref)
    for out in (torch.float32, torch.bfloat16):
        assert torch.equal(dequantize_fp8_rows(q, s, out), ref.to(out))


def test_rows_with_infinities_nan_and_the_borders_of_the_scale():
    from qwen3_moe_fused.quantize.fp8 import quantize_fp8_rows

    x = torch.zeros((9, 128), device=DEV)
    x[0, 5], x[0, 6] = float("inf"), 3.0
    x[1, 0], x[1, 1] = float("nan"), -448.0
    x[2, :] = float("-inf")
    x[3, 0] = 448.0
    x[4, 0] = 448.0 * (1 + 2.0 ** -23)  # the next scale
    x[5, 0] = 2.0 ** -140  # subnormal: the least scale
    x[6, 0] = torch.finfo(torch.float32).max
    x[7, 0], x[7, 1] = 448.0, 2.0 ** -9 * 1.5  # a tie between the grid's two smallest values
    x[8, 0], x[8, 1] = 448.0, -17.0  # a tie: to the even neighbour
    q, s = quantize_fp8_rows(x)
    ref, e, _ = quantize(x.double())
    assert torch.equal(s.view(torch.uint8).double() - 127, e)
    values = q.double() * torch.exp2(e).repeat_interleave(128, 1)
    assert torch.equal(values.isnan(), ref.isnan()) and torch.equal(values.nan_to_num(), ref.nan_to_num())
    assert q[0, 5].isnan() and not q[0, 6].isnan() and q[2].isnan().all()
    assert q[7, 1].float() == 2.0 ** -8 and q[8, 1].float() == -16.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 128, 256), (3, 130, 257), (2, 31, 5)])
def test_blocks_are_quantised_bit_for_bit(dtype, shape):
    from qwen3_moe_fused.quantize.fp8 import dequantize_fp8_blocks, quantize_fp8_blocks

    experts, n, k = shape
    w = make_rows(experts * n, k, dtype, sum(shape)).view(shape)
    q, s = quantize_fp8_blocks(w)
    assert q.shape == w.shape and s.shape == (experts, blocks_of(n), blocks_of(k))
    pad = torch.zeros((experts, blocks_of(n) * 128, blocks_of(k) * 128), dtype=torch.float64, device=DEV)
    pad[:, :n, :k] = w.double()
    amax = pad.abs().view(experts, blocks_of(n), 128, blocks_of(k), 128).amax(dim=(2, 4))
    e = scale_exponent(amax)
    assert torch.equal(s.double(), torch.exp2(e))
    v = w.double() / torch.exp2(e).repeat_interleave(128, 1)[:, :n].repeat_interleave(128, 2)[:, :, :k]
    step = torch.exp2((torch.frexp(v).exponent - 1).clamp(min=-6).double() - 3)
    assert torch.equal(q.double(), torch.round(v / step) * step)
    # any scales on the way back, rounded once
    s = s * 0.7
    for out in (torch.float32, torch.bfloat16):
        back = dequantize_fp8_blocks(q, s, out)
        assert torch.equal(back, dense(q, s).to(out))


# ---- the product and its input gradient -----------------------------------------------------------------------------------

# rows, experts, out, in, how the rows are dealt out
SHAPES = [
    (8, 128, 96, 256, "spread"),      # less than a row per expert
    (1, 3, 128, 128, "one"),
    (37, 5, 200, 328, "spread"),      # partial blocks both ways, 16-byte rows on neither side
    (70, 4, 33, 1001, "spread"),      # rows of odd length
    (300, 7, 256, 384, "spread"),
    (515, 2, 130, 64, "spread"),      # several row tiles per expert
    (129, 600, 64, 160, "spread"),    # more experts than a table of 512 holds
    (1000, 8, 768, 2048, "spread"),
    (700, 3, 384, 512, "one"),
    (90, 6, 272, 144, "few"),         # rows behind the last sequence
]


@pytest.mark.parametrize("rows,experts,n,k,kind", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_product_and_input_gradient(rows, experts, n, k, kind, dtype):
    from qwen3_moe_fused.quantize.layer_fp8 import moe_fused_linear_fp8

    counts = counts_of(rows, experts, kind)
    x, dy = make_rows(rows, k, dtype, 1, spread=False).requires_grad_(), make_rows(rows, n, dtype, 2, spread=False)
    w, s = make_weight(experts, n, k, 3)
    y = moe_fused_linear_fp8(x, w, s, sizes(counts))
    y.backward(dy)
    used, full = sum(counts), dense(w, s)
    for out, given, transposed in ((y.detach(), x.detach(), False), (x.grad, dy, True)):
        q, _, slack = quantize(given.double())
        ref, bound = product(q, slack, full, counts, transposed, cut_in(out))
        assert out.dtype == dtype
        assert_within(out[:used], ref[:used], bound[:used], "input gradient" if transposed else "forward")


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("index", [torch.int64, torch.int32, torch.uint8])
def test_output_types_and_row_count_types(out_dtype, index):
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import grouped_gemm_forward_fp8, grouped_gemm_forward_transposed_fp8

    counts = [3, 0, 41, 20]
    x, dy = make_rows(64, 256, torch.bfloat16, 4, spread=False), make_rows(64, 128, torch.bfloat16, 5, spread=False)
    w, s = make_weight(4, 128, 256, 6)
    y = grouped_gemm_forward_fp8(x, w, s, sizes(counts, index), out_dtype)
    dx = grouped_gemm_forward_transposed_fp8(dy, w, s, sizes(counts, index), out_dtype)
    for out, given, transposed in ((y, x, False), (dx, dy, True)):
        q, _, slack = quantize(given.double())
        assert out.dtype == out_dtype
        assert_within(out, *product(q, slack, dense(w, s), counts, transposed, cut_in(out)))


@pytest.mark.parametrize("rows", [24, 400, 3000])
def test_rows_outside_the_experts_are_left_as_they_were(rows):
    """Row counts that sum to less than the rows leave the others unwritten; more are cut at the last row, and negative ones
    count as none."""
    from qwen3_moe_fused import _lib
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import DX, FWD, fp8_weight, fp8_workspace

    n = k = 256
    x, dy = make_rows(rows, k, torch.bfloat16, 7, spread=False), make_rows(rows, n, torch.bfloat16, 8, spread=False)
    w, s = make_weight(3, n, k, 9)
    for counts in ([rows // 3, -5, rows // 4], [0, 0, 0], [rows // 2, rows, rows]):
        ms = sizes(counts)
        seen = [max(c, 0) for c in counts]
        used = min(sum(seen), rows)
        for transposed, given in ((False, x), (True, dy)):
            out = torch.full((rows + 8, 256), 7.0, device=DEV, dtype=torch.bfloat16)
            keep, ws, size = fp8_workspace(DX if transposed else FWD, x, rows, rows, n, k, 3)
            args = (ms.data_ptr(), _lib.I32, out.data_ptr(), rows, n, k, 3, _lib.BF16, _lib.BF16, ws, size, _lib.stream())
            if transposed:
                rc = _lib.lib().mfl_gemm_dx_fp8(given.data_ptr(), fp8_weight(w, s), *args)
            else:
                rc = _lib.lib().mfl_gemm_fwd_fp8(given.data_ptr(), rows, None, 1, fp8_weight(w, s), *args)
            assert rc == 0
            q, _, slack = quantize(given.double())
            ref, bound = product(q, slack, dense(w, s), seen, transposed, True)
            assert_within(out[:used], ref[:used], bound[:used])
            assert (out[used:] == 7.0).all()


def test_nan_and_infinity_stay_in_their_row_and_block():
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import grouped_gemm_forward_fp8

    for rows in (6, 200):
        x = make_rows(rows, 384, torch.bfloat16, 10, spread=False)
        w, s = make_weight(2, 256, 384, 11)
        clean = grouped_gemm_forward_fp8(x, w, s, sizes([rows - 2, 2]))
        x[1, 200], x[2, 3] = float("nan"), float("inf")
        s[1, 1, 2] = float("nan")  # the second expert's columns from 128 on
        y = grouped_gemm_forward_fp8(x, w, s, sizes([rows - 2, 2]))
        bad = torch.zeros_like(y, dtype=torch.bool)
        bad[1], bad[2], bad[-2:, 128:] = True, True, True
        assert torch.equal(y.isnan(), bad) and torch.equal(y[~bad], clean[~bad])


def test_partial_blocks_read_nothing_behind_them():
    """NaN weights of the next row, column or expert do not reach sums whose block ends before them."""
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import grouped_gemm_forward_fp8, grouped_gemm_forward_transposed_fp8

    for n, k in ((48, 208), (48, 77)):
        for rows in (5, 170):
            w, s = make_weight(3, n, k, 12)
            w[1] = torch.full_like(w[1].float(), float("nan")).to(FP8)
            counts = [rows, 0, 2]
            x, dy = make_rows(rows + 2, k, torch.float32, 13, False), make_rows(rows + 2, n, torch.float32, 14, False)
            full = dense(w, s)
            full[1] = 0
            for out, given, transposed in ((grouped_gemm_forward_fp8(x, w, s, sizes(counts)), x, False),
                                           (grouped_gemm_forward_transposed_fp8(dy, w, s, sizes(counts)), dy, True)):
                q, _, slack = quantize(given.double())
                assert_within(out, *product(q, slack, full, counts, transposed, cut_in(out)))


def test_gradient_against_differences():
    """The product is linear between points of the grid: rows and directions of small whole numbers, whose blocks share one
    scale, are on it, and so are the output gradients."""
    from qwen3_moe_fused.quantize.layer_fp8 import moe_fused_linear_fp8

    g = torch.Generator().manual_seed(15)
    rows, n, k, counts = 40, 160, 192, [13, 0, 27]
    x = torch.randint(-4, 5, (rows, k), generator=g).float()
    d = torch.randint(-2, 3, (rows, k), generator=g).float()
    dy = torch.randint(-7, 8, (rows, n), generator=g).float()
    w, s = make_weight(3, n, k, 16)
    x, d, dy = x.to(DEV).requires_grad_(), d.to(DEV), dy.to(DEV)
    y0 = moe_fused_linear_fp8(x, w, s, sizes(counts))
    y0.backward(dy)
    y1 = moe_fused_linear_fp8(x.detach() + d, w, s, sizes(counts))
    diff = ((y1 - y0.detach()).double() * dy.double()).sum()
    full = dense(w, s)
    size = (grouped(x.detach().double().abs() + d.double().abs(), full.abs(), counts) * dy.double().abs()).sum()
    assert abs(float(diff - (x.grad.double() * d.double()).sum())) <= 4 * (k + n) * GAMMA * float(size)


# ---- the gated unit -------------------------------------------------------------------------------------------------------

GATED = [
    # tokens, selected, experts, hidden, intermediate
    (1, 8, 128, 256, 96),
    (1, 1, 2, 128, 128),
    (5, 3, 7, 200, 72),
    (60, 4, 9, 1001, 33),
    (96, 4, 4, 512, 384),
    (700, 2, 6, 320, 272),
    (33, 2, 600, 128, 64),
]


def gated_reference(tokens, w, sort_idx, k, counts):
    q, _, slack = quantize(tokens.double())
    q = q[sort_idx.long() // k]
    slack = torch.zeros_like(q)
    e, de = product(q, slack, dense(*w[0]), counts, cut=cut_in(tokens))
    g, dg = product(q, slack, dense(*w[1]), counts, cut=cut_in(tokens))
    return e, de, g, dg


@pytest.mark.parametrize("tokens,k,experts,hidden,inter", GATED)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_gated_unit_and_its_backward(tokens, k, experts, hidden, inter, dtype):
    from qwen3_moe_fused.grouped_gemm.fused import grouped_glu_backward_fp8, grouped_glu_forward_fp8

    m_sizes, sort_idx, _, counts = routed(tokens, k, experts, 20)
    x = make_rows(tokens, hidden, dtype, 21, spread=False)
    w = [make_weight(experts, inter, hidden, 22 + i) for i in range(2)]
    w = [(q, s / s.mean() * (40.0 * hidden ** 0.5) ** -1) for q, s in w]  # projections of about unit variance
    h, e, g = grouped_glu_forward_fp8(x, *w[0], *w[1], m_sizes, sort_idx, k, return_products=True)
    re, de, rg, dg = gated_reference(x, w, sort_idx, k, counts)
    assert_within(e, re, de, "gate projection")
    assert_within(g, rg, dg, "up projection")
    assert_within(h, *gated(re, de, rg, dg), "gated unit")
    only = grouped_glu_forward_fp8(x, *w[0], *w[1], m_sizes, sort_idx, k)
    assert torch.equal(only, h)

    dh = make_rows(tokens * k, inter, dtype, 24, spread=False)
    dx = grouped_glu_backward_fp8(dh, e, g, *w[0], *w[1], m_sizes)
    a, ea, b, eb = gated_backward(dh.double(), e.double(), g.double())
    total, bound = 0, 0
    for v, err, (q, s) in ((a, ea, w[0]), (b, eb, w[1])):
        qv, _, slack = quantize(v, err)
        t, bd = product(qv, slack, dense(q, s), counts, True, cut_in(dx))
        total, bound = total + t, bound + 2 * bd  # (one sum over both terms: twice as many additions)
    assert_within(dx, total, bound, "gradient of the rows")


def test_gated_unit_without_gathered_rows():
    from qwen3_moe_fused.grouped_gemm.fused import grouped_glu_forward_fp8

    counts = [0, 17, 3]
    x = make_rows(20, 256, torch.bfloat16, 25, spread=False)
    w = [make_weight(3, 128, 256, 26 + i) for i in range(2)]
    idx = torch.arange(20, device=DEV, dtype=torch.int32)
    a = grouped_glu_forward_fp8(x, *w[0], *w[1], sizes(counts))
    assert torch.equal(a, grouped_glu_forward_fp8(x, *w[0], *w[1], sizes(counts), idx, 1))


def test_gated_unit_under_autograd_sums_each_tokens_rows():
    from qwen3_moe_fused.fused_mlp import moe_fused_glu_fp8
    from qwen3_moe_fused.grouped_gemm.fused import grouped_glu_backward_fp8, grouped_glu_forward_fp8
    from qwen3_moe_fused.kernels.routing import _combine

    m_sizes, sort_idx, inv, _ = routed(50, 3, 8, 28)
    x = make_rows(50, 256, torch.bfloat16, 29, spread=False).requires_grad_()
    w = [t for i in range(2) for t in make_weight(8, 128, 256, 30 + i)]
    h = moe_fused_glu_fp8(x, *w, m_sizes, sort_idx, inv, 3)
    dh = make_rows(150, 128, torch.bfloat16, 32, spread=False)
    h.backward(dh)
    h2, e, g = grouped_glu_forward_fp8(x.detach(), *w, m_sizes, sort_idx, 3, return_products=True)
    assert torch.equal(h, h2)
    rows = grouped_glu_backward_fp8(dh, e, g, *w, m_sizes)
    assert torch.equal(x.grad, _combine(rows, inv, None, 50, 3))


# ---- the expert MLP -------------------------------------------------------------------------------------------------------

def mlp_weights(experts, hidden, inter, seed):
    out = []
    for i, (n, k) in enumerate(((inter, hidden), (inter, hidden), (hidden, inter))):
        q, s = make_weight(experts, n, k, seed + i)
        out += [q, s / s.mean() * (40.0 * k ** 0.5) ** -1]
    return out


@pytest.mark.parametrize("tokens,k,experts,hidden,inter", GATED + [(1200, 4, 8, 256, 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_expert_mlp(tokens, k, experts, hidden, inter, dtype):
    from qwen3_moe_fused.fused_mlp import moe_fused_mlp_fp8

    m_sizes, sort_idx, inv, counts = routed(tokens, k, experts, 33)
    x = make_rows(tokens, hidden, dtype, 34, spread=False)
    w = mlp_weights(experts, hidden, inter, 35)
    y = moe_fused_mlp_fp8(x, *w, m_sizes, sort_idx, inv, k)
    h, dh = gated(*gated_reference(x, ((w[0], w[1]), (w[2], w[3])), sort_idx, k, counts))
    q, _, slack = quantize(h, dh)
    assert_within(y, *product(q, slack, dense(w[4], w[5]), counts, cut=cut_in(y)), "expert MLP")


def test_expert_mlp_backward_is_its_parts():
    from qwen3_moe_fused.fused_mlp import moe_fused_mlp_fp8
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import grouped_gemm_forward_transposed_fp8
    from qwen3_moe_fused.grouped_gemm.fused import grouped_glu_backward_fp8, grouped_glu_forward_fp8
    from qwen3_moe_fused.kernels.routing import _combine

    m_sizes, sort_idx, inv, _ = routed(70, 4, 8, 36)
    x = make_rows(70, 256, torch.bfloat16, 37, spread=False).requires_grad_()
    w = mlp_weights(8, 256, 128, 38)
    y = moe_fused_mlp_fp8(x, *w, m_sizes, sort_idx, inv, 4)
    dy = make_rows(280, 256, torch.bfloat16, 39, spread=False)
    y.backward(dy)
    _, e, g = grouped_glu_forward_fp8(x.detach(), *w[:4], m_sizes, sort_idx, 4, return_products=True)
    dh = grouped_gemm_forward_transposed_fp8(dy, w[4], w[5], m_sizes)
    assert torch.equal(x.grad, _combine(grouped_glu_backward_fp8(dh, e, g, *w[:4], m_sizes), inv, None, 70, 4))
    with torch.no_grad():
        assert torch.equal(moe_fused_mlp_fp8(x, *w, m_sizes, sort_idx, inv, 4), y)


# ---- empty calls, streams, graphs -----------------------------------------------------------------------------------------

def test_no_rows_and_no_tokens():
    from qwen3_moe_fused.fused_mlp import moe_fused_glu_fp8, moe_fused_mlp_fp8
    from qwen3_moe_fused.quantize.fp8 import dequantize_fp8_rows, quantize_fp8_rows
    from qwen3_moe_fused.quantize.layer_fp8 import moe_fused_linear_fp8

    w = mlp_weights(4, 128, 96, 40)
    none = torch.zeros(4, dtype=torch.int32, device=DEV)
    x = torch.empty((0, 128), device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = moe_fused_linear_fp8(x, w[0], w[1], none)
    y.sum().backward()
    assert y.shape == (0, 96) and x.grad.shape == (0, 128)
    idx = torch.empty(0, dtype=torch.int32, device=DEV)
    assert moe_fused_glu_fp8(x.detach(), *w[:4], none, idx, idx, 2).shape == (0, 96)
    assert moe_fused_mlp_fp8(x.detach(), *w, none, idx, idx, 2).shape == (0, 128)
    q, s = quantize_fp8_rows(x.detach())
    assert dequantize_fp8_rows(q, s).shape == (0, 128)


def test_another_stream_and_replayed_graphs():
    """Two graphs of one pool, replayed in turn with eager calls between them, and a call on a stream of its own."""
    from qwen3_moe_fused.fused_mlp import moe_fused_mlp_fp8

    w = mlp_weights(8, 256, 128, 41)
    cases = []
    for tokens, seed in ((3, 42), (300, 43)):
        m_sizes, sort_idx, inv, _ = routed(tokens, 2, 8, seed)
        cases.append((make_rows(tokens, 256, torch.bfloat16, seed, spread=False), m_sizes, sort_idx, inv))

    def run(c):
        return moe_fused_mlp_fp8(c[0], *w, *c[1:], 2)

    expect = [run(c).clone() for c in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [run(c) for c in cases]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(others, expect))
    graphs, outs, pool = [], [], None
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(run(c))
        pool = graph.pool()
        graphs.append(graph)
    for turn in range(4):
        for i in (0, 1):
            cases[i][0].mul_(-1)  # new inputs in place
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], run(cases[i])), (turn, i)


# ---- the module and the block ---------------------------------------------------------------------------------------------

def make_block(dtype, hidden=256, inter=128, experts=8, k=2, seed=50):
    from qwen3_moe_fused.modular_qwen3_moe_fused import Qwen3MoeFusedSparseMoeBlock
    from qwen3_moe_fused.quantize.layer_fp8 import MoeFusedLinearFp8

    torch.manual_seed(seed)
    block = Qwen3MoeFusedSparseMoeBlock(SimpleNamespace(num_experts=experts, num_experts_per_tok=k, norm_topk_prob=True,
                                                        hidden_size=hidden, moe_intermediate_size=inter, hidden_act="silu"))
    block = block.to(DEV).to(dtype)
    for name in ("gate_proj", "up_proj", "down_proj"):
        setattr(block, name, MoeFusedLinearFp8.from_linear(getattr(block, name)))
    return block


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens", [1, 130])
def test_block_runs_on_the_8_bit_projections(dtype, tokens):
    """The block against its parts called one by one, forward and backward."""
    from qwen3_moe_fused.fused_mlp import moe_fused_mlp_fp8
    from qwen3_moe_fused.kernels.routing import combine_rows
    from qwen3_moe_fused.modular_qwen3_moe_fused import route_tokens

    block = make_block(dtype)
    x = make_rows(tokens, 256, dtype, 51, spread=False).view(1, tokens, 256)
    dout = make_rows(tokens, 256, dtype, 52, spread=False).view(1, tokens, 256)
    results = []
    for parts in (False, True):
        block.zero_grad(set_to_none=True)
        xi = x.clone().requires_grad_()
        if parts:
            t = xi.view(tokens, 256)
            logits, weights, m_sizes, sort_idx, inv = route_tokens(block, t)
            w = [p for m in (block.gate_proj, block.up_proj, block.down_proj) for p in (m.weight, m.weight_scale_inv)]
            out = combine_rows(moe_fused_mlp_fp8(t, *w, m_sizes, sort_idx, inv, 2), inv, weights, sort_idx).view(x.shape)
        else:
            out, logits = block(xi)
        out.backward(dout)
        results.append((out.detach(), logits.detach(), xi.grad, block.gate.weight.grad))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(block(x)[0], results[0][0])


def test_block_with_a_hook_or_separate_steps_calls_the_modules():
    block = make_block(torch.bfloat16)
    x = make_rows(40, 256, torch.bfloat16, 53, spread=False).view(1, 40, 256)
    calls = []
    with torch.no_grad():
        expect = block(x)[0]
        handle = block.down_proj.register_forward_hook(lambda *a: calls.append(1))
        hooked = block(x)[0]
        handle.remove()
        block.fuse_front = False
        separate = block(x)[0]
    assert calls == [1]
    # h rounded to bf16 before it is quantised: a rounding of a step in places
    for other in (hooked, separate):
        assert (other.float() - expect.float()).norm() <= 0.05 * expect.float().norm()


def test_module_keeps_its_types_and_its_state(tmp_path):
    from qwen3_moe_fused.modular_qwen3_moe_fused import MoeFusedLinear
    from qwen3_moe_fused.quantize.fp8 import quantize_fp8_blocks
    from qwen3_moe_fused.quantize.layer_fp8 import MoeFusedLinearFp8

    torch.manual_seed(54)
    plain = MoeFusedLinear(200, 136, 3).to(DEV)
    q, s = quantize_fp8_blocks(plain.weight.detach())
    module = MoeFusedLinearFp8.from_linear(plain)
    assert torch.equal(module.weight.view(torch.uint8), q.view(torch.uint8)) and torch.equal(module.weight_scale_inv, s)
    for moved in (module.to(torch.bfloat16), module.half(), module.cpu().to(DEV)):
        assert moved.weight.dtype == FP8 and moved.weight_scale_inv.dtype == torch.float32 and not moved.weight.requires_grad
        assert torch.equal(moved.weight.view(torch.uint8), q.view(torch.uint8)) and torch.equal(moved.weight_scale_inv, s)
    torch.save(module.state_dict(), tmp_path / "state.pt")
    state = torch.load(tmp_path / "state.pt", weights_only=True)
    assert set(state) == {"weight", "weight_scale_inv"}
    for other in (MoeFusedLinearFp8(200, 136, 3, device=DEV), MoeFusedLinearFp8(200, 136, 3).to(DEV)):
        other.load_state_dict(state)
        x = make_rows(10, 200, torch.bfloat16, 55)
        assert torch.equal(other(x, sizes([4, 0, 6])), module(x, sizes([4, 0, 6])))
    other = MoeFusedLinearFp8(200, 136, 3, device=DEV)
    other.load_state_dict(plain.state_dict())  # a floating-point weight is quantised
    assert torch.equal(other.weight.view(torch.uint8), q.view(torch.uint8))


def test_lora_over_8_bit_weights():
    """An adapter over a frozen 8-bit projection: the base product's gradient plus the adapter's; the joined LoRA path, which
    does not know the scales, refuses."""
    from qwen3_moe_fused.fast_lora import get_lora_parameters
    from qwen3_moe_fused.functional import moe_fused_linear
    from qwen3_moe_fused.lora import HAVE_PEFT, LoraMoeFusedLinear
    from qwen3_moe_fused.modular_qwen3_moe_fused import MoeFusedLinear
    from qwen3_moe_fused.quantize.layer_fp8 import MoeFusedLinearFp8, moe_fused_linear_fp8

    if HAVE_PEFT:
        pytest.skip("written against the stand-in base class")
    torch.manual_seed(56)
    base = MoeFusedLinearFp8.from_linear(MoeFusedLinear(128, 96, 4).to(DEV))
    lora = LoraMoeFusedLinear(base, "default", r=8, lora_alpha=16).to(DEV)
    a, b = lora.lora_A["default"].weight, lora.lora_B["default"].weight
    assert a.dtype == torch.float32
    with torch.no_grad():
        b.normal_(0, 0.1)
    x = make_rows(30, 128, torch.float32, 57, spread=False).requires_grad_()
    ms, dy = sizes([10, 0, 15, 5]), make_rows(30, 96, torch.float32, 58, spread=False)
    lora(x, ms).backward(dy)
    got = (x.grad, a.grad, b.grad)
    x2, a2, b2 = x.detach().clone().requires_grad_(), a.detach().clone().requires_grad_(), b.detach().clone().requires_grad_()
    (moe_fused_linear_fp8(x2, base.weight, base.weight_scale_inv, ms)
     + moe_fused_linear(moe_fused_linear(x2, a2, ms), b2, ms) * 2.0).backward(dy)
    for u, v in zip(got, (x2.grad, a2.grad, b2.grad)):
        assert torch.equal(u, v)
    with pytest.raises(NotImplementedError):
        get_lora_parameters(lora)


# ---- sizes at which another kernel or tile takes over ---------------------------------------------------------------------

TAKEOVERS = [
    # rows, experts, out, in: rows whose bytes no 16-byte access fits, with rows for most experts (the weights are copied to
    # padded rows) and without; one step of the reduction; large tiles, partial rows and columns among them
    (700, 9, 200, 331),
    (700, 9, 331, 200),
    (700, 9, 47, 129),
    (20, 9, 200, 331),
    (600, 5, 256, 112),
    (600, 5, 112, 256),
    (9000, 8, 2000, 2064),
    (36000, 6, 2064, 288),
    (36000, 6, 288, 2064),
]


@pytest.mark.parametrize("rows,experts,n,k", TAKEOVERS)
def test_product_where_another_kernel_takes_over(rows, experts, n, k):
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import grouped_gemm_forward_fp8, grouped_gemm_forward_transposed_fp8

    counts = counts_of(rows, experts, "spread", 60)
    x, dy = make_rows(rows, k, torch.bfloat16, 61, spread=False), make_rows(rows, n, torch.bfloat16, 62, spread=False)
    w, s = make_weight(experts, n, k, 63)
    full = dense(w, s)
    for out, given, transposed in ((grouped_gemm_forward_fp8(x, w, s, sizes(counts)), x, False),
                                   (grouped_gemm_forward_transposed_fp8(dy, w, s, sizes(counts)), dy, True)):
        q, _, slack = quantize(given.double())
        assert_within(out, *product(q, slack, full, counts, transposed, True), "input gradient" if transposed else "forward")


@pytest.mark.parametrize("tokens,k,experts,hidden,inter", [(300, 3, 7, 331, 200), (300, 3, 7, 200, 331), (5000, 4, 6, 1040, 1168),
                                                           (400, 2, 5, 256, 144), (300, 2, 4, 100, 80)])
def test_gated_unit_and_mlp_where_another_kernel_takes_over(tokens, k, experts, hidden, inter):
    from qwen3_moe_fused.fused_mlp import moe_fused_mlp_fp8
    from qwen3_moe_fused.grouped_gemm.fused import grouped_glu_backward_fp8, grouped_glu_forward_fp8

    m_sizes, sort_idx, inv, counts = routed(tokens, k, experts, 64)
    x = make_rows(tokens, hidden, torch.bfloat16, 65, spread=False)
    w = mlp_weights(experts, hidden, inter, 66)
    h, e, g = grouped_glu_forward_fp8(x, *w[:4], m_sizes, sort_idx, k, return_products=True)
    re, de, rg, dg = gated_reference(x, ((w[0], w[1]), (w[2], w[3])), sort_idx, k, counts)
    assert_within(e, re, de, "gate projection")
    assert_within(g, rg, dg, "up projection")
    rh, dh = gated(re, de, rg, dg)
    assert_within(h, rh, dh, "gated unit")
    q, _, slack = quantize(rh, dh)
    y = moe_fused_mlp_fp8(x, *w, m_sizes, sort_idx, inv, k)
    assert_within(y, *product(q, slack, dense(w[4], w[5]), counts, cut=True), "expert MLP")
    dh = make_rows(tokens * k, inter, torch.bfloat16, 67, spread=False)
    dx = grouped_glu_backward_fp8(dh, e, g, *w[:4], m_sizes)
    a, ea, b, eb = gated_backward(dh.double(), e.double(), g.double())
    total, bound = 0, 0
    for v, err, (wq, s) in ((a, ea, w[0:2]), (b, eb, w[2:4])):
        qv, _, slack = quantize(v, err)
        t, bd = product(qv, slack, dense(wq, s), counts, True, True)
        total, bound = total + t, bound + 2 * bd
    assert_within(dx, total, bound, "gradient of the rows")


# ---- calls that lie a little apart ----------------------------------------------------------------------------------------

def off_grid(t):
    """The same values, contiguous, one element behind a 16-byte boundary."""
    raw = torch.empty(t.numel() + 1, dtype=torch.uint8 if t.dtype == FP8 else t.dtype, device=DEV)[1:]
    view = (raw.view(FP8) if t.dtype == FP8 else raw).view(t.shape)
    view.copy_(t)
    assert view.is_contiguous() and view.data_ptr() % 16 != 0
    return view


@pytest.mark.parametrize("rows", [6, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_operands_off_the_16_byte_grid(rows, dtype):
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import grouped_gemm_forward_fp8, grouped_gemm_forward_transposed_fp8

    n, k, counts = 272, 384, [rows - 4, 0, 4]
    x, dy = make_rows(rows, k, dtype, 70, spread=False), make_rows(rows, n, dtype, 71, spread=False)
    w, s = make_weight(3, n, k, 72)
    for wi, xi, di in ((w, off_grid(x), off_grid(dy)), (off_grid(w), x, dy), (off_grid(w), off_grid(x), off_grid(dy))):
        for out, given, transposed in ((grouped_gemm_forward_fp8(xi, wi, s, sizes(counts)), x, False),
                                       (grouped_gemm_forward_transposed_fp8(di, wi, s, sizes(counts)), dy, True)):
            q, _, slack = quantize(given.double())
            assert_within(out, *product(q, slack, dense(w, s), counts, transposed, cut_in(out)))


@pytest.mark.parametrize("tokens", [3, 200])
def test_mlp_operands_off_the_16_byte_grid(tokens):
    from qwen3_moe_fused.fused_mlp import moe_fused_mlp_fp8

    m_sizes, sort_idx, inv, counts = routed(tokens, 2, 8, 73)
    x, w = make_rows(tokens, 256, torch.bfloat16, 74, spread=False), mlp_weights(8, 256, 128, 75)
    h, dh = gated(*gated_reference(x, ((w[0], w[1]), (w[2], w[3])), sort_idx, 2, counts))
    q, _, slack = quantize(h, dh)
    expect = product(q, slack, dense(w[4], w[5]), counts, cut=True)
    shifted = [off_grid(t) for t in w[::2]]
    for xi, weights in ((off_grid(x), w), (x, [shifted[0], *w[1:]]), (x, [*w[:4], shifted[2], w[5]])):
        assert_within(moe_fused_mlp_fp8(xi, *weights, m_sizes, sort_idx, inv, 2), *expect)


@pytest.mark.parametrize("rows,experts,n,k", [(40, 3, 192, 9280), (40, 3, 9280, 192), (600, 3, 192, 9280), (600, 3, 9280, 192),
                                              (5000, 512, 128, 288), (5000, 513, 128, 288), (4096, 511, 128, 288)])
def test_long_reductions_and_many_experts(rows, experts, n, k):
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import grouped_gemm_forward_fp8, grouped_gemm_forward_transposed_fp8

    counts = counts_of(rows, experts, "spread", 76)
    x, dy = make_rows(rows, k, torch.bfloat16, 77, spread=False), make_rows(rows, n, torch.bfloat16, 78, spread=False)
    w, s = make_weight(experts, n, k, 79)
    for out, given, transposed in ((grouped_gemm_forward_fp8(x, w, s, sizes(counts, torch.int64)), x, False),
                                   (grouped_gemm_forward_transposed_fp8(dy, w, s, sizes(counts, torch.int64)), dy, True)):
        q, _, slack = quantize(given.double())
        assert_within(out, *product(q, slack, dense(w, s), counts, transposed, True))


def test_mlp_over_a_full_table_of_experts():
    from qwen3_moe_fused.fused_mlp import moe_fused_mlp_fp8

    m_sizes, sort_idx, inv, counts = routed(1500, 4, 512, 80)
    x, w = make_rows(1500, 512, torch.bfloat16, 81, spread=False), mlp_weights(512, 512, 128, 82)
    h, dh = gated(*gated_reference(x, ((w[0], w[1]), (w[2], w[3])), sort_idx, 4, counts))
    q, _, slack = quantize(h, dh)
    assert_within(moe_fused_mlp_fp8(x, *w, m_sizes, sort_idx, inv, 4), *product(q, slack, dense(w[4], w[5]), counts, cut=True))


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scales_whose_product_overflows(rows, dtype):
    """Huge rows on weights of zeros with huge scales are zero, and tiny scales of either kind meet huge ones of the other."""
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import grouped_gemm_forward_fp8

    x = make_rows(rows, 256, torch.float32, 83, spread=False)
    w, s = make_weight(2, 128, 256, 84)
    counts = [rows - 2, 2]
    zero = torch.zeros_like(w.float()).to(FP8)
    y = grouped_gemm_forward_fp8((x * 2.0 ** 110).to(dtype), zero, torch.full_like(s, 2.0 ** 40), sizes(counts))
    assert (y == 0).all()
    base = grouped_gemm_forward_fp8(x.to(dtype), w, s, sizes(counts))
    for up in (90, -90):
        y = grouped_gemm_forward_fp8((x * 2.0 ** up).to(dtype), w, s * 2.0 ** -up, sizes(counts))
        assert torch.equal(y, base)


def test_training_steps_in_a_graph_and_on_two_streams_at_once():
    from qwen3_moe_fused.fused_mlp import moe_fused_glu_fp8, moe_fused_mlp_fp8
    from qwen3_moe_fused.quantize.layer_fp8 import moe_fused_linear_fp8

    m_sizes, sort_idx, inv, _ = routed(300, 2, 8, 85)
    w = mlp_weights(8, 256, 128, 86)
    x = make_rows(300, 256, torch.bfloat16, 87, spread=False).requires_grad_()
    rows = make_rows(600, 256, torch.bfloat16, 88, spread=False).requires_grad_()
    dy, dh = make_rows(600, 256, torch.bfloat16, 89, False), make_rows(600, 128, torch.bfloat16, 90, False)

    def step():
        y = moe_fused_mlp_fp8(x, *w, m_sizes, sort_idx, inv, 2)
        h = moe_fused_glu_fp8(x, *w[:4], m_sizes, sort_idx, inv, 2)
        p = moe_fused_linear_fp8(rows, w[0], w[1], m_sizes)
        grads = [torch.autograd.grad(o, i, d)[0] for o, i, d in ((y, x, dy), (h, x, dh), (p, rows, dh))]
        return [t.detach() for t in (y, h, p)] + grads

    expect = step()
    streams, results = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s, r in zip(streams, results):
            with torch.cuda.stream(s):
                r.append(step())
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for got in r for a, b in zip(got, expect))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        with torch.no_grad():
            x.mul_(-1), rows.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), turn


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [5, 90])
def test_nan_and_infinity_in_every_type_and_through_the_mlp(dtype, tokens):
    """A token with an element that is no finite number comes out as NaN, the others as without it; a gated unit that overflows
    (its fp32 values are infinite) does the same to its rows."""
    from qwen3_moe_fused.fused_mlp import moe_fused_mlp_fp8
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import grouped_gemm_forward_fp8

    m_sizes, sort_idx, inv, counts = routed(tokens, 2, 8, 91)
    x, w = make_rows(tokens, 400, dtype, 92, spread=False), mlp_weights(8, 400, 272, 93)
    clean, rows = moe_fused_mlp_fp8(x, *w, m_sizes, sort_idx, inv, 2), x[sort_idx.long() // 2].contiguous()
    flat = grouped_gemm_forward_fp8(rows, w[0], w[1], m_sizes)
    x[1, 399], x[2, 130] = float("inf"), float("nan")
    bad = ((sort_idx // 2 == 1) | (sort_idx // 2 == 2)).cpu()
    for out, expect in ((moe_fused_mlp_fp8(x, *w, m_sizes, sort_idx, inv, 2), clean),
                        (grouped_gemm_forward_fp8(x[sort_idx.long() // 2].contiguous(), w[0], w[1], m_sizes), flat)):
        assert torch.equal(out.isnan().cpu(), bad[:, None].expand(out.shape)) and torch.equal(out[~bad], expect[~bad])
    x = make_rows(tokens, 400, dtype, 92, spread=False)
    up = w[3].clone()
    up[int((m_sizes > 0).nonzero()[0])] = 3e38  # the first expert with rows
    out = moe_fused_mlp_fp8(x, *w[:3], up, *w[4:], m_sizes, sort_idx, inv, 2)
    first = next(c for c in counts if c)
    assert out[:first].isnan().all() and torch.equal(out[first:], clean[first:])


@pytest.mark.parametrize("k", [9, 15, 17, 31, 135])
def test_narrow_odd_rows_of_weights(k):
    """Rows shorter than 16 bytes, and rows whose last piece has every kind of length, copied to padded rows."""
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import grouped_gemm_forward_fp8, grouped_gemm_forward_transposed_fp8

    counts = counts_of(700, 9, "spread", 94)
    x, dy = make_rows(700, k, torch.bfloat16, 95, spread=False), make_rows(700, 300, torch.bfloat16, 96, spread=False)
    w, s = make_weight(9, 300, k, 97)
    for out, given, transposed in ((grouped_gemm_forward_fp8(x, w, s, sizes(counts)), x, False),
                                   (grouped_gemm_forward_transposed_fp8(dy, w, s, sizes(counts)), dy, True)):
        q, _, slack = quantize(given.double())
        assert_within(out, *product(q, slack, dense(w, s), counts, transposed, True), "input gradient" if transposed else "forward")


@pytest.mark.parametrize("shift", [0, 1])
def test_mlp_through_the_c_interface_writes_its_workspace_only(shift):
    """Outputs on and off the 16-byte grid, with a workspace of the size that is asked for and guard bytes behind it."""
    from qwen3_moe_fused import _lib
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import MLP, MLP_OFF_GRID, fp8_weight
    from qwen3_moe_fused.grouped_gemm.fused import grouped_mlp_forward_fp8

    m_sizes, sort_idx, _, counts = routed(300, 2, 8, 98)
    for hidden, inter in ((256, 136), (331, 200)):
        x, w = make_rows(300, hidden, torch.bfloat16, 99, spread=False), mlp_weights(8, hidden, inter, 100)
        y, e, g = grouped_mlp_forward_fp8(x, *w, m_sizes, sort_idx, 2, return_products=True)
        ours = torch.full((3, 600 * max(hidden, inter) + 8), 7.0, device=DEV, dtype=torch.bfloat16)
        out = [ours[i, shift:shift + t.numel()].view(t.shape) for i, t in enumerate((y, e, g))]
        size = _lib.lib().mfl_fp8_workspace(MLP_OFF_GRID if shift else MLP, 300, 600, inter, hidden, 8)
        ws = torch.full((size + 4096,), 171, device=DEV, dtype=torch.uint8)
        rc = _lib.lib().mfl_mlp_fwd_fp8(x.data_ptr(), 300, sort_idx.data_ptr(), 2, *(fp8_weight(*w[i:i + 2]) for i in (0, 2, 4)),
                                        m_sizes.data_ptr(), _lib.I32, *(t.data_ptr() for t in out), 600, inter, hidden, 8,
                                        _lib.BF16, ws.data_ptr(), size, _lib.stream())
        assert rc == 0 and (ws[size:] == 171).all()
        for t, buf in zip(out, ours):
            assert (buf[:shift] == 7).all() and (buf[shift + t.numel():] == 7).all()
        re, de, rg, dg = gated_reference(x, ((w[0], w[1]), (w[2], w[3])), sort_idx, 2, counts)
        assert_within(out[1], re, de, "gate projection")
        assert_within(out[2], rg, dg, "up projection")
        q, _, slack = quantize(*gated(re, de, rg, dg))
        assert_within(out[0], *product(q, slack, dense(w[4], w[5]), counts, cut=True), "expert MLP")
        if not shift:
            assert all(torch.equal(a, b) for a, b in zip(out, (y, e, g)))


# ---- how far the expert MLP is from its definition as a whole ---------------------------------------------------------------

# The gated unit's values are rounded to the 8-bit grid from computed sums.  A value that is off by d lands on the other side of a
# border with probability d / step and is then off by a step, 1/8 of the value at most, so the mean square of what that adds is
# d |h| / 8.  For e, g of unit variance and sums off by s on average that is 1.8 s / 8 of the mean square of h (E[|silu'(e) silu(e)|] =
# 0.36, E[silu(e)^2] = 0.36, E|g| = 0.8), and the down projection keeps the ratio.  fp32 sums: some 24 roundings one behind the
# other, each with a standard deviation of 2^-24 / sqrt(3), so s = 0.8 * 1.7e-7, which gives 1.7e-4; twice that for the few values
# of a test.  Products cut off 2^-13 below the largest of eight (bf16 rows, more than 8 per expert): s <= 0.8 * 2^-13 sqrt(8 / 3)
# (the reference's CUT), 6.0e-3.
BORDERS, BORDERS_CUT = 3.5e-4, 6e-3


@pytest.mark.parametrize("tokens,k,experts", [(128, 8, 128), (300, 4, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_expert_mlp_is_as_near_as_its_type(tokens, k, experts, dtype):
    """Over the norm, and beyond the rounding of the output itself."""
    from qwen3_moe_fused.fused_mlp import moe_fused_mlp_fp8

    m_sizes, sort_idx, inv, counts = routed(tokens, k, experts, 101)
    x, w = make_rows(tokens, 2048, dtype, 102, spread=False), mlp_weights(experts, 2048, 256, 103)
    y = moe_fused_mlp_fp8(x, *w, m_sizes, sort_idx, inv, k)
    rows = quantize(x.double())[0][sort_idx.long() // k]
    e, g = (grouped(rows, dense(w[i], w[i + 1]), counts) for i in (0, 2))
    exact = grouped(quantize(e * torch.sigmoid(e) * g)[0], dense(w[4], w[5]), counts)
    off = [((t.double() - exact).norm() / exact.norm()).item() for t in (y, exact.to(dtype))]
    beyond = max(off[0] ** 2 - off[1] ** 2, 0.0) ** 0.5
    tiles_in_8_bit = dtype == torch.bfloat16 and tokens * k > 8 * experts
    assert beyond <= (BORDERS_CUT if tiles_in_8_bit else BORDERS), (beyond, *off)


@pytest.mark.parametrize("rows,width", [(24, 256), (400, 256), (400, 128)])  # decode kernel, tiles, any shape's kernel
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_counts_past_every_integer_are_cut_at_the_last_row(rows, width, index):
    from qwen3_moe_fused import _lib
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import DX, FWD, fp8_weight, fp8_workspace

    x = make_rows(rows, width, torch.bfloat16, 104, spread=False)
    w, s = make_weight(4, width, width, 105)
    top = torch.iinfo(index).max
    q, _, slack = quantize(x.double())
    for counts in ([7, top, top, 5], [top, top, 5, top], [-top, 3, top - 2, top], [0, top, -1, 1]):
        taken, left = [], rows
        for c in counts:
            taken.append(min(max(c, 0), left))
            left -= taken[-1]
        for transposed in (False, True):
            out = torch.full((rows + 512, width), 7.0, device=DEV, dtype=torch.bfloat16)
            _keep, ws, size = fp8_workspace(DX if transposed else FWD, x, rows, rows, width, width, 4)
            ms = sizes(counts, index)
            args = (ms.data_ptr(), _lib.itype_code(index), out.data_ptr(), rows, width, width, 4, _lib.BF16, _lib.BF16, ws, size,
                    _lib.stream())
            source = () if transposed else (rows, None, 1)
            call = _lib.lib().mfl_gemm_dx_fp8 if transposed else _lib.lib().mfl_gemm_fwd_fp8
            assert call(x.data_ptr(), *source, fp8_weight(w, s), *args) == 0
            assert_within(out[:rows], *product(q, slack, dense(w, s), taken, transposed, True))
            assert (out[rows:] == 7.0).all()


@pytest.mark.parametrize("rows,n", [(6, 128), (300, 128), (300, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_up_to_the_largest_magnitude_that_is_promised(rows, n, dtype):
    """2^111 against the largest weights, in both directions; every sum is a power of two times 7, which fp32 and bf16 hold."""
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import grouped_gemm_forward_fp8, grouped_gemm_forward_transposed_fp8

    w = torch.full((2, n, 256), 448.0, device=DEV).to(FP8)
    s = torch.full((2, 1, 2), 2.0 ** -60, device=DEV)
    for out, red in ((grouped_gemm_forward_fp8(torch.full((rows, 256), 2.0 ** 111, device=DEV, dtype=dtype), w, s, sizes([rows - 1, 1])), 256),
                     (grouped_gemm_forward_transposed_fp8(torch.full((rows, n), 2.0 ** 111, device=DEV, dtype=dtype), w, s,
                                                          sizes([rows - 1, 1])), n)):
        assert (out == red * 448.0 * 2.0 ** 51).all()


# ---- the decode kernel's own quantiser ------------------------------------------------------------------------------------

def blocks_around_their_largest(dtype):
    """Rows of 128 (a block each): a largest value at and next to the borders of the scale, and below it values of every exponent
    that the grid tells apart, down to what becomes zero, among them the middles between two neighbours."""
    g = torch.Generator().manual_seed(106)
    bits = {torch.bfloat16: 7, torch.float16: 10, torch.float32: 23}[dtype]
    down = torch.arange(0, 22).repeat_interleave(64)
    mantissa = torch.cat([torch.arange(32) / 32.0, torch.randint(0, 2 ** bits, (32,), generator=g) / 2.0 ** bits]).repeat(22)
    below = (1 + mantissa.double()) * torch.exp2(-down.double() - 1)
    below = torch.cat([below, -below])
    blocks = []
    for top in (1.0, 1.5, 1.75, 1.75 + 2.0 ** -bits, 2.0 - 2.0 ** -bits):
        for lo in range(0, below.numel(), 127):
            v = below[lo:lo + 127]
            blocks.append(torch.cat([torch.tensor([top], dtype=torch.float64), v, torch.zeros(127 - v.numel())])[
                torch.randperm(128, generator=g)])
    x = torch.stack(blocks)
    # (fp16: the least values are subnormal, others next to the largest)
    low, high = (-3, 13) if dtype == torch.float16 else (-100, 100)
    x = x * torch.exp2(torch.randint(low, high, (x.shape[0], 1), generator=g).double())
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_decode_kernel_quantises_like_the_quantiser(dtype):
    """Weights of ones on the diagonal: what comes out are the quantised rows, bit for bit (every sum has one term)."""
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import grouped_gemm_forward_fp8
    from qwen3_moe_fused.quantize.fp8 import dequantize_fp8_rows, quantize_fp8_rows

    k, experts = 1024, 16
    values = [blocks_around_their_largest(dtype).reshape(-1)]
    if dtype != torch.float32:  # every finite value of the type, next to its neighbours and in any order
        every = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype)
        every = every[every.isfinite()]
        # (16-bit outputs: quantised values past the type's largest would be infinite)
        every = every[every.abs() <= torch.finfo(dtype).max / 2]
        values += [every, every[torch.randperm(every.numel(), generator=torch.Generator().manual_seed(107))]]
    else:
        g = torch.Generator().manual_seed(108)
        bits = torch.randint(-2 ** 31, 2 ** 31, (2 ** 16,), generator=g).to(torch.int32).view(torch.float32)
        values.append(bits[bits.abs() <= 2.0 ** 120])
    out = torch.float16 if dtype == torch.float16 else torch.bfloat16
    w = torch.eye(k, device=DEV).to(FP8).expand(experts, k, k).contiguous()
    s = torch.ones((experts, k // 128, k // 128), device=DEV)
    for v in values:
        rows = -(-v.numel() // k)
        x = torch.zeros(rows * k, dtype=dtype)
        x[:v.numel()] = v
        x = x.view(rows, k).to(DEV)
        for part in x.split(8 * experts):
            part = part.contiguous()
            counts = [min(8, max(0, part.shape[0] - 8 * e)) for e in range(experts)]
            y = grouped_gemm_forward_fp8(part, w, s, sizes(counts), out)
            expect = dequantize_fp8_rows(*quantize_fp8_rows(part), out)
            assert expect.isfinite().all()
            assert torch.equal(y, expect)


# ---- whole tiles, several of them a workgroup -----------------------------------------------------------------------------

# A workgroup that goes on to another tile waits for that tile's copies behind the stores of whole row blocks, which it counts
# only where the columns are whole tiles: 128 x 128 tiles (564 and 768 for 512 workgroups) and 256 x 256 ones (1152 for 256), in
# reductions of whole blocks.

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,experts,n,k", [(6000, 16, 2048, 512), (6000, 16, 512, 2048), (36000, 6, 2048, 256), (36000, 6, 256, 2048)])
def test_products_in_whole_tiles_one_behind_the_other(rows, experts, n, k, dtype):
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import grouped_gemm_forward_fp8, grouped_gemm_forward_transposed_fp8

    counts = counts_of(rows, experts, "spread", 109)
    w, s = make_weight(experts, n, k, 110)
    full = dense(w, s)
    x, dy = make_rows(rows, k, dtype, 111, spread=False), make_rows(rows, n, dtype, 112, spread=False)
    for out, given, transposed in ((grouped_gemm_forward_fp8(x, w, s, sizes(counts)), x, False),
                                   (grouped_gemm_forward_transposed_fp8(dy, w, s, sizes(counts)), dy, True)):
        q, _, slack = quantize(given.double())
        assert_within(out, *product(q, slack, full, counts, transposed, cut_in(out)), "input gradient" if transposed else "forward")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,k,experts,hidden,inter", [(1500, 4, 16, 512, 1024), (1500, 4, 16, 256, 1024), (9000, 4, 6, 256, 2048),
                                                           (9000, 4, 6, 2048, 256)])
def test_gated_unit_and_mlp_in_whole_tiles_one_behind_the_other(tokens, k, experts, hidden, inter, dtype):
    """The quantised unit's kernel with and without the two products, 128 x (128 + 128) tiles, 384 and more for 256 workgroups."""
    from qwen3_moe_fused.grouped_gemm.fused import grouped_glu_backward_fp8, grouped_glu_forward_fp8, grouped_mlp_forward_fp8

    m_sizes, sort_idx, _, counts = routed(tokens, k, experts, 113)
    x, w = make_rows(tokens, hidden, dtype, 114, spread=False), mlp_weights(experts, hidden, inter, 115)
    re, de, rg, dg = gated_reference(x, ((w[0], w[1]), (w[2], w[3])), sort_idx, k, counts)
    rh, dh = gated(re, de, rg, dg)
    h, e, g = grouped_glu_forward_fp8(x, *w[:4], m_sizes, sort_idx, k, return_products=True)
    y, e2, g2 = grouped_mlp_forward_fp8(x, *w, m_sizes, sort_idx, k, return_products=True)
    for what, at, out in (("gate projection", (re, de), e), ("up projection", (rg, dg), g), ("gated unit", (rh, dh), h),
                          ("gate projection", (re, de), e2), ("up projection", (rg, dg), g2)):
        assert_within(out, *at, what)
    q, _, slack = quantize(rh, dh)
    assert_within(y, *product(q, slack, dense(w[4], w[5]), counts, cut=cut_in(y)), "expert MLP")
    assert torch.equal(y, grouped_mlp_forward_fp8(x, *w, m_sizes, sort_idx, k))
    del re, de, rg, dg, rh, dh, q, slack
    dh = make_rows(tokens * k, inter, dtype, 116, spread=False)
    dx = grouped_glu_backward_fp8(dh, e, g, *w[:4], m_sizes)
    a, ea, b, eb = gated_backward(dh.double(), e.double(), g.double())
    total, bound = 0, 0
    for v, err, (wq, s) in ((a, ea, w[0:2]), (b, eb, w[2:4])):
        qv, _, slack = quantize(v, err)
        t, bd = product(qv, slack, dense(wq, s), counts, True, cut_in(dx))
        total, bound = total + t, bound + 2 * bd
    assert_within(dx, total, bound, "gradient of the rows")
