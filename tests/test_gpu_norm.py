"""The residual's addition with the norm behind it, forward, backward and to 8-bit rows, against 64 bits."""
import pytest
import torch

import layer_reference as ref
from qwen3_moe_fused import _lib
from qwen3_moe_fused.kernels.norm import add_rms_norm, add_rms_norm_backward, add_rms_norm_fp8
from qwen3_moe_fused.quantize.fp8 import dequantize_fp8_rows, empty_fp8_rows, quantize_fp8_rows

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
EPS = 1e-6
# widths around every change of a row's threads, and such as no 16-byte access fits
WIDTHS = (1, 7, 8, 129, 512, 513, 1001, 1024, 1032, 2048, 2049, 4096, 4100, 8192, 8200, 16384, 20000, 32768)


def _inputs(rows, width, dtype, seed=0, residual=True, weight_dtype=None, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, width), generator=g) * std).to(dtype)
    r = (torch.randn((rows, width), generator=g) * 0.5 * std).to(dtype) if residual else None
    w = (1.0 + 0.1 * torch.randn(width, generator=g)).to(weight_dtype or dtype)
    return x, r, w, g


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def _check(y, s, x, r, w, dtype, eps=EPS):
    want_s = ref.stream(x, r)
    assert torch.equal(s.cpu().double(), want_s)
    want, _, _ = ref.norm(want_s, w, eps)
    assert ((y.cpu().double() - want).abs() <= ref.half_step(want, dtype)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("rows", (1, 5))
def test_forward(dtype, width, rows):
    for residual in (True, False):
        x, r, w, _ = _inputs(rows, width, dtype, width, residual)
        y, s = add_rms_norm(*_cuda(x, r, w), EPS)
        _check(y, s, x, r, w, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_leading_dimensions_other_weights_and_no_rows(dtype):
    x, r, w, _ = _inputs(12, 96, dtype, weight_dtype=torch.float32)
    y, s = add_rms_norm(x.view(3, 4, 96).cuda(), r.view(3, 4, 96).cuda(), w.cuda(), 1e-5)
    assert y.shape == s.shape == (3, 4, 96)
    _check(y.view(12, 96), s.view(12, 96), x, r, w, dtype, 1e-5)
    empty = torch.empty((0, 96), device="cuda", dtype=dtype)
    y, s = add_rms_norm(empty, empty.clone(), w.cuda())
    assert y.shape == s.shape == (0, 96)
    values, scales, s = add_rms_norm_fp8(empty, None, w.cuda())
    assert values.shape == (0, 96) and scales.shape == (0, 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off", (1, 3))
def test_rows_off_the_16_byte_grid(dtype, off):
    x, r, w, _ = _inputs(6, 264, dtype)

    def moved(t):
        room = torch.empty(t.numel() + off, device="cuda", dtype=t.dtype)
        room[off:] = t.flatten().cuda()
        return room[off:].view(t.shape)

    y, s = add_rms_norm(moved(x), moved(r), moved(w), EPS)
    _check(y, s, x, r, w, dtype)
    dy = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(dtype)
    a = add_rms_norm_backward(moved(dy), moved(dy), moved(s.cpu()), moved(w), EPS)
    b = add_rms_norm_backward(dy.cuda(), dy.cuda(), s, w.cuda(), EPS)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("std", (1e30, 1e-30))
def test_magnitudes_whose_squares_32_bits_do_not_hold(dtype, std):
    x, r, w, g = _inputs(4, 300, dtype, std=std)
    eps = 0.0 if std < 1 else EPS
    y, s = add_rms_norm(*_cuda(x, r, w), eps)
    _check(y, s, x, r, w, dtype, eps)
    if std > 1:  # (rows of 1e-30 without eps have gradients of 1e30)
        dy = torch.randn(x.shape, generator=g).to(dtype)
        dx, dw = add_rms_norm_backward(dy.cuda(), None, s, w.cuda(), eps)
        want = ref.norm_gradients(dy, None, s.cpu().double(), w, eps)
        bounds = ref.norm_gradient_bounds(dy, None, s.cpu().double(), w, eps, dtype, dtype)
        for a, b, c in zip((dx, dw), want, bounds):
            assert ((a.cpu().double() - b).abs() <= c).all()


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
def test_gradients_whose_row_sums_32_bits_do_not_hold(dtype):
    s, _, w, g = _inputs(4, 2048, dtype, residual=False, std=1e36)
    dy = (torch.randn(s.shape, generator=g).abs() * s.sign() * 256.0).to(dtype)  # 2048 terms of one sign, 2e38 each
    dx, dw = add_rms_norm_backward(dy.cuda(), None, s.cuda(), w.cuda(), EPS)
    want = ref.norm_gradients(dy, None, s.double(), w, EPS)
    bounds = ref.norm_gradient_bounds(dy, None, s.double(), w, EPS, dtype, dtype)
    for a, b, c in zip((dx, dw), want, bounds):
        assert ((a.cpu().double() - b).abs() <= c).all()


def test_a_row_without_a_finite_length_leaves_the_others_alone():
    x, r, w, _ = _inputs(9, 700, torch.bfloat16)
    x[2, 5], x[4, 699], x[6] = float("nan"), float("inf"), 0.0
    r[6] = 0.0
    y, s = add_rms_norm(*_cuda(x, r, w), EPS)
    keep = [0, 1, 3, 5, 6, 7, 8]
    _check(y[keep], s[keep], x[keep], r[keep], w, torch.bfloat16)
    assert y[2].isnan().all() and (y[6] == 0).all()
    # an infinite element: 1 / length is zero, and the element itself no number
    assert y[4, 699].isnan() and (y[4, :699] == 0).all()


# ---- 8-bit rows

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", (1, 17, 128, 130, 1001, 2048, 2050, 4096, 8200, 20000))
def test_quantised_rows_are_those_of_the_normed_rows(dtype, width):
    x, r, w, _ = _inputs(5, width, dtype, width)
    if width > 1000:
        x[1, 3], x[2, 500], x[3, 128:256] = float("nan"), float("inf"), 0.0
        r[3, 128:256] = 0.0
    x, r, w = _cuda(x, r, w)
    values, scales, s, y = add_rms_norm_fp8(x, r, w, EPS, return_normed=True)
    want_y, want_s = add_rms_norm(x, r, w, EPS)
    assert torch.equal(y.view(torch.uint8), want_y.view(torch.uint8)) and torch.equal(s.view(torch.uint8), want_s.view(torch.uint8))
    want, want_scales = quantize_fp8_rows(y)
    assert values.stride() == want.stride() and scales.stride() == want_scales.stride()
    assert torch.equal(values.view(torch.uint8), want.view(torch.uint8))
    assert torch.equal(scales.view(torch.uint8), want_scales.view(torch.uint8))
    padded = torch.as_strided(values.view(torch.uint8), (5, values.stride(0)), (values.stride(0), 1))[:, width:]
    assert (padded == 0).all()  # zeros behind the last column
    other, other_scales, s = add_rms_norm_fp8(x, None, w, EPS)
    assert s is x and torch.equal(dequantize_fp8_rows(other, other_scales, torch.float32).nan_to_num(),
                                  dequantize_fp8_rows(*quantize_fp8_rows(add_rms_norm(x, None, w, EPS)[0]), torch.float32).nan_to_num())


# ---- backward

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_backward(dtype, width):
    rows = 7 if width > 2100 else 37
    x, r, w, g = _inputs(rows, width, dtype, width)
    dy, ds = (torch.randn(x.shape, generator=g).to(dtype) for _ in range(2))
    leaves = [t.cuda().requires_grad_() for t in (x, r, w)]
    y, s = add_rms_norm(*leaves, EPS)
    got = torch.autograd.grad((y, s), leaves, (dy.cuda(), ds.cuda()))
    s64 = ref.stream(x, r)
    dx, dw = ref.norm_gradients(dy, ds, s64, w, EPS)
    bound, bound_w = ref.norm_gradient_bounds(dy, ds, s64, w, EPS, dtype, dtype)
    assert torch.equal(got[0], got[1])
    assert ((got[0].cpu().double() - dx).abs() <= bound).all()
    assert ((got[2].cpu().double() - dw).abs() <= bound_w).all()


@pytest.mark.parametrize("rows", (1, 2, 3000, 20011))
def test_backward_over_many_rows_is_the_same_every_time(rows):
    x, _, w, g = _inputs(rows, 136, torch.bfloat16, residual=False, weight_dtype=torch.float32)
    dy = torch.randn(x.shape, generator=g).to(torch.bfloat16)
    leaves = [x.cuda().requires_grad_(), w.cuda().requires_grad_()]
    y, s = add_rms_norm(leaves[0], None, leaves[1], EPS)
    assert s is leaves[0]
    got = torch.autograd.grad(y, leaves, dy.cuda(), retain_graph=True)
    dx, dw = ref.norm_gradients(dy, None, x.double(), w, EPS)
    bound, bound_w = ref.norm_gradient_bounds(dy, None, x.double(), w, EPS, torch.bfloat16, torch.float32)
    assert ((got[0].cpu().double() - dx).abs() <= bound).all() and ((got[1].cpu().double() - dw).abs() <= bound_w).all()
    again = torch.autograd.grad(y, leaves, dy.cuda())
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_gradient_against_differences():
    """Central differences of the definition in 64 bits: off by about h^2 times the third derivative, a few 1e-9 here."""
    x, r, w, g = _inputs(2, 24, torch.float32)
    dy, ds = torch.randn(x.shape, generator=g), torch.randn(x.shape, generator=g)
    leaves = [t.cuda().requires_grad_() for t in (x, r, w)]
    got = torch.autograd.grad(add_rms_norm(*leaves, EPS), leaves, (dy.cuda(), ds.cuda()))

    def loss(x, r, w):
        s = x + r
        return ((ref.norm(s, w, EPS)[0] * dy.double()).sum() + (s * ds.double()).sum()).item()

    h = 1e-5
    for which, grad in enumerate(got):
        flat = grad.cpu().double().flatten()
        for i in range(0, flat.numel(), 5):
            sides = []
            for sign in (1, -1):
                args = [t.double().clone() for t in (x, r, w)]
                args[which].view(-1)[i] += sign * h
                sides.append(loss(*args))
            slope = (sides[0] - sides[1]) / (2 * h)
            assert abs(flat[i].item() - slope) <= 2e-5 * (1 + abs(slope))


@pytest.mark.parametrize("needs", [(True, False, False), (False, True, False), (False, False, True), (True, False, True)])
def test_gradients_that_are_asked_for(needs):
    x, r, w, g = _inputs(11, 72, torch.float32)
    dy, ds = (torch.randn(x.shape, generator=g).cuda() for _ in range(2))
    everything = [t.cuda().requires_grad_() for t in (x, r, w)]
    want = torch.autograd.grad(add_rms_norm(*everything, EPS), everything, (dy, ds))
    some = [t.cuda().requires_grad_(n) for t, n in zip((x, r, w), needs)]
    got = torch.autograd.grad(add_rms_norm(*some, EPS), [t for t, n in zip(some, needs) if n], (dy, ds))
    assert all(torch.equal(a, b) for a, b in zip(got, [t for t, n in zip(want, needs) if n]))


def test_one_result_used_alone_and_shared_inputs():
    x, r, w, g = _inputs(5, 40, torch.float32)
    dy = torch.randn(x.shape, generator=g)
    leaves = [t.cuda().requires_grad_() for t in (x, r, w)]
    _, s = add_rms_norm(*leaves, EPS)
    got = torch.autograd.grad(s, leaves, dy.cuda(), allow_unused=True)  # the addition's gradient
    assert torch.equal(got[0].cpu(), dy) and torch.equal(got[1].cpu(), dy) and (got[2] is None or (got[2] == 0).all())
    y, _ = add_rms_norm(*leaves, EPS)
    got = torch.autograd.grad(y, leaves, dy.cuda())
    dx, _ = ref.norm_gradients(dy, None, ref.stream(x, r), w, EPS)
    bound, _ = ref.norm_gradient_bounds(dy, None, ref.stream(x, r), w, EPS, torch.float32, torch.float32)
    assert ((got[0].cpu().double() - dx).abs() <= bound).all()
    # the same tensor twice: both of its gradients
    one = x.cuda().requires_grad_()
    y, _ = add_rms_norm(one, one, w.cuda(), EPS)
    (grad,) = torch.autograd.grad(y, one, dy.cuda())
    dx, _ = ref.norm_gradients(dy, None, ref.stream(x, x), w, EPS)
    bound, _ = ref.norm_gradient_bounds(dy, None, ref.stream(x, x), w, EPS, torch.float32, torch.float32)
    assert ((grad.cpu().double() - 2 * dx).abs() <= 2 * bound + 2.0 ** -23 * dx.abs()).all()


def test_backward_through_the_quantised_form():
    x, r, w, g = _inputs(6, 200, torch.bfloat16)
    dy, ds = (torch.randn(x.shape, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    leaves = [t.cuda().requires_grad_() for t in (x, r, w)]
    want = torch.autograd.grad(add_rms_norm(*leaves, EPS), leaves, (dy, ds))
    values, scales, s, y = add_rms_norm_fp8(*leaves, EPS, return_normed=True)
    assert not values.requires_grad and not scales.requires_grad
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad((y, s), leaves, (dy, ds)), want))
    values, scales, s = add_rms_norm_fp8(*leaves, EPS)
    got = torch.autograd.grad(s, leaves[:2], ds)
    assert torch.equal(got[0], ds) and torch.equal(got[1], ds)


def test_second_derivatives_and_tangents_are_refused():
    x, r, w, _ = _inputs(3, 16, torch.float32)
    leaves = [t.cuda().requires_grad_() for t in (x, r, w)]
    y, _ = add_rms_norm(*leaves, EPS)
    (grad,) = torch.autograd.grad(y.sum(), leaves[:1], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.sum(), leaves[:1])
    from torch.autograd import forward_ad

    with forward_ad.dual_level(), pytest.raises(RuntimeError):
        add_rms_norm(forward_ad.make_dual(x.cuda(), r.cuda()), None, w.cuda(), EPS)


# ---- streams, graphs, in place

def test_captured_and_replayed_with_eager_passes_between():
    x, r, w, g = _inputs(33, 2048, torch.bfloat16)
    dy, ds = (torch.randn(x.shape, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    leaves = [t.cuda().requires_grad_() for t in (x, r, w)]

    def step():
        out = add_rms_norm(*leaves, EPS)
        grads = torch.autograd.grad(out, leaves, (dy, ds))
        return (*(t.detach() for t in out), *grads)  # (nothing of the graph lives on)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16))
        graph.replay()
        got = [t.clone() for t in captured]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_on_another_stream_than_the_default():
    x, r, w, _ = _inputs(64, 2048, torch.bfloat16)
    x, r, w = _cuda(x, r, w)
    want = add_rms_norm(x, r, w, EPS)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = add_rms_norm(x, r, w, EPS)
    b = add_rms_norm(x, r, w, EPS)
    torch.cuda.synchronize()
    for got in (a, b):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_results_in_the_place_of_operands():
    x, r, w, g = _inputs(19, 1001, torch.float16)
    xc, rc, wc = _cuda(x, r, w)
    y, s = add_rms_norm(xc, rc, wc, EPS)
    dy, ds = (torch.randn(x.shape, generator=g).to(torch.float16).cuda() for _ in range(2))
    dx, _ = add_rms_norm_backward(dy, ds, s, wc, EPS)
    a, b, lib = xc.clone(), rc.clone(), _lib.lib()
    _lib.check(lib.mfl_add_rms_norm(a.data_ptr(), b.data_ptr(), wc.data_ptr(), a.data_ptr(), b.data_ptr(), 19, 1001, EPS, _lib.F16,
                                    _lib.F16, _lib.stream()), "norm")
    assert torch.equal(a, y) and torch.equal(b, s)
    for place in range(3):
        ops = [dy.clone(), ds.clone(), s.clone()]
        _lib.check(lib.mfl_add_rms_norm_bwd(*(t.data_ptr() for t in ops), wc.data_ptr(), ops[place].data_ptr(), None, 19, 1001, EPS,
                                            _lib.F16, _lib.F16, None, 0, _lib.stream()), "norm backward")
        assert torch.equal(ops[place], dx)


def test_more_elements_than_32_bits_count():
    rows, width = (1 << 31) // 2048 + 3, 2048
    x = torch.zeros((rows, width), device="cuda", dtype=torch.bfloat16)
    tail, _, w, _ = _inputs(5, width, torch.bfloat16, residual=False)
    x[-5:] = tail.cuda()
    wc = w.cuda()
    y, _ = add_rms_norm(x, None, wc, EPS)
    _check(y[-5:], x[-5:], tail, None, w, torch.bfloat16)
    del y
    values, scales, _ = add_rms_norm_fp8(x, None, wc, EPS)
    want, want_scales = quantize_fp8_rows(add_rms_norm(tail.cuda(), None, wc, EPS)[0])
    assert torch.equal(values[-5:].view(torch.uint8), want.view(torch.uint8))
    assert torch.equal(scales[-5:].view(torch.uint8), want_scales.view(torch.uint8))
    dy = torch.zeros_like(x)
    dy[-5:] = tail.flip(0).cuda()
    dx, _ = add_rms_norm_backward(dy, None, x, wc, EPS, need_dw=False)
    want, _ = ref.norm_gradients(tail.flip(0), None, tail.double(), w, EPS)
    bound, _ = ref.norm_gradient_bounds(tail.flip(0), None, tail.double(), w, EPS, torch.bfloat16, torch.bfloat16)
    assert ((dx[-5:].cpu().double() - want).abs() <= bound).all()


def test_weight_gradient_of_no_rows():
    w, dw = torch.ones(72, device="cuda"), torch.full((72,), 5.0, device="cuda")
    rows = torch.empty((1, 72), device="cuda")
    rc = _lib.lib().mfl_add_rms_norm_bwd(rows.data_ptr(), None, rows.data_ptr(), w.data_ptr(), rows.data_ptr(), dw.data_ptr(), 0, 72, EPS,
                                         _lib.dtype_code(w.dtype), _lib.dtype_code(w.dtype), None, 0, _lib.stream())
    _lib.check(rc, "mfl_add_rms_norm_bwd")
    assert not dw.any()


@pytest.mark.parametrize("width", (2048, 16384, 32768, 20001))
@pytest.mark.parametrize("onto", ("dy", "ds", "s"))
def test_backward_onto_an_operand(width, onto):
    dtype = torch.bfloat16
    s, ds, w, g = _inputs(37, width, dtype, width)
    dy = torch.randn((37, width), generator=g).to(dtype)
    s, ds, w, dy = _cuda(s, ds, w, dy)
    want_dx, want_dw = add_rms_norm_backward(dy, ds, s, w, EPS)
    lib, dw = _lib.lib(), torch.empty_like(w)
    size = lib.mfl_add_rms_norm_bwd_workspace(37, width)
    ws = torch.empty(size, device="cuda", dtype=torch.uint8)
    dx = {"dy": dy, "ds": ds, "s": s}[onto]
    rc = lib.mfl_add_rms_norm_bwd(dy.data_ptr(), ds.data_ptr(), s.data_ptr(), w.data_ptr(), dx.data_ptr(), dw.data_ptr(), 37, width, EPS,
                                  _lib.dtype_code(dtype), _lib.dtype_code(dtype), ws.data_ptr(), size, _lib.stream())
    _lib.check(rc, "mfl_add_rms_norm_bwd")
    assert torch.equal(dx, want_dx) and torch.equal(dw, want_dw)


@pytest.mark.parametrize("width", (96, 2048, 16384, 32768))
def test_forward_onto_its_operands(width):
    dtype = torch.bfloat16
    x, r, w, _ = _inputs(21, width, dtype, width)
    x, r, w = _cuda(x, r, w)
    want, want_s = add_rms_norm(x, r, w, EPS)
    rc = _lib.lib().mfl_add_rms_norm(x.data_ptr(), r.data_ptr(), w.data_ptr(), x.data_ptr(), r.data_ptr(), 21, width, EPS,
                                     _lib.dtype_code(dtype), _lib.dtype_code(dtype), _lib.stream())
    _lib.check(rc, "mfl_add_rms_norm")
    assert torch.equal(x, want) and torch.equal(r, want_s)


@pytest.mark.parametrize("width", (1, 13, 200, 505, 1001))
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_single_row_is_written_out_from_where_it_stands(dtype, width):
    x, _, w, _ = _inputs(1, width, dtype, width, residual=False)
    values, scales, _ = add_rms_norm_fp8(x.cuda(), None, w.cuda())
    want = dequantize_fp8_rows(values, scales, dtype)
    tight = torch.zeros(7 + width, device="cuda", dtype=torch.uint8)
    tight[7:] = values.view(torch.uint8)[0]
    assert torch.equal(dequantize_fp8_rows(tight[7:].view(1, width).view(values.dtype), scales, dtype), want)


@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
@pytest.mark.parametrize("width", (512, 1024, 4096, 8192, 300, 1001, 2050, 9001, 20001))
@pytest.mark.parametrize("form", ("plain", "eight"))
def test_forward_onto_its_operands_in_every_width(dtype, width, form):
    x, r, w, _ = _inputs(23, width, dtype, width)
    x, r, w = _cuda(x, r, w)
    want, want_s = add_rms_norm(x, r, w, EPS)
    code, lib = _lib.dtype_code(dtype), _lib.lib()
    q, scale = quantize_fp8_rows(want)
    got_q, got_scale = empty_fp8_rows(x)

    def run(x, r, y, s):
        if form == "plain":
            rc = lib.mfl_add_rms_norm(x.data_ptr(), r.data_ptr(), w.data_ptr(), y.data_ptr(), s.data_ptr(), 23, width, EPS, code, code,
                                      _lib.stream())
        else:
            rc = lib.mfl_add_rms_norm_fp8(x.data_ptr(), r.data_ptr(), w.data_ptr(), got_q.data_ptr(), got_scale.data_ptr(), y.data_ptr(),
                                          s.data_ptr(), 23, width, EPS, code, code, _lib.stream())
            assert torch.equal(got_q.view(torch.uint8), q.view(torch.uint8))
            assert torch.equal(got_scale.view(torch.uint8), scale.view(torch.uint8))
        _lib.check(rc, "norm")
        assert torch.equal(y, want) and torch.equal(s, want_s)

    a, b = x.clone(), r.clone()
    run(a, b, a, b)  # y onto x, s onto the residual
    a, b = x.clone(), r.clone()
    run(a, b, torch.empty_like(x), a)  # s onto x


@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
@pytest.mark.parametrize("width", (512, 1024, 4096, 8192, 300, 1001, 2050, 9001, 20001, 32768))
@pytest.mark.parametrize("onto", ("dy", "ds", "s"))
def test_backward_onto_an_operand_in_every_width(dtype, width, onto):
    s, ds, w, g = _inputs(1500 if width <= 4096 else 700, width, dtype, width)  # (several rows a group)
    dy = torch.randn(s.shape, generator=g).to(dtype)
    s, ds, w, dy = _cuda(s, ds, w, dy)
    want, want_dw = add_rms_norm_backward(dy, ds, s, w, EPS)
    ops = {"dy": dy, "ds": ds, "s": s}
    lib, dw, code, rows = _lib.lib(), torch.empty_like(w), _lib.dtype_code(dtype), s.shape[0]
    size = lib.mfl_add_rms_norm_bwd_workspace(rows, width)
    ws = torch.empty(size, device="cuda", dtype=torch.uint8)
    rc = lib.mfl_add_rms_norm_bwd(dy.data_ptr(), ds.data_ptr(), s.data_ptr(), w.data_ptr(), ops[onto].data_ptr(), dw.data_ptr(), rows, width,
                                  EPS, code, code, ws.data_ptr(), size, _lib.stream())
    _lib.check(rc, "norm backward")
    assert torch.equal(ops[onto], want) and torch.equal(dw, want_dw)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("width", (40, 300, 2048, 12000, 20001))
def test_rows_whose_inverse_length_32_bits_do_not_hold(dtype, width):
    """Rows below 2^-128 without eps, one of ordinary values among them: both sides of the pass are the definition's."""
    g = torch.Generator().manual_seed(width)
    s = (torch.randn((5, width), generator=g) * 2.0 ** -131).to(dtype)
    s[3] = torch.randn(width, generator=g).to(dtype)
    w = (1.0 + 0.1 * torch.randn(width, generator=g)).to(dtype)
    dy = (torch.randn(s.shape, generator=g) * 2.0 ** -12).to(dtype)
    y, same = add_rms_norm(s.cuda(), None, w.cuda(), 0.0)
    _check(y, same, s, None, w, dtype, 0.0)
    dx, dw = add_rms_norm_backward(dy.cuda(), None, s.cuda(), w.cuda(), 0.0)
    want = ref.norm_gradients(dy, None, s.double(), w, 0.0)
    bounds = ref.norm_gradient_bounds(dy, None, s.double(), w, 0.0, dtype, dtype)
    for a, b, c in zip((dx, dw), want, bounds):
        assert ((a.cpu().double() - b).abs() <= c).all()
