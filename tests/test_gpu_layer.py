"""The whole expert layer for a few tokens against 64 bits, and the norm, the layer and the expert MLP as they are used together."""
from types import SimpleNamespace

import pytest
import torch

import layer_reference as ref
from qwen3_moe_fused import _lib
from qwen3_moe_fused.fused_mlp import moe_fused_layer, moe_fused_layer_fp8, moe_fused_mlp_fp8
from qwen3_moe_fused.kernels.norm import add_rms_norm, add_rms_norm_fp8
from qwen3_moe_fused.kernels.routing import route_and_sort
from qwen3_moe_fused.quantize.fp8 import quantize_fp8_blocks, quantize_fp8_rows

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6


class Case:
    def __init__(self, tokens, experts, k, hidden, inter, dtype, eight=False, norm=False, residual=False, renorm=True, seed=0, std=1.0):
        g = torch.Generator().manual_seed(seed)
        self.k, self.renorm, self.dtype, self.eight = k, renorm, dtype, eight
        self.x = (torch.randn((tokens, hidden), generator=g) * std).to(dtype)
        self.residual = torch.randn((tokens, hidden), generator=g).to(dtype) if residual else None
        self.norm = (1.0 + 0.1 * torch.randn(hidden, generator=g)).to(dtype) if norm else None
        self.router = (torch.randn((experts, hidden), generator=g) * hidden ** -0.5).to(dtype)
        scale = (hidden ** -0.5, hidden ** -0.5, inter ** -0.5)
        shapes = ((experts, inter, hidden), (experts, inter, hidden), (experts, hidden, inter))
        self.weights = [(torch.randn(s, generator=g) * f).to(dtype) for s, f in zip(shapes, scale)]
        self.scales = None
        if eight:
            # (scales that are no powers of two, as checkpoints have them)
            pairs = [quantize_fp8_blocks(w.cuda()) for w in self.weights]
            self.weights = [q.cpu() for q, _ in pairs]
            self.scales = [(s * (0.75 + 0.5 * torch.rand(s.shape, generator=g).cuda())).cpu() for _, s in pairs]

    def call(self, device="cuda", **changed):
        def at(t):
            return None if t is None else t.to(device)

        args = {"residual": at(self.residual), "norm_weight": at(self.norm), "eps": EPS, **changed}
        if self.eight:
            pairs = [at(t) for pair in zip(self.weights, self.scales) for t in pair]
            return moe_fused_layer_fp8(at(self.x), at(self.router), *pairs, self.k, self.renorm, **args)
        return moe_fused_layer(at(self.x), at(self.router), *map(at, self.weights), self.k, self.renorm, **args)

    def rows(self):
        """(rows that the experts get, as rounded to the type; stream to be added or None), float64."""
        s = ref.stream(self.x, self.residual)
        if self.norm is None:
            return s, None
        return ref.norm(s, self.norm, EPS)[0].float().to(self.dtype).double(), s

    def check(self, out, logits):
        rows, s = self.rows()
        want = rows @ self.router.double().t()
        got = logits.cpu().double()
        known = want.isfinite()
        # a sum in 64 bits, rounded once; what a row of another last bit (one in 2^29) would change is not allowed for
        assert ((got - want)[known].abs() <= ref.half_step(want, self.dtype)[known]).all()
        assert (~got[~known].isfinite()).all()
        want, bound = ref.layer(rows, s, logits.cpu(), *self.weights, self.k, self.renorm, self.dtype, self.scales)
        out = out.cpu().double()
        assert torch.equal(out.isnan(), want.isnan())
        error = (out - want).nan_to_num().abs()
        assert (error <= bound).all(), f"off by {(error / bound.clamp_min(1e-300)).max():.3g} of the bound"


SIZES = [
    # tokens, experts, k, hidden, inter
    (1, 8, 2, 64, 128),
    (1, 128, 8, 256, 96),
    (2, 4, 4, 16, 16),
    (3, 60, 4, 300, 100),
    (4, 16, 1, 1024, 64),
    (5, 60, 4, 1001, 333),
    (7, 8, 8, 72, 40),
    (8, 9, 3, 33, 17),
    (13, 5, 2, 520, 200),
    (16, 128, 8, 192, 64),
    (16, 1, 1, 128, 256),
    (16, 3, 3, 40, 1032),
    (1, 2, 1, 1, 1),
    (9, 300, 6, 48, 24),
    (6, 1024, 64, 40, 24),
]


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_layer(size, dtype):
    for norm, residual, renorm in ((False, False, True), (True, True, False), (True, False, True)):
        case = Case(*size, dtype, norm=norm, residual=residual, renorm=renorm, seed=sum(size))
        case.check(*case.call())


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_layer_in_8_bits(size, dtype):
    for norm, residual, renorm in ((False, False, False), (True, True, True)):
        case = Case(*size, dtype, eight=True, norm=norm, residual=residual, renorm=renorm, seed=sum(size))
        case.check(*case.call())


# rows that fill a wave's share, that do not, that take several chunks, either way
WIDE = [
    (5, 6, 2, 1024, 768),
    (2, 4, 2, 1536, 96),
    (3, 4, 2, 2050, 50),
    (4, 3, 2, 2048, 1536),
    (2, 3, 1, 4096, 768),
    (1, 2, 2, 5003, 24),
    (16, 2, 2, 6144, 40),
    (9, 3, 2, 24, 5001),
]


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("eight", (False, True))
@pytest.mark.parametrize("size", WIDE, ids=str)
def test_wide_rows(size, dtype, eight):
    case = Case(*size, dtype, eight=eight, norm=True, residual=True, seed=sum(size))
    case.check(*case.call())


@pytest.mark.parametrize("eight", (False, True))
def test_benchmark_sizes(eight):
    case = Case(3, 32, 8, 2048, 768, BF16, eight=eight, norm=True, residual=True)
    case.check(*case.call())


# 8-bit layers whose workgroups take many items of gate and up: the loop in which nothing is asked.  Rows of either chunk length that fit
# its loads, that are whole loads, that are neither, and of two chunks.
MANY = [
    # tokens, experts, k, hidden, inter
    (13, 40, 8, 2048, 768),
    (16, 72, 8, 1536, 400),
    (13, 64, 8, 1100, 500),
    (16, 36, 8, 4096, 768),
    (16, 80, 8, 1024, 768),
    (16, 128, 8, 256, 768),
    (16, 128, 8, 250, 700),
]


@pytest.mark.parametrize("size", MANY, ids=str)
def test_many_items_a_workgroup_in_8_bits(size):
    tokens, experts, k, hidden, inter = size
    case = Case(*size, BF16, eight=True, norm=tokens == 13, residual=tokens == 13, seed=sum(size))
    out, logits = case.call()
    hit = len({e for picked in ref.choose(logits.cpu(), k, True) for e, _ in picked})
    items, ahead = hit * 2 * ((inter + 15) // 16), 8 if hidden <= 1024 else 4
    # (from the first item of a workgroup the loop takes another turn while 2 ahead - 1 more are there; two turns at least)
    assert items > (3 * ahead - 1) * torch.cuda.get_device_properties(0).multi_processor_count
    case.check(out, logits)


@pytest.mark.parametrize("dtype", (BF16, F16))
@pytest.mark.parametrize("eight", (False, True))
def test_all_tokens_choose_the_same_experts(dtype, eight):
    case = Case(16, 12, 2, 136, 72, dtype, eight=eight)
    case.x[:, 0] = 4.0
    case.router[:, 0] = 0.0
    case.router[3, 0], case.router[7, 0] = 4.0, 3.0
    out, logits = case.call()
    assert all({e for e, _ in picked} == {3, 7} for picked in ref.choose(logits.cpu(), 2, True))
    case.check(out, logits)


def test_equal_logits_go_to_the_lower_expert():
    case = Case(5, 200, 7, 64, 32, BF16)
    case.router[:] = case.router[0]  # all equal
    out, logits = case.call()
    assert (logits == logits[:, :1]).all()
    case.check(out, logits)
    case.router[150:] = -case.router[0]  # two values, and zeros of both signs
    case.x[4] = 0.0
    case.x[4, ::2] = -0.0
    case.check(*case.call())


@pytest.mark.parametrize("eight", (False, True))
@pytest.mark.parametrize("norm", (False, True))
def test_a_token_that_is_no_number_leaves_the_others_alone(eight, norm):
    case = Case(9, 16, 3, 144, 80, BF16, eight=eight, norm=norm, residual=norm)
    want, want_logits = case.call()
    case.x[2, 7], case.x[5, 3], case.x[6, 140] = float("nan"), float("inf"), -float("inf")
    out, logits = case.call()
    keep = [0, 1, 3, 4, 7, 8]
    assert out[[2, 5, 6]].isnan().all()
    assert torch.equal(logits[keep], want_logits[keep])
    case.check(out, logits)


def test_infinite_and_missing_logits():
    case = Case(4, 6, 2, 32, 16, F32)
    case.router[1] = 0.0
    case.router[1, 0] = float("inf")
    case.router[4] = 0.0
    case.router[4, 1] = -float("inf")
    case.x[:, 1] = 1.0  # expert 4 is out of the question for every token
    case.x[:, 0] = torch.tensor([1.0, -1.0, -2.0, 0.0])  # expert 1: infinite, out, out, no number
    out, logits = case.call()
    assert out[[0, 3]].isnan().all() and out[[1, 2]].isfinite().all()
    case.check(out, logits)


def test_all_but_one_expert_out_of_the_question():
    case = Case(2, 4, 3, 16, 16, F32)
    case.x[:, 0] = 1.0
    case.router[:, 0] = torch.tensor([-float("inf"), -float("inf"), 0.0, -float("inf")])
    case.check(*case.call())


def test_no_tokens():
    case = Case(1, 8, 2, 64, 128, BF16)
    case.x = case.x[:0]
    out, logits = case.call()
    assert out.shape == (0, 64) and logits.shape == (0, 8)


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
def test_operands_off_the_16_byte_grid(dtype):
    case = Case(5, 8, 3, 128, 64, dtype, norm=True, residual=True)
    want = case.call()

    def moved(t):
        room = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)
        room[1:] = t.flatten().cuda()
        return room[1:].view(t.shape)

    case.x, case.residual, case.norm, case.router = map(moved, (case.x, case.residual, case.norm, case.router))
    case.weights = [moved(w) for w in case.weights]
    out, logits = case.call()
    assert torch.equal(out, want[0]) and torch.equal(logits, want[1])


def test_wide_values_of_the_gated_unit_in_fp16():
    """Products past 65504, which the type does not hold, and tiny ones: what the definition has, if the output fits."""
    case = Case(4, 4, 2, 64, 48, F16)
    case.weights[0] = case.weights[0] * 300
    case.weights[1] = case.weights[1] * 300
    case.weights[2] = case.weights[2] * 2.0 ** -8
    out, logits = case.call()
    assert out.isfinite().all()
    case.check(out, logits)


def _gated_units_of(case, wide):
    """Token 0's gated unit is 2^128 (1 - 2^-12) in column 3 (past bf16's largest value, not past fp32's), or with ``wide`` times four of
    that, of either sign in the experts' columns 3; token 1's values are small."""
    case.x[:] = 0.0
    case.x[0, :2] = 1.0
    case.x[1] = torch.randn(case.x.shape[1], generator=torch.Generator().manual_seed(5)).to(case.dtype) * 2.0 ** -40
    gate, up, down = case.weights
    gate[:, 3], up[:, 3] = 0.0, 0.0
    gate[:, 3, 0], up[:, 3, 0], up[:, 3, 1] = 2.0 ** 64, 2.0 ** 64, -(2.0 ** 52)
    if wide:
        up[:, 3] *= 4.0
    up[1, 3] *= -1.0
    down[:, :, 3] = torch.where(down[:, :, 3] < 0, -1.0, 1.0) * 2.0 ** -100


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("k", (1, 2))
def test_gated_unit_past_the_largest_bf16_value(dtype, k):
    """In bf16 the unit is two bf16 values: the larger one stays finite where the unit is."""
    case = Case(2, 2, k, 48, 40, dtype)
    _gated_units_of(case, wide=False)
    out, logits = case.call()
    assert out.isfinite().all() and out[0].abs().min() > 0
    case.check(out, logits)


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_infinite_gated_unit(dtype):
    """What the definition in 32 bits has: an infinity of the down projection's sign, and the other token as it is without it."""
    case = Case(2, 2, 1, 48, 40, dtype)
    _gated_units_of(case, wide=True)
    out, logits = case.call()
    ((expert, _),), _ = ref.choose(logits.cpu(), 1, True)
    sign = case.weights[2][expert, :, 3].sign() * (-1 if expert else 1)
    assert torch.equal(out[0].cpu(), sign * float("inf"))
    case.x[0] = 0.0
    assert torch.equal(case.call()[0][1], out[1]) and out[1].isfinite().all()


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
def test_an_expert_that_is_no_number_reaches_its_tokens_alone(dtype):
    case = Case(6, 8, 2, 80, 56, dtype)
    want, logits = case.call()
    picked = [{e for e, _ in p} for p in ref.choose(logits.cpu(), 2, True)]
    bad = next(e for e in range(8) if 0 < sum(e in p for p in picked) < 6)
    case.weights[0][bad, 17, 3] = float("nan")
    out, _ = case.call()
    for t in range(6):
        assert out[t].isnan().all() if bad in picked[t] else torch.equal(out[t], want[t])


def test_infinite_gated_unit_in_8_bits():
    """An infinite element becomes NaN on its way to the grid, as in the expert MLP, and the other token is as it is without it."""
    case = Case(2, 2, 2, 160, 200, BF16, eight=True)
    case.scales[0], case.scales[1] = case.scales[0] * 2.0 ** 80, case.scales[1] * 2.0 ** 80
    case.x[1] *= 2.0 ** -90
    out, _ = case.call()
    assert out[0].isnan().all() and out[1].isfinite().all()
    case.x[0] = 0.0
    assert torch.equal(case.call()[0][1], out[1])


@pytest.mark.parametrize("eight", (False, True))
def test_the_same_bits_every_time(eight):
    case = Case(16, 128, 8, 512, 256, BF16, eight=eight, norm=True, residual=True)
    first = case.call()
    for _ in range(4):
        again = case.call()
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


@pytest.mark.parametrize("eight", (False, True))
def test_captured_and_replayed_with_eager_calls_between(eight):
    case = Case(6, 32, 4, 512, 256, BF16, eight=eight, norm=True, residual=True)
    for name in ("x", "residual", "norm", "router"):
        setattr(case, name, getattr(case, name).cuda())
    case.weights = [w.cuda() for w in case.weights]
    case.scales = [s.cuda() for s in case.scales] if eight else None
    with torch.no_grad():
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            case.call()
        side.synchronize()
        first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(first):
            a = case.call()
        with torch.cuda.graph(second):
            b = case.call()
        for seed in range(4):
            case.x.copy_(torch.randn(case.x.shape, generator=torch.Generator().manual_seed(seed)).to(BF16))
            first.replay()
            got = [t.clone() for t in a]
            want = case.call()
            second.replay()
            torch.cuda.synchronize()
            for p, q, r in zip(got, want, b):
                assert torch.equal(p, q) and torch.equal(r, q)


def test_two_streams_at_once():
    cases = [Case(16, 64, 8, 1024, 512, BF16, norm=True, residual=True, seed=s) for s in range(2)]
    for case in cases:
        for name in ("x", "residual", "norm", "router"):
            setattr(case, name, getattr(case, name).cuda())
        case.weights = [w.cuda() for w in case.weights]
    want = [case.call() for case in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, case in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(case.call())
    torch.cuda.synchronize()
    for i in range(2):
        for out, logits in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(logits, want[i][1])


def test_tangents_batching_and_backward_are_refused():
    from torch.autograd import forward_ad

    case = Case(3, 8, 2, 64, 32, BF16)
    args = [t.cuda() for t in (case.x, case.router, *case.weights)]
    with forward_ad.dual_level(), pytest.raises(RuntimeError):
        moe_fused_layer(forward_ad.make_dual(args[0], args[0]), *args[1:], 2, True)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: moe_fused_layer(x, *args[1:], 2, True))(args[0][None])
    args[2].requires_grad_()
    with pytest.raises(AssertionError):
        moe_fused_layer(*args, 2, True)


# ---- together -------------------------------------------------------------------------------------------------------------------

def test_layer_with_norm_is_norm_then_layer_then_addition():
    case = Case(7, 32, 4, 512, 128, BF16, norm=True, residual=True)
    out, logits = case.call()
    y, s = add_rms_norm(case.x.cuda(), case.residual.cuda(), case.norm.cuda(), EPS)
    part, same = moe_fused_layer(y, case.router.cuda(), *(w.cuda() for w in case.weights), case.k, case.renorm)
    assert torch.equal(logits, same)
    # one rounding of the experts' sum and one of the result more
    want = s.double() + part.double()
    assert ((out.double() - want).abs() <= 2.0 ** -8 * (part.double().abs() + 2 * want.abs()) + 1e-30).all()


def test_layer_against_the_block():
    """The block rounds the gated unit's result twice, each expert's row, each weight and the sum: six half steps, and the same experts
    where its logits, from 32-bit sums, are the same."""
    from qwen3_moe_fused.modular_qwen3_moe_fused import Qwen3MoeFusedSparseMoeBlock

    config = SimpleNamespace(num_experts=32, num_experts_per_tok=4, norm_topk_prob=True, hidden_size=512,
                             moe_intermediate_size=256, hidden_act="silu")
    case = Case(8, 32, 4, 512, 256, BF16)
    block = Qwen3MoeFusedSparseMoeBlock(config).cuda().to(BF16)
    with torch.no_grad():
        block.gate.weight.copy_(case.router)
        for proj, w in zip((block.gate_proj, block.up_proj, block.down_proj), case.weights):
            proj.weight.copy_(w)
        want, want_logits = block(case.x.cuda().view(1, 8, 512))
    out, logits = case.call()
    same = [t for t in range(8) if [e for e, _ in ref.choose(logits[t:t + 1].cpu(), 4, True)[0]]
            == [e for e, _ in ref.choose(want_logits[t:t + 1].cpu(), 4, True)[0]]]
    assert len(same) >= 6
    error = (out - want[0]).double()[same].norm() / out.double()[same].norm()
    assert error <= 6 * 2.0 ** -8


def _mlp_call(case, tokens, quantized=None):
    k, dev = case.k, tokens.device
    logits = (tokens.float() @ case.router.to(dev).float().t()).to(tokens.dtype)
    weights, _, m_sizes, sort_idx, inv = route_and_sort(logits.detach(), k, True, tokens.dtype, case.router.shape[0])
    pairs = [t.to(dev) for pair in zip(case.weights, case.scales) for t in pair]
    return moe_fused_mlp_fp8(tokens, *pairs, m_sizes, sort_idx, inv, k, **({} if quantized is None else {"quantized": quantized}))


@pytest.mark.parametrize("tokens", (3, 700))  # the decode kernels, and the tiles
@pytest.mark.parametrize("hidden", (256, 208))
def test_norm_to_8_bit_rows_then_the_expert_mlp(tokens, hidden):
    case = Case(tokens, 8, 2, hidden, 256, BF16, eight=True, norm=True, residual=True)
    x, r, w = case.x.cuda(), case.residual.cuda(), case.norm.cuda()
    with torch.no_grad():
        values, scales, s, y = add_rms_norm_fp8(x, r, w, EPS, return_normed=True)
        assert torch.equal(_mlp_call(case, y, (values, scales)), _mlp_call(case, y))
    # a training step: the gradient goes through the normed rows
    grads = []
    for given in (True, False):
        leaves = [t.clone().requires_grad_() for t in (x, r, w)]
        values, scales, s, y = add_rms_norm_fp8(*leaves, EPS, return_normed=True)
        out = _mlp_call(case, y, (values, scales) if given else None)
        grads.append(torch.autograd.grad((out, s), leaves, (torch.ones_like(out), torch.ones_like(s))))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    assert all(t.isfinite().all() and t.abs().max() > 0 for t in grads[0])


def test_quantised_rows_of_another_form_are_refused():
    case = Case(40, 8, 2, 256, 128, BF16, eight=True)
    tokens = case.x.cuda()
    values, scales = quantize_fp8_rows(tokens)
    for bad in ((values[:39], scales), (values, scales[:, :1]), (values.view(torch.uint8), scales), (values.cpu(), scales),
                (values.clone(memory_format=torch.contiguous_format)[:, :128], scales)):
        with pytest.raises(AssertionError):
            _mlp_call(case, tokens, bad)
    assert _lib.lib() is not None
