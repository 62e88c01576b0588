"""How the 8-bit floating-point products are called, on the CPU: the tensors claim to be on the GPU, and the library is a
stand-in that sums every row of the left operand."""
import ctypes

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from qwen3_moe_fused import _lib
from qwen3_moe_fused.fused_mlp import moe_fused_glu_fp8, moe_fused_mlp_fp8
from qwen3_moe_fused.quantize.layer_fp8 import moe_fused_linear_fp8

FP8 = torch.float8_e4m3fn
TOKENS, K, EXPERTS, HIDDEN, INTER = 4, 2, 3, 256, 128
ROWS = TOKENS * K


def _array(address, *shape):
    return np.ctypeslib.as_array((ctypes.c_float * int(np.prod(shape))).from_address(address)).reshape(shape)


class _RowSums:
    """Every output's row r is filled with the sum of the row that it is made of (fp32 only)."""

    def __init__(self):
        self.calls = []

    def mfl_fp8_workspace(self, *sizes):
        return 0

    def _run(self, name, x, src_rows, idx, div, width, outs, rows):
        self.calls.append(name)
        source = _array(x, src_rows, width).sum(axis=1)
        index = np.arange(rows) if idx is None else np.ctypeslib.as_array((ctypes.c_int32 * rows).from_address(idx)) // div
        for at, n in outs:
            if at is not None:
                _array(at, rows, n)[:] = source[index][:, None]
        return 0

    def mfl_gemm_fwd_fp8(self, x, src, idx, div, w, ms, it, y, rows, n, k, *rest):
        return self._run("gemm_fwd", x, src, idx, div, k, [(y, n)], rows)

    def mfl_gemm_dx_fp8(self, dy, w, ms, it, dx, rows, n, k, *rest):
        return self._run("gemm_dx", dy, rows, None, 1, n, [(dx, k)], rows)

    def mfl_glu_fwd_fp8(self, x, src, idx, div, gate, up, ms, it, h, e, g, rows, n, k, *rest):
        return self._run("glu_fwd", x, src, idx, div, k, [(h, n), (e, n), (g, n)], rows)

    def mfl_glu_bwd_fp8(self, dh, e, g, gate, up, ms, it, dx, rows, n, k, *rest):
        return self._run("glu_bwd", dh, rows, None, 1, n, [(dx, k)], rows)

    def mfl_mlp_fwd_fp8(self, x, src, idx, div, gate, up, down, ms, it, y, e, g, rows, inter, hidden, *rest):
        return self._run("mlp_fwd", x, src, idx, div, hidden, [(y, hidden), (e, inter), (g, inter)], rows)

    def mfl_combine_rows(self, *args):
        self.calls.append("combine")
        return 0


@pytest.fixture
def library(monkeypatch):
    stand_in = _RowSums()
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(_lib, "lib", lambda: stand_in)
    monkeypatch.setattr(_lib, "stream", lambda: 0)
    return stand_in


def _weights():
    out = []
    for n, k in ((INTER, HIDDEN), (INTER, HIDDEN), (HIDDEN, INTER)):
        out += [torch.zeros((EXPERTS, n, k), dtype=torch.uint8).view(FP8), torch.ones(EXPERTS, n // 128, k // 128)]
    return out


def _call(which):
    """(a function of the left operand, its rows)"""
    w, sizes = _weights(), torch.tensor([3, 4, 1], dtype=torch.int32)
    idx = torch.arange(ROWS, dtype=torch.int32)
    if which == "linear":
        return lambda x: moe_fused_linear_fp8(x, w[0], w[1], sizes), ROWS
    if which == "glu":
        return lambda x: moe_fused_glu_fp8(x, *w[:4], sizes, idx, idx.clone(), K), TOKENS
    return lambda x: moe_fused_mlp_fp8(x, *w, sizes, idx, idx.clone(), K), TOKENS


WHICH = pytest.mark.parametrize("which", ["linear", "glu", "mlp"])


@WHICH
def test_a_trace_holds_the_call(library, which):
    call, rows = _call(which)
    a, b = torch.randn(rows, HIDDEN), torch.randn(rows, HIDDEN)
    with torch.no_grad():
        traced = torch.jit.trace(call, (a,), check_trace=False)
        del library.calls[:]
        got = traced(b)
        assert len(library.calls) == 1
        assert torch.equal(got, call(b)) and not torch.equal(got, call(a))


@WHICH
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(library, which, grad):
    call, rows = _call(which)
    x = torch.randn(rows, HIDDEN, requires_grad=grad)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises((NotImplementedError, RuntimeError)):
            call(forward_ad.make_dual(x, torch.ones_like(x)))


@WHICH
def test_a_plain_call_without_gradients_is_one_library_call(library, which):
    call, rows = _call(which)
    x = torch.randn(rows, HIDDEN)
    out = call(x)
    expect = x.sum(1) if which == "linear" else x.sum(1).repeat_interleave(K)
    assert len(library.calls) == 1 and not out.requires_grad
    assert torch.allclose(out, expect[:, None].expand_as(out), rtol=1e-4, atol=1e-4)


def test_an_adapter_over_8_bit_weights_keeps_its_type_whatever_the_base_class(monkeypatch):
    """The base class may move an adapter to the type of the base weight, as it does for 16-bit ones."""
    from qwen3_moe_fused import lora
    from qwen3_moe_fused.modular_qwen3_moe_fused import MoeFusedLinear
    from qwen3_moe_fused.quantize.layer_fp8 import MoeFusedLinearFp8

    def move(self, adapter_name, device=None):
        weight = self.get_base_layer().weight
        for adapters in (self.lora_A, self.lora_B):
            adapters[adapter_name].to(device=weight.device, dtype=weight.dtype)

    monkeypatch.setattr(lora.LoraLayer, "_move_adapter_to_device_of_base_layer", move)
    over = lora.LoraMoeFusedLinear(MoeFusedLinearFp8(32, 16, 2), "default", r=4)
    assert {p.dtype for p in (over.lora_A["default"].weight, over.lora_B["default"].weight)} == {torch.float32}
    over._move_adapter_to_device_of_base_layer("default", torch.device("cpu"))
    assert over.lora_A["default"].weight.dtype == torch.float32
    plain = lora.LoraMoeFusedLinear(MoeFusedLinear(32, 16, 2).to(torch.bfloat16), "default", r=4)
    assert plain.lora_A["default"].weight.dtype == torch.bfloat16


def _step(which, x):
    call, _ = _call(which)
    return call(x)


@WHICH
def test_saved_tensors_that_come_back_in_other_strides(library, monkeypatch, which):
    """A saved-tensor hook may hand equal tensors back that are laid out otherwise."""
    from qwen3_moe_fused import fused_mlp

    monkeypatch.setattr(fused_mlp, "_combine", lambda dx, inv, *a: dx.view(TOKENS, K, -1).sum(1))

    def strided(t):
        raw = torch.empty((*t.shape, 2), dtype=torch.uint8 if t.dtype == FP8 else t.dtype)
        out = (raw.view(FP8) if t.dtype == FP8 else raw)[..., 0]
        assert out.is_contiguous() == (out.numel() < 2)
        return out.copy_(t)

    _, rows = _call(which)
    grads = []
    for unpack in (lambda t: t, strided):
        x = torch.ones(rows, HIDDEN, requires_grad=True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            out = _step(which, x)
            out.backward(torch.arange(out.numel(), dtype=torch.float32).view_as(out))
        grads.append(x.grad)
    assert torch.equal(*grads)


@WHICH
def test_second_derivatives_and_batches_of_gradients_are_refused(library, monkeypatch, which):
    """A gradient that kernels have written is no function of anything for autograd: a second derivative would leave it out."""
    from qwen3_moe_fused import fused_mlp

    monkeypatch.setattr(fused_mlp, "_combine", lambda dx, inv, *a: dx.view(TOKENS, K, -1).sum(1))
    _, rows = _call(which)
    x = torch.ones(rows, HIDDEN, requires_grad=True)
    out = _step(which, x)
    dx, = torch.autograd.grad(out, x, torch.ones_like(out).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (dx.sum() + x.square().sum()).backward()
    out = _step(which, x)
    with pytest.raises((RuntimeError, AssertionError, NotImplementedError)):
        torch.autograd.grad(out, x, torch.ones(2, *out.shape), is_grads_batched=True)


def test_the_decode_sizes_are_the_librarys():
    import os
    import re

    from qwen3_moe_fused.grouped_gemm import forward_fp8

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "include", "moe_fused_linear.h")) as f:
        assert re.findall(r"#define MFL_FP8_DECODE_ROWS (\d+)", f.read()) == [str(forward_fp8._DECODE_ROWS)]
