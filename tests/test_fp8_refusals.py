"""Calls of the 8-bit floating-point products that are refused before anything reaches a device."""
import ctypes

import pytest
import torch

from qwen3_moe_fused import _lib

BF16, F32, I32, I64 = _lib.BF16, _lib.F32, _lib.I32, _lib.I64
NULL, SHAPE, DTYPE, ALIGN, WORKSPACE = -1, -2, -3, -4, -5


@pytest.fixture
def p():
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    yield at
    del buf


def test_workspaces():
    lib = _lib.lib()
    # values 256 bytes a row, scales 4 bytes a row, each rounded up to 256
    assert lib.mfl_fp8_workspace(0, 10, 80, 64, 208, 4) == 2560 + 256
    assert lib.mfl_fp8_workspace(1, 10, 80, 64, 208, 4) == 80 * 128 + 512
    assert lib.mfl_fp8_workspace(3, 0, 80, 64, 208, 4) == 2 * (80 * 128 + 512)
    assert lib.mfl_fp8_workspace(4, 10, 80, 64, 208, 4) >= 2560 + 256 + 80 * 128 + 512
    # weights in rows of 200 bytes are copied to rows of 208 where there are four rows per expert and more
    assert lib.mfl_fp8_workspace(0, 16, 16, 64, 200, 4) == 4096 + 256 + 4 * 64 * 208
    assert lib.mfl_fp8_workspace(2, 16, 16, 64, 200, 4) == 4096 + 256 + 2 * 4 * 64 * 208
    assert lib.mfl_fp8_workspace(0, 15, 15, 64, 200, 4) == 15 * 256 + 256
    for bad in ((0, 10, 0, 64, 200, 4), (0, -1, 8, 64, 200, 4), (0, 8, 8, 0, 200, 4), (9, 8, 8, 64, 200, 4), (0, 8, 8, 64, 200, 0)):
        assert lib.mfl_fp8_workspace(*bad) == 0


def test_products(p):
    lib, w = _lib.lib(), _lib.Fp8Weight(p, p)

    def fwd(x=p, src=4, idx=None, div=1, weight=w, ms=p, it=I32, y=p, rows=4, n=8, k=8, e=2, dt=BF16, out=BF16, ws=p, size=4096):
        return lib.mfl_gemm_fwd_fp8(x, src, idx, div, weight, ms, it, y, rows, n, k, e, dt, out, ws, size, None)

    def dx(x=p, weight=w, ms=p, it=I32, y=p, rows=4, n=8, k=8, e=2, dt=BF16, out=BF16, ws=p, size=4096):
        return lib.mfl_gemm_dx_fp8(x, weight, ms, it, y, rows, n, k, e, dt, out, ws, size, None)

    for call in (fwd, dx):
        assert call(ms=None) == NULL and call(x=None) == NULL and call(y=None) == NULL and call(weight=None) == NULL
        assert call(weight=_lib.Fp8Weight(p, None)) == NULL and call(weight=_lib.Fp8Weight(None, p)) == NULL
        assert call(n=0) == SHAPE and call(k=-1) == SHAPE and call(e=0) == SHAPE and call(rows=-1) == SHAPE
        assert call(rows=2 ** 31) == SHAPE
        assert call(dt=7) == DTYPE and call(out=7) == DTYPE and call(it=5) == DTYPE
        assert call(x=p + 1) == ALIGN and call(y=p + 1) == ALIGN and call(ms=p + 2) == ALIGN and call(ws=p + 16) == ALIGN
        assert call(weight=_lib.Fp8Weight(p, p + 1)) == ALIGN
        assert call(ws=None) == WORKSPACE and call(size=100) == WORKSPACE
        assert call(rows=0, x=None, y=None, ws=None, size=0) == 0
    assert fwd(idx=p, div=0) == SHAPE and fwd(idx=p, src=0) == SHAPE and fwd(src=3) == SHAPE and fwd(idx=p + 2) == ALIGN


def test_gated_unit_and_mlp(p):
    lib, w = _lib.lib(), _lib.Fp8Weight(p, p)

    def glu(x=p, src=4, idx=None, div=1, gate=w, up=w, ms=p, it=I32, h=p, e=None, g=None, rows=4, n=8, k=8, ex=2, dt=BF16, ws=p,
            size=4096):
        return lib.mfl_glu_fwd_fp8(x, src, idx, div, gate, up, ms, it, h, e, g, rows, n, k, ex, dt, ws, size, None)

    def mlp(x=p, src=4, idx=None, div=1, gate=w, up=w, down=w, ms=p, it=I32, h=p, e=None, g=None, rows=4, n=8, k=8, ex=2,
            dt=BF16, ws=p, size=4096):
        return lib.mfl_mlp_fwd_fp8(x, src, idx, div, gate, up, down, ms, it, h, e, g, rows, n, k, ex, dt, ws, size, None)

    def bwd(x=p, e=p, g=p, gate=w, up=w, ms=p, it=I32, h=p, rows=4, n=8, k=8, ex=2, dt=BF16, ws=p, size=4096):
        return lib.mfl_glu_bwd_fp8(x, e, g, gate, up, ms, it, h, rows, n, k, ex, dt, ws, size, None)

    for call in (glu, mlp, bwd):
        assert call(ms=None) == NULL and call(x=None) == NULL and call(h=None) == NULL
        assert call(gate=None) == NULL and call(up=None) == NULL
        assert call(n=0) == SHAPE and call(rows=-1) == SHAPE and call(ex=-3) == SHAPE
        assert call(dt=9) == DTYPE and call(it=9) == DTYPE
        assert call(h=p + 1) == ALIGN and call(e=p + 1, g=p) == ALIGN and call(e=p, g=p + 1) == ALIGN
        assert call(ws=None) == WORKSPACE and call(size=64) == WORKSPACE
        assert call(rows=0, ws=None, size=0) == 0
    assert mlp(down=None) == NULL and mlp(e=p) == NULL and bwd(e=None) == NULL
    for call in (glu, mlp):
        assert call(idx=p, div=0) == SHAPE and call(idx=p, src=0) == SHAPE and call(src=3) == SHAPE


def test_quantisers(p):
    lib = _lib.lib()
    assert lib.mfl_fp8_quant_rows(p, BF16, -1, 8, p, p, None) == SHAPE and lib.mfl_fp8_quant_rows(p, BF16, 1, 0, p, p, None) == SHAPE
    assert lib.mfl_fp8_quant_rows(p, 5, 1, 8, p, p, None) == DTYPE and lib.mfl_fp8_quant_rows(p, BF16, 1, 8, None, p, None) == NULL
    assert lib.mfl_fp8_quant_rows(p, BF16, 1, 8, p + 8, p, None) == ALIGN and lib.mfl_fp8_quant_rows(None, BF16, 0, 8, None, None, None) == 0
    assert lib.mfl_fp8_dequant_rows(p, p, 1, 8, None, F32, None) == NULL and lib.mfl_fp8_dequant_rows(p, p, 1, 8, p + 2, F32, None) == ALIGN
    assert lib.mfl_fp8_quant_blocks(p, BF16, 0, 8, 8, p, p, None) == SHAPE and lib.mfl_fp8_quant_blocks(p, 4, 1, 8, 8, p, p, None) == DTYPE
    assert lib.mfl_fp8_dequant_blocks(p, None, 1, 8, 8, p, F32, None) == NULL


def test_python_checks():
    from qwen3_moe_fused.fused_mlp import moe_fused_glu_fp8, moe_fused_mlp_fp8
    from qwen3_moe_fused.grouped_gemm.forward_fp8 import check_rows, grouped_gemm_forward_fp8
    from qwen3_moe_fused.quantize.fp8 import check_fp8_weight, quantize_fp8_blocks, quantize_fp8_rows
    from qwen3_moe_fused.quantize.layer_fp8 import moe_fused_linear_fp8

    x, ms = torch.zeros((4, 128), dtype=torch.bfloat16), torch.tensor([4])
    w, s = torch.zeros((1, 64, 128)).to(torch.float8_e4m3fn), torch.ones((1, 1, 1))
    for call in (lambda: grouped_gemm_forward_fp8(x, w, s, ms), lambda: moe_fused_linear_fp8(x, w, s, ms),
                 lambda: quantize_fp8_rows(x), lambda: quantize_fp8_blocks(w.float())):
        with pytest.raises(AssertionError):
            call()
    assert check_fp8_weight(x, w, s) == (1, 64, 128)
    for bad_w, bad_s in ((w.float(), s), (w[0], s), (w, s.double()), (w, torch.ones((1, 1, 2))), (w.transpose(1, 2), s),
                         (w.view(torch.uint8), s)):
        with pytest.raises(AssertionError):
            check_fp8_weight(x, bad_w, bad_s)
    with pytest.raises(AssertionError):
        check_rows(ms, x)
    with pytest.raises(AssertionError):  # frozen
        moe_fused_linear_fp8(x, w, s.clone().requires_grad_(), ms)
    idx = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: moe_fused_glu_fp8(x, w, s, w, s, ms, idx, idx, 1),
                 lambda: moe_fused_mlp_fp8(x, w, s, w, s, w, s, ms, idx.int()[:3], idx.int(), 1)):
        with pytest.raises(AssertionError):
            call()


def test_module_loads_only_what_it_can_hold():
    from qwen3_moe_fused.quantize.layer_fp8 import MoeFusedLinearFp8

    m = MoeFusedLinearFp8(130, 64, 2)
    good = {"weight": torch.zeros((2, 64, 130)).to(torch.float8_e4m3fn), "weight_scale_inv": torch.ones((2, 1, 2), dtype=torch.bfloat16)}
    m.load_state_dict(good)
    assert m.weight_scale_inv.dtype == torch.float32 and m.weight.dtype == torch.float8_e4m3fn
    for change in ({"weight": torch.zeros((2, 64, 130))}, {"weight": good["weight"][:1]}, {"weight_scale_inv": torch.ones((2, 1, 1))},
                   {"weight": torch.zeros((2, 64, 130)).to(torch.float8_e5m2)}, {"weight": torch.zeros((2, 64, 130), dtype=torch.int8)}):
        with pytest.raises(RuntimeError):
            m.load_state_dict({**good, **change})
    with pytest.raises(RuntimeError):  # a floating-point weight needs the GPU's quantiser
        m.load_state_dict({"weight": torch.zeros((2, 64, 130))})
    with pytest.raises(RuntimeError):
        m.load_state_dict({"weight": good["weight"]})
    assert m.to(torch.bfloat16).weight.dtype == torch.float8_e4m3fn


def test_widths_past_what_is_counted(p):
    """2^30 columns at most: more would not be countable in whole blocks."""
    lib, w, big = _lib.lib(), _lib.Fp8Weight(p, p), 2 ** 30 + 1
    assert lib.mfl_fp8_workspace(0, 1, 1, 1, 2 ** 31 - 1, 1) == 0
    for n, k in ((big, 8), (8, big), (8, 2 ** 31 - 1)):
        assert lib.mfl_gemm_fwd_fp8(p, 1, None, 1, w, p, I32, p, 1, n, k, 1, BF16, BF16, p, 4096, None) == SHAPE
        assert lib.mfl_gemm_dx_fp8(p, w, p, I32, p, 1, n, k, 1, BF16, BF16, p, 4096, None) == SHAPE
        assert lib.mfl_glu_fwd_fp8(p, 1, None, 1, w, w, p, I32, p, None, None, 1, n, k, 1, BF16, p, 4096, None) == SHAPE
        assert lib.mfl_glu_bwd_fp8(p, p, p, w, w, p, I32, p, 1, n, k, 1, BF16, p, 4096, None) == SHAPE
        assert lib.mfl_mlp_fwd_fp8(p, 1, None, 1, w, w, w, p, I32, p, None, None, 1, n, k, 1, BF16, p, 4096, None) == SHAPE
        assert lib.mfl_fp8_quant_blocks(p, BF16, 1, n, k, p, p, None) == SHAPE
        assert lib.mfl_fp8_dequant_blocks(p, p, 1, n, k, p, BF16, None) == SHAPE
    assert lib.mfl_fp8_quant_rows(p, BF16, 1, big, p, p, None) == SHAPE
    assert lib.mfl_fp8_dequant_rows(p, p, 1, big, p, BF16, None) == SHAPE


def test_mlp_workspace_holds_fp32_values_only_where_they_are_needed(p):
    """Tiles take the unit's result to quantised rows themselves: nothing of 4 bytes an element, 131072 rows of 768."""
    lib, w = _lib.lib(), _lib.Fp8Weight(p, p)
    rows = 16384 * 2048 + 16384 * 16 + 131072 * 768 + 131072 * 8
    assert lib.mfl_fp8_workspace(4, 16384, 131072, 768, 2048, 128) == rows
    assert lib.mfl_fp8_workspace(5, 16384, 131072, 768, 2048, 128) == rows + 131072 * 768 * 4
    values = 40 * 64 * 4
    for args, needed in (((10, 40, 64, 208, 4), False), ((10, 32, 64, 208, 4), True), ((10, 40, 64, 128, 4), True)):
        r, n, k = args[1:4]
        up = lambda b: -(-b // 256) * 256
        least = up(10 * (-(-k // 128) * 128)) + up(10 * 4) + up(r * 128) + up(r * 4)
        assert lib.mfl_fp8_workspace(4, *args) == least + (up(r * n * 4) if needed else 0)
        assert lib.mfl_fp8_workspace(5, *args) == least + up(r * n * 4)
    # weights off the grid need the larger one, and say so before anything is launched
    off = _lib.Fp8Weight(p + 1, p)
    small = lib.mfl_fp8_workspace(4, 10, 40, 64, 208, 4)
    assert lib.mfl_mlp_fwd_fp8(p, 10, p, 4, off, w, w, p, I32, p, None, None, 40, 64, 208, 4, BF16, p, small, None) == WORKSPACE
    assert lib.mfl_mlp_fwd_fp8(p, 10, p, 4, w, w, w, p, I32, p, p + 2, p + 2, 40, 64, 208, 4, BF16, p, small, None) == WORKSPACE
    assert values == lib.mfl_fp8_workspace(5, 10, 40, 64, 208, 4) - small
