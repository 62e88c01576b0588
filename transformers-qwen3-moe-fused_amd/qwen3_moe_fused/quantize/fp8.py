"""Quantisation to e4m3 (8-bit floating point) blocks, for rows and for expert weights.

Rows (activations, gradients): one power-of-two scale per row and 128 elements, kept as e8m0.  Weights (E, out, in): one fp32
scale per 128 x 128 block, as block-quantised checkpoints carry it (``weight_scale_inv``); the products take any finite fp32
scale, the quantiser here writes powers of two by the rows' rule: the smallest, 2^-117 at least, that brings the block's
largest finite magnitude to 448 or below.  Dividing by a power of two is exact, so every element is rounded once (nearest,
ties to even); elements that are infinite or no number become NaN and leave their block's scale to the others.
"""
from __future__ import annotations

from typing import Tuple

import torch

from .. import _lib

BLOCK = 128
FP8 = torch.float8_e4m3fn


def blocks_of(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def check_fp8_weight(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor) -> Tuple[int, int, int]:
    """The checks that the products share; returns the weight's (experts, out features, in features)."""
    assert weight.dtype == FP8 and weight.ndim == 3, "expert weights are (E, out, in) float8_e4m3fn"
    experts, n, k = weight.shape
    assert scale.dtype == torch.float32 and scale.shape == (experts, (n + 127) // 128, (k + 127) // 128)
    device = x.get_device()  # (x is on a GPU; an index compares faster than a device)
    assert weight.get_device() == device and scale.get_device() == device
    assert weight.is_contiguous() and scale.is_contiguous()
    return experts, n, k


def check_fp8_rows(values: torch.Tensor, scale: torch.Tensor, like: torch.Tensor) -> None:
    """That (values, scale) are quantised rows of ``like``'s shape and device, as ``quantize_fp8_rows`` lays them out."""
    assert values.dtype == FP8 and scale.dtype == torch.float8_e8m0fnu and values.shape == like.shape and like.ndim == 2
    rows, k = values.shape
    blocks = blocks_of(k)
    assert scale.shape == (rows, blocks)
    device = like.get_device()
    assert values.get_device() == device and scale.get_device() == device
    # (the last row has room behind its last column too: of a single row the stride does not say so, a copy keeps it and ends with the
    # column; where rows are whole blocks none is needed)
    for t, width, ld in ((values, k, blocks * BLOCK), (scale, blocks, (blocks + 3) // 4 * 4)):
        assert rows == 0 or (rows == 1 and width == ld) or (
            t.stride(0) == ld and t.untyped_storage().nbytes() >= t.storage_offset() + rows * ld), \
            "values and scales as quantize_fp8_rows lays them out"
    assert (k == 1 or values.stride(1) == 1) and (blocks == 1 or scale.stride(1) == 1)


def empty_fp8_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Room for ``x``'s quantised rows, laid out as ``quantize_fp8_rows`` says.  (Nothing is sliced that is whole: 2 us a tensor.)"""
    rows, k = x.shape
    blocks = blocks_of(k)
    ld, ld_scale = blocks * BLOCK, (blocks + 3) // 4 * 4
    values = torch.empty((rows, ld), device=x.device, dtype=FP8)
    scale = torch.empty((rows, ld_scale), device=x.device, dtype=torch.float8_e8m0fnu)
    return values if ld == k else values[:, :k], scale if ld_scale == blocks else scale[:, :blocks]


def quantize_fp8_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x`` (rows, K) in bf16 / fp16 / fp32 -> (values (rows, K) float8_e4m3fn, scales (rows, ceil(K / 128))
    float8_e8m0fnu).  Rows of the values lie a multiple of 128 bytes apart (zeros behind column K), those of the scales a
    multiple of 4."""
    assert x.is_cuda and x.ndim == 2 and x.is_contiguous()
    rows, k = x.shape
    dtype = _lib.dtype_code(x.dtype)
    with _lib.on_device_of(x):
        q, scale = empty_fp8_rows(x)
        rc = _lib.lib().mfl_fp8_quant_rows(x.data_ptr(), dtype, rows, k, q.data_ptr(), scale.data_ptr(), _lib.stream())
    _lib.check(rc, "mfl_fp8_quant_rows")
    return q, scale


def dequantize_fp8_rows(values: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that ``quantize_fp8_rows`` left, in ``dtype`` (exact in bf16 and fp32)."""
    assert values.is_cuda and values.ndim == 2 and values.dtype == FP8 and scale.dtype == torch.float8_e8m0fnu
    rows, k = values.shape
    blocks = blocks_of(k)
    assert scale.shape == (rows, blocks) and scale.device == values.device
    # (a single row, or none, may have any stride)
    assert rows <= 1 or (values.stride() == (blocks * BLOCK, 1) and scale.stride() == ((blocks + 3) // 4 * 4, 1)), \
        "values and scales as quantize_fp8_rows lays them out"
    assert values.stride(1) == 1 and scale.stride(1) == 1
    with _lib.on_device_of(values):
        out = torch.empty((rows, k), device=values.device, dtype=dtype)
        rc = _lib.lib().mfl_fp8_dequant_rows(values.data_ptr(), scale.data_ptr(), rows, k, out.data_ptr(),
                                             _lib.dtype_code(dtype), _lib.stream())
    _lib.check(rc, "mfl_fp8_dequant_rows")
    return out


def quantize_fp8_blocks(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``weight`` (E, out, in) in bf16 / fp16 / fp32 -> (float8_e4m3fn values of the same shape, fp32 scales)."""
    assert weight.is_cuda and weight.ndim == 3 and weight.is_contiguous()
    experts, n, k = weight.shape
    with _lib.on_device_of(weight):
        q = torch.empty(weight.shape, device=weight.device, dtype=FP8)
        scale = torch.empty((experts, blocks_of(n), blocks_of(k)), device=weight.device, dtype=torch.float32)
        rc = _lib.lib().mfl_fp8_quant_blocks(weight.data_ptr(), _lib.dtype_code(weight.dtype), experts, n, k, q.data_ptr(),
                                             scale.data_ptr(), _lib.stream())
    _lib.check(rc, "mfl_fp8_quant_blocks")
    return q, scale


def dequantize_fp8_blocks(weight: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``weight * scale`` block by block, the product rounded once to ``dtype``."""
    assert weight.is_cuda
    experts, n, k = check_fp8_weight(weight, weight, scale)
    with _lib.on_device_of(weight):
        out = torch.empty(weight.shape, device=weight.device, dtype=dtype)
        rc = _lib.lib().mfl_fp8_dequant_blocks(weight.data_ptr(), scale.data_ptr(), experts, n, k, out.data_ptr(),
                                               _lib.dtype_code(dtype), _lib.stream())
    _lib.check(rc, "mfl_fp8_dequant_blocks")
    return out
