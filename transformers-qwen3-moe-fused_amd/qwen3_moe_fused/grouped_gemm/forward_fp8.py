"""Grouped GEMM with expert weights in 8-bit floating point: forward and input gradient.

Host wrappers over ``mfl_gemm_fwd_fp8`` / ``mfl_gemm_dx_fp8``.  ``w`` (E, out, in) float8_e4m3fn with fp32 scales per 128 x 128
block; the rows (bf16, fp16 or fp32) are quantised by the call, one power-of-two scale per row and 128 elements of the
reduction (``quantize/fp8.py``).  Rows of magnitudes past 2^111 may overflow before the weights' scales are applied.  The contract
is otherwise that of ``grouped_gemm_forward``: output freshly allocated, rows past ``sum(m_sizes)`` left unwritten, ``m_sizes``
stays on the device.  The reference has no counterpart.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from ..quantize.fp8 import check_fp8_weight
from ._common import is_int_tensor

# MFL_FP8_*: whose workspace is asked for
FWD, DX, GLU, GLU_BWD, MLP, MLP_OFF_GRID = 0, 1, 2, 3, 4, 5
_NO_WORKSPACE = -5  # MFL_ERR_WORKSPACE
# Rows per expert up to which the forward product and the gated unit are called without scratch memory first: decode sizes do
# without, and asking for it and allocating it is a fifth of such a call's time on the host.
_DECODE_ROWS = 8  # MFL_FP8_DECODE_ROWS


def fp8_weight(weight: torch.Tensor, scale: torch.Tensor) -> "_lib.Fp8Weight":
    return _lib.Fp8Weight(weight.data_ptr(), scale.data_ptr())


def fp8_workspace(op: int, like: torch.Tensor, src_rows: int, rows: int, n: int, k: int, experts: int):
    """(scratch tensor or None, its address or None, its size) of a call."""
    size = _lib.lib().mfl_fp8_workspace(op, src_rows, rows, n, k, experts)
    if size == 0:
        return None, None, 0
    ws = torch.empty(size, device=like.device, dtype=torch.uint8)
    return ws, ws.data_ptr(), size


def call_with_workspace(call, op: int, like: torch.Tensor, src_rows: int, rows: int, n: int, k: int, experts: int) -> int:
    """``call(address, size)``'s status, with scratch memory where it needs some."""
    if rows <= _DECODE_ROWS * experts:
        rc = call(None, 0)
        if rc != _NO_WORKSPACE:
            return rc
    _keep, ws, size = fp8_workspace(op, like, src_rows, rows, n, k, experts)
    return call(ws, size)


def check_rows(m_sizes: torch.Tensor, *rows: torch.Tensor) -> None:
    """The left operands (one type and shape) and the row counts."""
    first = rows[0]
    assert first.is_cuda, "grouped GEMM runs on the GPU only"
    _lib.dtype_code(first.dtype)  # (TypeError for other types)
    for t in rows:
        assert t.ndim == 2 and t.shape == first.shape and t.dtype == first.dtype
        assert t.device == first.device and t.is_contiguous()
    assert m_sizes.ndim == 1 and is_int_tensor(m_sizes) and m_sizes.device == first.device and m_sizes.is_contiguous()


def grouped_gemm_forward_fp8(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, m_sizes: torch.Tensor,
                             dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y[r, n] = sum_k w[e(r), n, k] x[r, k]: ``x`` (rows, in), result (rows, out) in ``dtype`` (default: of ``x``)."""
    check_rows(m_sizes, x)
    rows, k = x.shape
    experts, n, k_w = check_fp8_weight(x, w, w_scale)
    assert k_w == k and m_sizes.numel() == experts
    with _lib.on_device_of(x):
        y = x.new_empty(rows, n, dtype=dtype)
        ms = _lib.as_index_tensor(m_sizes)
        entry, weight = _lib.lib().mfl_gemm_fwd_fp8, fp8_weight(w, w_scale)
        args = (x.data_ptr(), rows, None, 1, weight, ms.data_ptr(), _lib.itype_code(ms.dtype), y.data_ptr(), rows, n, k, experts,
                _lib.dtype_code(x.dtype), _lib.dtype_code(y.dtype))
        rc = call_with_workspace(lambda ws, size: entry(*args, ws, size, _lib.stream()), FWD, x, rows, rows, n, k, experts)
    _lib.check(rc, "mfl_gemm_fwd_fp8")
    return y


def grouped_gemm_forward_transposed_fp8(dy: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, m_sizes: torch.Tensor,
                                        dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """dx[r, k] = sum_n w[e(r), n, k] dy[r, n]: ``dy`` (rows, out), result (rows, in)."""
    check_rows(m_sizes, dy)
    rows, n = dy.shape
    experts, n_w, k = check_fp8_weight(dy, w, w_scale)
    assert n_w == n and m_sizes.numel() == experts
    with _lib.on_device_of(dy):
        dx = dy.new_empty(rows, k, dtype=dtype)
        ms = _lib.as_index_tensor(m_sizes)
        _keep, ws, ws_bytes = fp8_workspace(DX, dy, rows, rows, n, k, experts)
        rc = _lib.lib().mfl_gemm_dx_fp8(dy.data_ptr(), fp8_weight(w, w_scale), ms.data_ptr(), _lib.itype_code(ms.dtype),
                                        dx.data_ptr(), rows, n, k, experts, _lib.dtype_code(dy.dtype),
                                        _lib.dtype_code(dx.dtype), ws, ws_bytes, _lib.stream())
    _lib.check(rc, "mfl_gemm_dx_fp8")
    return dx
