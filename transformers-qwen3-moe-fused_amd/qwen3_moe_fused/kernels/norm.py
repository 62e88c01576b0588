"""The residual's addition and the root-mean-square norm behind it, which stand in front of the sparse block in a decoder layer.

    s = x + residual,   y = s / sqrt(mean(s^2) + eps) * weight

``s`` is rounded to the type of the tensors, as the stream that a model carries on, and the norm is that of the rounded values;
sums and products are in 64 bits, and ``y`` is rounded once (to 32 bits and from there to the type).  The reference leaves both to the
stock decoder layer, whose norm rounds once more between its two products.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _lib
from ..quantize.fp8 import empty_fp8_rows


WIDTH = 32768  # MFL_NORM_WIDTH


def most_rows(width: int) -> int:
    """The rows that one call takes at a width up to ``WIDTH``: a launch's threads are counted in 32 bits, and a row has 64 of them up to
    512 columns, twice as many for every doubling up to 1024."""
    lanes = 64
    while lanes < 1024 and lanes * 8 < width:
        lanes *= 2
    return (1 << 32) // lanes - 1024


def _check(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor) -> Tuple[int, int, int]:
    """Returns (rows, width, the type's code)."""
    assert x.is_cuda and x.ndim >= 1 and x.is_contiguous(), "the norm runs on the GPU, on dense rows"
    dtype, width = _lib.dtype_code(x.dtype), x.shape[-1]
    device = x.get_device()
    if residual is not None:
        assert residual.shape == x.shape and residual.dtype == x.dtype and residual.is_contiguous()
        assert residual.get_device() == device
    assert weight.shape == (width,) and weight.is_contiguous() and weight.get_device() == device
    assert weight.dtype in (x.dtype, torch.float32), "the norm's weight is of the rows' type or float32"
    assert width > 0
    return x.numel() // width, width, dtype


def _forward(x, residual, weight, eps):
    rows, width, dtype = _check(x, residual, weight)
    with _lib.on_device_of(x):
        y = torch.empty_like(x)
        s = x if residual is None else torch.empty_like(x)
        rc = _lib.lib().mfl_add_rms_norm(x.data_ptr(), _lib.ptr(residual), weight.data_ptr(), y.data_ptr(), s.data_ptr(), rows,
                                         width, eps, dtype, _lib.dtype_code(weight.dtype), _lib.stream())
    _lib.check(rc, "mfl_add_rms_norm")
    return y, s


def _forward_fp8(x, residual, weight, eps, return_normed):
    rows, width, dtype = _check(x, residual, weight)
    assert x.ndim == 2, "quantised rows are a matrix"
    with _lib.on_device_of(x):
        q, scale = empty_fp8_rows(x)
        s = x if residual is None else torch.empty_like(x)
        y = torch.empty_like(x) if return_normed else None
        rc = _lib.lib().mfl_add_rms_norm_fp8(x.data_ptr(), _lib.ptr(residual), weight.data_ptr(), q.data_ptr(), scale.data_ptr(),
                                             _lib.ptr(y), s.data_ptr(), rows, width, eps, dtype, _lib.dtype_code(weight.dtype),
                                             _lib.stream())
    _lib.check(rc, "mfl_add_rms_norm_fp8")
    return q, scale, s, y


def add_rms_norm_backward(dy: Optional[torch.Tensor], ds: Optional[torch.Tensor], s: torch.Tensor, weight: torch.Tensor, eps: float,
                          need_dx: bool = True, need_dw: bool = True) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dx, dw) from the gradients of the normed rows and of the stream ``s``, which is what the forward pass returned; ``dx`` is
    the residual's gradient too.  A row's own sums are in 64 bits, 1 / length, ``dy * weight`` and the sums over the rows in 32, these in the same
    order every time."""
    rows, width, dtype = _check(s, ds, weight)
    if dy is None:  # (nobody used the normed rows)
        return ds if need_dx else None, torch.zeros_like(weight) if need_dw else None
    assert dy.shape == s.shape and dy.dtype == s.dtype and dy.is_contiguous() and dy.device == s.device
    with _lib.on_device_of(s):
        dx = torch.empty_like(s) if need_dx else None
        dw = torch.empty_like(weight) if need_dw else None
        if rows == 0:
            return dx, dw.zero_() if need_dw else None
        lib, ws, size = _lib.lib(), None, 0
        if need_dw:
            size = lib.mfl_add_rms_norm_bwd_workspace(rows, width)
            ws = torch.empty(size, device=s.device, dtype=torch.uint8)
        rc = lib.mfl_add_rms_norm_bwd(dy.data_ptr(), _lib.ptr(ds), s.data_ptr(), weight.data_ptr(), _lib.ptr(dx), _lib.ptr(dw), rows,
                                      width, eps, dtype, _lib.dtype_code(weight.dtype), _lib.ptr(ws), size, _lib.stream())
    _lib.check(rc, "mfl_add_rms_norm_bwd")
    return dx, dw


class _AddRmsNorm(torch.autograd.Function):
    """``fp8``: False, or True for quantised rows in front of the other results; ``normed``: whether the normed rows are among them.
    Without a residual the stream is the input, which the caller has, and is no result."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, fp8, normed):
        ctx.set_materialize_grads(False)
        quantized = ()
        if fp8:
            *quantized, s, y = _forward_fp8(x, residual, weight, eps, normed)
            ctx.mark_non_differentiable(*quantized)
        else:
            y, s = _forward(x, residual, weight, eps)
        ctx.save_for_backward(s, weight)
        ctx.eps, ctx.skip, ctx.normed = eps, len(quantized), normed
        return (*quantized, *((y,) if normed else ()), *((s,) if residual is not None else ()))

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, *grads):
        grads = [None if g is None else _lib.dense(g) for g in grads[ctx.skip:]]
        dy = grads.pop(0) if ctx.normed else None
        ds = grads[0] if grads else None
        need_x, need_residual, need_w = ctx.needs_input_grad[:3]
        # (a saved-tensor hook may hand equal tensors back in other strides)
        s, weight = (_lib.dense(t) for t in ctx.saved_tensors)
        dx, dw = add_rms_norm_backward(dy, ds, s, weight, ctx.eps, need_x or need_residual, need_w)
        return dx if need_x else None, dx if need_residual else None, dw, None, None, None


def _watched(x, residual, weight) -> bool:
    """Whether the call has to be a node of the graph (or something that is watching has to see it)."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        return True
    return not _lib.plain_call()


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, s) of rows along the last dimension, bf16, fp16 or fp32 and dense, up to 32768 wide and
    ``most_rows`` long; ``weight`` in their type or float32.
    Without a ``residual`` (None) the stream ``s`` is ``x`` itself.  Differentiable once in ``x``, ``residual`` and ``weight``."""
    if not _watched(x, residual, weight):
        return _forward(x, residual, weight, eps)
    out = _AddRmsNorm.apply(x, residual, weight, eps, False, True)
    return out if residual is not None else (out[0], x)


def add_rms_norm_fp8(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                     return_normed: bool = False) -> Tuple[torch.Tensor, ...]:
    """(values, scales, s), or with ``return_normed`` (values, scales, s, y): ``add_rms_norm`` on a matrix with the normed rows
    quantised on the way, to what ``quantize_fp8_rows`` makes of ``y``.  ``moe_fused_mlp_fp8`` takes values and scales beside ``y``.
    The quantised rows carry no gradient; the others are differentiable as in ``add_rms_norm``."""
    if not _watched(x, residual, weight):
        q, scale, s, y = _forward_fp8(x, residual, weight, eps, return_normed)
    else:
        q, scale, *rest = _AddRmsNorm.apply(x, residual, weight, eps, True, return_normed)
        y = rest.pop(0) if return_normed else None
        s = rest[0] if rest else x
    return (q, scale, s, y) if return_normed else (q, scale, s)
