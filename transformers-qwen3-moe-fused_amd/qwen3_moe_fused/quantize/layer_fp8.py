"""Expert projection in 8-bit floating point: e4m3 weights with one fp32 scale per 128 x 128 block, frozen.

``moe_fused_linear_fp8`` is ``moe_fused_linear`` on such weights; its left operands, the rows in the forward pass and the
output's gradient in the backward pass, are quantised row by row on the way (``quantize/fp8.py``), and the gradient is that of
the product with the quantisation taken as the identity.  ``MoeFusedLinearFp8`` is the module: ``weight`` (float8_e4m3fn) and
``weight_scale_inv`` (fp32), the entries that block-quantised checkpoints have, stacked over the experts.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from .. import _lib
from ..grouped_gemm.forward_fp8 import grouped_gemm_forward_fp8, grouped_gemm_forward_transposed_fp8
from ..modular_qwen3_moe_fused import MoeFusedLinear
from .fp8 import FP8, blocks_of, quantize_fp8_blocks


class _GroupedGemmFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, weight_scale, m_sizes):
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(weight, weight_scale, m_sizes)
            ctx.dtype = x.dtype
        return grouped_gemm_forward_fp8(x, weight, weight_scale, m_sizes)

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dy):
        dx = None
        if ctx.needs_input_grad[0]:
            # (a saved-tensor hook may hand equal tensors back in other strides)
            weight, weight_scale, m_sizes = (_lib.dense(t) for t in ctx.saved_tensors)
            dx = grouped_gemm_forward_transposed_fp8(_lib.dense(dy), weight, weight_scale, m_sizes, ctx.dtype)
        return dx, None, None, None


def moe_fused_linear_fp8(input: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                         m_sizes: torch.Tensor) -> torch.Tensor:
    """``moe_fused_linear`` on ``weight`` (E, out, in) float8_e4m3fn with ``weight_scale`` (E, ceil(out / 128),
    ceil(in / 128)) fp32; both frozen.  Differentiable in ``input``."""
    assert not weight.requires_grad and not weight_scale.requires_grad, "8-bit expert weights are frozen"
    # (past autograd only where nobody watches: a tracer has to record the call, a forward-mode level has to refuse it)
    if not (torch.is_grad_enabled() and input.requires_grad) and _lib.plain_call():
        return grouped_gemm_forward_fp8(input, weight, weight_scale, m_sizes)
    return _GroupedGemmFp8.apply(input, weight, weight_scale, m_sizes)


class MoeFusedLinearFp8(MoeFusedLinear):
    """``weight``: floating-point (E, out, in) on the GPU, quantised here; without it the module is empty (zeros) and is to be
    loaded: ``load_state_dict`` takes ``weight`` with ``weight_scale_inv``, or a floating-point ``weight`` on the GPU."""

    def __init__(self, in_features: int, out_features: int, num_experts: int, *, weight: Optional[torch.Tensor] = None,
                 device: Optional[torch.device] = None) -> None:
        super().__init__(in_features, out_features, num_experts, device="meta")
        shape = (num_experts, out_features, in_features)
        if weight is not None:
            assert tuple(weight.shape) == shape
            device = weight.device if device is None else device
            q, scale = quantize_fp8_blocks(weight.detach().contiguous().to(device))
        else:
            q = torch.zeros(shape, device=device, dtype=torch.uint8).view(FP8)
            scale = torch.ones((num_experts, blocks_of(out_features), blocks_of(in_features)), device=device)
        self._set(q, scale)

    @classmethod
    def from_linear(cls, module: MoeFusedLinear) -> "MoeFusedLinearFp8":
        return cls(module.in_features, module.out_features, module.num_experts, weight=module.weight)

    def _set(self, q: torch.Tensor, scale: torch.Tensor) -> None:
        self.weight = nn.Parameter(q, requires_grad=False)
        self.weight_scale_inv = nn.Parameter(scale, requires_grad=False)

    def _apply(self, fn, recurse=True):
        # ``.to(dtype)`` and the like cast every floating-point parameter: the values and scales only change their place
        held = {name: self._parameters.pop(name) for name in ("weight", "weight_scale_inv")}
        try:
            super()._apply(fn, recurse)
            target = fn(torch.empty(0, device=held["weight"].device)).device
            held = {name: nn.Parameter(p.data.to(target) if not p.is_meta or target.type == "meta"
                                       else torch.empty_like(p.data, device=target), requires_grad=False)
                    for name, p in held.items()}
        finally:
            self._parameters.update(held)
        return self

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                              error_msgs) -> None:
        wkey, skey = prefix + "weight", prefix + "weight_scale_inv"
        if wkey not in state_dict:
            if strict:
                missing_keys.append(wkey)
            return
        data, scale = state_dict[wkey], state_dict.get(skey)
        shape, scale_shape = tuple(self.weight.shape), tuple(self.weight_scale_inv.shape)
        if tuple(data.shape) != shape or not data.dtype.is_floating_point:
            error_msgs.append(f"While loading {wkey}: expected a floating-point weight of shape {shape}, got "
                              f"{tuple(data.shape)} {data.dtype}")
        elif data.dtype == FP8:
            if scale is None:
                missing_keys.append(skey)
            elif tuple(scale.shape) != scale_shape or not scale.dtype.is_floating_point:
                error_msgs.append(f"While loading {skey}: expected scales of shape {scale_shape}, got {tuple(scale.shape)} "
                                  f"{scale.dtype}")
            else:
                where = data.device if self.weight.is_meta else self.weight.device
                self._set(data.detach().to(where, copy=True).contiguous(),
                          scale.detach().to(where, torch.float32, copy=True).contiguous())
        elif data.dtype.itemsize < 2 or scale is not None:
            error_msgs.append(f"While loading {wkey}: 8-bit values other than float8_e4m3fn, or scales of a weight that is "
                              f"{data.dtype}, are not taken")
        elif not (data.is_cuda or self.weight.is_cuda):
            error_msgs.append(f"While loading {wkey}: a {data.dtype} weight is quantised on the GPU: move it or the module there")
        else:
            self._set(*quantize_fp8_blocks(data.detach().to(self.weight.device if self.weight.is_cuda else data.device).contiguous()))

    def reset_parameters(self) -> None:
        """Values and scales come from a checkpoint or from another module."""

    def forward(self, x: torch.Tensor, m_sizes: torch.Tensor) -> torch.Tensor:
        return moe_fused_linear_fp8(x, self.weight, self.weight_scale_inv, m_sizes)

    _own_forward = forward
