"""Fused MoE modules (reference: qwen3_moe_fused/modular_qwen3_moe_fused.py).

``MoeFusedLinear`` keeps all experts of one projection in a single (E, out, in) parameter and
applies them with one grouped GEMM; ``Qwen3MoeFusedSparseMoeBlock`` is the whole sparse MLP:
router -> softmax/top-k -> stable expert sort -> gate/up GEMMs -> SiLU*mul -> down GEMM ->
un-sort + routing-weighted sum.  Parameter names and shapes match the reference so state dicts
load unchanged.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import nn

from . import _lib
from .functional import moe_fused_linear
from .kernels.routing import combine_rows, gather_rows, route_and_sort, router_has_a_kernel, router_linear
from .kernels.silu_mul import silu_mul


def moe_fused_kaiming_uniform_(weight: torch.Tensor) -> None:
    """Kaiming-uniform over in_features with gain a = sqrt(5), as nn.Linear initialises
    (modular_qwen3_moe_fused.py:21-26): U(-b, b) with b = sqrt(15 / in_features)."""
    fan_in = weight.shape[-1]
    limit = math.sqrt(15.0 / fan_in)
    with torch.no_grad():
        weight.uniform_(-limit, limit)


class MoeFusedLinear(nn.Module):
    __constants__ = ["in_features", "out_features", "num_experts"]

    def __init__(self, in_features: int, out_features: int, num_experts: int,
                 device: Optional[torch.device] = None, dtype: Optional[torch.dtype] = None) -> None:
        super().__init__()
        self.in_features, self.out_features, self.num_experts = in_features, out_features, num_experts
        self.weight = nn.Parameter(torch.empty((num_experts, out_features, in_features), device=device, dtype=dtype))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        moe_fused_kaiming_uniform_(self.weight)

    def forward(self, input: torch.Tensor, m_sizes: torch.Tensor) -> torch.Tensor:
        return moe_fused_linear(input, self.weight, m_sizes)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, num_experts={self.num_experts}"

    # what the block's one call stands in for: a class whose forward has been replaced runs on the separate steps
    _own_forward = forward


def route_tokens(block, hidden_2d: torch.Tensor, router_logits: Optional[torch.Tensor] = None):
    """Router half of the block, shared with the fast-LoRA forward: returns
    (router_logits, routing_weights (T,k), m_sizes, sort_idx, inv_sort_idx)."""
    if router_logits is None:
        router_logits = block.gate(hidden_2d)
    routing_weights, selected, m_sizes, sort_idx, inv_sort_idx = route_and_sort(
        router_logits.contiguous(), block.num_selected, block.norm_topk_prob, hidden_2d.dtype, block.num_experts)
    if getattr(block, "keep_routing", False):
        block.last_selected = selected  # (T, k) expert ids of this call, as the top-k kernel wrote them
    return router_logits, routing_weights, m_sizes, sort_idx, inv_sort_idx


class Qwen3MoeFusedRouter(nn.Linear):
    """The block's ``gate``: a plain bias-free linear layer (modular_qwen3_moe_fused.py:72 of the
    reference) under a class name of its own, so that transformers releases that collect
    ``router_logits`` with a forward hook on the router module (instead of from the block's return
    value, as the reference's release did) have a class to hook: its output is the raw logits."""

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        if torch.jit.is_scripting():  # (compiled from source, where neither the kernel nor super() can be called)
            return nn.functional.linear(input, self.weight, self.bias)
        else:
            out = None
            if self.bias is None and router_has_a_kernel(input, self.weight):
                out = router_linear(input, self.weight)
            return super().forward(input) if out is None else out

    _own_forward = forward  # (as in MoeFusedLinear)


def _stands_for_itself(module: nn.Module) -> bool:
    """Whether a module's call is its class's forward and nothing else: no hooks, no replaced forward."""
    return not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks
                or "forward" in module.__dict__ or type(module).forward is not type(module)._own_forward)


def _defined_forward(cls: type):
    """A foreign class's forward, or None where somebody outside its package has put another in its place.  (The package's own decorators
    are part of it.)"""
    forward = cls.forward
    at = getattr(forward, "__globals__", {}).get("__name__", "")
    return forward if at.split(".")[0] == cls.__module__.split(".")[0] else None


class Qwen3MoeFusedSparseMoeBlock(nn.Module):
    """``config`` needs: num_experts, num_experts_per_tok, norm_topk_prob, hidden_size,
    moe_intermediate_size, hidden_act == "silu" (a transformers ``Qwen3MoeConfig`` has them)."""

    def __init__(self, config) -> None:
        super().__init__()
        assert config.hidden_act == "silu"
        self.num_experts = config.num_experts
        self.num_selected = config.num_experts_per_tok
        self.norm_topk_prob = config.norm_topk_prob
        self.hidden_size = config.hidden_size
        self.moe_intermediate_size = config.moe_intermediate_size
        self.gate = Qwen3MoeFusedRouter(self.hidden_size, self.num_experts, bias=False)
        self.gate_proj = MoeFusedLinear(self.hidden_size, self.moe_intermediate_size, self.num_experts)
        self.up_proj = MoeFusedLinear(self.hidden_size, self.moe_intermediate_size, self.num_experts)
        self.down_proj = MoeFusedLinear(self.moe_intermediate_size, self.hidden_size, self.num_experts)

    # gather + gate_proj + up_proj + SiLU-mul as one kernel when both projections are plain (or
    # plain 4-bit) expert matrices in bf16; set to False to call the two modules one by one
    fuse_front = True
    # with fuse_front: set to True for the three projections as one node of the autograd graph, whose backward runs
    # the gated unit's backward inside the down projection's input gradient (dh is never written: 50 MB less memory
    # at 32768 routed rows).  Off by default: the kernel's epilogue then does the unit's arithmetic with the matrix
    # units idle, and a training step of the block takes 1.62-1.67 ms instead of 1.58-1.63 ms.
    fuse_backward = False
    # set to True for calls of up to 16 tokens without gradients as the whole layer in two launches (fused_mlp.moe_fused_layer; bf16,
    # fp16, fp32 and 8-bit expert matrices; 128 experts in bf16: one token 26 us a call against 45, 16 tokens 135 against 146).  Off
    # by default: the results are not those of the separate steps bit for bit, since less is rounded on the way.
    fuse_layer = False
    # set to True to keep the expert ids of the last call in ``last_selected`` (tests read the block's own routing)
    keep_routing = False

    def _fused_front(self, tokens, m_sizes, sort_idx, inv_sort_idx) -> Optional[torch.Tensor]:
        from .fused_mlp import moe_fused_glu, moe_fused_glu_4bit, moe_fused_glu_fp8
        from .quantize.layer import MoeFusedLinear4bit
        from .quantize.layer_fp8 import MoeFusedLinearFp8

        gate, up = self.gate_proj, self.up_proj
        if type(gate) is MoeFusedLinearFp8 and type(up) is MoeFusedLinearFp8:
            return moe_fused_glu_fp8(tokens, gate.weight, gate.weight_scale_inv, up.weight, up.weight_scale_inv, m_sizes,
                                     sort_idx, inv_sort_idx, self.num_selected)
        if tokens.dtype != torch.bfloat16 or type(gate) is not type(up):
            return None
        if type(gate) is MoeFusedLinear:
            if gate.weight.dtype != torch.bfloat16 or up.weight.dtype != torch.bfloat16:
                return None
            return moe_fused_glu(tokens, gate.weight, up.weight, m_sizes, sort_idx, inv_sort_idx, self.num_selected)
        if type(gate) is MoeFusedLinear4bit:
            for proj in (gate, up):
                if getattr(proj.weight, "quant_state", None) is None or proj.compute_dtype not in (None, torch.bfloat16):
                    return None
            return moe_fused_glu_4bit(tokens, gate.weight, up.weight, m_sizes, sort_idx, inv_sort_idx,
                                      self.num_selected)
        return None

    def whole_layer(self, tokens: torch.Tensor, residual: Optional[torch.Tensor] = None, norm_weight: Optional[torch.Tensor] = None,
                    eps: float = 1e-6) -> Optional[Tuple[torch.Tensor, torch.Tensor]]:
        """(out, router logits) of ``moe_fused_layer`` on the block's weights, or None where ``fuse_layer`` is off or the call is not one
        for it: more tokens, gradients, other kinds of weights, modules that somebody watches."""
        from .fused_mlp import LAYER_TOKENS, moe_fused_layer, moe_fused_layer_fp8
        from .quantize.layer_fp8 import MoeFusedLinearFp8

        if not (self.fuse_layer and self.fuse_front) or self.keep_routing or not 0 < tokens.shape[0] <= LAYER_TOKENS:
            return None
        gate, projs = self.gate, (self.gate_proj, self.up_proj, self.down_proj)
        kind = type(projs[0])
        if (type(gate) is not Qwen3MoeFusedRouter or gate.bias is not None or kind not in (MoeFusedLinear, MoeFusedLinearFp8)
                or any(type(m) is not kind for m in projs) or not all(map(_stands_for_itself, (gate, *projs)))):
            return None
        if torch.nn.modules.module._has_any_global_hook() or not _lib.plain_call() or torch.is_autocast_enabled("cuda"):
            return None
        same = [gate.weight] + ([p.weight for p in projs] if kind is MoeFusedLinear else [])
        same += [t for t in (residual, norm_weight) if t is not None]
        if not tokens.is_cuda or tokens.dtype not in (torch.bfloat16, torch.float16, torch.float32):
            return None
        if self.num_experts > 1024 or self.num_selected > 64 or projs[0].out_features > 1 << 17:  # (the call's limits)
            return None
        if any(t.dtype != tokens.dtype or t.device != tokens.device or not t.is_contiguous() for t in same):
            return None
        if torch.is_grad_enabled() and any(t.requires_grad for t in (tokens, *same)):
            return None
        if kind is MoeFusedLinear:
            return moe_fused_layer(tokens, gate.weight, *(m.weight for m in projs), self.num_selected, self.norm_topk_prob,
                                   residual, norm_weight, eps)
        pairs = [t for m in projs for t in (m.weight, m.weight_scale_inv)]
        return moe_fused_layer_fp8(tokens, gate.weight, *pairs, self.num_selected, self.norm_topk_prob, residual, norm_weight, eps)

    def _fused_mlp(self, tokens, m_sizes, sort_idx, inv_sort_idx, quantized=None) -> Optional[torch.Tensor]:
        """The three projections as one node of the graph when all are plain bf16 expert matrices and a gradient
        will be asked for: the backward then runs the gated unit's backward inside the down projection's input
        gradient.  Without gradients the front half and the down projection are the same two launches anyway."""
        from .fused_mlp import moe_fused_mlp, moe_fused_mlp_fp8
        from .quantize.layer_fp8 import MoeFusedLinearFp8

        projs = (self.gate_proj, self.up_proj, self.down_proj)
        if all(type(p) is MoeFusedLinearFp8 for p in projs):
            # 8-bit floating point: with the down projection in the call the gated unit's result is written in 8 bits only
            down = projs[2]
            if (down._forward_hooks or down._forward_pre_hooks or down._backward_hooks or down._backward_pre_hooks
                    or "forward" in down.__dict__ or MoeFusedLinearFp8.forward is not MoeFusedLinearFp8._own_forward
                    or torch.nn.modules.module._has_any_global_hook()):
                return None
            weights = [t for p in projs for t in (p.weight, p.weight_scale_inv)]
            return moe_fused_mlp_fp8(tokens, *weights, m_sizes, sort_idx, inv_sort_idx, self.num_selected, quantized)
        if not self.fuse_backward or tokens.dtype != torch.bfloat16 or not torch.is_grad_enabled():
            return None
        if any(type(p) is not MoeFusedLinear or p.weight.dtype != torch.bfloat16 for p in projs):
            return None
        if not (tokens.requires_grad or any(p.weight.requires_grad for p in projs)):
            return None
        return moe_fused_mlp(tokens, self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight, m_sizes,
                             sort_idx, inv_sort_idx, self.num_selected)

    # Rows up to which the block is one library call.  Beyond, the kernels hide the host's time (131072 rows on packed
    # weights: 1638 us either way), and the one buffer of all intermediates, 740 MB there, once cost a new state's first pass
    # more than the steps' own tensors (1870 against 1733 us).  Measured again at hidden 1024 to 4096 it did not (1730 either
    # way; buffers of 96 MB to 1.4 GB even or up to 3 % ahead), so the line is one of rows, not of the buffer's bytes.
    _ONE_CALL_ROWS = 65536

    def _one_call(self, tokens: torch.Tensor, logits: torch.Tensor) -> Optional[torch.Tensor]:
        """Everything behind the router projection as one library call, where the three projections are plain expert
        matrices in the tokens' type (both ways), or plain packed ones (without gradients)."""
        from .fused_mlp import moe_block_4bit, moe_block_of
        from .quantize.layer import MoeFusedLinear4bit

        gate, up, down = self.gate_proj, self.up_proj, self.down_proj
        kind = type(gate)
        if kind not in (MoeFusedLinear, MoeFusedLinear4bit) or type(up) is not kind or type(down) is not kind:
            return None
        if tokens.shape[0] == 0 or self.num_experts > 1024:
            return None
        if tokens.shape[0] * self.num_selected > self._ONE_CALL_ROWS:
            return None
        # Hooks and replaced forwards run on the separate steps.  (In bf16 and on packed weights those call the down
        # projection; what gate and up do is the fused front's, which calls neither unless ``fuse_front`` is off.)
        if kind.forward is not kind._own_forward:
            return None
        for proj in (gate, up, down):
            if (proj._forward_hooks or proj._forward_pre_hooks or proj._backward_hooks or proj._backward_pre_hooks
                    or "forward" in proj.__dict__):
                return None
        if torch.nn.modules.module._has_any_global_hook() or not _lib.plain_call():
            return None
        assert logits.shape[-1] == self.num_experts
        weights = (gate.weight, up.weight, down.weight)
        if kind is MoeFusedLinear:
            if tokens.dtype not in (torch.bfloat16, torch.float32):
                return None
            for w in weights:
                if w.dtype != tokens.dtype or not w.is_contiguous() or w.device != tokens.device:
                    return None
            out, ws = moe_block_of(tokens, logits, *weights, self.num_selected, self.norm_topk_prob)
        else:
            if tokens.dtype != torch.bfloat16 or (torch.is_grad_enabled() and (tokens.requires_grad or logits.requires_grad)):
                return None
            for proj in (gate, up, down):
                if getattr(proj.weight, "quant_state", None) is None or proj.compute_dtype not in (None, torch.bfloat16):
                    return None
            if not down.compute_type_is_set:  # as its own forward does on the first call
                down.set_compute_type(tokens)
                down.compute_type_is_set = True
            out, ws = moe_block_4bit(tokens, logits, *weights, self.num_selected, self.norm_topk_prob)
        if out is not None and self.keep_routing:
            n, k = tokens.shape[0], self.num_selected
            self.last_selected = ws[:n * k * 8].view(torch.int64).view(n, k).clone()  # (not the whole workspace)
        return out

    def forward(self, hidden_states: torch.Tensor, quantized: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                ) -> Tuple[torch.Tensor, torch.Tensor]:
        """``quantized``: what ``add_rms_norm_fp8`` made of the hidden states already, which 8-bit experts then do not make again."""
        batch, seq, hidden = hidden_states.shape
        tokens = hidden_states.reshape(batch * seq, hidden).contiguous()
        whole = self.whole_layer(tokens) if self.fuse_layer else None
        if whole is not None:
            return whole[0].view(batch, seq, hidden), whole[1]
        if self.fuse_front and not self.fuse_backward:
            router_logits = self.gate(tokens)
            out = self._one_call(tokens, router_logits.contiguous())
            if out is not None:
                return out.view(batch, seq, hidden), router_logits
            # (the separate steps take the logits as they are: the router is not called twice)
            routed = route_tokens(self, tokens, router_logits)
        else:
            routed = route_tokens(self, tokens)
        router_logits, routing_weights, m_sizes, sort_idx, inv_sort_idx = routed

        y = self._fused_mlp(tokens, m_sizes, sort_idx, inv_sort_idx, quantized) if self.fuse_front else None
        if y is None:
            h = self._fused_front(tokens, m_sizes, sort_idx, inv_sort_idx) if self.fuse_front else None
            if h is None:
                # every token once per selected expert, rows grouped by expert
                x = gather_rows(tokens, sort_idx, self.num_selected, inv_sort_idx)
                h = silu_mul(self.gate_proj(x, m_sizes), self.up_proj(x, m_sizes))
            y = self.down_proj(h, m_sizes)
        out = combine_rows(y, inv_sort_idx, routing_weights, sort_idx)
        return out.view(batch, seq, hidden), router_logits

    _own_forward = forward


def _hf_subclasses():
    """Model-level wiring (decoder layer / model / causal LM with the fused block swapped in),
    built on demand so that importing this module does not import transformers."""
    import inspect

    from transformers.models.qwen3_moe.modeling_qwen3_moe import (Qwen3MoeDecoderLayer, Qwen3MoeForCausalLM, Qwen3MoeMLP,
                                                                  Qwen3MoeModel, Qwen3MoeRMSNorm, Qwen3MoeSparseMoeBlock)

    # The reference was written against a transformers revision whose sparse block returns
    # (hidden_states, router_logits) (modular_qwen3_moe_fused.py:1,118); later releases return the
    # hidden states alone and the decoder layer adds them to the residual as they come.
    block_cls = Qwen3MoeFusedSparseMoeBlock
    if inspect.signature(Qwen3MoeSparseMoeBlock.forward).return_annotation is torch.Tensor:
        class _TensorBlock(Qwen3MoeFusedSparseMoeBlock):
            def forward(self, hidden_states: torch.Tensor,
                        quantized: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> torch.Tensor:
                # (a forward that somebody has put in the place of the block's takes the hidden states alone)
                given = () if quantized is None else (quantized,)
                return super().forward(hidden_states, *given)[0]

            _own_forward = forward

        block_cls = _TensorBlock

    stock_forward = inspect.signature(Qwen3MoeDecoderLayer.forward)
    stock_layer, stock_norm = _defined_forward(Qwen3MoeDecoderLayer), _defined_forward(Qwen3MoeRMSNorm)

    class Qwen3MoeFusedDecoderLayer(Qwen3MoeDecoderLayer):
        # set to True for the addition behind the attention and the norm in front of the experts as one kernel (kernels/norm.py), both
        # ways, with 8-bit experts also to the rows that they multiply; with the block's ``fuse_layer`` a call of up to 16 tokens without
        # gradients is two launches from there to the layer's result.  Off by default: the stock norm rounds once more.
        fuse_norm = False

        def __init__(self, config, layer_idx: int) -> None:
            super().__init__(config, layer_idx)
            sparse = (layer_idx not in config.mlp_only_layers and config.num_experts > 0
                      and (layer_idx + 1) % config.decoder_sparse_step == 0)
            self.mlp = (block_cls(config) if sparse
                        else Qwen3MoeMLP(config, intermediate_size=config.intermediate_size))

        def forward(self, hidden_states: torch.Tensor, *args, **kwargs):
            norm = self.post_attention_layernorm
            # (of releases whose block returns its logits the layer's results are another matter: their forward stays theirs)
            if (not self.fuse_norm or block_cls is Qwen3MoeFusedSparseMoeBlock or type(norm) is not Qwen3MoeRMSNorm
                    or norm._forward_hooks or norm._forward_pre_hooks or norm._backward_hooks or norm._backward_pre_hooks
                    or "forward" in norm.__dict__ or Qwen3MoeRMSNorm.forward is not stock_norm
                    or Qwen3MoeDecoderLayer.forward is not stock_layer
                    or torch.nn.modules.module._has_any_global_hook() or not _lib.plain_call()):
                return super().forward(hidden_states, *args, **kwargs)
            given = stock_forward.bind(self, hidden_states, *args, **kwargs)
            given.apply_defaults()
            rest = {k: v for k, v in list(given.arguments.items())[2:] if k != "kwargs"}
            rest.update(given.arguments.get("kwargs", {}))
            attention = self.self_attn(hidden_states=self.input_layernorm(hidden_states), **rest)[0]
            return self._feed_forward(attention, hidden_states, norm)

        def _feed_forward(self, x: torch.Tensor, residual: torch.Tensor, norm: nn.Module) -> torch.Tensor:
            from .kernels.norm import WIDTH, add_rms_norm, add_rms_norm_fp8, most_rows
            from .quantize.layer_fp8 import MoeFusedLinearFp8

            weight, eps = norm.weight, norm.variance_epsilon
            if (not x.is_cuda or x.dtype != residual.dtype or x.shape != residual.shape or x.device != residual.device
                    or x.dtype not in (torch.bfloat16, torch.float16, torch.float32) or weight.dtype not in (x.dtype, torch.float32)
                    or x.shape[-1] > WIDTH or x.numel() > most_rows(x.shape[-1]) * x.shape[-1]
                    or torch.is_autocast_enabled("cuda")):
                s = residual + x
                return s + self.mlp(norm(s))
            x, residual = _lib.dense(x), _lib.dense(residual)
            if isinstance(self.mlp, Qwen3MoeFusedSparseMoeBlock) and x.numel():
                flat, flat_residual = x.view(-1, x.shape[-1]), residual.view(-1, x.shape[-1])
                # (who watches the block's call, or has replaced it, may change what it is given)
                own = _stands_for_itself(self.mlp) and (Qwen3MoeFusedSparseMoeBlock.forward
                                                        is Qwen3MoeFusedSparseMoeBlock._own_forward)
                whole = self.mlp.whole_layer(flat, flat_residual, weight, eps) if own else None
                if whole is not None:
                    return whole[0].view(x.shape)
                if own and type(self.mlp.gate_proj) is MoeFusedLinearFp8:
                    values, scales, s, y = add_rms_norm_fp8(flat, flat_residual, weight, eps, return_normed=True)
                    return s.view(x.shape) + self.mlp(y.view(x.shape), quantized=(values, scales))
            y, s = add_rms_norm(x, residual, weight, eps)
            return s + self.mlp(y)

    # Releases that record outputs through forward hooks take the router logits from the stock router
    # class; the fused block's router is hooked the same way (output_router_logits, the auxiliary
    # load-balancing loss).  Older releases read them from the block's return value and have no table.
    record = {}
    if isinstance(getattr(Qwen3MoeModel, "_can_record_outputs", None), dict):
        # the recorder class has lived in two places; without it the model classes still build and the router
        # logits come from the block's return value only
        OutputRecorder = None
        for module in ("transformers.utils.output_capturing", "transformers.utils.generic"):
            try:
                OutputRecorder = getattr(__import__(module, fromlist=["OutputRecorder"]), "OutputRecorder")
                break
            except (ImportError, AttributeError):
                continue
        if OutputRecorder is not None:
            record = {"_can_record_outputs": {**Qwen3MoeModel._can_record_outputs,
                                              "router_logits": OutputRecorder(Qwen3MoeFusedRouter, index=0)}}

    class Qwen3MoeFusedModel(Qwen3MoeModel):
        locals().update(record)

        def __init__(self, config) -> None:
            super().__init__(config)
            self.layers = nn.ModuleList(Qwen3MoeFusedDecoderLayer(config, i) for i in range(config.num_hidden_layers))

    class Qwen3MoeFusedForCausalLM(Qwen3MoeForCausalLM):
        locals().update(record)

        def __init__(self, config) -> None:
            super().__init__(config)
            self.model = Qwen3MoeFusedModel(config)

    return Qwen3MoeFusedDecoderLayer, Qwen3MoeFusedModel, Qwen3MoeFusedForCausalLM


def __getattr__(name: str):
    names = ("Qwen3MoeFusedDecoderLayer", "Qwen3MoeFusedModel", "Qwen3MoeFusedForCausalLM")
    if name in names:
        classes = dict(zip(names, _hf_subclasses()))
        globals().update(classes)
        return classes[name]
    raise AttributeError(name)
