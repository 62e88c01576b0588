"""The norm and the whole expert layer where the modules call them: ``fuse_layer`` of the block, ``fuse_norm`` of the decoder layer."""
from types import SimpleNamespace

import pytest
import torch

from qwen3_moe_fused import _lib
from qwen3_moe_fused.fused_mlp import moe_fused_layer, moe_fused_layer_fp8
from qwen3_moe_fused.modular_qwen3_moe_fused import Qwen3MoeFusedSparseMoeBlock
from qwen3_moe_fused.quantize.layer_fp8 import MoeFusedLinearFp8

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _block(dtype=BF16, hidden=256, inter=128, experts=16, k=4, eight=False):
    torch.manual_seed(0)
    block = Qwen3MoeFusedSparseMoeBlock(SimpleNamespace(
        num_experts=experts, num_experts_per_tok=k, norm_topk_prob=True, hidden_size=hidden, moe_intermediate_size=inter,
        hidden_act="silu")).cuda().to(dtype)
    if eight:
        for name in ("gate_proj", "up_proj", "down_proj"):
            setattr(block, name, MoeFusedLinearFp8.from_linear(getattr(block, name)))
    return block


@pytest.fixture
def calls(monkeypatch):
    """Counts the library's calls by name."""
    seen, real = {}, _lib.lib()

    class Counting:
        def __getattr__(self, name):
            f = getattr(real, name)

            def call(*args):
                seen[name] = seen.get(name, 0) + 1
                return f(*args)

            return call

    counting = Counting()
    monkeypatch.setattr(_lib, "lib", lambda: counting)
    return seen


@pytest.mark.parametrize("eight", (False, True))
def test_block_calls_the_layer(calls, eight):
    block = _block(eight=eight)
    x = torch.randn((3, 4, 256), device="cuda", dtype=BF16)
    with torch.no_grad():
        want, want_logits = block(x)
        assert "mfl_moe_layer_fwd" not in calls
        block.fuse_layer = True
        out, logits = block(x)
        assert calls["mfl_moe_layer_fwd"] == 1 and out.shape == x.shape
        projs = (block.gate_proj, block.up_proj, block.down_proj)
        if eight:
            same, _ = moe_fused_layer_fp8(x.view(12, 256), block.gate.weight, *(t for m in projs for t in (m.weight, m.weight_scale_inv)), 4, True)
        else:
            same, _ = moe_fused_layer(x.view(12, 256), block.gate.weight, *(m.weight for m in projs), 4, True)
    assert torch.equal(out.view(12, 256), same)
    # (the tokens whose logits, from 32-bit sums there and 64-bit ones here, rounded alike chose the same experts)
    rows = (logits == want_logits).all(dim=1)
    assert rows.sum() >= 8
    error = (out - want).view(12, 256)[rows].double().norm() / want.view(12, 256)[rows].double().norm()
    assert error <= 6 * 2.0 ** -8  # six roundings more, as counted for the block in the layer's own tests


def test_calls_that_stay_with_the_separate_steps(calls):
    x = torch.randn((1, 4, 256), device="cuda", dtype=BF16)

    def stays(block, x=x):
        block.fuse_layer = True
        block(x)
        assert "mfl_moe_layer_fwd" not in calls

    stays(_block())  # gradients
    with torch.no_grad():
        stays(_block(), torch.randn((1, 17, 256), device="cuda", dtype=BF16))
        block = _block()
        block.keep_routing = True
        stays(block)
        assert block.last_selected.shape == (4, 4)
        for name in ("gate", "gate_proj", "up_proj", "down_proj"):
            block = _block()
            seen = []
            getattr(block, name).register_forward_hook(lambda *a, s=seen: s.append(1))
            stays(block)
            if name in ("gate", "down_proj"):
                assert seen
        block = _block()
        block.fuse_front = False
        stays(block)
        block = _block(eight=True)
        block.up_proj = _block().up_proj
        block.fuse_layer = True
        assert block.whole_layer(x.view(4, 256)) is None
        block = _block(experts=80, k=65)  # more experts a token than the call takes
        block.fuse_layer = True
        assert block.whole_layer(x.view(4, 256)) is None


def _models(dtype=BF16, **changed):
    pytest.importorskip("transformers")
    from transformers import Qwen3MoeConfig

    from qwen3_moe_fused.modular_qwen3_moe_fused import Qwen3MoeFusedModel

    torch.manual_seed(1)
    config = Qwen3MoeConfig(**{**dict(vocab_size=300, hidden_size=128, intermediate_size=96, num_hidden_layers=3,
                                      num_attention_heads=4, num_key_value_heads=2, head_dim=32, moe_intermediate_size=64,
                                      num_experts=8, num_experts_per_tok=2, norm_topk_prob=True, mlp_only_layers=[1]), **changed})
    model = Qwen3MoeFusedModel(config).cuda().to(dtype)
    if type(model.layers[0].mlp) is Qwen3MoeFusedSparseMoeBlock:
        pytest.skip("this transformers release has blocks that return their logits")
    return model


def _set(model, norm=True, layer=False):
    for decoder in model.layers:
        decoder.fuse_norm = norm
        if isinstance(decoder.mlp, Qwen3MoeFusedSparseMoeBlock):
            decoder.mlp.fuse_layer = layer


@pytest.mark.parametrize("batch,seq", ((2, 5), (2, 40)))
def test_model_with_the_fused_norm(calls, batch, seq):
    """fp32, where the stock norm's extra rounding is 2^-24: the same up to a few of those through three layers."""
    model = _models(F32).eval()
    ids = torch.randint(0, 300, (batch, seq), device="cuda")
    with torch.no_grad():
        want = model(input_ids=ids).last_hidden_state
        assert "mfl_add_rms_norm" not in calls
        _set(model)
        got = model(input_ids=ids).last_hidden_state
        assert calls["mfl_add_rms_norm"] == 3  # (the dense layer's norm too)
        torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4)
        _set(model, layer=True)
        few = model(input_ids=ids).last_hidden_state
        assert calls.get("mfl_moe_layer_fwd", 0) == (2 if batch * seq <= 16 else 0)
        torch.testing.assert_close(few, want, rtol=1e-4, atol=1e-4)


def test_gradients_through_the_fused_norm():
    """Two losses.  The mean square of what the last norm returns is mean(s^2) / (mean(s^2) + eps), all but a constant: the gradient that
    arrives, 2 y / n, and its part along y cancel in that norm, and what is left is the roundings of two equal terms, 2^-24 of their size
    a time.  Their size is that of the gradients of a loss whose arriving gradient is as large and does not cancel: the second one, with 2
    y / n moved by a column.  So both are held to 1e-4 of the second one's gradients."""
    model = _models(F32).train()
    ids = torch.randint(0, 300, (2, 24), device="cuda")
    grads = {}
    for norm in (False, True):
        _set(model, norm, layer=True)
        for loss in ("square", "moved"):
            model.zero_grad()
            y = model(input_ids=ids).last_hidden_state
            (y.square() if loss == "square" else y * 2 * y.detach().roll(1, -1)).mean().backward()
            grads[loss, norm] = {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}
    for loss in ("square", "moved"):
        assert grads[loss, False].keys() == grads[loss, True].keys()
        for n, g in grads[loss, False].items():
            assert (grads[loss, True][n] - g).abs().max() <= 1e-4 * grads["moved", False][n].abs().max(), (loss, n)


@pytest.mark.parametrize("tokens", (12, 90))
def test_8_bit_experts_get_the_norms_rows(calls, tokens):
    model = _models(BF16).eval()
    for decoder in model.layers:
        if isinstance(decoder.mlp, Qwen3MoeFusedSparseMoeBlock):
            for name in ("gate_proj", "up_proj", "down_proj"):
                setattr(decoder.mlp, name, MoeFusedLinearFp8.from_linear(getattr(decoder.mlp, name)))
    ids = torch.randint(0, 300, (1, tokens), device="cuda")
    with torch.no_grad():
        want = model(input_ids=ids).last_hidden_state
        _set(model)
        got = model(input_ids=ids).last_hidden_state
        assert calls["mfl_add_rms_norm_fp8"] == 2 and calls["mfl_mlp_fwd_fp8_rows"] == 2
        # bf16 through three layers, each with a rounding more or less, and tokens whose choice of experts that decides
        assert ((got - want).double().norm(dim=-1) / want.double().norm(dim=-1)).median() <= 0.05
        _set(model, layer=True)
        few = model(input_ids=ids).last_hidden_state
        assert calls.get("mfl_moe_layer_fwd", 0) == (2 if tokens <= 16 else 0)
        assert ((few - want).double().norm(dim=-1) / want.double().norm(dim=-1)).median() <= 0.05


def test_generation_with_a_cache():
    pytest.importorskip("transformers")
    from transformers import DynamicCache

    model = _models(F32).eval()
    ids = torch.randint(0, 300, (1, 9), device="cuda")
    _set(model, layer=True)
    with torch.no_grad():
        want = model(input_ids=ids).last_hidden_state
        cache = DynamicCache(config=model.config)
        first = model(input_ids=ids[:, :6], past_key_values=cache, use_cache=True).last_hidden_state
        rest = [model(input_ids=ids[:, i:i + 1], past_key_values=cache, use_cache=True).last_hidden_state for i in range(6, 9)]
    torch.testing.assert_close(torch.cat([first, *rest], 1), want, rtol=1e-4, atol=1e-4)


def test_hooks_keep_the_stock_forward(calls):
    model = _models(F32).eval()
    _set(model, layer=True)
    seen = []
    model.layers[0].post_attention_layernorm.register_forward_hook(lambda *a: seen.append(1))
    model.layers[2].mlp.gate.register_forward_hook(lambda *a: seen.append(2))
    ids = torch.randint(0, 300, (1, 4), device="cuda")
    with torch.no_grad():
        model(input_ids=ids)
    assert sorted(seen) == [1, 2]


@pytest.mark.parametrize("tokens", (12, 90))
def test_a_hook_in_front_of_8_bit_experts_decides_what_they_get(calls, tokens):
    """The rows that the norm quantised are not those that the hook returns."""
    model = _models(BF16, num_hidden_layers=1, mlp_only_layers=[]).eval()
    block = model.layers[0].mlp
    for name in ("gate_proj", "up_proj", "down_proj"):
        setattr(block, name, MoeFusedLinearFp8.from_linear(getattr(block, name)))
    ids = torch.randint(0, 300, (1, tokens), device="cuda")
    _set(model)
    seen = []
    block.register_forward_pre_hook(lambda module, args: (seen.append(args[0]), args[0].roll(1, 1))[1])
    block.register_forward_hook(lambda module, args, out: seen.append(out))
    with torch.no_grad():
        model(input_ids=ids)
        assert "mfl_mlp_fwd_fp8_rows" not in calls
        want = type(block).forward(block, seen[0].roll(1, 1))
    assert torch.equal(seen[1], want)


def test_cached_decoding_calls_the_layer_and_agrees_with_the_stock_steps(calls):
    pytest.importorskip("transformers")
    from transformers import DynamicCache

    model = _models(F32).eval()
    ids = torch.randint(0, 300, (1, 9), device="cuda")
    with torch.no_grad():
        want = model(input_ids=ids).last_hidden_state
        assert "mfl_moe_layer_fwd" not in calls and "mfl_add_rms_norm" not in calls
        _set(model, layer=True)
        cache, parts = DynamicCache(config=model.config), []
        for step, (lo, hi) in enumerate(((0, 6), (6, 7), (7, 8), (8, 9)), 1):
            parts.append(model(input_ids=ids[:, lo:hi], past_key_values=cache, use_cache=True).last_hidden_state)
            assert calls["mfl_moe_layer_fwd"] == 2 * step  # (layers 0 and 2; layer 1 is dense)
            assert calls["mfl_add_rms_norm"] == step
    torch.testing.assert_close(torch.cat(parts, 1), want, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("eight", (False, True))
@pytest.mark.parametrize("watch", ("autocast", "mode"))
def test_autocast_and_watched_calls_keep_the_separate_steps(calls, watch, eight):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watching(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    model = _models(BF16).eval()
    if eight:
        for decoder in model.layers:
            if isinstance(decoder.mlp, Qwen3MoeFusedSparseMoeBlock):
                for name in ("gate_proj", "up_proj", "down_proj"):
                    setattr(decoder.mlp, name, MoeFusedLinearFp8.from_linear(getattr(decoder.mlp, name)))
    ids = torch.randint(0, 300, (1, 7), device="cuda")
    results = []
    with torch.no_grad():
        for norm in (False, True):
            _set(model, norm, layer=norm)
            with torch.autocast("cuda", BF16) if watch == "autocast" else Watching():
                results.append(model(input_ids=ids).last_hidden_state)
    assert not {"mfl_moe_layer_fwd", "mfl_add_rms_norm", "mfl_add_rms_norm_fp8"} & set(calls)
    assert torch.equal(*results)


def test_checkpointed_layers_have_the_same_gradients(calls):
    model = _models(F32).train()
    _set(model)
    ids = torch.randint(0, 300, (2, 24), device="cuda")
    grads = []
    for on in (False, True):
        if on:
            model.gradient_checkpointing_enable({"use_reentrant": False})
        calls.clear()
        model.zero_grad()
        y = model(input_ids=ids).last_hidden_state
        (y * y.detach().roll(1, -1)).mean().backward()
        assert calls["mfl_add_rms_norm"] == (6 if on else 3) and calls["mfl_add_rms_norm_bwd"] == 3
        grads.append({n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None})
    assert grads[0].keys() == grads[1].keys()
    for n, g in grads[0].items():
        torch.testing.assert_close(grads[1][n], g, rtol=1e-5, atol=1e-5 * g.abs().max().item(), msg=n)
