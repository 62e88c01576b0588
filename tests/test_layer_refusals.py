"""Calls of the norm and of the whole expert layer that are refused before anything reaches a device."""
import ctypes

import pytest
import torch

from qwen3_moe_fused import _lib
from qwen3_moe_fused.fused_mlp import moe_fused_layer, moe_fused_layer_fp8
from qwen3_moe_fused.kernels.norm import add_rms_norm, add_rms_norm_backward, add_rms_norm_fp8, most_rows
from qwen3_moe_fused.quantize.fp8 import check_fp8_rows

BF16, F32, F16 = _lib.BF16, _lib.F32, _lib.F16
NULL, SHAPE, DTYPE, ALIGN, WORKSPACE, LIMIT = -1, -2, -3, -4, -5, -7


@pytest.fixture
def p():
    buf = ctypes.create_string_buffer(8192)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    yield at
    del buf


def test_norm(p):
    lib = _lib.lib()

    def fwd(x=p, r=None, w=p, y=p, s=p, rows=4, h=8, eps=1e-6, dt=BF16, wdt=BF16):
        return lib.mfl_add_rms_norm(x, r, w, y, s, rows, h, eps, dt, wdt, None)

    def fp8(x=p, r=None, w=p, y=None, s=p, rows=4, h=8, eps=1e-6, dt=BF16, wdt=BF16, q=p, scale=p):
        return lib.mfl_add_rms_norm_fp8(x, r, w, q, scale, y, s, rows, h, eps, dt, wdt, None)

    for call in (fwd, fp8):
        assert call(x=None) == NULL and call(w=None) == NULL and call(r=p, s=None) == NULL
        assert call(rows=-1) == SHAPE and call(h=0) == SHAPE and call(eps=-1.0) == SHAPE
        assert call(eps=float("nan")) == SHAPE and call(eps=float("inf")) == SHAPE
        assert call(h=32769) == LIMIT and call(rows=2 ** 40) == LIMIT
        assert call(dt=7) == DTYPE and call(wdt=F16) == DTYPE and call(wdt=9) == DTYPE and call(dt=F32) == DTYPE
        assert call(x=p + 1) == ALIGN and call(r=p + 1) == ALIGN and call(s=p + 1) == ALIGN and call(y=p + 1) == ALIGN
        assert call(w=p + 2, wdt=F32) == ALIGN
        assert call(rows=0, x=None, w=None) == 0
    assert fwd(y=None) == NULL and fp8(q=None) == NULL and fp8(scale=None) == NULL and fp8(q=p + 8) == ALIGN


def test_norm_backward(p):
    lib = _lib.lib()

    def bwd(dy=p, ds=None, s=p, w=p, dx=p, dw=p, rows=4, h=8, eps=1e-6, dt=BF16, wdt=BF16, ws=p, size=4096):
        return lib.mfl_add_rms_norm_bwd(dy, ds, s, w, dx, dw, rows, h, eps, dt, wdt, ws, size, None)

    assert lib.mfl_add_rms_norm_bwd_workspace(4, 8) >= 8 * 4
    for bad in ((0, 8), (-1, 8), (4, 0), (4, 32769)):
        assert lib.mfl_add_rms_norm_bwd_workspace(*bad) == 0
    assert bwd(dy=None) == NULL and bwd(s=None) == NULL and bwd(w=None) == NULL
    assert bwd(rows=-1) == SHAPE and bwd(h=-3) == SHAPE and bwd(h=40000) == LIMIT
    assert bwd(dt=5) == DTYPE and bwd(wdt=F16) == DTYPE
    assert bwd(dy=p + 1) == ALIGN and bwd(ds=p + 1) == ALIGN and bwd(dx=p + 1) == ALIGN and bwd(dw=p + 1) == ALIGN
    assert bwd(ws=p + 4) == ALIGN and bwd(ws=None) == WORKSPACE and bwd(size=16) == WORKSPACE
    assert bwd(dx=None, dw=None) == 0 and bwd(rows=0, dw=None, dy=None, s=None, w=None) == 0


def _call(p, **changed):
    fields = {"x": p, "residual": None, "norm_weight": None, "router": p, "w_gate": p, "w_up": p, "w_down": p, "s_gate": None,
              "s_up": None, "s_down": None, "T": 2, "E": 4, "k": 2, "H": 16, "I": 8, "renorm": 1, "dtype": BF16, "eps": 1e-6}
    assert not set(changed) - set(fields)
    return _lib.MoeLayer(**{**fields, **changed})


def test_layer(p):
    lib = _lib.lib()

    def run(out=p, logits=p, ws=p, size=8192, **changed):
        return lib.mfl_moe_layer_fwd(_call(p, **changed), out, logits, ws, size, None)

    assert lib.mfl_moe_layer_fwd(None, p, p, p, 8192, None) == NULL
    for name in ("x", "router", "w_gate", "w_up", "w_down"):
        assert run(**{name: None}) == NULL and run(**{name: p + 1}) == ALIGN
    assert run(out=None) == NULL and run(logits=None) == NULL and run(out=p + 1) == ALIGN and run(logits=p + 1) == ALIGN
    assert run(residual=p) == NULL  # without a norm there is nothing to add it for
    assert run(s_gate=p) == NULL and run(s_gate=p, s_up=p) == NULL and run(s_gate=p, s_up=p + 2, s_down=p) == ALIGN
    assert run(residual=p + 1, norm_weight=p) == ALIGN and run(norm_weight=p + 1) == ALIGN
    for name in ("E", "k", "H", "I"):
        assert run(**{name: 0}) == SHAPE
    assert run(T=-1) == SHAPE and run(k=5) == SHAPE and run(norm_weight=p, eps=-1.0) == SHAPE
    assert run(T=17) == LIMIT and run(E=1025) == LIMIT and run(E=100, k=65) == LIMIT and run(H=2 ** 24 + 1) == LIMIT
    assert run(I=2 ** 24 + 1) == LIMIT and run(dtype=9) == DTYPE
    assert run(ws=None) == WORKSPACE and run(size=100) == WORKSPACE and run(ws=p + 16) == ALIGN
    assert run(T=0, x=None, ws=None, size=0, out=None, logits=None) == 0


def test_layer_workspace(p):
    size = lambda **c: _lib.lib().mfl_moe_layer_workspace(_call(p, **c))  # noqa: E731
    assert _lib.lib().mfl_moe_layer_workspace(None) == 0
    plain = size()
    assert plain >= 2 * 2 * 16 * 4  # the gated unit's rows, fp32
    assert size(norm_weight=p) >= plain + 2 * 16 * 2 and size(norm_weight=p, residual=p) >= size(norm_weight=p) + 2 * 16 * 2
    assert size(s_gate=p, s_up=p, s_down=p) >= plain + 2 * 128 * 2
    for bad in ({"T": 0}, {"T": 17}, {"E": 0}, {"k": 5}, {"H": 0}, {"I": -1}, {"E": 1025}, {"dtype": 4}):
        assert size(**bad) == 0


# ---- the Python side, with a stand-in for the library and for the device ----------------------------------------------------------

class LibraryCalled(Exception):
    pass


class _StandIn:
    def __getattr__(self, name):
        if name.endswith("_workspace"):
            return lambda *args: 256

        def call(*args):
            raise LibraryCalled(name)

        return call


@pytest.fixture
def on_host(monkeypatch):
    """Host tensors pass for device tensors: what remains are the checks of shapes, types, devices and strides."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: t.device.type == "cpu"))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: {"cpu": 0, "meta": 1}[t.device.type])
    monkeypatch.setattr(_lib, "lib", lambda: _StandIn())
    monkeypatch.setattr(_lib, "stream", lambda: 0)
    monkeypatch.setattr(_lib, "on_device_of", lambda t: _lib._here)


def _strided(t):
    return torch.empty((*t.shape[:-1], t.shape[-1] + 1), dtype=t.dtype)[..., :-1]


BAD = [_strided, torch.Tensor.double, lambda t: t.to("meta"), lambda t: t[..., :-1].contiguous(), lambda t: t.to(torch.float16)]


@pytest.mark.parametrize("form", (add_rms_norm, add_rms_norm_fp8))
def test_norm_operands(on_host, form):
    good = [torch.zeros((3, 8), dtype=torch.bfloat16), torch.zeros((3, 8), dtype=torch.bfloat16), torch.ones(8, dtype=torch.bfloat16)]
    with pytest.raises(LibraryCalled):
        form(*good)
    with pytest.raises(LibraryCalled):
        form(good[0], None, good[2].float())
    for which in range(3):
        for bad in BAD:
            args = list(good)
            args[which] = bad(args[which])
            if which == 2 and bad is _strided:
                args[which] = torch.ones(16, dtype=torch.bfloat16)[::2]
            with pytest.raises((AssertionError, TypeError)):
                form(*args)
    with pytest.raises(AssertionError):  # (a residual is not spread over rows)
        form(good[0], good[1][:1], good[2])
    if form is add_rms_norm_fp8:
        with pytest.raises(AssertionError):
            form(good[0].view(3, 1, 8), None, good[2])


def test_norm_on_the_host():
    x, w = torch.zeros((3, 8)), torch.ones(8)
    for call in (lambda: add_rms_norm(x, None, w), lambda: add_rms_norm_fp8(x, None, w), lambda: add_rms_norm_backward(x, None, x, w, 1e-6)):
        with pytest.raises(AssertionError):
            call()


def _layer_args(eight, t=3, e=4, h=16, i=8):
    dt = torch.bfloat16
    args = [torch.zeros((t, h), dtype=dt), torch.zeros((e, h), dtype=dt)]
    for shape in ((e, i, h), (e, i, h), (e, h, i)):
        if eight:
            args += [torch.zeros(shape, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones((e, 1, 1))]
        else:
            args.append(torch.zeros(shape, dtype=dt))
    return args


@pytest.mark.parametrize("eight", (False, True))
def test_layer_operands(on_host, eight):
    form = moe_fused_layer_fp8 if eight else moe_fused_layer
    good = _layer_args(eight)
    norm, residual = torch.ones(16, dtype=torch.bfloat16), torch.zeros((3, 16), dtype=torch.bfloat16)
    with pytest.raises(LibraryCalled):
        form(*good, 2, True)
    with pytest.raises(LibraryCalled):
        form(*good, 2, True, residual=residual, norm_weight=norm)
    for which in range(len(good)):
        for bad in (_strided, torch.Tensor.double, lambda t: t.to("meta")):
            args = list(good)
            if args[which].dtype.itemsize == 1 and bad is _strided:
                args[which] = _strided(args[which].view(torch.uint8)).view(torch.float8_e4m3fn)
            else:
                args[which] = bad(args[which])
            if torch.equal(torch.tensor(args[which].stride()), torch.tensor(good[which].stride())) and args[which].dtype == good[which].dtype \
                    and args[which].device == good[which].device:
                continue
            with pytest.raises((AssertionError, TypeError)):
                form(*args, 2, True)
    with pytest.raises(AssertionError):
        form(*good, 2, True, residual=residual)
    with pytest.raises(AssertionError):
        form(*good, 2, True, norm_weight=norm[:8])
    with pytest.raises(AssertionError):
        form(*good, 2, True, norm_weight=norm, residual=residual[:1])
    for k in (0, 5, -1):
        with pytest.raises(AssertionError):
            form(*good, k, True)
    with pytest.raises(AssertionError):
        form(*_layer_args(eight, t=17), 2, True)
    # (it serves: there is no backward pass)
    good[0].requires_grad_()
    with pytest.raises(AssertionError):
        form(*good, 2, True)
    with torch.no_grad(), pytest.raises(LibraryCalled):
        form(*good, 2, True)


def _quantised(rows, k):
    blocks = (k + 127) // 128
    values = torch.zeros((rows, blocks * 128), dtype=torch.uint8).view(torch.float8_e4m3fn)[:, :k]
    return values, torch.zeros((rows, (blocks + 3) // 4 * 4), dtype=torch.uint8).view(torch.float8_e8m0fnu)[:, :blocks]


@pytest.mark.parametrize("rows", (0, 1, 2, 5))
@pytest.mark.parametrize("k", (1, 96, 128, 200, 512))
def test_quantised_rows_without_the_room_behind_them(rows, k):
    like = torch.zeros((rows, k))
    values, scales = _quantised(rows, k)
    check_fp8_rows(values, scales, like)

    def packed(t):
        return t.view(torch.uint8).contiguous().clone(memory_format=torch.contiguous_format).view(t.dtype)

    for whole, bad in ((k % 128 == 0, (packed(values), scales)), (k == 512, (values, packed(scales)))):
        if rows == 0 or whole:
            check_fp8_rows(*bad, like)
        else:
            with pytest.raises(AssertionError):
                check_fp8_rows(*bad, like)


@pytest.mark.parametrize("fuse", (False, True))
def test_a_replaced_forward_of_the_block_gets_the_hidden_states_alone(monkeypatch, fuse):
    pytest.importorskip("transformers")
    from transformers import Qwen3MoeConfig

    from qwen3_moe_fused.modular_qwen3_moe_fused import Qwen3MoeFusedModel, Qwen3MoeFusedSparseMoeBlock

    config = Qwen3MoeConfig(vocab_size=20, hidden_size=16, intermediate_size=16, num_hidden_layers=1, num_attention_heads=2,
                            num_key_value_heads=1, head_dim=8, moe_intermediate_size=8, num_experts=4, num_experts_per_tok=2)
    model = Qwen3MoeFusedModel(config).eval()
    model.layers[0].fuse_norm = model.layers[0].mlp.fuse_layer = fuse
    seen = []

    def replaced(self, hidden_states):
        seen.append(hidden_states.shape)
        return hidden_states, hidden_states.new_zeros(hidden_states.shape[1], 4)

    monkeypatch.setattr(Qwen3MoeFusedSparseMoeBlock, "forward", replaced)
    with torch.no_grad():
        model(input_ids=torch.zeros((1, 3), dtype=torch.long))
    assert seen == [(1, 3, 16)]


def _small_model(**changed):
    pytest.importorskip("transformers")
    from transformers import Qwen3MoeConfig

    from qwen3_moe_fused.modular_qwen3_moe_fused import Qwen3MoeFusedModel, Qwen3MoeFusedSparseMoeBlock

    config = Qwen3MoeConfig(**{**dict(vocab_size=20, hidden_size=16, intermediate_size=16, num_hidden_layers=1, num_attention_heads=2,
                                      num_key_value_heads=1, head_dim=8, moe_intermediate_size=8, num_experts=4,
                                      num_experts_per_tok=2, mlp_only_layers=[0]), **changed})  # (a dense layer runs on the host)
    model = Qwen3MoeFusedModel(config).eval()
    if type(model.layers[0].mlp) is Qwen3MoeFusedSparseMoeBlock:
        pytest.skip("this transformers release has blocks that return their logits")
    return model


@pytest.fixture
def own_half(monkeypatch):
    """A small model whose layers have the norm fused, and the calls of the half that goes past the norm's module."""
    model, calls = _small_model(), []
    cls = type(model.layers[0])
    real = cls._feed_forward
    monkeypatch.setattr(cls, "_feed_forward", lambda *args: (calls.append(1), real(*args))[1])
    model.layers[0].fuse_norm = True
    return model, calls


def test_a_replaced_forward_of_the_norms_class_is_called(own_half, monkeypatch):
    model, calls = own_half
    ids = torch.zeros((1, 3), dtype=torch.long)
    with torch.no_grad():
        model(input_ids=ids)
        assert calls == [1]
        seen, norm = [], type(model.layers[0].post_attention_layernorm)
        stock = norm.forward
        monkeypatch.setattr(norm, "forward", lambda self, hidden_states: (seen.append(self), stock(self, hidden_states))[1])
        model(input_ids=ids)
    assert calls == [1] and model.layers[0].post_attention_layernorm in seen


def test_a_forward_replaced_before_the_classes_are_built_is_known_too(monkeypatch):
    pytest.importorskip("transformers")
    import functools

    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeRMSNorm

    from qwen3_moe_fused.modular_qwen3_moe_fused import _defined_forward

    stock = Qwen3MoeRMSNorm.forward
    assert _defined_forward(Qwen3MoeRMSNorm) is stock
    monkeypatch.setattr(Qwen3MoeRMSNorm, "forward", functools.wraps(stock)(lambda self, hidden_states: stock(self, hidden_states)))
    assert _defined_forward(Qwen3MoeRMSNorm) is None
    decorated = {"__name__": "transformers.utils.deprecation"}
    exec("def wrapper(self, hidden_states):\n    return None", decorated)
    monkeypatch.setattr(Qwen3MoeRMSNorm, "forward", decorated["wrapper"])
    assert _defined_forward(Qwen3MoeRMSNorm) is decorated["wrapper"]


def test_a_replaced_forward_of_the_stock_layer_is_called(own_half, monkeypatch):
    model, calls = own_half
    stock_class = type(model.layers[0]).__mro__[1]
    seen, stock = [], stock_class.forward
    monkeypatch.setattr(stock_class, "forward", lambda self, *args, **kwargs: (seen.append(self), stock(self, *args, **kwargs))[1])
    with torch.no_grad():
        model(input_ids=torch.zeros((1, 3), dtype=torch.long))
    assert seen == [model.layers[0]] and not calls


@pytest.mark.parametrize("width", (1, 512, 513, 1024, 1025, 2048, 2049, 4096, 4097, 8192, 8193, 32768))
def test_rows_of_a_call(p, width):
    """The bound that the header names, from either side (nothing is launched: without rows to read the call ends with NULL)."""
    lib, most = _lib.lib(), most_rows(width)
    assert most == 2 ** 32 // max(64, min(1024, 1 << ((width + 7) // 8 - 1).bit_length())) - 1024
    assert width <= 4096 or most == 2 ** 22 - 2 ** 10
    for rows, code in ((most, NULL), (most + 1, LIMIT)):
        assert lib.mfl_add_rms_norm(None, None, p, p, p, rows, width, 1e-6, BF16, BF16, None) == code
        assert lib.mfl_add_rms_norm_fp8(None, None, p, p, p, None, p, rows, width, 1e-6, BF16, BF16, None) == code
    assert lib.mfl_add_rms_norm_bwd(None, None, p, p, p, None, most + 1, width, 1e-6, BF16, BF16, p, 4096, None) == NULL


def test_more_rows_than_a_call_takes_stay_with_the_separate_steps(on_host, monkeypatch):
    layer = _small_model().layers[0].to("meta", torch.bfloat16)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    with torch.no_grad():
        few, many = (torch.empty((1, rows, 16), device="meta", dtype=torch.bfloat16) for rows in (most_rows(16), most_rows(16) + 1))
        with pytest.raises(LibraryCalled):
            layer._feed_forward(few, few, layer.post_attention_layernorm)
        assert layer._feed_forward(many, many, layer.post_attention_layernorm).shape == many.shape


@pytest.mark.parametrize("rows", (1, 3))
@pytest.mark.parametrize("k", (1, 96, 128, 200, 512))
def test_quantised_rows_whose_storage_ends_with_the_last_column(rows, k):
    """A copy of a single row keeps its stride without the room that this stands for."""
    like = torch.zeros((rows, k))
    values, scales = _quantised(rows, k)

    def cut(t):
        copy = t.view(torch.uint8)
        copy = copy.clone() if rows == 1 else torch.empty_strided(copy.shape, copy.stride(), dtype=torch.uint8)
        assert copy.stride() == t.stride()
        return copy.view(t.dtype)

    for whole, bad in ((k % 128 == 0, (cut(values), scales)), (k == 512, (values, cut(scales)))):
        if whole:
            check_fp8_rows(*bad, like)
        else:
            with pytest.raises(AssertionError):
                check_fp8_rows(*bad, like)
    # a row of a table has the next one's room in front of it, the last one its own
    table, table_scales = _quantised(4, k)
    for at in range(0, 5 - rows):
        check_fp8_rows(table[at:at + rows], table_scales[at:at + rows], like)


@pytest.mark.parametrize("how", ("compiled", "mode", "traced"))
def test_a_layer_that_is_watched_keeps_the_separate_steps(own_half, how):
    from torch.utils.flop_counter import FlopCounterMode

    model, calls = own_half
    layer, x = model.layers[0].requires_grad_(False), torch.randn((1, 3, 16), generator=torch.Generator().manual_seed(0))
    given = {"position_embeddings": model.rotary_emb(x, torch.arange(3)[None])}
    with torch.no_grad():
        want = layer(x, **given)
        assert calls == [1]
        if how == "compiled":
            got = torch.compile(layer, backend="eager", fullgraph=True)(x, **given)
        elif how == "mode":
            with FlopCounterMode(display=False):
                got = layer(x, **given)
        else:
            seen = []
            torch.jit.trace(lambda t: seen.append(layer(t, **given)) or seen[-1], (x,), check_trace=False)
            got = seen[0]
    assert calls == [1] and torch.equal(got, want)
