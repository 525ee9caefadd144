"""The modules around a block's attention, as far as they go without a GPU: what they refuse, what they keep and what they
leave alone."""
from types import SimpleNamespace

import pytest
import torch

from peco_amd import model, processor, projection
from peco_amd.norm import LayerNorm
from peco_amd.projection import Int8Linear, QuantizedRows


@pytest.mark.parametrize("affine", [True, False])
def test_a_layer_norm_takes_rows_of_its_own_channels(affine):
    norm = LayerNorm(64, elementwise_affine=affine)
    for shape in ((128,), (2, 32), (64, 3), ()):
        with pytest.raises(ValueError, match="64 channels"):
            norm(torch.zeros(shape))
    with pytest.raises(ValueError, match="GPU"):  # rows of its channels come as far as the device
        norm(torch.zeros(2, 64))


def _int8_layer(outputs=8, channels=32, bias=True):
    g = torch.Generator().manual_seed(outputs + channels)
    codes = torch.randint(-127, 128, (outputs, channels), generator=g).to(torch.int8)
    return Int8Linear(QuantizedRows(codes, torch.rand(outputs, generator=g)), torch.rand(outputs, generator=g) if bias else None)


def _watch_forward(layers):
    layers[1].forward = lambda x: x
    return lambda: None


def _watch_instance(layers):
    return layers[2].register_forward_pre_hook(lambda module, args: None).remove


def _watch_all_inputs(layers):
    return torch.nn.modules.module.register_module_forward_pre_hook(lambda module, args: None).remove


def _watch_all_outputs(layers):
    return torch.nn.modules.module.register_module_forward_hook(lambda module, args, out: None).remove


@pytest.mark.parametrize("watch", [_watch_forward, _watch_instance, _watch_all_inputs, _watch_all_outputs])
def test_layers_that_something_watches_share_no_rows(watch, monkeypatch):
    """Rows are quantized for a part's three layers only where nothing would see them in the tensor's place."""
    monkeypatch.setattr(processor, "quantize_rows", lambda x: "rows")
    source, layers = torch.zeros(1, 5, 32), [_int8_layer() for _ in range(3)]
    assert processor._shared_rows(source, layers) == "rows"
    remove = watch(layers)
    try:
        assert processor._shared_rows(source, layers) is source
    finally:
        remove()


class _Attn(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.to_q, self.to_k, self.to_v = (torch.nn.Linear(32, 32) for _ in range(3))
        self.to_out = torch.nn.ModuleList([torch.nn.Linear(32, 32), torch.nn.Dropout(0.0)])


def _pipe(*attns):
    blocks = [SimpleNamespace(attn=a) for a in attns]
    return SimpleNamespace(transformer=SimpleNamespace(transformer_blocks=blocks[:1], single_transformer_blocks=blocks[1:]))


def _layers(attn):
    return attn.to_q, attn.to_k, attn.to_v, attn.to_out[0]


def _stand_in(monkeypatch, refused=lambda: None):
    """from_linear without a GPU; ``refused()`` is a layer that it does not take."""
    def make(layer):
        if layer is refused():
            raise ValueError("not this one")
        return _int8_layer(layer.out_features, layer.in_features)

    monkeypatch.setattr(projection.Int8Linear, "from_linear", make)


def test_a_refused_layer_leaves_the_transformer_as_it_was(monkeypatch):
    attns = _Attn(), _Attn()
    _stand_in(monkeypatch, lambda: attns[1].to_out[0])
    before = [_layers(a) for a in attns]
    with pytest.raises(ValueError, match="not this one"):
        model.quantize_projections(_pipe(*attns))
    assert all(a is b for attn, old in zip(attns, before) for a, b in zip(_layers(attn), old))
    _stand_in(monkeypatch)
    assert model.quantize_projections(_pipe(*attns)) == 8
    assert all(type(layer) is Int8Linear for attn in attns for layer in _layers(attn))
    assert model.quantize_projections(_pipe(*attns)) == 0


@pytest.mark.parametrize("attach", [
    lambda layer: layer.register_forward_hook(lambda *a: None),
    lambda layer: layer.register_forward_pre_hook(lambda *a: None),
    lambda layer: layer.register_full_backward_hook(lambda *a: None),
    lambda layer: layer.register_full_backward_pre_hook(lambda *a: None),
    lambda layer: setattr(layer, "forward", torch.nn.functional.relu),
])
def test_a_layer_with_something_attached_is_refused(attach, monkeypatch):
    """It would be lost with the layer."""
    _stand_in(monkeypatch)
    attns = _Attn(), _Attn()
    attach(attns[1].to_v)
    before = [_layers(a) for a in attns]
    with pytest.raises(RuntimeError, match=r"block 1.*to_v"):
        model.quantize_projections(_pipe(*attns))
    assert all(a is b for attn, old in zip(attns, before) for a, b in zip(_layers(attn), old))


def test_a_layer_in_several_places_stays_one(monkeypatch):
    _stand_in(monkeypatch)
    attns = _Attn(), _Attn()
    attns[1].to_q = attns[0].to_k = attns[0].to_q
    assert model.quantize_projections(_pipe(*attns, attns[0])) == 8  # (a block's attention that comes twice)
    assert attns[1].to_q is attns[0].to_q and attns[0].to_k is attns[0].to_q and attns[0].to_v is not attns[0].to_q


def test_an_output_projection_without_a_list(monkeypatch):
    _stand_in(monkeypatch)
    attns = _Attn(), _Attn(), _Attn()
    attns[0].to_out, attns[1].to_out, attns[2].to_out = torch.nn.Linear(32, 32), torch.nn.Identity(), None
    assert model.quantize_projections(_pipe(*attns)) == 10
    assert type(attns[0].to_out) is Int8Linear and type(attns[1].to_out) is torch.nn.Identity


def test_a_layer_that_moves_keeps_its_rows_on_16_bytes():
    """(Rows a fixed number of 16 bytes apart are what a call takes without a copy.)"""
    for channels, pitch in ((20, 32), (32, 32), (600, 640)):
        layer = _int8_layer(8, channels)
        codes, scales, bias = layer.codes.clone(), layer.scales.clone(), layer.bias.clone()
        assert layer.codes.stride() == (pitch, 1)
        for move in (lambda: layer.to("meta"), lambda: layer.to_empty(device="cpu"), layer.half, layer.double,
                     lambda: layer.to("cpu", torch.bfloat16)):
            move()
            assert layer.codes.shape == (8, channels) and layer.codes.stride() == (pitch, 1)
            assert layer.codes.dtype == torch.int8 and layer.scales.dtype == layer.bias.dtype == torch.float32
            assert layer.codes.device == layer.scales.device == layer.bias.device
            if layer.codes.device.type == "cpu":
                for kept, t in ((layer.codes, codes), (layer.scales, scales), (layer.bias, bias)):
                    assert kept.copy_(t) is kept
    layer = _int8_layer(8, 20, bias=False)
    assert layer.half().bias is None
    codes = layer.codes
    layer.float()
    assert layer.codes is codes  # (as it was)


def test_values_stay_through_a_cast():
    layer = _int8_layer(8, 20)
    codes, scales, bias = layer.codes.clone(), layer.scales.clone(), layer.bias.clone()
    for change in (layer.half, layer.double, layer.bfloat16):
        change()
        assert torch.equal(layer.codes, codes) and torch.equal(layer.scales, scales) and torch.equal(layer.bias, bias)
    assert layer.share_memory() is layer and layer.codes.is_shared() and layer.scales.is_shared()


def test_results_under_autocast_have_its_dtype(monkeypatch):
    """As those of the torch.nn.Linear whose place a layer takes; without it the rows' (codes: the layer's)."""
    asked = []
    monkeypatch.setattr(projection, "int8_linear", lambda x, weight, bias, dtype: asked.append(dtype))
    monkeypatch.setattr(processor, "quantize_rows", lambda x: codes)
    layers, x = [_int8_layer() for _ in range(3)], torch.zeros(2, 32)
    codes = QuantizedRows(torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2))

    def calls():
        asked.clear()
        layers[0](x), layers[0](codes), layers[0](x, dtype=torch.float32)
        processor._project(layers[0], x, processor._shared_rows(x, layers))
        processor._project(layers[0], codes, processor._shared_rows(codes, layers))
        return asked

    assert calls() == [torch.float32, torch.bfloat16, torch.float32, torch.float32, torch.bfloat16]
    kept = torch.get_autocast_dtype("cuda")
    try:  # (what torch.autocast sets, which does nothing without a GPU)
        torch.set_autocast_enabled("cuda", True)
        for dtype in (torch.float16, torch.bfloat16):
            torch.set_autocast_dtype("cuda", dtype)
            assert calls() == [dtype, dtype, torch.float32, dtype, dtype]
    finally:
        torch.set_autocast_enabled("cuda", False)
        torch.set_autocast_dtype("cuda", kept)
