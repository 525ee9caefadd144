"""The modules around a block's attention, as far as they go without a GPU: what they refuse, what they keep and what they
leave alone."""
import pytest
import torch

from peco_amd import processor
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
