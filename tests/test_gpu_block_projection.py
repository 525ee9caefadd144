"""The attention processor's call and the model wiring with 8-bit projections and layer norms of the heads."""
from types import SimpleNamespace

import pytest
import torch

from peco_amd import model, processor, projection
from peco_amd.norm import LayerNorm, layer_norm_rows
from peco_amd.projection import Int8Linear, QuantizedRows, int8_linear, quantize_rows
from peco_amd.rotary import RotaryAxes, RotaryPositions
from test_processor_call import _Attn, _rotary_tables

DEV = "cuda:0"
HEADS, DIM, VIDEO, TEXT = 3, 64, 210, 37


def _layer(attn, seen):
    """A processor whose attention keeps its inputs and gives a fixed function of them."""
    layer = processor.PecoAttention(0, processor.PecoConfig(), processor.InferenceContext(5, TEXT, TEXT))

    def attention(q, k, v):
        seen.extend(t.clone() for t in (q, k, v))
        return (q + 2 * k - v) / 2

    layer.attention = attention
    return layer


def _call(attn, hidden, text, freqs):
    seen = []
    out = _layer(attn, seen)(attn, hidden, text, image_rotary_emb=freqs)
    return (*seen, *out)


class _Each(torch.nn.Module):
    """An 8-bit layer that quantizes its own rows."""

    def __init__(self, layer):
        super().__init__()
        self.layer = layer

    def forward(self, x):
        return int8_linear(x, QuantizedRows(self.layer.codes, self.layer.scales), self.layer.bias)


def _pipe(attns):
    blocks = [SimpleNamespace(attn=a) for a in attns]
    return SimpleNamespace(transformer=SimpleNamespace(transformer_blocks=blocks[:1], single_transformer_blocks=blocks[1:]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dual", [False, True])
def test_call_with_8_bit_projections(dual, dtype, monkeypatch, announce):
    """The same bits as layers that each quantize their rows; each part's rows are quantized once."""
    announce()
    attn = _Attn(HEADS, DIM, dual, seed=1).to(DEV, dtype)
    plain = {n: m for n, m in attn.named_children() if isinstance(m, torch.nn.Linear)}
    assert model.quantize_projections(_pipe([attn])) == len(plain) + 1
    assert model.quantize_projections(_pipe([attn])) == 0
    assert all(type(getattr(attn, n)) is Int8Linear for n in plain) and type(attn.to_out[0]) is Int8Linear
    g = torch.Generator().manual_seed(3)
    hidden, text = (torch.randn(1, n, HEADS * DIM, generator=g).to(DEV, dtype) for n in (VIDEO, TEXT))
    freqs = tuple(t.to(DEV) for t in _rotary_tables(VIDEO, DIM))
    positions = RotaryPositions(RotaryAxes((16, 24, 24)), RotaryAxes.grid(5, 6, 7, device=DEV))
    calls = []
    monkeypatch.setattr(processor, "quantize_rows", lambda x: calls.append(x.shape) or quantize_rows(x))
    got = [_call(attn, hidden, text, f) for f in (freqs, positions)]
    assert calls == [hidden.shape, text.shape] * 2
    if dual:
        mixed = _Attn(HEADS, DIM, True, seed=1).to(DEV, dtype)  # the text's projections only
        for n in ("add_q_proj", "add_k_proj", "add_v_proj"):
            setattr(mixed, n, getattr(attn, n))
        calls.clear()
        q = _call(mixed, hidden, text, freqs)[0]
        assert calls == [text.shape] and torch.equal(q[:, :, VIDEO:], got[0][0][:, :, VIDEO:])
    for name in plain:
        setattr(attn, name, _Each(getattr(attn, name)))
    for f, out in zip((freqs, positions), got):
        assert all(torch.equal(a, b) for a, b in zip(out, _call(attn, hidden, text, f)))


@pytest.mark.gpu
def test_call_with_rows_from_the_norm(announce):
    """From the residual rows: the norm's rows in 8 bits go through the three projections as they are."""
    announce()
    attn = _Attn(HEADS, DIM, False, seed=2).to(DEV, torch.bfloat16)
    model.quantize_projections(_pipe([attn]))
    g = torch.Generator().manual_seed(4)
    x, text = (torch.randn(1, n, HEADS * DIM, generator=g).to(DEV, torch.bfloat16) for n in (VIDEO, TEXT))
    scale, shift = (torch.randn(1, HEADS * DIM, generator=g).to(DEV, torch.bfloat16) for _ in range(2))
    rows = layer_norm_rows(x, scale, shift, around_one=True)
    q, k, v, out, _ = _call(attn, rows, text, None)
    want = attn.to_v(rows).unflatten(2, (HEADS, DIM)).transpose(1, 2)
    assert want.dtype == torch.bfloat16 and torch.equal(v[:, :, :VIDEO], want)
    assert torch.equal(q[:, :, :VIDEO], attn.norm_q(attn.to_q(rows).unflatten(2, (HEADS, DIM))).transpose(1, 2))
    assert torch.equal(out, attn.to_out[0](((q + 2 * k - v) / 2)[:, :, :VIDEO].transpose(1, 2).flatten(2)))
    with pytest.raises(TypeError):
        attn.to_q = torch.nn.Linear(HEADS * DIM, HEADS * DIM, device=DEV, dtype=torch.bfloat16)
        _call(attn, rows, text, None)


@pytest.mark.gpu
def test_call_with_layer_norms_of_the_heads(announce):
    """A LayerNorm as the heads' norm gives the bits of the module on head-major rows."""
    announce()
    attn = _Attn(HEADS, DIM, False, seed=5).to(DEV, torch.bfloat16)
    for name in ("norm_q", "norm_k"):
        norm = LayerNorm(DIM, eps=1e-6, device=DEV, dtype=torch.bfloat16)
        torch.nn.init.uniform_(norm.weight, 0.5, 1.5)
        torch.nn.init.normal_(norm.bias)
        setattr(attn, name, norm)
    g = torch.Generator().manual_seed(6)
    x, text = (torch.randn(1, n, HEADS * DIM, generator=g).to(DEV, torch.bfloat16) for n in (VIDEO, TEXT))
    freqs = tuple(t.to(DEV) for t in _rotary_tables(VIDEO, DIM))
    q, k, _, _, _ = _call(attn, x, text, freqs)
    with torch.no_grad():
        for got, to, norm in ((q, attn.to_q, attn.norm_q), (k, attn.to_k, attn.norm_k)):
            video, words = (norm(to(t).unflatten(2, (HEADS, DIM)).transpose(1, 2)) for t in (x, text))
            assert torch.equal(got[:, :, VIDEO:], words)
            assert torch.equal(got[:, :, :VIDEO], processor._apply_rotary_emb(video, freqs))


@pytest.mark.gpu
def test_a_layer_that_something_watches_gets_the_tensor(announce):
    announce()
    attn = _Attn(HEADS, DIM, False, seed=7).to(DEV, torch.bfloat16)
    model.quantize_projections(_pipe([attn]))
    x, text = (torch.randn(1, n, HEADS * DIM, device=DEV, dtype=torch.bfloat16) for n in (VIDEO, TEXT))
    want, seen = _call(attn, x, text, None), []
    attn.to_k.register_forward_pre_hook(lambda module, args: seen.append(args[0]))
    got = _call(attn, x, text, None)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(type(t) is torch.Tensor for t in seen) and len(seen) == 2


def test_the_modules_have_the_reference_package_names():
    import peco.norm
    import peco.projection

    assert peco.projection is projection and peco.norm.LayerNorm is LayerNorm
