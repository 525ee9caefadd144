"""8-bit layers in a transformer's blocks on the GPU: layers that are refused, shared, watched or moved, and autocast."""
from types import SimpleNamespace

import pytest
import torch

from peco_amd import model
from peco_amd.projection import Int8Linear, QuantizedRows, int8_linear, quantize_rows
from test_gpu_block_projection import DEV, DIM, HEADS, TEXT, VIDEO, _call, _pipe
from test_processor_call import _Attn


def _attn(seed, dtype=torch.bfloat16):
    return _Attn(HEADS, DIM, False, seed=seed, norms=False).to(DEV, dtype)


def _inputs(dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(8)
    return [torch.randn(1, n, HEADS * DIM, generator=g).to(DEV, dtype) for n in (VIDEO, TEXT)]


@pytest.mark.gpu
def test_a_layer_on_the_cpu_leaves_the_transformer_as_it_was(announce):
    announce()
    attns = _attn(1), _attn(2)
    attns[1].to_out[0].cpu()
    with pytest.raises(ValueError):
        model.quantize_projections(_pipe(attns))
    assert not any(isinstance(m, Int8Linear) for attn in attns for m in attn.modules())
    attns[1].to_out[0].to(DEV)
    assert model.quantize_projections(_pipe(attns)) == 8


@pytest.mark.gpu
def test_a_forward_of_its_own_and_hooks_of_all_modules_see_the_tensor(announce):
    announce()
    attn, seen = _attn(3), []
    model.quantize_projections(_pipe([attn]))
    x, text = _inputs()
    want = _call(attn, x, text, None)
    inner = attn.to_k.forward
    attn.to_k.forward = lambda rows: seen.append(type(rows)) or inner(rows)
    assert all(torch.equal(a, b) for a, b in zip(_call(attn, x, text, None), want))
    assert seen == [torch.Tensor] * 2
    del attn.to_k.forward
    seen.clear()
    handle = torch.nn.modules.module.register_module_forward_pre_hook(
        lambda module, args: seen.append(type(args[0])) if type(module) is Int8Linear else None)
    try:
        assert all(torch.equal(a, b) for a, b in zip(_call(attn, x, text, None), want))
    finally:
        handle.remove()
    assert seen and set(seen) == {torch.Tensor}


@pytest.mark.gpu
def test_a_layer_that_moves(announce):
    """By the CPU and back the same bits, from codes that a call takes as they are."""
    announce()
    for channels in (72, 333, 1000):
        layer = Int8Linear.from_linear(torch.nn.Linear(channels, 200, device=DEV, dtype=torch.bfloat16))
        x = torch.randn(40, channels, device=DEV, dtype=torch.bfloat16)
        with torch.no_grad():
            want, stride = layer(x), layer.codes.stride()
            layer.cpu().to(DEV)
            assert layer.codes.stride() == stride and stride[0] % 16 == 0 and torch.equal(layer(x), want)
            sent = {k: v.cpu() for k, v in layer.state_dict().items()}
            layer.to("meta").to_empty(device=DEV).load_state_dict(sent)
            assert layer.codes.stride() == stride and torch.equal(layer(x), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast(dtype, announce):
    """fp32 rows under autocast: the results of the call with that dtype, in a layer alone and in the processor's call."""
    announce()
    attn = _attn(4, torch.float32)
    model.quantize_projections(_pipe([attn]))
    x, text = _inputs(torch.float32)
    with torch.no_grad(), torch.autocast("cuda", dtype):
        assert torch.equal(attn.to_q(x), attn.to_q(quantize_rows(x), dtype=dtype))
        assert attn.to_q(quantize_rows(x)).dtype == dtype and attn.to_q(x, dtype=torch.float32).dtype == torch.float32
        _, _, v, out, _ = _call(attn, x, text, None)
    assert v.dtype == out.dtype == dtype
    with torch.no_grad():
        want = attn.to_v(quantize_rows(x), dtype=dtype).unflatten(2, (HEADS, DIM)).transpose(1, 2)
        assert torch.equal(v[:, :, :VIDEO], want)
        assert attn.to_q(x).dtype == torch.float32


@pytest.mark.gpu
def test_results_of_few_rows_that_no_launch_holds(announce):
    """Refused before the result's gigabytes are allocated."""
    announce()
    weight = QuantizedRows(torch.zeros(1, 16, dtype=torch.int8, device=DEV).expand(1 << 27, 16),
                           torch.zeros(1, device=DEV).expand(1 << 27))
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for rows in (1, 17, 32):
        with pytest.raises(ValueError, match="2\\^27"):
            int8_linear(torch.zeros(rows, 16, device=DEV), weight)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20


@pytest.mark.gpu
def test_a_layer_of_codes_off_16_bytes(announce):
    announce()
    flat = torch.randint(-127, 128, (200 * 32 + 8,), device=DEV).to(torch.int8)
    scales, x = torch.rand(200, device=DEV), torch.randn(40, 32, device=DEV)
    weight = QuantizedRows(flat[8:].view(200, 32), scales)
    layer = Int8Linear(weight)
    assert layer.codes.data_ptr() % 16 == 0 and torch.equal(layer.codes, weight.codes)
    assert torch.equal(layer(x), int8_linear(x, weight))
