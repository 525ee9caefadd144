"""8-bit projections against their definition in 64 bits, and the block's path through them."""
import pytest
import torch

from norm_reference import product
from peco_amd.norm import layer_norm_rows
from peco_amd.projection import Int8Linear, QuantizedRows, int8_linear, quantize_rows

DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]

# rows, channels, outputs: single rows, ends inside tiles and blocks of every kind, and sizes that fill them
SIZES = [
    (1, 1, 1), (1, 16, 5), (2, 17, 33), (1, 2048, 640), (3, 1000, 1111), (16, 256, 64), (17, 255, 65), (31, 4096, 96),
    (33, 130, 257), (64, 512, 128), (65, 640, 300), (100, 96, 1000), (129, 1111, 130), (257, 384, 520), (300, 64, 2049),
    (1000, 200, 96), (1025, 1024, 1030), (2000, 127, 1999), (2048, 256, 2048), (4097, 72, 1048), (1, 16384, 48),
    (40, 16384, 80),
]


def _codes(g, *shape, extremes=True):
    codes = torch.randint(-127, 128, shape, generator=g, dtype=torch.int64).to(torch.int8)
    if extremes:
        codes.view(-1)[0] = -128
    return codes.to(DEV)


def _inputs(rows, channels, outputs, seed=0):
    g = torch.Generator().manual_seed(rows * 31 + channels + outputs + seed)
    a, w = _codes(g, rows, channels), _codes(g, outputs, channels)
    sa, sw = (torch.rand(n, generator=g).add_(0.1).div_(50).to(DEV) for n in (rows, outputs))
    return a, sa, w, sw, torch.randn(outputs, generator=g).to(DEV)


def _padded(codes, pitch):
    """The same codes in rows `pitch` bytes apart, what is between them set to other codes."""
    kept = torch.full((codes.shape[0], pitch), 77, dtype=torch.int8, device=DEV)
    kept[:, :codes.shape[1]] = codes
    return kept[:, :codes.shape[1]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,channels,outputs", SIZES)
def test_product(rows, channels, outputs, dtype, announce):
    announce()
    a, sa, w, sw, bias = _inputs(rows, channels, outputs)
    for b in (None, bias, bias.to(dtype)):
        ref, bound = product(a, sa, w, sw, b, dtype)
        out = int8_linear(QuantizedRows(a, sa), QuantizedRows(w, sw), b, dtype=dtype)
        assert out.shape == (rows, outputs) and out.dtype == dtype
        assert ((out.double() - ref).abs() <= bound).all()
    pitch = (channels + 15) // 16 * 16
    for p in (pitch, pitch + 48, channels + 1):  # codes between the rows count for nothing
        for q in (pitch, pitch + 16):
            got = int8_linear(QuantizedRows(_padded(a, p), sa), QuantizedRows(_padded(w, q), sw), b, dtype=dtype)
            assert torch.equal(got, out)
    apart = torch.zeros(rows, channels, 2, dtype=torch.int8, device=DEV)[..., 0].copy_(a)
    assert torch.equal(int8_linear(QuantizedRows(apart, sa), QuantizedRows(w, sw), b, dtype=dtype), out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,channels,outputs", SIZES)
def test_rows_are_quantized_as_quantize_rows_does(rows, channels, outputs, dtype, announce):
    announce()
    _, _, w, sw, bias = _inputs(rows, channels, outputs, 1)
    x = torch.randn(rows, channels, generator=torch.Generator().manual_seed(rows)).to(dtype).to(DEV)
    weight = QuantizedRows(_padded(w, (channels + 15) // 16 * 16), sw)
    out = int8_linear(x, weight, bias)
    assert torch.equal(out, int8_linear(quantize_rows(x), weight, bias, dtype=dtype))
    odd = torch.zeros(x.numel() + 1, dtype=dtype, device=DEV)[1:].view(x.shape).copy_(x)
    assert torch.equal(int8_linear(odd, weight, bias), out)
    # Each row is itself whatever the others are, and how many.
    assert torch.equal(int8_linear(x[:1], weight, bias), out[:1])
    assert torch.equal(int8_linear(x.flip(0), weight, bias), out.flip(0))


@pytest.mark.gpu
def test_shapes_strides_and_rows_that_are_not_finite(announce):
    announce()
    g = torch.Generator().manual_seed(3)
    weight = quantize_rows(torch.randn(96, 200, generator=g).to(DEV))
    x = torch.randn(2, 3, 5, 7, 200, generator=g).to(DEV).bfloat16()
    out = int8_linear(x, weight)
    assert out.shape == (2, 3, 5, 7, 96) and out.is_contiguous()
    assert torch.equal(out, int8_linear(x.view(-1, 200), weight).view(out.shape))
    swapped = x.transpose(1, 3)
    assert torch.equal(int8_linear(swapped, weight), out.transpose(1, 3))
    assert torch.equal(int8_linear(quantize_rows(swapped), weight, dtype=x.dtype), out.transpose(1, 3))
    rows = quantize_rows(x)
    turned = QuantizedRows(rows.codes.transpose(0, 2), rows.scales.transpose(0, 2))
    assert torch.equal(int8_linear(turned, weight, dtype=x.dtype), out.transpose(0, 2))
    assert torch.equal(int8_linear(x[:1, :1, :1, :1].expand(2, 3, 5, 7, 200), weight),
                       out[:1, :1, :1, :1].expand(2, 3, 5, 7, 96))
    assert int8_linear(x[:, :0], weight).shape == (2, 0, 5, 7, 96)
    assert torch.equal(int8_linear(x[0, 0, 0, 0], weight), out[0, 0, 0, 0])
    for n in (1, 12, 300):
        x = torch.randn(n, 200, generator=g).to(DEV)
        clean = int8_linear(x, weight)
        bad = x.clone()
        bad[n // 2, 3], bad[0, 199] = float("nan"), float("inf")
        out, odd = int8_linear(bad, weight), torch.zeros(n, dtype=torch.bool, device=DEV)
        odd[[0, n // 2]] = True
        assert out[odd].isnan().all() and torch.equal(out[~odd], clean[~odd])
        bad[:] = 0
        assert int8_linear(bad, weight).eq(0).all()


@pytest.mark.gpu
def test_the_longest_sums_are_exact(announce):
    """2^17 - 1 products of -128 and -128 or 127 come to the edge of 32 bits."""
    announce()
    k = (1 << 17) - 1
    for rows in (1, 20, 70, 300):
        a = torch.full((rows, k), -128, dtype=torch.int8, device=DEV)
        w = torch.full((40, k), -128, dtype=torch.int8, device=DEV)
        w[::2] = 127
        one = torch.ones(rows, device=DEV)
        out = int8_linear(QuantizedRows(a, one), QuantizedRows(w, torch.ones(40, device=DEV)), dtype=torch.float32)
        want = torch.tensor([-128 * 127 * k, 128 * 128 * k], dtype=torch.float32, device=DEV).repeat(20)
        assert torch.equal(out, want.expand(rows, 40))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 300, 3000])
def test_streams_and_graphs(rows, announce):
    announce()
    g = torch.Generator().manual_seed(rows)
    weight = quantize_rows(torch.randn(520, 640, generator=g).to(DEV))
    bias = torch.randn(520, generator=g).to(DEV)
    inputs = [torch.randn(rows, 640, generator=g).to(DEV).bfloat16() for _ in range(4)]
    want = [int8_linear(x, weight, bias) for x in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = int8_linear(inputs[1], weight, bias)
        held = inputs[0].clone()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = int8_linear(held, weight, bias)
    for x, expected in zip(inputs, want):
        held.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, expected)


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(announce):
    announce()
    g = torch.Generator().manual_seed(13)
    weight = quantize_rows(torch.randn(1100, 900, generator=g).to(DEV))
    inputs = [torch.randn(n, 900, generator=g).to(DEV).bfloat16() for n in (1500, 9)]
    want = [int8_linear(x, weight) for x in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append(int8_linear(inputs[k], weight))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[k]) for k in range(2) for out in got[k])


@pytest.mark.gpu
@pytest.mark.parametrize("quantized", [False, True])
def test_inputs_that_are_freed_while_a_copy_of_them_is_due(quantized, announce):
    """Inputs that the call copies (channels, codes, scales or the bias apart) belong to another stream, and are freed there
    before the call's stream has come to the copy: their memory must not be handed out until it has."""
    announce()
    g = torch.Generator().manual_seed(19)
    x = torch.randn(3000, 640, generator=g).to(DEV)
    weight, rows = quantize_rows(torch.randn(1200, 640, generator=g).to(DEV)), quantize_rows(x)
    bias = torch.randn(1200, generator=g).to(DEV)

    def apart(t):
        return torch.zeros(*t.shape, 2, dtype=t.dtype, device=DEV)[..., 0].copy_(t)

    def make():
        first = [apart(rows.codes), apart(rows.scales)] if quantized else [apart(x)]
        return first + [apart(weight.codes), apart(weight.scales), apart(bias)]

    def call(inputs):
        *first, codes, scales, added = inputs
        return int8_linear(QuantizedRows(*first) if quantized else first[0], QuantizedRows(codes, scales), added,
                           dtype=torch.float32)

    want = call(make())
    inputs = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        got = call(inputs)
    sizes = [(t.untyped_storage().nbytes(), t.untyped_storage().data_ptr()) for t in inputs]
    del inputs
    others = [torch.full((size,), 119, dtype=torch.uint8, device=DEV) for size, _ in sizes]
    assert not {t.data_ptr() for t in others} & {at for _, at in sizes}
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_results_past_32_bit_offsets(announce):
    """A result of more than 2^32 elements, and rows of codes more than 2^32 bytes behind the first."""
    announce()
    g = torch.Generator().manual_seed(1)
    rows, outputs = 300_000, 16_384
    a, sa, w, sw, bias = _inputs(4, 64, outputs)
    codes = torch.zeros(rows, 64, dtype=torch.int8, device=DEV)
    scales = torch.zeros(rows, device=DEV)
    codes[[0, 1, rows - 2, rows - 1]], scales[[0, 1, rows - 2, rows - 1]] = a, sa
    out = int8_linear(QuantizedRows(codes, scales), QuantizedRows(w, sw), bias)
    small = int8_linear(QuantizedRows(a, sa), QuantizedRows(w, sw), bias)
    assert torch.equal(out[[0, 1, rows - 2, rows - 1]], small)
    assert torch.equal(out[rows // 2], bias.bfloat16())
    del out, codes
    pitch = 1 << 22
    far = torch.zeros(1100 * pitch, dtype=torch.int8, device=DEV).view(1100, pitch)[:, :64]
    far[[0, 1, 1098, 1099]] = a
    scales = torch.zeros(1100, device=DEV)
    scales[[0, 1, 1098, 1099]] = sa
    assert torch.equal(int8_linear(QuantizedRows(far, scales), QuantizedRows(w, sw), bias)[[0, 1, 1098, 1099]], small)


@pytest.mark.gpu
def test_layer_from_a_linear_layer(announce):
    """Int8Linear against the layer's product: weight and rows are each within half a step of their row's range."""
    announce()
    torch.manual_seed(2)
    layer = torch.nn.Linear(333, 200, device=DEV, dtype=torch.bfloat16)
    quantized = Int8Linear.from_linear(layer)
    x = torch.randn(3, 50, 333, device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        want = x.double() @ layer.weight.double().T + layer.bias.double()
        out = quantized(x)
        rows, weight = quantize_rows(x), QuantizedRows(quantized.codes, quantized.scales)
        assert torch.equal(out, int8_linear(x, weight, layer.bias))
        assert torch.equal(out, quantized(rows))
        sx, sw = rows.scales.double()[..., None] / 2, weight.scales.double() / 2
        bound = sx * layer.weight.double().abs().sum(1) + x.double().abs().sum(-1, keepdim=True) * sw + 333 * sx * sw
        assert ((out.double() - want).abs() <= 1.01 * bound + 2.0 ** -8 * want.abs()).all()
        for moved in (quantized.half(), quantized.double()):
            assert moved.scales.dtype == moved.bias.dtype == torch.float32 and torch.equal(moved(x), out)
        other = Int8Linear.from_linear(torch.nn.Linear(333, 200, device=DEV, dtype=torch.bfloat16))
        other.load_state_dict(quantized.state_dict())
        assert torch.equal(other(x), out)


def test_refusals():
    codes, scales = torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4)
    weight = QuantizedRows(codes, scales)
    for bad, error in (((codes.float(), scales), TypeError), ((codes, scales.double()), TypeError),
                       ((codes, torch.zeros(3)), ValueError), ((None, scales), TypeError)):
        with pytest.raises(error):
            QuantizedRows(*bad)
    x = torch.zeros(2, 16)
    for args, error in (((x, codes), TypeError), ((1.0, weight), TypeError), ((torch.zeros(2, 15), weight), ValueError),
                        ((x.double(), weight), TypeError), ((x, weight, torch.zeros(5)), ValueError),
                        ((x, weight, torch.zeros(4).double()), TypeError), ((x, weight), ValueError),
                        ((x, QuantizedRows(codes[None], scales[None])), ValueError),
                        ((x[:, :0], QuantizedRows(codes[:, :0], scales)), ValueError),
                        ((weight, weight), ValueError)):
        with pytest.raises(error):
            int8_linear(*args)
    with pytest.raises(TypeError):
        int8_linear(x, weight, dtype=torch.float64)
    for bad, error in ((x, ValueError), (x.double(), TypeError), (torch.zeros(2, 0), ValueError),
                       (torch.zeros(1, 16385), ValueError), (None, TypeError)):
        with pytest.raises(error):
            quantize_rows(bad)


@pytest.mark.gpu
def test_refusals_on_the_gpu(announce):
    announce()
    weight = quantize_rows(torch.randn(8, 16, device=DEV))
    x = torch.randn(2, 16, device=DEV)
    with pytest.raises(RuntimeError):
        int8_linear(x.requires_grad_(), weight)
    with pytest.raises(RuntimeError):
        quantize_rows(x)
    with pytest.raises(ValueError):
        int8_linear(x.detach(), QuantizedRows(torch.zeros(8, 16, dtype=torch.int8), torch.zeros(8)))
    with pytest.raises(ValueError):
        int8_linear(x.detach(), weight, torch.zeros(8))
    wide = QuantizedRows(torch.zeros(1, 1 << 17, dtype=torch.int8, device=DEV), torch.zeros(1, device=DEV))
    with pytest.raises(ValueError):
        int8_linear(wide, wide)
    with torch.no_grad():
        assert int8_linear(x, weight).shape == (2, 8)


@pytest.mark.gpu
def test_norm_and_projection_in_a_row(announce):
    """A block's rows from the residual to the joint projection: the codes between the two are within half a step of
    the norm, so the product is within what those leave."""
    announce()
    g = torch.Generator().manual_seed(9)
    x = torch.randn(2, 70, 512, generator=g).to(DEV).bfloat16()
    scale, shift = (torch.randn(2, 512, generator=g).mul_(0.3).to(DEV).bfloat16() for _ in range(2))
    weight = quantize_rows(torch.randn(1536 // 2, 512, generator=g).to(DEV))
    bias = torch.randn(1536 // 2, generator=g).to(DEV).bfloat16()
    rows = layer_norm_rows(x, scale, shift, around_one=True)
    out = int8_linear(rows, weight, bias)
    ref, bound = product(rows.codes, rows.scales, weight.codes, weight.scales, bias, torch.bfloat16)
    assert ((out.double() - ref).abs() <= bound).all()
