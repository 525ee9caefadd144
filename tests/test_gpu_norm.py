"""Layer norm, its gradients and its quantized rows against their definitions in 64 bits."""
import pytest
import torch

from norm_reference import HALF_STEP, Norm, quantized
from peco_amd.norm import LayerNorm, layer_norm, layer_norm_rows
from peco_amd.projection import quantize_rows

DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]

# shape, entries of weight and bias (0: one for all)
SHAPES = [
    ((1, 1), 0), ((1, 8), 0), ((3, 5, 7), 3), ((5, 64), 0), ((2, 9, 3, 64), 2), ((1, 3, 37, 128), 0), ((70, 72), 0),
    ((3, 11, 130), 3), ((4, 512), 4), ((2, 17, 520), 2), ((9, 1024), 0), ((2, 5, 1111), 0), ((3, 3, 2048), 3),
    ((7, 2056), 0), ((2, 6, 4096), 2), ((5, 4099), 0), ((2, 3, 8192), 0), ((2, 2, 16384), 2), ((3, 16001), 0),
    ((2, 700, 64), 2), ((1200, 264), 0), ((2, 2, 3, 5, 96), 2),
]


def _inputs(shape, entries, dtype, wide, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    size = torch.exp(torch.randn(*shape[:-1], 1, generator=g))
    x = (torch.randn(shape, generator=g) * size + torch.randn(*shape[:-1], 1, generator=g)).to(dtype).to(DEV)
    affine = (entries, shape[-1]) if entries else (shape[-1],)
    kind = torch.float32 if wide else dtype
    weight, bias = ((torch.randn(affine, generator=g) * 0.5).to(kind).to(DEV) for _ in range(2))
    grad = torch.randn(shape, generator=g).to(dtype).to(DEV)
    return x, weight, bias, grad


def _layouts(x):
    """x as it is, head-major, in wider rows, off 16 bytes, with channels apart, and expanded."""
    yield x
    if x.dim() >= 3:
        yield x.transpose(-3, -2).contiguous().transpose(-3, -2)
    wide = torch.full((*x.shape[:-1], x.shape[-1] + 8), 3.0, dtype=x.dtype, device=DEV)
    wide[..., :x.shape[-1]] = x
    yield wide[..., :x.shape[-1]]
    yield torch.zeros(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape).copy_(x)
    yield torch.zeros(*x.shape, 2, dtype=x.dtype, device=DEV)[..., 0].copy_(x)
    if x.dim() >= 2:
        yield x[:1].expand(x.shape)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,entries", SHAPES)
def test_rows(shape, entries, dtype, announce):
    announce()
    for wide in (False, True):
        x, weight, bias, _ = _inputs(shape, entries, dtype, wide)
        for w, b, around in ((weight, bias, False), (weight, None, True), (None, bias, False), (None, None, False)):
            for part in _layouts(x):
                ref = Norm(part, w, b, 1e-5, around)
                out = layer_norm(part, w, b, 1e-5, around_one=around)
                assert out.shape == part.shape and out.stride() == torch.empty_like(part).stride()
                assert ((out.double() - ref.out).abs() <= ref.out_bound()).all()
    if shape[-1] > 1:
        # One row normalised alone has the same bits.
        one = layer_norm(x.reshape(-1, shape[-1])[-1:], None, None, 1e-5)
        assert torch.equal(one, layer_norm(x, None, None, 1e-5).reshape(-1, shape[-1])[-1:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,entries", SHAPES)
def test_gradients(shape, entries, dtype, announce):
    announce()
    for wide in (False, True):
        x, weight, bias, grad = _inputs(shape, entries, dtype, wide, 1)
        for around, part, by in ((False, x, grad), *((True, p, g) for p, g in zip(_layouts(x), _layouts(grad)))):
            leaves = [t.detach().requires_grad_() for t in (part, weight, bias)]
            out = layer_norm(*leaves, 1e-5, around_one=around)
            got = torch.autograd.grad(out, leaves, by, retain_graph=True)
            (dx, dx_bound), (dw, dw_off), (db, db_off) = Norm(part, weight, bias, 1e-5, around).gradients(by, entries > 0)
            half = HALF_STEP[weight.dtype] * 1.01
            assert ((got[0].double() - dx).abs() <= dx_bound).all()
            assert ((got[1].double() - dw).abs() <= half * dw.abs() + dw_off + 2.0 ** -25).all()
            assert ((got[2].double() - db).abs() <= half * db.abs() + db_off + 2.0 ** -25).all()
            again = torch.autograd.grad(out, leaves, by, retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(got, again))
            for i, t in enumerate(leaves):  # each alone
                assert torch.equal(torch.autograd.grad(out, t, by, retain_graph=True)[0], got[i])


@pytest.mark.gpu
def test_gradients_against_differences(announce):
    """fp32 rows moved by a small step along each gradient's own direction: the quotient of central differences h is the
    slope to h^2 of third derivatives, which for rows of deviation near 1, steps of 2^-7 and unit directions stay below
    2^-14 * 16 of the gradient's size, and to the sum's roundings (n values within 2^-20 of their size) over h."""
    announce()
    g = torch.Generator().manual_seed(5)
    x, grad = (torch.randn(2, 9, 96, generator=g).to(DEV) for _ in range(2))
    weight, bias = (torch.randn(2, 96, generator=g).to(DEV) for _ in range(2))
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    slopes = torch.autograd.grad((layer_norm(*leaves, 1e-3, around_one=True) * grad).sum(), leaves)
    h = 2.0 ** -7
    with torch.no_grad():
        for i, slope in enumerate(slopes):
            step = slope / slope.norm()
            values = []
            for sign in (1, -1):
                moved = [t + sign * h * step if j == i else t for j, t in enumerate(leaves)]
                values.append(float((layer_norm(*moved, 1e-3, around_one=True).double() * grad.double()).sum()))
            size = float(slope.norm())
            assert abs((values[0] - values[1]) / (2 * h) - size) <= 2.0 ** -10 * size + \
                2.0 ** -20 / h * float(grad.abs().sum())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,entries", SHAPES)
def test_quantized_rows(shape, entries, dtype, announce):
    """Codes of the norm's fp32 rows: every value within half a step of the row, and what fp32 leaves of the norm; the
    largest has code 127. (The factor of the codes has three roundings, the scale two: 127 steps * 3 2^-24 and 2^-23
    of the largest value are together below 2^-21 of it.)"""
    announce()
    x, weight, bias, _ = _inputs(shape, entries, dtype, False, 2)
    for part in _layouts(x):
        ref = Norm(part, weight, bias, 1e-5, True)
        rows = layer_norm_rows(part, weight, bias, 1e-5, around_one=True)
        assert rows.shape == part.shape and rows.scales.shape == part.shape[:-1]
        most = ref.out.abs().amax(-1, keepdim=True)
        off = ref.out_off.amax(-1, keepdim=True) + 2.0 ** -21 * most
        assert ((rows.dequantize(torch.float64) - ref.out).abs() <= most / 254 + off).all()
        assert ((rows.scales.double() * 127)[..., None] - most).abs().le(off).all()
        assert (rows.codes.abs().amax(-1) == 127).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,entries", SHAPES)
def test_row_quantization_is_exact(shape, entries, dtype, announce):
    announce()
    x = _inputs(shape, entries, dtype, False, 3)[0]
    for part in _layouts(x):
        rows, (codes, scales) = quantize_rows(part), quantized(part)
        assert torch.equal(rows.codes.cpu(), codes) and torch.equal(rows.scales.cpu(), scales)
    # Halves of a step go to the even code; rows of zeros, of tiny values, with infinities and NaN.
    steps = torch.arange(-127, 128, dtype=torch.float32) / 2
    ties = torch.cat((torch.tensor([127.0]), steps)).to(dtype).to(DEV)
    assert torch.equal(quantize_rows(ties).codes.cpu(), quantized(ties)[0])
    odd = torch.ones(6, 72, dtype=dtype, device=DEV)
    odd[0], odd[1, 3], odd[2, 70], odd[3, 0] = 0, float("inf"), float("nan"), -float("inf")
    if dtype != torch.float16:
        odd[4] = 2.0 ** -121
    rows = quantize_rows(odd)
    zero = [0, 4] if dtype != torch.float16 else [0]
    for i in range(6):
        if i in (1, 2, 3):
            assert rows.codes[i].eq(0).all() and rows.scales[i].isnan()
        elif i in zero:
            assert rows.codes[i].eq(0).all() and rows.scales[i] == 0
        else:
            assert rows.codes[i].eq(127).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels", [64, 100, 2048, 5000])
def test_rows_that_are_not_finite_or_constant(channels, dtype, announce):
    """A NaN or an infinity makes its own row NaN (output, gradient, codes) and no other; a constant row gives the bias."""
    announce()
    g = torch.Generator().manual_seed(channels)
    x = torch.randn(40, channels, generator=g).to(dtype).to(DEV)
    weight, bias = (torch.randn(channels, generator=g).to(dtype).to(DEV) for _ in range(2))
    clean, grad = layer_norm(x, weight, bias), torch.randn(40, channels, generator=g).to(dtype).to(DEV)
    bad = x.clone()
    bad[3, 5], bad[17, channels - 1], bad[39, 0], bad[20] = float("nan"), float("inf"), -float("inf"), 2.5
    odd = torch.zeros(40, dtype=torch.bool, device=DEV)
    odd[[3, 17, 39]] = True
    leaf = bad.requires_grad_()
    out = layer_norm(leaf, weight, bias)
    dx, = torch.autograd.grad(out, leaf, grad)
    assert out[odd].isnan().all() and dx[odd].isnan().all()
    odd[20] = True
    assert torch.equal(out[~odd], clean[~odd]) and dx[~odd].isfinite().all()
    assert torch.equal(out[20], bias)
    with torch.no_grad():
        rows, sound = layer_norm_rows(bad, weight, bias), layer_norm_rows(x, weight, bias)
    assert rows.scales[[3, 17, 39]].isnan().all() and rows.codes[[3, 17, 39]].eq(0).all()
    assert torch.equal(rows.codes[~odd], sound.codes[~odd]) and torch.equal(rows.scales[~odd], sound.scales[~odd])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,entries", [((2, 9, 3, 64), 2), ((1, 3, 37, 128), 0), ((2, 5, 1111), 0), ((3, 3, 2048), 3)])
def test_gradients_without_a_weight_or_a_bias(shape, entries, dtype, announce):
    announce()
    x, weight, bias, grad = _inputs(shape, entries, dtype, False, 7)
    half = HALF_STEP[dtype] * 1.01
    for w, b in ((None, None), (None, bias), (weight, None)):
        leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
        given = iter(leaves[1:])
        out = layer_norm(leaves[0], None if w is None else next(given), None if b is None else next(given), 1e-5)
        got = torch.autograd.grad(out, leaves, grad)
        (dx, dx_bound), (dw, dw_off), (db, db_off) = Norm(x, w, b, 1e-5, False).gradients(grad, entries > 0)
        assert ((got[0].double() - dx).abs() <= dx_bound).all()
        if w is not None:
            assert ((got[1].double() - dw).abs() <= half * dw.abs() + dw_off + 2.0 ** -25).all()
        if b is not None:
            assert ((got[1].double() - db).abs() <= half * db.abs() + db_off + 2.0 ** -25).all()
    frozen = x.detach()
    leaf = weight.detach().requires_grad_()
    only, = torch.autograd.grad(layer_norm(frozen, leaf, bias, 1e-5), leaf, grad)  # rows without a gradient
    assert ((only.double() - dw).abs() <= half * dw.abs() + dw_off + 2.0 ** -25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,entries", [((2, 7, 3, 64), 2), ((3, 5, 1111), 0), ((2, 9, 2048), 2)])
def test_saved_tensors_that_come_back_laid_out_anew(shape, entries, dtype, announce):
    """Hooks of saved tensors keep their sizes and values, not their strides: the gradients are the same bits."""
    announce()
    x, weight, bias, grad = _inputs(shape, entries, dtype, False, 2)

    def apart(t):  # the same values, every second element
        return torch.zeros(*t.shape, 2, dtype=t.dtype, device=DEV)[..., 0].copy_(t.detach())

    def dense(t):
        return t.detach().clone(memory_format=torch.contiguous_format)

    for part in _layouts(x):
        leaves = [t.detach().requires_grad_() for t in (part, weight, bias)]
        want = torch.autograd.grad(layer_norm(*leaves, 1e-5), leaves, grad)
        for pack in (dense, apart):
            with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
                out = layer_norm(*leaves, 1e-5)
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, grad), want))
    with torch.autograd.graph.save_on_cpu():
        out = layer_norm(*leaves, 1e-5)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, grad), want))


@pytest.mark.gpu
def test_leaves_that_change_before_the_gradient_are_refused(announce):
    """A module may be cast or moved between its forward and its backward call."""
    announce()
    for change in (torch.Tensor.bfloat16, torch.Tensor.cpu, lambda t: t[:32].clone()):
        for which in range(3):
            leaves = [torch.ones(64, device=DEV).requires_grad_() for _ in range(3)]
            out = layer_norm(*leaves)
            leaves[which].data = change(leaves[which].data)
            with pytest.raises(RuntimeError):
                torch.autograd.grad(out, [t for i, t in enumerate(leaves) if i != which], torch.ones_like(out))


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(announce):
    """Forward and backward of two inputs on two streams, several in flight, against one after the other."""
    announce()
    g = torch.Generator().manual_seed(11)
    inputs = [tuple(torch.randn(2, 900, 1024, generator=g).to(DEV) for _ in range(2)) for _ in range(2)]
    weight, bias = (torch.randn(2, 1024, generator=g).to(DEV).requires_grad_() for _ in range(2))

    def step(x, grad):
        x = x.detach().requires_grad_()
        out = layer_norm(x, weight, bias)
        return out.detach(), *torch.autograd.grad(out, (x, weight, bias), grad)

    want = [step(*i) for i in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append(step(*inputs[k]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for k in range(2) for out in got[k] for a, b in zip(out, want[k]))


@pytest.mark.gpu
def test_inputs_that_are_freed_while_a_copy_of_them_is_due(announce):
    """Inputs that the call copies (channels apart, weights of two types or apart) belong to another stream, and are freed
    there before the call's stream has come to the copy: their memory must not be handed out until it has."""
    announce()
    g = torch.Generator().manual_seed(17)
    x = torch.randn(6, 500, 1024, generator=g).to(DEV)
    weight, bias = (torch.randn(6, 1024, generator=g).to(DEV) for _ in range(2))

    def apart(t):
        return torch.zeros(*t.shape, 2, dtype=t.dtype, device=DEV)[..., 0].copy_(t)

    calls = [(layer_norm, lambda: (apart(x), apart(weight), apart(bias))),
             (layer_norm, lambda: (apart(x.half()), weight.clone(), bias.half())),
             (lambda *t: layer_norm_rows(*t).codes, lambda: (apart(x), apart(weight), apart(bias))),
             (lambda *t: quantize_rows(*t).codes, lambda: (apart(x),))]
    side = torch.cuda.Stream()
    for call, make in calls:
        want = call(*make())
        inputs = make()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            got = call(*inputs)
        sizes = [(t.untyped_storage().nbytes(), t.untyped_storage().data_ptr()) for t in inputs]
        del inputs
        others = [torch.full((size,), 119, dtype=torch.uint8, device=DEV) for size, _ in sizes]
        assert not {t.data_ptr() for t in others} & {at for _, at in sizes}
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [8, 100, 128, 777, 2048, 5000])
def test_rows_far_from_zero(channels, announce):
    """fp32 rows 10^4 to 10^6 times as far from 0 as they are wide (steps of 2^-10 around 2^13, of 2^-4 around
    -2^17), and constant ones: the bounds hold no term of the distance but its square."""
    announce()
    g = torch.Generator().manual_seed(channels)
    steps = torch.randint(-3, 4, (3, 40, channels), generator=g).float()
    x = torch.stack((8192 + steps[0] / 1024, -131072 + steps[1] / 16, torch.full((40, channels), 1000.1))).to(DEV)
    weight, bias = (torch.randn(3, channels, generator=g).to(DEV) for _ in range(2))
    grad = torch.randn(3, 40, channels, generator=g).to(DEV)
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    out = layer_norm(*leaves, 1e-6)
    ref = Norm(x.detach(), weight.detach(), bias.detach(), 1e-6, False)
    assert ((out.double() - ref.out).abs() <= ref.out_bound()).all()
    (dx, dx_bound), (dw, dw_off), _ = ref.gradients(grad, True)
    got = torch.autograd.grad(out, leaves, grad)
    assert ((got[0].double() - dx).abs() <= dx_bound).all()
    assert ((got[1].double() - dw).abs() <= 2.0 ** -24 * dw.abs() + dw_off).all()
    # A check of the bounds themselves. Rows at 8192: a plain mean is good to 48 2^-24 8192 = 0.023, which times the
    # inverse (up to 1000 for these steps) leaves 23 in n. Here its square, 550, stands at 48 2^-24 |n f|: 0.0016 of at most 9.
    assert float(ref.out_bound()[0].max()) < 0.0016 * 9 * 1.1


@pytest.mark.gpu
def test_mixed_weights_empty_rows_and_module(announce):
    announce()
    x = torch.randn(2, 6, 64, device=DEV).bfloat16()
    weight, bias = torch.randn(64, device=DEV), torch.randn(2, 64, device=DEV).bfloat16()
    for w, b in ((weight, bias), (weight.bfloat16(), bias.float())):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        out = layer_norm(*leaves)
        ref = Norm(x, w, b, 1e-6, False)
        assert ((out.double() - ref.out).abs() <= ref.out_bound()).all()
        dx, dw, db = torch.autograd.grad(out.float().sum(), leaves)
        assert dw.shape == w.shape and dw.dtype == w.dtype and db.shape == b.shape and db.dtype == b.dtype
        (want, bound), _, (bias_grad, _) = ref.gradients(torch.ones_like(x), True)
        assert ((dx.double() - want).abs() <= bound).all() and torch.equal(db.double(), bias_grad)
        # (dw is what rows of the two entries leave of sums that are near 0: 12 rows, 2^-24 * 100 of each.)
        assert (dw.double() - ref.n.sum((0, 1))).abs().max() <= 2.0 ** -8 * 12 * 8
    leaves = [torch.zeros(0, 5, 64, device=DEV).requires_grad_(), weight.requires_grad_()]
    out = layer_norm(*leaves)
    dx, dw = torch.autograd.grad(out.sum(), leaves)
    assert out.shape == dx.shape == (0, 5, 64) and dw.eq(0).all()
    module = LayerNorm(64, device=DEV, dtype=torch.bfloat16)
    assert torch.equal(module(x), layer_norm(x, module.weight, module.bias, module.eps))
    module(x).float().sum().backward()
    assert module.bias.grad.float().eq(12).all()
    with pytest.raises(ValueError):
        LayerNorm((2, 64))


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [128, 2048, 4100])
def test_streams_and_graphs(channels, announce):
    """A call on another stream, and forward and backward captured once and replayed on new inputs."""
    announce()
    g = torch.Generator().manual_seed(channels)
    inputs = [(torch.randn(2, 65, channels, generator=g).to(DEV), torch.randn(2, 65, channels, generator=g).to(DEV))
              for _ in range(4)]
    weight, bias = (torch.randn(2, channels, generator=g).to(DEV).requires_grad_() for _ in range(2))

    def step(x, grad):
        out = layer_norm(x, weight, bias, around_one=True)
        return out.detach(), *torch.autograd.grad(out, (x, weight, bias), grad)

    want = [step(x.clone().requires_grad_(), grad) for x, grad in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step(inputs[0][0].clone().requires_grad_(), inputs[0][1])
        held = inputs[0][0].clone().requires_grad_(), inputs[0][1].clone()
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(there, want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(*held)
    for (x, grad), expected in zip(inputs, want):
        with torch.no_grad():
            held[0].copy_(x)
            held[1].copy_(grad)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, expected))


@pytest.mark.gpu
def test_rows_past_32_bit_offsets(announce):
    """Rows more than 2^32 elements behind the first."""
    announce()
    channels, apart = 1024, 1 << 32
    x = torch.empty(apart + 4 * channels, dtype=torch.bfloat16, device=DEV).as_strided((2, 3, channels),
                                                                                     (apart, channels, 1))
    x.copy_(torch.randn(2, 3, channels, device=DEV))
    out = layer_norm(x)
    assert torch.equal(out, layer_norm(x.contiguous()))
    assert torch.equal(quantize_rows(x).codes, quantize_rows(x.contiguous()).codes)


def _refused(error, call, *args, **kwargs):
    with pytest.raises(error):
        call(*args, **kwargs)


def test_refusals():
    x, w = torch.zeros(2, 8), torch.zeros(8)
    _refused(ValueError, layer_norm, x, w)                                  # not on a GPU
    _refused(ValueError, layer_norm, torch.zeros(()))
    _refused(TypeError, layer_norm, x.double())
    _refused(TypeError, layer_norm, x, w.double())
    _refused(TypeError, layer_norm, x, w.bfloat16())
    _refused(ValueError, layer_norm, x, torch.zeros(3, 8))
    _refused(ValueError, layer_norm, x, torch.zeros(7))
    _refused(ValueError, layer_norm, x, None, torch.zeros(1, 8))
    _refused(ValueError, layer_norm, x, w, eps=-1.0)
    _refused(ValueError, layer_norm, x, w, eps=float("nan"))
    _refused(ValueError, layer_norm, x, around_one=True)
    _refused(ValueError, layer_norm, torch.zeros(2, 0))
    _refused(ValueError, layer_norm, torch.zeros(1, 16385))
    _refused(ValueError, layer_norm_rows, x, w)


@pytest.mark.gpu
def test_refusals_on_the_gpu(announce):
    announce()
    x, w = torch.zeros(2, 8, device=DEV), torch.zeros(8, device=DEV)
    _refused(RuntimeError, layer_norm_rows, x.requires_grad_(), w)
    _refused(ValueError, layer_norm, x, torch.zeros(8))
    out = layer_norm(x, w)
    _refused(RuntimeError, torch.autograd.grad, out, x, torch.ones(3, 2, 8, device=DEV), is_grads_batched=True)
    first, = torch.autograd.grad(layer_norm(x, w), x, torch.ones_like(x), create_graph=True)
    _refused(RuntimeError, torch.autograd.grad, first.sum(), x)
    with torch.autograd.forward_ad.dual_level():
        _refused(RuntimeError, layer_norm, torch.autograd.forward_ad.make_dual(x.detach(), x.detach()))
    many = torch.zeros(65536, 8, device=DEV)
    layer_norm(many, many)
    _refused(ValueError, layer_norm, many, many.clone().requires_grad_())
