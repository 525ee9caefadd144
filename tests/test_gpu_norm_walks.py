"""Layer norm, its codes and its gradients over more rows than one round of workgroups takes: every workgroup walks over
several rows with the next one's loads under way, changes its weight where the walk comes into another batch entry, and
ends on a round that is partly filled."""
import pytest
import torch

from norm_reference import HALF_STEP, U, Norm, quantized
from peco_amd.norm import layer_norm, layer_norm_rows
from peco_amd.projection import quantize_rows

DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]

# shape, entries, and the sets of lanes that share an entry's rows in the gradients at 256 CUs, rounded down. A CU holds 2048
# lanes at most, so a round of the forward kernel takes at most 65536 rows of 64 channels, 32768 of 128, 8192 of 264, 520 and
# (16 bits) 2048, 4096 of 1111 and (fp32) 2048, 1536 of 4100 and 1024 of 16384.
WALKS = [
    ((5, 20001, 64), 5, 6500), ((3, 16001, 128), 3, 5400), ((20001, 264), 0, 4000), ((4, 5003, 520), 4, 500),
    ((9001, 1111), 0, 1000), ((2, 5003, 2048), 2, 500), ((2, 2001, 4100), 2, 128), ((3, 701, 16384), 3, 85),
]


def _inputs(shape, entries, dtype):
    """Rows, fp32 weight and bias, and a gradient of small whole numbers (whose sums are exact)."""
    g = torch.Generator(device=DEV).manual_seed(sum(shape))

    def normal(*s):
        return torch.randn(s, generator=g, device=DEV)

    x = (normal(*shape) * torch.exp(normal(*shape[:-1], 1)) + normal(*shape[:-1], 1)).to(dtype)
    affine = (entries, shape[-1]) if entries else (shape[-1],)
    grad = torch.randint(-3, 4, shape, generator=g, device=DEV).to(dtype)
    return x, normal(*affine) * 0.5, normal(*affine) * 0.5, grad


def _pieces(t):
    """Few enough rows that every workgroup has one: 80 of each entry."""
    return t.split(80, t.dim() - 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,entries,sets", WALKS)
def test_rows(shape, entries, sets, dtype, announce):
    announce()
    x, weight, bias, _ = _inputs(shape, entries, dtype)
    for w, b, around in ((weight, bias, False), (weight.to(dtype), bias.to(dtype), True)):
        ref = Norm(x, w, b, 1e-5, around)
        out = layer_norm(x, w, b, 1e-5, around_one=around)
        assert ((out.double() - ref.out).abs() <= ref.out_bound()).all()
        assert torch.equal(out, torch.cat([layer_norm(p, w, b, 1e-5, around_one=around) for p in _pieces(x)], -2))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,entries,sets", WALKS)
def test_codes(shape, entries, sets, dtype, announce):
    """The norm's codes within half a step of the row and what fp32 leaves of the norm (the codes' factor has three roundings,
    the scale two: together below 2^-21 of the largest value); a tensor's codes as they are defined."""
    announce()
    x, weight, bias, _ = _inputs(shape, entries, dtype)
    ref = Norm(x, weight, bias, 1e-5, True)
    rows = layer_norm_rows(x, weight, bias, 1e-5, around_one=True)
    most = ref.out.abs().amax(-1, keepdim=True)
    off = ref.out_off.amax(-1, keepdim=True) + 2.0 ** -21 * most
    assert ((rows.dequantize(torch.float64) - ref.out).abs() <= most / 254 + off).all()
    assert ((rows.scales.double() * 127)[..., None] - most).abs().le(off).all()
    parts = [layer_norm_rows(p, weight, bias, 1e-5, around_one=True) for p in _pieces(x)]
    assert torch.equal(rows.codes, torch.cat([p.codes for p in parts], -2))
    assert torch.equal(rows.scales, torch.cat([p.scales for p in parts], -1))
    rows, (codes, scales) = quantize_rows(x), quantized(x)
    assert torch.equal(rows.codes.cpu(), codes) and torch.equal(rows.scales.cpu(), scales)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,entries,sets", WALKS)
def test_gradients(shape, entries, sets, dtype, announce):
    """dx as that of a few rows and within its bound, db exact, dw within what the order of its sums leaves: a set of lanes
    takes rows in turn, then up to 8 lanes and 8 sets of a workgroup and 512 workgroups (32 in turn, 16 wavefronts) are
    joined, less than 64 additions."""
    announce()
    x, weight, bias, grad = _inputs(shape, entries, dtype)
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    dx, dw, db = torch.autograd.grad(layer_norm(*leaves, 1e-5), leaves, grad)
    parts = []
    for p, g in zip(_pieces(x.detach()), _pieces(grad)):
        p.requires_grad_()
        parts.append(torch.autograd.grad(layer_norm(p, weight.detach(), bias.detach(), 1e-5), p, g)[0])
    assert torch.equal(dx, torch.cat(parts, -2))
    ref, d = Norm(x.detach(), weight.detach(), bias.detach(), 1e-5, False), grad.double()
    (want, bound), (dw_ref, _), (db_ref, _) = ref.gradients(grad, entries > 0)
    assert ((dx.double() - want).abs() <= bound).all()
    over = 1 if entries else 0
    assert torch.equal(db.double(), db_ref)
    chain = shape[-2] // sets + 1 + 64
    off = ((chain + 2) * U * (d * ref.n).abs() + d.abs() * ref.n_off).sum(over) + HALF_STEP[torch.float32] * dw_ref.abs()
    assert ((dw.double() - dw_ref).abs() <= off).all()
    # A check of the bound itself: sums without one row, or with one twice, are outside it in most columns.
    assert ((d * ref.n).abs().select(over, shape[-2] // 2) > off).double().mean() > 0.5


@pytest.mark.gpu
def test_weights_of_two_types_and_shapes(announce):
    """One weight for all rows beside a bias an entry and the other way round: the shared one's gradient is the two entries'
    sums added (one more rounding), and one to its type."""
    announce()
    g = torch.Generator().manual_seed(23)
    x = torch.randn(2, 6, 64, generator=g).to(DEV).bfloat16()
    grad = torch.randn(2, 6, 64, generator=g).to(DEV).bfloat16()
    one, each = torch.randn(64, generator=g).to(DEV), torch.randn(2, 64, generator=g).to(DEV)
    for w, b in ((one, each.bfloat16()), (one.bfloat16(), each), (each, one.bfloat16()), (each.bfloat16(), one)):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        got = torch.autograd.grad(layer_norm(*leaves), leaves, grad)
        ref, d = Norm(x, w, b, 1e-6, False), grad.double()
        (dx, bound), *_ = ref.gradients(grad, True)
        assert ((got[0].double() - dx).abs() <= bound).all()
        chain = 6 // 256 + 1 + 64
        for leaf, value, term, off in ((w, got[1], d * ref.n, d.abs() * ref.n_off), (b, got[2], d, torch.zeros_like(d))):
            over = (0, 1) if leaf.dim() == 1 else 1
            want = term.sum(over)
            limit = ((chain + 3) * U * term.abs() + off).sum(over) + HALF_STEP[leaf.dtype] * 1.01 * want.abs()
            assert value.shape == leaf.shape and value.dtype == leaf.dtype
            assert ((value.double() - want).abs() <= limit).all()
