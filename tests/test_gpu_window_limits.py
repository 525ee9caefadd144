"""Attention with a window and sinks at the limits of its inputs: scores of any size and values at the types' ends."""
import pytest
import torch

from peco_amd.window import window_attention
from tests.window_reference import seen_keys

DEV = "cuda:0"


def _gradients(q, k, v, g, window, sinks, **more):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = window_attention(*leaves, window, sinks, **more)
    return out.detach(), torch.autograd.grad(out, leaves, g)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 2.0 ** 10), (torch.bfloat16, 2.0 ** 30), (torch.float16, 2.0 ** 12)])
@pytest.mark.parametrize("left,right,sinks", [(-1, -1, 0), (80, 0, 3)])
def test_gradients_of_large_scores(dim, dtype, size, left, right, sinks, announce):
    """One weight of 1 a query and others of 0: its key's dV is the sum of such queries' gradients, which the products
    of 1 with 16-bit numbers give up to fp32 sums (200 terms: 2^-16 of their sizes) and one rounding.

    The backward pass forms the scores again: every fp32 sum has to come out as in the forward, since at these sizes
    (scaled scores past 2^16, steps of fp32 there 2^-8 and more) another order of the channels moves the exponents by
    whole numbers. Queries whose two largest scores are apart by less than 2^7 are given no gradient."""
    announce()
    unit = torch.finfo(dtype).eps / 2
    g0 = torch.Generator().manual_seed(8)
    q = (torch.sign(torch.randn(1, 2, 200, dim, generator=g0)) * size).to(dtype).to(DEV)
    k = (torch.randn(1, 2, 200, dim, generator=g0) * size).to(dtype).to(DEV)
    v, g = (torch.randn(1, 2, 200, dim, generator=g0).to(dtype).to(DEV) for _ in range(2))
    s = (q.double() @ k.double().transpose(2, 3).contiguous()).masked_fill(
        ~seen_keys(torch.arange(200), 200, left, right, sinks).to(DEV), -float("inf"))
    top = s.topk(2, -1)
    # (fp32 sums of `dim` terms are off by dim 2^-24 of the terms' sizes, which are at most 2^5 of the score's here.)
    clear = (top.values[..., 0] - top.values[..., 1]) * dim ** -0.5 > 2.0 ** 7 + 2.0 ** -12 * top.values[..., 0].abs()
    clear |= ~torch.isfinite(top.values[..., 1])
    assert clear.float().mean() > 0.8
    g = g * clear[..., None]
    out, grads = _gradients(q, k, v, g, (left, right), sinks)
    index = top.indices[..., :1].expand(-1, -1, -1, dim)
    assert torch.equal(out[clear], v.gather(2, index)[clear])
    want, mass = (torch.zeros(v.shape, dtype=torch.float64, device=DEV).scatter_add_(2, index, t.double())
                  for t in (g, g.abs()))
    assert ((grads[2].double() - want).abs() <= unit * want.abs() + 2.0 ** -16 * mass).all()
    assert all(torch.isfinite(t).all() for t in grads)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("which,dim", [(2, 64), (3, 64), (2, 128), (3, 128)])
def test_fp16_gradients_beside_an_infinity(which, dim, bad, announce):
    """An infinity or NaN in one row of v or of the gradient leaves the gradients of rows that do not meet it as they
    were, bit for bit. Their dS is far below fp16's steps without a factor (weights of one in 1500 of gradients of
    2^-14), and that factor comes from the lengths of the head's rows (the longest are others here)."""
    announce()
    gen = torch.Generator().manual_seed(15)
    sk, left = 2600, 1500
    q, k, v, g = (torch.randn(1, 2, sk, dim, generator=gen) for _ in range(4))
    # (Weights as of a scale of 1 / sqrt(D), while dQ = scale dS K and dK = scale dS^T Q are 2^6 times larger.)
    q, k = q * 2.0 ** -6, k * 2.0 ** -6
    g[:, :, 9], v[:, :, 9] = 2 * g.norm(dim=-1).amax() * dim ** -0.5, 2 * v.norm(dim=-1).amax() * dim ** -0.5
    clean = [t.half().to(DEV) for t in (q, k, v, g * 2.0 ** -14)]
    scale = 2.0 ** 12 * dim ** -0.5
    _, want = _gradients(*clean, (left, 0), 0, scale=scale)
    changed = [t.clone() for t in clean]
    changed[which][0, 1, 5, 3] = bad
    out, got = _gradients(*changed, (left, 0), 0, scale=scale)
    for i, first in enumerate((1700, 1800, 1800) if which == 2 else (200, 300, 300)):  # (whole tiles past the last reached)
        part = got[i][:, 1, first:]
        assert torch.isfinite(part).all() and (part != 0).float().mean() > 0.9
        assert torch.equal(part, want[i][:, 1, first:])
        assert torch.equal(got[i][:, 0], want[i][:, 0])
    assert not torch.isfinite(got[0][0, 1, 5]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [float("inf"), 2.0 ** 14])
@pytest.mark.parametrize("rows,left", [(200, 30), (1500, 800)])  # fine gradients, and not
def test_a_row_s_neighbours_do_not_change_its_bits(rows, left, size, dtype, announce):
    """One query is infinite, or so large that its scores take another form of the exponent: the rows beside it, in its
    tile and in its wavefront, come out bit for bit as they did, and so does their gradient."""
    announce()
    gen = torch.Generator().manual_seed(16)
    q, k, v, g = (torch.randn(1, 2, rows, 64, generator=gen).to(dtype).to(DEV) for _ in range(4))
    q *= 2
    changed, at = q.clone(), rows - 77
    changed[0, 1, at] *= size
    want, got = (_gradients(t, k, v, g, (left, 0), 3) for t in (q, changed))
    others = torch.arange(rows, device=DEV) != at
    assert torch.equal(got[0][:, :, others], want[0][:, :, others])
    assert torch.equal(got[1][0][:, :, others], want[1][0][:, :, others])
    assert not torch.equal(got[0][0, 1, at], want[0][0, 1, at])
