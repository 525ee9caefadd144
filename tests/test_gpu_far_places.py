"""Places that lie more than 2^32 bytes apart: a cache's pages, rows to be turned, queries and their gradients."""
import pytest
import torch

from peco_amd.paged import append_pages, paged_attention
from peco_amd.rotary import RotaryAxes, RotaryPositions, rotary_axes
from peco_amd.window import window_attention
from tests.test_gpu_paged import Cache

DEV = "cuda:0"


def _spread(shape, step):
    """A bf16 tensor of that shape whose entries of the first axis are `step` elements apart."""
    dense = torch.empty(shape[1:]).stride()
    return torch.empty(shape[0] * step, dtype=torch.bfloat16, device=DEV).as_strided(shape, (step, *dense))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[1, 1], [40, 200]])
def test_pages(new, announce):
    """Pages 160 MB apart, 7 GB in all: appended to and attended to as a compact cache is."""
    announce()
    cache = Cache(12, [400, 300], 16, 2, 64, torch.bfloat16)
    q, offsets, sizes = cache.queries(new, 4)
    k = torch.randn(q.shape[0], 2, 64, device=DEV).bfloat16()
    turn = RotaryPositions(RotaryAxes((16, 24, 24)), torch.randint(0, 99, (3, q.shape[0]), dtype=torch.int32, device=DEV))
    k_far, v_far = (_spread(cache.k_pages.shape, 80 << 20).copy_(t) for t in (cache.k_pages, cache.v_pages))
    assert k_far.stride(0) * 2 * (k_far.shape[0] - 1) > 1 << 32
    for k_pages, v_pages in ((k_far, v_far), (cache.k_pages, cache.v_pages)):
        append_pages(k, -k, k_pages, v_pages, cache.table, offsets, sizes, rotary=turn)
    for far, near in ((k_far, cache.k_pages), (v_far, cache.v_pages)):
        assert torch.equal(far.contiguous().view(torch.int16), near.view(torch.int16))
    args = (cache.table, offsets, sizes)
    assert torch.equal(paged_attention(q, k_far, v_far, *args, window=90, sinks=5),
                       paged_attention(q, cache.k_pages, cache.v_pages, *args, window=90, sinks=5))


@pytest.mark.gpu
def test_rows_queries_and_gradients(announce):
    announce()
    gen = torch.Generator().manual_seed(13)
    x, g, k, v = (torch.randn(6, 2, 70, 64, generator=gen).bfloat16().to(DEV) for _ in range(4))
    x_far, g_far = (_spread(x.shape, 1 << 29).copy_(t) for t in (x, g))  # 1 GB between batch entries
    axes, positions = RotaryAxes((16, 24, 24)), torch.randint(0, 99, (3, 70), dtype=torch.int32, device=DEV)

    def run(x, g):
        x = x.detach().requires_grad_()
        turned = rotary_axes(x, positions, axes)
        grads = [torch.autograd.grad(turned, x, g)[0]]
        leaves = [x, k.clone().requires_grad_(), v.clone().requires_grad_()]
        out = window_attention(*leaves, (20, 0), 3)
        return [turned.detach(), out.detach(), *grads, *torch.autograd.grad(out, leaves, g)]

    for a, b in zip(run(x_far, g_far), run(x, g)):
        assert torch.equal(a, b)
