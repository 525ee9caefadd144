"""Every key and every query row counts once: inputs whose weights are all equal, where one lost or doubled term shows.

With q = 0 (or k = 0) every score is 0 and a query's weights are 1 / n over the n keys it sees, exactly so in the running
sums (whole numbers below 2^24). Values, keys, queries and gradients that are one-hot in (index modulo D) then make each
result a sum of a few dozen terms of one size, so that a single term exceeds the bound, which comes from the roundings:
u = half a step of the type for weights and dS, u for the result, 2^-18 relative for exponentials, divisions and fp32 sums
(measured against n < 2^14 terms of 2^-24 each, of equal sign), and u^2 for the output with its rest that delta is taken
from. Each test also checks that an oracle that misses one key (or row) is told apart.
"""
import pytest
import torch

from peco_amd.paged import paged_attention
from peco_amd.window import window_attention
from tests.test_gpu_paged import Cache
from tests.window_reference import UNIT, seen_keys

DEV = "cuda:0"
FINE = 2.0 ** -18

CASES = [
    # query heads, key heads, queries, keys, left, right, sinks
    (1, 1, 1, 1, -1, 0, 0),
    (2, 2, 65, 65, 16, 0, 3),
    (2, 1, 129, 200, 31, 0, 7),
    (1, 1, 1, 5000, -1, 0, 0),          # one token: the walk in many parts
    (3, 1, 3, 4099, 2000, 0, 100),
    (2, 2, 130, 4000, -1, 0, 0),
    (1, 1, 2500, 2500, -1, -1, 0),      # few row and key tiles: every walk in parts
    (2, 1, 1300, 1300, 600, 0, 130),    # sinks of two tiles of the gradients' walks
    (1, 1, 3000, 3000, 200, 30, 300),
    (6, 2, 333, 777, 100, 100, 5),
]


def _one_hot(rows, dim):
    return torch.eye(dim, dtype=torch.float64, device=DEV)[torch.arange(rows, device=DEV) % dim]


def _signs(seed, *shape):
    return torch.randint(0, 2, shape, generator=torch.Generator().manual_seed(seed)).double().mul_(2).sub_(1).to(DEV)


def _weights(seen):
    return seen.double() / seen.sum(1, keepdim=True).clamp_min(1)


def _told_apart(got, right, wrong, bound, reached):
    """Within the bound of the right values; in the rows that miss a term, not within it of the wrong ones."""
    assert ((got.double() - right).abs() <= bound).all(), float(((got.double() - right).abs() - bound).max())
    miss = ((got.double() - wrong).abs() > bound).any(-1)
    assert miss[reached].all(), f"{int((~miss[reached]).sum())} of {int(reached.sum())} rows do not tell"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_heads,kv_heads,sq,sk,left,right,sinks", CASES)
def test_forward(q_heads, kv_heads, sq, sk, left, right, sinks, dim, dtype, announce):
    announce()
    q = torch.zeros(1, q_heads, sq, dim, dtype=dtype, device=DEV)
    k = torch.randn(1, kv_heads, sk, dim, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    v = _one_hot(sk, dim)
    out = window_attention(q, k, v.to(dtype).expand(1, kv_heads, -1, -1), (left, right), sinks)[0]
    seen = seen_keys(torch.arange(sk - sq, sk, device=DEV), sk, left, right, sinks)
    want = _weights(seen) @ v
    bound = (UNIT[dtype] + FINE) * want
    for lost in {0, sk // 2, sk - 1}:
        less = seen.clone()
        less[:, lost] = False
        reached = seen[:, lost] & (seen.sum(1) > 1)
        for h in range(q_heads):
            _told_apart(out[h], want, _weights(less) @ v, bound, reached)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,left,sinks", [(16, -1, 0), (100, 1000, 40), (128, 70, 0)])
def test_paged(page, left, sinks, dtype, announce):
    announce()
    dim, heads, lengths, new = 128, 2, [1, 64, 65, 5000, 700, 9000], [1, 1, 3, 1, 200, 2]
    cache = Cache(11, lengths, page, heads, dim, dtype)
    for b, n in enumerate(lengths):
        j = torch.arange(n, device=DEV)
        cache.v_pages[cache.table[b, j // page].long(), :, j % page] = _one_hot(n, dim).to(dtype)[:, None]
    q, offsets, sizes = cache.queries(new, 2 * heads)
    out = paged_attention(torch.zeros_like(q), cache.k_pages, cache.v_pages, cache.table, offsets, sizes, window=left, sinks=sinks)
    at = 0
    for n, fresh in zip(lengths, new):
        seen, v = seen_keys(torch.arange(n - fresh, n, device=DEV), n, left, 0, sinks), _one_hot(n, dim)
        want = _weights(seen) @ v
        lost = n - fresh
        less = seen.clone()
        less[:, lost] = False
        for h in range(2 * heads):
            _told_apart(out[at:at + fresh, h], want, _weights(less) @ v, (UNIT[dtype] + FINE) * want,
                        seen[:, lost] & (seen.sum(1) > 1))
        at += fresh


TINY = 2.0 ** -25  # half of fp16's smallest step


def _products(weights, d_s, x, unit, scale):
    """scale times a product of dS with x (summed over its first axis), and its bound."""
    r = scale * (d_s.T @ x)
    return r, scale * ((d_s.abs() * (unit + FINE) + weights * (unit ** 2 + FINE)).T @ x.abs()) + unit * r.abs() + TINY


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_heads,kv_heads,sq,sk,left,right,sinks", CASES)
def test_gradients(q_heads, kv_heads, sq, sk, left, right, sinks, dim, dtype, announce):
    announce()
    unit, group, scale = UNIT[dtype], q_heads // kv_heads, dim ** -0.5
    seen = seen_keys(torch.arange(sk - sq, sk, device=DEV), sk, left, right, sinks)
    weights, d = _weights(seen), torch.arange(dim, device=DEV)

    def run(q, k, v, g):
        leaves = [t.to(dtype).expand(1, heads, -1, -1).clone().requires_grad_()
                  for t, heads in ((q, q_heads), (k, kv_heads), (v, kv_heads))]
        out = window_attention(*leaves, (left, right), sinks)
        return torch.autograd.grad(out, leaves, g.to(dtype).expand(1, q_heads, -1, -1))

    def d_s(w, g, v):
        dp = g @ v.T
        return w * (dp - (w * dp).sum(1, keepdim=True))

    # dQ: keys one-hot, dP the sign of each key's one value.
    zeros, v, g = torch.zeros(sq, dim, dtype=torch.float64, device=DEV), torch.zeros(sk, dim, dtype=torch.float64, device=DEV), \
        torch.zeros(sq, dim, dtype=torch.float64, device=DEV)
    v[:, 0], g[:, 0] = _signs(2, sk), 1
    dq = run(zeros, _one_hot(sk, dim), v, g)[0][0]
    want, bound = _products(weights.T, d_s(weights, g, v).T, _one_hot(sk, dim), unit, scale)
    less = seen.clone()
    less[:, sk // 2] = False
    wrong = _products(weights.T, d_s(_weights(less), g, v).T, _one_hot(sk, dim), unit, scale)[0]
    # (Rows of few keys have dS near 0: a value equal to their mean says nothing.)
    reached = less.any(1) & seen[:, sk // 2] & (seen.sum(1) > 64)
    for h in range(q_heads):
        _told_apart(dq[h], want, wrong, bound, reached)

    # dK and dV: queries and gradients one-hot, values signs.
    q, v = _one_hot(sq, dim), _signs(3, sk, dim)
    grads = run(q, torch.zeros(sk, dim, dtype=torch.float64, device=DEV), v, q)
    want, bound = _products(weights, d_s(weights, q, v), q, unit, scale * group)
    want_v, mass = group * (weights.T @ q), group * (weights.T @ q)
    bound_v = (unit + FINE) * mass + unit * want_v + TINY
    lost = sq - 1 - (sq - 1) // 3  # (a row that other rows' neighbours see keys of as well)
    less = weights.clone()
    less[lost] = 0
    reached = seen[lost] & (seen.sum(1)[lost] > 64)
    # (One head's row is lost, not the group's.)
    wrong = want - (want - _products(less, d_s(less, q, v), q, unit, scale * group)[0]) / group
    wrong_v = want_v - (weights - less).T @ q
    for h in range(kv_heads):
        _told_apart(grads[1][0, h], want, wrong, bound, reached)
        _told_apart(grads[2][0, h], want_v, wrong_v, bound_v, seen[lost])
