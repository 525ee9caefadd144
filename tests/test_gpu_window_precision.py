"""How far the windowed attention's results are off in the mean, against a model of the roundings that its kernels name;
gradients against differences along their own direction; generation from a cache within each step's bounds."""
import math

import pytest
import torch

from peco_amd import _native
from peco_amd.paged import append_pages, paged_attention
from peco_amd.rotary import RotaryAxes, RotaryPositions, rotary_axes
from peco_amd.window import window_attention
from tests.window_reference import gradients, rows, seen_keys

DEV = "cuda:0"


def _rounded(x, dtype):
    return x.to(dtype).double()


def _head(q, k, v, g, seen, scale, dtype=None, fine=False, rest=True, low=0.0):
    """(out, dq, dk, dv) of one head in 64 bits. With ``dtype`` the roundings of the kernels: weights relative to a row's
    largest score (``low``: to one that many powers of e below it), summed as rounded; delta from the output and what its
    rounding left (``rest``: or from the rounded output alone); weights and dS rounded for their products (fp16: times
    powers of two that keep them out of the subnormal numbers); results rounded. ``fine``: gradients rounded alone."""
    s = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    w = torch.exp(s - s.amax(1, keepdim=True) + low)
    total = (w if dtype is None else _rounded(w, dtype)).sum(1, keepdim=True)
    out = (w if dtype is None else _rounded(w, dtype)) @ v / total
    if dtype is not None and fine:
        return [_rounded(t, dtype) for t in (out, *_head(q, k, v, g, seen, scale)[1:])]
    w = w / total
    for_delta = out
    if dtype is not None:
        for_delta = _rounded(out, dtype)
        for_delta = for_delta + _rounded(out - for_delta, dtype) if rest else for_delta
    d_s = w * (g @ v.T - (g * for_delta).sum(1, keepdim=True))
    if dtype is None:
        return out, scale * d_s @ k, scale * d_s.T @ q, w.T @ g
    up, by = 1.0, 1.0
    if dtype == torch.float16:
        up, by = 2.0 ** 14, 2.0 ** (14 - math.frexp(2 * float(g.norm(dim=1).max() * v.norm(dim=1).max()))[1])
    d_s = _rounded(d_s * by, dtype) / by
    return [_rounded(t, dtype) for t in (out, scale * d_s @ k, scale * d_s.T @ q, (_rounded(w * up, dtype) / up).T @ g)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("left", [1, 3, 7, 15])
@pytest.mark.parametrize("sinks", [0, 300])
def test_mean_errors_are_those_of_the_named_roundings(sinks, left, dim, dtype, announce):
    """Windows of 2 to 16 keys, where dS is a small difference and the weights are few: root mean squares over 4 heads of
    2000 rows, against the model's on the same inputs. Windows alone are fine calls, whose gradients are as good as their
    own rounding; with 300 sinks, whose scores lie 64 below all others here (weights below 2^-80), they are not, and
    weights, dS and delta come in as rounded. Two such means over 8000 rows of errors whose fourth moment is at most 30
    times the square of their second differ by chance by sqrt(2 * 29 / 4 / 8000) = 4% of each other at one standard
    deviation if the rows' channels all err together; they err apart, dim channels a row, and most roundings are the same
    on both sides. Twice the 4%, 8%, is allowed. An output whose rounding's rest is lost, or weights relative to less than
    the maximum (e^5 times; a power of two would change no rounding), make the gradients 11% to 75% worse, and a fine
    call's as rounded elsewhere 40% and more: told apart below."""
    announce()
    heads, n, scale = 4, 2000, dim ** -0.5
    gen = torch.Generator().manual_seed(left)
    q, k, v, g = (torch.randn(1, heads, n, dim, generator=gen) * x for x in (1.5, 1.0, 1.0, 1.0))
    if sinks:
        q[..., 0], k[..., 0], k[:, :, :sinks, 0] = 16, 0, -4 / scale
    q, k, v, g = (t.to(dtype).to(DEV) for t in (q, k, v, g))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = window_attention(*leaves, (left, 0), sinks)
    got = [out.detach(), *torch.autograd.grad(out, leaves, g)]
    seen = seen_keys(torch.arange(n, device=DEV), n, left, 0, sinks)
    others = {"coarse": {}} if not sinks else {"no rest": {"rest": False}, "low": {"low": 5.0}}
    squares = {name: [0.0] * 4 for name in ("kernel", "model", *others)}
    first = sinks + left  # (queries among the sinks see them alone, all alike: the weights are as elsewhere, few rows)
    for h in range(heads):
        args = [t[0, h].double() for t in (q, k, v, g)]
        right = _head(*args, seen, scale)
        results = {"kernel": [t[0, h].double() for t in got], "model": _head(*args, seen, scale, dtype, fine=not sinks),
                   **{name: _head(*args, seen, scale, dtype, **how) for name, how in others.items()}}
        for name, parts in results.items():
            for i, (a, b) in enumerate(zip(parts, right)):
                squares[name][i] += float((a - b)[first:].square().sum())
    size = {name: [math.sqrt(x / y) for x, y in zip(parts, squares["model"])] for name, parts in squares.items()}
    print({name: [round(x, 3) for x in parts] for name, parts in size.items()})
    for i, what in enumerate(("out", "dq", "dk", "dv")):
        assert size["kernel"][i] <= 1.08, (what, size)
        assert what not in ("dq", "dk") or min(size[name][i] for name in others) > 1.08, (what, size)


def test_which_calls_are_fine():
    """Up to 8 keys a query, or up to 2^20 pairs of a query and a key: their workspace holds a second number a row."""
    lib = _native.library()

    def numbers(batch, q_heads, kv_heads, queries, keys, left, right, sinks):
        floats = lib.peco_window_attention_grad_workspace_size(batch, q_heads, kv_heads, queries, keys, left, right, sinks, 128, 1)
        return floats / (batch * q_heads * queries)

    # (bf16, enough key tiles for walks in one part: nothing but the rows' numbers.)
    assert 2 <= numbers(1, 24, 24, 32896, 32896, 7, 0, 0) < 2.01
    assert 2 <= numbers(1, 24, 24, 32896, 32896, 3, 4, 0) < 2.01
    assert 1 <= numbers(1, 24, 24, 32896, 32896, 8, 0, 0) < 1.01
    assert 1 <= numbers(1, 24, 24, 32896, 32896, 2025, 0, 0) < 1.01
    assert 2 <= numbers(128, 8, 8, 32, 32, -1, 0, 0) < 2.01      # 2^15 rows of 32 keys
    assert 1 <= numbers(128, 8, 8, 33, 33, -1, 0, 0) < 1.01


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("at", [3, 700, 1990])
def test_values_that_are_not_seen_in_calls_that_are_not_fine(at, which, bad, dim, announce):
    """A NaN or infinity in one row of q, k, v or the gradient reaches the gradients of rows that it meets, and no other
    bit of any. 4 x 2000 rows of up to 305 keys."""
    announce()
    gen = torch.Generator().manual_seed(6)
    n, left, sinks = 2000, 300, 4
    clean = [torch.randn(1, h, n, dim, generator=gen).bfloat16().to(DEV) for h in (4, 2, 2, 4)]

    def run(q, k, v, g):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(window_attention(*leaves, (left, 0), sinks), leaves, g)

    want = run(*clean)
    tensors = [t.clone() for t in clean]
    tensors[which][0, 1, at, 7] = bad
    got = run(*tensors)
    seen = seen_keys(torch.arange(n), n, left, 0, sinks)
    queries = seen[:, at] if which in (1, 2) else torch.arange(n) == at  # rows of P that it may reach
    q_heads, kv_head = ([2, 3], 1) if which in (1, 2) else ([1], 0)
    keys = seen[queries].any(0)
    for i, (heads, reached) in enumerate(((q_heads, queries), ([kv_head], keys), ([kv_head], keys))):
        for h in range(got[i].shape[1]):
            same = ~reached.to(DEV) if h in heads else torch.ones(n, dtype=torch.bool, device=DEV)
            assert torch.equal(got[i][0, h, same], want[i][0, h, same]), ("qkv"[i], h)
    assert not torch.isfinite(got[0][0, q_heads[0], queries.to(DEV)]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_differences_along_the_gradient(which, dtype, announce):
    """The 64-bit function's central difference along the 64-bit gradient of q, k or v (the way in which a gradient that is
    zero, turned or scaled shows most), against the kernels' gradient times that way. Room: rows err apart, each by at
    most its elements' bounds; such a sum stays within 6 root sums of squares but once in 2^25 (Hoeffding). The
    difference's own third-order term is 2^-24 of it times the derivative's size, below 2^-9 of it here."""
    announce()
    gen = torch.Generator().manual_seed(3)
    q, k, v, g = (torch.randn(1, h, n, 64, generator=gen).to(dtype).to(DEV) for h, n in ((4, 150), (2, 190), (2, 190), (4, 150)))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(window_attention(*leaves, (60, 5), 7), leaves, g)
    refs, bounds = gradients(q, k, v, g, 60, 5, 7)
    way = refs[which] / refs[which].norm()
    seen, step, sums = seen_keys(torch.arange(40, 190, device=DEV), 190, 60, 5, 7), 2.0 ** -12, []
    for sign in (1, -1):
        moved = [t.double() for t in (q, k, v)]
        moved[which] = moved[which] + sign * step * way
        sums.append(sum((torch.softmax((moved[0][0, h] @ moved[1][0, h // 2].T / 8).masked_fill(~seen, -math.inf), -1) @
                         moved[2][0, h // 2] * g[0, h].double()).sum() for h in range(4)))
    difference = float(sums[0] - sums[1]) / (2 * step)
    product = float((grads[which].double() * way).sum())
    room = 6 * float((bounds[which] * way.abs()).sum(-1).square().sum().sqrt()) + 2.0 ** -9 * abs(difference)
    assert abs(difference - product) <= room
    assert difference > 4 * room  # (no gradient, half of it or one turned round would be told apart)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,queries,window,sinks", [(2, 300, (200, 0), 20), (8, 700, (-1, 0), 0)])  # fine, and not
def test_far_rows_backward(heads, queries, window, sinks, announce):
    """Key or value rows spread over more than 2^32 bytes (a view of a large buffer): the gradients of the compact call."""
    announce()
    keys, step = 700, 1 << 22  # 8 MiB between rows: 5.9 GB from first to last
    gen = torch.Generator().manual_seed(4)
    q, k, v, g = (torch.randn(1, h, n, 64, generator=gen).bfloat16().to(DEV)
                  for h, n in ((heads, queries), (1, keys), (1, keys), (heads, queries)))
    buffer = torch.empty(keys * step, dtype=torch.bfloat16, device=DEV)
    far = buffer.as_strided((1, 1, keys, 64), (step * keys, step * keys, step, 1))

    def run(*tensors):
        leaves = [t.detach().requires_grad_() for t in tensors]
        return torch.autograd.grad(window_attention(*leaves, window, sinks), leaves, g)

    want = run(q, k, v)
    for i in (1, 2):
        far.copy_((k, v)[i - 1])
        assert all(torch.equal(a, b) for a, b in zip(run(*[far if j == i else t for j, t in enumerate((q, k, v))]), want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_generation_within_each_step_s_bounds(dtype, announce):
    """A prompt, a frame of 9 tokens, then single tokens: every step's keys turned and appended, its queries turned and
    attended; each output within its own bound (64 bits, from the turned rows) and the cache's rows those turned rows."""
    announce()
    heads, kv_heads, dim, page, window, sinks = 4, 2, 64, 16, 40, 4
    steps = [75, 9, 1, 1, 1, 9, 1]
    total, axes = sum(steps), RotaryAxes((16, 24, 24), 256.0)
    gen = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(total, h, dim, generator=gen).to(dtype).to(DEV) for h in (heads, kv_heads, kv_heads))
    positions = torch.stack([torch.arange(total) // 9, torch.arange(total) % 9 // 3, torch.arange(total) % 3]).int().to(DEV)
    turned = [rotary_axes(t.transpose(0, 1)[None], positions, axes)[0].transpose(0, 1) for t in (q, k)]
    k_pages, v_pages = (torch.full((9, kv_heads, page, dim), float("nan"), dtype=dtype, device=DEV) for _ in "kv")
    table = torch.tensor([[5, 2, 7, 0, 1, 3, 8]], dtype=torch.int32, device=DEV)
    outs, at = [], 0
    for n in steps:
        part, ends = slice(at, at + n), [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, n], [at + n])]
        append_pages(k[part], v[part], k_pages, v_pages, table, *ends, rotary=RotaryPositions(axes, positions[:, part]))
        outs.append(paged_attention(turned[0][part], k_pages, v_pages, table, *ends, window=window, sinks=sinks))
        at += n
    out, j = torch.cat(outs), torch.arange(total, device=DEV)
    places = table[0, j // page].long(), j % page
    assert torch.equal(k_pages[places[0], :, places[1]], turned[1])
    assert torch.equal(v_pages[places[0], :, places[1]], v)
    seen = seen_keys(j, total, window, 0, sinks)
    for h in range(heads):
        ref, bound = rows(turned[0][:, h], turned[1][:, h // 2], v[:, h // 2], seen, dim ** -0.5)[:2]
        assert ((out[:, h].double() - ref).abs() <= bound).all()
        # (Bounds of a few times 2^-8 of the mean of |v| in bf16, an eighth of that in fp16: outputs are told from 0.)
        assert float(bound.mean()) < 0.2 * float(ref.abs().mean())
