"""Gradients of the attention with a window and sinks against the formula in 64 bits and against differences."""
import ctypes

import pytest
import torch

from peco_amd import _native
from peco_amd.window import window_attention
from tests.window_reference import gradients, seen_keys

DEV = "cuda:0"


def _inputs(seed, batch, q_heads, kv_heads, sq, sk, dim, dtype, size=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = [torch.randn(batch, heads, n, dim, generator=g).to(dtype).to(DEV)
               for heads, n in ((q_heads, sq), (kv_heads, sk), (kv_heads, sk))]
    return q, k, v, (torch.randn(q.shape, generator=g) * size).to(dtype).to(DEV)


def _gradients(q, k, v, g, window, sinks, **more):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = window_attention(*leaves, window, sinks, **more)
    return out.detach(), torch.autograd.grad(out, leaves, g)


def _near(grads, refs, bounds):
    for name, got, ref, bound in zip("qkv", grads, refs, bounds):
        assert torch.isfinite(got).all(), name
        off = (got.double() - ref).abs() - bound
        assert (off <= 0).all(), f"d{name} off by {float(off.max()):.3e} more than the bound at {int(off.argmax())}"


CASES = [
    # batch, query heads, key heads, queries, keys, left, right, sinks
    (1, 1, 1, 1, 1, -1, 0, 0),
    (1, 2, 1, 2, 2, 0, 0, 0),
    (2, 4, 2, 65, 65, 16, 0, 3),
    (1, 3, 3, 64, 64, -1, -1, 0),
    (1, 3, 1, 129, 129, 31, 0, 0),
    (2, 6, 2, 300, 300, 40, 0, 200),
    (1, 2, 2, 257, 641, 100, 0, 5),
    (1, 2, 2, 70, 33, -1, 0, 0),
    (1, 2, 1, 70, 33, 3, 0, 2),
    (1, 2, 2, 200, 90, 4, 30, 0),
    (1, 1, 1, 500, 500, 0, 0, 1),
    (1, 2, 2, 400, 400, 63, 64, 0),
    (1, 2, 2, 400, 400, 20, 17, 50),
    (1, 2, 2, 333, 333, 10, -1, 400),
    (1, 2, 2, 333, 333, 1 << 40, 1 << 40, 1 << 40),
    (1, 2, 1, 1, 300, -1, 0, 0),
    (1, 2, 1, 3, 1500, 1000, 0, 100),
    (1, 4, 2, 3000, 3000, 200, 0, 130),  # long walks of two sink tiles, in parts
    (1, 1, 1, 2500, 2500, -1, 0, 0),     # few key tiles: every walk in parts
    (1, 24, 24, 700, 700, 255, 0, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,q_heads,kv_heads,sq,sk,left,right,sinks", CASES)
def test_gradients(batch, q_heads, kv_heads, sq, sk, left, right, sinks, dim, dtype, announce):
    announce()
    q, k, v, g = _inputs(sq + sk, batch, q_heads, kv_heads, sq, sk, dim, dtype)
    out, grads = _gradients(q, k, v, g, (left, right), sinks)
    _near(grads, *gradients(q, k, v, g, left, right, sinks))
    assert torch.equal(out, window_attention(q, k, v, (left, right), sinks))
    _, again = _gradients(q, k, v, g, (left, right), sinks)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    hidden = ~seen_keys(torch.arange(sk - sq, sk), sk, left, right, sinks)
    assert (grads[0][:, :, hidden.all(1).to(DEV)] == 0).all()
    assert all((t[:, :, hidden.all(0).to(DEV)] == 0).all() for t in grads[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -10, 2.0 ** 5, 2.0 ** 10])
def test_fp16_gradients_of_any_size(size, announce):
    """Weights of one in 2000 and gradients down to fp16's subnormals: products taken in range."""
    announce()
    q, k, v, g = _inputs(2, 1, 2, 2, 2000, 2000, 64, torch.float16, size)
    _, grads = _gradients(q, k, v, g, (-1, -1), 0)
    _near(grads, *gradients(q, k, v, g, -1, -1, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_against_differences(dtype, announce):
    """The 64-bit function's central differences along a direction (step 2^-12: third-order terms of size 2^-24
    times a third derivative of at most 2^6 in the scores' units; 2^-9 of the sums covers them) against the
    gradients' products with it, within the gradients' own bounds."""
    announce()
    q, k, v, g = _inputs(3, 1, 4, 2, 150, 190, 64, dtype)
    _, grads = _gradients(q, k, v, g, (60, 5), 7)
    _, bounds = gradients(q, k, v, g, 60, 5, 7)
    gen = torch.Generator().manual_seed(4)
    for i, (t, grad, bound) in enumerate(zip((q, k, v), grads, bounds)):
        way, step = torch.randn(t.shape, generator=gen).to(DEV).double(), 2.0 ** -12
        sums = []
        for sign in (1, -1):
            moved = [x.double() for x in (q, k, v)]
            moved[i] = moved[i] + sign * step * way
            w = moved[0] @ moved[1].repeat_interleave(2, 1).transpose(2, 3).contiguous() / 8
            w = torch.softmax(w.masked_fill(~seen_keys(torch.arange(40, 190, device=DEV), 190, 60, 5, 7), -1e30), -1)
            sums.append(((w @ moved[2].repeat_interleave(2, 1)) * g.double()).sum())
        difference = float(sums[0] - sums[1]) / (2 * step)
        product = float((grad.double() * way).sum())
        room = float((bound * way.abs()).sum()) + 2.0 ** -9 * float(g.double().norm())
        assert abs(difference - product) <= room


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_padded_batch(dtype, announce):
    """Rows behind a sequence's length take and give no gradient, whatever they hold."""
    announce()
    sizes = [0, 1, 63, 64, 200, 333]
    q, k, v, g = _inputs(5, len(sizes), 4, 2, 333, 333, 64, dtype)
    for b, n in enumerate(sizes):
        for t, value in ((q, "nan"), (k, "inf"), (v, "-inf"), (g, "nan")):
            t[b, :, n:] = float(value)
    lengths = torch.tensor(sizes, dtype=torch.int32, device=DEV)
    for left, right, sinks in ((100, 0, 4), (-1, -1, 0)):
        _, grads = _gradients(q, k, v, g, (left, right), sinks, lengths=lengths)
        for b, n in enumerate(sizes):
            assert all((t[b, :, n:] == 0).all() for t in grads)
            if n:
                part = [t[b:b + 1, :, :n] for t in (q, k, v, g)]
                _near([t[b:b + 1, :, :n] for t in grads], *gradients(*part, left, right, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
def test_padded_batch_in_parts(dim, dtype, announce):
    """Few heads of long sequences: the walks of row tiles and of key tiles are cut, and parts beyond a sequence's
    end have nothing to add."""
    announce()
    sizes = [2600, 900, 5]
    q, k, v, g = _inputs(13, len(sizes), 2, 1, 2600, 2600, dim, dtype)
    for b, n in enumerate(sizes):
        for t, value in ((q, "nan"), (k, "inf"), (v, "-inf"), (g, "nan")):
            t[b, :, n:] = float(value)
    lengths = torch.tensor(sizes, dtype=torch.int32, device=DEV)
    _, grads = _gradients(q, k, v, g, (-1, 0), 0, lengths=lengths)
    for b, n in enumerate(sizes):
        assert all((t[b, :, n:] == 0).all() for t in grads)
        part = [t[b:b + 1, :, :n] for t in (q, k, v, g)]
        _near([t[b:b + 1, :, :n] for t in grads], *gradients(*part, -1, 0, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("at", [3, 130, 200])
def test_values_that_are_not_seen(which, at, announce):
    """A NaN in one row of q, k, v or the gradient reaches the gradients of rows it meets, and no others."""
    announce()
    sk, left, sinks = 300, 50, 5
    clean = list(_inputs(6, 1, 2, 2, sk, sk, 128, torch.bfloat16))
    _, want = _gradients(*clean, (left, 0), sinks)
    tensors = [t.clone() for t in clean]
    tensors[which][0, 1, at, 7] = float("nan")
    _, got = _gradients(*tensors, (left, 0), sinks)
    seen = seen_keys(torch.arange(sk), sk, left, 0, sinks)
    queries = seen[:, at] if which in (1, 2) else torch.arange(sk) == at   # rows of P that the NaN may reach
    keys = seen[queries].any(0)
    for i, reached in enumerate((queries, keys, keys)):
        assert torch.equal(got[i][:, 0], want[i][:, 0])
        assert torch.equal(got[i][0, 1, ~reached.to(DEV)], want[i][0, 1, ~reached.to(DEV)])
    assert not torch.isfinite(got[0][0, 1, queries.to(DEV)]).all()


@pytest.mark.gpu
def test_layouts_expanded_gradients_and_shared_inputs(announce):
    announce()
    q, k, v, g = _inputs(7, 2, 4, 2, 140, 140, 64, torch.bfloat16)
    _, want = _gradients(q, k, v, g, (30, 2), 4)

    def seen(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def odd(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t)

    for change in (seen, odd):
        _, grads = _gradients(*[change(t) for t in (q, k, v, g)], (30, 2), 4)
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
    ones = torch.ones((), dtype=torch.bfloat16, device=DEV).expand(q.shape)
    _, flat = _gradients(q, k, v, ones, (30, 2), 4)
    _, full = _gradients(q, k, v, ones.contiguous(), (30, 2), 4)
    assert all(torch.equal(a, b) for a, b in zip(flat, full))
    # One key head for all, by expand: autograd adds the heads' gradients up (in bf16, rounded again).
    one = k[:, :1].clone().requires_grad_()
    window_attention(q, one.expand(-1, 2, -1, -1), v, (30, 2), 4).backward(g)
    _, (_, each, _) = _gradients(q, one.detach().expand(-1, 2, -1, -1), v, g, (30, 2), 4)
    assert torch.equal(one.grad, each.sum(1, keepdim=True))
    # The same tensor as queries, keys and values.
    x = q[:, :2].clone().requires_grad_()
    window_attention(x, x, x, (30, 2), 4).backward(g[:, :2])
    _, parts = _gradients(q[:, :2], q[:, :2], q[:, :2], g[:, :2], (30, 2), 4)
    total = sum(p.double() for p in parts)
    assert ((x.grad.double() - total).abs() <= 2 * 2.0 ** -8 * sum(p.double().abs() for p in parts)).all()


@pytest.mark.gpu
def test_large_scores(announce):
    """One weight of 1 and others of 0: dV is the gradients' sum over each key's queries, dQ and dK vanish next to
    the sizes in play (dS of a weight of 1 is its rounding: |dP - delta| <= 2^-7 |dP|, times q or k)."""
    announce()
    g0 = torch.Generator().manual_seed(8)
    size = 2.0 ** 30
    q = (torch.sign(torch.randn(1, 1, 200, 64, generator=g0)) * size).bfloat16().to(DEV)
    k = (torch.randn(1, 1, 200, 64, generator=g0).bfloat16() * size).to(DEV)
    v, g = (torch.randn(1, 1, 200, 64, generator=g0).bfloat16().to(DEV) for _ in range(2))
    _, grads = _gradients(q, k, v, g, (-1, -1), 0)
    s = (q.double() @ k.double().transpose(2, 3))[0, 0]
    top = s.topk(2, -1)
    assert ((top.values[:, 0] - top.values[:, 1]) > 2.0 ** -12 * top.values[:, 0].abs()).all()
    want = torch.zeros(200, 64, dtype=torch.float64, device=DEV).index_add_(0, top.indices[:, 0], g[0, 0].double())
    mass = torch.zeros(200, 64, dtype=torch.float64, device=DEV).index_add_(0, top.indices[:, 0], g[0, 0].double().abs())
    assert ((grads[2][0, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * mass).all()
    assert all(torch.isfinite(t).all() for t in grads)


@pytest.mark.gpu
def test_replayed_step_and_streams(announce):
    """A forward and backward captured once; every replay equals the eager step on the new inputs."""
    announce()
    q, k, v, g = _inputs(9, 1, 4, 2, 500, 500, 64, torch.float16)
    args = ((100, 0), 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _, other = _gradients(q, k, v, g, *args)
    torch.cuda.current_stream().wait_stream(side)
    _, want = _gradients(q, k, v, g, *args)
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    torch.cuda.synchronize()
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = torch.autograd.grad(window_attention(*leaves, *args), leaves, g)
    for _ in range(4):
        for leaf in leaves:
            leaf.data.copy_(torch.randn(leaf.shape, device=DEV))
        _, want = _gradients(*leaves, g, *args)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.gpu
def test_training_step_with_rotation(announce):
    """rotary_axes and window_attention as a block uses them: the gradients of the unturned rows equal those of the
    turned ones turned back (both steps of the chain bit for bit)."""
    from peco_amd.rotary import RotaryAxes, rotary_axes

    announce()
    axes, positions = RotaryAxes((16, 24, 24), 256.0), RotaryAxes.grid(3, 5, 7, device=DEV)
    q, k, v, g = _inputs(10, 2, 4, 2, 105, 105, 64, torch.bfloat16)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    turned = [rotary_axes(t, positions, axes) for t in leaves[:2]]
    window_attention(*turned, leaves[2], (34, 0), 5).backward(g)
    _, inner = _gradients(*[t.detach() for t in turned], v, g, (34, 0), 5)
    for leaf, grad in zip(leaves[:2], inner[:2]):
        part = leaf.detach().requires_grad_()
        back, = torch.autograd.grad(rotary_axes(part, positions, axes), part, grad)
        assert torch.equal(leaf.grad, back)
    assert torch.equal(leaves[2].grad, inner[2])


@pytest.mark.gpu
def test_second_derivatives_are_refused_and_empty_inputs(announce):
    announce()
    q, k, v, g = _inputs(11, 1, 2, 2, 5, 5, 64, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(window_attention(*leaves, (1, 0)), leaves, g.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        grads[0].sum().backward()
    with torch.no_grad():
        assert not window_attention(*leaves, (1, 0)).requires_grad
    _, empty = _gradients(q[:, :, :0], k, v, g[:, :, :0].detach(), (1, 0), 0)
    assert empty[0].shape == (1, 2, 0, 64) and all((t == 0).all() for t in empty[1:])
    _, empty = _gradients(q, k[:, :, :0], v[:, :, :0], g.detach(), (1, 0), 0)
    assert (empty[0] == 0).all() and empty[1].shape == (1, 2, 0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,keys,sinks", [(3, 32896, 32896), (24, 118800, 118800), (1, 118800, 50000), (24, 7006, 256)])
def test_many_sinks_need_little_workspace(heads, keys, sinks, announce):
    """The walks of keys that every later token sees are cut for few heads only: at most 4 parts for each CU and one
    for each tile of 256 keys, of 256 KB."""
    announce()
    floats = _native.library().peco_window_attention_grad_workspace_size(1, heads, heads, keys, keys, 255, 0, sinks, 128, 1)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert floats <= heads * keys + 64 + (4 * cus + heads * (keys // 256 + 1)) * 256 * 256


@pytest.mark.gpu
def test_sinks_over_the_whole_sequence(announce):
    announce()
    q, k, v, g = _inputs(12, 1, 3, 3, 4000, 4000, 64, torch.bfloat16)
    _, grads = _gradients(q, k, v, g, (63, 0), 4000)
    _near(grads, *gradients(q, k, v, g, 63, 0, 4000))


def test_entry_refuses_bad_arguments():
    lib, null, some = _native.library(), ctypes.c_void_p(0), ctypes.c_void_p(4096)  # refused before it is read
    floats = lib.peco_window_attention_grad_workspace_size(1, 2, 1, 5, 5, 1, 0, 0, 64, 1)
    assert floats >= 10
    good = dict(q=some, k=some, v=some, out=some, grad=some, dq=some, dk=some, dv=some, strides=[1024, 512, 64] * 8,
                lengths=null, row_max=some, row_log=some, rest=some, work=some, floats=floats, batch=1, q_heads=2, kv_heads=1,
                queries=5, keys=5, left=1, right=0, sinks=0, scale=0.125, d=64, dtype=1)

    def call(**changes):
        a = {**good, **changes}
        a["strides"] = (ctypes.c_int64 * 24)(*a["strides"])
        return lib.peco_window_attention_grad(*a.values(), null)

    for name in ("q", "k", "v", "out", "grad", "dq", "dk", "dv", "row_max", "row_log", "rest", "work"):
        assert call(**{name: null}) == 1, name
    for change in (dict(batch=0), dict(q_heads=3, kv_heads=2), dict(queries=0), dict(keys=0), dict(left=-2), dict(sinks=-1),
                   dict(scale=0.0), dict(lengths=some, queries=4), dict(strides=[1024, 512, 60] * 8),
                   dict(dk=ctypes.c_void_p(4104))):
        assert call(**change) == 1, change
    assert call(d=96) == 20002 and call(dtype=2) == 20003 and call(floats=floats - 1) == 20001
    assert lib.peco_window_attention_grad_workspace_size(1, 3, 2, 5, 5, 1, 0, 0, 64, 1) == 0
