"""Rotary positions with several axes: the kernel, its gradient and the processor call against 64 bits."""
import pytest
import torch

from peco_amd import clustering_cuda, processor
from peco_amd.rotary import RotaryAxes, RotaryPositions, rotary_axes

DEV = "cuda:0"
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _turn(x, positions, axes, sign=1.0):
    """The definition in 64 bits: pairs as complex numbers times exp(i angle)."""
    half, pair, out = sum(axes.dims) // 2, 0, x.double().clone()
    for a, d in enumerate(axes.dims):
        for i in range(d // 2):
            step = 2 * pair / (2 * half) if axes.shared else 2 * i / d
            angle = sign * positions[..., a, :].double() * axes.theta ** -step  # [S] or [B, S]
            angle = angle if angle.dim() == 1 else angle[:, None]
            c0, c1 = (2 * pair, 2 * pair + 1) if axes.layout == "interleaved" else (pair, pair + half)
            u, v = x[..., c0].double(), x[..., c1].double()
            out[..., c0], out[..., c1] = u * angle.cos() - v * angle.sin(), v * angle.cos() + u * angle.sin()
            pair += 1
    return out


def _bound(ref, x, axes):
    """Half a step of the type, and in fp32: sine and cosine within 2^-22 (the fraction of a turn is rounded once,
    2^-25 turns at most, and the functions are good to 2 units in the last place), two products and a sum
    within 2^-22 of the pair's length; half the smallest fp16 step."""
    half, r = sum(axes.dims) // 2, torch.zeros_like(ref)
    sq = x.double().square()
    for i in range(half):
        c0, c1 = (2 * i, 2 * i + 1) if axes.layout == "interleaved" else (i, i + half)
        r[..., c0] = r[..., c1] = (sq[..., c0] + sq[..., c1]).sqrt()
    return UNIT[x.dtype] * 1.01 * ref.abs() + 2.0 ** -20 * r + 2.0 ** -25 * (x.dtype == torch.float16)


CASES = [
    # batch, heads, rows, D, axes, positions' type and range
    (1, 1, 1, 128, RotaryAxes((16, 56, 56), 256.0), torch.int32, 1 << 17),
    (2, 9, 17, 128, RotaryAxes((16, 56, 56), 256.0), torch.int64, 1 << 17),
    (1, 24, 333, 64, RotaryAxes((8, 24, 16)), torch.int32, 100),  # 16 channels stay
    (1, 3, 45, 72, RotaryAxes((6, 34)), torch.float32, 50),  # a chunk that turns in part
    (2, 5, 37, 128, RotaryAxes((32, 48, 48), 10000.0, "halves", True), torch.int32, 1 << 17),
    (1, 4, 29, 72, RotaryAxes((16, 8, 4, 4), 500.0, "halves"), torch.int32, 1 << 12),
    (1, 2, 257, 256, RotaryAxes((256,), 10000.0), torch.int32, 1 << 17),
    (3, 1, 5, 8, RotaryAxes((2,), 10000.0), torch.int32, 7),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("batch,heads,rows,dim,axes,kind,most", CASES)
def test_rows_and_gradient(batch, heads, rows, dim, axes, kind, most, dtype, announce):
    announce()
    g = torch.Generator().manual_seed(rows + dim)
    positions = torch.randint(0, most, (batch, len(axes.dims), rows), generator=g)
    positions = (positions + 0.25 if kind == torch.float32 else positions).to(kind).to(DEV)
    x = torch.randn(batch, heads, rows, dim, generator=g).to(dtype).to(DEV)
    seen = torch.randn(batch, rows, heads, dim, generator=g).to(dtype).to(DEV).transpose(1, 2)
    wide = torch.zeros(batch, heads, rows, dim + 8, dtype=dtype, device=DEV)
    wide[..., :dim] = x
    odd = torch.zeros(batch * heads * rows * dim + 1, dtype=dtype, device=DEV)[1:].view(x.shape).copy_(x)
    apart = torch.zeros(batch, heads, rows, dim, 2, dtype=dtype, device=DEV)[..., 0].copy_(x)
    for part in (x, seen, wide[..., :dim], odd, apart):
        for at in (positions, positions[0]) if batch > 1 else (positions,):
            ref = _turn(part, at, axes)
            leaf = part.detach().requires_grad_()
            out = rotary_axes(leaf, at, axes)
            assert out.shape == part.shape and out.stride() == torch.empty_like(part).stride()
            assert ((out.double() - ref).abs() <= _bound(ref, part, axes)).all()
            assert torch.equal(out, rotary_axes(part, at, axes))
            grad, = torch.autograd.grad(out, leaf, seen)
            back = _turn(seen, at, axes, -1.0)
            assert ((grad.double() - back).abs() <= _bound(back, seen, axes)).all()
    strided = positions.repeat_interleave(2, -1)[..., ::2]
    assert torch.equal(rotary_axes(x, strided, axes), rotary_axes(x, positions, axes))


@pytest.mark.gpu
def test_gradient_against_differences(announce):
    """The rotation is linear: a difference quotient with a step of 1 has only rounding in it. Values of size 1
    turned in fp32 are within 2^-20 |pair| each; a sum over n of them against unit weights within n times that."""
    announce()
    axes = RotaryAxes((16, 24, 24), 256.0)
    positions = RotaryAxes.grid(3, 4, 5, device=DEV)
    g = torch.Generator().manual_seed(1)
    x, step, weight = (torch.randn(1, 2, 60, 64, generator=g).to(DEV) for _ in range(3))
    leaf = x.clone().requires_grad_()
    (rotary_axes(leaf, positions, axes) * weight).sum().backward()
    moved = sum(sign * (rotary_axes(x + sign * step, positions, axes).double() * weight.double()).sum()
                for sign in (1, -1)) / 2
    size = (x.abs().max() + step.abs().max()) * 2 * weight.abs().max()
    assert abs(float(moved - (leaf.grad.double() * step.double()).sum())) <= 2.0 ** -20 * float(size) * x.numel()


@pytest.mark.gpu
def test_far_positions_expanded_gradients_and_non_finite_channels(announce):
    """64-bit positions near 2^40 (the product with the frequency is good to 2^-53 of its turns: 2^-14 turns and
    2^-11 radians), gradients without strides, and a NaN that stays in its pair."""
    announce()
    axes = RotaryAxes((64,), 10000.0)
    positions = (torch.arange(40) * 27487790694 + 5)[None].to(DEV)
    x = torch.randn(1, 2, 40, 64, device=DEV)
    ref = _turn(x, positions, axes)
    assert (rotary_axes(x, positions, axes).double() - ref).abs().max() <= 2.0 ** -10 * x.abs().max() * 1.5
    leaf = x.requires_grad_()
    near = torch.arange(40, device=DEV)[None]
    rotary_axes(leaf, near, axes).sum().backward()
    back = _turn(torch.ones_like(x), near, axes, -1.0)
    assert ((leaf.grad.double() - back).abs() <= _bound(back, torch.ones_like(x), axes)).all()
    with torch.no_grad():
        x = x.clone()
        x[0, 1, 7, 6] = float("nan")
        x[0, 0, 3, 9] = float("inf")
        out = rotary_axes(x, near, axes)
        bad = ~torch.isfinite(out)
        want = torch.zeros_like(bad)
        want[0, 1, 7, 6:8] = True
        want[0, 0, 3, 8:10] = True
        assert torch.equal(bad, want)
        assert rotary_axes(x[:, :, :0], near[:, :0], axes).shape == (1, 2, 0, 64)


@pytest.mark.gpu
def test_replayed_graph_and_side_stream(announce):
    announce()
    axes = RotaryAxes((16, 24, 24), 256.0)
    positions = RotaryAxes.grid(2, 5, 7, device=DEV)
    x = torch.randn(1, 3, 70, 64, device=DEV).bfloat16()
    rotary_axes(x, positions, axes)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary_axes(x, positions, axes)
    for i in range(4):
        x.copy_(torch.randn(1, 3, 70, 64, device=DEV))
        positions.add_(i)
        want = rotary_axes(x, positions, axes)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = rotary_axes(x, positions, axes)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)


class _Block(torch.nn.Module):
    def __init__(self, heads, dim):
        super().__init__()
        self.heads = heads
        self.to_q, self.to_k, self.to_v = (torch.nn.Linear(heads * dim, heads * dim) for _ in range(3))
        self.norm_q, self.norm_k = torch.nn.RMSNorm(dim, eps=1e-6), torch.nn.LayerNorm(dim)
        self.add_q_proj = None


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("per_batch", [False, True])
def test_processor_call_takes_positions(layout, per_batch, monkeypatch, announce):
    """Placed in one launch or by norm, rotary_axes and a copy: the same bits; and as near as two roundings of
    the type to the call with tables (fp32 cosines and sines of the same angles)."""
    announce()
    heads, dim, grid = 3, 64, (3, 6, 9)
    rows, text = grid[0] * grid[1] * grid[2], 11
    torch.manual_seed(5)
    block = _Block(heads, dim).to(DEV, torch.bfloat16)
    hidden = torch.randn(2, rows, heads * dim).to(DEV, torch.bfloat16)
    enc = torch.randn(2, text, heads * dim).to(DEV, torch.bfloat16)
    axes = RotaryAxes((16, 24, 24), 256.0, layout)
    positions = RotaryAxes.grid(*grid, device=DEV)
    if per_batch:
        positions = torch.stack((positions, positions + 5))
    layer = processor.PecoAttention(0, processor.PecoConfig(), processor.InferenceContext(5, text, text))
    layer.attention = lambda q, k, v: torch.cat((q, k, v), -1)
    launched = []
    place = clustering_cuda.place_heads
    monkeypatch.setattr(clustering_cuda, "place_heads", lambda *a: (launched.append(a), place(*a)))
    got = layer(block, hidden, enc, image_rotary_emb=RotaryPositions(axes, positions))
    assert len(launched) == (2 if layout == "interleaved" else 0)
    monkeypatch.setattr(processor, "_placeable", lambda part, buffer: False)
    ref = layer(block, hidden, enc, image_rotary_emb=RotaryPositions(axes, positions))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    if layout == "interleaved" and not per_batch:
        angle = torch.cat([positions[a].double()[:, None] * 256.0 ** (-torch.arange(0, d, 2, device=DEV).double() / d)
                           for a, d in enumerate(axes.dims)], 1).repeat_interleave(2, -1)
        tables = layer(block, hidden, enc, image_rotary_emb=(angle.cos().float(), angle.sin().float()))
        off = (tables[0].double() - got[0].double()).abs()
        assert (off <= 2 * 2.0 ** -8 * got[0].double().abs() + 2.0 ** -18 * got[0].abs().max()).all()
        assert torch.equal(tables[1], got[1])


def test_refusals():
    """No launch is reached: these run without a GPU."""
    axes, rows = RotaryAxes((16, 24, 24)), torch.zeros(1, 2, 5, 64)
    good = torch.zeros(3, 5, dtype=torch.int32)
    for kwargs in ({"dims": ()}, {"dims": (3, 5)}, {"dims": (2, 2, 2, 2, 2)}, {"dims": (300,)}, {"dims": (16,), "theta": 0},
                   {"dims": (16,), "theta": float("nan")}, {"dims": (16,), "layout": "pairs"},
                   {"dims": (10, 4), "layout": "halves"}, {"dims": (16.0,)}):
        with pytest.raises(ValueError):
            RotaryAxes(**kwargs)
    with pytest.raises(ValueError, match="B,H,S,D"):
        rotary_axes(rows[0], good, axes)
    with pytest.raises(TypeError, match="float16"):
        rotary_axes(rows.double(), good, axes)
    with pytest.raises(ValueError, match="multiples of 8"):
        rotary_axes(torch.zeros(1, 1, 5, 68), good, axes)
    with pytest.raises(TypeError, match="RotaryAxes"):
        rotary_axes(rows, good, (16, 24, 24))
    with pytest.raises(ValueError, match="more channels"):
        rotary_axes(rows, good, RotaryAxes((32, 24, 24)))
    with pytest.raises(TypeError, match="int32"):
        rotary_axes(rows, good.double(), axes)
    for shape in ((2, 5), (3, 4), (2, 3, 5), (3, 5, 1)):
        with pytest.raises(ValueError, match="must have shape"):
            rotary_axes(rows, torch.zeros(shape, dtype=torch.int32), axes)
    with pytest.raises(ValueError, match="GPU tensors"):
        rotary_axes(rows, good, axes)
    with pytest.raises(RuntimeError, match="no gradient"):
        rotary_axes(rows, torch.zeros(3, 5, requires_grad=True), axes)


def test_entry_refuses_bad_arguments():
    import ctypes

    from peco_amd import _native
    from peco_amd.rotary import plan_arguments

    lib, null = _native.library(), ctypes.c_void_p(0)
    some = ctypes.c_void_p(4096)  # refused before it is read
    plan = plan_arguments(RotaryAxes((16, 24, 24)), torch.zeros(3, 5, dtype=torch.int32))
    strides = (640, 320, 64)

    def call(x=some, out=some, plan=plan, strides=strides, sizes=(1, 2, 5, 64, 1)):
        return lib.peco_rotary_axes(x, *strides, out, *strides, *plan, *sizes, null)

    assert call(x=null) == 1 and call(out=null) == 1
    assert call(sizes=(0, 2, 5, 64, 1)) == 1 and call(sizes=(1, 2, 5, 56, 1)) == 1  # 64 channels turn
    assert call(sizes=(1, 2, 5, 68, 1)) == 20002 and call(sizes=(1, 2, 5, 64, 3)) == 20003
    assert call(strides=(640, 320, 60)) == 1 and call(x=ctypes.c_void_p(4104)) == 1
    for at, value in ((0, null), (1, 3), (4, None), (5, None), (6, 0), (6, 5)):
        assert call(plan=(*plan[:at], value, *plan[at + 1:])) == 1
    head = (some, *strides, some)
    assert lib.peco_place_heads_axes(*head, *plan[:7], 1, 0, 0, null, 0.0, 1, 2, 5, 0, 5, 64, 1, null) == 1
    assert lib.peco_place_heads_axes(*head, *plan, 0, null, 0.0, 1, 2, 5, 1, 5, 64, 1, null) == 1
