"""Attention with a sliding window and sinks against its definition in 64 bits."""
import pytest
import torch

from peco_amd.window import check_mask, window_attention
from tests.window_reference import attention, seen_keys

DEV = "cuda:0"


def _inputs(seed, batch, q_heads, kv_heads, sq, sk, dim, dtype, device=DEV):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(batch, heads, n, dim, generator=g).to(dtype).to(device)
            for heads, n in ((q_heads, sq), (kv_heads, sk), (kv_heads, sk))]


def _near(out, ref, bound):
    assert torch.isfinite(out).all()
    off = (out.double() - ref).abs() - bound
    assert (off <= 0).all(), f"off by {float(off.max()):.3e} more than the bound at {int(off.argmax())}"


CASES = [
    # batch, query heads, key heads, queries, keys, left, right, sinks
    (1, 1, 1, 1, 1, -1, 0, 0),
    (1, 2, 1, 2, 2, 0, 0, 0),
    (2, 4, 2, 65, 65, 16, 0, 3),
    (1, 3, 3, 64, 64, -1, -1, 0),
    (1, 3, 1, 129, 129, 31, 0, 0),       # three query heads a key head: rows of a tile end inside a token
    (2, 6, 2, 300, 300, 40, 0, 200),     # sinks that reach into the window of some rows
    (1, 2, 2, 257, 641, 100, 0, 5),      # queries behind cached keys
    (1, 2, 2, 70, 33, -1, 0, 0),         # more queries than keys: the first 37 see nothing
    (1, 2, 1, 70, 33, 3, 0, 2),
    (1, 2, 2, 200, 90, 4, 30, 0),        # queries before the first key that see some
    (1, 1, 1, 500, 500, 0, 0, 0),        # each its own key
    (1, 1, 1, 500, 500, 0, 0, 1),
    (1, 2, 2, 400, 400, 63, 64, 0),
    (1, 2, 2, 400, 400, 20, 17, 50),
    (1, 2, 2, 333, 333, -1, 10, 7),
    (1, 2, 2, 333, 333, 10, -1, 400),    # sinks past the end
    (1, 2, 2, 333, 333, 1 << 40, 1 << 40, 1 << 40),
    (1, 2, 1, 1, 300, -1, 0, 0),         # single tokens
    (3, 8, 2, 1, 5000, -1, 0, 0),        # cut into parts
    (1, 4, 1, 3, 9000, 2000, 0, 100),
    (1, 2, 2, 130, 4000, -1, 0, 0),
    (1, 24, 24, 1000, 1000, 255, 0, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,q_heads,kv_heads,sq,sk,left,right,sinks", CASES)
def test_forward(batch, q_heads, kv_heads, sq, sk, left, right, sinks, dim, dtype, announce):
    announce()
    q, k, v = _inputs(sq + sk, batch, q_heads, kv_heads, sq, sk, dim, dtype)
    out = window_attention(q, k, v, (left, right), sinks)
    _near(out, *attention(q, k, v, left, right, sinks))
    seen = seen_keys(torch.arange(sk - sq, sk), sk, left, right, sinks).any(1)
    assert (out[:, :, ~seen.to(DEV)] == 0).all()
    assert torch.equal(out, window_attention(q, k, v, (left, right), sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_layouts(dim, announce):
    """Views, gaps, misaligned rows, expanded heads: the bits of the contiguous call."""
    announce()
    q, k, v = _inputs(3, 2, 6, 3, 150, 150, dim, torch.bfloat16)
    want = window_attention(q, k, v, (50, 3), 9)

    def seen(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def gaps(t):
        wide = torch.full((*t.shape[:3], dim + 8), float("nan"), dtype=t.dtype, device=DEV)
        wide[..., :dim] = t
        return wide[..., :dim]

    def odd(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t)

    def apart(t):
        return torch.empty(*t.shape, 2, dtype=t.dtype, device=DEV)[..., 1].copy_(t)

    for change in (seen, gaps, odd, apart):
        parts = [change(t) for t in (q, k, v)]
        out = window_attention(*parts, (50, 3), 9)
        assert torch.equal(out, want) and out.stride() == torch.empty_like(parts[0]).stride()
    assert torch.equal(window_attention(q, seen(k), gaps(v), (50, 3), 9), want)
    one = k[:, :1].expand(-1, 3, -1, -1)
    assert torch.equal(window_attention(q, one, v, (50, 3), 9), window_attention(q, one.contiguous(), v, (50, 3), 9))


@pytest.mark.gpu
def test_far_rows(announce):
    """Key rows spread over more than 2^32 bytes (a view of a large buffer) read right."""
    announce()
    keys, step = 700, 1 << 22  # 8 MiB between rows: 5.9 GB from first to last
    q, k, v = _inputs(4, 1, 2, 1, 300, keys, 64, torch.bfloat16)
    buffer = torch.empty(keys * step, dtype=torch.bfloat16, device=DEV)
    far = buffer.as_strided((1, 1, keys, 64), (step * keys, step * keys, step, 1))
    far.copy_(k)
    out = window_attention(q, far, v, (200, 0), 20)
    assert torch.equal(out, window_attention(q, k, v, (200, 0), 20))
    far.copy_(v)
    assert torch.equal(window_attention(q, k, far, (200, 0), 20), out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_padded_batch(dtype, announce):
    """Lengths of none, one, some, all and more tokens; what lies behind them is NaN and infinity."""
    announce()
    sizes = [0, 1, 63, 64, 200, 333, 1000, -5]
    q, k, v = _inputs(5, len(sizes), 4, 2, 333, 333, 64, dtype)
    for b, n in enumerate(sizes):
        n = max(n, 0)
        q[b, :, n:], k[b, :, n:], v[b, :, n:] = float("nan"), float("inf"), float("-inf")
    lengths = torch.tensor(sizes, dtype=torch.int32, device=DEV)
    for mask in ((100, 0, 4), (-1, -1, 0), (10, 10, 0)):
        out = window_attention(q, k, v, mask[:2], mask[2], lengths=lengths)
        for b, n in enumerate(sizes):
            n = max(0, min(n, 333))
            assert (out[b, :, n:] == 0).all()
            if n:
                part = [t[b:b + 1, :, :n] for t in (q, k, v)]
                _near(out[b:b + 1, :, :n], *attention(*part, *mask))


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("sq,sk,left,right,sinks,at", [
    (300, 300, 50, 0, 0, 130), (300, 300, 50, 0, 10, 3), (200, 200, 20, 20, 0, 64), (2, 3000, 100, 0, 4, 2898),
    (130, 700, -1, 0, 0, 640)])
def test_values_that_a_query_does_not_see(sq, sk, left, right, sinks, at, bad, announce):
    """An infinity or NaN in one key or value reaches the queries that see it, and no other."""
    announce()
    q, k, v = _inputs(6, 1, 4, 2, sq, sk, 128, torch.bfloat16)
    clean = window_attention(q, k, v, (left, right), sinks)
    seen = seen_keys(torch.arange(sk - sq, sk), sk, left, right, sinks)[:, at].to(DEV)
    for which in (0, 1):
        kv = [k.clone(), v.clone()]
        kv[which][0, 1, at, 5] = bad
        out = window_attention(q, *kv, (left, right), sinks)
        assert torch.equal(out[:, :2], clean[:, :2])
        assert torch.equal(out[:, 2:, ~seen], clean[:, 2:, ~seen])
        if which:
            hit = out[:, 2:, seen]
            assert not torch.isfinite(hit[..., 5]).any()
            others = torch.arange(128, device=DEV) != 5
            ref, bound = attention(q, k, v, left, right, sinks)
            _near(hit[..., others], ref[:, 2:, seen][..., others], bound[:, 2:, seen][..., others])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("step", [0.004, 0.05, 0.17, 0.7, -0.004, -0.05, -0.7])
def test_rising_and_falling_scores(step, dtype, announce):
    """Scores that climb along the keys by powers of two of the weight a tile, below and past the 2^8 by which a row's
    weights may exceed its reference's, and that fall: forward and gradients."""
    from tests.window_reference import gradients

    announce()
    g = torch.Generator().manual_seed(14)
    signs = torch.sign(torch.randn(64, generator=g))
    climb = step * torch.arange(1000)[:, None] / 8 * signs
    q = (signs + 0.2 * torch.randn(1, 2, 150, 64, generator=g)).to(dtype).to(DEV)
    k = (climb + 0.2 * torch.randn(1, 1, 1000, 64, generator=g)).to(dtype).to(DEV)
    v = torch.randn(1, 1, 1000, 64, generator=g).to(dtype).to(DEV)
    grad = torch.randn(1, 2, 150, 64, generator=g).to(dtype).to(DEV)
    for left, right, sinks in ((-1, 0, 0), (400, 30, 40)):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = window_attention(*leaves, (left, right), sinks)
        _near(out, *attention(q, k, v, left, right, sinks))
        for got, ref, bound in zip(torch.autograd.grad(out, leaves, grad), *gradients(q, k, v, grad, left, right, sinks)):
            _near(got, ref, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** 8, 2.0 ** 30, 2.0 ** 55])
def test_large_scores(size, announce):
    """Scores of up to 2^116 times their scale: the weights of the largest are 1, of the others 0 (they are apart by
    more than 2^7, so exp underflows), whatever their size."""
    announce()
    g = torch.Generator().manual_seed(8)
    base = torch.randn(1, 2, 200, 64, generator=g)
    q = (torch.sign(base) * size).bfloat16().to(DEV)
    k = (torch.randn(1, 2, 200, 64, generator=g).bfloat16() * size).to(DEV)
    v = torch.randn(1, 2, 200, 64, generator=g).bfloat16().to(DEV)
    s = (q.double() @ k.double().transpose(2, 3)).masked_fill(
        ~seen_keys(torch.arange(200), 200, 80, 0, 3).to(DEV), -float("inf"))
    top = s.topk(2, -1)
    clear = (top.values[..., 0] - top.values[..., 1]) * 0.125 > 2.0 ** 7 + 2.0 ** -16 * top.values[..., 0].abs()
    clear[..., 0] = True
    assert clear.float().mean() > 0.6
    out = window_attention(q, k, v, (80, 0), 3)
    want = v.gather(2, top.indices[..., :1].expand(-1, -1, -1, 64))
    assert torch.equal(out[clear], want[clear])
    assert torch.isfinite(out).all()


@pytest.mark.gpu
def test_scale_streams_and_graph(announce):
    announce()
    q, k, v = _inputs(9, 1, 4, 4, 90, 2500, 64, torch.bfloat16)  # cut into parts: a workspace
    out = window_attention(q, k, v, (2000, 0), 4, scale=0.03)
    _near(out, *attention(q, k, v, 2000, 0, 4, 0.03))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = window_attention(q, k, v, (2000, 0), 4, scale=0.03)
    both = window_attention(q, k, v, (2000, 0), 4, scale=0.03)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, out) and torch.equal(both, out)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = window_attention(q, k, v, (2000, 0), 4)
    for i in range(4):
        q.copy_(torch.randn(q.shape, device=DEV))
        want = window_attention(q, k, v, (2000, 0), 4)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


@pytest.mark.gpu
def test_empty(announce):
    announce()
    q, k, v = _inputs(1, 1, 2, 2, 5, 5, 64, torch.bfloat16)
    assert window_attention(q[:, :, :0], k, v, (1, 0)).shape == (1, 2, 0, 64)
    assert (window_attention(q, k[:, :, :0], v[:, :, :0], (1, 0)) == 0).all()
    assert window_attention(q[:0], k[:0], v[:0], (1, 0)).shape == (0, 2, 5, 64)


def test_refusals():
    """No launch is reached: these run without a GPU."""
    q, k, v = _inputs(1, 2, 4, 2, 5, 7, 64, torch.bfloat16, "cpu")
    for window in ((-2, 0), (0,), (1.0, 0), (True, 0), 5, None):
        with pytest.raises(ValueError, match="window"):
            check_mask(window, 0, None, 64)
    for sinks in (-1, 1.5, True, None):
        with pytest.raises(ValueError, match="sinks"):
            check_mask((1, 0), sinks, None, 64)
    for scale in (0.0, -1.0, float("inf"), float("nan"), 1e-40):
        with pytest.raises(ValueError, match="scale"):
            check_mask((1, 0), 0, scale, 64)
    with pytest.raises(TypeError, match="torch tensors"):
        window_attention(q, k, None, (1, 0))
    with pytest.raises(ValueError, match="Expected Q"):
        window_attention(q[0], k, v, (1, 0))
    with pytest.raises(ValueError, match="Expected Q"):
        window_attention(q, k, v[:, :, :6], (1, 0))
    with pytest.raises(ValueError, match="batch and feature"):
        window_attention(q[:1], k, v, (1, 0))
    with pytest.raises(ValueError, match="multiple of the key heads"):
        window_attention(q[:, :3], k, v, (1, 0))
    with pytest.raises(ValueError, match="64 and 128"):
        window_attention(q[..., :32], k[..., :32], v[..., :32], (1, 0))
    with pytest.raises(TypeError, match="share dtype"):
        window_attention(q.float(), k, v, (1, 0))
    with pytest.raises(ValueError, match="as many queries"):
        window_attention(q, k, v, (1, 0), lengths=torch.ones(2, dtype=torch.int32))
    with pytest.raises(TypeError, match="int32"):
        window_attention(q, k[:, :, :5], v[:, :, :5], (1, 0), lengths=torch.ones(2))
    with pytest.raises(ValueError, match="GPU device"):
        window_attention(q, k, v, (1, 0))


def test_entry_refuses_bad_arguments():
    import ctypes

    from peco_amd import _native

    lib, null, some = _native.library(), ctypes.c_void_p(0), ctypes.c_void_p(4096)  # refused before it is read
    good = dict(q=some, k=some, v=some, out=some, strides=[1024, 512, 64] * 4, lengths=null, row_max=null, row_log=null,
                rest=null, work=null, floats=0, batch=1, q_heads=2, kv_heads=1, queries=5, keys=5, left=1, right=0, sinks=0,
                scale=0.125, d=64, dtype=1)

    def call(**changes):
        a = {**good, **changes}
        strides = (ctypes.c_int64 * 12)(*a.pop("strides"))
        return lib.peco_window_attention(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("out"), strides, *a.values(), null)

    for change in (dict(q=null), dict(out=null), dict(batch=0), dict(kv_heads=0), dict(q_heads=3, kv_heads=2),
                   dict(queries=0), dict(keys=0), dict(left=-2), dict(right=-2), dict(sinks=-1), dict(scale=0.0),
                   dict(scale=-1.0), dict(scale=float("nan")), dict(row_max=some), dict(row_max=some, row_log=some), dict(lengths=some, queries=4),
                   dict(strides=[1024, 512, 60] * 4), dict(k=ctypes.c_void_p(4104))):
        assert call(**change) == 1, change
    assert call(d=96) == 20002 and call(dtype=2) == 20003 and call(keys=1 << 30) == 20002
    floats = lib.peco_window_attention_workspace_size(1, 2, 1, 1, 50000, -1, 0, 0, 64)
    assert floats > 0 and call(queries=1, keys=50000, left=-1, work=some, floats=floats - 1) == 20001
    assert call(queries=1, keys=50000, left=-1, work=ctypes.c_void_p(4100), floats=floats) == 1
    assert lib.peco_window_attention_workspace_size(1, 2, 1, 5, 5, 1, 0, 0, 64) == 0
    assert lib.peco_window_attention_workspace_size(0, 24, 24, 7006, 7006, 2025, 0, 256, 128) == 0
