"""A paged cache: tokens appended and attended to, against the definition in 64 bits."""
import pytest
import torch

from peco_amd.paged import append_pages, paged_attention
from peco_amd.rotary import RotaryAxes, RotaryPositions, rotary_axes
from peco_amd.window import window_attention
from tests.window_reference import rows, seen_keys

DEV = "cuda:0"


class Cache:
    """Pages in a random order, with NaN wherever no token was written."""

    def __init__(self, seed, lengths, page, heads, dim, dtype, spare=2, width=None):
        self.g = torch.Generator().manual_seed(seed)
        held = [-(-max(n, 0) // page) for n in lengths]
        self.lengths, self.page, self.heads, self.dim, self.dtype = lengths, page, heads, dim, dtype
        order = torch.randperm(sum(held) + spare, generator=self.g).to(torch.int32)
        width = max(1, max(held)) if width is None else width
        self.table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(held):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.k = [torch.randn(max(n, 0), heads, dim, generator=self.g).to(dtype).to(DEV) for n in lengths]
        self.v = [torch.randn(max(n, 0), heads, dim, generator=self.g).to(dtype).to(DEV) for n in lengths]
        shape = (order.numel(), heads, page, dim)
        self.k_pages, self.v_pages = (torch.full(shape, float("nan"), dtype=dtype, device=DEV) for _ in range(2))
        for b, n in enumerate(lengths):
            for t in range(0, max(n, 0), page):
                p, m = int(self.table[b, t // page]), min(page, n - t)
                self.k_pages[p, :, :m] = self.k[b][t:t + m].transpose(0, 1)
                self.v_pages[p, :, :m] = self.v[b][t:t + m].transpose(0, 1)
        self.table = self.table.to(DEV)

    def queries(self, new, heads, tail=0):
        offsets = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
        q = torch.randn(sum(new) + tail, heads, self.dim, generator=self.g).to(self.dtype).to(DEV)
        return q, offsets, torch.tensor(self.lengths, dtype=torch.int32, device=DEV)

    def check(self, out, q, new, left, sinks, hide=None):
        at, group = 0, q.shape[1] // self.heads
        for b, n in enumerate(new):
            keys = max(self.lengths[b], 0)
            seen = seen_keys(torch.arange(keys - n, keys, device=DEV), keys, left, 0, sinks)
            if hide is not None:
                seen &= ~hide[b][None]
            for h in range(q.shape[1]):
                ref, bound = rows(q[at:at + n, h], self.k[b][:, h // group], self.v[b][:, h // group], seen,
                                  self.dim ** -0.5)[:2]
                got = out[at:at + n, h]
                assert torch.isfinite(got).all()
                off = (got.double() - ref).abs() - bound
                assert n == 0 or (off <= 0).all(), f"sequence {b} head {h}: {float(off.max()):.3e} past the bound"
            at += n


CASES = [
    # lengths, new tokens, page, query heads, key heads, window, sinks
    ([1], [1], 1, 1, 1, -1, 0),
    ([1, 5, 64, 65, 200], [1, 1, 1, 1, 1], 16, 4, 2, -1, 0),
    ([7, 300, 129, 1000], [7, 1, 40, 200], 16, 6, 2, 50, 3),
    ([333, 100], [333, 100], 100, 3, 3, -1, 0),       # prompts: every token is new
    ([500, 0, 70, 900], [3, 0, 70, 0], 7, 4, 4, 20, 0),  # sequences without tokens, without new ones
    ([2000], [1], 16, 8, 1, -1, 0),                   # cut into parts
    ([9000, 40], [2, 1], 128, 4, 2, 3000, 10),
    ([5000], [130], 64, 4, 2, 0, 0),                  # each its own key
    ([40, 30], [50, 30], 16, 2, 1, -1, 0),            # more new tokens than the cache has: the first see nothing
    ([700] * 70, [1] * 70, 32, 2, 2, 100, 4),         # more sequences than a wavefront has lanes
    ([260], [200], 300, 16, 1, -1, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths,new,page,q_heads,kv_heads,left,sinks", CASES)
def test_attention(lengths, new, page, q_heads, kv_heads, left, sinks, dim, dtype, announce):
    announce()
    cache = Cache(len(lengths) + page, lengths, page, kv_heads, dim, dtype)
    q, offsets, sizes = cache.queries(new, q_heads, tail=5)
    args = (cache.k_pages, cache.v_pages, cache.table, offsets, sizes)
    out = paged_attention(q, *args, window=left, sinks=sinks)
    cache.check(out, q, new, left, sinks)
    assert (out[sum(new):] == 0).all()
    given = torch.full_like(q, 7.0)
    assert paged_attention(q, *args, window=left, sinks=sinks, out=given) is given
    assert torch.equal(given[:sum(new)], out[:sum(new)]) and (given[sum(new):] == 7.0).all()


@pytest.mark.gpu
def test_layouts(announce):
    """Token-major pages, gaps, strided tables and queries: the bits of the plain call."""
    announce()
    cache = Cache(3, [300, 77, 1500], 16, 2, 64, torch.bfloat16)
    q, offsets, sizes = cache.queries([5, 1, 60], 6, tail=3)
    want = paged_attention(q, cache.k_pages, cache.v_pages, cache.table, offsets, sizes, window=90, sinks=2)
    k_pages = cache.k_pages.transpose(1, 2).contiguous().transpose(1, 2)
    v_pages = torch.zeros(*cache.v_pages.shape[:3], 72, dtype=torch.bfloat16, device=DEV)[..., :64].copy_(cache.v_pages)
    table = cache.table.repeat_interleave(2, 1)[:, ::2]
    many = torch.stack((offsets, offsets), 1)[:, 0], torch.stack((sizes, sizes), 1)[:, 1]
    other = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(paged_attention(other, k_pages, v_pages, table, *many, window=90, sinks=2), want)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape).copy_(q)
    assert torch.equal(paged_attention(odd, k_pages, v_pages, cache.table, offsets, sizes, window=90, sinks=2), want)
    out = torch.zeros(q.shape[0], 8, 64, dtype=q.dtype, device=DEV)[:, 1:7]
    assert torch.equal(paged_attention(q, k_pages, v_pages, cache.table, offsets, sizes, window=90, sinks=2, out=out), want)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[1, 1], [40, 200]])
def test_pages_that_are_not_held(new, announce):
    """Page numbers outside the cache hide their keys and are never read through; lengths and offsets past their
    tables are cut."""
    announce()
    cache = Cache(4, [900, 2500], 64, 2, 64, torch.bfloat16)
    q, offsets, sizes = cache.queries(new, 4)
    hide = [torch.zeros(n, dtype=torch.bool, device=DEV) for n in cache.lengths]
    for b, entry, value in ((0, 0, -1), (0, 5, cache.k_pages.shape[0]), (1, 20, -2147483648), (1, 21, 2147483647)):
        cache.table[b, entry] = value
        hide[b][64 * entry:64 * entry + 64] = True
    for left, sinks in ((-1, 0), (100, 30)):
        out = paged_attention(q, cache.k_pages, cache.v_pages, cache.table, offsets, sizes, window=left, sinks=sinks)
        cache.check(out, q, new, left, sinks, hide)
    # A length past the table counts as the table's 40 * 64 tokens.
    full = Cache(5, [2560, 2560], 64, 2, 64, torch.bfloat16)
    q, offsets, _ = full.queries(new, 4)
    far = torch.tensor([2147483647, 2561], dtype=torch.int32, device=DEV)
    out = paged_attention(q, full.k_pages, full.v_pages, full.table, offsets, far)
    full.check(out, q, new, -1, 0)
    low = torch.tensor([-7, -2147483648], dtype=torch.int32, device=DEV)
    assert (paged_attention(q, full.k_pages, full.v_pages, full.table, offsets, low) == 0).all()
    wild = torch.tensor([0, new[0], 2147483647], dtype=torch.int32, device=DEV)
    sizes = torch.tensor([2560, 2560], dtype=torch.int32, device=DEV)
    assert torch.equal(paged_attention(q, full.k_pages, full.v_pages, full.table, wild, sizes),
                       paged_attention(q, full.k_pages, full.v_pages, full.table, offsets, sizes))
    below = torch.tensor([-2147483648, -3, -3], dtype=torch.int32, device=DEV)
    assert (paged_attention(q, full.k_pages, full.v_pages, full.table, below, sizes) == 0).all()
    late = torch.tensor([1, 1, sum(new)], dtype=torch.int32, device=DEV)  # the first row is of no sequence
    out = paged_attention(q, full.k_pages, full.v_pages, full.table, late, sizes)
    assert (out[0] == 0).all() and (out[1:] != 0).any(-1).all()


@pytest.mark.gpu
def test_a_hidden_page_may_hold_anything(announce):
    """Tokens of earlier owners, NaN among them, in pages before the window and behind the last token."""
    announce()
    cache = Cache(6, [700], 16, 1, 128, torch.bfloat16)
    for new in ([1], [90]):
        q, offsets, sizes = cache.queries(new, 2)
        clean = paged_attention(q, cache.k_pages, cache.v_pages, cache.table, offsets, sizes, window=64, sinks=5)
        k_pages, v_pages = cache.k_pages.clone(), cache.v_pages.clone()
        first = 700 - new[0] - 64  # the first key of any window
        for entry in range(1, first // 16):
            k_pages[cache.table[0, entry]] = float("inf")
            v_pages[cache.table[0, entry]] = float("nan")
        out = paged_attention(q, k_pages, v_pages, cache.table, offsets, sizes, window=64, sinks=5)
        assert torch.equal(out, clean)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths,new,heads,page", [
    ([1], [1], 1, 1), ([5, 70, 200, 33], [5, 1, 90, 0], 3, 16), ([100] * 90, [1] * 90, 2, 7), ([3000], [2777], 24, 100)])
def test_append(lengths, new, heads, page, dim, dtype, announce):
    """The pages' other rows stay as they were; keys are turned as rotary_axes turns them, bit for bit."""
    announce()
    cache = Cache(7, lengths, page, heads, dim, dtype)
    rows_k, offsets, sizes = cache.queries(new, heads, tail=4)
    rows_v = torch.randn(rows_k.shape, device=DEV).to(dtype)
    tokens = rows_k.shape[0]
    positions = torch.randint(0, 5000, (3, tokens), dtype=torch.int32, device=DEV)
    plans = [None, RotaryAxes((16, 24, 24), 256.0), RotaryAxes((8, 16, 24)), RotaryAxes((16, 8, 8), 1e4, "halves", True)]
    for axes in plans:
        k_want, v_want = cache.k_pages.clone(), cache.v_pages.clone()
        turned = rows_k if axes is None else rotary_axes(rows_k.transpose(0, 1)[None], positions, axes)[0].transpose(0, 1)
        at = 0
        for b, n in enumerate(new):
            place = torch.arange(lengths[b] - n, lengths[b], device=DEV)
            page_of = cache.table[b, place // page].long()
            k_want[page_of, :, place % page] = turned[at:at + n]
            v_want[page_of, :, place % page] = rows_v[at:at + n]
            at += n
        for k, v in ((rows_k, rows_v), (rows_k.transpose(0, 1).contiguous().transpose(0, 1), rows_v)):
            k_pages, v_pages = cache.k_pages.clone(), cache.v_pages.clone()
            append_pages(k, v, k_pages, v_pages, cache.table, offsets, sizes,
                         rotary=None if axes is None else RotaryPositions(axes, positions))
            for got, want in ((k_pages, k_want), (v_pages, v_want)):
                assert torch.equal(got.view(torch.int16), want.view(torch.int16))


@pytest.mark.gpu
def test_append_passes_over_what_has_no_place(announce):
    announce()
    cache = Cache(8, [30, 40, 20], 16, 2, 64, torch.bfloat16, width=4)
    k, offsets, _ = cache.queries([10, 3, 20], 2)
    cache.table[0, 1] = cache.k_pages.shape[0]  # places 16..31 of sequence 0
    cache.table[1, 2] = -1                      # places 32..47 of sequence 1
    sizes = torch.tensor([20, 34, 70], dtype=torch.int32, device=DEV)  # sequence 2 ends past its 64 places
    k_pages, v_pages = cache.k_pages.clone(), cache.v_pages.clone()
    append_pages(k, k, k_pages, v_pages, cache.table, offsets, sizes)
    want = cache.k_pages.clone()
    want[cache.table[0, 0].long(), :, 10:16] = k[0:6].transpose(0, 1)
    want[cache.table[1, 1].long(), :, 15] = k[10]
    # Sequence 2 holds two pages: its places 50..69 lie behind them.
    assert torch.equal(k_pages.view(torch.int16), want.view(torch.int16))
    for offsets, sizes in (([0, 0, 0, 0], [20, 20, 20]), ([33, 33, 33, 33], [5, 5, 5]), ([0, 10, 13, 33], [0, -5, -2147483648])):
        before = k_pages.clone()
        append_pages(k, k, k_pages, v_pages, cache.table, torch.tensor(offsets, dtype=torch.int32, device=DEV),
                     torch.tensor(sizes, dtype=torch.int32, device=DEV))
        assert torch.equal(k_pages.view(torch.int16), before.view(torch.int16))


@pytest.mark.gpu
def test_generation_as_it_runs(announce):
    """A prompt, then single tokens: every step's keys turned and appended, its queries turned and attended, the
    steps after the first replayed from one captured graph. Each step's output equals window_attention's over the
    whole sequence within the two bounds (both within 2^-7 of the mean of |v|, bf16: 2 e + u and the joins' order)."""
    announce()
    heads, kv_heads, dim, page, prompt, steps = 4, 2, 64, 16, 75, 6
    axes, total = RotaryAxes((16, 24, 24), 256.0), 75 + 6
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(total, h, dim, generator=g).bfloat16().to(DEV) for h in (heads, kv_heads, kv_heads))
    positions = torch.stack([torch.arange(total) // 9, torch.arange(total) % 9 // 3, torch.arange(total) % 3]).int().to(DEV)

    def turn(x, at):
        return rotary_axes(x.transpose(0, 1)[None], at, axes)[0].transpose(0, 1)

    k_pages, v_pages = (torch.full((8, kv_heads, page, dim), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in "kv")
    table = torch.tensor([[5, 2, 7, 0, 1, 3]], dtype=torch.int32, device=DEV)

    def step(q, k, v, at, offsets, lengths):
        append_pages(k, v, k_pages, v_pages, table, offsets, lengths, rotary=RotaryPositions(axes, at))
        return paged_attention(turn(q, at), k_pages, v_pages, table, offsets, lengths, window=40, sinks=4)

    outs = [step(q[:prompt], k[:prompt], v[:prompt], positions[:, :prompt],
                 torch.tensor([0, prompt], dtype=torch.int32, device=DEV),
                 torch.tensor([prompt], dtype=torch.int32, device=DEV))]
    held = [t[prompt:prompt + 1].clone() for t in (q, k, v)] + [positions[:, prompt:prompt + 1].clone()]
    offsets = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([prompt + 1], dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = step(*held, offsets, lengths)
    for i in range(prompt, total):
        for t, x in zip(held, (q, k, v)):
            t.copy_(x[i:i + 1])
        held[3].copy_(positions[:, i:i + 1])
        lengths.fill_(i + 1)
        graph.replay()
        outs.append(result.clone())
    torch.cuda.synchronize()
    out = torch.cat(outs).transpose(0, 1)[None]
    whole = window_attention(turn(q, positions).transpose(0, 1)[None], turn(k, positions).transpose(0, 1)[None],
                             v.transpose(0, 1)[None], (40, 0), 4)
    assert torch.isfinite(out).all()
    assert (out.float() - whole.float()).abs().max() <= 2 * 2.0 ** -6 * v.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("first,last", [(0, 1), (700, 1100), (2000, 2000)])
def test_rows_of_no_sequence_in_a_wide_batch(first, last, announce):
    """A batch captured for 5000 new tokens that holds few: all other rows give 0."""
    announce()
    cache = Cache(8, [500, 1200], 16, 2, 64, torch.bfloat16)
    q = torch.randn(5000, 6, 64, device=DEV).bfloat16()
    offsets = torch.tensor([first, last, last], dtype=torch.int32, device=DEV)
    sizes = torch.tensor(cache.lengths, dtype=torch.int32, device=DEV)
    soil = torch.full_like(q, float("nan"))
    del soil  # (the result's memory, as a rule)
    out = paged_attention(q, cache.k_pages, cache.v_pages, cache.table, offsets, sizes)
    assert (out[:first] == 0).all() and (out[last:] == 0).all()
    assert (out[first:last] != 0).any(-1).all()


@pytest.mark.gpu
def test_expanded_places_to_write_are_refused(announce):
    announce()
    cache = Cache(9, [40], 16, 2, 64, torch.bfloat16)
    q, offsets, sizes = cache.queries([3], 2)
    wide = cache.k_pages[:1].expand(cache.k_pages.shape)
    args = (cache.table, offsets, sizes)
    for pages in ((wide, cache.v_pages), (cache.k_pages, wide)):
        with pytest.raises(ValueError, match="expanded"):
            append_pages(q, q, *pages, *args)
    with pytest.raises(ValueError, match="expanded"):
        paged_attention(q, cache.k_pages, cache.v_pages, *args, out=torch.empty_like(q[:1]).expand(q.shape))


def test_refusals():
    """No launch is reached: these run without a GPU."""
    q, pages = torch.zeros(3, 4, 64).bfloat16(), torch.zeros(5, 2, 16, 64).bfloat16()
    table, offsets, lengths = (torch.zeros(s, dtype=torch.int32) for s in ((2, 3), 3, 2))
    good = [q, pages, pages, table, offsets, lengths]

    def refused(kind, match, **changes):
        names = ["q", "k", "v", "table", "offsets", "lengths"]
        args = [changes.get(n, t) for n, t in zip(names, good)]
        with pytest.raises(kind, match=match):
            paged_attention(*args)
        if "q" not in changes:
            with pytest.raises(kind, match=match):
                append_pages(q[:, :2], q[:, :2], *args[1:])

    refused(TypeError, "torch tensors", k=None)
    refused(ValueError, "equal-shaped", v=pages[:, :, :8])
    refused(ValueError, "equal-shaped", k=pages[:0], v=pages[:0])
    refused(ValueError, "tokens,heads,D", q=q[0])
    refused(ValueError, "tokens,heads,D", q=q[..., :32])
    refused(ValueError, "64 and 128", q=q[..., :32], k=pages[..., :32], v=pages[..., :32])
    refused(TypeError, "share dtype", q=q.float())
    refused(TypeError, "share dtype", v=pages.half())
    refused(ValueError, "page_table", table=table[0])
    refused(ValueError, "page_table", table=table[:, :0])
    refused(ValueError, "offsets and lengths", offsets=offsets[:2])
    refused(ValueError, "offsets and lengths", lengths=offsets)
    refused(TypeError, "int32", table=table.long())
    refused(TypeError, "int32", lengths=lengths.float())
    refused(ValueError, "GPU device")
    with pytest.raises(ValueError, match="GPU device"):
        append_pages(q[:, :2], q[:, :2], *good[1:])


def test_entries_refuse_bad_arguments():
    import ctypes

    from peco_amd import _native
    from peco_amd.rotary import plan_arguments

    lib, null, some = _native.library(), ctypes.c_void_p(0), ctypes.c_void_p(4096)  # refused before it is read
    sizes = dict(batch=1, q_heads=2, kv_heads=1, tokens=3, pages=4, page=16, width=2, left=-1, sinks=0, scale=0.125,
                 d=64, dtype=1)
    head = dict(q=some, k=some, v=some, out=some, strides=[64] * 10, table=some, table_stride=2, offsets=some,
                lengths=some, clear=0, work=null, floats=0)

    def attend(**changes):
        a = {**head, **sizes, **changes}
        a["strides"] = (ctypes.c_int64 * 10)(*a["strides"])
        return lib.peco_paged_attention(*a.values(), null)

    for change in (dict(q=null), dict(v=null), dict(table=null), dict(offsets=null), dict(lengths=null), dict(batch=0),
                   dict(q_heads=3, kv_heads=2), dict(tokens=0), dict(pages=0), dict(page=0), dict(width=0),
                   dict(table_stride=-1), dict(left=-2), dict(sinks=-1), dict(scale=0.0), dict(strides=[64] * 9 + [63]),
                   dict(out=ctypes.c_void_p(4098))):
        assert attend(**change) == 1, change
    assert attend(d=32) == 20002 and attend(dtype=2) == 20003 and attend(width=1 << 26) == 20002
    floats = lib.peco_paged_attention_workspace_size(1, 2, 1, 3, 1000, 16, -1, 0, 64)
    assert floats > 0 and attend(width=1000, work=some, floats=floats - 1) == 20001

    plan = plan_arguments(RotaryAxes((16, 24, 24)), torch.zeros(3, 3, dtype=torch.int32))
    names = dict(k=some, v=some, kp=some, vp=some, strides=[64] * 10, table=some, table_stride=2, offsets=some,
                 lengths=some, plan=plan, batch=1, heads=2, tokens=3, pages=4, page=16, width=2, d=64, dtype=1)

    def append(**changes):
        a = {**names, **changes}
        a["strides"] = (ctypes.c_int64 * 10)(*a["strides"])
        values = list(a.values())
        return lib.peco_append_pages(*values[:9], *a["plan"], *values[10:], null)

    for change in (dict(k=null), dict(vp=null), dict(table=null), dict(batch=0), dict(heads=0), dict(tokens=0),
                   dict(pages=0), dict(page=0), dict(width=0), dict(strides=[60] * 10), dict(kp=ctypes.c_void_p(4100)),
                   dict(plan=(*plan[:4], None, *plan[5:]))):
        assert append(**change) == 1, change
    assert append(d=96) == 20002 and append(dtype=2) == 20003
