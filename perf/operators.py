"""Performance cases of the operators for clips that are generated in pieces or trained on.

Each case is a plain dict; its "kind" names the public entry point:

- "rotary": ``rotary.rotary_axes``, rotary positions with several axes over projected rows; with "train" the
  gradient of the rows too.
- "window": ``window.window_attention``, attention with a sliding window and first tokens that stay visible; with
  "train" the gradients of Q, K and V too.
- "append": ``paged.append_pages``, new keys (rotated) and values written to the pages of a cache.
- "paged": ``paged.paged_attention``, new tokens of several sequences over such a cache.

``listed`` holds the fixed cases, ``draw`` makes others of the same ranges, ``prepare`` the inputs, ``run`` one pass
(the framework's operators where ``own`` is set, else their plain form in torch), ``exact`` the same outputs in 64
bits from the definitions, ``work`` what a pass cannot do without.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---- cases ----

def _rotary(name, heads, grid, dim, axes, theta, layout, shared, dtype, train, first=0):
    return {"name": name, "kind": "rotary", "heads": heads, "frames": grid[0], "rows": grid[1], "columns": grid[2],
            "dim": dim, "time_dims": axes[0], "row_dims": axes[1], "column_dims": axes[2], "theta": theta,
            "layout": layout, "shared": shared, "dtype": dtype, "train": train, "first_frame": first}


def _window(name, batch, q_heads, kv_heads, queries, keys, dim, left, right, sinks, dtype, train):
    return {"name": name, "kind": "window", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads,
            "queries": queries, "keys": keys, "dim": dim, "left": left, "right": right, "sinks": sinks,
            "dtype": dtype, "train": train}


def _paged(name, sequences, q_heads, kv_heads, shortest, longest, new, page, dim, left, sinks, dtype):
    return {"name": name, "kind": "paged", "sequences": sequences, "q_heads": q_heads, "kv_heads": kv_heads,
            "shortest": shortest, "longest": longest, "new": new, "page": page, "dim": dim, "left": left,
            "sinks": sinks, "dtype": dtype}


def _append(name, sequences, heads, shortest, longest, new, page, dim, dtype):
    return {"name": name, "kind": "append", "sequences": sequences, "heads": heads, "shortest": shortest,
            "longest": longest, "new": new, "page": page, "dim": dim, "dtype": dtype}


def listed():
    return [
        # One frame's strip of tokens of a late frame on a head shard: a call that is all latency.
        _rotary("rotary_strip", 3, (1, 1, 45), 128, (16, 56, 56), 256.0, "interleaved", False, "bf16", False, 40000),
        # The 480p clip (5 latent frames of 30 x 45 tokens) in a training step: rows turned, gradients turned back.
        _rotary("rotary_480p_train", 24, (5, 30, 45), 128, (16, 56, 56), 256.0, "interleaved", False, "bf16", True),
        # The 720p clip (33 latent frames of 45 x 80 tokens), channel halves turned by one shared ladder.
        _rotary("rotary_720p_halves", 24, (33, 45, 80), 128, (32, 48, 48), 10000.0, "halves", True, "bf16", False),
        # Fine-tuning on short clips with shared key heads: a small training step.
        _window("window_small_train", 2, 8, 4, 777, 777, 64, 255, 0, 4, "fp16", True),
        # Fine-tuning on the 480p clip and its text: a window of one and a half frames, the text's rows stay visible.
        _window("window_480p_train", 1, 24, 24, 7006, 7006, 128, 2025, 0, 256, "bf16", True),
        # The 544p clip on one of eight GPUs (3 of 24 heads), a window to both sides, inference.
        _window("window_544p", 1, 3, 3, 32896, 32896, 128, 4079, 4079, 256, "bf16", False),
        # Two short sequences, one new token each: a call that is all latency.
        _paged("paged_token_small", 2, 4, 4, 500, 2112, 1, 16, 64, -1, 0, "fp16"),
        # A batch of sequences of up to the 480p clip's length, one new token each, three query heads a key head.
        _paged("paged_token_batch", 32, 24, 8, 600, 7006, 1, 64, 128, -1, 0, "bf16"),
        # One new token behind the whole 720p clip.
        _paged("paged_token_720p", 1, 24, 24, 119056, 119056, 1, 128, 128, -1, 0, "bf16"),
        # The next latent frame (30 x 45 tokens) of two 480p clips, a window of three frames and the text before it.
        _paged("paged_frame_480p", 2, 24, 24, 5656, 8356, 1350, 64, 128, 4050, 256, "bf16"),
        # One new token of each of a batch of sequences written to its cache.
        _append("append_token_batch", 32, 8, 60, 700, 1, 64, 128, "bf16"),
        # A latent frame (45 x 80 tokens) of two 720p clips, one of the first three, written to the cache.
        _append("append_frame_720p", 2, 24, 3856, 11056, 3600, 128, 128, "bf16"),
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rotary", "window", "window", "paged", "paged", "append"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    dim = rng.choice([64, 128])
    if kind == "rotary":
        frames, rows, columns = _spread(rng, 1, 33), _spread(rng, 1, 45), _spread(rng, 1, 80)
        axes = rng.choice([(16, 56, 56), (32, 48, 48), (44, 42, 42)]) if dim == 128 else \
            rng.choice([(16, 24, 24), (8, 24, 16)])
        layout = rng.choice(["interleaved", "interleaved", "halves"])
        if layout == "halves":
            axes = (32, 48, 48) if dim == 128 else (16, 24, 24)
        return {k: v for k, v in _rotary("", rng.randint(1, 24), (frames, rows, columns), dim, axes,
                                         rng.choice([256.0, 10000.0]), layout, rng.random() < 0.3,
                                         rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.5,
                                         rng.choice([0, rng.randint(0, 100000)])).items() if k != "name"}
    if kind == "window":
        kv = rng.choice([1, 2, 3, 4, 8])
        group = rng.choice([1, 1, 2, 3])
        train = rng.random() < 0.6
        keys = _spread(rng, 1, 7006 if train else 16384)
        queries = keys if rng.random() < 0.7 else _spread(rng, 1, keys)
        left = rng.choice([-1, _spread(rng, 1, 4096), _spread(rng, 1, 512)])
        right = rng.choice([0, 0, 0, _spread(rng, 1, 2048)])
        sinks = rng.choice([0, 4, _spread(rng, 1, 300)])
        # The plain form keeps whole score matrices: as many heads as fit beside the largest listed case.
        group = max(1, min(group, int(1.1e9 / (float(queries) * keys * kv)))) if queries * keys * kv > 4e8 else group
        kv = max(1, min(kv, int(1.1e9 / (float(queries) * keys * group))))
        return {k: v for k, v in _window("", rng.choice([1, 1, 2]) if keys < 3000 else 1, kv * group, kv, queries, keys,
                                         dim, left, right, sinks, dtype, train).items() if k != "name"}
    if kind == "paged":
        kv = rng.choice([1, 2, 4, 8, 24])
        group = rng.choice([1, 1, 3, 4, 8]) if kv <= 4 else rng.choice([1, 3])
        longest = _spread(rng, 64, 32768)
        sequences = max(1, min(_spread(rng, 1, 64), int(1.3e6 / (longest * kv))))
        new = rng.choice([1, 1, _spread(rng, 1, min(longest, 1350))])
        new = max(1, min(new, int(1e9 / (float(longest) * kv * group))))
        # The plain form keeps the padded batch's score matrices.
        sequences = max(1, min(sequences, int(6e8 / (float(new) * longest * kv * group))))
        return {k: v for k, v in _paged("", sequences, kv * group, kv, max(new, longest // rng.choice([1, 3, 10])),
                                        longest, new, rng.choice([16, 64, 100, 128]), dim,
                                        rng.choice([-1, _spread(rng, 1, 4096)]), rng.choice([0, 4, 256]),
                                        dtype).items() if k != "name"}
    new = rng.choice([1, _spread(rng, 1, 3600)])
    sequences = max(1, min(_spread(rng, 1, 64), 8000 // new))
    longest = max(new, _spread(rng, 64, 16384))
    return {k: v for k, v in _append("", sequences, rng.choice([1, 2, 8, 24]), max(new, longest // 4), longest, new,
                                     rng.choice([16, 64, 100, 128]), dim, dtype).items() if k != "name"}


# ---- inputs ----

def _grid_positions(first, frames, rows, columns):
    """int32 [3, frames * rows * columns]: each token's frame, row and column."""
    axes = torch.meshgrid(torch.arange(first, first + frames), torch.arange(rows), torch.arange(columns),
                          indexing="ij")
    return torch.stack([a.reshape(-1) for a in axes]).to(torch.int32).to(DEVICE)


def _sequence_lengths(case):
    """Host numbers: each sequence's length with the new tokens, and how many of them are new (ragged; the same for
    every seed, so that outputs of two seeds have one shape)."""
    rng = random.Random(case["longest"])
    lengths = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["sequences"])]
    lengths[0] = case["longest"]
    new = [rng.randint(-(-case["new"] // 2), case["new"]) for _ in lengths]
    new[0] = case["new"]
    return lengths, [min(a, b) for a, b in zip(new, lengths)]


def _cache(case, gen, heads):
    """Pages in a random order, the table of every sequence, and the ragged batch's offsets and lengths."""
    lengths, new = _sequence_lengths(case)
    page, dim, dtype = case["page"], case["dim"], _DTYPES[case["dtype"]]
    held = [-(-n // page) for n in lengths]
    pages, width = sum(held) + 3, max(held)
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((case["sequences"], width), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
    offsets = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEVICE)
    shape = (pages, heads, page, dim)
    return {"k_pages": torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype),
            "v_pages": torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype),
            "table": table, "offsets": offsets, "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEVICE),
            "tokens": sum(new), "most_new": max(new)}


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype, dim = _DTYPES[case["dtype"]], case["dim"]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device=DEVICE) * scale).to(dtype)

    state = {"case": case}
    if case["kind"] == "rotary":
        positions = _grid_positions(case["first_frame"], case["frames"], case["rows"], case["columns"])
        # As a projection leaves them: rows of all heads, seen head-major.
        rows = positions.shape[1]
        state |= {"positions": positions, "x": normal(1, rows, case["heads"], dim).transpose(1, 2)}
        if case["train"]:
            state |= {"x": state["x"].requires_grad_(), "grad": normal(1, rows, case["heads"], dim,
                                                                       scale=0.01).transpose(1, 2)}
    elif case["kind"] == "window":
        b, hq, hk = case["batch"], case["q_heads"], case["kv_heads"]
        state |= {"q": normal(b, hq, case["queries"], dim, scale=1.5), "k": normal(b, hk, case["keys"], dim),
                  "v": normal(b, hk, case["keys"], dim)}
        if case["train"]:
            for name in ("q", "k", "v"):
                state[name].requires_grad_()
            state["grad"] = normal(b, hq, case["queries"], dim, scale=0.01)
    elif case["kind"] == "paged":
        state |= _cache(case, gen, case["kv_heads"])
        state["q"] = normal(state["tokens"], case["q_heads"], dim, scale=1.5)
    else:
        state |= _cache(case, gen, case["heads"])
        state |= {"k": normal(state["tokens"], case["heads"], dim), "v": normal(state["tokens"], case["heads"], dim),
                  "positions": torch.randint(0, 4096, (3, state["tokens"]), generator=gen, device=DEVICE,
                                             dtype=torch.int32)}
    return state


def _axes(case):
    """(dims of the axes, theta, layout, one shared ladder)."""
    if case["kind"] == "append":
        return ((16, 56, 56) if case["dim"] == 128 else (16, 24, 24)), 256.0, "interleaved", False
    return (case["time_dims"], case["row_dims"], case["column_dims"]), case["theta"], case["layout"], case["shared"]


# ---- plain forms ----

def _frequencies(dims, theta, shared):
    """Per pair of channels: its axis and its frequency (float64)."""
    axis = torch.cat([torch.full((d // 2,), a) for a, d in enumerate(dims)])
    if shared:
        steps = torch.arange(sum(dims) // 2, dtype=torch.float64) * 2 / sum(dims)
    else:
        steps = torch.cat([torch.arange(d // 2, dtype=torch.float64) * 2 / d for d in dims])
    return axis.to(DEVICE), (theta ** -steps).to(DEVICE)


def _turn(x, positions, axes, sign=1.0):
    """x [..., S, D] turned by positions [A, S] (angles in 64 bits, the rows in 32)."""
    dims, theta, layout, shared = axes
    axis, freq = _frequencies(dims, theta, shared)
    angle = positions[axis].double().T * freq  # [S, pairs]
    cos, sin = angle.cos().float(), angle.sin().float() * sign
    pairs, wide = freq.shape[0], x.float()
    turned, rest = wide[..., :2 * pairs], wide[..., 2 * pairs:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if layout == "interleaved" else turned.split(pairs, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if layout == "interleaved" else torch.cat((a, b), -1)
    return torch.cat((turned, rest), -1).to(x.dtype)


def _visible(queries, keys, left, right, sinks):
    """bool [queries, keys]: the last query stands at the last key."""
    p = torch.arange(queries, device=DEVICE)[:, None] + (keys - queries)
    j = torch.arange(keys, device=DEVICE)[None, :]
    seen = torch.ones((queries, keys), dtype=torch.bool, device=DEVICE)
    if right >= 0:
        seen &= j <= p + right
    if left >= 0:
        seen &= (j >= p - left) | (j < sinks)
    return seen


def _weights(scores, seen):
    """Softmax over the seen keys, 0 in a row that sees none."""
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min_(-3e38)
    scores.sub_(top).exp_()
    return scores.div_(scores.sum(-1, keepdim=True).clamp_min_(1e-38))


def _plain_window(state):
    case = state["case"]
    q, k, v = (state[n].detach().float() for n in ("q", "k", "v"))
    b, hq, sq, d = q.shape
    hk, sk = k.shape[1:3]
    g, scale, dtype = hq // hk, 1.0 / math.sqrt(d), state["q"].dtype
    q = q.reshape(b, hk, g * sq, d)
    seen = _visible(sq, sk, case["left"], case["right"], case["sinks"]).repeat(g, 1)
    p = _weights(torch.matmul(q, k.transpose(2, 3)).mul_(scale), seen)
    out = torch.matmul(p, v)
    result = {"out": out.reshape(b, hq, sq, d).to(dtype)}
    if case["train"]:
        grad = state["grad"].float().reshape(b, hk, g * sq, d)
        result["v_grad"] = torch.matmul(p.transpose(2, 3), grad).to(dtype)
        ds = torch.matmul(grad, v.transpose(2, 3)).sub_((grad * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        result["q_grad"] = torch.matmul(ds, k).reshape(b, hq, sq, d).to(dtype)
        result["k_grad"] = torch.matmul(ds.transpose(2, 3), q).to(dtype)
    return result


def _token_places(state):
    """Each new token's sequence, its number among the sequence's new tokens and its position in the sequence."""
    offsets, lengths = state["offsets"].long(), state["lengths"].long()
    token = torch.arange(state["tokens"], device=DEVICE)
    sequence = torch.searchsorted(offsets, token, right=True) - 1
    number = token - offsets[sequence]
    return sequence, number, lengths[sequence] - (offsets[sequence + 1] - offsets[sequence]) + number


def _plain_paged(state):
    case = state["case"]
    b, m = state["table"].shape
    hk, page, d = state["k_pages"].shape[1:]
    hq, most, dtype = state["q"].shape[1], state["most_new"], state["q"].dtype
    g, keys = hq // hk, m * page
    at = state["table"].clamp_min(0).long()
    k, v = (state[n][at].transpose(1, 2).reshape(b, hk, keys, d).float() for n in ("k_pages", "v_pages"))
    sequence, number, position = _token_places(state)
    q = torch.zeros((b, most, hq, d), device=DEVICE)
    q[sequence, number] = state["q"].float()
    p_of = torch.full((b, most), -1, dtype=torch.long, device=DEVICE)
    p_of[sequence, number] = position
    j = torch.arange(keys, device=DEVICE)
    seen = j <= p_of[..., None]
    if case["left"] >= 0:
        seen &= (j >= p_of[..., None] - case["left"]) | (j < case["sinks"])
    q = q.reshape(b, most, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b, hk, g * most, d)
    p = _weights(torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(d)), seen.repeat(1, g, 1)[:, None])
    out = torch.matmul(p, v).reshape(b, hk, g, most, d).permute(0, 3, 1, 2, 4).reshape(b, most, hq, d)
    return out[sequence, number].to(dtype)


def _plain_append(state):
    sequence, _, position = _token_places(state)
    page = state["k_pages"].shape[2]
    at, slot = state["table"][sequence, position // page].long(), position % page
    turned = _turn(state["k"].transpose(0, 1), state["positions"], _axes(state["case"])).transpose(0, 1)
    state["k_pages"][at, :, slot] = turned
    state["v_pages"][at, :, slot] = state["v"]
    return {"k_pages": state["k_pages"], "v_pages": state["v_pages"]}


# ---- one pass ----

def _framework(state):
    case = state["case"]
    if case["kind"] == "rotary":
        from peco_amd.rotary import RotaryAxes, rotary_axes

        out = rotary_axes(state["x"], state["positions"], RotaryAxes(*_axes(case)))
        if not case["train"]:
            return {"out": out}
        return {"out": out.detach(), "x_grad": torch.autograd.grad(out, state["x"], state["grad"])[0]}
    if case["kind"] == "window":
        from peco_amd.window import window_attention

        out = window_attention(state["q"], state["k"], state["v"], (case["left"], case["right"]), case["sinks"])
        if not case["train"]:
            return {"out": out}
        grads = torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["grad"])
        return {"out": out.detach(), "q_grad": grads[0], "k_grad": grads[1], "v_grad": grads[2]}
    if case["kind"] == "paged":
        from peco_amd.paged import paged_attention

        return paged_attention(state["q"], state["k_pages"], state["v_pages"], state["table"], state["offsets"],
                               state["lengths"], window=case["left"], sinks=case["sinks"])
    from peco_amd.paged import append_pages
    from peco_amd.rotary import RotaryAxes, RotaryPositions

    append_pages(state["k"], state["v"], state["k_pages"], state["v_pages"], state["table"], state["offsets"],
                 state["lengths"], rotary=RotaryPositions(RotaryAxes(*_axes(case)), state["positions"]))
    return {"k_pages": state["k_pages"], "v_pages": state["v_pages"]}


def run(state):
    if own:
        return _framework(state)
    kind = state["case"]["kind"]
    with torch.no_grad():
        if kind == "rotary":
            axes = _axes(state["case"])
            result = {"out": _turn(state["x"], state["positions"], axes)}
            if state["case"]["train"]:
                result["x_grad"] = _turn(state["grad"], state["positions"], axes, -1.0)
            return result
        return {"window": _plain_window, "paged": _plain_paged, "append": _plain_append}[kind](state)


# ---- work ----

def _pairs(queries, keys, left, right, sinks):
    """Number of (query, key) pairs that are seen, and of keys that some query sees."""
    first = keys - queries
    p = torch.arange(first, keys, dtype=torch.int64)
    top = torch.clamp(p + right, max=keys - 1) if right >= 0 else torch.full_like(p, keys - 1)
    low = torch.clamp(p - left, min=0) if left >= 0 else torch.zeros_like(p)
    kept = torch.minimum(torch.minimum(low, torch.full_like(low, max(sinks, 0))), top + 1)
    seen = torch.clamp(top + 1, min=0) - torch.minimum(low, torch.clamp(top + 1, min=0)) + torch.clamp(kept, min=0)
    from_low = max(0, int(low[0]))
    return int(seen.sum()), int(top[-1]) + 1 - from_low + min(max(sinks, 0), from_low)


def work(case):
    size, dim = _BYTES[case["dtype"]], case["dim"]
    if case["kind"] == "rotary":
        rows = case["frames"] * case["rows"] * case["columns"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * rows * case["heads"] * dim * size + 12 * rows),
                "flops": passes * 6 * rows * case["heads"] * dim // 2}
    if case["kind"] == "window":
        pairs, _ = _pairs(case["queries"], case["keys"], case["left"], case["right"], case["sinks"])
        rows = case["batch"] * case["q_heads"] * case["queries"] * dim * size
        cols = case["batch"] * case["kv_heads"] * case["keys"] * dim * size
        if case["train"]:  # in: q, k, v, grad; out: out, the three gradients
            return {"bytes": 4 * rows + 4 * cols, "flops": 14 * dim * pairs * case["batch"] * case["q_heads"]}
        return {"bytes": 2 * rows + 2 * cols, "flops": 4 * dim * pairs * case["batch"] * case["q_heads"]}
    lengths, new = _sequence_lengths(case)
    if case["kind"] == "append":
        return {"bytes": sum(new) * (4 * case["heads"] * dim * size + 12), "flops": sum(new) * 3 * case["heads"] * dim}
    total = [_pairs(n, keys, case["left"], 0, case["sinks"]) for n, keys in zip(new, lengths)]
    return {"bytes": 2 * sum(t[1] for t in total) * case["kv_heads"] * dim * size +
            2 * sum(new) * case["q_heads"] * dim * size,
            "flops": 4 * dim * case["q_heads"] * sum(t[0] for t in total)}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    def turn(x, positions, axes, conjugate=False):
        """Pairs of channels as complex numbers times exp(i angle)."""
        dims, theta, layout, shared = axes
        z, pair = x.double(), 0
        out = z.clone()
        half = sum(dims) // 2
        for a, d in enumerate(dims):
            for i in range(d // 2):
                ladder = 2.0 * pair / (2 * half) if shared else 2.0 * i / d
                angle = positions[a].double() * theta ** (-ladder)
                c0, c1 = (2 * pair, 2 * pair + 1) if layout == "interleaved" else (pair, pair + half)
                phase = torch.polar(torch.ones_like(angle), -angle if conjugate else angle)
                w = torch.complex(z[..., c0], z[..., c1]) * phase
                out[..., c0], out[..., c1] = w.real, w.imag
                pair += 1
        return out

    def rows_of(q, k, v, position, left, right, sinks, grad=None):
        """One head: queries q [n, d] at position [n] (long) over k, v [m, d]; with grad the gradients as well."""
        q, k, v = q.double(), k.double(), v.double()
        scale, step = q.shape[1] ** -0.5, 4096
        j = torch.arange(k.shape[0], device=DEVICE)
        outs, dq, dk, dv = [], [], torch.zeros_like(k), torch.zeros_like(v)
        for i in range(0, q.shape[0], step):
            p = position[i:i + step, None]
            hidden = torch.zeros((p.shape[0], k.shape[0]), dtype=torch.bool, device=DEVICE)
            if right >= 0:
                hidden |= j > p + right
            if left >= 0:
                hidden |= (j < p - left) & (j >= sinks)
            s = (q[i:i + step] @ k.T) * scale
            s[hidden] = -math.inf
            none = hidden.all(1, keepdim=True)
            w = torch.softmax(s.masked_fill(none, 0.0), 1).masked_fill(none, 0.0)
            del s, hidden
            outs.append(w @ v)
            if grad is not None:
                g = grad[i:i + step].double()
                dv += w.T @ g
                dw = g @ v.T
                ds = w * (dw - (dw * w).sum(1, keepdim=True)) * scale
                dq.append(ds @ k)
                dk += ds.T @ q[i:i + step]
        return torch.cat(outs), torch.cat(dq) if grad is not None else None, dk, dv

    state = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "rotary":
            result = {"out": turn(state["x"].detach(), state["positions"], _axes(case))}
            if case["train"]:
                result["x_grad"] = turn(state["grad"], state["positions"], _axes(case), conjugate=True)
            return result
        if case["kind"] == "window":
            q, k, v = (state[n].detach() for n in ("q", "k", "v"))
            g = case["q_heads"] // case["kv_heads"]
            position = torch.arange(case["queries"], device=DEVICE) + case["keys"] - case["queries"]
            out, dq = (torch.empty(q.shape, dtype=torch.float64, device=DEVICE) for _ in range(2))
            dk, dv = (torch.zeros(k.shape, dtype=torch.float64, device=DEVICE) for _ in range(2))
            for b in range(case["batch"]):
                for h in range(case["q_heads"]):
                    grad = state["grad"][b, h] if case["train"] else None
                    o, a, c, e = rows_of(q[b, h], k[b, h // g], v[b, h // g], position, case["left"],
                                         case["right"], case["sinks"], grad)
                    out[b, h] = o
                    if case["train"]:
                        dq[b, h] = a
                        dk[b, h // g] += c
                        dv[b, h // g] += e
            return {"out": out, "q_grad": dq, "k_grad": dk, "v_grad": dv} if case["train"] else {"out": out}
        lengths, offsets, table = state["lengths"].tolist(), state["offsets"].tolist(), state["table"]
        page = case["page"]
        if case["kind"] == "paged":
            q, g = state["q"], case["q_heads"] // case["kv_heads"]
            out = torch.empty(q.shape, dtype=torch.float64, device=DEVICE)
            for b, n in enumerate(lengths):
                j = torch.arange(n, device=DEVICE)
                at, slot = table[b, j // page].long(), j % page
                first, last = offsets[b], offsets[b + 1]
                position = torch.arange(n - (last - first), n, device=DEVICE)
                for h in range(case["q_heads"]):
                    k, v = (state[name][at, h // g, slot] for name in ("k_pages", "v_pages"))
                    out[first:last, h] = rows_of(q[first:last, h], k, v, position, case["left"], 0,
                                                 case["sinks"])[0]
            return out
        k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
        turned = turn(state["k"].transpose(0, 1), state["positions"], _axes(case)).transpose(0, 1)
        for b, n in enumerate(lengths):
            first, last = offsets[b], offsets[b + 1]
            j = torch.arange(n - (last - first), n, device=DEVICE)
            at, slot = table[b, j // page].long(), j % page
            k_pages[at, :, slot] = turned[first:last]
            v_pages[at, :, slot] = state["v"][first:last].double()
        return {"k_pages": k_pages, "v_pages": v_pages}
