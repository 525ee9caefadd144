"""Performance cases of the operators around a block's attention: its layer norm and its projections in 8 bits.

Each case is a plain dict; its "kind" names the public entry points:

- "norm": ``norm.layer_norm``, rows normalised over their channels with a weight and a bias (one for all rows, or one
  for each batch entry, as a modulation gives them); with "train" the gradients of the rows, weight and bias too.
- "linear": ``projection.int8_linear``, rows quantized to 8 bits (a scale a row) and multiplied with a weight of 8-bit
  codes (a scale an output channel).
- "norm_linear": ``norm.layer_norm_rows`` and ``projection.int8_linear``, the norm's rows quantized as they are made
  and multiplied with such a weight.

``listed`` holds the fixed cases, ``draw`` makes others of the same ranges, ``prepare`` the inputs, ``run`` one pass
(the framework's operators where ``own`` is set, else their plain form in torch), ``exact`` the same outputs in 64
bits from the definitions, ``work`` what a pass cannot do without.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6


# ---- cases ----

def _norm(name, batch, heads, rows, channels, per_entry, dtype, train):
    """heads 0: rows [batch, rows, channels]; else the head-major view [batch, heads, rows, channels] of a projection."""
    return {"name": name, "kind": "norm", "batch": batch, "heads": heads, "rows": rows, "channels": channels,
            "per_entry": per_entry, "dtype": dtype, "train": train}


def _linear(name, rows, channels, outputs, bias, dtype):
    return {"name": name, "kind": "linear", "batch": 1, "rows": rows, "channels": channels, "outputs": outputs,
            "bias": bias, "dtype": dtype}


def _norm_linear(name, batch, rows, channels, outputs, per_entry, bias, dtype):
    return {"name": name, "kind": "norm_linear", "batch": batch, "rows": rows, "channels": channels,
            "outputs": outputs, "per_entry": per_entry, "bias": bias, "dtype": dtype}


def listed():
    return [
        # The norm of one new token in front of its projections: a call that is all latency.
        _norm("norm_token", 1, 0, 1, 2048, False, "bf16", False),
        # The 480p clip and its text (6750 + 256 tokens), modulated by the step's embedding, inference.
        _norm("norm_480p", 1, 0, 7006, 2048, True, "bf16", False),
        # The 720p clip (118800 + 256 tokens) at a wide model's channels.
        _norm("norm_720p", 1, 0, 119056, 4096, False, "fp16", False),
        # Fine-tuning on two 480p clips, each with its own modulation: a training step of the block's norm.
        _norm("norm_480p_train", 2, 0, 7006, 2048, True, "bf16", True),
        # The norm of the query heads of a 480p clip in a training step: many short rows, one small weight.
        _norm("norm_heads_train", 1, 24, 7006, 128, False, "bf16", True),
        # Full-precision fine-tuning with rows of an odd length.
        _norm("norm_odd_train", 3, 0, 777, 1111, False, "fp32", True),
        # One new token through the joint query/key/value projection: a call that streams the weight.
        _linear("linear_token", 1, 2048, 6144, True, "bf16"),
        # The prompt's 256 tokens through a projection.
        _linear("linear_text", 256, 4096, 4096, False, "fp16"),
        # The 480p clip and its text through the joint query/key/value projection.
        _linear("linear_480p", 7006, 2048, 6144, True, "bf16"),
        # The 720p clip and its text through the output projection of a wide model.
        _linear("linear_720p", 119056, 4096, 4096, False, "bf16"),
        # A few new tokens at odd sizes.
        _norm_linear("norm_linear_few", 1, 33, 1000, 1111, False, True, "fp16"),
        # The 480p clip and its text from the residual rows to queries, keys and values.
        _norm_linear("norm_linear_480p", 1, 7006, 2048, 6144, True, True, "bf16"),
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _channels(rng, low, high):
    """A row length: mostly a multiple of 64, some multiples of 8 and some odd ones."""
    n, step = _spread(rng, low, high), rng.choice([64, 64, 64, 8, 1])
    return max(low, n // step * step)


def draw(rng):
    kind = rng.choice(["norm", "norm", "linear", "linear", "norm_linear"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "norm":
        train = rng.random() < 0.5
        if rng.random() < 0.25:
            heads, dim = rng.randint(1, 32), rng.choice([64, 128])
            rows = _spread(rng, 1, min(32896, 100_000_000 // (heads * dim)))
            case = _norm("", rng.choice([1, 2]), heads, rows, dim, rng.random() < 0.3, dtype, train)
        else:
            channels = _channels(rng, 8, 8192)
            rows = _spread(rng, 1, max(1, min(32896, 100_000_000 // channels)))
            case = _norm("", rng.choice([1, 1, 2, 3]), 0, rows, channels, rng.random() < 0.5, dtype, train)
    else:
        channels, outputs = _channels(rng, 64, 8192), _channels(rng, 64, 8192)
        rows = min(_spread(rng, 1, 32896), int(1.9e12 / (channels * outputs)))
        if kind == "linear":
            case = _linear("", rows, channels, outputs, rng.random() < 0.5, dtype)
        else:
            batch = rng.choice([1, 1, 2, 3])
            # 16-bit rows: in fp32 the results' own precision would be finer than what a border between two codes moves.
            dtype = rng.choice(["bf16", "fp16"])
            case = _norm_linear("", batch, max(1, rows // batch), channels, outputs, rng.random() < 0.5,
                                rng.random() < 0.5, dtype)
    return {k: v for k, v in case.items() if k != "name"}


# ---- inputs ----

def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype, channels = _DTYPES[case["dtype"]], case["channels"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device=DEVICE) * scale

    def rows(*shape):
        """Rows as a residual stream has them: every row of its own size, a few channels much larger."""
        size = torch.exp(normal(*shape[:-1], 1, scale=0.5))
        wide = 1.0 + 7.0 * (torch.rand(shape[-1], generator=gen, device=DEVICE) < 0.01)
        return (normal(*shape) * size * wide + 0.1).to(dtype)

    state = {"case": case}
    heads = case.get("heads", 0)
    batch, count = case["batch"], case["rows"]
    if heads:
        state["x"] = rows(batch, count, heads, channels).transpose(1, 2)
    elif case["kind"] == "linear":
        state["x"] = rows(count, channels)
    else:
        state["x"] = rows(batch, count, channels)
    if case["kind"] != "linear":
        # A modulation (shift and scale around one) a batch entry, or a trained weight and bias.
        shape = (batch, channels) if case["per_entry"] else (channels,)
        state["weight"] = (normal(*shape, scale=0.2) + (0.0 if case["per_entry"] else 1.0)).to(dtype)
        state["bias"] = normal(*shape, scale=0.2).to(dtype)
    if case["kind"] == "norm":
        if case["train"]:
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_()
            state["grad"] = normal(*state["x"].shape, scale=0.01).to(dtype)
    else:
        # The weight as the program keeps it: codes in rows of whole 16 bytes, a scale an output channel.
        outputs, pitch = case["outputs"], -(-channels // 16) * 16
        codes = torch.empty((outputs, pitch), dtype=torch.int8, device=DEVICE)[:, :channels]
        state["codes"] = codes.copy_((normal(outputs, channels) * 40).round_().clamp_(-127, 127))
        state["scales"] = (0.5 + torch.rand(outputs, generator=gen, device=DEVICE)) / (40.0 * math.sqrt(channels))
        state["linear_bias"] = normal(outputs, scale=0.2).to(dtype) if case["bias"] else None
    return state


# ---- plain forms ----

def _affine(state, x):
    """Weight and bias in fp32, broadcast over x's rows."""
    w, b = state["weight"].detach().float(), state["bias"].detach().float()
    if state["case"]["per_entry"]:
        shape = (w.shape[0], *[1] * (x.dim() - 2), w.shape[1])
        w, b = (w + 1.0).view(shape), b.view(shape)
    return w, b


def _normalised(x):
    """Rows of x (fp32) minus their mean, over their deviation; and one over the deviation."""
    centred = x - x.mean(-1, keepdim=True)
    inverse = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + _EPS)
    return centred.mul_(inverse), inverse


def _plain_norm(state):
    case, x = state["case"], state["x"].detach()
    dtype = x.dtype
    w, b = _affine(state, x)
    normalised, inverse = _normalised(x.float())
    result = {"out": (normalised * w).add_(b).to(dtype)}
    if case["train"]:
        grad = state["grad"].float()
        over = tuple(range(1 if case["per_entry"] else 0, x.dim() - 1))
        result["bias_grad"] = grad.sum(over).to(dtype)
        result["weight_grad"] = (grad * normalised).sum(over).to(dtype)
        grad = grad * w
        along = (grad * normalised).mean(-1, keepdim=True)
        result["x_grad"] = (grad - grad.mean(-1, keepdim=True)).sub_(normalised.mul_(along)).mul_(inverse).to(dtype)
    return result


def _plain_product(state, rows, dtype):
    """fp32 rows quantized to 127 steps of their largest magnitude, times the weight's codes."""
    most = rows.abs().amax(-1, keepdim=True)
    codes = (rows * (127.0 / most)).round_()
    out = torch.matmul(codes, state["codes"].float().T).mul_(most / 127.0).mul_(state["scales"])
    return (out if state["linear_bias"] is None else out.add_(state["linear_bias"].float())).to(dtype)


def _plain_norm_linear(state):
    x = state["x"]
    w, b = _affine(state, x)
    return _plain_product(state, _normalised(x.float())[0].mul_(w).add_(b), x.dtype)


# ---- one pass ----

def _framework(state):
    case, x = state["case"], state["x"]
    if case["kind"] == "norm":
        from peco_amd.norm import layer_norm

        out = layer_norm(x, state["weight"], state["bias"], _EPS, around_one=case["per_entry"])
        if not case["train"]:
            return {"out": out}
        grads = torch.autograd.grad(out, (x, state["weight"], state["bias"]), state["grad"])
        return {"out": out.detach(), "x_grad": grads[0], "weight_grad": grads[1], "bias_grad": grads[2]}
    from peco_amd.projection import QuantizedRows, int8_linear

    weight = QuantizedRows(state["codes"], state["scales"])
    if case["kind"] == "linear":
        return int8_linear(x, weight, state["linear_bias"])
    from peco_amd.norm import layer_norm_rows

    rows = layer_norm_rows(x, state["weight"], state["bias"], _EPS, around_one=case["per_entry"])
    return int8_linear(rows, weight, state["linear_bias"], dtype=x.dtype)


def run(state):
    if own:
        return _framework(state)
    kind = state["case"]["kind"]
    with torch.no_grad():
        if kind == "norm":
            return _plain_norm(state)
        if kind == "linear":
            return _plain_product(state, state["x"].float(), state["x"].dtype)
        return _plain_norm_linear(state)


# ---- work ----

def work(case):
    size, channels = _BYTES[case["dtype"]], case["channels"]
    rows = case["batch"] * max(case.get("heads", 0), 1) * case["rows"]
    affine = 2 * channels * (case["batch"] if case.get("per_entry") else 1) * size if case["kind"] != "linear" else 0
    if case["kind"] == "norm":
        if case["train"]:  # in: x, grad, weight, bias; out: out and the three gradients
            return {"bytes": 4 * rows * channels * size + 2 * affine, "flops": 19 * rows * channels}
        return {"bytes": 2 * rows * channels * size + affine, "flops": 7 * rows * channels}
    outputs = case["outputs"]
    weight = outputs * (channels + 4 + (size if case["bias"] else 0))
    return {"bytes": rows * (channels + outputs) * size + affine + weight, "flops": 2 * rows * channels * outputs}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    state = prepare(case, seed)
    x = state["x"].detach().double()
    train = case.get("train", False)
    leaves = []

    def normed():
        w, b = state["weight"].detach().double(), state["bias"].detach().double()
        rows = x
        if train:
            rows, w, b = rows.requires_grad_(), w.requires_grad_(), b.requires_grad_()
            leaves.extend((rows, w, b))
        if case["per_entry"]:
            middle = [1] * (rows.dim() - 2)
            w, b = 1 + w.unflatten(0, (-1, *middle)), b.unflatten(0, (-1, *middle))
        variance, mean = torch.var_mean(rows, -1, correction=0, keepdim=True)
        return (rows - mean) / (variance + _EPS) ** 0.5 * w + b

    if case["kind"] == "norm":
        if not train:
            return {"out": normed()}
        out = normed()
        grads = torch.autograd.grad(out, leaves, state["grad"].double())
        return {"out": out.detach(), "x_grad": grads[0], "weight_grad": grads[1], "bias_grad": grads[2]}
    rows = x if case["kind"] == "linear" else normed()
    del x
    step = rows.abs().max(-1, keepdim=True).values / 127
    weight = state["codes"].double() * state["scales"].double()[:, None]
    out = (torch.round(rows / step) * step) @ weight.T
    return out if state["linear_bias"] is None else out + state["linear_bias"].double()
