"""Attention with a window and sinks from its definition in 64 bits, and how far a kernel may be from it.

``rows`` is one head. Bounds, with u half a step of the type (2^-8 bf16, 2^-11 fp16):
a score is a sum of D exact products in fp32, off by at most (D + 2) 2^-24 sum |q_i k_i|, so a weight is off by
that times scale, by 2^-21 for the exponential and its argument, and by u for its rounding (and by half the
smallest fp16 step, 2^-25 of the largest weight). Call it e, relative. Weights off by e move a weighted mean m of
x by at most 2 e sum w |x| (numerator and denominator, each by e), summation in fp32 by n 2^-24 sum w |x|.
"""
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def seen_keys(positions, keys, left, right, sinks):
    j = torch.arange(keys, device=positions.device)[None]
    p = positions[:, None]
    seen = torch.ones((positions.numel(), keys), dtype=torch.bool, device=positions.device)
    if right >= 0:
        seen &= j <= p + right
    if left >= 0:
        seen &= (j >= p - left) | (j < sinks)
    return seen


def rows(q, k, v, seen, scale):
    """(out, its bound, weights, error of a weight) of one head: q [n, d], k, v [m, d], seen [n, m]."""
    unit, d = UNIT[q.dtype], q.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    s = (q @ k.T * scale).masked_fill(~seen, -float("inf"))
    none = ~seen.any(1, keepdim=True)
    w = torch.softmax(s.masked_fill(none, 0.0), 1).masked_fill(none | ~seen, 0.0)
    out = w @ v
    e = unit + 2.0 ** -21 + scale * (d + 2) * 2.0 ** -24 * float((q.abs() @ k.abs().T).max() if seen.numel() else 0)
    tiny = 2.0 ** -25 * w.amax(1, keepdim=True) if unit == 2.0 ** -11 and w.numel() else torch.zeros_like(q[:, :1])
    mass = w @ v.abs()
    bound = (2 * e + seen.shape[1] * 2.0 ** -24) * 1.05 * mass + unit * out.abs() * 1.05 + \
        2 * tiny * v.abs().sum(0, keepdim=True) + 2.0 ** -25
    return out, bound, w, e


def attention(q, k, v, left, right, sinks, scale=None, lengths=None):
    """(out, bound) [B,HQ,SQ,D] for q [B,HQ,SQ,D], k, v [B,HK,SK,D]."""
    batch, heads, sq, d = q.shape
    group, sk = heads // k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    for b in range(batch):
        n = sk if lengths is None else max(0, min(int(lengths[b]), sk))
        first = sk - sq if lengths is None else 0
        last = sq if lengths is None else n
        seen = seen_keys(torch.arange(first, first + last, device=q.device), n, left, right, sinks)
        for h in range(heads):
            out[b, h, :last], bound[b, h, :last] = rows(q[b, h, :last], k[b, h // group, :n], v[b, h // group, :n], seen,
                                                        scale)[:2]
    return out, bound


def rows_grad(q, k, v, g, seen, scale):
    """((dq, dk, dv), (their bounds)) of one head, g [n, d] the gradient of out.

    A weight computed again is off by e - u and by the forward's sum of rounded weights, u: e in all; rounded for
    dV, u more. dP is off by (D + 2) 2^-24 sum |g||v|, delta by the bound of out under |g| and D 2^-24 sum |g||out|;
    dS takes both, the weight's e, its rounding u and (fp16) half a smallest step of its scaled value, 2^-37 of
    2 max|g| max|v|. The products' sums are fp32 (n 2^-24), the results rounded once.
    """
    unit, d = UNIT[q.dtype], q.shape[1]
    out, off, w, e = rows(q, k, v, seen, scale)
    q, k, v, g = q.double(), k.double(), v.double(), g.double()
    dp = g @ v.T
    delta = (g * out).sum(1, keepdim=True)
    ds = w * (dp - delta)
    dp_off = (d + 2) * 2.0 ** -24 * (g.abs() @ v.abs().T)
    delta_off = (g.abs() * (off + d * 2.0 ** -24 * out.abs())).sum(1, keepdim=True)
    ds_off = w * (e * (dp.abs() + delta.abs()) + dp_off + delta_off) + unit * ds.abs()
    if unit == 2.0 ** -11 and seen.numel():
        ds_off = ds_off + seen * (2.0 ** -36 * float(g.norm(dim=1).max()) * float(v.norm(dim=1).max()))
    tiny = 2.0 ** -25 if unit == 2.0 ** -11 else 0.0
    results, bounds = [], []
    for weight, weight_off, x, mul in ((ds, ds_off, k, scale), (ds.T, ds_off.T, q, scale),
                                       (w.T, ((e + unit) * w).T + seen.T * tiny * 2.0 ** -14, g, 1.0)):
        r = mul * (weight @ x)
        b = mul * (weight_off @ x.abs() + x.shape[0] * 2.0 ** -24 * (weight.abs() @ x.abs()))
        results.append(r)
        bounds.append(1.05 * b + unit * 1.05 * r.abs() + tiny + 2.0 ** -60)
    return results, bounds


def gradients(q, k, v, g, left, right, sinks, scale=None, lengths=None):
    """((dq, dk, dv), (bounds)) of the whole tensors; the bound of a shared head is the sum of its heads'."""
    batch, heads, sq, d = q.shape
    group, sk = heads // k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    results = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)]
    bounds = [torch.zeros_like(t) for t in results]
    for b in range(batch):
        n = sk if lengths is None else max(0, min(int(lengths[b]), sk))
        first, last = (sk - sq, sq) if lengths is None else (0, n)
        seen = seen_keys(torch.arange(first, first + last, device=q.device), n, left, right, sinks)
        for h in range(heads):
            r, o = rows_grad(q[b, h, :last], k[b, h // group, :n], v[b, h // group, :n], g[b, h, :last], seen, scale)
            for to, part in ((results, r), (bounds, o)):
                to[0][b, h, :last] = part[0]
                to[1][b, h // group, :n] += part[1]
                to[2][b, h // group, :n] += part[2]
    return results, bounds
