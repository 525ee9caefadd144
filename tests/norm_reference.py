"""Layer norm, its gradients, row quantization and the 8-bit product from their definitions in 64 bits, with bounds on
what fp32 arithmetic and one rounding may leave between them and the kernels."""
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALLEST = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}  # half the least fp16 step
U = 2.0 ** -24
# A sum over a row adds at most 32 values in turn in a lane, then 6 steps over lanes and 7 over wavefronts; with the
# product by 1 / C and the operation that uses it, fewer than 48 roundings.
ROW = 48


def broadcast(t, x):
    """A weight [C] or [B, C] against rows x [B, ..., C]."""
    return t.double() if t.dim() == 1 else t.double().reshape(t.shape[0], *[1] * (x.dim() - 2), t.shape[1])


class Norm:
    def __init__(self, x, weight, bias, eps, around_one):
        self.x, self.x_type = x.double(), x.dtype
        self.factor = torch.ones((), dtype=torch.float64, device=x.device) if weight is None else \
            broadcast(weight, x) + float(around_one)
        plus = torch.zeros((), dtype=torch.float64, device=x.device) if bias is None else broadcast(bias, x)
        self.mean = self.x.mean(-1, keepdim=True)
        self.inverse = ((self.x - self.mean).square().mean(-1, keepdim=True) + eps).rsqrt()
        self.n = (self.x - self.mean) * self.inverse
        self.out = self.n * self.factor + plus
        # The deviations are taken from a mean that is off by `shift` and their own mean, which is good to ROW U of
        # their size; the sum of squares less that square is good to ROW U of either.
        shift = ROW * U * self.x.abs().mean(-1, keepdim=True)
        wide = (self.x - self.mean).abs().mean(-1, keepdim=True) + shift
        self.n_off = ROW * U * (self.inverse * wide + self.n.abs() * (2 + (shift * self.inverse).square()))
        self.out_off = self.n_off * self.factor.abs() + 3 * U * ((self.n * self.factor).abs() + plus.abs())

    def out_bound(self):
        return HALF_STEP[self.x_type] * 1.01 * self.out.abs() + self.out_off + SMALLEST[self.x_type]

    def gradients(self, grad, per_entry):
        """(dx, dw, db) and their bounds, dw and db without their rounding to a type."""
        d = grad.double()
        g = d * self.factor
        s1, s2 = g.mean(-1, keepdim=True), (g * self.n).mean(-1, keepdim=True)
        dx = self.inverse * (g - s1 - self.n * s2)
        size1 = g.abs().mean(-1, keepdim=True)
        s2_off = 2 * ROW * U * (g * self.n).abs().mean(-1, keepdim=True) + (g.abs() * self.n_off).mean(-1, keepdim=True)
        off = self.inverse * (ROW * U * (size1 + g.abs() + (self.n * s2).abs()) + self.n.abs() * s2_off +
                              self.n_off * s2.abs())
        bound = HALF_STEP[self.x_type] * 1.01 * dx.abs() + off + SMALLEST[self.x_type]
        over = tuple(range(1 if per_entry else 0, d.dim() - 1))

        def add(t):  # (torch's sum over no axes is one over all)
            return t.sum(over) if over else t

        rows = d[..., 0].numel() // (d.shape[0] if per_entry else 1)
        # A column's sum: at least 256 sets of lanes take rows in turn where there are as many, then up to 8 sets of a
        # workgroup and 512 workgroups (32 in turn, 16 wavefronts) are joined.
        chain = rows // 256 + 1 + 8 + 4 + 32 + 16
        dw, db = add(d * self.n), add(d)
        dw_off = add((chain + 2) * U * (d * self.n).abs() + d.abs() * self.n_off)
        return (dx, bound), (dw, dw_off), (db, chain * U * add(d.abs()))


def quantized(x):
    """(codes, scales) of rows x in fp32 arithmetic on the CPU, for rows that are finite."""
    x = x.float().cpu()
    most = x.abs().amax(-1, keepdim=True)
    kept = most >= 127 * 2.0 ** -126
    one, steps = torch.tensor(1.0), torch.tensor(127.0)
    by = torch.where(kept, steps * (one / most), torch.zeros(()))
    return (x * by).round().to(torch.int8), torch.where(kept, most * (one / steps), torch.zeros(()))[..., 0]


def product(codes, scales, weight, weight_scales, bias, dtype):
    """The product's definition, and a bound: conversion, two scales and the bias are 4 operations in fp32."""
    # (Sums below 2^53 are exact in 64-bit floating point.)
    out = torch.matmul(codes.double(), weight.double().T.contiguous()) * scales.double()[..., None] * weight_scales.double()
    size = out.abs()
    if bias is not None:
        out, size = out + bias.double(), size + bias.double().abs()
    return out, HALF_STEP[dtype] * 1.01 * out.abs() + 4 * U * size + SMALLEST[dtype]
