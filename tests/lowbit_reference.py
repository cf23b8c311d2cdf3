"""Plain 64-bit implementations of the low-bit operators on the CPU, for their tests."""
from __future__ import annotations

import torch

F64 = torch.float64
TOP = {torch.int8: 127, torch.float8_e4m3fn: 448}
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half a step, relative to the value


def f32(t: torch.Tensor) -> torch.Tensor:
    """Rounded to 32 bits, held in 64."""
    return t.to(torch.float32).to(F64)


def half_even(t: torch.Tensor) -> torch.Tensor:
    return torch.round(t)


def e4m3(t: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 number, ties to even: numbers up to 2^-6 lie 2^-9 apart, above 1/8 of their power of two."""
    e = torch.frexp(t.abs())[1] - 1
    step = torch.ldexp(torch.ones_like(t), torch.clamp_min(e, -6) - 3)
    return (half_even(t / step) * step).clamp(-448, 448)


def norm(x, residual, weight, eps, dtype):
    """(codes as numbers, scales, hidden, inv_rms) in 64 bits; the roundings of the definition are kept."""
    h = x.to(F64) if residual is None else f32(x.to(F64) + residual.to(F64)).to(x.dtype).to(F64)
    z = f32(h * weight.to(F64))
    a = z.abs().amax(-1)
    s = f32(a / TOP[dtype])
    t = z / torch.where(s > 0, s, torch.ones_like(s)).unsqueeze(-1)
    t = torch.where((s > 0).unsqueeze(-1), t, torch.zeros_like(t))
    codes = half_even(t).clamp(-127, 127) if dtype == torch.int8 else e4m3(t)
    inv = 1 / torch.sqrt((h * h).mean(-1) + eps)
    return codes, s * inv, h, inv


def norm_backward(grad, hidden, weight, inv_rms, grad_hidden=None):
    """(grad_x, grad_weight, bound of grad_x's error in 32-bit arithmetic, the same for grad_weight), before the last rounding."""
    g, h, w, inv = grad.to(F64), hidden.to(F64), weight.to(F64), inv_rms.to(F64).unsqueeze(-1)
    n, u = h * inv, g * w
    c = (u * n).mean(-1, keepdim=True)
    dx = inv * (u - n * c)
    if grad_hidden is not None:
        dx = dx + grad_hidden.to(F64)
    dims = tuple(range(g.dim() - 1))
    dw = (g * n).sum(dims)
    eps = 2.0 ** -24
    # u and n carry one rounding each, their products and the outer ones a few more; the mean is a tree of lane sums of at
    # most 24 terms (16 registers, or a stretch of 8 per visit), then at most 6 + 16 joining additions
    mean_abs = (u * n).abs().mean(-1, keepdim=True)
    visits = 24 + h.shape[-1] // 1024
    bound_x = eps * (inv * (5 * u.abs() + n.abs() * (visits + 30) * mean_abs) + 2 * dx.abs())
    rows = max(1, g.numel() // max(1, g.shape[-1]))
    bound_w = eps * (rows + 4) * (g * n).abs().sum(dims)
    return dx, dw, bound_x, bound_w


def quantize_4bit(weight, group, scale_dtype):
    """(codes [n, groups * group] as whole numbers, scales)."""
    n, k = weight.shape
    groups = -(-k // group)
    w = torch.zeros(n, groups * group, dtype=F64)
    w[:, :k] = weight.to(F64)
    w = w.view(n, groups, group)
    s = (w.abs().amax(-1) / 7).to(torch.float32).to(scale_dtype)
    s64 = s.to(F64).unsqueeze(-1)
    t = torch.where(s64 > 0, w / torch.where(s64 > 0, s64, torch.ones_like(s64)), torch.zeros_like(w))
    return half_even(t).clamp(-7, 7).view(n, groups * group).to(torch.int8), s


def pack(codes):
    """Whole numbers -8 .. 7 [n, even] to bytes, the even element in the lower half."""
    c = codes.to(torch.int16) & 15
    return (c[:, 0::2] | (c[:, 1::2] << 4)).to(torch.uint8)


def unpack(packed):
    p = packed.to(torch.int16)
    both = torch.stack((p & 15, p >> 4), -1).view(p.shape[0], -1)
    return (both - 16 * (both >= 8).to(torch.int16)).to(torch.int8)


def matvec(x, x_scales, codes, scales, k):
    """(products, bound of their error in 32-bit sums), before the last rounding."""
    group = codes.shape[1] // scales.shape[1]
    rows = x.reshape(-1, k).to(F64)
    q, s = codes[:, :k].to(F64), scales.to(F64).repeat_interleave(group, 1)[:, :k]
    y = rows @ (q * s).T
    eps = 2.0 ** -24
    if x_scales is None:
        # any order of summation, the weights as integers of up to 31 beside an offset of up to 24 that is taken off again
        bound = eps * (k + 8) * (rows.abs() @ (55 * s.abs()).T)
    else:
        # sums within a group are whole numbers below 2^24; the groups' terms are added in some order, after three roundings
        parts = torch.stack([(rows[:, a:a + group] @ (q * s)[:, a:a + group].T).abs() for a in range(0, k, group)]).sum(0)
        xs = x_scales.reshape(-1, 1).to(F64)
        y, bound = y * xs, eps * (scales.shape[1] + 4) * parts * xs.abs()
    lead = x.shape[:-1]
    return y.view(*lead, codes.shape[0]), bound.view(*lead, codes.shape[0])


def outside(got, want, bound):
    """The largest excess of |got - want| over half a step of got's type and the bound; at most 0 when all is well."""
    d = (got.to(F64) - want).abs()
    # the rounded value is compared, so the step is taken where the bound could carry it; 2^-150: fp32's smallest half step
    small = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[got.dtype]
    return float((d - (STEP[got.dtype] * (want.abs() + bound) + bound + small)).max()) if d.numel() else 0.0


def matvec_bound(x, codes, scales, k):
    """Bound of the error of products of floating rows, from the roundings that 32-bit sums of the terms themselves make: relative to
    sum |code x scale|, so that a column whose code is 0 counts for nothing.  Products with a code are exact (fp32 rows as three
    parts, so three products).  Within a group each addition is off by at most a whole step (twice half of one, should the matrix
    unit cut off what it does not hold); a group's scaling and each addition of groups, wavefronts and visits by half a step."""
    group = codes.shape[1] // scales.shape[1]
    parts = 3 if x.dtype == torch.float32 else 1
    terms = x.reshape(-1, k).to(F64).abs() @ (codes[:, :k].to(F64) * scales.to(F64).repeat_interleave(group, 1)[:, :k]).abs().T
    bound = 2.0 ** -24 * (2 * parts * group + scales.shape[1] + 24) * terms
    return bound.view(*x.shape[:-1], codes.shape[0])
