"""Plain statements in 64 bits of the products with 4-bit weights and of rotary positions, with what an output may be off
by, for the tests of ``b200t2w.w4`` and ``b200t2w.rotary``."""

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # steps of subnormal numbers


def weights(n, k, group, zeros, scale_dtype, gen, device="cpu"):
    """Random codes over all 16 values, scales over three powers of two, zeros over all 16 values."""
    codes = torch.randint(0, 16, (n, k), generator=gen, dtype=torch.uint8)
    scales = (torch.exp2(torch.rand(n, k // group, generator=gen) * 3 - 1) * k ** -0.5 / 4).to(scale_dtype)
    z = torch.randint(0, 16, (n, k // group), generator=gen, dtype=torch.uint8) if zeros else None
    return tuple(None if x is None else x.to(device) for x in (codes, scales, z))


def dense(w):
    """(code - zero) * scale in 64 bits."""
    codes, scales, zeros = w
    n, k = codes.shape
    c = codes.double().view(n, scales.shape[1], -1) - (8 if zeros is None else zeros.double().unsqueeze(2))
    return (c * scales.double().unsqueeze(2)).view(n, k)


def product(x, w):
    """y = x W^T and the sum of magnitudes B = |x| |W|^T."""
    d, x = dense(w), x.double()
    return x @ d.T, x.abs() @ d.abs().T


def sum_error(k, b):
    """What fp32 sums of k products with magnitudes adding up to b may be off by.

    Products are exact (8 or 11 bits by 5).  A step of a tensor-core product adds 16 of them and the running sum of its group,
    each cut to 24 bits of the largest: 17 * 2^-23 of what has been added so far, which over a group's at most 8 steps (and
    their magnitudes b_g) is at most 17 * 2^-23 * b_g for every step: 8 * 17 * 2^-23 < 2^-15.  Most of that is never there: cut terms
    are of either sign; but it is the bound.  The groups' sums are scaled and added in fp32: at most k / 32 + 16
    roundings of 2^-24 of b, the last ones being joins of parts."""
    return (2.0 ** -15 + (k / 32 + 16) * 2.0 ** -24) * b


def rounded(y, error, dtype):
    """The error and half a step of the rounded value (which may be off by the error itself)."""
    return error + HALF_STEP[dtype] * (y.abs() + error) + TINY[dtype]


def linear(x, w, bias=None, residual=None):
    """The value, and how far from it an output may be."""
    y, b = product(x, w)
    e = sum_error(x.shape[1], b)
    for extra in (bias, residual):
        if extra is not None:
            y = y + extra.double()
            e = e + 2.0 ** -24 * (y.abs() + e)  # one fp32 addition
    return y, rounded(y, e, x.dtype)


def gated(x, gate, up, act):
    """act(g) u and how far an output may be from it.  SiLU and GELU have slopes of at most 1.13; their fp32 forms (an
    exponential with an error of 2 + 1.2 |s| steps of 2^-23, s its argument, a quotient, products) are off by at most
    (8 + 1.2 |s|) 2^-23 of the value, |s| <= 1.6 (|g| + 0.045 |g|^3) for GELU."""
    (g, bg), (u, bu) = product(x, gate), product(x, up)
    eg, eu = sum_error(x.shape[1], bg), sum_error(x.shape[1], bu)
    if act == "silu":
        s = g
    else:
        s = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    a = g * torch.sigmoid(s)
    ea = 1.13 * eg + (8 + 1.2 * s.abs().clamp(max=200)) * 2.0 ** -23 * a.abs()
    e = ea * u.abs() + (a.abs() + ea) * eu + 2.0 ** -24 * (a * u).abs()
    return a * u, rounded(a * u, e, x.dtype)


def turned(x, positions, axis, inv_freq, rotary_dim, adjacent, inverse):
    """x [rows, heads, head_dim] turned, in 64 bits; positions [axes, rows], axis and inv_freq for each pair."""
    angle = positions.double()[axis] * inv_freq[:, None]  # [pairs, rows]
    if inverse:
        angle = -angle
    cos, sin = torch.cos(angle).T[:, None], torch.sin(angle).T[:, None]
    y, d = x.double().clone(), rotary_dim
    if adjacent:
        a, b = y[..., 0:d:2].clone(), y[..., 1:d:2].clone()
        y[..., 0:d:2], y[..., 1:d:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = y[..., :d // 2].clone(), y[..., d // 2:d].clone()
        y[..., :d // 2], y[..., d // 2:d] = a * cos - b * sin, b * cos + a * sin
    return y
