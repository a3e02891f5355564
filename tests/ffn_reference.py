"""The gated feed-forward projection, its gradients and 4-bit weights from their definitions, in 64 bits, with the bounds
that 32-bit sums and one rounding to 16 bits allow."""
import math

import torch

import inputs

ACTIVATIONS = ("silu", "gelu", "gelu_tanh")
DTYPES = (torch.bfloat16, torch.float16)


def half_step(dtype) -> float:
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def act_and_slope(g, act):
    """act(g) = g P(g) and its derivative P(g) + g P'(g), both tails without cancellation."""
    if act == "silu":
        p = torch.sigmoid(g)
        return g * p, p + g * p * torch.sigmoid(-g)
    if act == "gelu":
        p = 0.5 * torch.erfc(-g / math.sqrt(2.0))
        return g * p, p + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    c = 2 * math.sqrt(2 / math.pi)
    z = c * (g + 0.044715 * g ** 3)
    p = torch.sigmoid(z)
    return g * p, p + g * p * torch.sigmoid(-z) * c * (1 + 3 * 0.044715 * g * g)


def sum_error(n: int) -> float:
    """Relative to the sum of the terms' magnitudes: n terms added in fp32, each addition off by at most one unit in
    the last place (the tensor cores may truncate where the adders round)."""
    return n * 2.0 ** -23


def gated(x, w, act):
    """(h, bound of |kernel - h|, g, u) for x [T, K] and w [2I, K]."""
    dtype = x.dtype
    x, w = x.double(), w.double()
    inter, k = w.shape[0] // 2, x.shape[1]
    p = x @ w.t()
    mag = (x.abs() @ w.abs().t()) * sum_error(k)
    g, u = p[:, :inter], p[:, inter:]
    a, _ = act_and_slope(g, act)
    h = a * u
    # slopes are below 1.13 in magnitude; 1e-5 for the exponential and the division of the activation
    bound = (half_step(dtype) + 1e-5) * h.abs() + 1.13 * mag[:, :inter] * u.abs() + a.abs() * mag[:, inter:]
    return h, bound + 2 * mag[:, :inter] * mag[:, inter:] + torch.finfo(dtype).smallest_normal * half_step(dtype), g, u


def gated_backward(x, w, act, dh):
    """(dx, its bound, dw, its bound): every gradient of a projection is rounded once to the 16-bit type (half a step of
    it, plus 2^-14 for g and u in 24 bits and for the activation's slope) and enters sums of n terms."""
    dtype = x.dtype
    x, w, dh = x.double(), w.double(), dh.double()
    inter, k, t = w.shape[0] // 2, x.shape[1], x.shape[0]
    p = x @ w.t()
    mag = (x.abs() @ w.abs().t()) * sum_error(k)
    g, u = p[:, :inter], p[:, inter:]
    a, s = act_and_slope(g, act)
    he = half_step(dtype)
    tiny = torch.finfo(dtype).smallest_normal * he
    d = torch.cat((dh * u * s, dh * a), 1)
    # second derivatives are below 0.8 in magnitude
    off = torch.cat((dh.abs() * (1.13 * mag[:, inter:] + 0.8 * u.abs() * mag[:, :inter]), dh.abs() * 1.13 * mag[:, :inter]), 1)
    off = off + (he + 2.0 ** -14) * torch.cat((dh.abs() * u.abs() * 1.13, dh.abs() * a.abs()), 1) + tiny
    dx, dw = d @ w, d.t() @ x
    bx = he * dx.abs() + off @ w.abs() + sum_error(2 * inter) * ((d.abs() + off) @ w.abs()) + tiny
    bw = he * dw.abs() + off.t() @ x.abs() + sum_error(t) * ((d.abs() + off).t() @ x.abs()) + tiny
    return dx, bx, dw, bw


def unpack(codes):
    return torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)


def dequantize(codes, scale, zero):
    """W in 64 bits."""
    q = unpack(codes).double().view(*scale.shape, -1)
    z = 8.0 if zero is None else zero.double()[..., None]
    return ((q - z) * scale.double()[..., None]).flatten(1)


def inside(got, want, bound, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(off[bad].max()), float(bound[bad].min()))


def rows(t, k, seed, dtype, std=1.0):
    return (std * torch.randn(t, k, generator=inputs.gen(seed))).to(dtype)


def random_int4(n, k, group, seed, zero=True, scale_dtype=torch.bfloat16):
    """(codes, scale, zero) with every code, steps spread over a factor of 16 and zero points over their whole range."""
    gen = inputs.gen(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=gen, dtype=torch.uint8)
    scale = (torch.exp2(-8 + 4 * torch.rand(n, k // group, generator=gen))).to(scale_dtype)
    return codes, scale, torch.randint(0, 16, (n, k // group), generator=gen, dtype=torch.uint8) if zero else None
