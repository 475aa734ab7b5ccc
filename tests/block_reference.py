"""Plain 64-bit forms of the norm and rotation of queries and keys, the gated projections and the dropout, for the tests that hold the kernels
to them.  Each comes with the size of what its roundings act on, from which the tests' tolerances are made:

  2^-8    half a step of bf16, relative to the value: every output is rounded once
  2^-11   half a step of fp16: what the gated projections keep for the backward pass
  2^-23   an addition or product in float32, or in a tensor core's accumulator (which may cut off instead of rounding)
"""
import math

import numpy as np
import torch

BF, F16, F32 = 2.0 ** -8, 2.0 ** -11, 2.0 ** -23


def heads(x, w, positions, eps, theta, rotary, interleaved, sign=1):
    """(rotated, what it is rounded from: the sum of the magnitudes behind each element); x (..., tokens, heads, dim) double, positions (..., tokens)"""
    x, size = norm(x, w, eps), norm(x, w, eps).abs()
    return rotate(x, positions, theta, rotary, interleaved, sign), rotate(size, positions, theta, rotary, interleaved, sign, True)


def norm(x, w, eps):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w


def rotate(x, positions, theta, rotary, interleaved, sign=1, sizes=False):
    """sizes: the sum of the two elements of a pair in place of either"""
    i = torch.arange(rotary // 2, device=x.device, dtype=torch.float64)
    angle = sign * positions.double()[..., None, None] * theta ** (-2 * i / max(rotary, 1))
    c, s = torch.cos(angle), torch.sin(angle)
    part, rest = x[..., :rotary], x[..., rotary:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :rotary // 2], part[..., rotary // 2:])
    u, v = (a + b, a + b) if sizes else (a * c - b * s, a * s + b * c)
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((turned, rest), -1)


def heads_bwd(x, w, g, positions, eps, theta, rotary, interleaved):
    """(dx, its size, dw, its size), the last two None without a scale"""
    size = rotate(g.abs(), positions, theta, rotary, interleaved, -1, True)
    g = rotate(g, positions, theta, rotary, interleaved, -1)
    if w is None:
        return g, size, None, None
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    n, a, m = x * r, g * w, size * w.abs()
    dx = r * (a - n * (a * n).mean(-1, keepdim=True))
    axes = tuple(range(x.dim() - 1))
    return dx, r * (m + n.abs() * (m * n.abs()).mean(-1, keepdim=True)), (g * n).sum(axes), (size * n.abs()).sum(axes)


def act(g, name):
    """(act, its derivative)"""
    if name == "relu":
        return g.clamp_min(0), (g > 0).double()
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    phi = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def gated(x, wg, wu, name):
    """(h, how far it may be off)"""
    g, u = x @ wg, x @ wu
    dg, du = x.shape[1] * F32 * (x.abs() @ wg.abs()), x.shape[1] * F32 * (x.abs() @ wu.abs())
    a, _ = act(g, name)
    h = a * u
    # every one of the three has a slope of at most 1.13; 2^-20 for the functions that it is made of, of |g| and not of act(g): the error of exp(v) is one of v
    return h, BF * h.abs() + (1.2 * dg + 2.0 ** -20 * g.abs()) * (u.abs() + du) + a.abs() * du + 1e-38


def gated_bwd(x, wg, wu, name, grad, pieces=1):
    """[(dx, how far it may be off), ...] for x and both weights; pieces: of bf16 that the gradients at the projections are the sum of"""
    k, (m, f) = x.shape[1], grad.shape
    g, u = x @ wg, x @ wu
    # what the projections are when the backward pass sees them: accumulated, then in fp16 (2^-24: its smallest steps)
    eg, eu = (k * F32 * (x.abs() @ w.abs()) + F16 * v.abs() + 2.0 ** -24 for w, v in ((wg, g), (wu, u)))
    a, da = act(g, name)
    bend = (g.abs() <= eg).double() if name == "relu" else 0.8 * eg + 2.0 ** -20 * (1 + g.abs())       # of the derivative
    dg, du = grad * u * da, grad * a
    r = BF ** pieces                            # (the second is of what the first left, at most BF of it)
    err_g = r * dg.abs() + grad.abs() * (bend * (u.abs() + eu) + 1.2 * eu)
    err_u = r * du.abs() + grad.abs() * (1.2 * eg + 2.0 ** -20 * g.abs())

    def total(value, parts, n):
        """`value` of products a @ b whose second factor may be off by e, n terms in all"""
        return value, 1.01 * BF * value.abs() + sum(1.01 * (p.abs() @ e) + pieces * n * F32 * (p.abs() @ q.abs()) for p, q, e in parts) + 1e-38

    dx = (dg @ wg.T + du @ wu.T).T
    dx, e = total(dx, [(wg, dg.T, err_g.T), (wu, du.T, err_u.T)], 2 * f)
    return [(dx.T, e.T), total(x.T @ dg, [(x.T, dg, err_g)], m), total(x.T @ du, [(x.T, du, err_u)], m)]


def philox(counter, key):
    """Philox4x32 with ten rounds; counter (n, 4) and key (2,) of 32-bit words"""
    c = [np.asarray(v, dtype=np.uint64) for v in np.asarray(counter).T]
    k = [int(v) for v in key]
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, -1).astype(np.uint32)


def kept(n, p, seed, site, first=0):
    """the mask of elements first .. first + n, and the factor"""
    lo, hi = first // 8, (first + n + 7) // 8
    i = np.arange(lo, hi, dtype=np.uint64)
    counter = np.stack((i & np.uint64(0xFFFFFFFF), i >> np.uint64(32), np.full_like(i, site), np.zeros_like(i)), -1)
    words = philox(counter, (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    bits = np.stack((words & np.uint32(0xFFFF), words >> np.uint32(16)), -1).reshape(-1)[first - 8 * lo:][:n]
    t = round(p * 65536)
    return bits >= t, 65536 / (65536 - t) if t < 65536 else 0.0
