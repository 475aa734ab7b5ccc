"""The angles of kernels.qk_norm_rope at far positions, by pairs whose rotation all but cancels: y = a cos - b sin with (a, b) along (sin, cos) is what the angle
is off by, times the pair's length."""
import math
from fractions import Fraction

import pytest
import torch

from train_gpt_b200 import kernels

N, DIGITS = 512, 160                # positions, bits behind the point of a turn

pytestmark = pytest.mark.gpu


def _pi():
    """pi 2^DIGITS, by Machin's formula"""
    def arctan_of_one_over(n):
        total, term, k = 0, (1 << (DIGITS + 20)) // n, 1
        while term:
            total += term // k if k % 4 == 1 else -(term // k)
            term //= n * n
            k += 2
        return total
    return (4 * (4 * arctan_of_one_over(5) - arctan_of_one_over(239))) >> 20


def _turns(theta, rotary):
    """theta^(-2 i / rotary) / 2 pi times 2^DIGITS for i < rotary / 2, by square roots of integers (rotary / 2 is a power of two)"""
    one = 1 << DIGITS
    step = one // theta
    for _ in range(int(math.log2(rotary // 2))):
        step = math.isqrt(step << DIGITS)
    out, t = [], (one * one) // (2 * _pi())
    for _ in range(rotary // 2):
        out.append(t)
        t = (t * step) >> DIGITS
    return out


def _cancelling(theta, rotary, positions):
    """(x, cos, sin): pairs (i, i + rotary / 2) in bf16 for which x_i cos - x_j sin is near 0, and the exact cosines and sines as doubles"""
    one = 1 << DIGITS
    fraction = torch.tensor([[float(Fraction((p * t) % one, one)) for t in _turns(theta, rotary)] for p in positions], dtype=torch.float64)
    c, s = torch.cos(2 * math.pi * fraction), torch.sin(2 * math.pi * fraction)
    best = None
    for length in torch.linspace(1, 2, 64, dtype=torch.float64).tolist():
        a, b = ((length * v).to(torch.bfloat16).double() for v in (s, c))
        left = (a * c - b * s).abs()
        if best is None:
            best = [left, a, b]
        else:
            better = left < best[0]
            best = [torch.where(better, n, o) for n, o in zip((left, a, b), best)]
    return torch.cat(best[1:], -1), c, s


@pytest.mark.parametrize("theta,rotary", [(300, 512), (2, 256), (10000, 128), (500000, 64)])
def test_far_angles(theta, rotary):
    gen = torch.Generator().manual_seed(rotary)
    positions = (2 ** 31 - 1 - torch.randint(0, 2 ** 22, (N,), generator=gen)).tolist()
    x, c, s = _cancelling(theta, rotary, positions)
    q = x.to(torch.bfloat16).cuda().view(1, N, 1, rotary)
    got, _ = kernels.qk_norm_rope(q, q, None, None, 0.0, torch.tensor(positions, device="cuda"), theta=float(theta))
    y = got.double().cpu().view(N, rotary)[:, :rotary // 2]
    a, b = x[:, :rotary // 2], x[:, rotary // 2:]
    off = (a * c - b * s - y) / (a * s + b * c)                                     # of the angle
    angle = 2.0 ** 31 * theta ** (-2 * torch.arange(rotary // 2, dtype=torch.float64) / rotary)
    # Two roundings of 2^-53 to the turn, float32's of it (2^-23), of sine and cosine (2 ulp) and of two products (2^-22 in all, the pair's length being 1
    # to 2), bf16's of what is left (2^-8 of it).
    assert (off.abs() <= angle * 2.0 ** -52 + 2.0 ** -23 + 2.0 ** -21 + 2.0 ** -8 * y.abs()).all()
    # All positions are about 2^31, so that an error of the table is the same in all; the other roundings differ from one to the next, and their mean is a twentieth.
    mean = off.mean(0).abs()
    assert (mean <= angle * 2.0 ** -53 * 1.1 + 2.0 ** -24).all(), float((mean / (angle * 2.0 ** -53 + 2.0 ** -24)).max())
