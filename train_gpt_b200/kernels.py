"""RMSNorm: the call surface of train-gpt's `kernels.py` on B200 kernels.

`rms_norm(x, scale, eps)` is the fused single-rounding norm (kernels.py:44-53 with the
variance pass of :66 folded in) with the recompute backward of kernels.py:104-118;
`_rms_norm_pure(x, scale, eps)` is the three-rounding form (kernels.py:30-33).  Both are
positional-only in the reference's order; `eps` is static (not differentiated).
`rms_norm_quant` is the fused norm + 1x128 e4m3 quantise the FP8 linear layers consume.

`sandwich_norm` and `sandwich_norm_quant` have no counterpart there: the junction between two blocks that have a norm on
both sides, with the block's gate and the scaled residual add between the norms.  Nor have `qk_norm_rope` (a norm per head of
queries and keys with the rotation by position), `gated_linear` (the gated feed-forward's two projections, its activation and the
product) and `dropout` (from a counter-based generator, with the residual add behind it).
"""
from __future__ import annotations

import torch

from . import _lib, ops


def rms_norm(x: torch.Tensor, scale: torch.Tensor, eps: float) -> torch.Tensor:
    return ops._host().rms_norm(x, scale, eps, False)


def _rms_norm_pure(x: torch.Tensor, scale: torch.Tensor, eps: float) -> torch.Tensor:
    return ops._host().rms_norm(x, scale, eps, True)


class NormedQuantized:
    """Output of `rms_norm_quant`: the norm's bf16 result in quantised form (q, scales),
    usable as `a_quantized=` of `fp8.block_scaled_matmul` by every GEMM that consumes the
    same normed activation, plus the bf16 tensor itself when it was asked for."""

    __slots__ = ("q", "scales", "y")

    def __init__(self, q, scales, y):
        self.q, self.scales, self.y = q, scales, y

    def as_pair(self):
        return self.q, self.scales


def rms_norm_quant(x, scale, eps: float, pure: bool = False, want_y: bool = False) -> NormedQuantized:
    """model.py:76-77 `_norm(...)` followed by the quantiser of fp8.py:66, one kernel.
    Forward only (no autograd); training code pairs it with `rms_norm`'s backward."""
    q, s, y, _ = ops._host().rmsnorm_quant_fwd(x, scale, eps, pure, want_y, False)
    return NormedQuantized(q, s, y)


def sandwich_norm(x, branch, post_scale, scale, eps: float, gate=None, residual_scale: float = 1.0, quantize: bool = False):
    """The junction behind a block whose output is `branch`, x being the residual stream:

        x_new = bf16(residual_scale * x + G * rms(branch) * post_scale),   h = bf16(rms(x_new) * scale)

    with rms(v) = v * rsqrt(mean(v^2) + eps), float32 between the two roundings (h is the norm of x_new as it is kept).
    x, branch (..., D) bf16, D a multiple of 8 up to 8192; post_scale, scale (D,) bf16; gate None (G = 1), (D,) bf16 for one
    per channel, or (..., 1) bf16 for one per token; residual_scale and eps are static.

    Returns (x_new, h), or with quantize=True (D a multiple of 128) (x_new, h, q, scales), q and scales the 1x128 e4m3 form
    of h that `fp8.block_scaled_matmul` takes as `a_quantized`; they carry no gradient, h does.  Differentiable once, in reverse mode, in x,
    branch, both scales and the gate; the backward pass keeps x_new and branch and computes the factors again.  32768 x 2048
    forward and backward is one kernel each way and a small one for the scales' gradients."""
    return ops._host().sandwich_norm(x, branch, post_scale, scale, eps, gate, residual_scale, quantize)


def sandwich_norm_quant(x, branch, post_scale, scale, eps: float, gate=None, residual_scale: float = 1.0, want_y: bool = False):
    """`sandwich_norm` for inference: (x_new, NormedQuantized of h), h itself written only if it is asked for.
    Forward only (no autograd)."""
    x_new, h, q, s = ops._host().sandwich_norm_fwd(x, branch, post_scale, scale, eps, gate, residual_scale, want_y, True)
    return x_new, NormedQuantized(q, s, h)


def qk_norm_rope(q, k, q_scale, k_scale, eps: float, positions=None, *, theta: float = 10000.0, rotary_dim: int | None = None,
                 interleaved: bool = False):
    """Queries and keys of an attention, each head normed and rotated by its token's position, in one pass over both:

        y = R(t) (x * rsqrt(mean(x^2) + eps) * scale)        over a head's dim elements, float32 with one rounding

    q (..., H, D), k (..., K, D) bf16 with the same leading axes, any strides (column slices of one projection and transposed tensors are
    read as they lie where heads begin at 16-byte boundaries with unit stride along D); D a multiple of 16 up to 512.  q_scale, k_scale
    (D,) bf16, or both None for the rotation without a norm.  R(t) turns the pair (i, i + rotary_dim / 2), or (2 i, 2 i + 1) with `interleaved`,
    by t * theta^(-2 i / rotary_dim), theta from 1e-30 to 1e30; rotary_dim (default D, a multiple of 16, 0 for none) is the part of a head that is rotated.
    positions int32 or int64, expandable to the leading axes: a token's t, |t| < 2^31; None: its place along the last of them.

    Returns (q', k'), contiguous.  Differentiable once, in reverse mode, in q, k and the scales; the backward pass keeps q and k
    (with scales) and the positions, and works out norms and angles again."""
    return ops._host().qk_norm_rope(q, k, q_scale, k_scale, eps, positions, theta, -1 if rotary_dim is None else ops.rotary_dim_of(rotary_dim), interleaved)


def gated_linear(x, w_gate, w_up, activation: str = "silu"):
    """act(x w_gate) * (x w_up), the first half of a gated feed-forward, as one kernel: both projections, the activation and the
    product, float32 between the bf16 inputs and the one rounding.

    x (..., D), w_gate and w_up (D, F) bf16, D and F multiples of 8; rows of any pitch (the weights may be column slices of one matrix).
    activation "silu", "gelu" (by erf) or "relu".  Returns (..., F) bf16.

    Differentiable once, in reverse mode.  With gradients on, both projections are kept in 16 bits (fp16 with a power of two per 64 columns
    of a row) for the backward pass: 11 bits of a value, fewer where it is below 2^-28 of the largest of its 64, nothing below 2^-40 of it.  The
    backward pass rounds the gradients at them to bf16 (to the sum of two in small problems) and makes dx and both weight gradients in one launch."""
    if activation not in _lib.TG_GATED:
        raise ValueError(f"unknown activation {activation!r}; use one of {sorted(_lib.TG_GATED)}")
    return ops._host().gated_linear(x, w_gate, w_up, _lib.TG_GATED[activation])


def dropout(x, p: float, seed: torch.Tensor, site: int = 0, residual=None):
    """bf16(residual + keep * x / (1 - p)) with a mask that is never stored: element e is kept where the 16 random bits that Philox4x32-10
    gives for (seed, site, e) are at least round(65536 p), and the factor is that of the rounded p.

    x bf16 of any shape, residual None or like x; 0 <= p <= 1 (0 keeps everything); seed an int64 CUDA tensor of one element, so that a captured graph
    draws new masks when it changes; site an integer in [0, 2^32), another one for every place of a model that drops out.  The mask depends on
    an element's place in the contiguous order of x alone.  Differentiable once, in reverse mode, in x and residual: the backward
    pass draws the mask again, so the seed must not change before it (an error; a graph of one's own whose replay changes it is not noticed:
    torch.autograd.graph.increment_version(seed) behind the replay makes it one)."""
    return ops._host().dropout(x, p, seed, site, residual)
