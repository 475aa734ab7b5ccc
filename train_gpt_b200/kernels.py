"""RMSNorm: the call surface of train-gpt's `kernels.py` on B200 kernels.

`rms_norm(x, scale, eps)` is the fused single-rounding norm (kernels.py:44-53 with the
variance pass of :66 folded in) with the recompute backward of kernels.py:104-118;
`_rms_norm_pure(x, scale, eps)` is the three-rounding form (kernels.py:30-33).  Both are
positional-only in the reference's order; `eps` is static (not differentiated).
`rms_norm_quant` is the fused norm + 1x128 e4m3 quantise the FP8 linear layers consume.

`sandwich_norm` and `sandwich_norm_quant` have no counterpart there: the junction between two blocks that have a norm on
both sides, with the block's gate and the scaled residual add between the norms.
"""
from __future__ import annotations

import torch

from . import ops


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
