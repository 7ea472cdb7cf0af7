"""Root-mean-square norm on the sm_100a kernels, with the residual's addition and an
8-bit output.

    h = x + residual               rounded to x's dtype: the new residual stream
    y = h * rsqrt(mean(h^2) + eps) * weight

over the last dimension of x [..., dim], dim up to 16384, in bfloat16, float16 or
float32; weight [dim] has x's dtype or is float32. Sums are float32. The norm reads
the rounded h, the stream that a model passes on. x and residual may be strided;
outputs are contiguous.
"""
from __future__ import annotations

from typing import Optional

import torch

from .._ext import C


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6):
    """y, or (y, h) with a residual; differentiable (once, in reverse mode) in x, weight and
    residual."""
    y, h = C().rms_norm(x, weight, residual, eps)
    return y if h is None else (y, h)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                 eps: float = 1e-6, group: int = 0):
    """The norm's output in 8 bits: (y8, scale), or (y8, scale, h) with a residual.

    y8 (float8_e4m3fn, x's shape) times scale (float32 [..., dim / group]) stands for y.
    scale is the largest |y| of its `group` columns (16, 32, 64 or 128, dividing dim) or,
    with group 0, of its row, over 448, the largest e4m3 value; 1 where all are zero or
    one is NaN. Not differentiable: for inference."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (residual is not None and residual.requires_grad)):
        raise RuntimeError("rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    y8, scale, h = C().rms_norm_fp8(x, weight, residual, eps, group)
    return (y8, scale) if h is None else (y8, scale, h)
