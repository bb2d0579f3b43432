"""Root-mean-square norm in front of the expert layer: the residual's addition fused in, a backward pass, and an output in
8 bits for `momoe.fp8` experts.

    r = x + residual (rounded to the stream's type),   y = r / sqrt(mean(r^2) + eps) * weight

`rms_norm` / `RMSNorm` are differentiable; `rms_norm_fp8` is forward-only.  `PreNormMoE` chains norm, router and experts."""
from typing import NamedTuple

import torch
import torch.nn as nn

from ._lib import native
from .fp8 import Fp8Rows


def rms_norm(x, weight, residual=None, eps=1e-6):
    """x [..., D] (bfloat16, float16 or float32; D a multiple of 8 up to 16384), weight [D] in x's type or float32.
    Returns y, or (y, x + residual) when a residual (like x) is given.  Differentiable (once) in x, weight and residual."""
    out = native.rms_norm(x, weight, residual, eps)
    return out[0] if residual is None else (out[0], out[1])


class Fp8Norm(NamedTuple):
    """Result of `rms_norm_fp8`: y, its 8-bit rows, and the rounded sum (None without a residual)."""
    y: torch.Tensor
    rows: Fp8Rows
    residual: torch.Tensor | None


def rms_norm_fp8(x, weight, residual=None, eps=1e-6):
    """`rms_norm` that also gives y as 8-bit rows (converted from the 32-bit value, not from the rounded y).  Forward only."""
    y, q, scale, *r = native.rms_norm_fp8(x, weight, residual, eps)
    return Fp8Norm(y, Fp8Rows(q, scale), r[0] if r else None)


class RMSNorm(nn.Module):
    """`rms_norm` with a learned weight (ones at first)."""

    def __init__(self, embedding_dim, eps=1e-6, weight: torch.Tensor | None = None, device="cuda", dtype=torch.bfloat16):
        super().__init__()
        self.D = embedding_dim
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(embedding_dim, device=device, dtype=dtype) if weight is None
                                   else weight.clone().detach())

    def forward(self, x, residual=None):
        return rms_norm(x, self.weight, residual, self.eps)


class PreNormMoE(nn.Module):
    """Norm, router and experts as a transformer block chains them: `y, r = block(x, residual)` with r = x + residual and
    y = moe(norm(r)).  Without a residual r is x.  When `moe.experts_fp8` is set the norm hands the experts 8-bit rows."""

    def __init__(self, norm: RMSNorm, moe: nn.Module):
        super().__init__()
        self.norm = norm
        self.moe = moe

    def forward(self, x_BSD, residual=None):
        if getattr(self.moe, "experts_fp8", None) is not None:
            y, rows, r = rms_norm_fp8(x_BSD, self.norm.weight, residual, self.norm.eps)
            return self.moe(y, rows), (r if r is not None else x_BSD)
        if residual is None:
            return self.moe(self.norm(x_BSD)), x_BSD
        y, r = self.norm(x_BSD, residual)
        return self.moe(y), r
