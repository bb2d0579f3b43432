"""Root-mean-square norm in front of the expert layer: the residual's addition fused in, a backward pass, and an output in
8 bits for `momoe.fp8` experts.

    r = x + residual (rounded to the stream's type),   y = r / sqrt(mean(r^2) + eps) * weight

`rms_norm` / `RMSNorm` are differentiable; `rms_norm_fp8` is forward-only.  `PreNormMoE` chains norm, router and experts."""
from typing import NamedTuple

import torch
import torch.nn as nn

from . import _lib, ops
from ._lib import as_rows, lib, pitch, ptr, stream_ptr
from .fp8 import BLOCK, Fp8Rows

MAX_D = 16384


def _check(x, weight, residual):
    dev = _lib.require_one_device(x, weight, residual)
    if x.dtype not in _lib.TYPES:
        raise RuntimeError("rms_norm works on bfloat16, float16 or float32, but got: %s" % x.dtype)
    D = x.shape[-1] if x.dim() > 0 else 0
    if D == 0 or D % 8 != 0 or D > MAX_D:
        raise RuntimeError("the normed width must be a multiple of 8 up to %d, but got: %d" % (MAX_D, D))
    if weight.dim() != 1 or weight.shape[0] != D or weight.dtype not in (x.dtype, torch.float32):
        raise RuntimeError("the weight must be [%d] in %s or float32, but got: %s in %s"
                           % (D, x.dtype, list(weight.shape), weight.dtype))
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise RuntimeError("the residual must be like x, %s in %s, but got: %s in %s"
                           % (list(x.shape), x.dtype, list(residual.shape), residual.dtype))
    return dev, D


def _weight(w):
    w = w.detach().contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


def _forward(x, w, residual, eps, want_y, want_rows, want_rstd):
    """x, residual: rows [M, D].  Returns r (None without a residual), y, rstd, q, scale (None where not wanted)."""
    M, D = x.shape
    dev = x.device
    r = torch.empty((M, D), dtype=x.dtype, device=dev) if residual is not None else None
    y = torch.empty((M, D), dtype=x.dtype, device=dev) if want_y else None
    rstd = torch.empty(M, dtype=torch.float32, device=dev) if want_rstd else None
    q = scale = None
    if want_rows:
        q = torch.empty((M, D), dtype=torch.float8_e4m3fn, device=dev)
        scale = torch.empty((M, -(-D // BLOCK)), dtype=torch.float8_e8m0fnu, device=dev)
    if M > 0:
        ops._call("momoe_rms_norm", 1, lib.momoe_rms_norm, ptr(x), pitch(x), ptr(residual),
                  pitch(residual) if residual is not None else 0, ptr(w), _lib.TYPES[x.dtype], _lib.TYPES[w.dtype], M, D,
                  eps, ptr(r), ptr(y), ptr(rstd), ptr(q), ptr(scale), stream_ptr())
    return r, y, rstd, q, scale


class RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        dev, D = _check(x, weight, residual)
        ctx.set_materialize_grads(False)
        w = _weight(weight)
        with torch.cuda.device(dev):
            rows = as_rows(x.detach())
            res = as_rows(residual.detach()) if residual is not None else None
            r, y, rstd, _, _ = _forward(rows, w, res, eps, True, False, any(ctx.needs_input_grad))
        ctx.save_for_backward(r if r is not None else rows, w, rstd)
        y = y.view(x.shape)
        return (y, r.view(x.shape)) if r is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, gr=None):
        r, w, rstd = ctx.saved_tensors
        M, D = r.shape
        need_x, need_w, need_res = ctx.needs_input_grad[:3]
        shape = gy.shape if gy is not None else gr.shape if gr is not None else None
        if shape is None:
            return None, None, None, None
        if gy is None:                       # only the sum was used
            return (gr if need_x else None), (torch.zeros_like(w) if need_w else None), (gr if need_res else None), None
        dev = r.device
        with torch.cuda.device(dev):
            gy = gy.reshape(M, D).contiguous()
            gy = gy if gy.data_ptr() % 16 == 0 else gy.clone()
            if gr is not None:
                gr = gr.reshape(M, D).contiguous()
                gr = gr if gr.data_ptr() % 16 == 0 else gr.clone()
            gx = torch.empty((M, D), dtype=r.dtype, device=dev)
            gw = torch.empty_like(w) if need_w else None
            if M > 0:
                nbytes = int(lib.momoe_rms_norm_backward_workspace_bytes(M, D)) if need_w else 0
                ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if need_w else None
                ops._call("momoe_rms_norm_backward", 2 if need_w else 1, lib.momoe_rms_norm_backward, ptr(gy), ptr(gr),
                          ptr(r), pitch(r), ptr(w), ptr(rstd), _lib.TYPES[r.dtype], _lib.TYPES[w.dtype], M, D, ptr(gx),
                          ptr(gw), ptr(ws), nbytes, stream_ptr())
            elif need_w:
                gw.zero_()
        gx = gx.view(shape)
        return (gx if need_x else None), gw, (gx if need_res else None), None


def rms_norm(x, weight, residual=None, eps=1e-6):
    """x [..., D] (bfloat16, float16 or float32; D a multiple of 8 up to 16384), weight [D] in x's type or float32.
    Returns y, or (y, x + residual) when a residual (like x) is given.  Differentiable in x, weight and residual."""
    return RMSNormFunction.apply(x, weight, residual, float(eps))


class Fp8Norm(NamedTuple):
    """Result of `rms_norm_fp8`: y, its 8-bit rows, and the rounded sum (None without a residual)."""
    y: torch.Tensor
    rows: Fp8Rows
    residual: torch.Tensor | None


def rms_norm_fp8(x, weight, residual=None, eps=1e-6):
    """`rms_norm` that also gives y as 8-bit rows (converted from the 32-bit value, not from the rounded y).  Forward only."""
    dev, D = _check(x, weight, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_fp8 has no backward pass: call it under torch.no_grad()")
    with torch.cuda.device(dev):
        r, y, _, q, scale = _forward(as_rows(x.detach()), _weight(weight),
                                     as_rows(residual.detach()) if residual is not None else None, float(eps), True, True,
                                     False)
    return Fp8Norm(y.view(x.shape), Fp8Rows(q, scale), r.view(x.shape) if r is not None else None)


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
