"""Root-mean-square norm in front of the expert layer: the residual's addition fused in, a backward pass, and an output in
8 bits for `momoe.fp8` experts.

    r = x + residual (rounded to the stream's type),   y = r / sqrt(mean(r^2) + eps) * weight

`rms_norm` / `RMSNorm` are differentiable; `rms_norm_fp8` is forward-only.  `PreNormMoE` chains norm, router and experts."""
from typing import NamedTuple

import torch
import torch.nn as nn

from . import _lib, ops
from ._lib import aligned, as_rows, lib, on_device, pitch, raw_stream
from .fp8 import BLOCK, E4M3, E8M0, Fp8Rows

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
    return dev


def _learns(x, weight, residual):
    return torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                        (residual is not None and residual.requires_grad))


def _forward(x, weight, residual, eps, want_rows, want_rstd):
    """Runs the kernel on checked tensors.  Returns the input rows [M, D] (the sum r where there is a residual), the weight
    as the kernel read it, y, rstd and the 8-bit rows (None where not wanted)."""
    dev, dtype = x.device, x.dtype
    x = as_rows(x)
    w = aligned(weight if weight.is_contiguous() else weight.contiguous())
    M, D = x.shape
    y = torch.empty((M, D), dtype=dtype, device=dev)
    r = rstd = rows = res_ptr = r_ptr = None
    res_pitch = 0
    if residual is not None:
        residual = as_rows(residual)
        r = torch.empty((M, D), dtype=dtype, device=dev)
        res_ptr, r_ptr, res_pitch = residual.data_ptr(), r.data_ptr(), pitch(residual)
    if want_rstd:
        rstd = torch.empty(M, dtype=torch.float32, device=dev)
    if want_rows:
        rows = Fp8Rows(torch.empty((M, D), dtype=E4M3, device=dev), torch.empty((M, -(-D // BLOCK)), dtype=E8M0, device=dev))
    if M > 0:
        ops._call("momoe_rms_norm", 1, lib.momoe_rms_norm, x.data_ptr(), pitch(x), res_ptr, res_pitch, w.data_ptr(),
                  _lib.TYPES[dtype], _lib.TYPES[w.dtype], M, D, eps, r_ptr, y.data_ptr(),
                  rstd.data_ptr() if want_rstd else None, rows.q.data_ptr() if want_rows else None,
                  rows.scale.data_ptr() if want_rows else None, raw_stream(dev))
    return (x if r is None else r), w, y, rstd, rows


class RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        shape = x.shape
        with on_device(x.device):
            r, w, y, rstd, _ = _forward(x, weight, residual, eps, False, True)
        ctx.save_for_backward(r, w, rstd)
        ctx.shape = shape
        if len(shape) != 2:
            y = y.view(shape)
            r = r.view(shape) if residual is not None else r
        return (y, r) if residual is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, gr=None):
        r, w, rstd = ctx.saved_tensors
        need_x, need_w, need_res, _ = ctx.needs_input_grad
        if gy is None:                       # only the sum was used, or nothing
            gw = torch.zeros_like(w) if need_w and gr is not None else None
            return (gr if need_x else None), gw, (gr if need_res else None), None
        D = w.shape[0]
        dev = w.device
        with on_device(dev):
            r = r if r.dim() == 2 else r.view(-1, D)
            M = r.shape[0]
            gy = aligned(gy if gy.is_contiguous() else gy.contiguous())
            if gr is not None:
                gr = aligned(gr if gr.is_contiguous() else gr.contiguous())
            gx = torch.empty((M, D), dtype=r.dtype, device=dev)
            gw = torch.empty_like(w) if need_w else None
            if M > 0:
                nbytes = _lib.rms_norm_backward_workspace_bytes(M, D) if need_w else 0
                ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if need_w else None
                ops._call("momoe_rms_norm_backward", 2 if need_w else 1, lib.momoe_rms_norm_backward, gy.data_ptr(),
                          gr.data_ptr() if gr is not None else None, r.data_ptr(), pitch(r), w.data_ptr(),
                          rstd.data_ptr(), _lib.TYPES[r.dtype], _lib.TYPES[w.dtype], M, D, gx.data_ptr(),
                          gw.data_ptr() if need_w else None, ws.data_ptr() if need_w else None, nbytes, raw_stream(dev))
            elif need_w:
                gw.zero_()
        if len(ctx.shape) != 2:
            gx = gx.view(ctx.shape)
        return (gx if need_x else None), gw, (gx if need_res else None), None


def rms_norm(x, weight, residual=None, eps=1e-6):
    """x [..., D] (bfloat16, float16 or float32; D a multiple of 8 up to 16384), weight [D] in x's type or float32.
    Returns y, or (y, x + residual) when a residual (like x) is given.  Differentiable in x, weight and residual."""
    dev = _check(x, weight, residual)
    if _learns(x, weight, residual):
        return RMSNormFunction.apply(x, weight, residual, float(eps))
    with on_device(dev):
        r, _, y, _, _ = _forward(x.detach(), weight.detach(), residual.detach() if residual is not None else None,
                                 float(eps), False, False)
    if x.dim() != 2:
        y, r = y.view(x.shape), (r.view(x.shape) if residual is not None else r)
    return (y, r) if residual is not None else y


class Fp8Norm(NamedTuple):
    """Result of `rms_norm_fp8`: y, its 8-bit rows, and the rounded sum (None without a residual)."""
    y: torch.Tensor
    rows: Fp8Rows
    residual: torch.Tensor | None


def rms_norm_fp8(x, weight, residual=None, eps=1e-6):
    """`rms_norm` that also gives y as 8-bit rows (converted from the 32-bit value, not from the rounded y).  Forward only."""
    dev = _check(x, weight, residual)
    if _learns(x, weight, residual):
        raise RuntimeError("rms_norm_fp8 has no backward pass: call it under torch.no_grad()")
    with on_device(dev):
        r, _, y, _, rows = _forward(x.detach(), weight.detach(), residual.detach() if residual is not None else None,
                                    float(eps), True, False)
    if x.dim() != 2:
        y, r = y.view(x.shape), (r.view(x.shape) if residual is not None else r)
    return Fp8Norm(y, rows, r if residual is not None else None)


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
