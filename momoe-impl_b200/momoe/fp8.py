"""The experts' forward pass in 8-bit floating point: e4m3 rows and weights with a power of two (e8m0) for each block of
128, multiplied on the tensor cores with 32-bit accumulation.  Forward only.  `Fp8Experts` takes half the memory of bfloat16
weights and needs nothing else; a `MoE` layer keeps its 16-bit weights beside it.

    experts = quantize_experts(moe.momoe.Wl1_ND2H, moe.momoe.Wl2_NHD)       # once, when the weights are final
    y_MD, tokens_per_expert_N = experts_forward(x_MD, topk_idx_MK, topk_w_MK, experts)

`MoE.quantize_experts()` does the first and makes the module use the second."""
from typing import NamedTuple

import torch

from . import _lib, ops
from ._lib import as_rows, lib, native, on_device, pitch, ptr, raw_stream

BLOCK = 128                      # values that share a scale
# Calls with at most this many rows per expert on average stream the weights past the rows; more take the row-tile kernels.
# Whole passes, streaming against tiles: one token 26.0 / 30.0 us, 1 row an expert 87 / 91.5, 4 rows 130 / 133.5, 8 rows 142.5 /
# 145, 12 rows 147.6 / 148.5, 24 rows 167 / 155 (D2048 H1024, top-8 of 128).
STREAM_MAX_AVG_ROWS = 8
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


class Fp8Rows(NamedTuple):
    """Rows in 8 bits: the value of column c is q[m, c] * scale[m, c // 128]."""
    q: torch.Tensor              # float8_e4m3fn [M, D]
    scale: torch.Tensor          # float8_e8m0fnu [M, ceil(D / 128)]


class Fp8Experts(NamedTuple):
    """Expert weights in 8 bits, the contraction axis last, one scale for each 128 x 128 block."""
    W1_N2HD: torch.Tensor        # float8_e4m3fn [N, 2H, D]: rows [:H] linear half, [H:] gate half
    S1: torch.Tensor             # float8_e8m0fnu [N, 2, ceil(H / 128), ceil(D / 128)]
    W2_NDH: torch.Tensor         # float8_e4m3fn [N, D, H]
    S2: torch.Tensor             # float8_e8m0fnu [N, ceil(D / 128), ceil(H / 128)]

    @property
    def sizes(self):
        """(N, D, H)."""
        return self.W2_NDH.shape


def _blocks(n):
    return -(-n // BLOCK)


def quantize_rows(x):
    """x [..., D] (bfloat16, float16 or float32; D a multiple of 8) -> Fp8Rows of the [M, D] view.  The scale of a block
    is the smallest power of two that brings its largest magnitude to 448 at most (1 for a block of zeros, NaN for a block
    that holds an infinity or a NaN), so only the conversion to e4m3 rounds.  x is taken as a constant: no gradient passes."""
    _lib.require_cuda(x)
    if x.dtype not in _lib.TYPES:
        raise RuntimeError("quantize_rows works on bfloat16, float16 or float32, but got: %s" % x.dtype)
    if x.dim() == 0 or x.shape[-1] == 0 or x.shape[-1] % 8 != 0:
        raise RuntimeError("the width of 8-bit rows must be a multiple of 8, but got: %s" % list(x.shape))
    with on_device(x.device):
        r = as_rows(x.detach())
        M, D = r.shape
        rows = Fp8Rows(torch.empty((M, D), dtype=E4M3, device=x.device),
                       torch.empty((M, _blocks(D)), dtype=E8M0, device=x.device))
        if M > 0:
            ops._call("momoe_quantize_rows", 1, lib.momoe_quantize_rows, ptr(r), pitch(r), _lib.TYPES[r.dtype], M, D,
                      ptr(rows.q), ptr(rows.scale), raw_stream(x.device))
    return rows


def _quantize_weights(W, groups):
    N, Kd, C = W.shape
    W = W.detach().contiguous()
    if W.dtype not in (torch.bfloat16, torch.float32):
        W = W.to(torch.float32)
    q = torch.empty((N, C, Kd), dtype=E4M3, device=W.device)
    S = torch.empty((N, groups, _blocks(C // groups), _blocks(Kd)), dtype=E8M0, device=W.device)
    ops._call("momoe_fp8_quantize_weights", 1, lib.momoe_fp8_quantize_weights, ptr(W), _lib.TYPES[W.dtype], N, Kd, groups,
              C // groups, ptr(q), ptr(S), raw_stream(W.device))
    return q, S


def quantize_experts(Wl1_ND2H, Wl2_NHD):
    """Up/gate weights [N, D, 2H] and down weights [N, H, D], as `MoMoE` holds them -> Fp8Experts.  No gradient passes."""
    dev = _lib.require_one_device(Wl1_ND2H, Wl2_NHD)
    if Wl1_ND2H.dim() != 3 or Wl2_NHD.dim() != 3:
        raise RuntimeError("expert weights must be [N, D, 2H] and [N, H, D], but got: %s and %s"
                           % (list(Wl1_ND2H.shape), list(Wl2_NHD.shape)))
    N, H, D = Wl2_NHD.shape
    if tuple(Wl1_ND2H.shape) != (N, D, 2 * H):
        raise RuntimeError("expert weights must be [N, D, 2H] and [N, H, D], but got: %s and %s"
                           % (list(Wl1_ND2H.shape), list(Wl2_NHD.shape)))
    if N == 0 or D == 0 or H == 0 or D % 16 != 0 or H % 16 != 0:
        raise RuntimeError("8-bit experts need D and H in multiples of 16, but got: D = %d, H = %d" % (D, H))
    with on_device(dev):
        W1, S1 = _quantize_weights(Wl1_ND2H, 2)
        W2, S2 = _quantize_weights(Wl2_NHD, 1)
    return Fp8Experts(W1, S1, W2, S2.view(N, _blocks(D), _blocks(H)))


def experts_forward(x, topk_idx_MK, topk_w_MK, experts):
    """Weighted sum of the K chosen experts' outputs for each token, in 8 bits.

    x: bfloat16 [M, D] (converted on the way; other float types are cast to bfloat16 first), or Fp8Rows;
    topk_idx_MK int32 [M, K]: expert ids (one named twice counts with both weights); topk_w_MK float32 [M, K]; experts:
    Fp8Experts.  D, H multiples of 16 up to 2^22, N <= 1024, K <= 32, M K up to 8.2 million.  Returns (y bfloat16 [M, D],
    tokens_per_expert_N int64 [N]).  The hidden values are converted to 8-bit rows once, from 32 bits.  No host synchronisation: an expert id out of range (202) is reported through the
    device's status word like the other problems only the device can see."""
    q, scale = x if isinstance(x, Fp8Rows) else (x, None)
    _lib.require_cuda(q)
    y, sizes = native.experts_forward(q, scale, topk_idx_MK, topk_w_MK, *experts, STREAM_MAX_AVG_ROWS,
                                      ops.status_word(q.device))
    return y, sizes
