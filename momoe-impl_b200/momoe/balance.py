"""Balance loss and z-loss of the router, with tokens per expert and sequence, differentiable in the gate logits.

With p the softmax over the Ng = N - Ks gating logits of a token, T_b the tokens of sequence b, B' the sequences that are
not empty, T all tokens, Kg = K - Ks:

    loss = balance_coef / B' * sum_b sum_e  [Ng / (Kg T_b) * count_be] * [mean of p_e over sequence b]
         + z_coef / T * sum_t (log sum_e exp logit_te)^2

The counts carry no gradient.  Perfectly even routing gives a first term of balance_coef.  It complements the bias update
of `MoE`, which balances over the whole batch; `MoE.balance_coef` / `MoE.z_coef` switch it on there."""
import torch

from . import _lib, ops
from ._lib import aligned, lib, on_device, raw_stream

MAX_EXPERTS, MAX_SEQUENCES = 1024, 65535


def _loss(logits, idx, Ks, balance_coef, z_coef, cu, seq_len, B):
    """Checked contiguous tensors -> loss [], counts [B, N], the backward pass's coefficients [B, N]."""
    M, N = logits.shape
    dev = logits.device
    loss = torch.empty((), dtype=torch.float32, device=dev)
    counts = torch.empty((B, N), dtype=torch.int64, device=dev)
    g = torch.empty((B, N), dtype=torch.float32, device=dev)
    if M == 0:
        return loss.zero_(), counts.zero_(), g.zero_()
    nbytes = _lib.balance_loss_workspace_bytes(M, N, B)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    ops._call("momoe_balance_loss", 2, lib.momoe_balance_loss, logits.data_ptr(), _lib.TYPES[logits.dtype],
              idx.data_ptr(), cu.data_ptr() if cu is not None else None, seq_len, M, N, idx.shape[1], Ks, B, balance_coef,
              z_coef, loss.data_ptr(), counts.data_ptr(), g.data_ptr(), ws.data_ptr(), nbytes, raw_stream(dev))
    return loss, counts, g


def _loss_backward(logits, g, Ks, z_coef, cu, seq_len, B, G_loss, add=None):
    """Gradient of the logits; `add`: a gradient from elsewhere that is overwritten with the sum."""
    M, N = logits.shape
    out = add if add is not None else torch.empty_like(logits)
    if M > 0:
        ops._call("momoe_balance_loss_backward", 1, lib.momoe_balance_loss_backward, logits.data_ptr(),
                  _lib.TYPES[logits.dtype], cu.data_ptr() if cu is not None else None, seq_len, g.data_ptr(), M, N, Ks, B,
                  z_coef, G_loss.data_ptr(), add.data_ptr() if add is not None else None, out.data_ptr(),
                  raw_stream(logits.device))
    return out


class BalanceLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, idx, Ks, balance_coef, z_coef, cu, seq_len, B):
        with on_device(logits.device):
            x = aligned(logits.contiguous())
            loss, counts, g = _loss(x, idx, Ks, balance_coef, z_coef, cu, seq_len, B)
        ctx.save_for_backward(x, g, cu)
        ctx.args = (Ks, z_coef, seq_len, B)
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, G_loss, _):
        x, g, cu = ctx.saved_tensors
        Ks, z_coef, seq_len, B = ctx.args
        with on_device(x.device):
            out = _loss_backward(x, g, Ks, z_coef, cu, seq_len, B, G_loss)
        return out, None, None, None, None, None, None, None


def balance_loss(logits_MN, topk_idx_MK, num_shared_experts=0, balance_coef=1.0, z_coef=0.0, cu_seqlens=None,
                 seq_len=None):
    """logits_MN bfloat16 or float32 [M, N]; topk_idx_MK int32 [M, K] (ids outside [0, N) are not counted).

    The rows are packed sequences: cu_seqlens int32 [B + 1] on the device, ascending, sequence b is rows cu_seqlens[b] up
    to cu_seqlens[b + 1] (empty ones count for nothing; rows outside, such as padding, are not read and get a zero
    gradient); or seq_len, consecutive sequences of that many rows (B = ceil(M / seq_len)); or neither, one sequence.
    Returns (loss float32 [], tokens_per_expert_BN int64 [B, N]); shared experts are counted but not balanced."""
    dev = _lib.require_one_device(logits_MN, topk_idx_MK, cu_seqlens)
    Ks = num_shared_experts
    if logits_MN.dtype not in (torch.bfloat16, torch.float32):
        raise RuntimeError("the logits must be bfloat16 or float32, but got: %s" % logits_MN.dtype)
    if logits_MN.dim() != 2 or topk_idx_MK.dim() != 2 or topk_idx_MK.shape[0] != logits_MN.shape[0]:
        raise RuntimeError("the logits must be [M, N] and the expert ids [M, K], but got: %s and %s"
                           % (list(logits_MN.shape), list(topk_idx_MK.shape)))
    M, N = logits_MN.shape
    K = topk_idx_MK.shape[1]
    if not 0 <= Ks < K <= N or N > MAX_EXPERTS:
        raise RuntimeError("0 <= shared experts < K <= N <= %d is needed, but got: Ks = %d, K = %d, N = %d"
                           % (MAX_EXPERTS, Ks, K, N))
    if cu_seqlens is not None and seq_len is not None:
        raise RuntimeError("give cu_seqlens or seq_len, not both")
    with on_device(dev):
        if topk_idx_MK.dtype != torch.int32:
            topk_idx_MK = topk_idx_MK.to(torch.int32)
        idx = topk_idx_MK.contiguous()
        if cu_seqlens is not None:
            if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2 or cu_seqlens.is_floating_point():
                raise RuntimeError("cu_seqlens must be whole numbers [B + 1], but got: %s in %s"
                                   % (list(cu_seqlens.shape), cu_seqlens.dtype))
            cu_seqlens = cu_seqlens.to(torch.int32).contiguous()
            B, seq_len = cu_seqlens.shape[0] - 1, 0
        else:
            seq_len = max(M, 1) if seq_len is None else min(int(seq_len), max(M, 1))
            if seq_len <= 0:
                raise RuntimeError("seq_len must be positive, but got: %d" % seq_len)
            B = max(1, -(-M // seq_len))
        if B > MAX_SEQUENCES:
            raise RuntimeError("at most %d sequences, but got: %d" % (MAX_SEQUENCES, B))
        return BalanceLossFunction.apply(logits_MN, idx, Ks, float(balance_coef), float(z_coef), cu_seqlens, seq_len, B)
