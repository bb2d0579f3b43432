"""Balance loss and z-loss of the router, with tokens per expert and sequence, differentiable in the gate logits.

With p the softmax over the Ng = N - Ks gating logits of a token, T_b the tokens of sequence b, B' the sequences that are
not empty, T all tokens, Kg = K - Ks:

    loss = balance_coef / B' * sum_b sum_e  [Ng / (Kg T_b) * count_be] * [mean of p_e over sequence b]
         + z_coef / T * sum_t (log sum_e exp logit_te)^2

The counts carry no gradient.  Perfectly even routing gives a first term of balance_coef.  It complements the bias update
of `MoE`, which balances over the whole batch; `MoE.balance_coef` / `MoE.z_coef` switch it on there."""
from ._lib import native


def balance_loss(logits_MN, topk_idx_MK, num_shared_experts=0, balance_coef=1.0, z_coef=0.0, cu_seqlens=None,
                 seq_len=None):
    """logits_MN bfloat16 or float32 [M, N]; topk_idx_MK whole numbers [M, K] (ids outside [0, N) are not counted).

    The rows are packed sequences: cu_seqlens [B + 1] on the device, ascending, sequence b is rows cu_seqlens[b] up
    to cu_seqlens[b + 1] (empty ones count for nothing; rows outside, such as padding, are not read and get a zero
    gradient; bounds outside [0, M] count as 0 and M; a table that does not ascend, which only the device can see, gives a
    loss and gradients of NaN and counts of 0); or seq_len, consecutive sequences of that many rows (B =
    ceil(M / seq_len)); or neither, one sequence.
    Returns (loss float32 [], tokens_per_expert_BN int64 [B, N]); shared experts are counted but not balanced."""
    loss, counts = native.balance_loss(logits_MN, topk_idx_MK, num_shared_experts, balance_coef, z_coef, cu_seqlens,
                                       seq_len)
    return loss, counts
