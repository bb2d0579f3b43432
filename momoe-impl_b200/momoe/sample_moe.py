"""`MoE`: router + MoMoE + aux-loss-free bias update, same interface as the reference wrapper
(momoe/sample_moe.py:16-68 there).

By default the wrapper runs router and experts as one autograd node that keeps the routing in its compact form
(top-k ids, weights, permutation): the dense `mask_NM` / `s_NM` of the two-module composition, the dense `G_s_NM` and
the dense router backward are never materialised.  `MoE.fused = False` restores the literal composition
`TopKRouter -> MoMoE`; both give the same output bit for bit.

Two things the reference does not have are switched on by attributes: `balance_coef` / `z_coef` add the router's balance
loss and z-loss (`momoe.balance`; the value is `MoE.aux_loss`, to be added to the training loss), and `quantize_experts()`
makes forward-only calls run the experts in 8 bits (`momoe.fp8`)."""
import weakref

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import balance, fp8, ops
from ._lib import native, require_cuda
from .momoe import MoMoE, _CHECK, compact_routing_of
from .topk_router import TopKRouter


class FusedMoEFunction(torch.autograd.Function):
    """Gate GEMM -> router kernel -> permutation -> experts, and the matching backward, on compact routing data.
    Stands in for momoe/topk_router.py:85-145 plus momoe/momoe.py:847-903 of the reference.  With a balance or z
    coefficient there is a third output, the router's auxiliary loss, each of the B sequences balanced on its own."""

    @staticmethod
    def forward(ctx, x_BSD, Wg_DN, Wl1_ND2H, Wl2_NHD, biases_N, K, Ks, save_percent, balance_coef, z_coef):
        B, S, D = x_BSD.shape
        assert Wg_DN.dtype == torch.bfloat16, "Wg_DN must be of type torch.bfloat16"
        assert Wl1_ND2H.device == Wl2_NHD.device, \
            "All weights must be on the same device, but got: Wl1_ND2H.device = {}, Wl2_NHD.device = {}".format(
                Wl1_ND2H.device, Wl2_NHD.device)
        require_cuda(Wl1_ND2H, Wg_DN)
        dev = Wl1_ND2H.device
        N, H, _ = Wl2_NHD.shape
        x_MD = x_BSD.reshape(B * S, D).to(device=dev, dtype=torch.bfloat16).contiguous()
        Wg = Wg_DN.detach()
        W1 = Wl1_ND2H.detach().to(torch.bfloat16).contiguous()
        W2 = Wl2_NHD.detach().to(torch.bfloat16).contiguous()
        with torch.cuda.device(dev):
            logits_MN = x_MD @ Wg
            topk_idx, topk_w, d = ops.route_topk(logits_MN, biases_N, K, Ks, dense=False, normalisers=True)
            plan = ops.RoutingPlan.from_topk(topk_idx, topk_w, N, D, H, save_percent)
            y_MD, a_save, b_save = ops.experts_forward(plan, x_MD, W1, W2,
                                                          inference=not any(ctx.needs_input_grad))
            ctx.aux = balance_coef != 0 or z_coef != 0
            if ctx.aux:
                aux_loss, _, g_BN = native.balance_forward(logits_MN, topk_idx, Ks, balance_coef, z_coef, None, S, B)
        ctx.plan = plan
        ctx.shape = (B, S, D)
        ctx.Ks = Ks
        ctx.z_coef = z_coef
        ctx.x_device = x_BSD.device
        saved = [x_MD, Wg, W1, W2, d["Ng_M"], d["Ks_M"]]
        if ctx.aux:
            saved += [logits_MN, g_BN]
        ctx.has_ab = a_save is not None
        if ctx.has_ab:
            saved += [a_save, b_save]
        ctx.save_for_backward(*saved)
        ctx.mark_non_differentiable(plan.sizes)
        ops.status_post(dev)
        if _CHECK:
            ops.check_status(dev)
        y_BSD = y_MD.reshape(B, S, D).to(device=x_BSD.device)
        return (y_BSD, plan.sizes, aux_loss) if ctx.aux else (y_BSD, plan.sizes)

    @staticmethod
    def backward(ctx, G_y_BSD, _, G_aux=None):
        saved = ctx.saved_tensors
        x_MD, Wg, W1, W2, Ng_M, Ks_M = saved[:6]
        a_save, b_save = (saved[-2], saved[-1]) if ctx.has_ab else (None, None)
        B, S, D = ctx.shape
        plan = ctx.plan
        dev = W1.device
        g_MD = G_y_BSD.reshape(B * S, D).to(device=dev, dtype=torch.bfloat16).contiguous()
        with torch.cuda.device(dev):
            G_x, G_W1, G_W2, gs_part = ops.experts_backward(plan, g_MD, x_MD, W1, W2, a_save, b_save,
                                                            need_gs_dense=False)
            G_L = ops.router_backward_compact(plan, gs_part, Ng_M, Ks_M, ctx.Ks)
            if ctx.aux:
                # the experts' share of the logits' gradient is in 16 bits already; the sum is formed in 32 and rounded
                # once more, like every gradient that reaches the two gate GEMMs
                G_L = native.balance_backward(saved[6], saved[7], ctx.Ks, ctx.z_coef, None, S, G_aux, G_L)
            G_x = torch.addmm(G_x, G_L, Wg.T)
            G_Wg = x_MD.T @ G_L
        ops.status_post(dev)
        if _CHECK:
            ops.check_status(dev)
        return G_x.reshape(B, S, D).to(ctx.x_device), G_Wg, G_W1, G_W2, None, None, None, None, None, None


def _version(w):
    """Counts the in-place changes of a tensor; tensors made in inference mode have no count."""
    return None if w.is_inference() else w._version


def _refs(tensors):
    return tuple(weakref.ref(t) for t in tensors)


def _same(refs, tensors):
    return all(ref() is t for ref, t in zip(refs, tensors))


class MoE(nn.Module):
    balance_coef = 0.0     # weight of the balance loss (each of a batch's sequences on its own)
    z_coef = 0.0           # weight of the z-loss
    aux_loss = None        # their sum of the latest forward pass, float32 [], differentiable; None if both are 0
    experts_fp8 = None     # 8-bit weights of forward-only calls, from quantize_experts()
    # (tensors of experts_fp8, the weights that they stand for with their versions), by weak references; no weights: none of
    # this layer's.  In a saved state (): those, else None.
    _fp8_weights = None

    def __init__(self, embedding_dim, intermediate_dim, num_experts, num_chosen_experts, num_shared_experts,
                 save_percent=0, bias_update_rate=1e-4, Wg_DN: torch.Tensor | None = None,
                 Wl1_ND2H: torch.Tensor | None = None, Wl2_NHD: torch.Tensor | None = None):
        super().__init__()
        self.D = embedding_dim
        self.H = intermediate_dim
        self.N = num_experts
        self.K = num_chosen_experts
        self.Ks = num_shared_experts
        self.save_percent = save_percent
        self.bias_update_rate = bias_update_rate
        self.router = TopKRouter(embedding_dim=self.D, num_experts=self.N, num_chosen_experts=self.K,
                                 num_shared_experts=self.Ks, Wg_DN=Wg_DN)
        self.momoe = MoMoE(embedding_dim=self.D, intermediate_dim=self.H, num_experts=self.N,
                           num_chosen_experts=self.K, save_percent=self.save_percent, Wl1_ND2H=Wl1_ND2H,
                           Wl2_NHD=Wl2_NHD)
        dev = self.momoe.Wl1_ND2H.device
        self.biases_N = nn.Parameter(
            torch.cat([torch.zeros(self.N - self.Ks, device=dev, dtype=torch.float32),
                       torch.full((self.Ks,), float("-inf"), device=dev, dtype=torch.float32)], dim=-1),
            requires_grad=False)
        self.fused = True

    def __getstate__(self):
        state = dict(self.__dict__)
        state.pop("aux_loss", None)         # belongs to the graph of a forward pass, not to a copy of the layer
        # a copy has weights of its own, for which its 8-bit ones stand if they stand for this layer's
        state["_fp8_weights"] = None if self.experts_fp8 is None or self._fp8_fresh() else ()
        return state

    def __setstate__(self, state):
        super().__setstate__(state)
        if self.experts_fp8 is not None:
            if self._fp8_weights == ():
                self._fp8_weights = _refs(self.experts_fp8), ()
            self._fp8_fresh()

    def _fp8_fresh(self):
        """Whether the 8-bit weights stand for the layer's weights as they are; ones that were set by hand do from the first
        look on."""
        weights = self.momoe.Wl1_ND2H, self.momoe.Wl2_NHD
        if self._fp8_weights is None or not _same(self._fp8_weights[0], self.experts_fp8):
            self._fp8_weights = _refs(self.experts_fp8), tuple(zip(_refs(weights), map(_version, weights)))
        seen = self._fp8_weights[1]
        return len(seen) == 2 and all(ref() is w and version == _version(w) for (ref, version), w in zip(seen, weights))

    def quantize_experts(self):
        """From now on forward passes use an 8-bit copy of the expert weights as they are now.  Such passes have no
        backward: they run under torch.no_grad() (or with nothing that requires a gradient).  The copy is held beside the
        16-bit weights, is no part of state_dict() and does not follow `.to()`.  When the weights have
        changed since (in place or by other ones; changes through `.data`, and in-place changes of tensors made in inference
        mode, are not seen), forward raises; call this again, or set `experts_fp8 = None` to go back to 16 bits."""
        self.experts_fp8 = fp8.quantize_experts(self.momoe.Wl1_ND2H, self.momoe.Wl2_NHD)
        self._fp8_weights = None
        self._fp8_fresh()

    def _forward_fp8(self, x_BSD, rows):
        if torch.is_grad_enabled() and (x_BSD.requires_grad or any(p.requires_grad for p in self.parameters())):
            raise RuntimeError("8-bit experts have no backward pass: call the layer under torch.no_grad()")
        if forward_ad.unpack_dual(x_BSD).tangent is not None:
            raise RuntimeError("8-bit experts have no forward-mode derivative")
        if not self._fp8_fresh():
            raise RuntimeError("the expert weights have changed since quantize_experts(): call it again")
        Wg = self.router.Wg_DN
        assert Wg.dtype == torch.bfloat16, "Wg_DN must be of type torch.bfloat16"
        dev = Wg.device
        require_cuda(Wg)
        ops.status_poll(dev)
        B, S, D = x_BSD.shape
        with torch.cuda.device(dev):
            x_MD = x_BSD.detach().reshape(B * S, D).to(device=dev, dtype=torch.bfloat16)
            topk_idx, topk_w, _ = ops.route_topk(x_MD @ Wg.detach(), self.biases_N.detach(), self.K, self.Ks, dense=False)
            y_MD, sizes_N = fp8.experts_forward(x_MD if rows is None else rows, topk_idx, topk_w, self.experts_fp8)
        ops.status_post(dev)
        if _CHECK:
            ops.check_status(dev)
        return y_MD.reshape(B, S, D).to(device=x_BSD.device), sizes_N

    def forward(self, x_BSD, rows_fp8=None):
        """x_BSD [B, S, D] -> y_BSD.  rows_fp8: the same rows in 8 bits (momoe.fp8.Fp8Rows), if the caller has them, for
        a layer with 8-bit experts; the router always reads x_BSD."""
        self.aux_loss = None        # before the new graph is built: an old one must not keep its gradient nodes alive
        aux = self.balance_coef != 0 or self.z_coef != 0
        if self.experts_fp8 is not None:
            if aux:
                raise RuntimeError("balance_coef and z_coef are for training: 8-bit experts have no backward pass")
            y_BSD, sizes_N = self._forward_fp8(x_BSD, rows_fp8)
        elif rows_fp8 is not None:
            raise RuntimeError("8-bit rows need 8-bit experts: call quantize_experts() first")
        elif self.fused:
            ops.status_poll(self.momoe.Wl1_ND2H.device)  # raises if an earlier pass left a device-side error code
            out = FusedMoEFunction.apply(x_BSD, self.router.Wg_DN, self.momoe.Wl1_ND2H, self.momoe.Wl2_NHD,
                                         self.biases_N, self.K, self.Ks, self.save_percent, float(self.balance_coef),
                                         float(self.z_coef))
            y_BSD, sizes_N = out[:2]
            if aux:
                self.aux_loss = out[2]
        else:
            x_in = x_BSD
            x_BSD, mask_NM, s_NM = self.router(x_BSD, self.biases_N)
            y_BSD, sizes_N = self.momoe(x_BSD, mask_NM, s_NM)
            if aux:
                topk_idx, _ = compact_routing_of(mask_NM, s_NM)
                Wg = self.router.Wg_DN
                logits_MN = x_in.reshape(-1, self.D).to(device=Wg.device, dtype=torch.bfloat16) @ Wg
                self.aux_loss, _ = balance.balance_loss(logits_MN, topk_idx, self.Ks, self.balance_coef, self.z_coef,
                                                        seq_len=x_in.shape[1])
        # DeepSeek-style auxiliary-loss-free balancing: push the bias of under-loaded experts up
        B, S, _ = x_BSD.shape
        c_avg = B * S * (self.K - self.Ks) / (self.N - self.Ks)
        with torch.no_grad():
            ops.bias_update_(self.biases_N.data, sizes_N, self.Ks, c_avg, self.bias_update_rate)
        return y_BSD
