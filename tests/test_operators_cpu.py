"""What the operators around the expert layer refuse on the host, before anything is launched, and the sizes they ask
for."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__
    __graft_entry__.build()
    from momoe import _lib
    return _lib


ONE = C.c_void_p(256)      # never dereferenced: every call below fails its checks first
ODD = C.c_void_p(264)


def test_norm_arguments(lib):
    f = lib.lib.momoe_rms_norm
    def call(x=ONE, xs=64, res=None, rs=0, w=ONE, t=0, wt=0, M=4, D=64, eps=1e-6, r=None, y=ONE, rstd=None, q=None, s=None):
        return f(x, xs, res, rs, w, t, wt, M, D, eps, r, y, rstd, q, s, None)
    assert call(M=0) == 0
    assert call(M=-1) == -1 and call(D=0) == -1 and call(D=60) == -2 and call(D=16392) == -4
    assert call(t=3) == -2 and call(t=0, wt=1) == -2 and call(t=2, wt=0) == -2
    assert call(x=None) == -1 and call(w=None) == -1 and call(y=None) == -1
    assert call(res=ONE) == -1 and call(r=ONE) == -1 and call(q=ONE) == -1 and call(s=ONE) == -1
    assert call(x=ODD) == -1 and call(w=ODD) == -1 and call(y=ODD) == -1 and call(xs=60) == -1 and call(xs=-8) == -1
    assert call(eps=-1.0) == -1 and call(eps=float("nan")) == -1
    b = lib.lib.momoe_rms_norm_backward
    def back(gy=ONE, gr=None, r=ONE, rs=64, w=ONE, rstd=ONE, t=0, wt=0, M=4, D=64, gx=ONE, gw=ONE, ws=ONE, n=None):
        n = lib.lib.momoe_rms_norm_backward_workspace_bytes(M, D) if n is None else n
        return b(gy, gr, r, rs, w, rstd, t, wt, M, D, gx, gw, ws, n, None)
    assert back(n=4) == -1 and back(ws=None) == -1 and back(gx=None) == -1 and back(rstd=None) == -1 and back(M=0) == -1
    assert back(gr=ODD) == -1 and back(rs=3) == -1 and back(D=12) == -2
    assert lib.lib.momoe_rms_norm_backward_workspace_bytes(4, 64) == 4 * 64 * 4
    assert lib.lib.momoe_rms_norm_backward_workspace_bytes(0, 64) == 0


def test_balance_arguments(lib):
    f = lib.lib.momoe_balance_loss
    def call(x=ONE, t=0, idx=ONE, cu=None, S=10, M=10, N=16, K=2, Ks=0, B=1, loss=ONE, c=ONE, g=ONE, ws=ONE, n=None):
        n = lib.lib.momoe_balance_loss_workspace_bytes(M, N, B) if n is None else n
        return f(x, t, idx, cu, S, M, N, K, Ks, B, 1.0, 0.0, loss, c, g, ws, n, None)
    assert call(M=0) == -1 and call(N=0) == -1 and call(B=0) == -1 and call(Ks=-1) == -1 and call(Ks=2) == -1
    assert call(K=17) == -1 and call(t=1) == -2 and call(N=1025) == -4 and call(cu=ONE, B=65536) == -4
    assert call(S=0) == -1 and call(S=3) == -1 and call(S=9, B=3) == -1          # 10 rows of 9 are two sequences
    assert call(x=None) == -1 and call(idx=None) == -1 and call(loss=None) == -1 and call(c=None) == -1
    assert call(g=None) == -1 and call(ws=None) == -1 and call(n=8) == -1 and call(x=ODD) == -1
    b = lib.lib.momoe_balance_loss_backward
    def back(x=ONE, t=0, cu=None, S=10, g=ONE, M=10, N=16, Ks=0, B=1, up=ONE, add=None, out=ONE):
        return b(x, t, cu, S, g, M, N, Ks, B, 0.0, up, add, out, None)
    assert back(up=None) == -1 and back(out=None) == -1 and back(add=ODD) == -1 and back(S=4) == -1 and back(t=1) == -2


def test_fp8_arguments(lib):
    L = lib.lib
    assert L.momoe_quantize_rows(ONE, 64, 0, 4, 60, ONE, ONE, None) == -2
    assert L.momoe_quantize_rows(ONE, 64, 5, 4, 64, ONE, ONE, None) == -2
    assert L.momoe_quantize_rows(None, 64, 0, 4, 64, ONE, ONE, None) == -1
    assert L.momoe_quantize_rows(ONE, 64, 0, 0, 64, ONE, ONE, None) == 0
    assert L.momoe_fp8_quantize_weights(ONE, 0, 4, 40, 2, 32, ONE, ONE, None) == -2
    assert L.momoe_fp8_quantize_weights(ONE, 1, 4, 64, 2, 32, ONE, ONE, None) == -2
    assert L.momoe_fp8_quantize_weights(ONE, 0, 4, 64, 2, 32, None, ONE, None) == -1
    assert L.momoe_fp8_quantize_weights(ONE, 0, 65536, 64, 2, 32, ONE, ONE, None) == -4
    plan = lib.Plan(M=4, N=8, K=2, D=72, H=32, reserved=0, rows_capacity=128 * 9, sched=16, tile_expert=16,
                    pad_off=16, row_token=16, row_weight=16, pos_MK=16, status=16, pair_info=16)
    p = C.byref(plan)
    assert L.momoe_fp8_up_swiglu(p, ONE, ONE, ONE, ONE, ONE, ONE, ONE, None) == -2    # D not a multiple of 16
    plan.D = 64
    def dispatch(x=ONE, M=4, N=8, K=2, D=64, rows=128 * 9, ws=ONE, n=None, dst=ONE):
        n = L.momoe_fp8_dispatch_workspace_bytes(M, N, K) if n is None else n
        return L.momoe_fp8_dispatch_rows(x, None, ONE, ONE, M, N, K, D, ONE, ONE, ONE, ONE, ONE, ONE, ONE, rows, ws, n, dst,
                                         ONE, ONE, None)
    assert dispatch(x=None) == -1 and dispatch(D=72) == -2 and dispatch(K=9) == -1 and dispatch(N=1025) == -4
    assert dispatch(N=40, K=33) == -4 and dispatch(rows=128 * 8) == -1 and dispatch(dst=ODD) == -1
    assert dispatch(M=20000, rows=1 << 20, n=8) == -1 and dispatch(M=20000, rows=1 << 20, ws=None) == -1
    assert dispatch(M=8 << 20, rows=1 << 40) == -4                               # more tiles than a table entry counts
    assert L.momoe_fp8_dispatch_workspace_bytes(4, 8, 2) == 0
    assert L.momoe_fp8_dispatch_workspace_bytes(20000, 8, 2) > 8 * 4
    for f in (L.momoe_fp8_up_swiglu, L.momoe_fp8_up_swiglu_decode):
        assert f(p, ONE, ONE, ONE, ONE, None, ONE, ONE, None) == -1 and f(p, ONE, ODD, ONE, ONE, ONE, ONE, ONE, None) == -1
        assert f(None, ONE, ONE, ONE, ONE, ONE, ONE, ONE, None) == -1
    for f in (L.momoe_fp8_down_scale, L.momoe_fp8_down_scale_decode):
        assert f(p, ONE, ONE, ONE, ONE, None, ONE, ONE, None) == -1 and f(p, ONE, ONE, ONE, ONE, ONE, None, ONE, None) == -1
        assert f(p, ONE, ONE, ONE, ONE, ONE, ONE, None, None) == -1 and f(p, ONE, ONE, ONE, ONE, ONE, ODD, ONE, None) == -1
    assert L.momoe_fp8_combine_rows(ONE, ONE, ONE, 4, 2, 60, ONE, None) == -2
    assert L.momoe_fp8_combine_rows(ONE, ONE, ONE, 4, 0, 64, ONE, None) == -1
    assert L.momoe_fp8_combine_rows(ODD, ONE, ONE, 4, 2, 64, ONE, None) == -1
    for f in (L.momoe_fp8_up_swiglu, L.momoe_fp8_up_swiglu_decode, L.momoe_fp8_down_scale, L.momoe_fp8_down_scale_decode):
        assert f(p, None, ONE, ONE, ONE, ONE, ONE, ONE, None) == -1
    def whole(M=4, N=8, K=2, D=64, H=32, x=ONE, ws=ONE, n=None):
        n = L.momoe_fp8_experts_workspace_bytes(M, N, K, D, H) if n is None else n
        return L.momoe_fp8_experts_forward(x, None, ONE, ONE, M, N, K, D, H, ONE, ONE, ONE, ONE, 16, ONE, ONE, ws, n, ONE,
                                           None)
    assert whole(D=40) == -2 and whole(H=24) == -2 and whole(M=0) == -1 and whole(n=100) == -1 and whole(ws=C.c_void_p(128)) == -1
    assert whole(x=None) == -1 and whole(K=9) == -1 and whole(N=1025) == -4
    assert L.momoe_fp8_experts_workspace_bytes(0, 8, 2, 64, 32) == 0


def test_there_is_no_cpu_path(lib):
    from momoe import balance, fp8, norm
    x, w = torch.zeros(4, 64), torch.ones(64)
    ids = torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: norm.rms_norm(x, w), lambda: norm.rms_norm_fp8(x, w), lambda: fp8.quantize_rows(x),
                 lambda: balance.balance_loss(x, ids), lambda: fp8.quantize_experts(torch.zeros(2, 64, 64), torch.zeros(2, 32, 64)),
                 lambda: norm.RMSNorm(64, device="cpu")(x.bfloat16())):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_row_numbers_stay_inside_32_bits(lib):
    """Kernels step past the last row before they compare, so the largest row counts are refused."""
    L, M = lib.lib, 2 ** 30 + 1
    assert L.momoe_rms_norm(ONE, 8, None, 0, ONE, 0, 0, M, 8, 1e-6, None, ONE, None, None, None, None) == -4
    assert L.momoe_rms_norm_backward(ONE, None, ONE, 8, ONE, ONE, 0, 0, M, 8, ONE, None, None, 0, None) == -4
    assert L.momoe_balance_loss(ONE, 0, ONE, None, M, M, 8, 2, 0, 1, 1.0, 0.0, ONE, ONE, ONE, ONE, 1 << 40, None) == -4
    assert L.momoe_balance_loss_backward(ONE, 0, None, M, ONE, M, 8, 0, 1, 0.0, ONE, None, ONE, None) == -4
