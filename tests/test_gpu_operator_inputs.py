"""What callers hand to the operators around the expert layer besides the usual tensors."""
import pytest
import torch

pytestmark = pytest.mark.gpu

WHOLE = [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.uint32, torch.int64]


@pytest.fixture(scope="module")
def momoe():
    import __graft_entry__
    __graft_entry__.build()
    import momoe
    import momoe.balance
    import momoe.fp8
    import momoe.norm
    return momoe


def top(dtype):
    return min(torch.iinfo(dtype).max, 2 ** 31 - 1)


@pytest.mark.parametrize("dtype", WHOLE)
@pytest.mark.parametrize("N", [8, 130, 300])
def test_ids_and_bounds_of_every_whole_type(momoe, dtype, N):
    """Narrow types hold neither -1 nor N nor M: the limits must not be formed in them."""
    g = torch.Generator().manual_seed(N)
    M = 600
    ids = torch.stack([torch.randperm(min(N, top(dtype) + 1), generator=g)[:3] for _ in range(M)]).int().cuda()
    logits = torch.randn(M, N, generator=g).cuda()
    cu = torch.tensor([0, 5, 90, 127], dtype=torch.int32, device="cuda")

    def both(ids, cu):
        leaf = logits.clone().requires_grad_(True)
        loss, counts = momoe.balance.balance_loss(leaf, ids, 0, 0.5, 0.1, cu_seqlens=cu)
        return loss.detach(), counts, torch.autograd.grad(loss, leaf)[0]
    want = both(ids, cu)
    assert int(want[1].sum()) == 127 * 3
    assert all(torch.equal(a, b) for a, b in zip(both(ids.to(dtype), cu), want))
    assert all(torch.equal(a, b) for a, b in zip(both(ids, cu.to(dtype)), want))
    if torch.iinfo(dtype).min < 0:
        out = ids.clone()
        out[3] = -1
        assert all(torch.equal(a, b) for a, b in zip(both(out.to(dtype), cu), both(out, cu)))


@pytest.mark.parametrize("dtype", WHOLE)
def test_expert_ids_of_every_whole_type(momoe, dtype):
    from momoe import ops
    g = torch.Generator().manual_seed(0)
    for N in (8, 300):
        e = momoe.fp8.quantize_experts(torch.randn(N, 64, 64, generator=g).cuda() * 0.1, torch.randn(N, 32, 64, generator=g).cuda() * 0.1)
        ids = torch.stack([torch.randperm(min(N, top(dtype) + 1), generator=g)[:2] for _ in range(40)]).int().cuda()
        x, w = torch.randn(40, 64, generator=g).bfloat16().cuda(), torch.rand(40, 2, generator=g).cuda()
        want = momoe.fp8.experts_forward(x, ids, w, e)
        got = momoe.fp8.experts_forward(x, ids.to(dtype), w, e)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        ops.check_status()


def test_tangents_are_refused(momoe):
    """Forward-mode gradients: none of the operators has them, and none drops them."""
    from torch.autograd import forward_ad
    x, w = torch.randn(6, 64, device="cuda"), torch.ones(64, device="cuda")
    e = momoe.fp8.quantize_experts(torch.randn(4, 64, 64, device="cuda"), torch.randn(4, 32, 64, device="cuda"))
    ids, top = torch.zeros(6, 2, dtype=torch.int32, device="cuda"), torch.rand(6, 2, device="cuda")
    ids[:, 1] = 1
    moe = momoe.MoE(64, 32, 4, 2, 0)
    moe.quantize_experts()
    calls = [lambda: momoe.norm.rms_norm(x, w), lambda: momoe.norm.rms_norm(x, w, x), lambda: momoe.norm.rms_norm_fp8(x, w),
             lambda: momoe.fp8.experts_forward(x.bfloat16(), ids, top, e), lambda: momoe.balance.balance_loss(x, ids)]
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for f in (lambda: momoe.norm.rms_norm(dual(x), w), lambda: momoe.norm.rms_norm(x, dual(w)),
                          lambda: momoe.norm.rms_norm(x, w, dual(x)), lambda: momoe.norm.rms_norm_fp8(dual(x), w),
                          lambda: momoe.fp8.experts_forward(dual(x.bfloat16()), ids, top, e),
                          lambda: momoe.fp8.experts_forward(x.bfloat16(), ids, dual(top), e),
                          lambda: momoe.balance.balance_loss(dual(x), ids)):
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        f()
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            moe(dual(x.bfloat16()[None]))
        for f in calls:                                     # nothing to lose: inside a level, without tangents
            f()


@pytest.mark.parametrize("bounds", [[0, 30, 20, 50], [10, 5], [60, 0], [0, 60, 59], [0, 60, 0, 60, 0, 60], [7] + list(range(600, 0, -1))])
def test_bounds_that_do_not_ascend_give_nan(momoe, bounds):
    """Not numbers from whatever the workspace held."""
    g = torch.Generator().manual_seed(1)
    M = 700
    logits, ids = torch.randn(M, 40, generator=g).cuda(), torch.randint(0, 40, (M, 2), generator=g).int().cuda()

    def run(bounds):
        leaf = logits.clone().requires_grad_(True)
        cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")
        loss, counts = momoe.balance.balance_loss(leaf, ids, 0, 0.5, 0.1, cu_seqlens=cu)
        return loss.detach(), counts, torch.autograd.grad(loss, leaf)[0]
    want = run([0, 20, 700])
    loss, counts, grad = run(bounds)
    assert torch.isnan(loss) and not counts.any()
    inside = torch.zeros(M, dtype=torch.bool, device="cuda")
    inside[bounds[0]:bounds[-1]] = True
    assert torch.isnan(grad[inside]).all() and not grad[~inside].any()
    assert all(torch.equal(a, b) for a, b in zip(run([-3, 20, 701]), want))    # outside [0, M]: as 0 and M
    assert all(torch.equal(a, b) for a, b in zip(run([0, 20, 700]), want))


def test_status_is_cleared_outside_of_the_mode_it_was_first_used_in(momoe, monkeypatch):
    from momoe import ops
    monkeypatch.setattr(ops, "_status_words", {})
    monkeypatch.setattr(ops, "_status_reports", {})
    with torch.inference_mode():
        e = momoe.fp8.quantize_experts(torch.randn(4, 64, 64, device="cuda"), torch.randn(4, 32, 64, device="cuda"))
        x, w = torch.randn(3, 64, device="cuda").bfloat16(), torch.ones(3, 1, device="cuda")
        momoe.fp8.experts_forward(x, torch.full((3, 1), 4, device="cuda"), w, e)
        ops.status_post("cuda")
    with pytest.raises(RuntimeError, match="202"):
        ops.check_status()
    ops.check_status()
    momoe.fp8.experts_forward(x, torch.full((3, 1), 4, device="cuda"), w, e)
    ops.status_post("cuda")
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="202"):
        ops.status_poll("cuda")
    ops.check_status()


def test_layer_made_in_inference_mode(momoe):
    """Its parameters have no version counter; swapped ones are noticed all the same."""
    x = torch.randn(1, 5, 64, device="cuda").bfloat16()
    with torch.inference_mode():
        moe = momoe.MoE(64, 32, 4, 2, 0)
        moe.quantize_experts()
        bias = moe.biases_N.clone()
        want = moe(x)
        moe.biases_N.copy_(bias)
        assert torch.equal(moe(x), want)
        moe.momoe.Wl2_NHD = torch.nn.Parameter(moe.momoe.Wl2_NHD.clone(), requires_grad=False)
        with pytest.raises(RuntimeError, match="changed"):
            moe(x)
        moe.quantize_experts()
        moe.biases_N.copy_(bias)
        assert torch.equal(moe(x), want)


def test_eight_bit_weights_set_by_hand_after_others(momoe):
    """Ones that replace stale ones are the caller's; the stale ones stay refused, in copies as well."""
    import copy
    import io

    def saved(layer):
        file = io.BytesIO()
        torch.save(layer, file)
        file.seek(0)
        return torch.load(file, weights_only=False)
    x = torch.randn(1, 5, 64, device="cuda").bfloat16()
    with torch.no_grad():
        moe = momoe.MoE(64, 32, 4, 2, 0)
        moe.quantize_experts()
        old = moe.experts_fp8
        moe.momoe.Wl1_ND2H.mul_(0.5)
        with pytest.raises(RuntimeError, match="changed"):
            moe(x)
        for twin in (copy.deepcopy(moe), saved(moe)):
            with pytest.raises(RuntimeError, match="changed"):
                twin(x)
        moe.experts_fp8 = momoe.fp8.quantize_experts(moe.momoe.Wl1_ND2H, moe.momoe.Wl2_NHD)
        bias = moe.biases_N.clone()
        want = moe(x)
        for twin in (copy.deepcopy(moe), saved(moe)):
            twin.biases_N.copy_(bias)
            assert torch.equal(twin(x), want)
        moe.experts_fp8 = None
        moe(x)
        moe.momoe.Wl1_ND2H.mul_(2)
        moe.experts_fp8 = old
        moe(x)
        moe.momoe.Wl1_ND2H.mul_(2)
        with pytest.raises(RuntimeError, match="changed"):
            moe(x)


def test_stale_eight_bit_weights_in_a_saved_state(momoe):
    x = torch.randn(1, 5, 64, device="cuda").bfloat16()
    with torch.no_grad():
        moe = momoe.MoE(64, 32, 4, 2, 0)
        moe.quantize_experts()
        state = dict(moe.__getstate__(), _fp8_weights=())
        moe.__setstate__(state)
        with pytest.raises(RuntimeError, match="changed"):
            moe(x)
        moe.quantize_experts()
        moe(x)


def test_eight_bit_weights_are_freed_when_they_are_given_up(momoe):
    with torch.no_grad():
        moe = momoe.MoE(256, 128, 16, 2, 0)
        x = torch.randn(1, 5, 256, device="cuda").bfloat16()
        moe(x)
        before = torch.cuda.memory_allocated()
        moe.quantize_experts()
        moe(x)
        size = sum(t.numel() for t in moe.experts_fp8)
        assert torch.cuda.memory_allocated() >= before + size
        moe.quantize_experts()
        moe(x)
        assert torch.cuda.memory_allocated() < before + 2 * size
        moe.experts_fp8 = None
        assert torch.cuda.memory_allocated() < before + size
