"""8-bit experts whose blocks are of very unlike size: blocks of zeros, columns far above their neighbours, columns that
are not finite.  A result row is kept as fp16 with one power of two for each 256 columns, so what its largest value is
taken from decides what is left of the others."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# tokens, and the most rows an expert for which the streaming form is used: streaming, a tile for a thread block, pairs
FORMS = [(50, 2 ** 20), (50, 0), (900, 0)]


@pytest.fixture(scope="module")
def fp8():
    import __graft_entry__
    __graft_entry__.build()
    from momoe import fp8
    return fp8


def inputs(M, N, D, H, size, std, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    x = (size * r(M, D)).bfloat16().cuda()
    idx = torch.stack([torch.randperm(N, generator=g)[:1] for _ in range(M)]).int().cuda()
    w = (0.1 + torch.rand(M, 1, generator=g)).cuda()
    return x, idx, w, (std * r(N, D, 2 * H)).bfloat16().cuda(), (std * r(N, H, D)).bfloat16().cuda()


def spread(W1, W2, at, zero, seed):
    """The layer's hidden channels in blocks of 128 at new places: block i of the result is block at[i], or (None) one whose
    up and gate columns (zero = "W1"), down rows ("W2") or both are zeros, the others as in any layer."""
    N, D, H = W1.shape[0], W1.shape[1], W2.shape[1]
    g = torch.Generator().manual_seed(seed)
    n = 128 * len(at)
    U = (torch.randn(N, D, 2, n, generator=g) * float(W1.float().std())).bfloat16().cuda()
    V = (torch.randn(N, n, D, generator=g) * float(W2.float().std())).bfloat16().cuda()
    halves = W1.view(N, D, 2, H)
    for i, b in enumerate(at):
        new = slice(128 * i, 128 * i + 128)
        if b is None:
            if zero != "W2":
                U[..., new] = 0
            if zero != "W1":
                V[:, new] = 0
        else:
            k = min(128, H - 128 * b)
            U[..., new], V[:, new] = 0, 0
            U[..., 128 * i:128 * i + k] = halves[..., 128 * b:128 * b + k]
            V[:, 128 * i:128 * i + k] = W2[:, 128 * b:128 * b + k]
    return U.reshape(N, D, 2 * n).contiguous(), V


@pytest.mark.parametrize("zero", ["both", "W1", "W2"])
@pytest.mark.parametrize("M,stream", FORMS)
def test_blocks_of_zeros_change_nothing(fp8, monkeypatch, M, stream, zero):
    """Hidden channels that contribute nothing add zeros to the accumulators, which is exact: the same bits, at any size of
    the rows and weights."""
    monkeypatch.setattr(fp8, "STREAM_MAX_AVG_ROWS", stream)
    for D, H, at in ((512, 384, (0, None, 1, None, 2)), (400, 144, (0, 1, None)), (272, 128, (None, None, None, None, 0))):
        for size, std in ((1.0, 0.02), (0.1, 0.02), (0.03, 0.02), (1.0, 0.002)):
            x, idx, w, W1, W2 = inputs(M, 4, D, H, size, std, H)
            want, _ = fp8.experts_forward(x, idx, w, fp8.quantize_experts(W1, W2))
            assert (want != 0).float().mean() > 0.99
            got, _ = fp8.experts_forward(x, idx, w, fp8.quantize_experts(*spread(W1, W2, at, zero, 1)))
            assert torch.equal(got, want), (D, size, std, float((got.double() - want.double()).norm() / want.double().norm()))


@pytest.mark.parametrize("M,stream", FORMS)
@pytest.mark.parametrize("exponent", [20, 28])
def test_columns_beside_much_larger_ones(fp8, monkeypatch, M, stream, exponent):
    """128 columns that share a power of two with larger ones.  With L the largest value of the 256, stored as 2^13 at least,
    the smallest step of fp16, 2^-24, is off by 2^-38 L at most; else each of the two runs has an fp16 (2^-11) and a bfloat16
    (2^-8) rounding."""
    monkeypatch.setattr(fp8, "STREAM_MAX_AVG_ROWS", stream)
    x, idx, w, W1, W2 = inputs(M, 4, 400, 256, 1.0, 0.05, 3)
    want = fp8.experts_forward(x, idx, w, fp8.quantize_experts(W1, W2))[0].double()
    for large, small in ((slice(0, 128), slice(128, 256)), (slice(128, 256), slice(0, 128)), (slice(256, 384), slice(384, 400))):
        W = W2.float()
        W[:, :, large] *= 2.0 ** exponent
        got = fp8.experts_forward(x, idx, w, fp8.quantize_experts(W1, W))[0].double()
        L = got[:, large].abs().amax(1, keepdim=True) * (1 + 2.0 ** -7)
        off = (got[:, small] - want[:, small]).abs()
        assert (off <= (2.0 ** -7 + 2.0 ** -10) * want[:, small].abs() + 2.0 ** -38 * L).all(), float((off / L).max())
        assert torch.equal(got[:, large], want[:, large] * 2.0 ** exponent)


@pytest.mark.parametrize("M,stream", FORMS)
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_bad_weight_spoils_its_own_columns_only(fp8, monkeypatch, M, stream, bad):
    """The block that holds it is NaN; the 128 columns beside it keep their values (two runs, an fp16 and a bfloat16 rounding
    each, the fp16 one off by 2^-38 of the largest for small values)."""
    monkeypatch.setattr(fp8, "STREAM_MAX_AVG_ROWS", stream)
    x, idx, w, W1, W2 = inputs(M, 4, 512, 256, 1.0, 0.05, 4)
    want = fp8.experts_forward(x, idx, w, fp8.quantize_experts(W1, W2))[0].double()
    W = W2.clone()
    W[2, 130, 140] = bad
    got = fp8.experts_forward(x, idx, w, fp8.quantize_experts(W1, W))[0].double()
    here = idx[:, 0] == 2
    assert torch.isnan(got[here][:, 128:256]).all() and torch.equal(got[~here], want[~here])
    beside = torch.cat([got[here][:, :128], got[here][:, 256:]], 1)
    ref = torch.cat([want[here][:, :128], want[here][:, 256:]], 1)
    L = want[here].abs().amax(1, keepdim=True) * (1 + 2.0 ** -7)
    assert ((beside - ref).abs() <= (2.0 ** -7 + 2.0 ** -10) * ref.abs() + 2.0 ** -38 * L).all()
