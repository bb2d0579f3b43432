"""Balance loss, z-loss and counts against their definitions in 64 bits, the gradient against the formula and against
differences, at the sequences and masks where they can go wrong.

Tolerances, u = 2^-24: every sum has terms of one sign, so a relative error of u for each addition of a chain (at most a
few hundred here: 2^-16) plus the exponential's (2^-19 at logits 30 apart) bounds the loss at 2^-15; the gradient
p (g - sum g p + z) is bounded against the sum of its terms' magnitudes, plus half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -15


@pytest.fixture(scope="module")
def balance():
    import __graft_entry__
    __graft_entry__.build()
    from momoe import balance
    return balance


def make(M, N, K, Ks, seed, dtype, masked=0.05):
    g = torch.Generator().manual_seed(seed)
    logits = 2 * torch.randn(M, N, generator=g)
    Ng = N - Ks
    logits[:, :Ng] = logits[:, :Ng].masked_fill(torch.rand(M, Ng, generator=g) < masked, float("-inf"))
    idx = torch.rand(M, Ng, generator=g).topk(K - Ks).indices
    idx = torch.cat([idx, torch.arange(Ng, N).expand(M, Ks)], 1).int()
    return logits.to(dtype).cuda(), idx.cuda()


def definition(logits, idx, Ks, bc, zc, bounds):
    """loss, counts, gradient, and the magnitudes that bound the gradient's error; 64 bits."""
    M, N = logits.shape
    K, Ng = idx.shape[1], N - Ks
    lens = [b - a for a, b in zip(bounds, bounds[1:])]
    n_seq, T = max(1, sum(n > 0 for n in lens)), max(1, sum(lens))
    loss = torch.zeros((), dtype=torch.float64, device=logits.device)
    grad, size = torch.zeros(M, N, dtype=torch.float64, device=logits.device), torch.zeros(M, N, dtype=torch.float64, device=logits.device)
    counts = torch.zeros(len(lens), N, dtype=torch.long, device=logits.device)
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        rows = slice(bounds[b], bounds[b + 1])
        ids = idx[rows].flatten().long()
        counts[b] = torch.bincount(ids[(ids >= 0) & (ids < N)], minlength=N)
        z = logits[rows, :Ng].double()
        lse = torch.logsumexp(z, 1)
        dead = torch.isneginf(lse)
        p = torch.softmax(z, 1).masked_fill(dead[:, None], 0)
        lse = lse.masked_fill(dead, 0)
        f = counts[b, :Ng].double() * Ng / ((K - Ks) * n)
        loss += bc / n_seq * (f * p.mean(0)).sum() + zc / T * (lse ** 2).sum()
        g, zt = bc / (n_seq * n) * f, (2 * zc / T * lse)[:, None]
        dot = (p @ g)[:, None]
        grad[rows, :Ng] = p * (g - dot + zt)
        size[rows, :Ng] = p * (abs(g) + abs(dot) + abs(zt))
    return loss, counts, grad, size


def check(balance, logits, idx, Ks, bc, zc, bounds, up=1.75, **kw):
    leaf = logits.clone().requires_grad_(True)
    loss, counts = balance.balance_loss(leaf, idx, Ks, bc, zc, **kw)
    want, c, grad, size = definition(logits, idx, Ks, bc, zc, bounds)
    assert loss.dtype == torch.float32 and loss.shape == () and counts.dtype == torch.int64
    assert torch.equal(counts, c)
    assert abs(float(loss.detach()) - float(want)) <= F32 * abs(float(want)), (float(loss.detach()), float(want))
    got, = torch.autograd.grad(loss, leaf, torch.tensor(up, device="cuda"))
    assert got.dtype == logits.dtype
    f = torch.finfo(got.dtype)
    off = (got.double() - up * grad).abs()
    assert (off <= f.eps / 2 * (up * grad).abs() + F32 * up * size + f.tiny * f.eps / 2).all(), float((off / (up * size).clamp(min=1e-300)).max())
    return loss, counts, got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K,Ks", [(1, 2, 1, 0), (7, 8, 2, 0), (130, 31, 3, 1), (64, 33, 2, 0), (515, 64, 4, 2),
                                      (1024, 100, 8, 4), (2047, 128, 8, 0), (333, 130, 5, 0), (900, 256, 8, 1),
                                      (77, 384, 6, 0), (50, 601, 9, 3), (40, 1000, 32, 0), (20, 1024, 8, 7)])
def test_one_sequence_and_even_sequences(balance, M, N, K, Ks, dtype):
    logits, idx = make(M, N, K, Ks, M + N, dtype)
    check(balance, logits, idx, Ks, 0.3, 0.02, [0, M])
    S = max(1, M // 3)
    check(balance, logits, idx, Ks, 0.3, 0.0, list(range(0, M, S)) + [M], seq_len=S)
    check(balance, logits, idx, Ks, 0.0, 1.0, [0, M], seq_len=10 ** 12)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bounds", [[0, 0, 5, 5, 6, 300, 300], [3, 40, 41, 260], [0, 0], [300, 300], [0, 300], [10, 11],
                                    [0, 16, 32, 48, 300], list(range(0, 301, 2))])
def test_packed_sequences_with_padding_nobody_wrote(balance, bounds, dtype):
    logits, idx = make(300, 96, 6, 2, 4, dtype)
    logits[:bounds[0]] = float("nan")
    logits[bounds[-1]:] = float("nan")
    idx[bounds[-1]:] = 2 ** 31 - 1
    if bounds[-1] > bounds[0]:
        logits[bounds[0], :94] = float("-inf")               # every expert masked: the row counts for nothing
    for cu in (torch.tensor(bounds, dtype=torch.int32, device="cuda"), torch.tensor(bounds, device="cuda")):
        _, _, g = check(balance, logits, idx, 2, 0.5, 0.1, bounds, cu_seqlens=cu)
        assert not g[:, 94:].any() and not g[:bounds[0]].any() and not g[bounds[-1]:].any()


def test_many_rows_many_sequences_twice_the_same(balance):
    logits, idx = make(40001, 160, 8, 0, 11, torch.bfloat16)
    g = torch.Generator().manual_seed(1)
    bounds = [0] + torch.randint(0, 39000, (700,), generator=g).sort().values.tolist() + [39000]
    cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    a = check(balance, logits, idx, 0, 0.01, 0.001, bounds, cu_seqlens=cu)
    b = check(balance, logits, idx, 0, 0.01, 0.001, bounds, cu_seqlens=cu)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_as_many_sequences_as_rows(balance):
    logits, idx = make(9001, 24, 2, 0, 13, torch.bfloat16)
    check(balance, logits, idx, 0, 0.4, 0.2, list(range(9002)), seq_len=1)


def test_even_routing_gives_the_coefficient_and_ids_outside_are_not_counted(balance):
    logits = torch.zeros(64, 16, dtype=torch.bfloat16, device="cuda")
    idx = (torch.arange(64)[:, None] * 2 + torch.arange(2)).remainder(16).int().cuda()
    loss, counts = balance.balance_loss(logits, idx, 0, 0.25)
    assert float(loss) == pytest.approx(0.25, rel=F32) and (counts == 8).all()
    idx[0], idx[1, 0] = -1, 16
    check(balance, logits, idx, 0, 0.25, 0.1, [0, 64])
    check(balance, logits, idx.long() + 2 ** 32 * (idx < 0), 0, 0.25, 0.1, [0, 64])      # wide ids are not wrapped around
    idx[5] = 3                                               # the same expert twice counts twice
    check(balance, logits, idx, 0, 0.25, 0.1, [0, 64])


def test_gradient_against_differences(balance):
    logits, idx = make(24, 20, 3, 0, 6, torch.float32, masked=0)
    leaf = logits.clone().requires_grad_(True)
    loss, _ = balance.balance_loss(leaf, idx, 0, 0.7, 0.3, seq_len=9)
    loss.backward()
    g = torch.Generator().manual_seed(2)
    for _ in range(4):
        d = torch.randn(24, 20, generator=g).double().cuda()
        f = lambda t: definition(logits.double() + t * d, idx, 0, 0.7, 0.3, [0, 9, 18, 24])[0]
        slope = float((f(1e-5) - f(-1e-5)) / 2e-5)
        assert abs(slope - float((leaf.grad.double() * d).sum())) <= F32 * float((leaf.grad.double() * d).abs().sum()) + 1e-9


def test_bad_values_stay_in_their_rows_and_strided_logits(balance):
    logits, idx = make(50, 72, 4, 0, 7, torch.float32)
    wide = torch.full((50, 100), 9.0, device="cuda")
    wide[:, 1:73] = logits
    a = check(balance, wide[:, 1:73], idx, 0, 0.5, 0.1, [0, 50])
    b = check(balance, logits, idx.flip(0).flip(0), 0, 0.5, 0.1, [0, 50])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    logits[7, 3] = float("nan")
    leaf = logits.clone().requires_grad_(True)
    loss, _ = balance.balance_loss(leaf, idx, 0, 0.5, 0.1)
    loss.backward()
    assert torch.isnan(loss) and torch.isnan(leaf.grad[7]).any()
    assert torch.isfinite(leaf.grad[[i for i in range(50) if i != 7]]).all()


def test_capture_empty_batch_and_refusals(balance):
    logits, idx = make(600, 64, 4, 0, 8, torch.bfloat16)
    def step(x):
        leaf = x.detach().requires_grad_(True)
        loss, counts = balance.balance_loss(leaf, idx, 0, 0.5, 0.1, seq_len=100)
        return loss, counts, torch.autograd.grad(loss, leaf)[0]
    want = step(logits)
    buf = torch.zeros_like(logits)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(buf)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(buf)
    for _ in range(2):
        buf.copy_(logits)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, out))
    loss, counts = balance.balance_loss(logits[:0].detach().requires_grad_(True), idx[:0], 0, 1.0)
    assert float(loss) == 0 and counts.shape == (1, 64) and not counts.any()
    loss.backward()
    cu = torch.tensor([0, 600], device="cuda")
    for bad in (lambda: balance.balance_loss(logits.half(), idx), lambda: balance.balance_loss(logits, idx[:5]),
                lambda: balance.balance_loss(logits, idx, 4), lambda: balance.balance_loss(logits, idx, -1),
                lambda: balance.balance_loss(logits, idx, cu_seqlens=cu, seq_len=3),
                lambda: balance.balance_loss(logits, idx, cu_seqlens=cu[:1]), lambda: balance.balance_loss(logits, idx, seq_len=0),
                lambda: balance.balance_loss(logits, idx, cu_seqlens=cu.float()), lambda: balance.balance_loss(logits.cpu(), idx),
                lambda: balance.balance_loss(torch.zeros(2, 1032, device="cuda"), idx[:2])):
        with pytest.raises(RuntimeError):
            bad()
