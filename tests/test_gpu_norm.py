"""The norm with the residual's addition against its formula in 64 bits, its gradient against the formula and against
differences, its 8-bit rows, odd layouts, and what it leaves alone.

Tolerances, u = 2^-24: a sum of up to 32 terms a thread, 5 + 16 partial sums, a division, a square root and a division
cost rstd at most 64 u; the products behind it a few u more: 2^-17 relative with room to spare.  Rounding to the output's
type adds half a step, eps / 2."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -17
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SHAPES = [(1, 8), (3, 136), (257, 1024), (5, 1032), (130, 2176), (1, 4096), (33, 4104), (7, 8192), (4, 8200), (2, 16384),
          (5000, 64), (1000, 2048), (400, 7176)]        # the last three: several rows for each group of the backward pass


@pytest.fixture(scope="module")
def norm():
    import __graft_entry__
    __graft_entry__.build()
    from momoe import norm
    return norm


def make(M, D, dtype, seed, residual=True, wtype=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    x, w = (r(M, D) * torch.exp(r(D))).to(dtype), (1 + 0.2 * r(D)).to(wtype or dtype)
    res = (2 * r(M, D)).to(dtype) if residual else None
    gy, gr = r(M, D).to(dtype), r(M, D).to(dtype)
    return [t.cuda() if t is not None else None for t in (x, w, res, gy, gr)]


def formula(x, w, res, eps):
    """r (rounded as the stream's type), rstd, xhat, y in 64 bits."""
    r = x if res is None else (x.float() + res.float()).to(x.dtype)
    v = r.double()
    rstd = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    return r, rstd, v * rstd, v * rstd * w.double()


def near(got, want, scale, what):
    """|got - want| <= eps / 2 |want| + F32 * scale; below the smallest normal number of the type half a step there."""
    f = torch.finfo(got.dtype)
    tol = f.eps / 2 * want.abs() + F32 * scale + f.tiny * f.eps / 2
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), "%s: %d values off, worst %g" % (what, int(bad.sum()), float((got.double() - want).abs().max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D", SHAPES)
def test_forward_and_gradient_against_the_formula(norm, M, D, dtype):
    for residual, wtype in ((True, None), (False, torch.float32)):
        x, w, res, gy, gr = make(M, D, dtype, M + D, residual, wtype)
        leaves = [t.clone().requires_grad_(True) if t is not None else None for t in (x, w, res)]
        out = norm.rms_norm(leaves[0], leaves[1], leaves[2], 1e-5)
        y, r = out if residual else (out, None)
        r64, rstd, xhat, y64 = formula(x, w, res, 1e-5)
        near(y, y64, y64.abs(), "y")
        if residual:
            assert torch.equal(r, r64)
        torch.autograd.backward([y, r] if residual else [y], [gy, gr] if residual else [gy])
        gh = gy.double() * w.double()
        gx = rstd * (gh - xhat * (gh * xhat).mean(1, keepdim=True))
        size = rstd * (gh.abs() + xhat.abs() * (gh * xhat).abs().mean(1, keepdim=True))
        if residual:
            gx, size = gx + gr.double(), size + gr.double().abs()
            near(leaves[2].grad, gx, size, "g residual")
            assert leaves[2].grad.data_ptr() != leaves[0].grad.data_ptr()
        near(leaves[0].grad, gx, size, "g x")
        # the sum over rows: at most M / 148 rows a group, then the groups, in u each
        terms = (gy.double() * xhat)
        near(leaves[1].grad, terms.sum(0), terms.abs().sum(0) * (1 + M / 148 / 128), "g w")


def test_gradient_against_differences(norm):
    x, w, res, gy, gr = make(6, 72, torch.float32, 3)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, res)]
    y, r = norm.rms_norm(*leaves, 1e-6)
    torch.autograd.backward([y, r], [gy, gr])
    def loss(x, w, res):
        v = x + res                                          # 64 bits: no rounding of the sum
        y = v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6) * w
        return (y * gy.double()).sum() + (v * gr.double()).sum()
    g = torch.Generator().manual_seed(9)
    for i in range(3):
        args = [t.double() for t in (x, w, res)]
        d = torch.randn(args[i].shape, generator=g).double().cuda()
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + 1e-5 * d, args[i] - 1e-5 * d
        slope = float((loss(*up) - loss(*down)) / 2e-5)
        # the kernel rounds the sum of x and residual to 32 bits: 2^-24 relative in each value, 2^-17 in sums of 432 terms
        assert abs(slope - float((leaves[i].grad.double() * d).sum())) <= 2.0 ** -15 * float((leaves[i].grad.double() * d).abs().sum())


@pytest.mark.parametrize("M,D,dtype", [(1, 16, torch.bfloat16), (5, 144, torch.float32), (300, 2048, torch.bfloat16),
                                       (3, 7168, torch.float16), (2, 16384, torch.bfloat16), (1, 8, torch.bfloat16)])
def test_eight_bit_rows(norm, M, D, dtype):
    x, w, res, _, _ = make(M, D, dtype, 5)
    w[D // 2:D // 2 + 8] = 0
    if D > 128:
        w[:128] = 0                                          # a block of zeros
    out = norm.rms_norm_fp8(x, w, res, 1e-5)
    r64, _, _, y64 = formula(x, w, res, 1e-5)
    y, r = norm.rms_norm(x, w, res, 1e-5)
    assert torch.equal(out.y, y) and torch.equal(out.residual, r)
    check_rows(out.rows, y64, F32)


def check_rows(rows, want, rel):
    """8-bit rows against 64-bit values that the kernel had up to a relative error `rel`."""
    M, D = want.shape
    scale = rows.scale.double()
    assert scale.shape == (M, -(-D // 128)) and rows.q.shape == (M, D)
    top = torch.nn.functional.pad(want.abs(), (0, -D % 128)).view(M, -1, 128).amax(2)
    zero = top == 0
    assert (scale[zero] == 1).all()
    assert (top[~zero] <= 448 * scale[~zero] * (1 + rel)).all() and (top[~zero] > 224 * scale[~zero] * (1 - rel)).all()
    wide = scale.repeat_interleave(128, 1)[:, :D]
    # e4m3 is off by half a step: 2^-4 relative, 2^-10 of the scale below 2^-6 of it
    tol = torch.maximum(want.abs() * 2.0 ** -4, wide * 2.0 ** -10) + rel * want.abs()
    assert ((rows.q.double() * wide - want).abs() <= tol).all()


def test_no_rounding_of_y_before_the_eight_bit_rows(norm):
    """A value whose bfloat16 rounding crosses a border of e4m3 shows which of the two the rows were made from."""
    x = torch.full((1, 128), 1.0, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(128, dtype=torch.float32, device="cuda")
    w[1] = 1.0625 + 2.0 ** -12        # just above the middle of 1 and 1.125; bfloat16 rounds it to the middle (tie: 1.0)
    out = norm.rms_norm_fp8(x, w, None, 0.0)
    scale = float(out.rows.scale.float()[0, 0])
    assert float(out.y[0, 1]) == 1.0625 and float(out.rows.q.float()[0, 1]) * scale == 1.125


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_views_and_other_streams(norm, dtype):
    x, w, res, gy, _ = make(40, 512, dtype, 1)
    want = norm.rms_norm(x[:, :256].contiguous(), w[:256].contiguous(), res[:, 256:].contiguous())
    for a, b in ((x[:, :256], res[:, 256:]), (x[:, :256].t().contiguous().t(), res[:, 256:].clone())):
        got = norm.rms_norm(a, w[:256], b)
        assert all(torch.equal(p, q) for p, q in zip(want, got))
    odd = torch.empty(40 * 256 + 1, dtype=dtype, device="cuda")[1:].view(40, 256).copy_(x[:, :256])   # not 16-byte aligned
    got = norm.rms_norm(odd, w[:256], res[:, 256:])
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    got = norm.rms_norm(x[:, :256].reshape(2, 4, 5, 256), w[:256], res[:, 256:].reshape(2, 4, 5, 256))
    assert got[0].shape == (2, 4, 5, 256) and torch.equal(got[0].view(40, 256), want[0])
    # a broadcast gradient and a strided input under autograd
    a = x[::2, :256].detach().requires_grad_(True)
    y = norm.rms_norm(a, w[:256])
    y.sum().backward()
    b = x[::2, :256].contiguous().requires_grad_(True)
    norm.rms_norm(b, w[:256]).backward(torch.ones(20, 256, dtype=dtype, device="cuda"))
    assert torch.equal(a.grad, b.grad)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = norm.rms_norm(x[:, :256], w[:256], res[:, 256:])
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_partial_gradients_empty_input_and_bad_values(norm):
    x, w, res, gy, gr = make(9, 264, torch.bfloat16, 2)
    # only the sum is used, only the norm is used, only the weight learns
    a, v = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y, r = norm.rms_norm(a, v, res)
    gx, gw = torch.autograd.grad(r, (a, v), gr, allow_unused=True)
    assert torch.equal(gx, gr) and (gw is None or not gw.any())
    y, r = norm.rms_norm(x, v, res)
    gw, = torch.autograd.grad(y, v, gy)
    y, r = norm.rms_norm(a, v, res)
    full = torch.autograd.grad((y, r), (a, v), (gy, torch.zeros_like(gr)))
    assert torch.equal(gw, full[1])
    alone = torch.autograd.grad(norm.rms_norm(a, v, res)[0], a, gy)[0]
    assert torch.equal(alone, full[0])
    e = torch.empty(0, 264, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = norm.rms_norm(e, v)
    ge, gw = torch.autograd.grad(y, (e, v), torch.empty_like(y))
    assert y.shape == (0, 264) and ge.shape == (0, 264) and not gw.any()
    assert norm.rms_norm_fp8(e.detach(), w).rows.q.shape == (0, 264)
    # a NaN and an infinity stay in their rows; zeros are normed to zeros
    x[2, 5], x[4, 200], x[6] = float("nan"), float("inf"), 0
    res[6] = 0
    out = norm.rms_norm_fp8(x, w, res)
    good = [i for i in range(9) if i not in (2, 4)]
    assert torch.isfinite(out.y[good]).all() and torch.isnan(out.y[2]).all() and torch.isnan(out.y[4, 200])
    assert not out.y[6].any() and (out.rows.scale.float()[6] == 1).all() and not out.rows.q.float()[6].any()
    assert torch.isnan(out.rows.scale.float()[2]).all() and torch.isfinite(out.rows.scale.float()[good]).all()


def test_same_result_twice_and_from_a_captured_graph(norm):
    x, w, res, gy, gr = make(3001, 640, torch.bfloat16, 8)
    def step(x):
        a, v, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True), res.detach().requires_grad_(True)
        y, r = norm.rms_norm(a, v, b)
        return (y, r) + torch.autograd.grad((y, r), (a, v, b), (gy, gr))
    want = step(x)
    assert all(torch.equal(p, q) for p, q in zip(want, step(x)))
    buf = torch.zeros_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(buf)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(buf)
    buf.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, out))


def test_refusals(norm):
    x, w, res, _, _ = make(4, 64, torch.bfloat16, 0)
    for bad in (lambda: norm.rms_norm(x[:, :60], w[:60]), lambda: norm.rms_norm(x, w[:32]), lambda: norm.rms_norm(x, w.half()),
                lambda: norm.rms_norm(x, w, res[:2]), lambda: norm.rms_norm(x, w, res.float()),
                lambda: norm.rms_norm(x.double(), w.double()), lambda: norm.rms_norm(x, w.cpu()),
                lambda: norm.rms_norm(torch.zeros(1, 16392, device="cuda"), torch.zeros(16392, device="cuda")),
                lambda: norm.rms_norm_fp8(x, w.requires_grad_(True)),
                lambda: norm.rms_norm(x, w.detach(), eps=-1.0)):
        with pytest.raises(RuntimeError):
            bad()
