"""8-bit rows, 8-bit weights and the experts' forward pass on them, stage by stage against 64 bits.

Each stage is fed what the previous kernel wrote, so that a value next to a border of e4m3 cannot blur the next stage.
Tolerances: a product of two e4m3 values and powers of two is exact in 32 bits; the tensor core adds 32 of them and the
accumulator at a time, at most 2^-21 of the sum of magnitudes an addition, over at most 4096 / 32 additions: 2^-14.
exp and the division of the activation: 2^-20 relative.  e4m3 is off by half a step (2^-4 relative, 2^-10 of the scale
below 2^-6 of it), bfloat16 by 2^-8 relative."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ACC = 2.0 ** -14
# M, N, K, D, H, skew
SHAPES = [
    (1, 8, 2, 64, 32, 0.0),
    (1, 128, 8, 2048, 768, 0.0),
    (5, 4, 4, 16, 16, 0.0),           # smaller than one block in every axis; every expert sees every token
    (37, 6, 3, 144, 272, 0.0),        # ragged in both widths
    (70, 2, 1, 512, 640, 0.0),        # more than one 32-row block
    (300, 4, 2, 528, 400, 1.0),
    (900, 4, 1, 656, 400, 0.5),       # enough rows an expert for pairs of tiles
    (1000, 16, 4, 640, 1152, 2.0),    # skewed: empty experts, experts of many tiles
    (257, 3, 1, 2176, 128, 0.0),
    (129, 1, 1, 128, 4096, 0.0),
    (640, 5, 3, 4096, 48, 0.0),
    (90, 40, 6, 256, 144, 3.0),       # few rows on average, some experts with several 32-row blocks
    (1400, 1000, 3, 64, 32, 1.0),     # many experts
    (50, 24, 13, 144, 64, 0.5),       # more experts a token than the weighted sum reads at once
    (33, 9, 7, 272, 48, 0.0),
    (40, 4, 2, 2576, 1680, 0.5),      # so few items that two thread blocks share an item's k axis, in both GEMMs
    (6000, 40, 3, 96, 64, 1.0),       # more pairs than one launch dispatches
]


@pytest.fixture(scope="module")
def fp8():
    import __graft_entry__
    __graft_entry__.build()
    from momoe import fp8
    return fp8


def rows_of(v):
    """Values in 64 bits -> codes and scales by the definition."""
    C = v.shape[-1]
    top = torch.nn.functional.pad(v.abs(), (0, -C % 128)).unflatten(-1, (-1, 128)).amax(-1)
    m, x = torch.frexp(top / 448)
    e = torch.where(m > 0.5, x, x - 1)
    scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), e), 1.0)
    scale = torch.where(torch.isfinite(top), scale, float("nan"))
    return (v / wide(scale, C)).float().to(torch.float8_e4m3fn), scale


def wide(scale, C):
    return scale.repeat_interleave(128, -1)[..., :C]


def value(q, scale):
    return q.double() * wide(scale.double(), q.shape[-1])


def weights(fp8, N, D, H, seed):      # channels of unlike size
    g = torch.Generator().manual_seed(seed)
    W1 = (torch.randn(N, D, 2 * H, generator=g) * torch.exp(torch.randn(N, D, 1, generator=g)) / D ** 0.5).bfloat16().cuda()
    W2 = (torch.randn(N, H, D, generator=g) / H ** 0.5).bfloat16().cuda()
    return W1, W2


def block_values(q, S):
    """Dequantised [.., C, Kd] of codes [.., C, Kd] and block scales."""
    C, Kd = q.shape[-2:]
    return q.double() * S.double().repeat_interleave(128, -2)[..., :C, :].repeat_interleave(128, -1)[..., :Kd]


def routing(M, N, K, seed, skew):
    from helpers import make_routing
    return make_routing(M, N, K, seed, skew)


def unpack_scales(buf, rows, blocks):
    """Expert-major scale bytes as the GEMMs read them -> scales [rows, blocks]."""
    g = -(-blocks // 4)
    r, b = torch.arange(rows, device=buf.device)[:, None], torch.arange(blocks, device=buf.device)[None]
    at = (r // 128 * g + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4
    return torch.exp2(buf[at].double() - 127)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_rows(fp8, dtype):
    for M, D in ((1, 8), (3, 128), (130, 136), (7, 2048), (1001, 264)):
        g = torch.Generator().manual_seed(M)
        x = (torch.randn(M, D, generator=g) * torch.exp(3 * torch.randn(M, 1, generator=g))).to(dtype).cuda()
        x[0, :min(D, 128)] = 0
        got = fp8.quantize_rows(x)
        q, scale = rows_of(x.double())
        # the largest rows overflow float16: an infinity makes its block's scale NaN (by the definition), no other
        fine = torch.isfinite(scale)
        assert torch.isnan(got.scale.double()[~fine]).all() and torch.equal(got.scale.double()[fine], scale[fine])
        at = wide(fine, D)
        assert torch.equal(got.q.float()[at], q.float()[at])
        view = fp8.quantize_rows(torch.cat([x, x], 1)[:, :D] if D % 8 == 0 else x)
        assert torch.equal(view.q.view(torch.uint8), got.q.view(torch.uint8))
    assert fp8.quantize_rows(x[:0]).scale.shape == (0, 3)


def test_scale_borders_and_bad_values(fp8):
    """448 * 2^e keeps its power, the next larger value takes the next one; tiny, huge and bad values."""
    x = torch.zeros(8, 128, device="cuda")
    x[0, 3] = 448.0
    x[1, 3] = torch.nextafter(torch.tensor(448.0), torch.tensor(1e9))
    x[2, 3] = -1.75 * 2.0 ** -20
    x[3, 3] = 2.0 ** -149                    # smallest subnormal: the scale stops at 2^-127
    x[4, 3] = torch.finfo(torch.float32).max
    x[5, 3], x[5, 4] = float("inf"), 1.0
    x[6, 3] = float("nan")
    r = fp8.quantize_rows(x)
    s = r.scale.view(torch.uint8).flatten().tolist()
    assert s == [127, 128, 127 - 28, 0, 127 + 120, 255, 255, 127]
    v = value(r.q, r.scale)
    assert float(v[0, 3]) == 448 and float(v[1, 3]) == 448 and float(v[2, 3]) == -1.75 * 2.0 ** -20
    assert torch.isnan(v[5]).all() and torch.isnan(v[6]).all() and not v[7].any() and torch.isfinite(v[:5]).all()


@pytest.mark.parametrize("N,D,H", [(1, 16, 16), (3, 144, 272), (2, 512, 128), (4, 2176, 48)])
def test_quantize_experts(fp8, N, D, H):
    W1, W2 = weights(fp8, N, D, H, 3)
    W2[0, :, :min(D, 128)] = 0
    for cast in (torch.bfloat16, torch.float32):
        e = fp8.quantize_experts(W1.to(cast), W2.to(cast))
        assert e.sizes == (N, D, H)
        for q, S, w in ((e.W1_N2HD.view(N, 2, H, D), e.S1, W1.double().transpose(1, 2).reshape(N, 2, H, D)),
                        (e.W2_NDH, e.S2, W2.double().transpose(1, 2))):
            C, Kd = w.shape[-2:]
            top = torch.nn.functional.pad(w.abs(), (0, -Kd % 128, 0, -C % 128)).unflatten(-1, (-1, 128)).unflatten(-3, (-1, 128)).amax((-3, -1))
            assert S.shape == top.shape
            s = S.double()
            assert (s[top == 0] == 1).all()
            assert (top <= 448 * s).all() and (top > 224 * s)[top > 0].all()
            step = s.repeat_interleave(128, -2)[..., :C, :].repeat_interleave(128, -1)[..., :Kd]
            assert torch.equal(q.float(), (w / step).float().to(torch.float8_e4m3fn).float())


class Stages:
    """The tables and buffers of one forward pass, as the whole call carves them from its workspace."""

    def __init__(self, M, N, K, D, H):
        from momoe import _lib, ops
        self.lib, self.ptr, self.st, self.status = _lib.lib, _lib.ptr, _lib.stream_ptr(), ops.status_word("cuda")
        self.check = _lib.check
        tiles = -(-M * K // 128) + min(N, M * K)
        rows = tiles * 128
        i32 = lambda n: torch.full((n,), 77, dtype=torch.int32, device="cuda")
        u8 = lambda n: torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
        self.sizes = torch.empty(N, dtype=torch.int64, device="cuda")
        self.tile_expert, self.pair_info, self.sched, self.tile_rows, self.pos = i32(tiles), i32(tiles), i32(8), i32(tiles), i32(M * K)
        self.row_weight = torch.full((rows,), float("nan"), device="cuda")
        self.xs, self.xsc = u8(rows * D), u8(tiles * -(-D // 512) * 512)
        self.hs, self.hsc = u8(rows * H), u8(tiles * -(-H // 512) * 512)
        self.ys = torch.full((rows, D), float("nan"), dtype=torch.float16, device="cuda")
        self.yscale = torch.full((rows, -(-D // 256)), float("nan"), device="cuda")
        self.M, self.N, self.K, self.D, self.H, self.rows, self.tiles = M, N, K, D, H, rows, tiles
        p = lambda t: t.data_ptr()
        self.c = _lib.Plan(M=M, N=N, K=K, D=D, H=H, reserved=0, rows_capacity=rows, sched=p(self.sched),
                           tile_expert=p(self.tile_expert), pad_off=0, row_token=0,
                           row_weight=p(self.row_weight), pos_MK=p(self.pos), status=p(self.status), pair_info=p(self.pair_info))

    def dispatch(self, x, scale, idx, w):
        nbytes = self.lib.momoe_fp8_dispatch_workspace_bytes(self.M, self.N, self.K)
        ws = torch.full((max(nbytes, 1),), 0x7F, dtype=torch.uint8, device="cuda")
        p = self.ptr
        self.check(self.lib.momoe_fp8_dispatch_rows(p(x), p(scale), p(idx), p(w), self.M, self.N, self.K, self.D,
                                                    p(self.sizes), p(self.tile_expert), p(self.pair_info), p(self.sched),
                                                    p(self.tile_rows), p(self.row_weight), p(self.pos), self.rows, p(ws),
                                                    nbytes, p(self.xs), p(self.xsc), p(self.status), self.st), "dispatch")

    def gemms(self, e, stream):
        import ctypes
        ref, p, L = ctypes.byref(self.c), self.ptr, self.lib
        up = L.momoe_fp8_up_swiglu_decode if stream else L.momoe_fp8_up_swiglu
        down = L.momoe_fp8_down_scale_decode if stream else L.momoe_fp8_down_scale
        rows = p(self.tile_rows)
        self.check(up(ref, rows, p(self.xs), p(self.xsc), p(e.W1_N2HD), p(e.S1), p(self.hs), p(self.hsc), self.st), "up")
        self.check(down(ref, rows, p(self.hs), p(self.hsc), p(e.W2_NDH), p(e.S2), p(self.ys), p(self.yscale), self.st),
                   "down")

    def combine(self):
        y = torch.empty(self.M, self.D, dtype=torch.bfloat16, device="cuda")
        p = self.ptr
        self.check(self.lib.momoe_fp8_combine_rows(p(self.ys), p(self.yscale), p(self.pos), self.M, self.K, self.D, p(y),
                                                   self.st), "combine")
        return y


def check_tables(s, idx, w):
    """The layout against its definition: whole tiles of one expert each, every pair in a row of its own."""
    sizes = torch.bincount(idx.flatten().long(), minlength=s.N)
    assert torch.equal(s.sizes, sizes)
    nt = -(-sizes // 128)
    T = int(nt.sum())
    assert s.sched.tolist()[:4] == [T, 0, T * 128, int((-(-nt // 2)).sum())]
    assert torch.equal(s.tile_expert[:T].long(), torch.repeat_interleave(torch.arange(s.N, device="cuda"), nt))
    pairs, t0 = [], 0
    for n in nt.tolist():
        pairs += [(t0 + j) * 2 + (1 if j + 1 < n else 0) for j in range(0, n, 2)]
        t0 += n
    assert s.pair_info[:len(pairs)].tolist() == pairs
    rows = torch.cat([torch.tensor([min(128, n - j) for j in range(0, n, 128)], dtype=torch.int32) for n in sizes.tolist()])
    assert torch.equal(s.tile_rows[:T].cpu(), rows)
    pos = s.pos.long()
    assert len(pos.unique()) == s.M * s.K
    assert torch.equal(s.tile_expert[pos // 128], idx.flatten())
    assert (pos % 128 < s.tile_rows[pos // 128]).all()           # real rows come first in a tile
    assert torch.equal(s.row_weight[pos], w.flatten())


@pytest.mark.parametrize("stream", [False, True])
@pytest.mark.parametrize("M,N,K,D,H,skew", SHAPES)
def test_stages_against_64_bits(fp8, monkeypatch, M, N, K, D, H, skew, stream):
    from momoe import ops
    idx, w = routing(M, N, K, M + D, skew)
    e = fp8.quantize_experts(*weights(fp8, N, D, H, D + H))
    g = torch.Generator().manual_seed(1)
    x = torch.randn(M, D, generator=g).bfloat16().cuda()
    s = Stages(M, N, K, D, H)
    s.dispatch(x, None, idx, w)
    s.gemms(e, stream)
    torch.cuda.synchronize()
    ops.check_status()
    check_tables(s, idx, w)
    real = s.pos.long()
    token = torch.arange(M, device="cuda").repeat_interleave(K)
    expert = idx.flatten().long()
    # dispatch: the converted row of each token, bit for bit
    q, scale = rows_of(x.double())
    xq = s.xs.view(torch.float8_e4m3fn).view(s.rows, D)[real]
    assert torch.equal(xq.float(), q[token].float())
    assert torch.equal(unpack_scales(s.xsc, s.rows, -(-D // 128))[real], scale[token])
    xv = value(xq, scale[token])
    hq = s.hs.view(torch.float8_e4m3fn).view(s.rows, H)[real]
    hscale = unpack_scales(s.hsc, s.rows, -(-H // 128))[real]
    hv = value(hq, hscale)
    W1v = block_values(e.W1_N2HD.view(N, 2, H, D), e.S1)
    W2v = block_values(e.W2_NDH, e.S2)
    for n in range(N):
        at = (expert == n).nonzero().flatten()
        if len(at) == 0:
            continue
        a, b = xv[at] @ W1v[n, 0].T, xv[at] @ W1v[n, 1].T
        da, db = ACC * (xv[at].abs() @ W1v[n, 0].abs().T), ACC * (xv[at].abs() @ W1v[n, 1].abs().T)
        sg = torch.sigmoid(b)
        h = a * b * sg
        # |d(b sigmoid(b))/db| <= 1.1
        dh = da * (b * sg).abs() + 1.1 * db * a.abs() + 1.1 * da * db + 2.0 ** -20 * h.abs()
        top = torch.nn.functional.pad(h.abs(), (0, -H % 128)).unflatten(-1, (-1, 128)).amax(-1)
        dtop = torch.nn.functional.pad(dh, (0, -H % 128)).unflatten(-1, (-1, 128)).amax(-1)
        sc = hscale[at]
        assert (top - dtop <= 448 * sc).all() and (top + dtop >= 224 * sc).all()
        tol = torch.maximum((h.abs() + dh) * 2.0 ** -4, wide(sc, H) * 2.0 ** -10) + dh
        assert ((hv[at] - h).abs() <= tol).all(), "h of expert %d: %g" % (n, float(((hv[at] - h).abs() / tol).max()))
        wt = w.flatten()[at, None].double()
        y = hv[at] @ W2v[n].T * wt
        dy = ACC * (hv[at].abs() @ W2v[n].abs().T) * wt
        # fp16 at a power of two: 2^-11 relative, and half a step of its smallest numbers, 2^-25 of that power
        yv = s.ys.double() * s.yscale.double().repeat_interleave(256, 1)[:, :D]
        off = (yv[real[at]] - y).abs()
        fine = 2.0 ** -25 * s.yscale.double().repeat_interleave(256, 1)[:, :D][real[at]]
        assert (off <= 2.0 ** -11 * (y.abs() + dy) + dy + fine).all(), "y of expert %d" % n
        # the power of two is a bound, and not so far above the values that their precision suffers
        assert torch.isfinite(s.ys[real[at]]).all()
        assert (s.ys[real[at]].abs().amax(1) > 2.0 ** -8).all()
    # the combine: one rounding of the sum of K values, each up to 2^-24 (fma) off
    want = s.combine()
    vals = yv[real].view(M, K, D)
    assert ((want.double() - vals.sum(1)).abs() <= 2.0 ** -8 * vals.sum(1).abs() + 2.0 ** -19 * vals.abs().sum(1)).all()
    # the whole call is these stages, bit for bit, from 16-bit and from 8-bit rows
    monkeypatch.setattr(fp8, "STREAM_MAX_AVG_ROWS", 2 ** 20 if stream else 0)
    for rows_in in (x, fp8.Fp8Rows(q, scale.to(torch.float8_e8m0fnu)), fp8.quantize_rows(x)):
        y, sizes = fp8.experts_forward(rows_in, idx, w, e)
        assert torch.equal(y, want) and torch.equal(sizes, s.sizes)
    ops.check_status()


def test_bad_rows_stay_alone_and_strides(fp8):
    M, N, K, D, H = 200, 8, 2, 256, 192
    idx, w = routing(M, N, K, 0, 0.0)
    e = fp8.quantize_experts(*weights(fp8, N, D, H, 0))
    x = torch.randn(M, D, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    want, sizes = fp8.experts_forward(x, idx, w, e)
    bad = x.clone()
    bad[3, 7], bad[9, 200] = float("nan"), float("inf")
    y, _ = fp8.experts_forward(bad, idx, w, e)
    good = [i for i in range(M) if i not in (3, 9)]
    assert torch.equal(y[good], want[good]) and torch.isnan(y[3]).all() and torch.isnan(y[9]).all()
    y, _ = fp8.experts_forward(torch.cat([x, x], 1)[:, D:], idx.long(), w.t().contiguous().t(), e)
    assert torch.equal(y, want)
    odd = torch.empty(M * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(M, D).copy_(x)
    assert torch.equal(fp8.experts_forward(odd, idx, w, e)[0], want)
    assert torch.equal(fp8.experts_forward(x.float(), idx, w, e)[0], want)
    zero, none = fp8.experts_forward(x[:0], idx[:0], w[:0], e)
    assert zero.shape == (0, D) and none.tolist() == [0] * N


@pytest.mark.parametrize("stream", [False, True])
def test_same_bits_every_time(fp8, monkeypatch, stream):
    """Rows of an expert are placed in no fixed order, across several tiles; the results do not depend on it."""
    monkeypatch.setattr(fp8, "STREAM_MAX_AVG_ROWS", 2 ** 20 if stream else 0)
    for M, N, K in ((700, 5, 3), (9000, 6, 2)):
        idx, w = routing(M, N, K, 1, 2.0)
        e = fp8.quantize_experts(*weights(fp8, N, 256, 144, 6))
        x = torch.randn(M, 256, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
        want, sizes = fp8.experts_forward(x, idx, w, e)
        assert int(sizes.max()) > 256
        for _ in range(12):
            y, n = fp8.experts_forward(x, idx, w, e)
            assert torch.equal(y, want) and torch.equal(n, sizes)
        order = torch.randperm(M, generator=torch.Generator().manual_seed(7)).cuda()
        y, _ = fp8.experts_forward(x[order], idx[order], w[order], e)
        assert torch.equal(y, want[order])


@pytest.mark.parametrize("stream", [False, True])
def test_result_rows_keep_their_range(fp8, monkeypatch, stream):
    """Values far beyond fp16 and far below it, and rows of unlike size, come out with one bfloat16 rounding: the
    intermediate rows carry a power of two each."""
    monkeypatch.setattr(fp8, "STREAM_MAX_AVG_ROWS", 2 ** 20 if stream else 0)
    M, N, K, D, H = 60, 4, 2, 384, 160
    idx, w = routing(M, N, K, 2, 0.0)
    W1, W2 = weights(fp8, N, D, H, 4)
    x = torch.randn(M, D, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    for exponent, columns in ((0, 0), (40, 0), (-50, 0), (0, 20)):
        W = W2.clone()
        W[:, :, :256] *= 2.0 ** columns                     # one block of columns much larger than the other
        e = fp8.quantize_experts(W1, (W.float() * 2.0 ** exponent))
        y, _ = fp8.experts_forward(x, idx, w * 3, e)
        base = fp8.quantize_experts(W1, W2)
        want, _ = fp8.experts_forward(x, idx, w * 3, base)
        # powers of two pass through every stage unchanged
        want = want.double() * 2.0 ** exponent
        want[:, :256] *= 2.0 ** columns
        assert torch.equal(y.double(), want)
    y, _ = fp8.experts_forward(x, idx, -w * 2.0 ** 30, base)
    assert torch.equal(y.double(), fp8.experts_forward(x, idx, w, base)[0].double() * -2.0 ** 30)
    y, _ = fp8.experts_forward(x, idx, torch.zeros_like(w), base)
    assert not y.any()
    big = x.clone()
    big[7] *= 2.0 ** 60                                      # both halves of the activation grow: h is 2^120 and more
    y, _ = fp8.experts_forward(big, idx, w, base)
    plain, _ = fp8.experts_forward(x, idx, w, base)
    others = [i for i in range(M) if i != 7]
    assert torch.equal(y[others], plain[others]) and not torch.isnan(y[7]).any()


def test_capture_other_stream_and_two_graphs(fp8):
    from momoe import ops
    N, K, D, H = 16, 4, 384, 256
    e = fp8.quantize_experts(*weights(fp8, N, D, H, 1))
    cases = []
    for M in (3, 700):
        idx, w = routing(M, N, K, M, 0.5)
        x = torch.randn(M, D, generator=torch.Generator().manual_seed(M)).bfloat16().cuda()
        cases.append((x, idx, w, fp8.experts_forward(x, idx, w, e)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [fp8.experts_forward(x, idx, w, e) for x, idx, w, _ in cases]
    s.synchronize()
    for (y, n), (_, _, _, (want, sizes)) in zip(got, cases):
        assert torch.equal(y, want) and torch.equal(n, sizes)
    graphs = []
    for x, idx, w, want in cases:
        buf, ibuf = torch.zeros_like(x), idx.flip(0).contiguous()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fp8.experts_forward(buf, ibuf, w, e)
        graphs.append((graph, buf, ibuf, out))
    for _ in range(2):
        for (graph, buf, ibuf, out), (x, idx, w, want) in zip(graphs, cases):
            buf.copy_(x)
            ibuf.copy_(idx)
            graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, out), (_, _, _, want) in zip(graphs, cases):
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    ops.check_status()


def test_an_expert_named_twice_counts_twice_and_bad_ids_are_reported(fp8):
    from momoe import ops
    e = fp8.quantize_experts(*weights(fp8, 8, 64, 32, 1))
    x = torch.randn(4, 64, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    w = torch.tensor([[0.5, 0.5], [1.0, 0.25], [0.75, 0.25], [0.0, 2.0]], device="cuda")
    t = lambda ids: torch.tensor(ids, dtype=torch.int32, device="cuda")
    ops.check_status()
    y, sizes = fp8.experts_forward(x, t([[0, 1], [2, 3], [4, 4], [5, 6]]), w, e)
    assert sizes.tolist() == [1, 1, 1, 1, 2, 1, 1, 0]
    one, _ = fp8.experts_forward(x[2:3], t([[4]]), torch.ones(1, 1, device="cuda"), e)
    # 0.75 o + 0.25 o and o, each rounded to bfloat16 once
    assert ((y[2].double() - one[0].double()).abs() <= 2 * 2.0 ** -8 * one[0].double().abs()).all()
    ops.check_status()
    for ids in (t([[0, 1], [2, 8], [4, 5], [5, 6]]), t([[0, 1], [2, 3], [4, -1], [5, 6]]),
                t([[0, 1], [2, 3], [4, 5], [5, 6]]).long() + 2 ** 32):
        fp8.experts_forward(x, ids, w, e)
        with pytest.raises(RuntimeError, match="202"):
            ops.check_status()
    many = t([[0, 1]]).expand(9000, 2).clone()               # the two-launch dispatch reports as well
    many[4321, 1] = 99
    fp8.experts_forward(x[:1].expand(9000, 64), many, torch.ones(9000, 2, device="cuda"), e)
    with pytest.raises(RuntimeError, match="202"):
        ops.check_status()
    ops.check_status()


def test_refusals(fp8):
    N, K, D, H = 4, 2, 64, 32
    W1, W2 = weights(fp8, N, D, H, 2)
    e = fp8.quantize_experts(W1, W2)
    idx, w = routing(6, N, K, 0, 0.0)
    x = torch.zeros(6, D, dtype=torch.bfloat16, device="cuda")
    r = fp8.quantize_rows(x)
    for bad in (lambda: fp8.experts_forward(x[:, :48], idx, w, e), lambda: fp8.experts_forward(x[:5], idx, w, e),
                lambda: fp8.experts_forward(x, idx, w[:, :1], e), lambda: fp8.experts_forward(x.cpu(), idx, w, e),
                lambda: fp8.experts_forward(x.clone().requires_grad_(True), idx, w, e),
                lambda: fp8.experts_forward(x, idx, w.clone().requires_grad_(True), e),
                lambda: fp8.experts_forward(x.int(), idx, w, e),
                lambda: fp8.experts_forward(fp8.Fp8Rows(r.q, r.scale[:5]), idx, w, e),
                lambda: fp8.experts_forward(fp8.Fp8Rows(r.q.view(torch.uint8), r.scale), idx, w, e),
                lambda: fp8.experts_forward(x, idx, w, e._replace(S1=e.S1[:, :1])),
                lambda: fp8.experts_forward(x, idx, w, e._replace(W2_NDH=e.W2_NDH.transpose(1, 2))),
                lambda: fp8.experts_forward(x, torch.zeros(6, 5, dtype=torch.int32, device="cuda"), torch.zeros(6, 5, device="cuda"), e),
                lambda: fp8.quantize_experts(W1, W2[:, :24]), lambda: fp8.quantize_experts(W1[:, :40, :], W2[:, :, :40]),
                lambda: fp8.quantize_rows(x[:, :4]), lambda: fp8.quantize_rows(x.int()), lambda: fp8.quantize_rows(x.cpu())):
        with pytest.raises(RuntimeError):
            bad()


# ------------------------------------------------------------------------------------------------- the layer
def layer(D, H, N, K, Ks, seed, **kw):
    import momoe
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    return momoe.MoE(D, H, N, K, Ks, Wg_DN=(r(D, N) / D ** 0.5).bfloat16().cuda(),
                     Wl1_ND2H=(r(N, D, 2 * H) / D ** 0.5).bfloat16().cuda(),
                     Wl2_NHD=(r(N, H, D) / H ** 0.5).bfloat16().cuda(), **kw)


def test_prenorm_layer_in_eight_bits_is_its_operators_in_a_row(fp8):
    from momoe import norm, ops
    B, S, D, H, N, K, Ks = 3, 41, 256, 128, 12, 4, 1
    moe = layer(D, H, N, K, Ks, 0)
    block = norm.PreNormMoE(norm.RMSNorm(D, weight=1 + 0.1 * torch.randn(D, device="cuda").bfloat16()), moe)
    x, res = torch.randn(2, B, S, D, device="cuda").bfloat16()
    bias = moe.biases_N.detach().clone()
    with torch.no_grad():
        y16, r16 = block(x, res)
        moe.biases_N.copy_(bias)
        moe.quantize_experts()
        y, r = block(x, res)
        assert torch.equal(r, r16) and y.shape == (B, S, D) and y.dtype == torch.bfloat16
        n = norm.rms_norm_fp8(x, block.norm.weight, res)
        logits = n.y.view(-1, D) @ moe.router.Wg_DN
        idx, w, _ = ops.route_topk(logits, bias, K, Ks, dense=False)
        want, sizes = fp8.experts_forward(n.rows, idx, w, moe.experts_fp8)
        assert torch.equal(y.view(-1, D), want)
        # the bias moved as it does in 16 bits
        c_avg = B * S * (K - Ks) / (N - Ks)
        step = moe.bias_update_rate * torch.sign(c_avg - sizes[:N - Ks].float())
        assert torch.allclose(moe.biases_N[:N - Ks], bias[:N - Ks] + step, rtol=0, atol=1e-9)
        # e4m3 in x, W and h, each off by up to 2^-4 and on average about 2^-5.3 of its value: y follows to some 8 %
        assert float((y.float() - y16.float()).norm() / y16.float().norm()) < 0.12
        alone = block(x)
        assert torch.equal(alone[1], x)
    import copy
    twin = copy.deepcopy(moe)
    with torch.no_grad():
        twin.biases_N.copy_(moe.biases_N)
        assert torch.equal(twin(x), moe(x))
    # refusals: gradients, stale weights, rows without 8-bit experts, training coefficients
    with pytest.raises(RuntimeError, match="no backward"):
        moe(x)
    with torch.no_grad():
        moe.balance_coef = 0.1
        with pytest.raises(RuntimeError, match="training"):
            moe(x)
        moe.balance_coef = 0.0
        moe.momoe.Wl2_NHD.mul_(0.5)
        with pytest.raises(RuntimeError, match="changed"):
            moe(x)
        moe.quantize_experts()
        twin = copy.deepcopy(moe)
        twin.biases_N.copy_(moe.biases_N)
        assert torch.equal(twin(x), moe(x))
        moe.experts_fp8 = None
        with pytest.raises(RuntimeError, match="8-bit experts"):
            moe(x, n.rows)
        moe(x)
    ops.check_status()


def test_eight_bit_weights_that_stand_for_other_weights_are_refused(fp8):
    """Swapped parameters, a copy of a layer whose weights have moved on, and a copy that is changed before its first pass."""
    import copy
    import io
    moe = layer(128, 64, 8, 2, 0, 0)
    x = torch.randn(1, 5, 128, device="cuda").bfloat16()
    with torch.no_grad():
        moe.quantize_experts()
        want = moe(x)
        twin = copy.deepcopy(moe)
        twin.momoe.Wl1_ND2H.mul_(0.5)
        with pytest.raises(RuntimeError, match="changed"):
            twin(x)
        with pytest.raises(RuntimeError, match="changed"):
            copy.deepcopy(twin)(x)
        twin.quantize_experts()
        twin(x)
        file = io.BytesIO()
        torch.save(moe, file)
        file.seek(0)
        again = torch.load(file, weights_only=False)
        again.biases_N.copy_(moe.biases_N)
        assert torch.equal(again(x), moe(x)) and want.shape == x.shape
        moe.momoe.Wl2_NHD = torch.nn.Parameter(moe.momoe.Wl2_NHD.detach().clone())
        with pytest.raises(RuntimeError, match="changed"):
            moe(x)
        moe.quantize_experts()
        moe(x)
        plain = copy.deepcopy(layer(128, 64, 8, 2, 0, 0))       # one without 8-bit weights, which get set by hand
        plain.experts_fp8 = moe.experts_fp8
        plain(x)


@pytest.mark.parametrize("fused", [True, False])
def test_layer_with_balance_loss_trains_on_the_sum_of_both(fp8, fused):
    """The auxiliary loss and its share of the gradients are those of the operator on the layer's own logits."""
    from momoe import balance, norm, ops
    B, S, D, H, N, K, Ks = 4, 33, 192, 64, 10, 4, 1
    def run(coefs, use_y=True):
        moe = layer(D, H, N, K, Ks, 5)
        moe.fused = fused
        moe.balance_coef, moe.z_coef = coefs
        block = norm.PreNormMoE(norm.RMSNorm(D), moe)
        g = torch.Generator().manual_seed(3)
        x = torch.randn(B, S, D, generator=g).bfloat16().cuda().requires_grad_(True)
        y, r = block(x, torch.ones_like(x))
        loss = (y.float() * torch.randn(B, S, D, generator=g).cuda()).sum() * (1.0 if use_y else 0.0)
        if moe.aux_loss is not None:
            loss = loss + 100 * moe.aux_loss
        loss.backward()
        return moe, block, x, y
    plain, pblock, px, py = run((0.0, 0.0))
    assert plain.aux_loss is None
    moe, block, x, y = run((0.2, 0.05))
    assert torch.equal(y, py)
    import copy
    twin = copy.deepcopy(moe)                                # the loss belongs to the graph, not to a copy of the layer
    assert twin.aux_loss is None and twin.balance_coef == 0.2 and moe.aux_loss is not None
    # the operator on the same logits
    with torch.no_grad():
        n, _ = norm.rms_norm(x, block.norm.weight, torch.ones_like(x))
        logits = n.view(-1, D) @ moe.router.Wg_DN
        idx, _, _ = ops.route_topk(logits, layer(D, H, N, K, Ks, 5).biases_N, K, Ks, dense=False)
    leaf = logits.detach().requires_grad_(True)
    aux, counts = balance.balance_loss(leaf, idx, Ks, 0.2, 0.05, seq_len=S)
    assert counts.shape == (B, N) and int(counts.sum()) == B * S * K
    assert float(aux.detach()) == float(moe.aux_loss.detach())
    (100 * aux).backward()
    # gate weights: the two shares add up; each term is rounded to 16 bits on its way (2^-8 of the larger one, twice, and
    # the products are rounded once more)
    share = n.view(-1, D).double().T @ leaf.grad.double()
    got = moe.router.Wg_DN.grad.double() - plain.router.Wg_DN.grad.double()
    mags = n.view(-1, D).double().abs().T @ (leaf.grad.double().abs() * 2.0 ** -7)
    both = moe.router.Wg_DN.grad.double().abs() + plain.router.Wg_DN.grad.double().abs()
    # the logits' gradient of the experts is not at hand: bound it through the gate gradient's own size per column
    lim = mags + 2.0 ** -7 * both + 2.0 ** -7 * both.amax(0, keepdim=True)
    assert ((got - share).abs() <= lim).all(), float(((got - share).abs() / lim).max())
    assert torch.equal(moe.momoe.Wl1_ND2H.grad, plain.momoe.Wl1_ND2H.grad)
    # alone: the upstream gradient of y is zero, so only the operator's share remains
    only, oblock, ox, _ = run((0.2, 0.05), use_y=False)
    got = only.router.Wg_DN.grad.double()
    assert ((got - share).abs() <= 2.0 ** -8 * share.abs() + mags).all()
    assert not only.momoe.Wl2_NHD.grad.any() and ox.grad.any()
    ops.check_status()
