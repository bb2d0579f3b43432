"""Measured cases of the operators around the expert layer: the residual addition with its root-mean-square norm, the
router's balance loss, and the experts in 8-bit floating point.

`own` chooses what `run` computes: the plain form (elementary torch operations) or the calls of this repository's package.
Both take the state that `prepare` makes.

Formats that the two sides share:
  8-bit rows     q e4m3 [M, D], scale e8m0 [M, ceil(D/128)]: one power of two for each 128 columns, the smallest 2^e with
                 max|x| <= 448 * 2^e (1 for a block of zeros); the value is q * scale.
  8-bit experts  W1 e4m3 [N, 2H, D] (rows [0, H) linear half, [H, 2H) gate half), S1 e8m0 [N, 2, ceil(H/128), ceil(D/128)];
                 W2 e4m3 [N, D, H], S2 e8m0 [N, ceil(D/128), ceil(H/128)]: one power of two for each 128 x 128 block.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
BALANCE, Z = 0.01, 0.001


# ------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decoded token: the latency of the pre-norm in front of the expert layer
        dict(name="norm fp8, 1 token", op="norm_fp8", M=1, D=2048, dtype="bf16", residual=True),
        # a prompt in front of a wide layer
        dict(name="norm fp8, 8192 x 7168", op="norm_fp8", M=8192, D=7168, dtype="bf16", residual=True),
        # the training step of the headline layer's width and tokens
        dict(name="norm train, 16384 x 2048", op="norm_train", M=16384, D=2048, dtype="bf16", residual=True),
        # an odd number of rows of a width that is no multiple of 128 times a power of two, residual stream in 32 bits
        dict(name="norm train, 4099 x 2176 fp32", op="norm_train", M=4099, D=2176, dtype="fp32", residual=True),
        # the smallest training batch of the published charts
        dict(name="balance, 1024 x 32", op="balance", M=1024, N=32, K=4, Ks=0, B=2, ragged=False),
        # the headline layer's router: 8 sequences of 2048 tokens
        dict(name="balance, 16384 x 128", op="balance", M=16384, N=128, K=8, Ks=0, B=8, ragged=False),
        # packed sequences of unlike lengths with padding rows behind them and masked experts, 4 shared experts
        dict(name="balance, 65521 x 256 ragged", op="balance", M=65521, N=256, K=12, Ks=4, B=37, ragged=True),
        # one decoded token through an inference layer
        dict(name="experts, 1 token", op="experts", M=1, D=2048, H=768, N=128, K=8, rows8=False),
        # a batch of decoded tokens, input already in 8 bits
        dict(name="experts, 64 tokens", op="experts", M=64, D=2048, H=768, N=128, K=8, rows8=True),
        # an odd prompt through a layer whose sizes are no powers of two
        dict(name="experts, 1031 tokens", op="experts", M=1031, D=2176, H=1152, N=64, K=6, rows8=False),
        # the pre-normed rows of a prompt, wide experts
        dict(name="experts, 4096 tokens", op="experts", M=4096, D=2048, H=1408, N=64, K=8, rows8=True),
        # the headline layer's sizes
        dict(name="experts, 16384 tokens", op="experts", M=16384, D=2048, H=1024, N=128, K=8, rows8=False),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))
    return max(step, min(hi, int(v)) // step * step)


def draw(rng):
    op = rng.choice(["norm_fp8", "norm_train", "balance", "experts", "experts"])
    if op.startswith("norm"):
        step = 16 if op == "norm_fp8" else 8
        D = _log(rng, 64, 8192, step)
        return dict(op=op, M=_log(rng, 1, min(65536, 8192 * 7168 // D // (2 if op == "norm_train" else 1))), D=D,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), residual=rng.random() < 0.75)
    if op == "balance":
        N = _log(rng, 8, 512)
        Ks = rng.choice([0, 0, 1, 4]) if N >= 16 else 0
        M = _log(rng, 1, min(65536, 65521 * 256 // N))
        return dict(op=op, M=M, N=N, K=Ks + rng.randint(1, 8 if N - Ks >= 8 else 1), Ks=Ks, B=rng.randint(1, max(1, min(64, M // 4))),
                    ragged=rng.random() < 0.6)
    M, N = _log(rng, 1, 16384), _log(rng, 4, 128)
    K = rng.randint(1, min(8, N))
    while True:
        D, H = _log(rng, 64, 4096, 16), _log(rng, 32, 2048, 16)
        if M * K * D * H <= 16384 * 8 * 2048 * 1024 and N * D * H <= 128 * 2048 * 1024:
            return dict(op=op, M=M, D=D, H=H, N=N, K=K, rows8=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------------ the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1 + 7919 * seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = dict(case)
    if case["op"].startswith("norm"):
        M, D, t = case["M"], case["D"], DTYPES[case["dtype"]]
        channel = torch.exp(0.7 * randn(D))                 # some channels of a residual stream are much larger than others
        s.update(x=(randn(M, D) * channel).to(t), w=(1 + 0.1 * randn(D)).to(t))
        s["res"] = (3 * randn(M, D) * channel).to(t) if case["residual"] else None
        if case["op"] == "norm_train":
            s["gy"] = (0.1 * randn(M, D)).to(t)
            s["gr"] = (0.1 * randn(M, D)).to(t) if case["residual"] else None
        return s
    if case["op"] == "balance":
        M, N, K, Ks, B = (case[k] for k in ("M", "N", "K", "Ks", "B"))
        Ng = N - Ks
        logits = randn(M, N) + 0.5 * randn(N)
        if case["ragged"]:
            logits[:, :Ng] = logits[:, :Ng].masked_fill(rand(M, Ng) < 0.02, float("-inf"))   # experts out of service
        picks = torch.topk(logits[:, :Ng] + 1e-3 * randn(Ng), K - Ks).indices.sort(dim=1).values
        shared = torch.arange(Ng, N, device="cuda").expand(M, Ks)
        used = M
        if case["ragged"]:
            # cut points from uniform numbers: some sequences are empty, the last sixteenth of the rows is padding
            used = M - M // 16
            cuts = (rand(B - 1) * (used + 1)).long().sort().values if B > 1 else torch.empty(0, dtype=torch.long, device="cuda")
        else:
            cuts = torch.arange(1, B, device="cuda") * M // B
        zero = torch.zeros(1, dtype=torch.long, device="cuda")
        logits[used:] = float("nan")                        # nobody writes padding rows
        s.update(logits=logits.bfloat16(), idx=torch.cat([picks, shared], 1).int().contiguous(),
                 cu=torch.cat([zero, cuts, zero + used]).int(), up=0.5 + rand(1)[0])
        return s
    M, D, H, N, K = (case[k] for k in ("M", "D", "H", "N", "K"))
    x = (randn(M, D) * torch.exp(0.3 * randn(D))).bfloat16()
    score = randn(M, N) + 0.5 * randn(N)                     # a mildly unbalanced router
    top = torch.topk(score, K)
    idx, order = top.indices.sort(dim=1)
    s.update(x=x, idx=idx.int(), w=torch.softmax(top.values, dim=1).gather(1, order).contiguous())
    if case["rows8"]:
        s["q"], s["scale"] = _to_rows8(x.float())
        del s["x"]
    W1, S1, W2, S2 = [], [], [], []
    for e in range(0, N, 16):                                # a few experts at a time: the 32-bit weights are never held whole
        n = min(16, N - e)
        q, sc = _to_blocks8(0.02 * randn(n, 2, H, D))
        W1.append(q.view(n, 2 * H, D))
        S1.append(sc)
        q, sc = _to_blocks8(0.02 * randn(n, D, H))
        W2.append(q)
        S2.append(sc)
    s.update(W1=torch.cat(W1), S1=torch.cat(S1), W2=torch.cat(W2), S2=torch.cat(S2))
    return s


def _exponents(amax):
    """The biased exponent byte of the smallest 2^e with amax <= 448 * 2^e; 127 where amax is 0."""
    m, x = torch.frexp(amax)                                 # amax = m * 2^x with 0.5 <= m < 1, and 448 = 0.875 * 2^9
    return torch.where(amax > 0, x - 9 + (m > 0.875).int() + 127, torch.full_like(x, 127)).clamp(0, 254)


def _scale_of(byte):
    return torch.ldexp(torch.ones_like(byte, dtype=torch.float32), byte - 127)


def _to_rows8(v):
    """v [.., C] in 32 bits -> e4m3 of the same shape and e8m0 [.., ceil(C/128)]."""
    C = v.shape[-1]
    blocks = torch.nn.functional.pad(v, (0, -C % 128)).unflatten(-1, (-1, 128))
    byte = _exponents(blocks.abs().amax(-1))
    q = (blocks / _scale_of(byte).unsqueeze(-1)).flatten(-2)[..., :C].contiguous()
    return q.to(torch.float8_e4m3fn), byte.to(torch.uint8).view(torch.float8_e8m0fnu)


def _to_blocks8(v):
    """v [.., R, C] in 32 bits -> e4m3 of the same shape and e8m0 [.., ceil(R/128), ceil(C/128)]."""
    R, C = v.shape[-2:]
    blocks = torch.nn.functional.pad(v, (0, -C % 128, 0, -R % 128)).unflatten(-1, (-1, 128)).unflatten(-3, (-1, 128))
    byte = _exponents(blocks.abs().amax((-3, -1)))           # [.., R/128, C/128]
    q = blocks / _scale_of(byte)[..., :, None, :, None]
    q = q.flatten(-2).flatten(-3, -2)[..., :R, :C].contiguous()
    return q.to(torch.float8_e4m3fn), byte.to(torch.uint8).view(torch.float8_e8m0fnu)


def _from_rows8(q, scale):
    return q.float() * scale.float().repeat_interleave(128, -1)[..., :q.shape[-1]]


def _from_blocks8(q, scale):
    R, C = q.shape[-2:]
    return q.float() * scale.float().repeat_interleave(128, -2)[..., :R, :].repeat_interleave(128, -1)[..., :C]


# -------------------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _run_own(s)
    return {"norm_fp8": _norm_fp8, "norm_train": _norm_train, "balance": _balance, "experts": _experts}[s["op"]](s)


def _run_own(s):
    package = os.path.join(os.getcwd(), "momoe-impl_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from momoe import balance, fp8, norm
    if s["op"] == "norm_fp8":
        out = norm.rms_norm_fp8(s["x"], s["w"], s["res"], EPS)
        rows = out.rows
        return dict(y=out.y, r=out.residual, q=rows.q, scale=rows.scale) if s["residual"] else dict(y=out.y, q=rows.q, scale=rows.scale)
    if s["op"] == "norm_train":
        x, w = s["x"].detach().requires_grad_(True), s["w"].detach().requires_grad_(True)
        if not s["residual"]:
            y = norm.rms_norm(x, w, eps=EPS)
            gx, gw = torch.autograd.grad(y, (x, w), s["gy"])
            return dict(y=y, gx=gx, gw=gw)
        y, r = norm.rms_norm(x, w, s["res"], EPS)
        gx, gw = torch.autograd.grad((y, r), (x, w), (s["gy"], s["gr"]))
        return dict(y=y, r=r, gx=gx, gw=gw)
    if s["op"] == "balance":
        logits = s["logits"].detach().requires_grad_(True)
        loss, counts = balance.balance_loss(logits, s["idx"], s["Ks"], BALANCE, Z, s["cu"])
        glogits, = torch.autograd.grad(loss, logits, s["up"])
        return dict(loss=loss, counts=counts, glogits=glogits)
    rows = fp8.Fp8Rows(s["q"], s["scale"]) if s["rows8"] else s["x"]
    y, counts = fp8.experts_forward(rows, s["idx"], s["w"], fp8.Fp8Experts(s["W1"], s["S1"], s["W2"], s["S2"]))
    return dict(y=y, counts=counts)


def _rms(s):
    """The rounded sum r (also in 32 bits), 1 / rms and the normed rows in 32 bits."""
    r = s["x"] if s["res"] is None else (s["x"].float() + s["res"].float()).to(s["x"].dtype)
    v = r.float()
    rstd = torch.rsqrt((v * v).mean(1, keepdim=True) + EPS)
    return r, v, rstd, v * rstd * s["w"].float()


def _norm_fp8(s):
    r, _, _, y = _rms(s)
    q, scale = _to_rows8(y)
    out = dict(y=y.to(s["x"].dtype), q=q, scale=scale)
    if s["residual"]:
        out["r"] = r
    return out


def _norm_train(s):
    r, v, rstd, y = _rms(s)
    gy, xhat = s["gy"].float(), v * rstd
    gh = gy * s["w"].float()
    gx = rstd * (gh - xhat * (gh * xhat).mean(1, keepdim=True))
    out = dict(y=y.to(s["x"].dtype), gw=(gy * xhat).sum(0).to(s["w"].dtype))
    if s["residual"]:
        gx = gx + s["gr"].float()
        out["r"] = r
    out["gx"] = gx.to(s["x"].dtype)
    return out


def _balance(s):
    M, N, K, Ks, B, cu = s["M"], s["N"], s["K"], s["Ks"], s["B"], s["cu"].long()
    Ng = N - Ks
    row = torch.arange(M, device=cu.device)
    seq = torch.searchsorted(cu, row, right=True) - 1        # sequence of each row; rows at or behind cu[B] have none
    real = seq < B
    seq = seq.clamp(max=B - 1)
    z = torch.where(real[:, None], s["logits"][:, :Ng].float(), 0.0)
    top = z.amax(1, keepdim=True)
    alive = torch.isfinite(top) & real[:, None]              # a row with every expert masked counts for nothing
    top = torch.where(alive, top, 0.0)
    ex = torch.where(alive, torch.exp(z - top), 0.0)
    total = ex.sum(1, keepdim=True)
    p = ex / torch.where(alive, total, 1.0)
    lse = torch.where(alive, top + torch.log(torch.where(alive, total, 1.0)), 0.0)
    lens = cu[1:] - cu[:-1]
    n_seq = (lens > 0).sum().clamp(min=1)
    inv = torch.where(lens > 0, 1.0 / lens.clamp(min=1), 0.0)[:, None]
    one = torch.where(real, 1, 0)[:, None].expand(M, K)
    counts = torch.zeros(B, N, dtype=torch.long, device=cu.device)
    counts.view(-1).index_add_(0, (seq[:, None] * N + s["idx"].long()).flatten(), one.flatten())
    P = torch.zeros(B, Ng, dtype=torch.float64, device=cu.device).index_add_(0, seq, p.double()).float() * inv
    f = counts[:, :Ng].float() * (inv * (Ng / (K - Ks)))
    T = lens.sum().clamp(min=1)
    loss = BALANCE * (f * P).sum() / n_seq + Z * (lse * lse).double().sum().float() / T
    gp = (BALANCE * f * inv / n_seq)[seq]
    glog = p * (gp - (gp * p).sum(1, keepdim=True)) + (2 * Z / T) * lse * p
    glogits = torch.zeros(M, N, device=cu.device)
    glogits[:, :Ng] = torch.where(real[:, None], glog * s["up"], 0.0)
    return dict(loss=loss, counts=counts, glogits=glogits.bfloat16())


def _experts(s):
    M, D, H, N, K = (s[k] for k in ("M", "D", "H", "N", "K"))
    q, scale = (s["q"], s["scale"]) if s["rows8"] else _to_rows8(s["x"].float())
    x = _from_rows8(q, scale)
    e, order = s["idx"].flatten().long().sort(stable=True)
    counts = torch.bincount(e, minlength=N)
    used = counts.nonzero().flatten()                        # only touched experts' weights are read
    place = (counts > 0).long().cumsum(0)[e] - 1
    at = torch.arange(M * K, device=e.device) - (counts.cumsum(0) - counts)[e]
    rows = torch.zeros(len(used), int(counts.max()), D, device=e.device)
    rows[place, at] = x[order // K]
    W1 = _from_blocks8(s["W1"][used].view(-1, 2, H, D), s["S1"][used]).flatten(1, 2)
    a, b = torch.bmm(rows, W1.transpose(1, 2)).split(H, dim=2)
    h = _from_rows8(*_to_rows8(a * b * torch.sigmoid(b)))
    out = torch.bmm(h, _from_blocks8(s["W2"][used], s["S2"][used]).transpose(1, 2))
    pairs = torch.empty(M * K, D, device=e.device)
    pairs[order] = out[place, at]
    y = (pairs.view(M, K, D) * s["w"].unsqueeze(2)).sum(1)
    return dict(y=y.bfloat16(), counts=counts)


# ------------------------------------------------------------------------------------------ what a pass has to move
def work(case):
    M = case["M"]
    if case["op"].startswith("norm"):
        D, b, res = case["D"], 4 if case["dtype"] == "fp32" else 2, 1 if case["residual"] else 0
        if case["op"] == "norm_fp8":
            return dict(bytes=M * D * (b * (2 + 2 * res) + 1) + M * -(-D // 128) + D * b, flops=6 * M * D)
        # forward: x, res -> y, r; backward: r, gy, gr -> gx (and the weight's gradient)
        return dict(bytes=M * D * b * (2 + 2 * res + 3 + res) + 3 * D * b, flops=16 * M * D)
    if case["op"] == "balance":
        N, K = case["N"], case["K"]
        return dict(bytes=M * N * 6 + M * K * 4 + case["B"] * N * 8, flops=20 * M * N)   # logits twice, their gradient
    D, H, N, K = (case[k] for k in ("D", "H", "N", "K"))
    touched = N * (1 - (1 - K / N) ** M)
    return dict(bytes=touched * 3 * D * H + M * D * (2 + (1 if case["rows8"] else 2)) + 8 * M * K + 8 * N,
                flops=6 * M * K * D * H)


# --------------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("norm"):
        x, w = s["x"].double(), s["w"].double()
        r = x if s["res"] is None else (x + s["res"].double()).to(s["x"].dtype).double()
        k = 1.0 / torch.sqrt(r.pow(2).sum(1) / case["D"] + EPS)
        y = torch.einsum("md,m,d->md", r, k, w)
        out = dict(y=y)
        if case["residual"]:
            out["r"] = r
        if case["op"] == "norm_fp8":
            out["q"], out["scale"] = _exact_rows8(y)
            return out
        gy = s["gy"].double()
        c = torch.einsum("md,md,d->m", gy, r, w) * k.pow(3) / case["D"]
        out["gx"] = gy * w * k[:, None] - r * c[:, None]
        if case["residual"]:
            out["gx"] = out["gx"] + s["gr"].double()
        out["gw"] = torch.einsum("md,md,m->d", gy, r, k)
        return out
    if case["op"] == "balance":
        return _exact_balance(case, s)
    D, H, N, K = (case[k] for k in ("D", "H", "N", "K"))
    if case["rows8"]:
        x = s["q"].double() * s["scale"].double().repeat_interleave(128, 1)[:, :D]
    else:
        q, sc = _exact_rows8(s["x"].double())
        x = q * sc.repeat_interleave(128, 1)[:, :D]
    y = torch.zeros(case["M"], D, dtype=torch.float64, device="cuda")
    for e in range(N):
        m, k = (s["idx"] == e).nonzero(as_tuple=True)
        if len(m) == 0:
            continue
        half = []
        for i in range(2):
            sc = s["S1"][e, i].double().repeat_interleave(128, 0)[:H].repeat_interleave(128, 1)[:, :D]
            half.append(x[m] @ (s["W1"][e, i * H:(i + 1) * H].double() * sc).T)
        h, hs = _exact_rows8(half[0] * half[1] / (1 + torch.exp(-half[1])))
        h = h * hs.repeat_interleave(128, 1)[:, :H]
        sc = s["S2"][e].double().repeat_interleave(128, 0)[:D].repeat_interleave(128, 1)[:, :H]
        y[m] += (h @ (s["W2"][e].double() * sc).T) * s["w"][m, k, None].double()
    return dict(y=y, counts=None)


def _exact_rows8(v):
    """Values of 8-bit rows in 64 bits: codes and scales."""
    C = v.shape[1]
    top = torch.nn.functional.pad(v.abs(), (0, -C % 128)).view(len(v), -1, 128).amax(2)
    e = torch.ceil(torch.log2(top / 448))
    e = torch.where(448 * torch.exp2(e - 1) >= top, e - 1, e)   # log2 of a border may come out a little high or low
    e = torch.where(448 * torch.exp2(e) < top, e + 1, e)
    scale = torch.where(top > 0, torch.exp2(e), 1.0)
    u = v / scale.repeat_interleave(128, 1)[:, :C]
    # e4m3: three bits behind the leading one, steps of 2^-9 below 2^-6
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(u / step) * step, scale


def _exact_balance(case, s):
    M, N, K, Ks, B = (case[k] for k in ("M", "N", "K", "Ks", "B"))
    Ng, cu = N - Ks, s["cu"].tolist()
    lens = [cu[b + 1] - cu[b] for b in range(B)]
    n_seq, T = max(1, sum(n > 0 for n in lens)), max(1, sum(lens))
    loss = torch.zeros((), dtype=torch.float64, device="cuda")
    grad = torch.zeros(M, N, dtype=torch.float64, device="cuda")
    for b in range(B):
        if lens[b] == 0:
            continue
        rows = slice(cu[b], cu[b + 1])
        z = s["logits"][rows, :Ng].double()
        lse = torch.logsumexp(z, 1)
        dead = torch.isneginf(lse)
        p = torch.softmax(z, 1).masked_fill(dead[:, None], 0.0)
        lse = lse.masked_fill(dead, 0.0)
        f = torch.bincount(s["idx"][rows].flatten().long(), minlength=N)[:Ng].double() * Ng / ((K - Ks) * lens[b])
        loss = loss + BALANCE / n_seq * (f * p.mean(0)).sum() + Z / T * lse.pow(2).sum()
        g = BALANCE / (n_seq * lens[b]) * f
        grad[rows, :Ng] = p * (g - (p @ g)[:, None] + (2 * Z / T) * lse[:, None])
    return dict(loss=loss, counts=None, glogits=grad * s["up"].double())
