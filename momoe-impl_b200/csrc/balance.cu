// Balance loss and z-loss of a router with per-expert counts, and the gradient of its logits.
//
// With p the softmax over the Ng = N - Ks gating logits of a token, T_b the tokens of sequence b, B' the sequences that
// are not empty, T all tokens and Kg = K - Ks the routed experts a token has:
//   count[b,e] = how often e is among the experts of sequence b's tokens
//   f[b,e] = Ng / (Kg T_b) * count[b,e],   P[b,e] = mean of p[.,e] over sequence b
//   loss = balance_coef / B' * sum_b sum_e f[b,e] P[b,e]  +  z_coef / T * sum_t lse_t^2
// The counts carry no gradient, so with g[b,e] = balance_coef f[b,e] / (B' T_b)
//   dloss/dlogit[t,e] = p[t,e] (g[b,e] - sum_j g[b,j] p[t,j] + 2 z_coef / T * lse_t)
// Rows outside every sequence are neither read nor counted and get a zero gradient; a row whose gating logits are all
// -inf has p = 0 and lse = 0.  A table of sequences that does not ascend gives a loss and coefficients of NaN, and no counts.
//
// Bound by HBM for large batches (the logits are read once in each direction and the gradient written once) and by the
// launches for small ones.  Forward, two launches: blocks of rows leave partial sums, one slot for each (row block,
// sequence) that meet; then the slots of a sequence are added in a fixed order, 32 experts a block, and the last block
// to finish adds the blocks' shares of the loss, also in a fixed order: no result depends on timing.  At 65521 rows of 256
// logits in 37 sequences the partial sums take 21 us, their sum 7 and the gradient 26, against 16 us for the bytes alone.
// Of a warp's time the partial sums wait 42 % for loads and 9 % for exchanges between lanes, the gradient 25 % and 14 %: a warp
// has one set of rows in flight.  At 1024 x 32: 3.7, 5.7, 2.9.
#include <cmath>

#include "internal.h"
#include "../../include/momoe_b200.h"

namespace momoe {

constexpr int BAL_THREADS = 256;
constexpr int BAL_WARPS = BAL_THREADS / 32;
constexpr int BAL_MAX_EXPERTS = 1024;

__device__ __forceinline__ float bal_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ float bal_to_float(float v) { return v; }
__device__ __forceinline__ float bal_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void bal_from_float(float v, float& o) { o = v; }
__device__ __forceinline__ void bal_from_float(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) BalVec {
    T v[V];
};

// How a row of N logits lies in a warp: L lanes a row (32 / L rows side by side), lane l of them holds the logits
// (l + i L) V .. + V - 1, i < NV.  Few lanes a row keep the reductions short, which is what a row costs; V = 8 needs rows
// that are a multiple of 8 long.
template <typename T, int L, int V, int NV>
struct BalRow {
    static constexpr int C = V * NV;

    static __device__ __forceinline__ int column(int l, int i) { return (l + i * L) * V; }

    // columns from Ng on, and the whole row where `in` is false, count as -inf
    static __device__ __forceinline__ void load(const T* row, bool in, int N, int Ng, int l, float (&x)[C]) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = column(l, i);
            BalVec<T, V> q;
            if (in && j < N) q = *reinterpret_cast<const BalVec<T, V>*>(row + j);
#pragma unroll
            for (int u = 0; u < V; ++u) x[i * V + u] = in && j + u < Ng ? bal_to_float(q.v[u]) : -INFINITY;
        }
    }
    static __device__ __forceinline__ float max(float v) {
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    }
    static __device__ __forceinline__ float sum(float v) {
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
    // x -> probabilities; returns the log of the sum (0, and p = 0, where every logit is -inf).
    static __device__ __forceinline__ float softmax(float (&x)[C]) {
        float mx = x[0];
#pragma unroll
        for (int i = 1; i < C; ++i) mx = fmaxf(mx, x[i]);
        mx = max(mx);
        const bool dead = mx == -INFINITY;
        const float base = dead ? 0.0f : mx;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            x[i] = __expf(x[i] - base);      // 2 + 1.2 |x| units of the last place: 2^-17 at e^-100
            s += x[i];
        }
        s = sum(s);
        // a NaN among the logits is lost by the maximum, not by the sum: it is not 0, so it reaches the result
        const bool none = dead && s == 0.0f;
        const float inv = none ? 0.0f : 1.0f / s;
#pragma unroll
        for (int i = 0; i < C; ++i) x[i] *= inv;
        return none ? 0.0f : base + logf(s);
    }
};

// The B sequences of M rows: a table of B + 1 row numbers, or (null) consecutive sequences of S rows.
struct BalSeqs {
    const int* cu;
    int S, B, M;
    // first row of sequence b (b = B: the end of the last one), kept inside [0, M]
    __device__ __forceinline__ int bound(int b) const {
        if (cu == nullptr) return static_cast<int>(min(static_cast<long long>(b) * S, static_cast<long long>(M)));
        return min(max(__ldg(cu + b), 0), M);
    }
    // last sequence that starts at or before `row` (-1: none)
    __device__ __forceinline__ int of(int row) const {
        if (cu == nullptr) return min(row / S, B - 1);
        int lo = -1, hi = B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (bound(mid) <= row) lo = mid;
            else hi = mid;
        }
        return lo;
    }
};

struct BalArgs {
    const void* logits;
    const int* topk;
    BalSeqs seq;
    int M, N, K, Ks, B;
    int R;               // rows of a row block
    int n_blk;
    float balance_coef, z_coef;
    float* slot_p;       // [n_blk + B, N]
    int* slot_count;     // [n_blk + B, N]
    float* slot_z;       // [n_blk + B]
    float* share;        // [column blocks * B]
    unsigned* ticket;
    int* totals;         // [3]: sequences that are not empty, all their tokens, whether a bound is below the one before
    float* loss;
    long long* counts;   // [B, N]
    float* g;            // [B, N]
};

template <typename T, int L, int V, int NV>
__global__ void __launch_bounds__(BAL_THREADS) balance_partial_kernel(const BalArgs a) {
    using Row = BalRow<T, L, V, NV>;
    constexpr int SIDE = 32 / L;                // rows side by side in a warp
    extern __shared__ float sm[];               // [8 warps, N] sums, then N counters
    __shared__ float s_z[BAL_WARPS];
    int* s_cnt = reinterpret_cast<int*>(sm + BAL_WARPS * a.N);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, l = lane % L;
    const int c = blockIdx.x;
    const int row0 = c * a.R, row1 = min(a.M, row0 + a.R);
    if (c == 0) {
        // once for the whole call, whatever the number of sequences
        __shared__ unsigned s_tot[3];
        if (threadIdx.x < 3) s_tot[threadIdx.x] = 0u;
        if (threadIdx.x == 0) *a.ticket = 0u;
        __syncthreads();
        unsigned n = 0u, tokens = 0u, bad = 0u;
        for (int i = threadIdx.x; i < a.B; i += BAL_THREADS) {
            const int len = a.seq.bound(i + 1) - a.seq.bound(i);
            if (len > 0) {
                ++n;
                tokens += static_cast<unsigned>(len);
            }
            if (len < 0) bad = 1u;
        }
        atomicAdd(&s_tot[0], n);
        atomicAdd(&s_tot[1], tokens);
        atomicOr(&s_tot[2], bad);
        __syncthreads();
        if (threadIdx.x < 3) a.totals[threadIdx.x] = static_cast<int>(s_tot[threadIdx.x]);
    }
    const T* logits = static_cast<const T*>(a.logits);
    const int Ng = a.N - a.Ks;
    int b = a.seq.of(row0);
    if (b < 0) b = 0;
    for (; b < a.seq.B; ++b) {
        const int start = a.seq.bound(b);
        const int end = a.seq.bound(b + 1);
        if (start >= row1 || end < start) break;
        const int lo = max(start, row0), hi = min(end, row1);
        if (hi <= lo) continue;
        for (int e = threadIdx.x; e < a.N; e += BAL_THREADS) s_cnt[e] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < (hi - lo) * a.K; i += BAL_THREADS) {
            const int e = __ldg(a.topk + static_cast<size_t>(lo) * a.K + i);
            if (e >= 0 && e < a.N) atomicAdd(&s_cnt[e], 1);
        }
        float acc[Row::C], z = 0.0f;
#pragma unroll
        for (int i = 0; i < Row::C; ++i) acc[i] = 0.0f;
        for (int m0 = lo + w * SIDE; m0 < hi; m0 += BAL_WARPS * SIDE) {
            const int m = m0 + lane / L;
            float x[Row::C];
            Row::load(logits + static_cast<size_t>(m) * a.N, m < hi, a.N, Ng, l, x);
            const float lse = Row::softmax(x);
#pragma unroll
            for (int i = 0; i < Row::C; ++i) acc[i] += x[i];
            z = fmaf(lse, lse, z);
        }
        // rows side by side, then the warps
#pragma unroll
        for (int o = 16; o >= L; o >>= 1) {
#pragma unroll
            for (int i = 0; i < Row::C; ++i) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
            z += __shfl_xor_sync(0xffffffffu, z, o);
        }
        if (lane < L) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int j = Row::column(l, i);
#pragma unroll
                for (int u = 0; u < V; ++u)
                    if (j + u < a.N) sm[w * a.N + j + u] = acc[i * V + u];
            }
        }
        if (lane == 0) s_z[w] = z;
        __syncthreads();
        // row blocks and sequences both ascend along the rows, so block + sequence is a slot of its own
        const size_t slot = static_cast<size_t>(c + b);
        for (int e = threadIdx.x; e < a.N; e += BAL_THREADS) {
            float p = 0.0f;
#pragma unroll
            for (int i = 0; i < BAL_WARPS; ++i) p += sm[i * a.N + e];
            a.slot_p[slot * a.N + e] = p;
            a.slot_count[slot * a.N + e] = s_cnt[e];
        }
        if (threadIdx.x == 0) {
            float t = 0.0f;
            for (int i = 0; i < BAL_WARPS; ++i) t += s_z[i];
            a.slot_z[slot] = t;
        }
        __syncthreads();
    }
}

// Block (x, b): experts 32 x .. + 31 of sequence b, 32 threads down the sequence's slots for each expert.
__global__ void __launch_bounds__(1024) balance_finish_kernel(const BalArgs a) {
    __shared__ float s_p[32][33];
    __shared__ int s_c[32][33];
    __shared__ float s_red[32];
    __shared__ bool s_last;
    const int tx = threadIdx.x, ty = threadIdx.y, tid = ty * 32 + tx;
    const int b = blockIdx.y;
    const int start = a.seq.bound(b), end = a.seq.bound(b + 1);
    const int n = a.totals[0], tokens = a.totals[1];
    const bool bad = a.totals[2] != 0;          // then nothing is read of the slots, which need not have been written

    const int e = blockIdx.x * 32 + tx;
    const int Ng = a.N - a.Ks;
    const int T_b = bad ? 0 : end - start;
    float p = 0.0f;
    int cnt = 0;
    if (T_b > 0 && e < a.N) {
        const int c1 = (end - 1) / a.R;
        for (int c = start / a.R + ty; c <= c1; c += 32) {
            const size_t i = static_cast<size_t>(c + b) * a.N + e;
            p += a.slot_p[i];
            cnt += a.slot_count[i];
        }
    }
    s_p[ty][tx] = p;
    s_c[ty][tx] = cnt;
    __syncthreads();
    // warp ty now owns expert 32 x + ty
    p = bal_sum(s_p[tx][ty]);
    cnt = __reduce_add_sync(0xffffffffu, s_c[tx][ty]);
    const int eo = blockIdx.x * 32 + ty;
    float term = 0.0f;
    if (eo < a.N) {
        float f = 0.0f;
        if (T_b > 0 && eo < Ng)
            f = static_cast<float>(cnt) * (static_cast<float>(Ng) / (static_cast<float>(a.K - a.Ks) * static_cast<float>(T_b)));
        const float gf = T_b > 0 ? a.balance_coef * f / (static_cast<float>(n) * static_cast<float>(T_b)) : 0.0f;
        term = gf * p;
        if (tx == 0) {
            a.counts[static_cast<size_t>(b) * a.N + eo] = cnt;
            a.g[static_cast<size_t>(b) * a.N + eo] = bad ? NAN : gf;
        }
    }
    // z-loss of the sequence, added by its first block
    float z = 0.0f;
    if (blockIdx.x == 0 && T_b > 0) {
        const int c1 = (end - 1) / a.R;
        for (int c = start / a.R + tid; c <= c1; c += 1024) z += a.slot_z[c + b];
        z = bal_sum(z) * (a.z_coef / static_cast<float>(tokens));
    }
    __syncthreads();
    if (tx == 0) s_red[ty] = term + z;
    __syncthreads();
    if (ty == 0) {
        const float share = bal_sum(s_red[tx]);
        if (tx == 0) {
            a.share[static_cast<size_t>(b) * gridDim.x + blockIdx.x] = share;
            __threadfence();
            s_last = atomicAdd(a.ticket, 1u) == gridDim.x * gridDim.y - 1u;
        }
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    float total = 0.0f;
    for (unsigned i = tid; i < gridDim.x * gridDim.y; i += 1024) total += __ldcg(a.share + i);
    total = bal_sum(total);
    __syncthreads();
    if (tx == 0) s_red[ty] = total;
    __syncthreads();
    if (ty == 0) {
        total = bal_sum(s_red[tx]);
        if (tx == 0) *a.loss = bad ? NAN : total;
    }
}

// `add` (may be null, may be `out` itself): a gradient of the logits from elsewhere, added in 32 bits.  A warp takes RW
// consecutive rows, so that the coefficients of their sequence are mostly read once.
template <typename T, int L, int V, int NV>
__global__ void __launch_bounds__(BAL_THREADS)
balance_backward_kernel(const T* __restrict__ logits, const BalSeqs seq, const float* __restrict__ g, int N, int Ks, int RW,
                        float z_coef, const float* __restrict__ up, const T* add, T* out) {
    using Row = BalRow<T, L, V, NV>;
    constexpr int SIDE = 32 / L;
    const int lane = threadIdx.x & 31, l = lane % L;
    const int first_row = (blockIdx.x * BAL_WARPS + (threadIdx.x >> 5)) * RW;
    const int end_row = min(seq.M, first_row + RW);
    if (first_row >= end_row) return;
    const int Ng = N - Ks;
    const int first = seq.bound(0), last = seq.bound(seq.B);
    const float scale = __ldg(up);
    const float zt = 2.0f * z_coef / static_cast<float>(max(last - first, 1));
    int b = -1;                                 // sequence whose coefficients gv holds
    float gv[Row::C];
#pragma unroll
    for (int i = 0; i < Row::C; ++i) gv[i] = 0.0f;
    for (int m0 = first_row; m0 < end_row; m0 += SIDE) {
        const int m = m0 + lane / L;
        const bool here = m < end_row;
        const bool real = here && m >= first && m < last;
        float x[Row::C];
        Row::load(logits + static_cast<size_t>(m) * N, real, N, Ng, l, x);
        if (real && (b < 0 || m >= seq.bound(b + 1))) {
            b = seq.of(m);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int j = Row::column(l, i);
                if (V % 4 == 0) {
#pragma unroll
                    for (int u = 0; u < V; u += 4)
                        if (j + u < N) {
                            const float4 q = __ldg(reinterpret_cast<const float4*>(g + static_cast<size_t>(b) * N + j + u));
                            gv[i * V + u] = q.x;
                            gv[i * V + (u + 1) % V] = q.y;
                            gv[i * V + (u + 2) % V] = q.z;
                            gv[i * V + (u + 3) % V] = q.w;
                        }
                } else {
#pragma unroll
                    for (int u = 0; u < V; ++u)
                        if (j + u < N) gv[i * V + u] = __ldg(g + static_cast<size_t>(b) * N + j + u);
                }
            }
        }
        const float lse = Row::softmax(x);
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < Row::C; ++i) dot = fmaf(gv[i], x[i], dot);     // x is 0 in columns without a coefficient
        dot = Row::sum(dot) - zt * lse;
        if (!here) continue;
        const size_t row = static_cast<size_t>(m) * N;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = Row::column(l, i);
            if (j >= N) continue;
            BalVec<T, V> q;
            if (add != nullptr) q = *reinterpret_cast<const BalVec<T, V>*>(add + row + j);
#pragma unroll
            for (int u = 0; u < V; ++u) {
                float v = real && j + u < Ng ? x[i * V + u] * scale * (gv[i * V + u] - dot) : 0.0f;
                if (add != nullptr) v += bal_to_float(q.v[u]);
                bal_from_float(v, q.v[u]);
            }
            *reinterpret_cast<BalVec<T, V>*>(out + row + j) = q;
        }
    }
}

// Rows of a row block: enough blocks for four an SM, at least 16 rows so that the partial sums stay a small share.
static int bal_rows(int M) {
    const int want = (M + sm_count() * 4 - 1) / (sm_count() * 4);
    return (want < 16 ? 16 : want + BAL_WARPS - 1) / BAL_WARPS * BAL_WARPS;
}

struct BalLayout {
    size_t p, count, z, share, ticket, totals, bytes;
};
static BalLayout bal_layout(int M, int N, int B) {
    const size_t slots = static_cast<size_t>((M + bal_rows(M) - 1) / bal_rows(M)) + B;
    BalLayout l;
    l.p = 0;
    l.count = l.p + slots * N * 4;
    l.z = l.count + slots * N * 4;
    l.share = l.z + slots * 4;
    l.ticket = l.share + static_cast<size_t>((N + 31) / 32) * B * 4;
    l.totals = l.ticket + 4;
    l.bytes = l.totals + 12;
    return l;
}

static int bal_check(int32_t M, int32_t N, int32_t Ks, int32_t B, int32_t type) {
    if (M < 0 || N <= 0 || Ks < 0 || Ks >= N || B <= 0) return MOMOE_ERR_ARG;
    if (type != 0 && type != 2) return MOMOE_ERR_UNSUPPORTED;
    // row numbers stay inside 32 bits, with room for a step past the last row
    if (N > BAL_MAX_EXPERTS || B > 65535 || M > 1 << 30) return MOMOE_ERR_TOO_LARGE;
    return MOMOE_OK;
}

// Without a table of bounds the sequences have seq_len rows each and cover all M rows.
static bool bal_uniform(const int32_t* cu, int32_t seq_len, int32_t M, int32_t B) {
    return cu != nullptr || (seq_len > 0 && B == (M - 1) / seq_len + 1);
}

// 16 logits a lane in accesses of 8 where the row length allows it (32 above 512 experts), else one by one across a warp.
#define BAL_DISPATCH(T, CALL)                                   \
    if (N % 8 == 0) {                                           \
        if (N <= 32) { CALL(T, 2, 8, 2); }                      \
        else if (N <= 64) { CALL(T, 4, 8, 2); }                 \
        else if (N <= 128) { CALL(T, 8, 8, 2); }                \
        else if (N <= 256) { CALL(T, 16, 8, 2); }               \
        else if (N <= 512) { CALL(T, 32, 8, 2); }               \
        else { CALL(T, 32, 8, 4); }                             \
    }                                                           \
    else if (N <= 32) { CALL(T, 32, 1, 1); }                    \
    else if (N <= 64) { CALL(T, 32, 1, 2); }                    \
    else if (N <= 128) { CALL(T, 32, 1, 4); }                   \
    else if (N <= 256) { CALL(T, 32, 1, 8); }                   \
    else if (N <= 512) { CALL(T, 32, 1, 16); }                  \
    else { CALL(T, 32, 1, 32); }

}  // namespace momoe

using namespace momoe;

#define MOMOE_API extern "C" __attribute__((visibility("default")))

MOMOE_API size_t momoe_balance_loss_workspace_bytes(int32_t M, int32_t N, int32_t B) {
    if (M <= 0 || N <= 0 || B <= 0) return 0;
    return bal_layout(M, N, B).bytes;
}

MOMOE_API int momoe_balance_loss(const void* logits_MN, int32_t type, const int32_t* topk_idx_MK,
                                 const int32_t* cu_seqlens, int32_t seq_len, int32_t M, int32_t N, int32_t K,
                                 int32_t Ks, int32_t B, float balance_coef, float z_coef, float* loss,
                                 int64_t* counts_BN, float* grad_BN, void* workspace, size_t workspace_bytes,
                                 momoe_stream_t stream) {
    int rc = bal_check(M, N, Ks, B, type);
    if (rc != MOMOE_OK) return rc;
    if (M == 0 || K <= Ks || K > N || !bal_uniform(cu_seqlens, seq_len, M, B)) return MOMOE_ERR_ARG;
    if (logits_MN == nullptr || topk_idx_MK == nullptr || loss == nullptr || counts_BN == nullptr ||
        grad_BN == nullptr || workspace == nullptr)
        return MOMOE_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(logits_MN) & 15) != 0) return MOMOE_ERR_ARG;
    if (workspace_bytes < momoe_balance_loss_workspace_bytes(M, N, B) ||
        (reinterpret_cast<uintptr_t>(workspace) & 3) != 0)
        return MOMOE_ERR_ARG;
    if (static_cast<int64_t>(bal_rows(M)) * K > 0x7fffffff) return MOMOE_ERR_TOO_LARGE;
    const BalLayout l = bal_layout(M, N, B);
    char* ws = static_cast<char*>(workspace);
    BalArgs a;
    a.logits = logits_MN;
    a.topk = topk_idx_MK;
    a.seq = BalSeqs{cu_seqlens, seq_len, B, M};
    a.M = M; a.N = N; a.K = K; a.Ks = Ks; a.B = B;
    a.R = bal_rows(M);
    a.n_blk = (M + a.R - 1) / a.R;
    a.balance_coef = balance_coef;
    a.z_coef = z_coef;
    a.slot_p = reinterpret_cast<float*>(ws + l.p);
    a.slot_count = reinterpret_cast<int*>(ws + l.count);
    a.slot_z = reinterpret_cast<float*>(ws + l.z);
    a.share = reinterpret_cast<float*>(ws + l.share);
    a.ticket = reinterpret_cast<unsigned*>(ws + l.ticket);
    a.totals = reinterpret_cast<int*>(ws + l.totals);
    a.loss = loss;
    a.counts = reinterpret_cast<long long*>(counts_BN);
    a.g = grad_BN;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t smem = static_cast<size_t>(BAL_WARPS + 1) * N * 4;   // 36 KiB at most
#define BAL_PARTIAL(T, L, V, NV) balance_partial_kernel<T, L, V, NV><<<a.n_blk, BAL_THREADS, smem, st>>>(a)
    if (type == 0) { BAL_DISPATCH(__nv_bfloat16, BAL_PARTIAL) }
    else { BAL_DISPATCH(float, BAL_PARTIAL) }
#undef BAL_PARTIAL
    balance_finish_kernel<<<dim3((N + 31) / 32, B), dim3(32, 32), 0, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? MOMOE_OK : MOMOE_ERR_CUDA;
}

MOMOE_API int momoe_balance_loss_backward(const void* logits_MN, int32_t type, const int32_t* cu_seqlens,
                                          int32_t seq_len, const float* grad_BN, int32_t M, int32_t N, int32_t Ks, int32_t B,
                                          float z_coef, const float* grad_loss, const void* add_MN, void* G_logits_MN,
                                          momoe_stream_t stream) {
    int rc = bal_check(M, N, Ks, B, type);
    if (rc != MOMOE_OK) return rc;
    if (M == 0 || !bal_uniform(cu_seqlens, seq_len, M, B)) return MOMOE_ERR_ARG;
    if (logits_MN == nullptr || grad_BN == nullptr || grad_loss == nullptr || G_logits_MN == nullptr)
        return MOMOE_ERR_ARG;
    if (((reinterpret_cast<uintptr_t>(logits_MN) | reinterpret_cast<uintptr_t>(add_MN) |
          reinterpret_cast<uintptr_t>(G_logits_MN) | reinterpret_cast<uintptr_t>(grad_BN)) & 15) != 0)
        return MOMOE_ERR_ARG;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // rows of a warp: four blocks an SM, at least 8 (up to 32 experts a warp has room for 16, so in small calls half of its
    // lanes have no row; such a call is a launch's latency)
    int RW = (M + sm_count() * 4 * BAL_WARPS - 1) / (sm_count() * 4 * BAL_WARPS);
    RW = RW < 8 ? 8 : RW;
    const int grid = ((M + RW - 1) / RW + BAL_WARPS - 1) / BAL_WARPS;
#define BAL_BACKWARD(T, L, V, NV)                                                                               \
    balance_backward_kernel<T, L, V, NV><<<grid, BAL_THREADS, 0, st>>>(                                         \
        static_cast<const T*>(logits_MN), BalSeqs{cu_seqlens, seq_len, B, M}, grad_BN, N, Ks, RW, z_coef, grad_loss,  \
        static_cast<const T*>(add_MN), static_cast<T*>(G_logits_MN))
    if (type == 0) { BAL_DISPATCH(__nv_bfloat16, BAL_BACKWARD) }
    else { BAL_DISPATCH(float, BAL_BACKWARD) }
#undef BAL_BACKWARD
    return cudaGetLastError() == cudaSuccess ? MOMOE_OK : MOMOE_ERR_CUDA;
}
