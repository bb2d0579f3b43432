// Around the 8-bit expert GEMMs: the weights' conversion, the dispatch of token rows into expert-major order (which converts
// them on the way), and one call that runs the whole forward pass (dispatch, two GEMMs, combine) out of one workspace.
#include "fp8.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "../../include/momoe_b200.h"

namespace momoe {

__device__ __forceinline__ float f8_value(float v) { return v; }
__device__ __forceinline__ float f8_value(__nv_bfloat16 v) { return __bfloat162float(v); }

// W [N, Kd, G * C] -> q [N, G * C, Kd] (k contiguous, as the MMA reads it) and one scale for each 128 x 128 block
// [N, G, ceil(C / 128), ceil(Kd / 128)].  A block of columns never crosses a group (the linear and the gate half of the
// up projection).  Runs once when a model is loaded; the weights are read twice, once for the maximum of a block and once for
// its codes, and written once.
template <typename T>
__global__ void __launch_bounds__(256) fp8_quantize_weights_kernel(const T* __restrict__ W, int Kd, int G, int C,
                                                                   uint8_t* __restrict__ q, uint8_t* __restrict__ S) {
    __shared__ float s[128][33];     // 32 columns of the block at a time
    __shared__ uint32_t s_top[8];
    const int kb = blockIdx.x, cb = blockIdx.y % ((C + 127) / 128), grp = blockIdx.y / ((C + 127) / 128);
    const size_t e = blockIdx.z;
    const int k0 = kb * 128, c0 = cb * 128;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const T* src = W + e * Kd * static_cast<size_t>(G) * C + static_cast<size_t>(grp) * C;
    const size_t pitch = static_cast<size_t>(G) * C;
    uint32_t top = 0u;
    for (int k = w; k < 128; k += 8)
        for (int c = lane; c < 128; c += 32)
            if (k0 + k < Kd && c0 + c < C) top = max(top, abs_bits(f8_value(src[(k0 + k) * pitch + c0 + c])));
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) s_top[w] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, s_top[lane & 7]);
    const uint32_t byte = fp8_scale_byte(top);
    const float inv = fp8_inv_scale(byte);
    if (threadIdx.x == 0) S[((e * G + grp) * ((C + 127) / 128) + cb) * gridDim.x + kb] = static_cast<uint8_t>(byte);
    for (int cq = 0; cq < 4; ++cq) {
        for (int k = w; k < 128; k += 8) {
            const int c = c0 + cq * 32 + lane;
            s[k][lane] = k0 + k < Kd && c < C ? f8_value(src[(k0 + k) * pitch + c]) * inv : 0.0f;
        }
        __syncthreads();
        // 8 threads a column, 16 values of k each (Kd is a multiple of 16)
        const int cl = threadIdx.x >> 3, kc = threadIdx.x & 7;
        const int c = c0 + cq * 32 + cl, k = k0 + kc * 16;
        if (c < C && k < Kd) {
            uint32_t p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                p[i] = fp8_pack4(s[kc * 16 + 4 * i][cl], s[kc * 16 + 4 * i + 1][cl], s[kc * 16 + 4 * i + 2][cl],
                                 s[kc * 16 + 4 * i + 3][cl]);
            *reinterpret_cast<uint4*>(q + ((e * G + grp) * C + c) * static_cast<size_t>(Kd) + k) =
                make_uint4(p[0], p[1], p[2], p[3]);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ dispatch
// Expert-major layout and row conversion in one pass over the tokens.  A thread block has a chunk of tokens; it needs, for
// each expert, the pairs of all tokens (where the expert's 128-row tiles start) and a row number inside the expert that no
// other block hands out.
//   up to DISPATCH_SMALL_PAIRS pairs: every block counts all pairs itself, so the pass is one launch (an id costs a few
//       cycles, a launch several microseconds);
//   more: a first kernel counts each chunk and reserves its rows with one atomic for each (chunk, expert).
// Rows inside an expert are handed out by atomics, in no fixed order.  No result depends on it: a row's values do not
// depend on its place, and a token's K rows are added in the order of k.
constexpr int DISPATCH_SMALL_PAIRS = 16384;
constexpr int DISPATCH_MAX_EXPERTS = 1024;
constexpr int DISPATCH_MAX_TOPK = 32;

struct DispatchArgs {
    const void* x;              // bf16 [M, D], or e4m3 with x_scale
    const uint8_t* x_scale;
    const int* topk_idx;
    const float* topk_w;
    int M, N, K, D;
    int chunk;                  // tokens of a block
    int* total;                 // large: pairs of each expert [N]
    int* chunk_base;            // large: rows reserved before a chunk's own [n_chunks, N]
    long long* sizes;
    int* tile_expert;
    int* pair_info;
    int* sched;
    int* tile_rows;
    float* row_weight;
    int* pos;
    uint8_t* dst;
    uint8_t* dst_scale;
    int* status;
};

__device__ __forceinline__ int dispatch_expert(const DispatchArgs& a, int i, bool report) {
    const int e = __ldg(a.topk_idx + i);
    if (e >= 0 && e < a.N) return e;
    if (report) atomicCAS(a.status, 0, DEV_BAD_EXPERT_ID);
    return 0;                   // stay in bounds: the pair goes to expert 0, and the report says so
}

__global__ void __launch_bounds__(256) fp8_count_kernel(const DispatchArgs a) {
    __shared__ int s_cnt[DISPATCH_MAX_EXPERTS];
    for (int e = threadIdx.x; e < a.N; e += 256) s_cnt[e] = 0;
    __syncthreads();
    const int m0 = blockIdx.x * a.chunk, m1 = min(a.M, m0 + a.chunk);
    for (int i = m0 * a.K + threadIdx.x; i < m1 * a.K; i += 256) atomicAdd(&s_cnt[dispatch_expert(a, i, true)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e < a.N; e += 256)
        if (s_cnt[e] != 0) a.chunk_base[static_cast<size_t>(blockIdx.x) * a.N + e] = atomicAdd(a.total + e, s_cnt[e]);
}

// 16 columns of a row as e4m3, scaled by `inv`.
__device__ __forceinline__ uint4 fp8_convert16(const float (&v)[16], float inv) {
    uint4 o;
    o.x = fp8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    o.y = fp8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
    o.z = fp8_pack4(v[8] * inv, v[9] * inv, v[10] * inv, v[11] * inv);
    o.w = fp8_pack4(v[12] * inv, v[13] * inv, v[14] * inv, v[15] * inv);
    return o;
}

// A token's row is read once, converted (ROWS8: copied) and stored to the K expert-major rows of its experts, the scales in
// the blocks the GEMMs read.  A lane holds 16 columns, 8 lanes a block of 128, a warp the 512 columns whose four scale
// bytes make one word.  One warp a token, or (ONE, few tokens) one block a token, its warps on different columns.  Bound by
// HBM: M D (2 + K) bytes from 16-bit rows, M D (1 + K) from 8-bit ones (68 us at 16384 tokens, D2048, top-8: 0.75 of the
// measured copy rate); by latency for few tokens (one token 4.9 us with one warp a token, 3.3 with one block).  Padding rows
// of dst are left as they are.
template <bool ROWS8, bool SMALL, bool ONE>
__global__ void __launch_bounds__(256) fp8_dispatch_kernel(const DispatchArgs a) {
    constexpr int STEP = ONE ? 8 : 1;    // warps that share a token
    __shared__ int s_next[DISPATCH_MAX_EXPERTS];     // next row of each expert for this block
    __shared__ int s_total[DISPATCH_MAX_EXPERTS];
    __shared__ unsigned s_first[DISPATCH_MAX_EXPERTS];    // first tile | first pair << 16 of each expert
    __shared__ unsigned s_warp[8];
    __shared__ int s_pos[DISPATCH_MAX_TOPK];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int m0 = blockIdx.x * a.chunk, m1 = min(a.M, m0 + a.chunk);
    const bool first = blockIdx.x == 0;
    grid_launch_dependents();
    constexpr int U = ONE ? 1 : 4;       // groups of 512 columns in flight
    const int n_chunks = a.D >> 4;
    const int n_blocks = (a.D + FP8_BLOCK - 1) / FP8_BLOCK;
    const int n_groups = (n_blocks + FP8_GROUP - 1) / FP8_GROUP;
    uint4 lo[U], hi[U];
    uint32_t byte[U];
    auto fetch = [&](int m, int g0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = (g0 + u) * 32 + lane;      // (g0 of a warp that shares its token: its own group)
            lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
            byte[u] = 127u;
            if (c < n_chunks) {
                if constexpr (ROWS8) {
                    lo[u] = __ldg(static_cast<const uint4*>(a.x) + static_cast<size_t>(m) * n_chunks + c);
                    byte[u] = __ldg(a.x_scale + static_cast<size_t>(m) * n_blocks + (c >> 3));
                } else {
                    const uint4* src = static_cast<const uint4*>(a.x) + (static_cast<size_t>(m) * n_chunks + c) * 2;
                    lo[u] = __ldg(src);
                    hi[u] = __ldg(src + 1);
                }
            }
        }
    };
    // the first columns are on their way while the layout is worked out
    const int m_first = ONE ? m0 : m0 + warp, g_first = ONE ? warp : 0;
    if (m_first < m1) fetch(m_first, g_first);
    if constexpr (SMALL) {
        for (int e = tid; e < a.N; e += 256) s_next[e] = s_total[e] = 0;
        __syncthreads();
        const int before = m0 * a.K;
        for (int i = tid; i < a.M * a.K; i += 256) {
            const int e = dispatch_expert(a, i, first);
            atomicAdd(&s_total[e], 1);
            if (i < before) atomicAdd(&s_next[e], 1);
        }
    } else {
        // experts that the chunk does not name have no entry in chunk_base: what is read there is not used
        for (int e = tid; e < a.N; e += 256) {
            s_total[e] = __ldg(a.total + e);
            s_next[e] = __ldg(a.chunk_base + static_cast<size_t>(blockIdx.x) * a.N + e);
        }
    }
    __syncthreads();
    // exclusive scan of tiles (low half) and tile pairs (high half) over the experts, four of them a thread
    unsigned mine[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int e = tid * 4 + j;
        const unsigned nt = e < a.N ? static_cast<unsigned>(s_total[e] + TILE_M - 1) / TILE_M : 0u;
        mine[j] = sum;
        sum += nt | ((nt + 1) / 2) << 16;
    }
    unsigned incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    unsigned base = incl - sum, all = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i < warp) base += s_warp[i];
        all += s_warp[i];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (tid * 4 + j < a.N) s_first[tid * 4 + j] = base + mine[j];
    __syncthreads();
    if (first && tid == 0) {
        a.sched[SCHED_N_TILES] = static_cast<int>(all & 0xFFFFu);
        a.sched[SCHED_N_SAVED_TILES] = 0;
        a.sched[SCHED_PAD_ROWS] = static_cast<int>((all & 0xFFFFu) * TILE_M);
        a.sched[SCHED_N_PAIRS] = static_cast<int>(all >> 16);
    }
    // the tables of the tiles: the experts are shared out among the blocks, a thread each
    for (int e = blockIdx.x + gridDim.x * tid; e < a.N; e += gridDim.x * 256) {
        const int cnt = s_total[e], t0 = static_cast<int>(s_first[e] & 0xFFFFu), p0 = static_cast<int>(s_first[e] >> 16);
        const int nt = (cnt + TILE_M - 1) / TILE_M;
        a.sizes[e] = cnt;
        for (int t = 0; t < nt; ++t) {
            a.tile_expert[t0 + t] = e;
            a.tile_rows[t0 + t] = min(cnt - t * TILE_M, TILE_M);
            if ((t & 1) == 0) a.pair_info[p0 + t / 2] = (t0 + t) * 2 + (t + 1 < nt ? 1 : 0);
        }
    }

    for (int m = m_first; m < m1; m += ONE ? 1 : 8) {
        int p = 0;
        if (lane < a.K && (!ONE || warp == 0)) {
            const int i = m * a.K + lane;
            const int e = dispatch_expert(a, i, false);
            p = static_cast<int>(s_first[e] & 0xFFFFu) * TILE_M + atomicAdd(&s_next[e], 1);
            a.pos[i] = p;
            a.row_weight[p] = __ldg(a.topk_w + i);
            if constexpr (ONE) s_pos[lane] = p;
        }
        if constexpr (ONE) {
            __syncthreads();             // a block has one token, so this runs once
            if (lane < a.K) p = s_pos[lane];
        }
        for (int g0 = g_first; g0 < n_groups; g0 += U * STEP) {
            if (g0 != g_first || m != m_first) fetch(m, g0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (g0 + u >= n_groups) break;
                const int c = (g0 + u) * 32 + lane;
                uint4 o = lo[u];
                if constexpr (!ROWS8) {
                    const uint32_t raw[8] = {lo[u].x, lo[u].y, lo[u].z, lo[u].w, hi[u].x, hi[u].y, hi[u].z, hi[u].w};
                    float v[16];
                    uint32_t top = 0u;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        v[2 * i] = __uint_as_float(raw[i] << 16);
                        v[2 * i + 1] = __uint_as_float(raw[i] & 0xFFFF0000u);
                        top = max(top, max(abs_bits(v[2 * i]), abs_bits(v[2 * i + 1])));
                    }
#pragma unroll
                    for (int d = 4; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
                    byte[u] = fp8_scale_byte(top);
                    o = fp8_convert16(v, fp8_inv_scale(byte[u]));
                }
                const uint32_t word = __reduce_or_sync(0xffffffffu, (lane & 7) == 0 ? byte[u] << lane : 0u);
                if (lane < a.K)
                    *reinterpret_cast<uint32_t*>(a.dst_scale + fp8_atom_offset(p, g0 + u, n_groups)) = word;
                for (int k = 0; k < a.K; ++k) {
                    const size_t row = static_cast<size_t>(__shfl_sync(0xffffffffu, p, k));
                    if (c < n_chunks) *reinterpret_cast<uint4*>(a.dst + row * a.D + static_cast<size_t>(c) * 16) = o;
                }
            }
        }
    }
}

// y[m, :] = bf16(sum over k of rows[pos[m, k], :] * scale), 32-bit sums in the order of k, one rounding.  A thread has
// 8 columns and all K rows in flight (8 at a time above 8, one by one took 101 against 84 us at 8192 tokens, D2048, top-12);
// bound by HBM: M (K + 1) D 2 bytes (104 us at 16384 tokens, D2048, top-8: 0.89 of the measured copy rate).
template <int KT>
__global__ void __launch_bounds__(256) fp8_combine_kernel(const uint4* __restrict__ rows, const float* __restrict__ scale,
                                                          const int* __restrict__ pos, int M, int K, int vec_per_row,
                                                          int n_scale, uint4* __restrict__ dst) {
    grid_wait();
    const long long total = static_cast<long long>(M) * vec_per_row;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
        const int m = static_cast<int>(i / vec_per_row);
        const int c = static_cast<int>(i - static_cast<long long>(m) * vec_per_row);
        const int* p = pos + static_cast<size_t>(m) * (KT > 0 ? KT : K);
        float a[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        auto add = [&](const uint4& q, float s) {
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                a[2 * j] = fmaf(f.x, s, a[2 * j]);
                a[2 * j + 1] = fmaf(f.y, s, a[2 * j + 1]);
            }
        };
        // U rows in flight
        constexpr int U = KT > 0 ? KT : 8;
        for (int k0 = 0; k0 < (KT > 0 ? KT : K); k0 += U) {
            uint4 q[U];
            float s[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (KT == 0 && k0 + k >= K) break;
                const size_t row = static_cast<size_t>(__ldca(p + k0 + k));
                q[k] = __ldcg(rows + row * vec_per_row + c);
                s[k] = __ldca(scale + row * n_scale + (c >> 5));
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (KT == 0 && k0 + k >= K) break;
                add(q[k], s[k]);
            }
        }
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a[2 * j], a[2 * j + 1]);
            o[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
        dst[i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

static int fp8_combine(const void* rows, const float* scale, const int32_t* pos, int M, int K, int D, void* y,
                       cudaStream_t st, bool dependent) {
    const int vec = D / 8, n_scale = (D + FP8_YBLOCK - 1) / FP8_YBLOCK;
    const long long want = (static_cast<long long>(M) * vec + 255) / 256, cap = sm_count() * 16;
    const int grid = static_cast<int>(want < cap ? want : cap);
    const uint4* r = static_cast<const uint4*>(rows);
    uint4* d = static_cast<uint4*>(y);
#define COMBINE(KT)                                                                                                    \
    if (dependent)                                                                                                     \
        return launch_dependent(fp8_combine_kernel<KT>, grid, 256, 0, st, 1, r, scale, pos, M, K, vec, n_scale, d) ==  \
               cudaSuccess ? MOMOE_OK : MOMOE_ERR_CUDA;                                                                \
    fp8_combine_kernel<KT><<<grid, 256, 0, st>>>(r, scale, pos, M, K, vec, n_scale, d);                                \
    break
    switch (K) {
        case 1: COMBINE(1);
        case 2: COMBINE(2);
        case 3: COMBINE(3);
        case 4: COMBINE(4);
        case 5: COMBINE(5);
        case 6: COMBINE(6);
        case 7: COMBINE(7);
        case 8: COMBINE(8);
        default: COMBINE(0);
    }
#undef COMBINE
    return cudaGetLastError() == cudaSuccess ? MOMOE_OK : MOMOE_ERR_CUDA;
}

static bool dispatch_small(int M, int K) { return static_cast<long long>(M) * K <= DISPATCH_SMALL_PAIRS; }
// Tokens of a block: one up to four blocks an SM, else one a warp, more where that makes more than four blocks an SM (a block
// has a set-up of its own).
static int dispatch_chunk(int M, int K) {
    const int want = (M + 4 * sm_count() - 1) / (4 * sm_count());
    if (want <= 1 && dispatch_small(M, K)) return 1;
    return (want + 7) / 8 * 8;
}

// Parts of the workspace of a whole forward pass, each on a 256-byte boundary.
struct Fp8Workspace {
    size_t tile_expert, pair_info, sched, tile_rows, row_weight, pos, dispatch, dispatch_bytes, x_scale, h, h_scale, rows,
        y_scale, bytes;
    long long tiles;
};
static Fp8Workspace fp8_workspace(int M, int N, int K, int D, int H) {
    Fp8Workspace w;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += (bytes + 255) & ~static_cast<size_t>(255);
        return o;
    };
    const size_t msum = static_cast<size_t>(M) * K;
    // an expert without a token has no tile: fewer than momoe_tile_capacity when there are fewer pairs than experts
    const size_t tiles = (msum + TILE_M - 1) / TILE_M + (msum < static_cast<size_t>(N) ? msum : N), rows = tiles * TILE_M;
    w.tiles = static_cast<long long>(tiles);
    w.tile_expert = take(tiles * 4);
    w.pair_info = take(tiles * 4);
    w.sched = take(SCHED_WORDS * 4);
    w.tile_rows = take(tiles * 4);
    w.row_weight = take(rows * 4);
    w.pos = take(msum * 4);
    w.dispatch_bytes = momoe_fp8_dispatch_workspace_bytes(M, N, K);
    w.dispatch = take(w.dispatch_bytes);
    w.x_scale = take(tiles * ((D + 511) / 512) * FP8_ATOM);
    w.h = take(rows * H);
    w.h_scale = take(tiles * ((H + 511) / 512) * FP8_ATOM);
    w.rows = take(rows * D * 2);     // 8-bit input rows, later the 16-bit result rows
    w.y_scale = take(rows * ((D + FP8_YBLOCK - 1) / FP8_YBLOCK) * 4);
    w.bytes = at;
    return w;
}

}  // namespace momoe

using namespace momoe;

#define MOMOE_API extern "C" __attribute__((visibility("default")))

MOMOE_API int momoe_fp8_quantize_weights(const void* W, int32_t type, int32_t N, int32_t Kd, int32_t groups, int32_t C,
                                         uint8_t* q, uint8_t* S, momoe_stream_t stream) {
    if (W == nullptr || q == nullptr || S == nullptr || N <= 0 || Kd <= 0 || groups <= 0 || C <= 0) return MOMOE_ERR_ARG;
    if ((type != 0 && type != 2) || Kd % 16 != 0) return MOMOE_ERR_UNSUPPORTED;
    const long long by = static_cast<long long>(groups) * ((C + 127LL) / 128);
    if (N > 65535 || by > 65535 || Kd > FP8_MAX_WIDTH) return MOMOE_ERR_TOO_LARGE;
    if ((reinterpret_cast<uintptr_t>(q) & 15) != 0) return MOMOE_ERR_ARG;
    const dim3 grid((Kd + 127) / 128, static_cast<unsigned>(by), N);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type == 0)
        fp8_quantize_weights_kernel<<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(W), Kd, groups, C, q, S);
    else
        fp8_quantize_weights_kernel<<<grid, 256, 0, st>>>(static_cast<const float*>(W), Kd, groups, C, q, S);
    return cudaGetLastError() == cudaSuccess ? MOMOE_OK : MOMOE_ERR_CUDA;
}

MOMOE_API size_t momoe_fp8_dispatch_workspace_bytes(int32_t M, int32_t N, int32_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || dispatch_small(M, K)) return 0;
    const int c = dispatch_chunk(M, K);
    return (1 + static_cast<size_t>((M + c - 1) / c)) * N * 4;
}

MOMOE_API int momoe_fp8_dispatch_rows(const void* x, const uint8_t* x_scale, const int32_t* topk_idx_MK,
                                      const float* topk_w_MK, int32_t M, int32_t N, int32_t K, int32_t D,
                                      int64_t* sizes_N, int32_t* tile_expert, int32_t* pair_info, int32_t* sched,
                                      int32_t* tile_rows, float* row_weight, int32_t* pos_MK, int64_t rows_capacity,
                                      void* workspace, size_t workspace_bytes, uint8_t* dst_sorted, uint8_t* dst_scale,
                                      int32_t* status, momoe_stream_t stream) {
    if (x == nullptr || topk_idx_MK == nullptr || topk_w_MK == nullptr || sizes_N == nullptr || tile_expert == nullptr ||
        pair_info == nullptr || sched == nullptr || tile_rows == nullptr || row_weight == nullptr || pos_MK == nullptr ||
        dst_sorted == nullptr || dst_scale == nullptr || status == nullptr)
        return MOMOE_ERR_ARG;
    if (M <= 0 || N <= 0 || K <= 0 || K > N || D <= 0) return MOMOE_ERR_ARG;
    if (D % 16 != 0) return MOMOE_ERR_UNSUPPORTED;
    if (N > DISPATCH_MAX_EXPERTS || K > DISPATCH_MAX_TOPK || D > FP8_MAX_WIDTH) return MOMOE_ERR_TOO_LARGE;
    // tiles and pairs share a word in the scan
    const int64_t msum = static_cast<int64_t>(M) * K, tiles = (msum + TILE_M - 1) / TILE_M + (msum < N ? msum : N);
    if (tiles > 0xFFFF) return MOMOE_ERR_TOO_LARGE;
    if (rows_capacity < tiles * TILE_M) return MOMOE_ERR_ARG;
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(dst_sorted) |
          reinterpret_cast<uintptr_t>(dst_scale)) & 15) != 0)
        return MOMOE_ERR_ARG;
    const size_t need = momoe_fp8_dispatch_workspace_bytes(M, N, K);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return MOMOE_ERR_ARG;
    DispatchArgs a;
    a.x = x; a.x_scale = x_scale; a.topk_idx = topk_idx_MK; a.topk_w = topk_w_MK;
    a.M = M; a.N = N; a.K = K; a.D = D;
    a.chunk = dispatch_chunk(M, K);
    a.total = static_cast<int*>(workspace);
    a.chunk_base = need > 0 ? a.total + N : nullptr;
    a.sizes = reinterpret_cast<long long*>(sizes_N);
    a.tile_expert = tile_expert; a.pair_info = pair_info; a.sched = sched;
    a.tile_rows = tile_rows; a.row_weight = row_weight; a.pos = pos_MK;
    a.dst = dst_sorted; a.dst_scale = dst_scale; a.status = status;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int grid = (M + a.chunk - 1) / a.chunk;
    if (a.chunk == 1) {
        if (x_scale != nullptr) fp8_dispatch_kernel<true, true, true><<<grid, 256, 0, st>>>(a);
        else fp8_dispatch_kernel<false, true, true><<<grid, 256, 0, st>>>(a);
    } else if (need == 0) {
        if (x_scale != nullptr) fp8_dispatch_kernel<true, true, false><<<grid, 256, 0, st>>>(a);
        else fp8_dispatch_kernel<false, true, false><<<grid, 256, 0, st>>>(a);
    } else {
        if (cudaMemsetAsync(a.total, 0, static_cast<size_t>(N) * 4, st) != cudaSuccess) return MOMOE_ERR_CUDA;
        fp8_count_kernel<<<grid, 256, 0, st>>>(a);
        if (x_scale != nullptr) fp8_dispatch_kernel<true, false, false><<<grid, 256, 0, st>>>(a);
        else fp8_dispatch_kernel<false, false, false><<<grid, 256, 0, st>>>(a);
    }
    return cudaGetLastError() == cudaSuccess ? MOMOE_OK : MOMOE_ERR_CUDA;
}

MOMOE_API int momoe_fp8_combine_rows(const void* y_sorted, const float* y_scale, const int32_t* pos_MK, int32_t M, int32_t K,
                                     int32_t D, void* y_MD, momoe_stream_t stream) {
    if (y_sorted == nullptr || y_scale == nullptr || pos_MK == nullptr || y_MD == nullptr || M <= 0 || K <= 0 || D <= 0)
        return MOMOE_ERR_ARG;
    if (D % 8 != 0) return MOMOE_ERR_UNSUPPORTED;
    if (((reinterpret_cast<uintptr_t>(y_sorted) | reinterpret_cast<uintptr_t>(y_MD)) & 15) != 0) return MOMOE_ERR_ARG;
    return fp8_combine(y_sorted, y_scale, pos_MK, M, K, D, y_MD, static_cast<cudaStream_t>(stream), false);
}

MOMOE_API size_t momoe_fp8_experts_workspace_bytes(int32_t M, int32_t N, int32_t K, int32_t D, int32_t H) {
    if (M <= 0 || N <= 0 || K <= 0 || D <= 0 || H <= 0) return 0;
    return fp8_workspace(M, N, K, D, H).bytes;
}

MOMOE_API int momoe_fp8_experts_launches(int32_t M, int32_t N, int32_t K) {
    (void)N;
    return dispatch_small(M, K) ? 4 : 5;
}

MOMOE_API int momoe_fp8_experts_forward(const void* x_MD, const uint8_t* x_scale, const int32_t* topk_idx_MK,
                                        const float* topk_w_MK, int32_t M, int32_t N, int32_t K, int32_t D, int32_t H,
                                        const uint8_t* W1_N2HD, const uint8_t* S1, const uint8_t* W2_NDH,
                                        const uint8_t* S2, int32_t stream_max_avg_rows, void* y_MD, int64_t* sizes_N,
                                        void* workspace, size_t workspace_bytes, int32_t* status,
                                        momoe_stream_t stream) {
    if (M <= 0 || N <= 0 || K <= 0 || D <= 0 || H <= 0) return MOMOE_ERR_ARG;
    if (D % 16 != 0 || H % 16 != 0) return MOMOE_ERR_UNSUPPORTED;
    if (D > FP8_MAX_WIDTH || H > FP8_MAX_WIDTH) return MOMOE_ERR_TOO_LARGE;
    if (x_MD == nullptr || y_MD == nullptr || workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)
        return MOMOE_ERR_ARG;
    const Fp8Workspace l = fp8_workspace(M, N, K, D, H);
    if (workspace_bytes < l.bytes) return MOMOE_ERR_ARG;
    char* ws = static_cast<char*>(workspace);
    auto i32 = [&](size_t at) { return reinterpret_cast<int32_t*>(ws + at); };
    auto u8 = [&](size_t at) { return reinterpret_cast<uint8_t*>(ws + at); };
    momoe_plan_t plan;
    plan.M = M; plan.N = N; plan.K = K; plan.D = D; plan.H = H; plan.reserved = 0;
    plan.rows_capacity = l.tiles * TILE_M;
    plan.sched = i32(l.sched);
    plan.tile_expert = i32(l.tile_expert);
    plan.pad_off = nullptr;
    plan.row_token = nullptr;
    plan.row_weight = reinterpret_cast<float*>(ws + l.row_weight);
    plan.pos_MK = i32(l.pos);
    plan.status = status;
    plan.pair_info = i32(l.pair_info);
    int rc = momoe_fp8_dispatch_rows(x_MD, x_scale, topk_idx_MK, topk_w_MK, M, N, K, D, sizes_N, i32(l.tile_expert),
                                     i32(l.pair_info), i32(l.sched), i32(l.tile_rows),
                                     reinterpret_cast<float*>(ws + l.row_weight), i32(l.pos), plan.rows_capacity,
                                     ws + l.dispatch, l.dispatch_bytes, u8(l.rows), u8(l.x_scale), status, stream);
    if (rc != MOMOE_OK) return rc;
    // with few rows an expert, the kernels that stream the weights
    const bool decode = static_cast<int64_t>(M) * K <= static_cast<int64_t>(stream_max_avg_rows) * N;
    const auto up = decode ? momoe_fp8_up_swiglu_decode : momoe_fp8_up_swiglu;
    const auto down = decode ? momoe_fp8_down_scale_decode : momoe_fp8_down_scale;
    rc = up(&plan, i32(l.tile_rows), u8(l.rows), u8(l.x_scale), W1_N2HD, S1, u8(l.h), u8(l.h_scale), stream);
    if (rc != MOMOE_OK) return rc;
    float* y_scale = reinterpret_cast<float*>(ws + l.y_scale);
    rc = down(&plan, i32(l.tile_rows), u8(l.h), u8(l.h_scale), W2_NDH, S2, ws + l.rows, y_scale, stream);
    if (rc != MOMOE_OK) return rc;
    // launched early beside the tile kernel its blocks wait there for long and slow it down (1124 against 1098 us at 16384
    // tokens, D2048 H1024, top-8 of 128); behind the streaming kernel it saves a launch gap (30.7 against 32.5 us, 1 token)
    return fp8_combine(ws + l.rows, y_scale, plan.pos_MK, M, K, D, y_MD, static_cast<cudaStream_t>(stream), decode);
}
