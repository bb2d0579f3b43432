// Around the 8-bit expert GEMMs: the weights' conversion, the row gather that converts on the way, and one call that runs
// the whole forward pass (permutation, gather, two GEMMs, combine) out of one workspace.
#include "fp8.cuh"
#include "internal.h"
#include "../../include/momoe_b200.h"

namespace momoe {

int fp8_check_plan(const momoe_plan_t* p);

__device__ __forceinline__ float f8_value(float v) { return v; }
__device__ __forceinline__ float f8_value(__nv_bfloat16 v) { return __bfloat162float(v); }

// W [N, Kd, G * C] -> q [N, G * C, Kd] (k contiguous, as the MMA reads it) and one scale for each 128 x 128 block
// [N, G, ceil(C / 128), ceil(Kd / 128)].  A block of columns never crosses a group (the linear and the gate half of the
// up projection).  Runs once when a model is loaded; bound by HBM, one read and one write of the weights.
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

// One warp a token: its row is read once, converted (ROWS8: copied) and stored to the K expert-major rows of its experts,
// the scales in the blocks the GEMMs read.  A lane holds 16 columns, 8 lanes a block of 128, the warp the 512 columns
// whose four scale bytes make one word.  Bound by HBM: M D (2 + K) bytes from 16-bit rows, M D (1 + K) from 8-bit ones.
// Padding rows are left as they are.  A token that names an expert twice would have both copies in one row: reported.
template <bool ROWS8>
__global__ void __launch_bounds__(256) fp8_gather_kernel(const void* __restrict__ x, const uint8_t* __restrict__ x_scale,
                                                         const int* __restrict__ pos_MK, int M, int K, int D,
                                                         uint8_t* __restrict__ dst, uint8_t* __restrict__ dst_scale,
                                                         int* status) {
    constexpr int U = 4;             // groups of 512 columns in flight
    const int lane = threadIdx.x & 31;
    const int warps_total = gridDim.x * 8;
    const int n_chunks = D >> 4;
    const int n_blocks = (D + FP8_BLOCK - 1) / FP8_BLOCK;
    const int n_groups = (n_blocks + FP8_GROUP - 1) / FP8_GROUP;
    for (int m = blockIdx.x * 8 + (threadIdx.x >> 5); m < M; m += warps_total) {
        const int p = lane < K ? __ldg(pos_MK + static_cast<size_t>(m) * K + lane) : -1 - lane;
        const unsigned same = __match_any_sync(0xffffffffu, p);
        if ((same & (same - 1u)) != 0u) atomicCAS(status, 0, DEV_REPEATED_EXPERT);
        for (int g0 = 0; g0 < n_groups; g0 += U) {
            uint4 lo[U], hi[U];
            uint32_t byte[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = (g0 + u) * 32 + lane;
                lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
                byte[u] = 127u;
                if (c < n_chunks) {
                    if constexpr (ROWS8) {
                        lo[u] = __ldg(static_cast<const uint4*>(x) + static_cast<size_t>(m) * n_chunks + c);
                        byte[u] = __ldg(x_scale + static_cast<size_t>(m) * n_blocks + (c >> 3));
                    } else {
                        const uint4* src = static_cast<const uint4*>(x) + (static_cast<size_t>(m) * n_chunks + c) * 2;
                        lo[u] = __ldg(src);
                        hi[u] = __ldg(src + 1);
                    }
                }
            }
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
                    const float inv = fp8_inv_scale(byte[u]);
                    o.x = fp8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                    o.y = fp8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
                    o.z = fp8_pack4(v[8] * inv, v[9] * inv, v[10] * inv, v[11] * inv);
                    o.w = fp8_pack4(v[12] * inv, v[13] * inv, v[14] * inv, v[15] * inv);
                }
                const uint32_t word = __reduce_or_sync(0xffffffffu, (lane & 7) == 0 ? byte[u] << lane : 0u);
                if (lane < K)
                    *reinterpret_cast<uint32_t*>(dst_scale + fp8_atom_offset(p, g0 + u, n_groups)) = word;
                for (int k = 0; k < K; ++k) {
                    const size_t row = static_cast<size_t>(__shfl_sync(0xffffffffu, p, k));
                    if (c < n_chunks) *reinterpret_cast<uint4*>(dst + row * D + static_cast<size_t>(c) * 16) = o;
                }
            }
        }
    }
}

// Parts of the workspace of a whole forward pass, each on a 256-byte boundary.
struct Fp8Workspace {
    size_t cumsums, idx, which, pad_off, tile_expert, pair_info, sched, row_token, row_weight, pos, perm, x_scale, h,
        h_scale, rows, bytes;
};
static Fp8Workspace fp8_workspace(int M, int N, int K, int D, int H) {
    Fp8Workspace w;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += (bytes + 255) & ~static_cast<size_t>(255);
        return o;
    };
    const size_t tiles = static_cast<size_t>(momoe_tile_capacity(M, K, N)), rows = tiles * TILE_M;
    const size_t msum = static_cast<size_t>(M) * K;
    w.cumsums = take((N + 1) * 4);
    w.idx = take(msum * 4);
    w.which = take(msum * 4);
    w.pad_off = take((N + 1) * 4);
    w.tile_expert = take(tiles * 4);
    w.pair_info = take(tiles * 4);
    w.sched = take(SCHED_WORDS * 4);
    w.row_token = take(rows * 4);
    w.row_weight = take(rows * 4);
    w.pos = take(msum * 4);
    w.perm = take(momoe_permutation_workspace_bytes(M, N, K));
    w.x_scale = take(tiles * ((D + 511) / 512) * FP8_ATOM);
    w.h = take(rows * H);
    w.h_scale = take(tiles * ((H + 511) / 512) * FP8_ATOM);
    w.rows = take(rows * D * 2);     // 8-bit input rows, later the 16-bit result rows
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
    const long long by = static_cast<long long>(groups) * ((C + 127) / 128);
    if (N > 65535 || by > 65535) return MOMOE_ERR_TOO_LARGE;
    if ((reinterpret_cast<uintptr_t>(q) & 15) != 0) return MOMOE_ERR_ARG;
    const dim3 grid((Kd + 127) / 128, static_cast<unsigned>(by), N);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type == 0)
        fp8_quantize_weights_kernel<<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(W), Kd, groups, C, q, S);
    else
        fp8_quantize_weights_kernel<<<grid, 256, 0, st>>>(static_cast<const float*>(W), Kd, groups, C, q, S);
    return cudaGetLastError() == cudaSuccess ? MOMOE_OK : MOMOE_ERR_CUDA;
}

MOMOE_API int momoe_fp8_gather_rows(const momoe_plan_t* plan, const void* x, const uint8_t* x_scale, uint8_t* dst_sorted,
                                    uint8_t* dst_scale, momoe_stream_t stream) {
    int rc = fp8_check_plan(plan);
    if (rc != MOMOE_OK) return rc;
    if (x == nullptr || dst_sorted == nullptr || dst_scale == nullptr) return MOMOE_ERR_ARG;
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(dst_sorted) |
          reinterpret_cast<uintptr_t>(dst_scale)) & 15) != 0)
        return MOMOE_ERR_ARG;
    if (plan->K > 32) return MOMOE_ERR_TOO_LARGE;
    const int want = (plan->M + 7) / 8, cap = sm_count() * 8;
    const int grid = want < cap ? want : cap;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (x_scale != nullptr)
        fp8_gather_kernel<true><<<grid, 256, 0, st>>>(x, x_scale, plan->pos_MK, plan->M, plan->K, plan->D, dst_sorted,
                                                      dst_scale, plan->status);
    else
        fp8_gather_kernel<false><<<grid, 256, 0, st>>>(x, x_scale, plan->pos_MK, plan->M, plan->K, plan->D, dst_sorted,
                                                       dst_scale, plan->status);
    return cudaGetLastError() == cudaSuccess ? MOMOE_OK : MOMOE_ERR_CUDA;
}

MOMOE_API size_t momoe_fp8_experts_workspace_bytes(int32_t M, int32_t N, int32_t K, int32_t D, int32_t H) {
    if (M <= 0 || N <= 0 || K <= 0 || D <= 0 || H <= 0) return 0;
    return fp8_workspace(M, N, K, D, H).bytes;
}

MOMOE_API int momoe_fp8_experts_launches(int32_t M, int32_t N, int32_t K) {
    return momoe_permutation_launches(M, N, K) + 4;
}

MOMOE_API int momoe_fp8_experts_forward(const void* x_MD, const uint8_t* x_scale, const int32_t* topk_idx_MK,
                                        const float* topk_w_MK, int32_t M, int32_t N, int32_t K, int32_t D, int32_t H,
                                        const uint8_t* W1_N2HD, const uint8_t* S1, const uint8_t* W2_NDH,
                                        const uint8_t* S2, int32_t decode_max_avg_rows, void* y_MD, int64_t* sizes_N,
                                        void* workspace, size_t workspace_bytes, int32_t* status,
                                        momoe_stream_t stream) {
    if (M <= 0 || N <= 0 || K <= 0 || D <= 0 || H <= 0) return MOMOE_ERR_ARG;
    if (D % 16 != 0 || H % 16 != 0) return MOMOE_ERR_UNSUPPORTED;
    if (x_MD == nullptr || y_MD == nullptr || workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)
        return MOMOE_ERR_ARG;
    const Fp8Workspace l = fp8_workspace(M, N, K, D, H);
    if (workspace_bytes < l.bytes) return MOMOE_ERR_ARG;
    char* ws = static_cast<char*>(workspace);
    auto i32 = [&](size_t at) { return reinterpret_cast<int32_t*>(ws + at); };
    auto u8 = [&](size_t at) { return reinterpret_cast<uint8_t*>(ws + at); };
    momoe_plan_t plan;
    plan.M = M; plan.N = N; plan.K = K; plan.D = D; plan.H = H; plan.reserved = 0;
    plan.rows_capacity = momoe_sorted_rows_capacity(M, K, N);
    plan.sched = i32(l.sched);
    plan.tile_expert = i32(l.tile_expert);
    plan.pad_off = i32(l.pad_off);
    plan.row_token = i32(l.row_token);
    plan.row_weight = reinterpret_cast<float*>(ws + l.row_weight);
    plan.pos_MK = i32(l.pos);
    plan.status = status;
    plan.pair_info = i32(l.pair_info);
    int rc = momoe_build_permutation(topk_idx_MK, topk_w_MK, M, N, K, 0, sizes_N, i32(l.cumsums), i32(l.idx),
                                     i32(l.which), i32(l.pad_off), i32(l.tile_expert), i32(l.pair_info), i32(l.sched),
                                     i32(l.row_token), reinterpret_cast<float*>(ws + l.row_weight), i32(l.pos),
                                     plan.rows_capacity, ws + l.perm, l.x_scale - l.perm, status, stream);
    if (rc != MOMOE_OK) return rc;
    if ((rc = momoe_fp8_gather_rows(&plan, x_MD, x_scale, u8(l.rows), u8(l.x_scale), stream)) != MOMOE_OK) return rc;
    // as for 16-bit experts: with few rows an expert, the kernels that stream the weights
    const bool decode = static_cast<int64_t>(M) * K <= static_cast<int64_t>(decode_max_avg_rows) * N;
    rc = decode ? momoe_fp8_up_swiglu_decode(&plan, u8(l.rows), u8(l.x_scale), W1_N2HD, S1, u8(l.h), u8(l.h_scale), stream)
                : momoe_fp8_up_swiglu(&plan, u8(l.rows), u8(l.x_scale), W1_N2HD, S1, u8(l.h), u8(l.h_scale), stream);
    if (rc != MOMOE_OK) return rc;
    rc = decode ? momoe_fp8_down_scale_decode(&plan, u8(l.h), u8(l.h_scale), W2_NDH, S2, ws + l.rows, stream)
                : momoe_fp8_down_scale(&plan, u8(l.h), u8(l.h_scale), W2_NDH, S2, ws + l.rows, stream);
    if (rc != MOMOE_OK) return rc;
    return momoe_combine_rows(&plan, ws + l.rows, D, y_MD, stream);
}
