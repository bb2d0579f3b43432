// Root-mean-square norm with the residual's addition, its backward pass, and an 8-bit output.
//
//   r = round(x + residual)            (rounded once, to the stream's type; the norm sees the rounded value, so that the
//                                       backward pass, which reads r, differentiates exactly what the forward computed)
//   y = r * rstd * w,   rstd = 1 / sqrt(mean(r^2) + eps)
//   q, scale: the same y, before its rounding, as e4m3 with a power of two for each 128 columns
//
//   backward, with gh = gy * w, xhat = r * rstd:  gx = rstd * (gh - xhat * mean(gh * xhat)) + gr,  gw = sum over rows of
//   gy * xhat.  gx is the gradient of x and of the residual alike.
//
// Everything is bound by HBM: each tensor crosses it once, a row lives in registers between its two uses.  A row belongs
// to a warp up to 512 columns and to a thread block above; a thread holds 2 chunks of 8 columns (4 above 8192 columns), so
// that a block has few idle threads at widths between powers of two and enough blocks fit an SM to keep 60 KiB and more
// in flight.  Sums are 32-bit.  Of the measured copy rate: 8-bit output 0.94 (8192 x 7168 bf16, 86 us), forward 0.98 and
// backward 0.84 without its 4.5 us of partial sums (16384 x 2048 bf16, 42 and 48 us).
#include <cmath>

#include "fp8.cuh"
#include "internal.h"
#include "../../include/momoe_b200.h"

namespace momoe {

constexpr int NORM_MAX_THREADS = 512;
constexpr int NORM_MAX_D = NORM_MAX_THREADS * 4 * 8;
constexpr int QUANT_MAX_D = 1 << 30;         // column numbers too, with room for the rest of a block
constexpr int NORM_MAX_M = 1 << 30;          // row numbers stay inside 32 bits, with room for a step past the last row

// How a row of n chunks is shared out: chunks a thread holds, threads of a row, rows of a block.
struct NormShape {
    int ch, tpr, rows;
};
static NormShape norm_shape(int D) {
    const int n = D >> 3;
    if (n <= 64) return {2, 32, 4};
    const int ch = n <= 2 * NORM_MAX_THREADS ? 2 : 4;
    return {ch, ((n + ch - 1) / ch + 31) / 32 * 32, 1};
}

__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Sum over the threads of a row (a warp, or the whole block); every one of them gets it.  `buf` is written again only
// after the next barrier.
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float v, float* buf) {
    v = lanes_sum(v);
    if constexpr (BLOCK) {
        const int n = blockDim.x >> 5, lane = threadIdx.x & 31;
        __syncthreads();
        if (lane == 0) buf[threadIdx.x >> 5] = v;
        __syncthreads();
        v = lanes_sum(lane < n ? buf[lane] : 0.0f);
    }
    return v;
}

template <typename T>
struct NormArgs {
    const T* x;
    const T* res;        // may be null
    long long x_stride, res_stride;
    const void* w;
    int w_fp32;
    int M, D;
    float eps;
    T* r;                // null when there is no residual
    T* y;                // may be null (8-bit output only)
    float* rstd;         // may be null
    uint8_t* q;          // may be null
    uint8_t* scale;
};

template <typename T>
__device__ __forceinline__ void load_weight8(const void* w, int w_fp32, int col, float (&v)[8]) {
    if (w_fp32) load8(static_cast<const float*>(w) + col, v);
    else load8(static_cast<const T*>(w) + col, v);
}

template <typename T, int CH, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? NORM_MAX_THREADS : 128) rms_norm_kernel(const NormArgs<T> g) {
    __shared__ float buf[32];
    const int TPR = BLOCK ? blockDim.x : 32;
    const int t = BLOCK ? threadIdx.x : threadIdx.x & 31;
    const int m = BLOCK ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 5);
    if (m >= g.M) return;                       // whole warps leave, and only where a row is a warp's
    const int n_chunks = g.D >> 3;
    const T* x = g.x + m * g.x_stride;
    Raw8<T> rx[CH], re[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = t + i * TPR;
        if (c < n_chunks) rx[i].load(x + c * 8);
    }
    if (g.res != nullptr) {
        const T* res = g.res + m * g.res_stride;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c = t + i * TPR;
            if (c < n_chunks) re[i].load(res + c * 8);
        }
    }
    float v[CH][8];
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = t + i * TPR;
        if (c >= n_chunks) continue;
        rx[i].unpack(v[i]);
        if (g.res != nullptr) {
            float a[8];
            re[i].unpack(a);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] += a[j];
            store8(g.r + static_cast<size_t>(m) * g.D + c * 8, v[i]);        // leaves the rounded sum in v
        }
    }
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if (t + i * TPR < n_chunks) {
#pragma unroll
            for (int j = 0; j < 8; ++j) sq = fmaf(v[i][j], v[i][j], sq);
        }
    sq = row_sum<BLOCK>(sq, buf);
    const float rstd = 1.0f / sqrtf(sq / static_cast<float>(g.D) + g.eps);
    if (t == 0 && g.rstd != nullptr) g.rstd[m] = rstd;
    const int n_blocks = (g.D + FP8_BLOCK - 1) / FP8_BLOCK;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = t + i * TPR;
        if (c - (t & 31) >= n_chunks) break;    // the whole warp is past the row's end
        const bool in = c < n_chunks;
        if (in) {
            float w[8];
            load_weight8<T>(g.w, g.w_fp32, c * 8, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * rstd * w[j];
        }
        if (g.q != nullptr) {
            // 16 consecutive lanes hold a block of 128 columns
            uint32_t top = 0u;
            if (in) {
#pragma unroll
                for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[i][j]));
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const uint32_t byte = fp8_scale_byte(top);
            if (in) {
                const float inv = fp8_inv_scale(byte);
                uint2 p;
                p.x = fp8_pack4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
                p.y = fp8_pack4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
                *reinterpret_cast<uint2*>(g.q + static_cast<size_t>(m) * g.D + c * 8) = p;
                if ((c & 15) == 0) g.scale[static_cast<size_t>(m) * n_blocks + (c >> 4)] = static_cast<uint8_t>(byte);
            }
        }
        if (in && g.y != nullptr) store8(g.y + static_cast<size_t>(m) * g.D + c * 8, v[i]);
    }
}

// ------------------------------------------------------------------------------------------------ backward
// Every group (a warp or a block) walks rows g, g + G, g + 2G, ... and keeps the weight's gradient of its columns in
// registers; the groups' partial sums go to `part` [G, D] and a second kernel adds them in a fixed order, so the result
// does not depend on timing.
template <typename T>
struct NormBwdArgs {
    const T* gy;
    const T* gr;         // may be null
    const T* r;
    long long r_stride;
    const void* w;
    int w_fp32;
    const float* rstd;
    int M, D, G;
    T* gx;
    float* part;         // null: no weight gradient
};

// AHEAD: a row is asked for while the one before is worked on.  That pays where a block is so large that an SM holds one.
// Backward kernel without and with it: 69 / 51 us (4096 x 8192 fp16), 64 / 46 (4096 x 7168 bf16); but 48 / 55 us with six
// blocks an SM (16384 x 2048 bf16), since it costs registers.
template <typename T, int CH, bool BLOCK, bool AHEAD>
__global__ void __launch_bounds__(BLOCK ? NORM_MAX_THREADS : 128) rms_norm_backward_kernel(const NormBwdArgs<T> g) {
    __shared__ float buf[32];
    const int TPR = BLOCK ? blockDim.x : 32;
    const int t = BLOCK ? threadIdx.x : threadIdx.x & 31;
    const int group = BLOCK ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 5);
    if (group >= g.G) return;
    const int n_chunks = g.D >> 3;
    const float inv_d = 1.0f / static_cast<float>(g.D);
    float gw[CH][8];
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) gw[i][j] = 0.0f;
    // all three tensors are asked for before the first is used (with 4 chunks there is no room to hold the third)
    Raw8<T> ny[CH], nr[CH], ne[CH];
    float n_rstd = 0.0f;
    auto fetch = [&](int m) {
        const T* gy = g.gy + static_cast<size_t>(m) * g.D;
        const T* gr = g.gr + static_cast<size_t>(m) * g.D;
        const T* r = g.r + m * g.r_stride;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c = t + i * TPR;
            if (c < n_chunks) {
                ny[i].load(gy + c * 8);
                nr[i].load(r + c * 8);
                if (CH <= 2 && g.gr != nullptr) ne[i].load(gr + c * 8);
            }
        }
        n_rstd = g.rstd[m];
    };
    if (AHEAD && group < g.M) fetch(group);
#pragma unroll 1
    for (int m = group; m < g.M; m += g.G) {
        const T* gr = g.gr + static_cast<size_t>(m) * g.D;
        if (!AHEAD) fetch(m);
        Raw8<T> ry[CH], rr[CH], re[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            ry[i] = ny[i];
            rr[i] = nr[i];
            re[i] = ne[i];
        }
        const float rstd = n_rstd;
        if (AHEAD && m + g.G < g.M) fetch(m + g.G);
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c = t + i * TPR;
            if (c < n_chunks) {
                float w[8], a[8], b[8];
                load_weight8<T>(g.w, g.w_fp32, c * 8, w);
                ry[i].unpack(a);
                rr[i].unpack(b);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    b[j] *= rstd;                              // xhat
                    gw[i][j] = fmaf(a[j], b[j], gw[i][j]);
                    dot = fmaf(a[j] * w[j], b[j], dot);        // gh * xhat
                }
            }
        }
        dot = row_sum<BLOCK>(dot, buf) * inv_d;
        T* gx = g.gx + static_cast<size_t>(m) * g.D;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c = t + i * TPR;
            if (c < n_chunks) {
                // gh and xhat again from the values as they were read: cheaper than registers to keep them
                float w[8], a[8], b[8], o[8];
                load_weight8<T>(g.w, g.w_fp32, c * 8, w);
                ry[i].unpack(a);
                rr[i].unpack(b);
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = rstd * (a[j] * w[j] - b[j] * rstd * dot);
                if (g.gr != nullptr) {
                    float e[8];
                    if (CH > 2) re[i].load(gr + c * 8);
                    re[i].unpack(e);
#pragma unroll
                    for (int j = 0; j < 8; ++j) o[j] += e[j];
                }
                store8(gx + c * 8, o);
            }
        }
    }
    if (g.part != nullptr) {
        float* part = g.part + static_cast<size_t>(group) * g.D;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c = t + i * TPR;
            if (c < n_chunks) store8(part + c * 8, gw[i]);
        }
    }
}

// gw[d] = sum over g of part[g, d]: 32 columns a block, 32 threads down the groups for each.
template <typename W>
__global__ void __launch_bounds__(1024) rms_norm_weight_grad_kernel(const float* __restrict__ part, int G, int D,
                                                                    W* __restrict__ gw) {
    __shared__ float s[32][33];
    const int d = blockIdx.x * 32 + threadIdx.x;
    float v = 0.0f;
    if (d < D) {
#pragma unroll 8
        for (int i = threadIdx.y; i < G; i += 32) v += part[static_cast<size_t>(i) * D + d];
    }
    s[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    v = lanes_sum(s[threadIdx.x][threadIdx.y]);
    const int o = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && o < D) gw[o] = static_cast<W>(v);
}

// x -> q, scale without a norm: the same blocks of 128 columns.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, long long x_stride, int M, int D,
                                                            uint8_t* __restrict__ q, uint8_t* __restrict__ scale) {
    const int n_blocks = (D + FP8_BLOCK - 1) / FP8_BLOCK;
    const long long total = static_cast<long long>(M) * n_blocks;
    const int l = threadIdx.x & 15;
    // half a warp a block of 128 columns; both halves run the same number of turns because of the shuffles
    for (long long i0 = (blockIdx.x * 256LL + threadIdx.x) / 32 * 2; i0 < total; i0 += gridDim.x * 16LL) {
        const long long i = i0 + ((threadIdx.x >> 4) & 1);
        const long long m = i / n_blocks;
        const int b = static_cast<int>(i - m * n_blocks);
        const int col = b * FP8_BLOCK + l * 8;
        const bool in = i < total && col < D;
        float v[8];
        uint32_t top = 0u;
        if (in) {
            load8(x + m * x_stride + col, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[j]));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (!in) continue;
        const uint32_t byte = fp8_scale_byte(top);
        const float inv = fp8_inv_scale(byte);
        uint2 p;
        p.x = fp8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        p.y = fp8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
        *reinterpret_cast<uint2*>(q + m * D + col) = p;
        if (l == 0) scale[m * n_blocks + b] = static_cast<uint8_t>(byte);
    }
}

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Blocks of a row's size that an SM holds in the backward pass, at 80 registers a thread.
static int norm_resident(int tpr) { return 768 / tpr > 0 ? 768 / tpr : 1; }

// Groups of the backward pass: as many as are resident, no more, since each leaves a row of partial sums.
static int norm_groups(int M, int D) {
    const NormShape s = norm_shape(D);
    const int groups = sm_count() * norm_resident(s.tpr);
    return M < groups ? M : groups;
}

template <typename T>
static int norm_launch(const NormArgs<T>& g, cudaStream_t st) {
    const NormShape s = norm_shape(g.D);
    if (s.rows > 1) rms_norm_kernel<T, 2, false><<<(g.M + 3) / 4, 128, 0, st>>>(g);
    else if (s.ch == 2) rms_norm_kernel<T, 2, true><<<g.M, s.tpr, 0, st>>>(g);
    else rms_norm_kernel<T, 4, true><<<g.M, s.tpr, 0, st>>>(g);
    return cudaGetLastError() == cudaSuccess ? MOMOE_OK : MOMOE_ERR_CUDA;
}

template <typename T>
static int norm_backward_launch(const NormBwdArgs<T>& g, void* gw, cudaStream_t st) {
    const NormShape s = norm_shape(g.D);
    if (s.rows > 1) rms_norm_backward_kernel<T, 2, false, false><<<(g.G + 3) / 4, 128, 0, st>>>(g);
    else if (s.ch == 2 && norm_resident(s.tpr) > 1) rms_norm_backward_kernel<T, 2, true, false><<<g.G, s.tpr, 0, st>>>(g);
    else if (s.ch == 2) rms_norm_backward_kernel<T, 2, true, true><<<g.G, s.tpr, 0, st>>>(g);
    else rms_norm_backward_kernel<T, 4, true, false><<<g.G, s.tpr, 0, st>>>(g);
    if (gw != nullptr) {
        const dim3 grid((g.D + 31) / 32), block(32, 32);
        if (g.w_fp32) rms_norm_weight_grad_kernel<<<grid, block, 0, st>>>(g.part, g.G, g.D, static_cast<float*>(gw));
        else rms_norm_weight_grad_kernel<<<grid, block, 0, st>>>(g.part, g.G, g.D, static_cast<T*>(gw));
    }
    return cudaGetLastError() == cudaSuccess ? MOMOE_OK : MOMOE_ERR_CUDA;
}

template <typename T>
static NormArgs<T> norm_args(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                             const void* weight, int w_fp32, int M, int D, float eps, void* r, void* y, float* rstd,
                             uint8_t* q, uint8_t* scale) {
    return NormArgs<T>{static_cast<const T*>(x), static_cast<const T*>(residual), x_stride, residual_stride, weight,
                       w_fp32, M, D, eps, static_cast<T*>(r), static_cast<T*>(y), rstd, q, scale};
}
template <typename T>
static NormBwdArgs<T> norm_backward_args(const void* gy, const void* gr, const void* r, int64_t r_stride,
                                         const void* weight, int w_fp32, const float* rstd, int M, int D, int G,
                                         void* gx, float* part) {
    return NormBwdArgs<T>{static_cast<const T*>(gy), static_cast<const T*>(gr), static_cast<const T*>(r), r_stride,
                          weight, w_fp32, rstd, M, D, G, static_cast<T*>(gx), part};
}

// Shared checks of one tensor type: 0 bf16, 1 fp16, 2 fp32; the weight has the same type or is fp32.
static int norm_check(int32_t M, int32_t D, int32_t type, int32_t weight_type) {
    if (M < 0 || D <= 0) return MOMOE_ERR_ARG;
    if (type < 0 || type > 2 || (weight_type != type && weight_type != 2)) return MOMOE_ERR_UNSUPPORTED;
    if (D % 8 != 0) return MOMOE_ERR_UNSUPPORTED;
    if (D > NORM_MAX_D || M > NORM_MAX_M) return MOMOE_ERR_TOO_LARGE;
    return MOMOE_OK;
}

}  // namespace momoe

using namespace momoe;

#define MOMOE_API extern "C" __attribute__((visibility("default")))

MOMOE_API int momoe_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                             const void* weight, int32_t type, int32_t weight_type, int32_t M, int32_t D, float eps,
                             void* r, void* y, float* rstd, uint8_t* q, uint8_t* scale, momoe_stream_t stream) {
    int rc = norm_check(M, D, type, weight_type);
    if (rc != MOMOE_OK) return rc;
    if (M == 0) return MOMOE_OK;
    if (x == nullptr || weight == nullptr || (y == nullptr && q == nullptr)) return MOMOE_ERR_ARG;
    if ((residual != nullptr) != (r != nullptr) || (q != nullptr) != (scale != nullptr)) return MOMOE_ERR_ARG;
    if (x_stride < 0 || residual_stride < 0 || x_stride % 8 != 0 || residual_stride % 8 != 0) return MOMOE_ERR_ARG;
    if (!aligned16(x) || !aligned16(residual) || !aligned16(weight) || !aligned16(r) || !aligned16(y) ||
        (reinterpret_cast<uintptr_t>(q) & 7) != 0)
        return MOMOE_ERR_ARG;
    if (!(eps >= 0.0f)) return MOMOE_ERR_ARG;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int wf = weight_type == 2;
    if (type == 0)
        return norm_launch(norm_args<__nv_bfloat16>(x, x_stride, residual, residual_stride, weight, wf, M, D, eps, r, y,
                                                    rstd, q, scale), st);
    if (type == 1)
        return norm_launch(norm_args<__half>(x, x_stride, residual, residual_stride, weight, wf, M, D, eps, r, y, rstd,
                                             q, scale), st);
    return norm_launch(norm_args<float>(x, x_stride, residual, residual_stride, weight, wf, M, D, eps, r, y, rstd, q,
                                        scale), st);
}

MOMOE_API size_t momoe_rms_norm_backward_workspace_bytes(int32_t M, int32_t D) {
    if (M <= 0 || D <= 0) return 0;
    return static_cast<size_t>(norm_groups(M, D)) * D * sizeof(float);
}

MOMOE_API int momoe_rms_norm_backward(const void* gy, const void* gr, const void* r, int64_t r_stride,
                                      const void* weight, const float* rstd, int32_t type, int32_t weight_type,
                                      int32_t M, int32_t D, void* gx, void* gw, void* workspace,
                                      size_t workspace_bytes, momoe_stream_t stream) {
    int rc = norm_check(M, D, type, weight_type);
    if (rc != MOMOE_OK) return rc;
    if (M == 0) return MOMOE_ERR_ARG;   // nothing to launch: the caller clears gw itself
    if (gy == nullptr || r == nullptr || weight == nullptr || rstd == nullptr || gx == nullptr) return MOMOE_ERR_ARG;
    if (r_stride < 0 || r_stride % 8 != 0) return MOMOE_ERR_ARG;
    if (!aligned16(gy) || !aligned16(gr) || !aligned16(r) || !aligned16(weight) || !aligned16(gx) ||
        !aligned16(workspace))
        return MOMOE_ERR_ARG;
    if (gw != nullptr && (workspace == nullptr || workspace_bytes < momoe_rms_norm_backward_workspace_bytes(M, D)))
        return MOMOE_ERR_ARG;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int wf = weight_type == 2, G = norm_groups(M, D);
    float* part = gw != nullptr ? static_cast<float*>(workspace) : nullptr;
    if (type == 0)
        return norm_backward_launch(norm_backward_args<__nv_bfloat16>(gy, gr, r, r_stride, weight, wf, rstd, M, D, G,
                                                                      gx, part), gw, st);
    if (type == 1)
        return norm_backward_launch(norm_backward_args<__half>(gy, gr, r, r_stride, weight, wf, rstd, M, D, G, gx,
                                                               part), gw, st);
    return norm_backward_launch(norm_backward_args<float>(gy, gr, r, r_stride, weight, wf, rstd, M, D, G, gx, part), gw,
                                st);
}

MOMOE_API int momoe_quantize_rows(const void* x, int64_t x_stride, int32_t type, int32_t M, int32_t D, uint8_t* q,
                                  uint8_t* scale, momoe_stream_t stream) {
    if (M < 0 || D <= 0) return MOMOE_ERR_ARG;
    if (type < 0 || type > 2 || D % 8 != 0) return MOMOE_ERR_UNSUPPORTED;
    if (D > QUANT_MAX_D) return MOMOE_ERR_TOO_LARGE;
    if (M == 0) return MOMOE_OK;
    if (x == nullptr || q == nullptr || scale == nullptr) return MOMOE_ERR_ARG;
    if (x_stride < 0 || x_stride % 8 != 0 || !aligned16(x) || (reinterpret_cast<uintptr_t>(q) & 7) != 0)
        return MOMOE_ERR_ARG;
    const long long blocks128 = static_cast<long long>(M) * ((D + FP8_BLOCK - 1) / FP8_BLOCK);
    const long long want = (blocks128 + 15) / 16, cap = sm_count() * 8;
    const int grid = static_cast<int>(want < cap ? want : cap);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type == 0)
        quantize_rows_kernel<<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(x), x_stride, M, D, q, scale);
    else if (type == 1)
        quantize_rows_kernel<<<grid, 256, 0, st>>>(static_cast<const __half*>(x), x_stride, M, D, q, scale);
    else
        quantize_rows_kernel<<<grid, 256, 0, st>>>(static_cast<const float*>(x), x_stride, M, D, q, scale);
    return cudaGetLastError() == cudaSuccess ? MOMOE_OK : MOMOE_ERR_CUDA;
}
