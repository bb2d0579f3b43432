// The experts' two 8-bit forward GEMMs for token batches with few rows an expert, sm_100a.
//
// Bound by the weights' way across HBM: 3 D H bytes for each touched expert.  As in the 16-bit kernels for this case the
// WEIGHTS are the M side of the MMA (128 weight rows = 128 TMEM lanes) and the tokens its N side, so that shared memory
// holds weights in flight and not padding rows.  Two forms:
//   NT = 32   up to 16 rows an expert: 6 stages x 32 KiB of weights (up), 5 x 32 KiB (down); an expert with more rows takes a
//             pass over its weights for each 32 of them
//   NT = 128  more rows: a whole 128-row tile in one pass, the MMA's N is the tile's 32-row blocks that hold real rows;
//             4 stages x 32 KiB of weights beside 16 KiB of rows
//
//   up    an item is 128 columns of h: two MMAs a k slice, the linear rows and the gate rows of W1[e], into two accumulators
//         whose lane j holds a[j] and b[j] of the same column, so the epilogue thread has both; h needs the maximum over
//         the item's 128 columns (the scale of 8-bit rows): a warp reduction for each token and one meeting of four warps
//   down  an item is 128 columns of y (NT = 32), or 256 in two MMAs, so that a row crosses from L2 half as often (NT = 128)
//
// One CTA (320 threads) an SM, persistent over items = (128-row tile, column block).  Warp 0 loads, warp 1 issues MMAs,
// warps 2..5 are the epilogue (a thread has one weight column and 32 tokens at a time), warps 6..9 write scales to TMEM
// (see the row-tile kernel).  With NT = 128 there is one accumulator: the MMAs of an item wait for
// the read-out of the item before, while the ring goes on filling; they need less than half of the time that the
// weights take.
#include <cstring>

#include "fp8.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "../../include/momoe_b200.h"

namespace momoe {

int fp8_check_plan(const momoe_plan_t* p);

constexpr int D8_THREADS = 320;
constexpr int D8_K = 128;                        // values of a k slice
constexpr int D8_W = 128 * D8_K;                 // 16 KiB: 128 weight rows
constexpr int D8_X = 32 * D8_K;                  // 4 KiB: 32 token rows

template <bool UP, int NT>
struct D8 {
    static constexpr int NW = UP || NT > 32 ? 2 : 1;         // weight blocks of 128 rows an item has
    static constexpr int SL = NW == 1 ? 2 : 1;               // k slices of a stage: 32 KiB of weights each way
    static constexpr int SLICE = NW * D8_W + NT / 32 * D8_X;
    static constexpr int STAGE = SL * SLICE;
    static constexpr int STAGES = NT > 32 ? 4 : UP ? 6 : 5;
    static constexpr int SMEM = STAGES * STAGE + 1024;
    static constexpr int BUFS = NT > 32 ? 1 : 2;             // accumulators
    static constexpr int SF_COL = 256;                       // TMEM: accumulators below, two copies of the scales from here
    static constexpr int TMEM_COLS = 512;
};

struct Fp8DecArgs {
    const int* sched;
    const int* tile_expert;
    const int* row_token;
    const float* row_weight;
    int* status;
    int n_cblk;
    int nkb;
    int out_cols;
    const uint8_t* x_scale;
    const uint8_t* w_scale;
    uint8_t* h;
    uint8_t* h_scale;
    __nv_bfloat16* y;
};

struct D8Item {
    int tile, cb, e;
    int n_pass;      // passes over the weights
    int n_sub;       // 32-row blocks of a pass
};
template <int NT>
__device__ __forceinline__ D8Item d8_item(const Fp8DecArgs& g, int item) {
    D8Item w;
    w.tile = item / g.n_cblk;
    w.cb = item - w.tile * g.n_cblk;
    w.e = __ldg(g.tile_expert + w.tile);
    const int* rt = g.row_token + static_cast<size_t>(w.tile) * TILE_M;
    const int r1 = __ldg(rt + 32), r2 = __ldg(rt + 64), r3 = __ldg(rt + 96);
    const int blocks = 1 + (r1 >= 0) + (r2 >= 0) + (r3 >= 0);     // real rows come first in a tile
    w.n_pass = NT == 32 ? blocks : 1;
    w.n_sub = NT == 32 ? 1 : blocks;
    return w;
}

template <bool UP, int NT>
__global__ void __launch_bounds__(D8_THREADS, 1)
fp8_decode_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Fp8DecArgs g) {
    using C = D8<UP, NT>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_full[C::STAGES];
    __shared__ uint64_t bar_empty[C::STAGES];
    __shared__ uint64_t bar_sf_full[2];
    __shared__ uint64_t bar_sf_empty[2];
    __shared__ uint64_t bar_acc_full[C::BUFS];
    __shared__ uint64_t bar_acc_empty[C::BUFS];
    __shared__ uint64_t bar_meet;                    // up: the four epilogue warps have written their part of s_top
    __shared__ uint32_t s_top[UP ? 2 : 1][UP ? 4 : 1][UP ? 32 : 1];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t stage_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int total_items = __ldg(g.sched + SCHED_N_TILES) * g.n_cblk;
    if (total_items <= 0 || static_cast<int>(blockIdx.x) >= total_items) return;
    const int n_groups = (g.nkb + FP8_GROUP - 1) / FP8_GROUP;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&bar_sf_full[b]), 4);
            mbar_init(smem_u32(&bar_sf_empty[b]), 1);
        }
        for (int b = 0; b < C::BUFS; ++b) {
            mbar_init(smem_u32(&bar_acc_full[b]), 1);
            mbar_init(smem_u32(&bar_acc_empty[b]), 4);
        }
        mbar_init(smem_u32(&bar_meet), 4);
        fence_mbar_init();
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_slot), C::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
    volatile int* abortp = &abort_flag;

    if (warp == 0) {
        // ================================================================ loads
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int item = blockIdx.x; ok && item < total_items; item += gridDim.x) {
                const D8Item w = d8_item<NT>(g, item);
                for (int ps = 0; ok && ps < w.n_pass; ++ps) {
                    const int row0 = w.tile * TILE_M + ps * 32;
                    for (int kb = 0; kb < g.nkb; kb += C::SL) {
                        ok = mbar_wait(smem_u32(&bar_empty[stage]), phase ^ 1u, abortp, g.status, DEV_TIMEOUT_PRODUCER);
                        if (!ok) break;
                        const uint32_t full = smem_u32(&bar_full[stage]);
                        mbar_arrive_expect_tx(full, C::SL * (C::NW * D8_W + w.n_sub * D8_X));
#pragma unroll
                        for (int h = 0; h < C::SL; ++h) {      // a slice past the end of the k axis is zero-filled
                            const uint32_t sw = stage_base + stage * C::STAGE + h * C::SLICE;
                            const int k0 = (kb + h) * (D8_K / 2);      // tensor maps count in 16-bit units
#pragma unroll
                            for (int i = 0; i < C::NW; ++i) {
                                if constexpr (UP) tma_load_3d(sw + i * D8_W, &tmW, full, k0, w.cb * 128, w.e * 2 + i);
                                else tma_load_3d(sw + i * D8_W, &tmW, full, k0, (w.cb * C::NW + i) * 128, w.e);
                            }
                            for (int t = 0; t < w.n_sub; ++t)
                                tma_load_2d(sw + C::NW * D8_W + t * D8_X, &tmX, full, k0, row0 + t * 32);
                        }
                        if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ================================================================ MMAs
        if (lane == 0) {
            // descriptor halves as in the row-tile kernels: only the start address changes from MMA to MMA
            constexpr uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);
            const uint32_t lo0 = ((stage_base >> 4) & 0x3FFFu) | (1u << 16);
            int stage = 0;
            uint32_t phase = 0, lo = lo0;
            int it = 0, gi = 0;
            bool ok = true;
            for (int item = blockIdx.x; ok && item < total_items; item += gridDim.x) {
                const D8Item w = d8_item<NT>(g, item);
                const uint32_t n_field = static_cast<uint32_t>(w.n_sub * 32 >> 3) << 17;
                for (int ps = 0; ok && ps < w.n_pass; ++ps, ++it) {
                    const int ab = it % C::BUFS;
                    ok = mbar_wait(smem_u32(&bar_acc_empty[ab]), ((it / C::BUFS) & 1u) ^ 1u, abortp, g.status,
                                   DEV_TIMEOUT_MMA);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t tmem_d = tmem_base + ab * (C::NW * NT);
                    for (int grp = 0; ok && grp < n_groups; ++grp, ++gi) {
                        const uint32_t sf = tmem_base + C::SF_COL + (gi & 1) * 16;
                        ok = mbar_wait(smem_u32(&bar_sf_full[gi & 1]), (gi >> 1) & 1u, abortp, g.status, DEV_TIMEOUT_MMA);
                        if (!ok) break;
                        tc_fence_after();
                        const int kb0 = grp * FP8_GROUP;
#pragma unroll
                        for (int j = 0; j < FP8_GROUP; ++j) {
                            if (ok && kb0 + j < g.nkb) {
                                if (j % C::SL == 0) {
                                    ok = mbar_wait(smem_u32(&bar_full[stage]), phase, abortp, g.status, DEV_TIMEOUT_MMA);
                                    tc_fence_after();
                                }
                                if (ok) {
                                    const uint32_t idesc = umma_idesc_fp8(128, 0, j) | n_field;
                                    const uint32_t w_lo = lo + (j % C::SL * C::SLICE >> 4);
                                    const uint32_t x_lo = w_lo + (C::NW * D8_W >> 4);
#pragma unroll
                                    for (int i = 0; i < C::NW; ++i) {
#pragma unroll
                                        for (uint32_t k = 0; k < 4; ++k)
                                            umma_fp8_lohi(tmem_d + i * NT, w_lo + (i * D8_W >> 4) + k * 2u, desc_hi,
                                                          x_lo + k * 2u, desc_hi, idesc, sf + 4 * i, sf + 4 * C::NW,
                                                          (kb0 + j + static_cast<int>(k)) != 0 ? 1u : 0u);
                                    }
                                    if (j % C::SL == C::SL - 1 || kb0 + j + 1 == g.nkb) {
                                        umma_commit(smem_u32(&bar_empty[stage]));
                                        lo += C::STAGE >> 4;
                                        if (++stage == C::STAGES) { stage = 0; phase ^= 1u; lo = lo0; }
                                    }
                                }
                            }
                        }
                        if (ok) umma_commit(smem_u32(&bar_sf_empty[gi & 1]));
                    }
                    if (ok) umma_commit(smem_u32(&bar_acc_full[ab]));
                }
            }
        }
    } else if (warp >= 6) {
        // ================================================================ scales (four whole warps)
        int gi = 0;
        bool ok = true;
        const uint32_t sf0 = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + C::SF_COL;
        const int w_blocks = UP ? g.n_cblk : (g.out_cols + 127) / 128;
        for (int item = blockIdx.x; ok && item < total_items; item += gridDim.x) {
            const D8Item w = d8_item<NT>(g, item);
            const int i = (lane >> 2) & 1;
            const uint8_t* ws;
            bool have = true;
            if constexpr (UP) {
                ws = g.w_scale + ((static_cast<size_t>(w.e) * 2 + i) * w_blocks + w.cb) * g.nkb;
            } else {
                const int wb = w.cb * C::NW + (C::NW == 2 ? i : 0);
                ws = g.w_scale + (static_cast<size_t>(w.e) * w_blocks + wb) * g.nkb;
                have = wb < w_blocks;
            }
            const uint8_t* xs = g.x_scale + static_cast<size_t>(w.tile) * n_groups * FP8_ATOM + lane * 16;
            for (int ps = 0; ok && ps < w.n_pass; ++ps) {
                for (int grp = 0; grp < n_groups; ++grp, ++gi) {
                    uint4 xw;
                    if constexpr (NT == 32) {
                        // row ps * 32 + lane: word ps of the lane's 16 bytes
                        xw.x = __ldg(reinterpret_cast<const uint32_t*>(xs + static_cast<size_t>(grp) * FP8_ATOM) + ps);
                        xw.y = xw.z = xw.w = xw.x;
                    } else {
                        xw = __ldg(reinterpret_cast<const uint4*>(xs + static_cast<size_t>(grp) * FP8_ATOM));
                    }
                    const int kb = grp * FP8_GROUP + (lane & 3);
                    uint32_t word = have && kb < g.nkb ? __ldg(ws + kb) : 127u;
                    word <<= 8 * (lane & 3);
                    word |= __shfl_xor_sync(0xffffffffu, word, 1);
                    word |= __shfl_xor_sync(0xffffffffu, word, 2);
                    const uint32_t w0 = __shfl_sync(0xffffffffu, word, 0), w1 = __shfl_sync(0xffffffffu, word, 4);
                    ok = mbar_wait(smem_u32(&bar_sf_empty[gi & 1]), ((gi >> 1) & 1u) ^ 1u, abortp, g.status,
                                   DEV_TIMEOUT_PRODUCER);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t sf = sf0 + (gi & 1) * 16;
                    tmem_st4(sf, w0, w0, w0, w0);
                    if constexpr (C::NW == 2) tmem_st4(sf + 4, w1, w1, w1, w1);
                    tmem_st4(sf + 4 * C::NW, xw.x, xw.y, xw.z, xw.w);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&bar_sf_full[gi & 1]));
                }
            }
        }
    } else {
        // ================================================================ epilogue (warps 2..5)
        const int q = warp & 3;
        int it = 0, meet = 0;
        bool ok = true;
        for (int item = blockIdx.x; ok && item < total_items; item += gridDim.x) {
            const D8Item w = d8_item<NT>(g, item);
            for (int ps = 0; ok && ps < w.n_pass; ++ps, ++it) {
                const int ab = it % C::BUFS;
                ok = mbar_wait(smem_u32(&bar_acc_full[ab]), (it / C::BUFS) & 1u, abortp, g.status, DEV_TIMEOUT_EPILOGUE);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + ab * (C::NW * NT);
                auto hand_back = [&]() {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&bar_acc_empty[ab]));
                };
#pragma unroll 1
                for (int sub = 0; sub < w.n_sub; ++sub) {
                    const size_t row0 = static_cast<size_t>(w.tile) * TILE_M + (ps + sub) * 32;
                    uint32_t r[32];
                    tmem_ld32(taddr + sub * 32, r);
                    if constexpr (UP) {
                        uint32_t rb[32];
                        tmem_ld32(taddr + NT + sub * 32, rb);
                        tmem_ld_wait();
                        if (sub + 1 == w.n_sub) hand_back();
                        const int col = w.cb * 128 + q * 32 + lane;
                        float v[32];
                        uint32_t mine = 0u;
#pragma unroll
                        for (int t = 0; t < 32; ++t) {
                            const float b = __uint_as_float(rb[t]);
                            v[t] = b * __fdividef(1.0f, 1.0f + __expf(-b)) * __uint_as_float(r[t]);
                            // columns past H have zero weights, so v is zero there
                            const uint32_t top = __reduce_max_sync(0xffffffffu, abs_bits(v[t]));
                            if (lane == t) mine = top;
                        }
                        const int mb = meet & 1;
                        s_top[mb][q][lane] = mine;
                        // s_top[mb] is written again two meetings later, after every warp has been at the next one
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&bar_meet));
                        ok = mbar_wait(smem_u32(&bar_meet), static_cast<uint32_t>(mb), abortp, g.status,
                                       DEV_TIMEOUT_EPILOGUE);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        ++meet;
                        mine = max(max(s_top[mb][0][lane], s_top[mb][1][lane]), max(s_top[mb][2][lane], s_top[mb][3][lane]));
                        const uint32_t byte = fp8_scale_byte(mine);
                        const float inv = fp8_inv_scale(byte);
                        if (q == 0)
                            g.h_scale[fp8_atom_offset(row0 + lane, w.cb >> 2, (g.n_cblk + 3) >> 2) + (w.cb & 3)] =
                                static_cast<uint8_t>(byte);
                        uint8_t* dst = g.h + row0 * g.out_cols + col;
#pragma unroll
                        for (int t = 0; t < 32; ++t) {
                            const float s = __shfl_sync(0xffffffffu, inv, t);
                            if (col < g.out_cols) dst[static_cast<size_t>(t) * g.out_cols] = fp8_one(v[t] * s);
                        }
                    } else {
                        const float wgt = __ldg(g.row_weight + row0 + lane);   // lane t holds the weight of token t
#pragma unroll
                        for (int i = 0; i < C::NW; ++i) {
                            if (i > 0) tmem_ld32(taddr + i * NT + sub * 32, r);
                            tmem_ld_wait();
                            if (i + 1 == C::NW && sub + 1 == w.n_sub) hand_back();
                            const int col = (w.cb * C::NW + i) * 128 + q * 32 + lane;
                            __nv_bfloat16* dst = g.y + row0 * g.out_cols + col;
#pragma unroll
                            for (int t = 0; t < 32; ++t) {
                                const float s = __shfl_sync(0xffffffffu, wgt, t);
                                if (col < g.out_cols)
                                    dst[static_cast<size_t>(t) * g.out_cols] = __float2bfloat16_rn(__uint_as_float(r[t]) * s);
                            }
                        }
                    }
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (*abortp) {
        // a wait was abandoned: give loads still in flight time to land before shared memory is released
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) __nanosleep(1000);
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
}

template <bool UP, int NT>
static int d8_launch(const CUtensorMap& tmW, const CUtensorMap& tmX, const Fp8DecArgs& g, cudaStream_t stream) {
    static bool attr_set[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MOMOE_ERR_CUDA;
    if (!attr_set[dev]) {
        if (cudaFuncSetAttribute(fp8_decode_kernel<UP, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 D8<UP, NT>::SMEM) != cudaSuccess)
            return MOMOE_ERR_CUDA;
        attr_set[dev] = true;
    }
    fp8_decode_kernel<UP, NT><<<sm_count(), D8_THREADS, D8<UP, NT>::SMEM, stream>>>(tmW, tmX, g);
    return cudaGetLastError() == cudaSuccess ? MOMOE_OK : MOMOE_ERR_CUDA;
}

// Rows an expert has on average up to which 32-row passes are used.
static bool d8_narrow(const momoe_plan_t* p) {
    return static_cast<int64_t>(p->M) * p->K <= 16 * static_cast<int64_t>(p->N);
}

static void d8_args(const momoe_plan_t* p, Fp8DecArgs& g) {
    memset(&g, 0, sizeof(g));
    g.sched = p->sched;
    g.tile_expert = p->tile_expert;
    g.row_token = p->row_token;
    g.row_weight = p->row_weight;
    g.status = p->status;
}
static inline bool d8_aligned(const void* p) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace momoe

using namespace momoe;

#define MOMOE_API extern "C" __attribute__((visibility("default")))

MOMOE_API int momoe_fp8_up_swiglu_decode(const momoe_plan_t* plan, const uint8_t* x_sorted, const uint8_t* x_scale,
                                         const uint8_t* W1_N2HD, const uint8_t* S1, uint8_t* h_sorted,
                                         uint8_t* h_scale, momoe_stream_t stream) {
    int rc = fp8_check_plan(plan);
    if (rc != MOMOE_OK) return rc;
    if (!d8_aligned(x_sorted) || !d8_aligned(x_scale) || !d8_aligned(W1_N2HD) || S1 == nullptr ||
        !d8_aligned(h_sorted) || !d8_aligned(h_scale))
        return MOMOE_ERR_ARG;
    const int D = plan->D, H = plan->H;
    CUtensorMap tmW, tmX;
    if ((rc = encode_tmap_3d(&tmW, W1_N2HD, static_cast<uint64_t>(plan->N) * 2, H, D / 2, 128, D8_K / 2)) != MOMOE_OK)
        return rc;
    if ((rc = encode_tmap_2d(&tmX, x_sorted, plan->rows_capacity, D / 2, 32, D8_K / 2)) != MOMOE_OK) return rc;
    Fp8DecArgs g;
    d8_args(plan, g);
    g.n_cblk = (H + 127) / 128;
    g.nkb = (D + D8_K - 1) / D8_K;
    g.out_cols = H;
    g.x_scale = x_scale;
    g.w_scale = S1;
    g.h = h_sorted;
    g.h_scale = h_scale;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return d8_narrow(plan) ? d8_launch<true, 32>(tmW, tmX, g, st) : d8_launch<true, 128>(tmW, tmX, g, st);
}

MOMOE_API int momoe_fp8_down_scale_decode(const momoe_plan_t* plan, const uint8_t* h_sorted, const uint8_t* h_scale,
                                          const uint8_t* W2_NDH, const uint8_t* S2, void* y_sorted,
                                          momoe_stream_t stream) {
    int rc = fp8_check_plan(plan);
    if (rc != MOMOE_OK) return rc;
    if (!d8_aligned(h_sorted) || !d8_aligned(h_scale) || !d8_aligned(W2_NDH) || S2 == nullptr || !d8_aligned(y_sorted))
        return MOMOE_ERR_ARG;
    const int D = plan->D, H = plan->H;
    CUtensorMap tmW, tmX;
    if ((rc = encode_tmap_3d(&tmW, W2_NDH, plan->N, D, H / 2, 128, D8_K / 2)) != MOMOE_OK) return rc;
    if ((rc = encode_tmap_2d(&tmX, h_sorted, plan->rows_capacity, H / 2, 32, D8_K / 2)) != MOMOE_OK) return rc;
    Fp8DecArgs g;
    d8_args(plan, g);
    const bool narrow = d8_narrow(plan);
    g.n_cblk = narrow ? (D + 127) / 128 : (D + 255) / 256;
    g.nkb = (H + D8_K - 1) / D8_K;
    g.out_cols = D;
    g.x_scale = h_scale;
    g.w_scale = S2;
    g.y = static_cast<__nv_bfloat16*>(y_sorted);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return narrow ? d8_launch<false, 32>(tmW, tmX, g, st) : d8_launch<false, 128>(tmW, tmX, g, st);
}
