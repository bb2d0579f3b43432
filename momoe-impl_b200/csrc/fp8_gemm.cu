// The experts' two forward GEMMs on 8-bit rows and weights (e4m3, a power of two for each block of 128), sm_100a.
//
//   up    a = x W1[e][:H]^T, b = x W1[e][H:]^T, h = b sigmoid(b) a in 32 bits, h -> 8-bit rows (128 columns a scale)
//   down  y[r, :] = row_weight[r] * (h W2[e]^T), as fp16 with a power of two for each (row, 256 columns) (fp8.cuh)
//
// Weights are K-major ([N, 2H, D] and [N, D, H]) with one scale for each 128 x 128 block.  All scales are powers of two,
// so the tensor core applies them (kind::mxf8f6f4, block-scaled): accumulation is fp32 over the whole k axis and there is
// no per-block pass over the accumulators, which fp32 scales would need.
//
// Bound at large row counts by the tensor pipe at the clock that the power limit leaves and by the tiles' way out of L2, 10
// TB/s at 16384 tokens (D2048 H1024, top-8 of 128: up 2.2, down 1.8 PFLOP/s).  The structure is that of the 16-bit grouped
// GEMM: a CTA pair computes 256 x 256, each CTA loads its 128 rows of A and half of B, ring of 3 stages of two 128-byte k
// slices (a slice is 128 values here), warp 0 loads, warp 1 of the leader issues the MMAs, warps 2..9 are the epilogue.
//
// With few rows an expert the second tile of a pair is mostly missing and half of its MMAs and A loads are for nothing.
// Then (CG = 1) a CTA computes 128 x 256 by itself, in 4 stages of one slice, and loads the 32-row blocks of A that hold
// real rows.  It takes half as many loads of B more, 48 KiB a slice for 128 rows against 64 KiB for 256.
//
// What differs from the 16-bit kernel:
//
// Scales.  Warps 10..13 of each CTA (one for each TMEM lane quarter) write the scales of four slices (512 k) straight into
// TMEM: 4 columns for the CTA's 128 rows, 8 for the 256 weight columns (one word each, repeated).  The MMAs of the four
// slices pick their byte of each word through the scale ids of the instruction descriptor.  Two TMEM copies alternate; a
// copy is overwritten after the commit behind the MMAs that read it has arrived.  (Copies from shared memory by tcgen05.cp
// sit between the MMAs in the tensor pipe: 536 against 515 us for the up GEMM of 16384 tokens, D2048 H1024, top-8 of 128.)
//
// TMEM.  Two accumulators of 256 columns and 24 columns of scales do not fit 512 columns, so the accumulators overlap: the
// first takes columns 0..255, the second 224..479, the scales 480..503.  The epilogue reads the 32 shared columns of a
// tile first and hands them back at once (`bar_ovl`), so the next tile's MMAs wait for an eighth of the read-out, not all.
//
// Padding rows hold anything: no row of a forward pass depends on another, and no consumer reads their results.
#include <cstring>
#include <type_traits>

#include "fp8.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "../../include/momoe_b200.h"

namespace momoe {

constexpr int F8_EPI_WARPS = 8;
constexpr int F8_SF_WARPS = 4;
constexpr int F8_THREADS = 32 * (2 + F8_EPI_WARPS + F8_SF_WARPS);
constexpr int F8_TILE_N = 256;
constexpr int F8_K = 128;                                 // values of a k slice (128 bytes)
constexpr int F8_A_BYTES = TILE_M * F8_K;                 // 16 KiB
// of CG thread blocks that share a tile: bytes of a CTA's part of a k slice, slices of a stage, stages
template <int CG>
constexpr int F8_SLICE_BYTES = F8_A_BYTES + F8_TILE_N / CG * F8_K;
template <int CG>
constexpr int F8_SLICES = CG;
template <int CG>
constexpr int F8_STAGES = CG == 2 ? 3 : 4;
template <int CG>
constexpr int F8_STAGE_BYTES = F8_SLICES<CG> * F8_SLICE_BYTES<CG>;
constexpr int F8_PIECE = 2048;                            // staging of results: 32 rows x 64 bytes
template <bool UP>
constexpr int F8_PIECES = UP ? 1 : 2;                     // pieces an epilogue warp has
template <bool UP, int CG>
constexpr int F8_SMEM_BYTES = F8_STAGES<CG> * F8_STAGE_BYTES<CG> + F8_EPI_WARPS * F8_PIECES<UP> * F8_PIECE + 1024;
constexpr int F8_ACC1 = 224;                              // first column of the second accumulator
constexpr int F8_SF_COL = 480;
constexpr int F8_SF_COLS = 12;                            // 4 for A, 8 for B

struct Fp8Args {
    const int* sched;
    const int* tile_expert;
    const int* pair_info;
    const int* tile_rows;
    int* status;
    int n_nblk;                 // column blocks of 128 (up, both halves) or 256 (down)
    int nkb;                    // k slices
    int out_cols;               // H (up) or D (down)
    const uint8_t* a_scale;     // blocks of 512 bytes, [tile, ceil(nkb / 4)]
    const uint8_t* b_scale;     // up: [N, 2, n_nblk, nkb]; down: [N, ceil(D / 128), nkb]
    int b_blocks;               // down: ceil(D / 128)
    uint8_t* h_scale;           // up: scales of h, blocks of 512 bytes
    const float* row_weight;    // down
    float* y_scale;             // down: [rows, n_nblk]
};

__device__ __forceinline__ uint32_t f8_pack_f16(float lo, float hi) {
    const __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}
// The short exponential and division are off by some 2^-20 relative; the value is rounded to e4m3 (2^-4) next.
__device__ __forceinline__ float f8_swiglu(float a, float b) { return b * __fdividef(1.0f, 1.0f + __expf(-b)) * a; }

struct Fp8Work {
    int tile, nb, e;
    int rows;          // the tile's real rows, which come first; pairs: TILE_M, or 0 for a missing second tile
};
template <int CG>
__device__ __forceinline__ Fp8Work f8_work(const Fp8Args& g, int item, uint32_t cta_rank) {
    Fp8Work w;
    w.nb = item % g.n_nblk;
    if constexpr (CG == 2) {
        const int info = __ldcg(g.pair_info + item / g.n_nblk);
        w.tile = (info >> 1) + static_cast<int>(cta_rank);
        w.rows = cta_rank == 0 || (info & 1) != 0 ? TILE_M : 0;
        w.e = __ldcg(g.tile_expert + (info >> 1));
    } else {
        w.tile = item / g.n_nblk;
        w.rows = __ldcg(g.tile_rows + w.tile);
        w.e = __ldcg(g.tile_expert + w.tile);
    }
    return w;
}
// The same variable in the CTA that issues the MMAs.
template <int CG>
__device__ __forceinline__ uint32_t f8_lead(uint32_t addr) {
    return CG == 2 ? mapa_shared(addr, 0) : addr;
}
// All MMAs so far have completed: an arrival in every CTA of the tile.
template <int CG>
__device__ __forceinline__ void f8_commit(uint32_t bar) {
    if constexpr (CG == 2) umma_commit_pair(bar, 3);
    else umma_commit(bar);
}

template <bool UP, int CG>
__global__ void __cluster_dims__(CG, 1, 1) __launch_bounds__(F8_THREADS, 1)
fp8_grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                        const __grid_constant__ CUtensorMap tmO, const Fp8Args g) {
    extern __shared__ uint8_t smem_raw[];
    constexpr int STAGES = F8_STAGES<CG>, SLICES = F8_SLICES<CG>;
    constexpr int SLICE_BYTES = F8_SLICE_BYTES<CG>, STAGE_BYTES = F8_STAGE_BYTES<CG>;
    __shared__ uint64_t bar_full[STAGES];
    __shared__ uint64_t bar_empty[STAGES];
    __shared__ uint64_t bar_sf_full[2];              // leader: both CTAs' scale warps have written this copy
    __shared__ uint64_t bar_sf_empty[2];             // both: the MMAs that read this copy have completed
    __shared__ uint64_t bar_acc_full[2];
    __shared__ uint64_t bar_acc_empty[2];            // leader
    __shared__ uint64_t bar_ovl;                     // leader: the shared columns of the latest tile have been read
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    // [meeting][column half][row]: up, the bits of the largest magnitude; down, its exponent alone, since memory is short
    __shared__ std::conditional_t<UP, uint32_t, uint8_t> s_top[2][2][TILE_M];

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t cta_rank = CG == 2 ? cluster_ctarank() : 0u;
    const bool leader = cta_rank == 0;
    const int cluster_id = blockIdx.x / CG;
    const int n_clusters = gridDim.x / CG;
    const uint32_t stage_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t epi_base = stage_base + STAGES * STAGE_BYTES;

    const int n_groups = (g.nkb + FP8_GROUP - 1) / FP8_GROUP;
    grid_launch_dependents();

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&bar_sf_full[b]), CG * F8_SF_WARPS);
            mbar_init(smem_u32(&bar_sf_empty[b]), 1);
            mbar_init(smem_u32(&bar_acc_full[b]), 1);
            mbar_init(smem_u32(&bar_acc_empty[b]), CG * F8_EPI_WARPS);
        }
        mbar_init(smem_u32(&bar_ovl), CG * F8_EPI_WARPS / 2);   // four warps of each CTA read the shared columns
        fence_mbar_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
        tma_prefetch_desc(&tmO);
    }
    if (warp == 1) {
        if constexpr (CG == 2) {
            tmem_alloc_pair(smem_u32(&tmem_slot), 512);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(&tmem_slot), 512);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
    volatile int* abortp = &abort_flag;
    // everything above ran beside the tail of the kernel before; from here on its results are read
    grid_wait();
    const int total_items = __ldcg(g.sched + (CG == 2 ? SCHED_N_PAIRS : SCHED_N_TILES)) * g.n_nblk;

    if (warp == 0) {
        // ================================================================ loads
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            const int r = static_cast<int>(cta_rank);
            for (int item = cluster_id; ok && item < total_items; item += n_clusters) {
                const Fp8Work w = f8_work<CG>(g, item, cta_rank);
                // of a tile of its own a CTA loads the blocks of 32 rows that hold real ones: the rest of a stage holds
                // what it held before, and so do the rows of the accumulator that nothing reads
                const int blocks = CG == 2 ? 4 : (w.rows + 31) >> 5;
                const uint32_t bytes = CG == 2 ? 2 * STAGE_BYTES : SLICE_BYTES - (4 - blocks) * (F8_A_BYTES / 4);
                for (int kb = 0; kb < g.nkb; kb += SLICES) {
                    ok = mbar_wait(smem_u32(&bar_empty[stage]), phase ^ 1u, abortp, g.status, DEV_TIMEOUT_PRODUCER);
                    if (!ok) break;
                    if (leader) mbar_arrive_expect_tx(smem_u32(&bar_full[stage]), bytes);
                    const uint32_t full = f8_lead<CG>(smem_u32(&bar_full[stage]));
                    // tensor maps count in 16-bit units; a slice past the end of the k axis is zero-filled
#pragma unroll
                    for (int h = 0; h < SLICES; ++h) {
                        const uint32_t sa = stage_base + stage * STAGE_BYTES + h * SLICE_BYTES;
                        const int k0 = (kb + h) * (F8_K / 2);
                        // up: 128 rows of the linear half of W1[e] and the matching gate rows; of a pair, the leader
                        // loads the former and its peer the latter
                        if constexpr (CG == 2) {
                            tma_load_2d_pair(sa, &tmA, full, k0, w.tile * TILE_M);
                            if constexpr (UP) tma_load_3d_pair(sa + F8_A_BYTES, &tmB, full, k0, w.nb * 128, w.e * 2 + r);
                            else tma_load_3d_pair(sa + F8_A_BYTES, &tmB, full, k0, w.nb * F8_TILE_N + r * 128, w.e);
                        } else {
                            for (int i = 0; i < blocks; ++i)
                                tma_load_2d(sa + i * (F8_A_BYTES / 4), &tmA, full, k0, w.tile * TILE_M + i * 32);
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const uint32_t sb = sa + F8_A_BYTES + i * 128 * F8_K;
                                if constexpr (UP) tma_load_3d(sb, &tmB, full, k0, w.nb * 128, w.e * 2 + i);
                                else tma_load_3d(sb, &tmB, full, k0, w.nb * F8_TILE_N + i * 128, w.e);
                            }
                        }
                    }
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
            }
        }
    } else if (warp == 1) {
        // ================================================================ MMAs (leader CTA only)
        if (lane == 0 && leader) {
            constexpr uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);   // SBO 1024, version 1, 128-byte swizzle
            const uint32_t a_lo0 = ((stage_base >> 4) & 0x3FFFu) | (1u << 16);
            constexpr uint32_t b_off = F8_A_BYTES >> 4;
            int stage = 0;
            uint32_t phase = 0;
            uint32_t a_lo = a_lo0;
            int it = 0, gi = 0;        // tiles and scale groups so far
            bool ok = true;
            for (int item = cluster_id; ok && item < total_items; item += n_clusters, ++it) {
                const int ab = it & 1;
                ok = mbar_wait(smem_u32(&bar_acc_empty[ab]), ((it >> 1) & 1u) ^ 1u, abortp, g.status, DEV_TIMEOUT_MMA);
                if (ok && it > 0) ok = mbar_wait(smem_u32(&bar_ovl), (it - 1) & 1u, abortp, g.status, DEV_TIMEOUT_MMA);
                if (!ok) break;
                tc_fence_after();
                const uint32_t tmem_d = tmem_base + ab * F8_ACC1;
                for (int grp = 0; ok && grp < n_groups; ++grp, ++gi) {
                    const uint32_t sf = tmem_base + F8_SF_COL + (gi & 1) * F8_SF_COLS;
                    ok = mbar_wait(smem_u32(&bar_sf_full[gi & 1]), (gi >> 1) & 1u, abortp, g.status, DEV_TIMEOUT_MMA);
                    if (!ok) break;
                    tc_fence_after();
                    const int kb0 = grp * FP8_GROUP;
#pragma unroll
                    for (int j = 0; j < FP8_GROUP; ++j) {
                        if (kb0 + j < g.nkb) {
                            if (j % SLICES == 0) {
                                ok = ok && mbar_wait(smem_u32(&bar_full[stage]), phase, abortp, g.status, DEV_TIMEOUT_MMA);
                                tc_fence_after();
                            }
                            if (ok) {
                                const uint32_t idesc = umma_idesc_fp8(CG * TILE_M, F8_TILE_N, j);
                                const uint32_t lo = a_lo + j % SLICES * (SLICE_BYTES >> 4);
#pragma unroll
                                for (uint32_t k = 0; k < 4; ++k) {
                                    const uint32_t more = (kb0 + j + static_cast<int>(k)) != 0 ? 1u : 0u;
                                    if constexpr (CG == 2)
                                        umma_fp8_pair_lohi(tmem_d, lo + k * 2u, desc_hi, lo + b_off + k * 2u, desc_hi,
                                                           idesc, sf, sf + 4, more);
                                    else
                                        umma_fp8_lohi(tmem_d, lo + k * 2u, desc_hi, lo + b_off + k * 2u, desc_hi, idesc, sf,
                                                      sf + 4, more);
                                }
                                if (j % SLICES == SLICES - 1 || kb0 + j + 1 == g.nkb) {
                                    f8_commit<CG>(smem_u32(&bar_empty[stage]));
                                    a_lo += STAGE_BYTES >> 4;
                                    if (++stage == STAGES) { stage = 0; phase ^= 1u; a_lo = a_lo0; }
                                }
                            }
                        }
                    }
                    if (ok) f8_commit<CG>(smem_u32(&bar_sf_empty[gi & 1]));
                }
                if (ok) f8_commit<CG>(smem_u32(&bar_acc_full[ab]));
            }
        }
    } else if (warp >= 2 + F8_EPI_WARPS) {
        // ================================================================ scales (both CTAs, four whole warps)
        int gi = 0;
        bool ok = true;
        const uint32_t full0 = f8_lead<CG>(smem_u32(&bar_sf_full[0]));
        const uint32_t sf0 = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + F8_SF_COL;
        for (int item = cluster_id; ok && item < total_items; item += n_clusters) {
            const Fp8Work w = f8_work<CG>(g, item, cta_rank);
            const int tile = w.rows > 0 ? w.tile : w.tile - 1;     // a missing half reads its partner's scales
            const uint4* src = reinterpret_cast<const uint4*>(g.a_scale + static_cast<size_t>(tile) * n_groups * FP8_ATOM);
            // the two blocks of 128 weight columns of this item
            const int i = (lane >> 2) & 1;
            const uint8_t* bs;
            bool have;
            if constexpr (UP) {
                bs = g.b_scale + ((static_cast<size_t>(w.e) * 2 + i) * g.n_nblk + w.nb) * g.nkb;
                have = true;
            } else {
                bs = g.b_scale + (static_cast<size_t>(w.e) * g.b_blocks + w.nb * 2 + i) * g.nkb;
                have = w.nb * 2 + i < g.b_blocks;
            }
            for (int grp = 0; grp < n_groups; ++grp, ++gi) {
                const uint4 a = __ldcg(src + grp * 32 + lane);
                const int kb = grp * FP8_GROUP + (lane & 3);
                uint32_t word = have && kb < g.nkb ? __ldg(bs + kb) : 127u;
                word <<= 8 * (lane & 3);
                word |= __shfl_xor_sync(0xffffffffu, word, 1);
                word |= __shfl_xor_sync(0xffffffffu, word, 2);
                const uint32_t b0 = __shfl_sync(0xffffffffu, word, 0), b1 = __shfl_sync(0xffffffffu, word, 4);
                ok = mbar_wait(smem_u32(&bar_sf_empty[gi & 1]), ((gi >> 1) & 1u) ^ 1u, abortp, g.status,
                               DEV_TIMEOUT_PRODUCER);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t sf = sf0 + (gi & 1) * F8_SF_COLS;
                tmem_st4(sf, a.x, a.y, a.z, a.w);
                tmem_st4(sf + 4, b0, b0, b0, b0);
                tmem_st4(sf + 8, b1, b1, b1, b1);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_relaxed(full0 + static_cast<uint32_t>((gi & 1) * sizeof(uint64_t)));
            }
        }
    } else {
        // ================================================================ epilogue (warps 2..9, both CTAs)
        const int q = warp & 3;
        const int row = q * 32 + lane;
        const int half = (warp - 2) >> 2;
        const uint32_t acc_empty_leader = f8_lead<CG>(smem_u32(&bar_acc_empty[0]));
        const uint32_t ovl_leader = f8_lead<CG>(smem_u32(&bar_ovl));
        constexpr int PIECES = F8_PIECES<UP>;
        const uint32_t stage_area = epi_base + (warp - 2) * PIECES * F8_PIECE;
        int it = 0;
        bool ok = true;
        int meet = 0;                      // meetings with the warp of the other column half so far
        int n_stored = 0;                  // pieces handed to TMA stores so far (lane 0 owns the bulk groups)
        // an item's table entries, and down the rows' weights, are asked for an item ahead
        Fp8Work next = {};
        float w_next = 0.0f;
        auto ask = [&](int item) {
            next = f8_work<CG>(g, item, cta_rank);
            if constexpr (!UP) {
                if (q * 32 < next.rows) w_next = __ldcg(g.row_weight + static_cast<size_t>(next.tile) * TILE_M + row);
            }
        };
        if (cluster_id < total_items) ask(cluster_id);
        for (int item = cluster_id; ok && item < total_items; item += n_clusters, ++it) {
            const Fp8Work w = next;
            const int ab = it & 1;
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + ab * F8_ACC1;
            // the accumulator whose neighbour follows above shares its last 32 columns, the other one its first
            const bool shares = ab == 0 ? half == 1 : half == 0;
            auto hand_back_shared = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_relaxed(ovl_leader);
            };
            auto hand_back_all = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_relaxed(acc_empty_leader + ab * static_cast<uint32_t>(sizeof(uint64_t)));
            };
            const bool live = q * 32 < w.rows;         // this warp has real rows
            const float wgt = w_next;
            const size_t grow = static_cast<size_t>(w.tile) * TILE_M + row;
            if (item + n_clusters < total_items) ask(item + n_clusters);
            ok = mbar_wait(smem_u32(&bar_acc_full[ab]), (it >> 1) & 1u, abortp, g.status, DEV_TIMEOUT_EPILOGUE) &&
                 *abortp == 0;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                // the partner warp may be on its way into the meeting below: it must not wait for this one
                asm volatile("bar.arrive %0, 64;" ::"r"(1 + q) : "memory");
                break;
            }
            tc_fence_after();
            if ((CG == 1 || !UP) && !live) {           // so is its partner's
                if (shares) hand_back_shared();
                hand_back_all();
                continue;
            }
            if constexpr (UP) {
                // columns 32c .. 32c + 31 of the block, first the chunk that touches the shared columns
                const int s0 = half;                     // position of the first chunk inside this warp's 64 columns
                float h0[32], h1[32];
                {
                    uint32_t ra[32], rb[32];
                    const int c = half * 2 + s0;
                    tmem_ld32(taddr + c * 32, ra);
                    tmem_ld32(taddr + 128 + c * 32, rb);
                    tmem_ld_wait();
                    if (shares) hand_back_shared();
#pragma unroll
                    for (int i = 0; i < 32; ++i) h0[i] = f8_swiglu(__uint_as_float(ra[i]), __uint_as_float(rb[i]));
                    const int c1 = half * 2 + (s0 ^ 1);
                    tmem_ld32(taddr + c1 * 32, ra);
                    tmem_ld32(taddr + 128 + c1 * 32, rb);
                    tmem_ld_wait();
                    hand_back_all();
#pragma unroll
                    for (int i = 0; i < 32; ++i) h1[i] = f8_swiglu(__uint_as_float(ra[i]), __uint_as_float(rb[i]));
                }
                // columns past H have zero weights, so h is zero there and leaves the maximum alone
                uint32_t top = 0u;
#pragma unroll
                for (int i = 0; i < 32; ++i) top = max(top, max(abs_bits(h0[i]), abs_bits(h1[i])));
                s_top[meet & 1][half][row] = top;
                // two warps share a row's 128 columns; this half of s_top is written again two meetings later, after the
                // partner has been at the next one, i.e. after it has read this one
                asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory");
                top = max(top, s_top[meet & 1][half ^ 1][row]);
                ++meet;
                const uint32_t byte = fp8_scale_byte(top);
                const float inv = fp8_inv_scale(byte);
                const int col0 = w.nb * 128 + half * 64;
                if (CG == 1 || live) {
                    if (half == 0)
                        g.h_scale[fp8_atom_offset(grow, w.nb >> 2, (g.n_nblk + 3) >> 2) + (w.nb & 3)] =
                            static_cast<uint8_t>(byte);
                    if (col0 < g.out_cols) {
                        const uint32_t slot = stage_area + n_stored % PIECES * F8_PIECE;
                        if (n_stored >= PIECES && lane == 0) bulk_wait_read<PIECES - 1>();
                        __syncwarp();
                        // [32 rows x 64 bytes], 64-byte swizzle: 16-byte chunk j of row r at chunk j ^ ((r >> 1) & 3)
                        const uint32_t base = slot + lane * 64;
                        const uint32_t x = (lane >> 1) & 3;
                        uint32_t p[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            p[i] = fp8_pack4(h0[4 * i] * inv, h0[4 * i + 1] * inv, h0[4 * i + 2] * inv, h0[4 * i + 3] * inv);
                        const uint32_t j0 = 2 * s0, j1 = 2 * (s0 ^ 1);
                        st_shared_v4(base + ((j0 ^ x) << 4), p[0], p[1], p[2], p[3]);
                        st_shared_v4(base + (((j0 + 1) ^ x) << 4), p[4], p[5], p[6], p[7]);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            p[i] = fp8_pack4(h1[4 * i] * inv, h1[4 * i + 1] * inv, h1[4 * i + 2] * inv, h1[4 * i + 3] * inv);
                        st_shared_v4(base + ((j1 ^ x) << 4), p[0], p[1], p[2], p[3]);
                        st_shared_v4(base + (((j1 + 1) ^ x) << 4), p[4], p[5], p[6], p[7]);
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_2d(&tmO, slot, col0 / 2, w.tile * TILE_M + q * 32);
                            bulk_commit();
                        }
                        ++n_stored;
                    }
                }
            } else {
                // The largest sum of a row decides its power of two, so all are read before the first is stored.  Three chunks of
                // 32 columns stay in registers, among them the one that may hold shared columns; the other is read again.
                auto chunk = [&](int i) { return half == 0 ? i : 4 + ((i + 3) & 3); };   // half 1 starts with its last chunk
                auto top_of = [](const uint32_t (&r)[32]) {
                    float top = 0.0f;
#pragma unroll
                    for (int j = 0; j < 32; ++j) top = fmaxf(top, fabsf(__uint_as_float(r[j])));   // passes NaN over
                    if (top == INFINITY) {
                        top = 0.0f;
#pragma unroll
                        for (int j = 0; j < 32; ++j) top = fmaxf(top, finite_or_zero(__uint_as_float(r[j])));
                    }
                    return top;
                };
                uint32_t r0[32], r1[32], r[32];
                tmem_ld32(taddr + chunk(0) * 32, r0);
                tmem_ld32(taddr + chunk(1) * 32, r1);
                tmem_ld_wait();
                if (shares) hand_back_shared();
                float top = fmaxf(top_of(r0), top_of(r1));
#pragma unroll 1
                for (int i = 2; i < 4; ++i) {
                    tmem_ld32(taddr + chunk(i) * 32, r);
                    tmem_ld_wait();
                    top = fmaxf(top, top_of(r));
                }
                // as in the up GEMM, two warps share a row's columns
                int et = static_cast<int>(__float_as_uint(top) >> 23);
                s_top[meet & 1][half][row] = static_cast<uint8_t>(et);
                asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory");
                et = max(et, static_cast<int>(s_top[meet & 1][half ^ 1][row]));
                ++meet;
                const int e = fp8_row_exponent(et, wgt);
                if (half == 0) g.y_scale[grow * g.n_nblk + w.nb] = pow2f(-e);
                const float factor = wgt * pow2f(e);
                // results leave through shared memory by TMA: with one row a thread, stores straight from registers touch
                // 32 sectors an instruction and take longer than the tile's MMAs (328 against 285 us, 16384 tokens, D2048
                // H1024, top-8 of 128)
                auto store = [&](int c, const uint32_t (&v)[32]) {
                    const int col0 = w.nb * F8_TILE_N + c * 32;
                    if (col0 >= g.out_cols) return;
                    const uint32_t slot = stage_area + n_stored % PIECES * F8_PIECE;
                    if (n_stored >= PIECES && lane == 0) bulk_wait_read<PIECES - 1>();
                    __syncwarp();
                    // [32 rows x 64 bytes], 64-byte swizzle: 16-byte chunk j of row r at chunk j ^ ((r >> 1) & 3)
                    const uint32_t base = slot + lane * 64;
                    const uint32_t x = (lane >> 1) & 3;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t p[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            p[u] = f8_pack_f16(__uint_as_float(v[j * 8 + 2 * u]) * factor,
                                               __uint_as_float(v[j * 8 + 2 * u + 1]) * factor);
                        st_shared_v4(base + ((j ^ x) << 4), p[0], p[1], p[2], p[3]);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tmO, slot, col0, w.tile * TILE_M + q * 32);   // columns past D are not written
                        bulk_commit();
                    }
                    ++n_stored;
                };
                store(chunk(0), r0);
                tmem_ld32(taddr + chunk(2) * 32, r0);
                store(chunk(1), r1);
                store(chunk(3), r);
                tmem_ld_wait();
                hand_back_all();
                store(chunk(2), r0);
            }
        }
        if (lane == 0) bulk_wait_all<0>();   // the staging area must outlive every store issued from it
        __syncwarp();
    }

    tc_fence_before();
    __syncthreads();
    if (*abortp) {
        // a wait was abandoned: give loads still in flight time to land before shared memory is released
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) __nanosleep(1000);
    }
    if constexpr (CG == 2) cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (CG == 2) tmem_dealloc_pair(tmem_base, 512);
        else tmem_dealloc(tmem_base, 512);
    }
}

template <bool UP, int CG>
static int f8_launch(const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmO, const Fp8Args& g,
                     cudaStream_t stream) {
    static int blocks[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MOMOE_ERR_CUDA;
    const auto kernel = fp8_grouped_gemm_kernel<UP, CG>;
    constexpr int smem = F8_SMEM_BYTES<UP, CG>;
    if (blocks[dev] == 0) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
            return MOMOE_ERR_CUDA;
        int n = sm_count() / CG;
        if (CG == 2) {
            cudaLaunchConfig_t cfg;
            memset(&cfg, 0, sizeof(cfg));
            cfg.gridDim = dim3(static_cast<unsigned>(n * CG));
            cfg.blockDim = dim3(F8_THREADS);
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = CG;
            attr.val.clusterDim.y = 1;
            attr.val.clusterDim.z = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            int most = 0;
            if (cudaOccupancyMaxActiveClusters(&most, kernel, &cfg) != cudaSuccess) (void)cudaGetLastError();
            if (most > 0 && most < n) n = most;
        }
        blocks[dev] = n * CG;
    }
    // (the cluster shape is the kernel's own attribute)
    return launch_dependent(kernel, blocks[dev], F8_THREADS, smem, stream, 1, tmA, tmB, tmO, g) == cudaSuccess
               ? MOMOE_OK : MOMOE_ERR_CUDA;
}

// Whether a CTA works on a tile of its own: up to F8_SINGLE_ROWS rows an expert on average.  Whole passes in us, on tiles of
// their own and in pairs:  rows an expert       48          128          192          256          384
//   D2176 H1152, top-6 of 64                115 / 132    138 / 163    177 / 194    219 / 220    299 / 291
//   D2048 H1024, top-8 of 128               173 / 215    227 / 266    298 / 313    353 / 380    497 / 468
//   D7168 H2048, top-4 of 32                262 / 338    358 / 400    473 / 460    566 / 528    773 / 695
constexpr long long F8_SINGLE_ROWS = 192;
static bool f8_single(const momoe_plan_t* p) {
    return static_cast<long long>(p->M) * p->K <= F8_SINGLE_ROWS * static_cast<long long>(p->N);
}

int fp8_check_plan(const momoe_plan_t* p) {
    if (p == nullptr || p->sched == nullptr || p->tile_expert == nullptr || p->pair_info == nullptr ||
        p->row_weight == nullptr || p->status == nullptr)
        return MOMOE_ERR_ARG;
    if (p->M <= 0 || p->N <= 0 || p->K <= 0 || p->D <= 0 || p->H <= 0 || p->rows_capacity <= 0) return MOMOE_ERR_ARG;
    if (p->D % 16 != 0 || p->H % 16 != 0) return MOMOE_ERR_UNSUPPORTED;   // TMA row pitch of 8-bit rows: 16 bytes
    if (p->D > FP8_MAX_WIDTH || p->H > FP8_MAX_WIDTH) return MOMOE_ERR_TOO_LARGE;
    if (p->rows_capacity % TILE_M != 0) return MOMOE_ERR_ARG;
    return MOMOE_OK;
}

static inline int f8_cdiv(int a, int b) { return (a + b - 1) / b; }
static inline bool f8_aligned(const void* p, uintptr_t n) {
    return p != nullptr && (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

}  // namespace momoe

using namespace momoe;

#define MOMOE_API extern "C" __attribute__((visibility("default")))

MOMOE_API int momoe_fp8_up_swiglu(const momoe_plan_t* plan, const int32_t* tile_rows, const uint8_t* x_sorted,
                                  const uint8_t* x_scale, const uint8_t* W1_N2HD, const uint8_t* S1, uint8_t* h_sorted,
                                  uint8_t* h_scale, momoe_stream_t stream) {
    int rc = fp8_check_plan(plan);
    if (rc != MOMOE_OK) return rc;
    if (tile_rows == nullptr || !f8_aligned(x_sorted, 16) || !f8_aligned(x_scale, 16) || !f8_aligned(W1_N2HD, 16) ||
        S1 == nullptr || !f8_aligned(h_sorted, 16) || !f8_aligned(h_scale, 16))
        return MOMOE_ERR_ARG;
    const int D = plan->D, H = plan->H;
    CUtensorMap tmA, tmB, tmO;
    const bool single = f8_single(plan);
    if ((rc = encode_tmap_2d(&tmA, x_sorted, plan->rows_capacity, D / 2, single ? 32 : TILE_M, F8_K / 2)) != MOMOE_OK)
        return rc;
    if ((rc = encode_tmap_3d(&tmB, W1_N2HD, static_cast<uint64_t>(plan->N) * 2, H, D / 2, 128, F8_K / 2)) != MOMOE_OK)
        return rc;
    if ((rc = encode_tmap_2d(&tmO, h_sorted, plan->rows_capacity, H / 2, 32, 32, TMAP_SWIZZLE_64B)) != MOMOE_OK) return rc;
    Fp8Args g;
    memset(&g, 0, sizeof(g));
    g.sched = plan->sched;
    g.tile_expert = plan->tile_expert;
    g.pair_info = plan->pair_info;
    g.tile_rows = tile_rows;
    g.status = plan->status;
    g.n_nblk = f8_cdiv(H, 128);
    g.nkb = f8_cdiv(D, F8_K);
    g.out_cols = H;
    g.a_scale = x_scale;
    g.b_scale = S1;
    g.h_scale = h_scale;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return single ? f8_launch<true, 1>(tmA, tmB, tmO, g, st) : f8_launch<true, 2>(tmA, tmB, tmO, g, st);
}

MOMOE_API int momoe_fp8_down_scale(const momoe_plan_t* plan, const int32_t* tile_rows, const uint8_t* h_sorted,
                                   const uint8_t* h_scale, const uint8_t* W2_NDH, const uint8_t* S2, void* y_sorted,
                                   float* y_scale, momoe_stream_t stream) {
    int rc = fp8_check_plan(plan);
    if (rc != MOMOE_OK) return rc;
    if (tile_rows == nullptr || !f8_aligned(h_sorted, 16) || !f8_aligned(h_scale, 16) || !f8_aligned(W2_NDH, 16) ||
        S2 == nullptr || !f8_aligned(y_sorted, 16) || y_scale == nullptr)
        return MOMOE_ERR_ARG;
    const int D = plan->D, H = plan->H;
    CUtensorMap tmA, tmB, tmO;
    const bool single = f8_single(plan);
    if ((rc = encode_tmap_2d(&tmA, h_sorted, plan->rows_capacity, H / 2, single ? 32 : TILE_M, F8_K / 2)) != MOMOE_OK)
        return rc;
    if ((rc = encode_tmap_3d(&tmB, W2_NDH, plan->N, D, H / 2, 128, F8_K / 2)) != MOMOE_OK) return rc;
    if ((rc = encode_tmap_2d(&tmO, y_sorted, plan->rows_capacity, D, 32, 32, TMAP_SWIZZLE_64B)) != MOMOE_OK) return rc;
    Fp8Args g;
    memset(&g, 0, sizeof(g));
    g.sched = plan->sched;
    g.tile_expert = plan->tile_expert;
    g.pair_info = plan->pair_info;
    g.tile_rows = tile_rows;
    g.status = plan->status;
    g.n_nblk = f8_cdiv(D, F8_TILE_N);
    g.nkb = f8_cdiv(H, F8_K);
    g.out_cols = D;
    g.a_scale = h_scale;
    g.b_scale = S2;
    g.b_blocks = f8_cdiv(D, 128);
    g.row_weight = plan->row_weight;
    g.y_scale = y_scale;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return single ? f8_launch<false, 1>(tmA, tmB, tmO, g, st) : f8_launch<false, 2>(tmA, tmB, tmO, g, st);
}
