// The experts' two 8-bit forward GEMMs for token batches with few rows an expert, sm_100a.
//
// Bound by the weights' way across HBM: 3 D H bytes for each touched expert.  As in the 16-bit kernels for this case the
// WEIGHTS are the M side of the MMA (128 weight rows = 128 TMEM lanes) and the tokens its N side, so that shared memory
// holds weights in flight and not padding rows: 4 stages of 32 KiB of weights and up to 16 KiB of rows an SM.  The MMA's N is
// the tile's 32-row blocks that hold real rows, up to the whole 128-row tile, so an expert's weights pass once for each
// tile.  (A form with 32 rows a pass and 6 stages was no faster at 1 row an expert, 98 against 100 us, and slower from 8 on,
// 149 against 137 us: D2048 H1024, top-8 of 128.)
//
//   up    an item is 128 columns of h: two MMAs a k slice, the linear rows and the gate rows of W1[e], into two accumulators
//         whose lane j holds a[j] and b[j] of the same column, so the epilogue thread has both; h needs the maximum over
//         the item's 128 columns (the scale of 8-bit rows): a warp reduction for each token and one meeting of four warps
//   down  an item is 256 columns of y in two MMAs; a result row needs its largest sum (its power of two): the same
//
// One CTA (320 threads) an SM, persistent over items = (128-row tile, column block).  Warp 0 loads, warp 1 issues MMAs,
// warps 2..5 are the epilogue (a thread has one weight column and 32 tokens at a time), warps 6..9 write scales to TMEM
// (see the row-tile kernel).  There is one accumulator: the MMAs of an item wait for the read-out of the item before, while
// the ring goes on filling.
//
// With so few items that half of the SMs would idle (one token) and more than 12 k slices, two CTAs of a cluster share an
// item's k axis: the second stores its accumulators into the first one's shared memory, which adds them and goes on.
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

constexpr int D8_NT = 128;                       // tokens of a tile, columns of an accumulator
constexpr int D8_STAGE = 2 * D8_W + D8_NT / 32 * D8_X;       // one k slice: two blocks of 128 weight rows, the token rows
constexpr int D8_STAGES = 4;
template <int SPLIT>
constexpr int D8_SMEM = D8_STAGES * D8_STAGE + (SPLIT > 1 ? 4 * 64 * 32 * 4 : 0) + 1024;
constexpr int D8_SF_COL = 256;                   // TMEM: accumulators in columns 0..255, two copies of the scales behind
constexpr int D8_TMEM_COLS = 512;

struct Fp8DecArgs {
    const int* sched;
    const int* tile_expert;
    const int* tile_rows;
    const float* row_weight;
    int* status;
    int tile_cap;            // entries of tile_expert and tile_rows
    int n_cblk;
    int nkb;
    int out_cols;
    const uint8_t* x_scale;
    const uint8_t* w_scale;
    uint8_t* h;
    uint8_t* h_scale;
    __half* y;
    float* y_scale;          // down: [rows, n_cblk]
};

struct D8Item {
    int tile, cb, e;
    int rows;        // real rows of the tile (they come first)
    int n_sub;       // 32-row blocks that hold them
};
__device__ __forceinline__ D8Item d8_item(const Fp8DecArgs& g, int item) {
    D8Item w;
    w.tile = item / g.n_cblk;
    w.cb = item - w.tile * g.n_cblk;
    w.e = __ldcg(g.tile_expert + w.tile);
    w.rows = __ldcg(g.tile_rows + w.tile);
    w.n_sub = (w.rows + 31) >> 5;
    return w;
}

// What an epilogue warp keeps between read-outs.
struct D8Epi {
    uint32_t bar_acc_empty, bar_meet, bar_part_full, bar_part_free;
    uint32_t part;           // split: this lane's place in the buffer of the first CTA
    uint32_t* s_top;         // [2][4 quarters][32 tokens]
    volatile int* abortp;
    int rank;
    int meet, parts;
};

template <int T>
__device__ __forceinline__ void d8_tmem_ld(uint32_t taddr, uint32_t (&r)[T]) {
    if constexpr (T == 8) tmem_ld8(taddr, r);
    else tmem_ld32(taddr, r);
}

// The first T tokens of a 32-row block out of the accumulators (columns taddr and taddr + D8_NT), by the four epilogue
// warps; `last`: hand the accumulators back; left: real rows from row0 on; wgt: down, the weight of row0 + lane.  False when a
// wait was abandoned.
template <bool UP, int SPLIT, int T>
__device__ __forceinline__ bool d8_read_out(const Fp8DecArgs& g, D8Epi& c, const D8Item& w, size_t row0, uint32_t taddr,
                                            bool last, int left, float wgt) {
    const int lane = threadIdx.x & 31, q = (threadIdx.x >> 5) & 3;
    uint32_t r[T], rb[T];
    d8_tmem_ld<T>(taddr, r);
    d8_tmem_ld<T>(taddr + D8_NT, rb);
    tmem_ld_wait();
    if (last) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(c.bar_acc_empty);
    }
    if constexpr (SPLIT > 1) {
        // [quarter][T columns of both accumulators][lane] floats in the first CTA's shared memory
        if (c.rank != 0) {
            bool ok = mbar_wait_cluster(c.bar_part_free, (c.parts & 1u) ^ 1u, c.abortp, g.status, DEV_TIMEOUT_EPILOGUE);
            if (!__all_sync(0xffffffffu, ok)) return false;
            const uint32_t dst = mapa_shared(c.part, 0);
#pragma unroll
            for (int t = 0; t < T; ++t) {
                st_cluster_f32(dst + t * 128, r[t]);
                st_cluster_f32(dst + (T + t) * 128, rb[t]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(mapa_shared(c.bar_part_full, 0));
            ++c.parts;
            return true;
        }
        bool ok = mbar_wait_cluster(c.bar_part_full, c.parts & 1u, c.abortp, g.status, DEV_TIMEOUT_EPILOGUE);
        if (!__all_sync(0xffffffffu, ok)) return false;
        ++c.parts;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            r[t] = __float_as_uint(__uint_as_float(r[t]) + ld_shared_f32(c.part + t * 128));
            rb[t] = __float_as_uint(__uint_as_float(rb[t]) + ld_shared_f32(c.part + (T + t) * 128));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(c.bar_part_free, 1));
    }
    // lane t gets the largest of token t's columns (up: 128, the rest has zero weights; down: the finite ones of 256)
    float v[T];
    uint32_t mine = 0u;
#pragma unroll
    for (int t = 0; t < T; ++t) {
        uint32_t top;
        if constexpr (UP) {
            const float b = __uint_as_float(rb[t]);
            // off by some 2^-20 relative, before a rounding to e4m3 (2^-4)
            v[t] = b * __fdividef(1.0f, 1.0f + __expf(-b)) * __uint_as_float(r[t]);
            top = __reduce_max_sync(0xffffffffu, abs_bits(v[t]));
        } else {
            top = __reduce_max_sync(0xffffffffu, abs_bits(fmaxf(fabsf(__uint_as_float(r[t])), fabsf(__uint_as_float(rb[t])))));
        }
        if (lane == t) mine = top;
    }
    if constexpr (!UP) {
        if (__any_sync(0xffffffffu, mine >= 0x7F800000u)) {
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const uint32_t top = __reduce_max_sync(
                    0xffffffffu, __float_as_uint(fmaxf(finite_or_zero(__uint_as_float(r[t])), finite_or_zero(__uint_as_float(rb[t])))));
                if (lane == t) mine = top;
            }
        }
    }
    const int mb = c.meet & 1;
    uint32_t* s_top = c.s_top + mb * 128;
    s_top[q * 32 + lane] = mine;
    // this half of s_top is written again two meetings later, after every warp has been at the next one
    __syncwarp();
    if (lane == 0) mbar_arrive(c.bar_meet);
    bool ok = mbar_wait(c.bar_meet, static_cast<uint32_t>(mb), c.abortp, g.status, DEV_TIMEOUT_EPILOGUE);
    if (!__all_sync(0xffffffffu, ok)) return false;
    ++c.meet;
    mine = max(max(s_top[lane], s_top[32 + lane]), max(s_top[64 + lane], s_top[96 + lane]));
    if constexpr (UP) {
        const int col = w.cb * 128 + q * 32 + lane;
        const uint32_t byte = fp8_scale_byte(mine);
        const float inv = fp8_inv_scale(byte);
        if (q == 0 && lane < T)
            g.h_scale[fp8_atom_offset(row0 + lane, w.cb >> 2, (g.n_cblk + 3) >> 2) + (w.cb & 3)] = static_cast<uint8_t>(byte);
        uint8_t* dst = g.h + row0 * g.out_cols + col;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const float s = __shfl_sync(0xffffffffu, inv, t);
            if (col < g.out_cols) dst[static_cast<size_t>(t) * g.out_cols] = fp8_one(v[t] * s);
        }
    } else {
        const int e = fp8_row_exponent(static_cast<int>(mine >> 23), wgt);
        if (q == 0 && lane < left && lane < T) g.y_scale[(row0 + lane) * g.n_cblk + w.cb] = pow2f(-e);
        const float factor = wgt * pow2f(e);
        const int col = w.cb * 256 + q * 32 + lane;
        __half* dst = g.y + row0 * g.out_cols + col;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const float s = __shfl_sync(0xffffffffu, factor, t);
            if (col < g.out_cols) dst[0] = __float2half_rn(__uint_as_float(r[t]) * s);
            if (col + 128 < g.out_cols) dst[128] = __float2half_rn(__uint_as_float(rb[t]) * s);
            dst += g.out_cols;
        }
    }
    return true;
}

template <bool UP, int SPLIT>
__global__ void __launch_bounds__(D8_THREADS, 1)
fp8_decode_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Fp8DecArgs g) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_full[D8_STAGES];
    __shared__ uint64_t bar_empty[D8_STAGES];
    __shared__ uint64_t bar_sf_full[2];
    __shared__ uint64_t bar_sf_empty[2];
    __shared__ uint64_t bar_acc_full;
    __shared__ uint64_t bar_acc_empty;
    __shared__ uint64_t bar_meet;                    // the four epilogue warps have written their part of s_top
    __shared__ uint32_t s_top[2][4][32];
    __shared__ uint64_t bar_part_full[4];            // split: the other CTA's part of a quarter's accumulators has arrived
    __shared__ uint64_t bar_part_free[4];            // split, other CTA: its buffer has been read
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t stage_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int n_groups = (g.nkb + FP8_GROUP - 1) / FP8_GROUP;
    // this CTA's part of the k axis, in groups of four slices
    const int rank = SPLIT > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int grp0 = n_groups * rank / SPLIT, grp1 = n_groups * (rank + 1) / SPLIT;
    const int kb_lo = grp0 * FP8_GROUP, kb_hi = min(g.nkb, grp1 * FP8_GROUP);
    const int first_item = blockIdx.x / SPLIT, step_item = gridDim.x / SPLIT;
    grid_launch_dependents();

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < D8_STAGES; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&bar_sf_full[b]), 4);
            mbar_init(smem_u32(&bar_sf_empty[b]), 1);
        }
        mbar_init(smem_u32(&bar_acc_full), 1);
        mbar_init(smem_u32(&bar_acc_empty), 4);
        mbar_init(smem_u32(&bar_meet), 4);
        for (int w = 0; w < 4; ++w) {
            mbar_init(smem_u32(&bar_part_full[w]), 1);
            mbar_init(smem_u32(&bar_part_free[w]), 1);
        }
        fence_mbar_init();
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_slot), D8_TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (SPLIT > 1) cluster_sync_all();     // the other CTA's barriers exist before anything arrives on them
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
    volatile int* abortp = &abort_flag;
    // everything above ran beside the tail of the kernel before; from here on its results are read
    grid_wait();
    // the first item's entries are asked for together with the schedule (and clamped to the tables, which may be shorter)
    const int n_tiles = __ldcg(g.sched + SCHED_N_TILES);
    const D8Item first = d8_item(g, min(first_item, g.tile_cap * g.n_cblk - 1));
    const int total_items = n_tiles * g.n_cblk;

    if (warp == 0) {
        // ================================================================ loads
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int item = first_item; ok && item < total_items; item += step_item) {
                const D8Item w = item == first_item ? first : d8_item(g, item);
                for (int kb = kb_lo; kb < kb_hi; ++kb) {
                    ok = mbar_wait(smem_u32(&bar_empty[stage]), phase ^ 1u, abortp, g.status, DEV_TIMEOUT_PRODUCER);
                    if (!ok) break;
                    const uint32_t full = smem_u32(&bar_full[stage]);
                    mbar_arrive_expect_tx(full, 2 * D8_W + w.n_sub * D8_X);
                    const uint32_t sw = stage_base + stage * D8_STAGE;
                    const int k0 = kb * (D8_K / 2);      // tensor maps count in 16-bit units
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if constexpr (UP) tma_load_3d(sw + i * D8_W, &tmW, full, k0, w.cb * 128, w.e * 2 + i);
                        else tma_load_3d(sw + i * D8_W, &tmW, full, k0, w.cb * 256 + i * 128, w.e);
                    }
                    for (int t = 0; t < w.n_sub; ++t)
                        tma_load_2d(sw + 2 * D8_W + t * D8_X, &tmX, full, k0, w.tile * TILE_M + t * 32);
                    if (++stage == D8_STAGES) { stage = 0; phase ^= 1u; }
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
            for (int item = first_item; ok && item < total_items; item += step_item, ++it) {
                const D8Item w = item == first_item ? first : d8_item(g, item);
                const uint32_t n_field = static_cast<uint32_t>(w.n_sub * 32 >> 3) << 17;
                ok = mbar_wait(smem_u32(&bar_acc_empty), (it & 1u) ^ 1u, abortp, g.status, DEV_TIMEOUT_MMA);
                if (!ok) break;
                tc_fence_after();
                for (int grp = grp0; ok && grp < grp1; ++grp, ++gi) {
                    const uint32_t sf = tmem_base + D8_SF_COL + (gi & 1) * 16;
                    ok = mbar_wait(smem_u32(&bar_sf_full[gi & 1]), (gi >> 1) & 1u, abortp, g.status, DEV_TIMEOUT_MMA);
                    if (!ok) break;
                    tc_fence_after();
                    const int kb0 = grp * FP8_GROUP;
#pragma unroll
                    for (int j = 0; j < FP8_GROUP; ++j) {
                        if (ok && kb0 + j < kb_hi) {
                            ok = mbar_wait(smem_u32(&bar_full[stage]), phase, abortp, g.status, DEV_TIMEOUT_MMA);
                            if (ok) {
                                tc_fence_after();
                                const uint32_t idesc = umma_idesc_fp8(128, 0, j) | n_field;
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
#pragma unroll
                                    for (uint32_t k = 0; k < 4; ++k)
                                        umma_fp8_lohi(tmem_base + i * D8_NT, lo + (i * D8_W >> 4) + k * 2u, desc_hi,
                                                      lo + (2 * D8_W >> 4) + k * 2u, desc_hi, idesc, sf + 4 * i, sf + 8,
                                                      (kb0 - kb_lo + j + static_cast<int>(k)) != 0 ? 1u : 0u);
                                }
                                umma_commit(smem_u32(&bar_empty[stage]));
                                lo += D8_STAGE >> 4;
                                if (++stage == D8_STAGES) { stage = 0; phase ^= 1u; lo = lo0; }
                            }
                        }
                    }
                    if (ok) umma_commit(smem_u32(&bar_sf_empty[gi & 1]));
                }
                if (ok) umma_commit(smem_u32(&bar_acc_full));
            }
        }
    } else if (warp >= 6) {
        // ================================================================ scales (four whole warps)
        int gi = 0;
        bool ok = true;
        const uint32_t sf0 = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + D8_SF_COL;
        const int w_blocks = UP ? g.n_cblk : (g.out_cols + 127) / 128;
        for (int item = first_item; ok && item < total_items; item += step_item) {
            const D8Item w = item == first_item ? first : d8_item(g, item);
            const int i = (lane >> 2) & 1;
            const int wb = UP ? w.cb : w.cb * 2 + i;
            const bool have = wb < w_blocks;
            const uint8_t* ws = g.w_scale + ((static_cast<size_t>(w.e) * (UP ? 2 : 1) + (UP ? i : 0)) * w_blocks + wb) * g.nkb;
            const uint4* xs = reinterpret_cast<const uint4*>(g.x_scale + static_cast<size_t>(w.tile) * n_groups * FP8_ATOM);
            for (int grp = grp0; grp < grp1; ++grp, ++gi) {
                const uint4 xw = __ldcg(xs + grp * 32 + lane);
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
                tmem_st4(sf + 4, w1, w1, w1, w1);
                tmem_st4(sf + 8, xw.x, xw.y, xw.z, xw.w);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bar_sf_full[gi & 1]));
            }
        }
    } else {
        // ================================================================ epilogue (warps 2..5)
        const int q = warp & 3;
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
        D8Epi c;
        c.bar_acc_empty = smem_u32(&bar_acc_empty);
        c.bar_meet = smem_u32(&bar_meet);
        c.bar_part_full = smem_u32(&bar_part_full[q]);
        c.bar_part_free = smem_u32(&bar_part_free[q]);
        c.part = stage_base + D8_STAGES * D8_STAGE + (q * 64 * 32 + lane) * 4;
        c.s_top = &s_top[0][0][0];
        c.abortp = abortp;
        c.rank = rank;
        c.meet = c.parts = 0;
        int it = 0;
        bool ok = true;
        for (int item = first_item; ok && item < total_items; item += step_item, ++it) {
            const D8Item w = item == first_item ? first : d8_item(g, item);
            // down: the first rows' weights are asked for while the accumulators fill
            const size_t tile0 = static_cast<size_t>(w.tile) * TILE_M;
            float wgt = UP ? 0.0f : __ldcg(g.row_weight + tile0 + lane);
            ok = mbar_wait(smem_u32(&bar_acc_full), it & 1u, abortp, g.status, DEV_TIMEOUT_EPILOGUE);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            for (int sub = 0; ok && sub < w.n_sub; ++sub) {
                const size_t row0 = tile0 + sub * 32;
                const bool last = sub + 1 == w.n_sub;
                // a token more costs a reduction and a store, so a few rows take the short form
                const int left = w.rows - sub * 32;
                if (!UP && sub > 0) wgt = __ldcg(g.row_weight + row0 + lane);
                ok = left <= 8 ? d8_read_out<UP, SPLIT, 8>(g, c, w, row0, taddr + sub * 32, last, left, wgt)
                               : d8_read_out<UP, SPLIT, 32>(g, c, w, row0, taddr + sub * 32, last, left, wgt);
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
    if constexpr (SPLIT > 1) cluster_sync_all();     // the other CTA may still write here
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, D8_TMEM_COLS);
    }
}

template <bool UP, int SPLIT>
static int d8_launch(const CUtensorMap& tmW, const CUtensorMap& tmX, const Fp8DecArgs& g, cudaStream_t stream) {
    static bool attr_set[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MOMOE_ERR_CUDA;
    if (!attr_set[dev]) {
        if (cudaFuncSetAttribute(fp8_decode_kernel<UP, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 D8_SMEM<SPLIT>) != cudaSuccess)
            return MOMOE_ERR_CUDA;
        attr_set[dev] = true;
    }
    return launch_dependent(fp8_decode_kernel<UP, SPLIT>, sm_count() / SPLIT * SPLIT, D8_THREADS, D8_SMEM<SPLIT>, stream,
                            SPLIT, tmW, tmX, g) == cudaSuccess ? MOMOE_OK : MOMOE_ERR_CUDA;
}

// Whether two CTAs share an item's k axis: when the items leave half of the SMs idle, and the k axis is long enough to pay
// for the meeting.  Whole passes of one token, with the up GEMM shared and not: 20.4 / 18.5 us at 8 k slices, 20.5 / 20.2 at
// 12, 21.4 / 22.4 at 16, 24.6 / 28.7 at 32 (H512, top-4 of 32), 37.0 / 45.2 at 56 (top-8 of 64).
static bool d8_split(const momoe_plan_t* p, const Fp8DecArgs& g) {
    const long long msum = static_cast<long long>(p->M) * p->K;
    const long long tiles = msum / TILE_M + (msum < p->N ? msum : p->N);      // an upper bound
    return tiles * g.n_cblk * 2 <= sm_count() && g.nkb > 3 * FP8_GROUP;
}

static void d8_args(const momoe_plan_t* p, const int32_t* tile_rows, Fp8DecArgs& g) {
    memset(&g, 0, sizeof(g));
    g.sched = p->sched;
    g.tile_expert = p->tile_expert;
    g.tile_rows = tile_rows;
    g.row_weight = p->row_weight;
    g.status = p->status;
    g.tile_cap = static_cast<int>(p->rows_capacity / TILE_M);
}
static inline bool d8_aligned(const void* p) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace momoe

using namespace momoe;

#define MOMOE_API extern "C" __attribute__((visibility("default")))

MOMOE_API int momoe_fp8_up_swiglu_decode(const momoe_plan_t* plan, const int32_t* tile_rows, const uint8_t* x_sorted,
                                         const uint8_t* x_scale, const uint8_t* W1_N2HD, const uint8_t* S1, uint8_t* h_sorted,
                                         uint8_t* h_scale, momoe_stream_t stream) {
    int rc = fp8_check_plan(plan);
    if (rc != MOMOE_OK) return rc;
    if (tile_rows == nullptr || !d8_aligned(x_sorted) || !d8_aligned(x_scale) || !d8_aligned(W1_N2HD) || S1 == nullptr ||
        !d8_aligned(h_sorted) || !d8_aligned(h_scale))
        return MOMOE_ERR_ARG;
    const int D = plan->D, H = plan->H;
    CUtensorMap tmW, tmX;
    if ((rc = encode_tmap_3d(&tmW, W1_N2HD, static_cast<uint64_t>(plan->N) * 2, H, D / 2, 128, D8_K / 2)) != MOMOE_OK)
        return rc;
    if ((rc = encode_tmap_2d(&tmX, x_sorted, plan->rows_capacity, D / 2, 32, D8_K / 2)) != MOMOE_OK) return rc;
    Fp8DecArgs g;
    d8_args(plan, tile_rows, g);
    g.n_cblk = (H + 127) / 128;
    g.nkb = (D + D8_K - 1) / D8_K;
    g.out_cols = H;
    g.x_scale = x_scale;
    g.w_scale = S1;
    g.h = h_sorted;
    g.h_scale = h_scale;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return d8_split(plan, g) ? d8_launch<true, 2>(tmW, tmX, g, st) : d8_launch<true, 1>(tmW, tmX, g, st);
}

MOMOE_API int momoe_fp8_down_scale_decode(const momoe_plan_t* plan, const int32_t* tile_rows, const uint8_t* h_sorted,
                                          const uint8_t* h_scale, const uint8_t* W2_NDH, const uint8_t* S2, void* y_sorted,
                                          float* y_scale, momoe_stream_t stream) {
    int rc = fp8_check_plan(plan);
    if (rc != MOMOE_OK) return rc;
    if (tile_rows == nullptr || !d8_aligned(h_sorted) || !d8_aligned(h_scale) || !d8_aligned(W2_NDH) || S2 == nullptr ||
        !d8_aligned(y_sorted) || y_scale == nullptr)
        return MOMOE_ERR_ARG;
    const int D = plan->D, H = plan->H;
    CUtensorMap tmW, tmX;
    if ((rc = encode_tmap_3d(&tmW, W2_NDH, plan->N, D, H / 2, 128, D8_K / 2)) != MOMOE_OK) return rc;
    if ((rc = encode_tmap_2d(&tmX, h_sorted, plan->rows_capacity, H / 2, 32, D8_K / 2)) != MOMOE_OK) return rc;
    Fp8DecArgs g;
    d8_args(plan, tile_rows, g);
    g.n_cblk = (D + 255) / 256;
    g.nkb = (H + D8_K - 1) / D8_K;
    g.out_cols = D;
    g.x_scale = h_scale;
    g.w_scale = S2;
    g.y = static_cast<__half*>(y_sorted);
    g.y_scale = y_scale;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return d8_split(plan, g) ? d8_launch<false, 2>(tmW, tmX, g, st) : d8_launch<false, 1>(tmW, tmX, g, st);
}
