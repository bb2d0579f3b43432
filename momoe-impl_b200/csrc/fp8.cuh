// 8-bit rows: e4m3 values with one power of two (e8m0 byte, 2^(byte - 127)) for each block of 128.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

namespace momoe {

constexpr int FP8_BLOCK = 128;          // values that share a scale
constexpr int FP8_GROUP = 4;            // blocks whose scale bytes share a 32-bit word
constexpr int FP8_MAX_WIDTH = 1 << 22;  // of expert rows: up to 65535 tiles times column blocks are counted in 32 bits
constexpr int FP8_ATOM = 512;           // bytes of the scales of 128 rows x 4 blocks

// Scales of expert-major rows lie as the tensor core reads them: 512 bytes for each (128-row tile, 4 blocks of 128
// columns), byte (row % 32) * 16 + (row % 128) / 32 * 4 + block % 4.
__host__ __device__ __forceinline__ size_t fp8_atom_offset(size_t row, int group, int n_groups) {
    return ((row >> 7) * static_cast<size_t>(n_groups) + group) * FP8_ATOM + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// The byte of the smallest 2^e with amax <= 448 * 2^e, from the bit pattern of amax >= 0.  448 = 1.75 * 2^8, so this is
// integer arithmetic and exact.  127 (a scale of 1) for a block of zeros; 255 (NaN) where the block holds an infinity or
// a NaN, so that the block's products are NaN as they would be in 32 bits.  A power of two makes the division below
// exact: the one rounding is the conversion to e4m3.
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t amax_bits) {
    if (amax_bits >= 0x7F800000u) return 255u;
    if (amax_bits == 0u) return 127u;
    const int b = static_cast<int>(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return static_cast<uint32_t>(b < 0 ? 0 : b);
}
// 1 / scale (NaN for byte 255); byte is at most 247 otherwise.
__device__ __forceinline__ float fp8_inv_scale(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float((254u - byte) << 23);
}
// Larger magnitude of two as bit patterns: orders infinities and NaN above every finite value.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
__device__ __forceinline__ uint8_t fp8_one(float a) { return __nv_cvt_float_to_fp8(a, __NV_SATFINITE, __NV_E4M3); }

// Result rows of the down GEMM on their way to the weighted sum: fp16 with one power of two for each (row, 256 columns).
// bf16 rows would add a second rounding as large as that of the result itself; fp16 rows have the same size and one 16 times
// smaller, and the power of two keeps them in range.  It comes from the largest finite sum of the row's 256 columns, which is
// stored as 2^13 to 2^15.  Values down to 2^-27 of the largest keep their 11 bits; smaller ones are off by up to 2^-38 of it.
// (A bound from the blocks' scales is known before the sums are and 0.5 to 1.5 us a call cheaper, but a block of zeros has a
// scale of 1, which says nothing about it: beside it real results fell below fp16's normal numbers.)
constexpr int FP8_YBLOCK = 256;

// Magnitude of a sum that sets the power: infinities and NaN stay what they are whatever the power is, and do not set it.
__device__ __forceinline__ float finite_or_zero(float v) { return abs_bits(v) < 0x7F800000u ? fabsf(v) : 0.0f; }
// Exponent e of a row: stored value = sum * w * 2^e.  et: biased exponent of the largest finite sum; w: the row's weight.
__device__ __forceinline__ int fp8_row_exponent(int et, float w) {
    const int ew = static_cast<int>((__float_as_uint(w) >> 23) & 255u);
    // |sum| < 2^(et - 126) and |w| < 2^(ew - 126); the second limit keeps w * 2^e finite
    return min(max(267 - et - ew, -126), min(126, 253 - ew));
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }   // |e| <= 126

// Eight consecutive values of a row as they lie in memory, read past L1 (each is used once), and in 32 bits.
__device__ __forceinline__ uint4 ld_stream(const void* p) {
    uint4 q;
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "l"(p));
    return q;
}
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
    uint4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = ld_stream(p);
        b = ld_stream(p + 4);
    }
    __device__ __forceinline__ void unpack(float (&v)[8]) const {
        v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
        v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
    }
};
template <>
struct Raw8<__nv_bfloat16> {
    uint4 q;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { q = ld_stream(p); }
    __device__ __forceinline__ void unpack(float (&v)[8]) const {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};
template <>
struct Raw8<__half> {
    uint4 q;
    __device__ __forceinline__ void load(const __half* p) { q = ld_stream(p); }
    __device__ __forceinline__ void unpack(float (&v)[8]) const {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
};
// The same through L1, for what other threads read as well.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    Raw8<T> r;
    const uint4* q = reinterpret_cast<const uint4*>(p);
    if constexpr (sizeof(T) == 4) {
        r.a = __ldg(q);
        r.b = __ldg(q + 1);
    } else {
        r.q = __ldg(q);
    }
    r.unpack(v);
}
// Rounds the eight values to T, stores them and leaves the rounded values in v.
template <typename T>
__device__ __forceinline__ void store8(T* p, float (&v)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* p, float (&v)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ void store8<__half>(__half* p, float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
        const float2 f = __half22float2(h);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace momoe
