// The 8-bit block format shared by the quantiser, the RMSNorm output, the matrix product and the optimizer's first moment.
//
// A block is 128 consecutive values along the axis a product reduces over.  amax = the largest finite magnitude, e = the smallest
// whole number with amax <= 448 * 2^e (e >= -127), code = e4m3(x * 2^-e), scale byte = e + 127.  The scale is a power of two because
// v_mfma_scale_f32_*_f8f6f4 multiplies by exactly such a byte per operand row inside the matrix pipe (no fp32 epilogue per block), because
// a block then decodes exactly into bf16 (3 mantissa bits; scale bytes 0..2 reach below its smallest number), and because a floating-point code's relative error does not depend on the
// scale - only one binade of its 18 can be lost to the rounding of e.  Non-finite values become the NaN code and do not enter amax.
#pragma once
#include "common.h"

namespace spn {

static constexpr int QBLK = 128;               // values per scale
static constexpr uint32_t F32_INF_BITS = 0x7f800000u;

// 2^(f - 127) for f in 0..254
__device__ __forceinline__ float pow2_field(int f) { return __uint_as_float(f == 0 ? 0x00400000u : (uint32_t)f << 23); }
// magnitude bits of x, 0 for non-finite values: unsigned order = magnitude order
__device__ __forceinline__ uint32_t finite_bits(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < F32_INF_BITS ? b : 0u;
}
// scale byte of a block with largest magnitude `bits`: the exponent that brings it into (224, 448]; 448 = 1.75 * 2^8
__device__ __forceinline__ int e4m3_scale_byte(uint32_t bits) {
    const int E = (int)(bits >> 23);
    const int b = (E < 1 ? 1 : E) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return b < 0 ? 0 : b;
}
// Largest value over the 16 lanes that share lane >> 4, by DPP (quad permutations, then the mirrors of half rows and rows: no LDS pipe)
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float row16_max(float v) {
    v = fmaxf(v, dpp_f32<0xB1>(v));      // lane ^ 1
    v = fmaxf(v, dpp_f32<0x4E>(v));      // lane ^ 2
    v = fmaxf(v, dpp_f32<0x141>(v));     // 7 - lane of 8
    return fmaxf(v, dpp_f32<0x140>(v));  // 15 - lane of 16
}
// Largest of eight magnitudes, NaN if one of them is (v_maximum3: the v_max forms drop a quiet NaN, but a signalling one makes them drop the
// numbers beside it).  Two values per instruction, no separate absolute values; the s_nop are the two wait states between a vector result
// and a DPP or lane-swap instruction that reads it, which the compiler does not count behind inline asm.
__device__ __forceinline__ float max8_abs(float a, float b, float c, float d, float e, float f, float g, float h) {
    float m;
    asm("v_maximum3_f32 %0, |%1|, |%2|, |%3|\n\tv_maximum3_f32 %0, |%4|, |%5|, %0\n\tv_maximum3_f32 %0, |%6|, |%7|, %0\n\t"
        "v_maximum3_f32 %0, |%8|, |%8|, %0\n\ts_nop 1"
        : "=&v"(m) : "v"(a), "v"(b), "v"(c), "v"(d), "v"(e), "v"(f), "v"(g), "v"(h));
    return m;
}
__device__ __forceinline__ float max8_abs(const float (&x)[8]) { return max8_abs(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]); }
__device__ __forceinline__ float max8_finite(const float (&x)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t b = finite_bits(x[e]);
        m = m > b ? m : b;
    }
    return __uint_as_float(m);
}
// the same without infinities and NaN: a lane that holds one (rare) looks again
__device__ __forceinline__ bool not_finite(float m) { return !(m < __uint_as_float(F32_INF_BITS)); }
__device__ __forceinline__ float max8_scale(const float (&x)[8]) {
    float m = max8_abs(x);
    if (not_finite(m)) m = max8_finite(x);
    return m;
}
// scale byte of the block that 16 lanes hold in eight values each
__device__ __forceinline__ int e4m3_block_byte(const float (&x)[8]) { return e4m3_scale_byte(__float_as_uint(row16_max(max8_scale(x)))); }
// eight values times a power of two -> eight codes: v_cvt_pk_fp8_f32 rounds to nearest even and turns infinities and NaN into the NaN code;
// finite values cannot overflow under their block's scale
__device__ __forceinline__ u32x2 e4m3_pack8(const float (&x)[8], float inv) {
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[4] * inv, x[5] * inv, hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[6] * inv, x[7] * inv, hi, true);
    return u32x2{(uint32_t)lo, (uint32_t)hi};
}
__device__ __forceinline__ void e4m3_unpack8(u32x2 c, float scale, float (&x)[8]) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[0], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[0], true);
    const f32x2 d = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[1], false), f = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[1], true);
    x[0] = a[0] * scale; x[1] = a[1] * scale; x[2] = b[0] * scale; x[3] = b[1] * scale;
    x[4] = d[0] * scale; x[5] = d[1] * scale; x[6] = f[0] * scale; x[7] = f[1] * scale;
}

// ---- eight consecutive elements of fp32 / bf16 / fp16 memory at any element alignment (the hardware takes unaligned vector accesses in
// global memory: rows of odd pitch need no second code path).  Loads come as bits and are converted by a separate call: a conversion inside
// a guard would wait for its load before the next one is issued, so kernels issue all their loads first.
typedef _Float16 f16_t;
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Vec8 { uint32_t w[2 * sizeof(T)]; };

// `count` of the eight valid (any number <= 0: none), zeros behind them; RAGGED = false: count is >= 8 or <= 0
template <bool RAGGED, typename T>
__device__ __forceinline__ Vec8<T> fetch8(const T* p, int count) {
    Vec8<T> t;
#pragma unroll
    for (int k = 0; k < 2 * (int)sizeof(T); ++k) t.w[k] = 0u;
    if (count >= 8) {
        t = *(const Vec8<T>*)p;
    } else if (RAGGED && count > 0) {
#pragma unroll
        for (int e = 0; e < 7; ++e) {
            if (e >= count) continue;
            if constexpr (sizeof(T) == 4) t.w[e] = __builtin_bit_cast(uint32_t, p[e]);
            else t.w[e >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, p[e]) << (16 * (e & 1));
        }
    }
    return t;
}
template <typename T>
__device__ __forceinline__ Vec8<T> fetch8_whole(const T* p) { return *(const Vec8<T>*)p; }
template <typename T>
__device__ __forceinline__ void to_f32(const Vec8<T>& t, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (sizeof(T) == 4) x[e] = __uint_as_float(t.w[e]);
        else x[e] = (float)__builtin_bit_cast(T, (uint16_t)(t.w[e >> 1] >> (16 * (e & 1))));
    }
}
// two numbers rounded to 16 bits each in one instruction (written one by one the compiler takes two conversions and a merge)
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef T T2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, T2));
}
template <bool RAGGED, typename T>
__device__ __forceinline__ void put8(T* p, int count, const float (&x)[8]) {
    if (count >= 8) {
        Vec8<T> t;
#pragma unroll
        for (int k = 0; k < 2 * (int)sizeof(T); ++k) {
            if constexpr (sizeof(T) == 4) t.w[k] = __float_as_uint(x[k]);
            else t.w[k] = pack2<T>(x[2 * k], x[2 * k + 1]);
        }
        *(Vec8<T>*)p = t;
    } else if (RAGGED && count > 0) {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < count) p[e] = (T)x[e];
    }
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, int count, float (&x)[8]) { to_f32(fetch8<true>(p, count), x); }
template <typename T>
__device__ __forceinline__ void store8(T* p, int count, const float (&x)[8]) { put8<true>(p, count, x); }
// element types at the C boundary
enum ElemType { ET_F32 = 0, ET_BF16 = 1, ET_F16 = 2, ET_E4M3 = 3 };

__host__ __device__ static inline int qblocks(int64_t k) { return (int)((k + QBLK - 1) / QBLK); }
__host__ __device__ static inline int qscale_pitch(int64_t k) { return (qblocks(k) + 3) & ~3; }

}  // namespace spn
