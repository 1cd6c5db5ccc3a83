// AdamW over many tensors in one launch, moments in 32 or 8 bits.
//
//   m = b1 m + (1 - b1) g ;  v = b2 v + (1 - b2) g^2 ;  p = p (1 - lr wd) - lr / bc1 * m / (sqrt(v / bc2) + eps)
//
// torch.optim.AdamW's arithmetic (train_negplus.py:77-84).  The tensors' addresses that do not change between steps (parameters and
// moments) live in a device table the caller builds once; the gradients', which autograd may replace every step, travel in the kernel's
// argument block: no upload per step, and a captured launch carries them.
//
// 8-bit moments, blocks of 128 with one byte of scale each: m as e4m3 (fp8.h), v as an UNSIGNED code of 5 exponent and 3 mantissa
// bits - v spans the square of m's range, and an element whose v fell to 0 while its m did not would take a step of m / eps; a positive
// v is never stored as 0.  Both are rounded stochastically with 16 random bits each from a hash of (seed, step, element index): where
// gradients are small v falls by a share of 1 - b2 per step (0.1 % at b2 = 0.999); rounding to nearest would drop every change of less than half a
// code's step (3-6 %), and the average would never decay.  The update itself uses the unrounded moments in fp32.
//
// Bound by HBM: 16 bytes per element with 8-bit moments and fp32 gradients, 28 with fp32 moments.  16 lanes hold a block of 128, so its scale is one DPP
// reduction; chunks of 4 096 elements of one tensor are the unit of work, 4 workgroups per CU walk them (404 us below; 2: 410, 8: 402).
// Measured: 123.65 M parameters in 150 tensors, 8 bits: 387-407 us, 4.9-5.1 TB/s (a copy: 5.0).  330 ragged tensors, 32 bits, bf16 gradients: 40 us.  Both moments decoded to bf16: 134 us.
#include "fp8.h"
#include "kernels.h"

namespace spn {

static constexpr int AM_CHUNK = 4096;          // elements of one tensor per work item

// 32-bit mixing: two multiply-xorshift rounds, every input bit reaches every output bit.  Shifts and factors are from Chris Wellons' published search
// for 32-bit integer hashes of low bias (2018).
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x7feb352du;
    x = (x ^ (x >> 15)) * 0x846ca68bu;
    return x ^ (x >> 16);
}

// v: codes are the top bits of an fp32 number scaled by 2^-byte so that the block's largest has exponent field <= 31 (mantissa <= 1.75 there)
__device__ __forceinline__ int ue5m3_scale_byte(uint32_t bits) {
    const int E = (int)(bits >> 23);
    const int b = (E < 1 ? 1 : E) - 31 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return b < 0 ? 0 : b;
}
__device__ __forceinline__ float ue5m3_decode(uint32_t code, int byte) {
    return code == 0xffu ? __uint_as_float(0x7fc00000u) : ldexpf(__uint_as_float(code << 20), byte);
}

// One element.  The fused multiply-adds are written out so that the result does not depend on what the compiler contracts around it: they
// are the ones adamw_kernel (elementwise.hip) compiles to, whose last n % 4 elements take the second form of v - a tensor gives the same
// bits through either kernel.
__device__ __forceinline__ void adamw_element(float& p, float g, float& m, float& v, const AdamGroup& h, float decay, float step_size, float rsqrt_bc2,
                                              bool last) {
#pragma clang fp contract(off)
    const float q = h.omb2 * g;
    m = __builtin_fmaf(h.omb1, g, h.b1 * m);
    v = last ? __builtin_fmaf(g, q, h.b2 * v) : __builtin_fmaf(h.b2, v, g * q);
    const float denom = __builtin_fmaf(rsqrt_bc2, sqrtf(v), h.eps);
    p = __builtin_fmaf(decay, p, -(step_size * (m / denom)));
}

// The same step where the moments are kept in 8 bits: square root and quotient by the one-ulp instructions (the moments' own rounding is
// 2^-4 of a value; the exact forms cost a third of the kernel's vector instructions).  The root instruction takes numbers below 2^-126 for 0, which
// would divide m by eps alone: small v are brought up by 2^64 first.
__device__ __forceinline__ void adamw_element8(float& p, float g, float& m, float& v, const AdamGroup& h, float decay, float step_size, float rsqrt_bc2) {
    m = __builtin_fmaf(h.omb1, g, h.b1 * m);
    v = __builtin_fmaf(h.b2, v, g * (h.omb2 * g));
    const bool small = v < 0x1p-100f;
    const float root = __builtin_amdgcn_sqrtf(small ? v * 0x1p64f : v);
    const float denom = __builtin_fmaf(rsqrt_bc2, small ? root * 0x1p-32f : root, h.eps);
    p = __builtin_fmaf(decay, p, -(step_size * (m * __builtin_amdgcn_rcpf(denom))));
}

__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
__device__ __forceinline__ uint32_t row16_max_u32(uint32_t v) {
    v = max_u32(v, dpp_u32<0xB1>(v));
    v = max_u32(v, dpp_u32<0x4E>(v));
    v = max_u32(v, dpp_u32<0x141>(v));
    return max_u32(v, dpp_u32<0x140>(v));
}

// Stochastic rounding to 8 bits: the value times the power of two that lines the code's exponent field up with fp32's, 20 random low bits
// added (16 of them random), the upper bits kept - below the smallest normal code fp32's own subnormals do the fixed-point rounding.
// FINITE: the block holds no infinity or NaN (decided for 16 lanes at once).
template <bool FINITE>
__device__ __forceinline__ void adamw_encode(const float (&M)[8], const float (&V)[8], int sm, int sv, uint32_t idx, uint32_t key, u32x2& cm, u32x2& cv) {
    uint32_t c[8], d[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t r = mix32((idx + e) ^ key);
        c[e] = (__float_as_uint(ldexpf(fabsf(M[e]), 7 - sm)) + ((r & 0xffffu) << 4)) >> 20;
        d[e] = (__float_as_uint(ldexpf(V[e], -sv)) + ((r >> 16) << 4)) >> 20;
        d[e] = max_u32(d[e], V[e] > 0.f ? 1u : 0u);
        if constexpr (!FINITE) {
            c[e] = (__float_as_uint(M[e]) & 0x7fffffffu) < F32_INF_BITS ? c[e] : 0x7fu;
            d[e] = __float_as_uint(V[e]) < F32_INF_BITS ? d[e] : 0xffu;
        }
        c[e] |= (__float_as_uint(M[e]) >> 24) & 0x80u;
    }
    cm = u32x2{c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24};
    cv = u32x2{d[0] | d[1] << 8 | d[2] << 16 | d[3] << 24, d[4] | d[5] << 8 | d[6] << 16 | d[7] << 24};
}

// 2048 elements of one tensor from `start` on, 8 per thread: 16 lanes hold a block
// FULL: the tensor reaches past them
template <int BITS, bool FULL, typename TG>
__device__ __forceinline__ void adamw_piece(const AdamTensor& t, const TG* g, int64_t start, const AdamGroup& h, float decay, float step_size,
                                            float rsqrt_bc2, float inv_scale, uint32_t key) {
    const int64_t i = start + (int)threadIdx.x * 8, left = t.n - i;
    const int cnt = FULL || left >= 8 ? 8 : left > 0 ? (int)left : 0;
    float P[8], G[8], M[8], V[8];
    const Vec8<float> rp = fetch8<!FULL>(t.p + i, cnt);
    const Vec8<TG> rg = fetch8<!FULL>(g + i, cnt);
    if constexpr (BITS == 32) {
        const Vec8<float> rm = fetch8<!FULL>((const float*)t.m + i, cnt), rv = fetch8<!FULL>((const float*)t.v + i, cnt);
        to_f32(rp, P);
        to_f32(rg, G);
        to_f32(rm, M);
        to_f32(rv, V);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            adamw_element(P[e], G[e] * inv_scale, M[e], V[e], h, decay, step_size, rsqrt_bc2, i + e >= (t.n & ~(int64_t)3));
        put8<!FULL>(t.p + i, cnt, P);
        put8<!FULL>((float*)t.m + i, cnt, M);
        put8<!FULL>((float*)t.v + i, cnt, V);
    } else {
        // codes and scale bytes exist up to the next multiple of 128: whole blocks are read and written
        const bool live = FULL || (i & ~(int64_t)(QBLK - 1)) < t.n;
        u32x2 cm = {0, 0}, cv = {0, 0};
        int bm = 0, bv = 0;
        if (live) {
            cm = *(const u32x2*)((const uint8_t*)t.m + i);
            cv = *(const u32x2*)((const uint8_t*)t.v + i);
            bm = t.m_scale[i >> 7];
            bv = t.v_scale[i >> 7];
        }
        to_f32(rp, P);
        to_f32(rg, G);
        e4m3_unpack8(cm, pow2_field(bm), M);
#pragma unroll
        for (int e = 0; e < 8; ++e) V[e] = ue5m3_decode((cv[e >> 2] >> (8 * (e & 3))) & 0xffu, bv);
#pragma unroll
        for (int e = 0; e < 8; ++e) adamw_element8(P[e], G[e] * inv_scale, M[e], V[e], h, decay, step_size, rsqrt_bc2);
        put8<!FULL>(t.p + i, cnt, P);
        uint32_t am = 0, av = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (!FULL && e >= cnt) { M[e] = 0.f; V[e] = 0.f; }    // what lies behind the tensor's end stays zero
            am = max_u32(am, __float_as_uint(M[e]) & 0x7fffffffu);
            av = max_u32(av, __float_as_uint(V[e]));                // v >= 0: a sign bit means NaN
        }
        am = row16_max_u32(am);
        av = row16_max_u32(av);
        const bool finite = am < F32_INF_BITS && av < F32_INF_BITS;
        if (!finite) {
            am = row16_max_u32(__float_as_uint(max8_finite(M)));
            av = row16_max_u32(__float_as_uint(max8_finite(V)));
        }
        const int sm = e4m3_scale_byte(am), sv = ue5m3_scale_byte(av);
        const uint64_t at = (uint64_t)(t.index0 + i);      // a multiple of 8: the upper half is the same for all eight
        const uint32_t idx = (uint32_t)at;
        if (at >> 32) key ^= mix32((uint32_t)(at >> 32));
        if (finite) adamw_encode<true>(M, V, sm, sv, idx, key, cm, cv);
        else adamw_encode<false>(M, V, sm, sv, idx, key, cm, cv);
        if (live) {
            *(u32x2*)((uint8_t*)t.m + i) = cm;
            *(u32x2*)((uint8_t*)t.v + i) = cv;
            if ((threadIdx.x & 15) == 0) {
                t.m_scale[i >> 7] = (uint8_t)sm;
                t.v_scale[i >> 7] = (uint8_t)sv;
            }
        }
    }
}

template <int BITS, typename TG>
__device__ __forceinline__ void adamw_chunk(const AdamTensor& t, const TG* g, int64_t start, const AdamGroup& h, float step_size, float rsqrt_bc2,
                                            float inv_scale, uint32_t key) {
    const float decay = __builtin_fmaf(-h.lr, h.wd, 1.0f);
    for (int64_t s = start; s < t.n && s < start + AM_CHUNK; s += 2048) {
        if (s + 2048 <= t.n) adamw_piece<BITS, true, TG>(t, g, s, h, decay, step_size, rsqrt_bc2, inv_scale, key);
        else adamw_piece<BITS, false, TG>(t, g, s, h, decay, step_size, rsqrt_bc2, inv_scale, key);
    }
}

template <int BITS>
__global__ __launch_bounds__(256) void adamw_multi_kernel(const AdamMulti a) {
    if (a.found_inf && *a.found_inf != 0.f) return;
    __shared__ float bc[AM_GROUPS][2];
    __shared__ uint32_t skey;
    if ((int)threadIdx.x < a.n_groups) {
        if (a.step_dev) {
            const double t = (double)*a.step_dev;
            bc[threadIdx.x][0] = (float)(1.0 - pow(a.beta[threadIdx.x][0], t));
            bc[threadIdx.x][1] = (float)(1.0 / sqrt(1.0 - pow(a.beta[threadIdx.x][1], t)));
        } else {
            bc[threadIdx.x][0] = a.bc1[threadIdx.x];
            bc[threadIdx.x][1] = a.rsqrt_bc2[threadIdx.x];
        }
        if (threadIdx.x == 0) {
            const uint32_t step = a.step_dev ? (uint32_t)*a.step_dev : (uint32_t)a.step;
            skey = mix32(a.seed ^ mix32(step + 0x9e3779b9u));
        }
    }
    __syncthreads();
    const float inv_scale = a.grad_scale ? a.inv_scale / *a.grad_scale : a.inv_scale;
    for (int c = a.chunk_begin + (int)blockIdx.x; c < a.chunk_end; c += (int)gridDim.x) {
        const int ti = a.chunks[2 * c];
        const int64_t start = (int64_t)a.chunks[2 * c + 1] * AM_CHUNK;
        const void* g = a.g[ti - a.tensor_begin];
        if (!g) continue;
        const AdamTensor t = a.table[ti];
        const AdamGroup h = a.group[t.group];
        const float step_size = h.lr / bc[t.group][0], rsqrt_bc2 = bc[t.group][1];
        const int gt = a.gtype[ti - a.tensor_begin];
        if (gt == ET_F32) adamw_chunk<BITS>(t, (const float*)g, start, h, step_size, rsqrt_bc2, inv_scale, skey);
        else if (gt == ET_BF16) adamw_chunk<BITS>(t, (const bf16_t*)g, start, h, step_size, rsqrt_bc2, inv_scale, skey);
        else adamw_chunk<BITS>(t, (const f16_t*)g, start, h, step_size, rsqrt_bc2, inv_scale, skey);
    }
}

int adamw_multi(const AdamMulti& a, int bits, hipStream_t st) {
    const int chunks = a.chunk_end - a.chunk_begin;
    if (chunks <= 0) return SPN_OK;
    const int cap = 4 * device_cu_count();
    const int grid = chunks < cap ? chunks : cap;
    if (bits == 8) hipLaunchKernelGGL(adamw_multi_kernel<8>, dim3(grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(adamw_multi_kernel<32>, dim3(grid), dim3(256), 0, st, a);
    SPN_CHECK_LAUNCH();
    return SPN_OK;
}

// Both 8-bit moments as plain numbers (checkpoints, inspection): n a multiple of 128.
template <typename T>
__global__ __launch_bounds__(256) void adamw_moments_kernel(const uint8_t* __restrict__ m, const uint8_t* __restrict__ ms,
                                                            const uint8_t* __restrict__ v, const uint8_t* __restrict__ vs, T* __restrict__ mo,
                                                            T* __restrict__ vo, int64_t n) {
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 2048) {
        const u32x2 cm = *(const u32x2*)(m + i), cv = *(const u32x2*)(v + i);
        float x[8];
        e4m3_unpack8(cm, pow2_field(ms[i >> 7]), x);
        store8(mo + i, 8, x);
        const int bv = vs[i >> 7];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = ue5m3_decode((cv[e >> 2] >> (8 * (e & 3))) & 0xffu, bv);
        store8(vo + i, 8, x);
    }
}

int adamw_moments(const uint8_t* m, const uint8_t* ms, const uint8_t* v, const uint8_t* vs, void* mo, void* vo, int type, int64_t n, hipStream_t st) {
    if (n == 0) return SPN_OK;
    if ((uintptr_t)m % 8 || (uintptr_t)v % 8) return SPN_ERR_ARG;
    const int64_t want = (n + 2047) / 2048;
    const int grid = (int)(want < 8192 ? want : 8192);
    if (type == ET_F32) hipLaunchKernelGGL(adamw_moments_kernel<float>, dim3(grid), dim3(256), 0, st, m, ms, v, vs, (float*)mo, (float*)vo, n);
    else if (type == ET_BF16) hipLaunchKernelGGL(adamw_moments_kernel<bf16_t>, dim3(grid), dim3(256), 0, st, m, ms, v, vs, (bf16_t*)mo, (bf16_t*)vo, n);
    else return SPN_ERR_ARG;
    SPN_CHECK_LAUNCH();
    return SPN_OK;
}

}  // namespace spn
