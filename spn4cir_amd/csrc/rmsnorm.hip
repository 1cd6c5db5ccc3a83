// Root-mean-square norm with the residual's addition, forward and backward.
//
//   h = T(x + r)  (x itself without a residual),  rstd = 1 / sqrt(mean(h^2) + eps),  y = h * rstd * gamma
//   dxh = dy * gamma,  dh = rstd * (dxh - xh * mean(dxh * xh)) + dh_in,  dgamma = sum over rows of dy * xh,  xh = h * rstd
//
// The sum is rounded to the stream's type first and the rounded value is normalised: the backward pass, which reads h, then differentiates
// exactly what the forward pass computed.  All arithmetic in fp32.  y leaves in 8-bit blocks (fp8.h) if asked: the row is in registers,
// 16 lanes hold a block of 128, so the scale costs one 4-step reduction and no pass over memory.
// Bound by HBM: x, r (forward) and dy, h, dh (backward) are read once, h, y, dx written once.  A wave owns a row of up to 1 024 columns, a workgroup
// of 4 waves a wider one (up to 64 columns per lane, in registers).  Loads are issued as raw bits before any is converted, the forward pass has
// the next row's in flight under the current row's reduction.  dgamma: one partial row per workgroup, then a fold in a
// fixed order; of few rows, column sums by further workgroups of the same launch.
// Measured (a copy reaches 5.0 TB/s on this part, reads alone more): forward 19712 x 768, bf16 + fp32 stream -> bf16: 31.0 us, 5.9 TB/s;
// backward of it 34.9 + 4.7 us (fold), 6.1 TB/s; forward 16384 x 4096 bf16 + bf16 -> 8-bit blocks: 81-92 us, 5.1-5.8 TB/s; 4 x 4096: 3.4 us.
#include "fp8.h"
#include "kernels.h"
#include <type_traits>

namespace spn {

static constexpr int RMS_MAX_W = 16384;

// sum over the TPR threads that share a row
template <int TPR>
__device__ __forceinline__ float rms_row_sum(float s, float* red) {
    s = wave_sum(s);
    if constexpr (TPR > 64) {
        const int w = threadIdx.x >> 6;
        __syncthreads();                                   // the previous row's partials have been read
        if ((threadIdx.x & 63) == 0) red[w] = s;
        __syncthreads();
        s = 0.f;
#pragma unroll
        for (int k = 0; k < TPR / 64; ++k) s += red[k];
    }
    return s;
}

struct NoRes {};

// Persistent: a wave (TPR = 64) or workgroup (256) walks its rows with gamma in registers and the next row's loads in flight under the
// current row's reduction and stores.  RAGGED: W is no multiple of 8.
template <typename TX, typename TR, int TPR, int NV, bool RAGGED>
__global__ __launch_bounds__(256) void rmsnorm_fwd_kernel(const RmsArgs a) {
    __shared__ float red[4];
    constexpr bool RES = !__is_same(TR, NoRes);
    using TR1 = std::conditional_t<RES, TR, TX>;
    const int t = threadIdx.x % TPR, Wp = qblocks(a.W) * QBLK, sp = qscale_pitch(a.W);
    constexpr int rpb = 256 / TPR;
    const int64_t stride = (int64_t)gridDim.x * rpb;
    int64_t row = (int64_t)blockIdx.x * rpb + threadIdx.x / TPR;
    Vec8<float> gm[NV];
    Vec8<TX> xn[NV];
    Vec8<TR1> rn[NV];
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            xn[i] = fetch8<RAGGED>((const TX*)a.x + r * a.ldx + c, a.W - c);
        }
        if constexpr (RES) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (t + i * TPR) * 8;
                rn[i] = fetch8<RAGGED>((const TR*)a.r + r * a.ldr + c, a.W - c);
            }
        }
    };
    if (row < a.rows) fetch(row);
#pragma unroll
    for (int i = 0; i < NV; ++i) gm[i] = fetch8<RAGGED>(a.gamma + (t + i * TPR) * 8, a.W - (t + i * TPR) * 8);
    for (; row < a.rows; row += stride) {
        float v[NV][8];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            to_f32(xn[i], v[i]);
            if constexpr (RES) {
                float r[8];
                to_f32(rn[i], r);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] = (float)(TR)(v[i][e] + r[e]);
            }
        }
        if (row + stride < a.rows) fetch(row + stride);
        if constexpr (RES) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (t + i * TPR) * 8;
                put8<RAGGED>((TR*)a.h + row * a.W + c, a.W - c, v[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) s += v[i][e] * v[i][e];
        const float rs = 1.0f / sqrtf(rms_row_sum<TPR>(s, red) / (float)a.W + a.eps);
        if (t == 0) a.rstd[row] = rs;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            float gf[8];
            to_f32(gm[i], gf);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = (RAGGED ? c + e < a.W : c < a.W) ? v[i][e] * rs * gf[e] : 0.f;   // zero codes behind W, also where rs is NaN
            if (a.yt == ET_E4M3) {                         // uniform
                const int sb = e4m3_block_byte(v[i]);
                if (c < Wp) *(u32x2*)((uint8_t*)a.y + row * Wp + c) = e4m3_pack8(v[i], pow2_field(254 - sb));
                if ((t & 15) == 0 && (c >> 7) < sp) a.y_scale[row * sp + (c >> 7)] = c < Wp ? (uint8_t)sb : (uint8_t)127;
            } else if (a.yt == ET_BF16) {
                put8<RAGGED>((bf16_t*)a.y + row * a.W + c, a.W - c, v[i]);
            } else if (a.yt == ET_F16) {
                put8<RAGGED>((f16_t*)a.y + row * a.W + c, a.W - c, v[i]);
            } else {
                put8<RAGGED>((float*)a.y + row * a.W + c, a.W - c, v[i]);
            }
        }
        if (a.yt == ET_E4M3) {
            // scale bytes behind the columns the row's vectors cover
            for (int b = (TPR * NV * 8) / QBLK + t; b < sp; b += TPR) a.y_scale[row * sp + b] = 127;
        }
    }
}

template <typename TX, typename TR>
static int rms_fwd_launch(const RmsArgs& a, hipStream_t st) {
    const int nv = (a.W + 7) / 8;
    // workgroups per CU, 19712 x 768 and 16384 x 4096: 8: 33.0 and 97.5 us, 16: 31.6 and 93.5, 32: 31.0 and 92.1
#define SPN_RMS_FWD(TPR_, NV_)                                                                                             \
    do {                                                                                                                   \
        const int64_t blocks = (a.rows + 256 / TPR_ - 1) / (256 / TPR_), cap = 32 * (int64_t)device_cu_count();            \
        const dim3 grid((unsigned)(blocks < cap ? blocks : cap));                                                          \
        if (a.W % 8) hipLaunchKernelGGL((rmsnorm_fwd_kernel<TX, TR, TPR_, NV_, true>), grid, dim3(256), 0, st, a);         \
        else hipLaunchKernelGGL((rmsnorm_fwd_kernel<TX, TR, TPR_, NV_, false>), grid, dim3(256), 0, st, a);                \
    } while (0)
    if (nv <= 64) SPN_RMS_FWD(64, 1);
    else if (nv <= 128) SPN_RMS_FWD(64, 2);
    else if (nv <= 256) SPN_RMS_FWD(256, 1);
    else if (nv <= 512) SPN_RMS_FWD(256, 2);
    else if (nv <= 1024) SPN_RMS_FWD(256, 4);
    else SPN_RMS_FWD(256, 8);
#undef SPN_RMS_FWD
    SPN_CHECK_LAUNCH();
    return SPN_OK;
}

int rmsnorm_fwd(const RmsArgs& a, hipStream_t st) {
    if (a.rows < 0 || a.W <= 0 || !a.x || !a.gamma || !a.y || !a.rstd || (a.r && !a.h) || (a.yt == ET_E4M3 && !a.y_scale)) return SPN_ERR_ARG;
    if (a.W > RMS_MAX_W || a.ldx < a.W || (a.r && a.ldr < a.W)) return SPN_ERR_SHAPE;
    if (a.rows == 0) return SPN_OK;
    if (a.yt < ET_F32 || a.yt > ET_E4M3 || a.xt < ET_F32 || a.xt > ET_F16 || (a.yt == ET_E4M3 && (uintptr_t)a.y % 8)) return SPN_ERR_ARG;
    if (!a.r) {
        if (a.xt == ET_F32) return rms_fwd_launch<float, NoRes>(a, st);
        if (a.xt == ET_BF16) return rms_fwd_launch<bf16_t, NoRes>(a, st);
        return rms_fwd_launch<f16_t, NoRes>(a, st);
    }
    if (a.rt == ET_F32) {
        if (a.xt == ET_F32) return rms_fwd_launch<float, float>(a, st);
        if (a.xt == ET_BF16) return rms_fwd_launch<bf16_t, float>(a, st);
        return rms_fwd_launch<f16_t, float>(a, st);
    }
    if (a.rt != a.xt) return SPN_ERR_ARG;
    if (a.xt == ET_BF16) return rms_fwd_launch<bf16_t, bf16_t>(a, st);
    return rms_fwd_launch<f16_t, f16_t>(a, st);
}

// dgamma of 32 columns straight from dy, h and rstd: 4 threads of 8 columns x 64 row lanes, eight rows in flight per thread.  Rows behind the last are
// read as the last one and left out: a guard around a load would wait for it.  WHOLE: all 32 columns exist.
template <typename TD, typename TH, bool WHOLE>
__device__ __forceinline__ void rms_columns(const RmsBwdArgs& a, int block, float (*red)[33]) {
    const int rl = threadIdx.x >> 2, c = block * 32 + (threadIdx.x & 3) * 8, cnt = a.W - c;
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = 0.f;
    for (int64_t r0 = rl; r0 < a.rows; r0 += 512) {
        Vec8<TD> rd[8];
        Vec8<TH> rh[8];
        float rs[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t r = r0 + k * 64 < a.rows ? r0 + k * 64 : a.rows - 1;
            const TD* pd = (const TD*)a.dy + r * a.lddy + c;
            const TH* ph = (const TH*)a.h + r * a.ldh + c;
            rd[k] = WHOLE ? fetch8_whole(pd) : fetch8<true>(pd, cnt);
            rh[k] = WHOLE ? fetch8_whole(ph) : fetch8<true>(ph, cnt);
            rs[k] = a.rstd[r];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float d[8], x[8];
            to_f32(rd[k], d);
            to_f32(rh[k], x);
            if (r0 + k * 64 < a.rows) {
#pragma unroll
                for (int e = 0; e < 8; ++e) s[e] += d[e] * (x[e] * rs[k]);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) red[rl][(threadIdx.x & 3) * 8 + e] = s[e];
    __syncthreads();
    const int col = threadIdx.x & 31, part = threadIdx.x >> 5;
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += red[part * 8 + k][col];
    __syncthreads();
    red[part][col] = t;
    __syncthreads();
    if (threadIdx.x < 32 && block * 32 + col < a.W) {
        t = red[0][col];
#pragma unroll
        for (int k = 1; k < 8; ++k) t += red[k][col];
        a.dgamma[block * 32 + col] = t;
    }
}

template <typename TD, typename TH, int TPR, int NV, bool RAGGED>
__global__ __launch_bounds__(256) void rmsnorm_bwd_kernel(const RmsBwdArgs a) {
    __shared__ float shared[TPR == 256 ? 64 * 33 : 4 * TPR * NV * 8 > 64 * 33 ? 4 * TPR * NV * 8 : 64 * 33];
    __shared__ float red[4];
    if ((int)blockIdx.x >= a.row_blocks) {                 // uniform
        const int block = (int)blockIdx.x - a.row_blocks;
        if (block * 32 + 32 <= a.W) rms_columns<TD, TH, true>(a, block, (float(*)[33])shared);
        else rms_columns<TD, TH, false>(a, block, (float(*)[33])shared);
        return;
    }
    const int t = threadIdx.x % TPR;
    constexpr int rpb = 256 / TPR;
    float dg[NV][8];
    Vec8<float> gm[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        gm[i] = fetch8<RAGGED>(a.gamma + (t + i * TPR) * 8, a.W - (t + i * TPR) * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) dg[i][e] = 0.f;
    }
    const int64_t steps = (a.rows + rpb - 1) / rpb;        // every thread of a workgroup takes part in every reduction
    for (int64_t k = blockIdx.x; k < steps; k += a.row_blocks) {
        const int64_t row = k * rpb + threadIdx.x / TPR;
        const bool live = row < a.rows;
        const int W = live ? a.W : 0;
        const float rs = live ? a.rstd[row] : 0.f;
        Vec8<TD> rd[NV];
        Vec8<TH> rh[NV], rp[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            rd[i] = fetch8<RAGGED>((const TD*)a.dy + row * a.lddy + c, W - c);
            rh[i] = fetch8<RAGGED>((const TH*)a.h + row * a.ldh + c, W - c);
        }
        if (a.dh) {                                        // uniform
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (t + i * TPR) * 8;
                rp[i] = fetch8<RAGGED>((const TH*)a.dh + row * a.lddh + c, W - c);
            }
        }
        float xh[NV][8], u[NV][8];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float gf[8];
            to_f32(rd[i], u[i]);
            to_f32(rh[i], xh[i]);
            to_f32(gm[i], gf);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                xh[i][e] *= rs;
                dg[i][e] += u[i][e] * xh[i][e];
                u[i][e] *= gf[e];
                s += u[i][e] * xh[i][e];
            }
        }
        s = rms_row_sum<TPR>(s, red) / (float)a.W;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            float d[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = rs * (u[i][e] - xh[i][e] * s);
            if (a.dh) {
                float p[8];
                to_f32(rp[i], p);
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] += p[e];
            }
            put8<RAGGED>((TH*)a.dx + row * a.W + c, W - c, d);
            if (a.dx2) {
                if (a.dx2t == ET_BF16) put8<RAGGED>((bf16_t*)a.dx2 + row * a.W + c, W - c, d);
                else if (a.dx2t == ET_F16) put8<RAGGED>((f16_t*)a.dx2 + row * a.W + c, W - c, d);
                else put8<RAGGED>((float*)a.dx2 + row * a.W + c, W - c, d);
            }
        }
    }
    if (a.row_blocks < (int)gridDim.x) return;             // others sum the columns
    // one partial row per workgroup
    float* w = a.ws + (size_t)blockIdx.x * ((a.W + 3) & ~3);
    if constexpr (TPR == 256) {
#pragma unroll
        for (int i = 0; i < NV; ++i) put8<RAGGED>(w + (t + i * TPR) * 8, a.W - (t + i * TPR) * 8, dg[i]);
    } else {
        float(*const part)[TPR * NV * 8] = (float(*)[TPR * NV * 8])shared;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) part[threadIdx.x / TPR][(t + i * TPR) * 8 + e] = dg[i][e];
        __syncthreads();
        for (int c = threadIdx.x; c < a.W; c += 256) w[c] = (part[0][c] + part[1][c]) + (part[2][c] + part[3][c]);
    }
}

// dgamma[c] = sum of the partial rows: 16 columns per workgroup, 64 row lanes of four columns each, all of a lane's loads in flight
__global__ __launch_bounds__(256) void rms_fold_kernel(const float* __restrict__ ws, int n, int W, int ld, float* __restrict__ out) {
    __shared__ f32x4 red[64][4];
    const int q = threadIdx.x & 3, rl = threadIdx.x >> 2, c = blockIdx.x * 16 + q * 4;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (c < ld) {
#pragma unroll 8
        for (int r = rl; r < n; r += 64) s += *(const f32x4*)(ws + (size_t)r * ld + c);
    }
    red[rl][q] = s;
    __syncthreads();
    if (threadIdx.x < 16) {
        const int col = blockIdx.x * 16 + threadIdx.x;
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 64; ++k) t += red[k][threadIdx.x >> 2][threadIdx.x & 3];
        if (col < W) out[col] = t;
    }
}

static int rms_bwd_blocks(int64_t rows, int W) {
    // two workgroups per CU, each with one partial row of dgamma (19712 x 768: 35.0 us; one per CU 39.3, four 38.1)
    const int rpb = W <= 1024 ? 4 : 1;
    const int64_t want = (rows + rpb - 1) / rpb, cap = 2 * (int64_t)device_cu_count();
    return (int)(want < cap ? want : cap);
}
// Few rows of a matrix that stays in the caches: further workgroups of the same launch sum dgamma's columns from a second read - no partial rows,
// no fold, no workspace, one launch (a call costs the host 9.1 instead of 13.1 us, which bounds it at these sizes).  A workgroup of 32 columns
// reads 50 KB per us, so long columns lose.  On the GPU, columns / fold, us: 4 x 4096 3.1 / 5.7, 128 x 8192 4.2 / 10.2, 512 x 4096 4.5 / 14.2,
// 1024 x 2048 6.1 / 10.6, 2048 x 1024 7.9 / 8.5 (bf16), 2048 x 768 (bf16, fp32 h) 10.8 / 8.7, 1237 x 1001 (fp16) 11.2 / 8.8
// (the last two lose 2 us where a graph replays them and the host does not count); not taken: 2048 x 2048
// 14.7 / 12.7, 4096 x 512 12.3 / 7.8, 2048 x 8192 39 / 28.
static bool rms_bwd_columns(int64_t rows, int W) { return rows <= 2048 && rows * W <= (1 << 21); }
size_t rmsnorm_bwd_ws_bytes(int64_t rows, int W) {
    return rms_bwd_columns(rows, W) ? 0 : (size_t)rms_bwd_blocks(rows, W) * ((W + 3) & ~3) * sizeof(float);
}

template <typename TD, typename TH>
static int rms_bwd_launch(const RmsBwdArgs& args, hipStream_t st) {
    RmsBwdArgs a = args;
    const bool columns = rms_bwd_columns(a.rows, a.W);
    a.row_blocks = rms_bwd_blocks(a.rows, a.W);
    const int nv = (a.W + 7) / 8, blocks = a.row_blocks + (columns ? (a.W + 31) / 32 : 0);
#define SPN_RMS_BWD(TPR_, NV_)                                                                                             \
    do {                                                                                                                   \
        if (a.W % 8) hipLaunchKernelGGL((rmsnorm_bwd_kernel<TD, TH, TPR_, NV_, true>), dim3(blocks), dim3(256), 0, st, a); \
        else hipLaunchKernelGGL((rmsnorm_bwd_kernel<TD, TH, TPR_, NV_, false>), dim3(blocks), dim3(256), 0, st, a);        \
    } while (0)
    if (nv <= 64) SPN_RMS_BWD(64, 1);
    else if (nv <= 128) SPN_RMS_BWD(64, 2);
    else if (nv <= 256) SPN_RMS_BWD(256, 1);
    else if (nv <= 512) SPN_RMS_BWD(256, 2);
    else if (nv <= 1024) SPN_RMS_BWD(256, 4);
    else SPN_RMS_BWD(256, 8);
#undef SPN_RMS_BWD
    SPN_CHECK_LAUNCH();
    if (columns) return SPN_OK;
    hipLaunchKernelGGL(rms_fold_kernel, dim3((a.W + 15) / 16), dim3(256), 0, st, a.ws, blocks, a.W, (a.W + 3) & ~3, a.dgamma);
    SPN_CHECK_LAUNCH();
    return SPN_OK;
}

int rmsnorm_bwd(const RmsBwdArgs& a, hipStream_t st) {
    if (a.rows <= 0 || a.W <= 0 || !a.dy || !a.h || !a.gamma || !a.rstd || !a.dx || !a.dgamma) return SPN_ERR_ARG;
    if (a.W > RMS_MAX_W || a.lddy < a.W || a.ldh < a.W || (a.dh && a.lddh < a.W)) return SPN_ERR_SHAPE;
    if (a.dyt < ET_F32 || a.dyt > ET_F16 || a.ht < ET_F32 || a.ht > ET_F16 || (a.dx2 && (a.dx2t < ET_F32 || a.dx2t > ET_F16))) return SPN_ERR_ARG;
    const size_t need = rmsnorm_bwd_ws_bytes(a.rows, a.W);
    if (need && (!a.ws || a.ws_bytes < need || (uintptr_t)a.ws % 16)) return SPN_ERR_WORKSPACE;
    if (a.dyt == ET_F32) {
        if (a.ht == ET_F32) return rms_bwd_launch<float, float>(a, st);
        if (a.ht == ET_BF16) return rms_bwd_launch<float, bf16_t>(a, st);
        return rms_bwd_launch<float, f16_t>(a, st);
    }
    if (a.dyt == ET_BF16) {
        if (a.ht == ET_F32) return rms_bwd_launch<bf16_t, float>(a, st);
        if (a.ht == ET_BF16) return rms_bwd_launch<bf16_t, bf16_t>(a, st);
        return rms_bwd_launch<bf16_t, f16_t>(a, st);
    }
    if (a.ht == ET_F32) return rms_bwd_launch<f16_t, float>(a, st);
    if (a.ht == ET_BF16) return rms_bwd_launch<f16_t, bf16_t>(a, st);
    return rms_bwd_launch<f16_t, f16_t>(a, st);
}

}  // namespace spn
