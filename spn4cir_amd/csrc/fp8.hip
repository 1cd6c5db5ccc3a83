// Quantiser and decoder of the 8-bit block format (fp8.h).
//
// Rows form: blocks along each row (what a product that reduces over the columns reads).  Transposed form: the transposed matrix in blocks
// along ITS rows, i.e. along the columns of x (what dW = dY^T X reduces over).  Square form: one scale for 128 x 128 values, so the
// transposed matrix holds the same codes - a weight is quantised once and serves the forward product and dX.
// Bound by HBM.  When the transposed form is wanted a workgroup takes a 128 x 128 tile: every value is read once, stays in registers (a
// thread holds 8 rows x 8 columns), both scales come from it, the transposed codes turn through 16 KB of LDS so that both outputs leave
// in whole 128-byte lines; the column sums (a bias gradient) ride along.
// Measured: both forms of [8192, 8192] bf16 54 us, 5.0 TB/s; of [19712, 2304] with column sums 40 + 5.7 us (fold), 4.6 TB/s; square blocks of
// fp32 [8192, 4096] 42 us, 4.8 TB/s; rows alone, [16384, 4096] bf16 34.9 us, 5.8 TB/s; stored blocks of that size along their columns 29.5 us, 4.6 TB/s; decoding [16384, 4096] to bf16 34 us, 6.0 TB/s.  A copy reaches 5.0.
#include "fp8.h"
#include "kernels.h"

namespace spn {

struct E4m3In {};

// eight values of row r from column c on: fetched as bits, converted later
template <typename T>
struct QIn {
    Vec8<T> v;
    __device__ __forceinline__ void fetch(const QuantArgs& a, int64_t r, int64_t c, int count) { v = fetch8<true>((const T*)a.x + r * a.ldx + c, count); }
    __device__ __forceinline__ void fetch_whole(const QuantArgs& a, int64_t r, int64_t c) { v = fetch8_whole((const T*)a.x + r * a.ldx + c); }
    __device__ __forceinline__ void get(int, float (&x)[8]) const { to_f32(v, x); }
};
template <>
struct QIn<E4m3In> {
    u32x2 v;
    int s;
    __device__ __forceinline__ void fetch(const QuantArgs& a, int64_t r, int64_t c, int count) {
        v = u32x2{0, 0};
        s = 0;
        if (count > 0) {                                   // codes behind C are zeros up to the next multiple of 128
            v = *(const u32x2*)((const uint8_t*)a.x + r * a.ldx + c);
            s = a.x_scale[r * a.x_pitch + (c >> 7)];
        }
    }
    __device__ __forceinline__ void fetch_whole(const QuantArgs& a, int64_t r, int64_t c) { fetch(a, r, c, 8); }
    __device__ __forceinline__ void get(int count, float (&x)[8]) const {
        e4m3_unpack8(v, pow2_field(s), x);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e >= count) x[e] = 0.f;
    }
};

// 16 blocks per workgroup: 2^bits of a row (16 / 2^bits rows), so that no index is divided
static int block_bits(int blocks) { int b = 0; while (b < 4 && (1 << b) < blocks) ++b; return b; }
// a launch holds fewer than 2^32 threads along x: more rows take more launches
static constexpr int64_t ROW_BLOCKS = (1 << 24) - 1;
static unsigned row_blocks(int64_t rows, int bits) {
    const int64_t n = (rows + (16 >> bits) - 1) >> (4 - bits);
    return (unsigned)(n < ROW_BLOCKS ? n : ROW_BLOCKS);
}
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const QuantArgs a, int64_t row0, int bits) {
    const int nb = qblocks(a.C), sp = qscale_pitch(a.C), l = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int b = (int)(blockIdx.y << bits) + (g & ((1 << bits) - 1));
    const int64_t r = row0 + ((int64_t)blockIdx.x << (4 - bits)) + (g >> bits);
    if (r >= a.R || b >= sp) return;
    if (b >= nb) {                                         // the padding of the scale row
        if (l == 0) a.q_scale[r * sp + b] = 127;
        return;
    }
    const int64_t c = (int64_t)b * QBLK + l * 8, left = a.C - c;
    float x[8];
    const int cnt = left > 8 ? 8 : (int)left;
    QIn<T> in;
    in.fetch(a, r, c, cnt);
    in.get(cnt, x);
    const int sb = e4m3_block_byte(x);
    *(u32x2*)(a.q + r * ((int64_t)nb * QBLK) + c) = e4m3_pack8(x, pow2_field(254 - sb));
    if (l == 0) a.q_scale[r * sp + b] = (uint8_t)sb;
}

// op over the lanes l, l + 16, l + 32, l + 48, in every lane
template <typename F>
__device__ __forceinline__ float rows4(float v, F op) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// 128 x 128 tile per workgroup, column blocks fastest
template <typename T>
__global__ __launch_bounds__(256) void quantize_tile_kernel(const QuantArgs a, int tiles_c) {
    __shared__ __attribute__((aligned(16))) float cmax[4][QBLK], csum[4][QBLK];
    __shared__ __attribute__((aligned(16))) uint8_t tr[QBLK][QBLK + 8];
    const int tc = (int)(blockIdx.x % tiles_c);
    const int64_t tr_i = blockIdx.x / tiles_c;
    const int l = threadIdx.x & 15, rg = threadIdx.x >> 4, wave = threadIdx.x >> 6;
    const int64_t r0 = tr_i * QBLK + rg * 8, c0 = (int64_t)tc * QBLK + l * 8;
    const int64_t lc = a.C - c0;
    const int cc = lc >= 8 ? 8 : lc > 0 ? (int)lc : 0;
    float x[8][8];
    {
        // a whole tile's loads carry no guards: behind a guard the compiler waits for each load where the paths meet
        QIn<T> in[8];
        if ((tr_i + 1) * QBLK <= a.R && (int64_t)(tc + 1) * QBLK <= a.C) {
#pragma unroll
            for (int p = 0; p < 8; ++p) in[p].fetch_whole(a, r0 + p, c0);
#pragma unroll
            for (int p = 0; p < 8; ++p) in[p].get(8, x[p]);
        } else {
#pragma unroll
            for (int p = 0; p < 8; ++p) in[p].fetch(a, r0 + p < a.R ? r0 + p : 0, c0, r0 + p < a.R ? cc : 0);
#pragma unroll
            for (int p = 0; p < 8; ++p) in[p].get(cc, x[p]);
        }
    }

    // Largest magnitudes: rows over the 16 lanes of a row; columns over the thread's 8 rows, the wave's 4 row groups (lane swaps of rows of 16
    // and of halves: the swapped pair holds both partners' values in every lane), the 4 waves (LDS)
    float rmax[8], cm[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) rmax[p] = max8_abs(x[p]);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        cm[e] = max8_abs(x[0][e], x[1][e], x[2][e], x[3][e], x[4][e], x[5][e], x[6][e], x[7][e]);
    const float hot = max8_abs(rmax);
    if (not_finite(hot)) {                                 // infinities and NaN do not enter the scales
#pragma unroll
        for (int p = 0; p < 8; ++p) rmax[p] = max8_finite(x[p]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float y[8];
#pragma unroll
            for (int p = 0; p < 8; ++p) y[p] = x[p][e];
            cm[e] = max8_finite(y);
        }
    }
#pragma unroll
    for (int p = 0; p < 8; ++p) rmax[p] = row16_max(rmax[p]);
#pragma unroll
    for (int e = 0; e < 8; ++e) cm[e] = rows4(cm[e], [](float u, float v) { return fmaxf(u, v); });
    if ((threadIdx.x & 63) < 16) {
        *(f32x4*)&cmax[wave][l * 8] = f32x4{cm[0], cm[1], cm[2], cm[3]};
        *(f32x4*)&cmax[wave][l * 8 + 4] = f32x4{cm[4], cm[5], cm[6], cm[7]};
    }
    if (a.colsum) {                                        // block-uniform
        float cs[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float s = 0.f;
#pragma unroll
            for (int p = 0; p < 8; ++p) s += x[p][e];
            cs[e] = rows4(s, [](float u, float v) { return u + v; });
        }
        if ((threadIdx.x & 63) < 16) {
            *(f32x4*)&csum[wave][l * 8] = f32x4{cs[0], cs[1], cs[2], cs[3]};
            *(f32x4*)&csum[wave][l * 8 + 4] = f32x4{cs[4], cs[5], cs[6], cs[7]};
        }
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const f32x4 lo = *(const f32x4*)&cmax[w][l * 8], hi = *(const f32x4*)&cmax[w][l * 8 + 4];
#pragma unroll
        for (int e = 0; e < 4; ++e) { cm[e] = fmaxf(cm[e], lo[e]); cm[4 + e] = fmaxf(cm[4 + e], hi[e]); }
    }
    if (a.colsum && threadIdx.x < QBLK && (int64_t)tc * QBLK + threadIdx.x < a.C)
        a.ws[tr_i * a.C + (int64_t)tc * QBLK + threadIdx.x] =
            (csum[0][threadIdx.x] + csum[1][threadIdx.x]) + (csum[2][threadIdx.x] + csum[3][threadIdx.x]);
    if (a.square) {                                        // block-uniform: one maximum for the tile
        const float m = row16_max(max8_abs(cm));
#pragma unroll
        for (int e = 0; e < 8; ++e) { cm[e] = m; rmax[e] = m; }
    }
    const int nbc = qblocks(a.C), spc = qscale_pitch(a.C);
    if (a.q) {
        const int64_t Cp = (int64_t)nbc * QBLK;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            if (r0 + p >= a.R) continue;
            const int sb = e4m3_scale_byte(__float_as_uint(rmax[p]));
            *(u32x2*)(a.q + (r0 + p) * Cp + c0) = e4m3_pack8(x[p], pow2_field(254 - sb));
            if (l == 0) a.q_scale[(r0 + p) * spc + tc] = (uint8_t)sb;
            if (tc == nbc - 1 && nbc + l < spc) a.q_scale[(r0 + p) * spc + nbc + l] = 127;
        }
    }
    if (a.qt) {
        const int nbr = qblocks(a.R), spr = qscale_pitch(a.R);
        const int64_t Rp = (int64_t)nbr * QBLK;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int sb = e4m3_scale_byte(__float_as_uint(cm[e]));
            float y[8];
#pragma unroll
            for (int p = 0; p < 8; ++p) y[p] = x[p][e];
            *(u32x2*)(&tr[l * 8 + e][rg * 8]) = e4m3_pack8(y, pow2_field(254 - sb));
            if (rg == 0 && c0 + e < a.C) {
                a.qt_scale[(c0 + e) * spr + tr_i] = (uint8_t)sb;
                if (tr_i == nbr - 1)
                    for (int b = nbr; b < spr; ++b) a.qt_scale[(c0 + e) * spr + b] = 127;
            }
        }
        __syncthreads();
        // 128 rows of 128 bytes: 8 lanes of 16 bytes per row
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 32 + (threadIdx.x >> 3), b = (threadIdx.x & 7) * 16;
            const int64_t c = (int64_t)tc * QBLK + row;
            const u32x2 lo = *(const u32x2*)(&tr[row][b]), hi = *(const u32x2*)(&tr[row][b + 8]);
            if (c < a.C) *(u32x4*)(a.qt + c * Rp + tr_i * QBLK + b) = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
    }
}

// column sums of the tile rows' partials: 16 columns x 16 row lanes per workgroup, four loads in flight per lane
__global__ __launch_bounds__(256) void qcolsum_fold_kernel(const float* __restrict__ ws, int64_t n, int64_t C, float* __restrict__ out) {
    __shared__ float red[16][17];
    const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4;
    const int64_t c = (int64_t)blockIdx.x * 16 + cl;
    float s = 0.f;
    if (c < C) {
#pragma unroll 4
        for (int64_t r = rl; r < n; r += 16) s += ws[r * C + c];
    }
    red[rl][cl] = s;
    __syncthreads();
    if (rl == 0 && c < C) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += red[k][cl];
        out[c] = s;
    }
}

size_t quantize_fp8_ws_bytes(int64_t R, int64_t C) { return (size_t)qblocks(R) * C * sizeof(float); }

template <typename T>
static int quantize_launch(const QuantArgs& a, hipStream_t st) {
    if (!a.qt && !a.square && !a.colsum) {
        const int bits = block_bits(qscale_pitch(a.C));
        const unsigned gy = (unsigned)((qscale_pitch(a.C) + 15) >> 4);
        if (gy > 65535) return SPN_ERR_SHAPE;
        const int64_t step = ROW_BLOCKS << (4 - bits);
        for (int64_t r = 0; r < a.R; r += step) {
            hipLaunchKernelGGL(quantize_rows_kernel<T>, dim3(row_blocks(a.R - r, bits), gy), dim3(256), 0, st, a, r, bits);
            SPN_CHECK_LAUNCH();
        }
        return SPN_OK;
    }
    const int64_t tiles = (int64_t)qblocks(a.R) * qblocks(a.C);
    if (tiles >= (1ll << 24) || (a.colsum && (a.C + 15) / 16 >= (1ll << 24))) return SPN_ERR_SHAPE;        // 2^32 threads
    hipLaunchKernelGGL(quantize_tile_kernel<T>, dim3((unsigned)tiles), dim3(256), 0, st, a, qblocks(a.C));
    SPN_CHECK_LAUNCH();
    if (a.colsum) {
        hipLaunchKernelGGL(qcolsum_fold_kernel, dim3((unsigned)((a.C + 15) / 16)), dim3(256), 0, st, a.ws, (int64_t)qblocks(a.R), a.C, a.colsum);
        SPN_CHECK_LAUNCH();
    }
    return SPN_OK;
}

int quantize_fp8(const QuantArgs& a, hipStream_t st) {
    if (!a.x || a.R <= 0 || a.C <= 0 || (!a.q && !a.qt) || (a.q && !a.q_scale) || (a.qt && !a.qt_scale)) return SPN_ERR_ARG;
    if ((uintptr_t)a.q % 8 || (uintptr_t)a.qt % 16) return SPN_ERR_ARG;
    if (a.R >= (1ll << 31) || a.C >= (1ll << 31) || a.ldx < a.C) return SPN_ERR_SHAPE;
    if (a.colsum && (!a.ws || a.ws_bytes < quantize_fp8_ws_bytes(a.R, a.C))) return SPN_ERR_WORKSPACE;
    switch (a.type) {
        case ET_F32: return quantize_launch<float>(a, st);
        case ET_BF16: return quantize_launch<bf16_t>(a, st);
        case ET_F16: return quantize_launch<f16_t>(a, st);
        case ET_E4M3:
            if (!a.x_scale || a.ldx % 8 || (uintptr_t)a.x % 8) return SPN_ERR_ARG;
            if (a.x_pitch < qblocks(a.C)) return SPN_ERR_SHAPE;
            return quantize_launch<E4m3In>(a, st);
        default: return SPN_ERR_ARG;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale, int64_t R, int64_t C,
                                                         T* __restrict__ out, int64_t row0, int bits) {
    const int nb = qblocks(C), l = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int b = (int)(blockIdx.y << bits) + (g & ((1 << bits) - 1));
    const int64_t r = row0 + ((int64_t)blockIdx.x << (4 - bits)) + (g >> bits);
    if (r >= R || b >= nb) return;
    const int64_t c = (int64_t)b * QBLK + l * 8, left = C - c;
    float x[8];
    e4m3_unpack8(*(const u32x2*)(q + r * ((int64_t)nb * QBLK) + c), pow2_field(scale[r * qscale_pitch(C) + b]), x);
    store8(out + r * C + c, left >= 8 ? 8 : left > 0 ? (int)left : 0, x);
}

int dequantize_fp8(const uint8_t* q, const uint8_t* scale, int64_t R, int64_t C, void* out, int type, hipStream_t st) {
    if (!q || !scale || !out || R < 0 || C <= 0 || (uintptr_t)q % 8) return SPN_ERR_ARG;
    if (R == 0) return SPN_OK;
    const int bits = block_bits(qblocks(C));
    if (R >= (1ll << 31) || C >= (1ll << 31) || ((qblocks(C) + 15) >> 4) > 65535) return SPN_ERR_SHAPE;
    const int64_t step = ROW_BLOCKS << (4 - bits);
    for (int64_t r = 0; r < R; r += step) {
        const dim3 grid(row_blocks(R - r, bits), (unsigned)((qblocks(C) + 15) >> 4));
        if (type == ET_F32) hipLaunchKernelGGL(dequantize_kernel<float>, grid, dim3(256), 0, st, q, scale, R, C, (float*)out, r, bits);
        else if (type == ET_BF16) hipLaunchKernelGGL(dequantize_kernel<bf16_t>, grid, dim3(256), 0, st, q, scale, R, C, (bf16_t*)out, r, bits);
        else if (type == ET_F16) hipLaunchKernelGGL(dequantize_kernel<f16_t>, grid, dim3(256), 0, st, q, scale, R, C, (f16_t*)out, r, bits);
        else return SPN_ERR_ARG;
        SPN_CHECK_LAUNCH();
    }
    return SPN_OK;
}

}  // namespace spn
