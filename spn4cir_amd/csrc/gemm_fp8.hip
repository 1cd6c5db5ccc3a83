// C[M, N] = act(A[M, K] . B[N, K]^T + bias) on 8-bit blocks (fp8.h): codes e4m3, one power-of-two scale per row and 128 values of k.
//
//   C[m, n] = sum over blocks kb of 2^(sa[m, kb] + sb[n, kb] - 254) * sum over k in kb of A[m, k] B[n, k]
//
// v_mfma_scale_f32_32x32x64_f8f6f4 applies both scales inside the matrix pipe; fp32 accumulators.  Measured (single products beside a large one):
// the unit aligns the products of 8 consecutive k (the 8 bytes of a register pair) to the largest sum of exponents among them and drops
// what lies 13 bits below; groups are then added in fp32.  Against 64 bits that is 1.5e-5 of the result for normal data and 4.5e-5 with
// a hundredth of the channels 20 times as loud, at every K - three orders below what the codes themselves cost, so the full-rate
// instruction is used for fp32 outputs too (the half-rate fp8 instruction does the same; only products in bf16 would be exact).  K is padded to whole blocks with zero
// codes by whoever wrote the operands, so the k loop has no tail; rows behind M / N read as zeros through the buffer descriptors.
//
// Three kernels: 256 x 256 tiles (large products: matrix unit, at the power limit), smaller tiles with the k blocks dealt to groups of waves (bound by the
// 26-32 bytes per cycle that a CU takes from L2), and up to 32 rows straight from registers (bound by the weights' bytes in flight).
// Few tiles over a long k are split into slices of k, summed in their order by a second kernel.
#include "fp8.h"
#include "kernels.h"
#include <atomic>

namespace spn {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// Operand order (B, A): a lane then owns row m = lane & 31 of C and, for g = 0..3, the columns 8 g + 4 (lane >> 5) + 0..3 (registers 4g..4g+3).
__device__ __forceinline__ f32x16 mfma_fp8(i32x8 b, i32x8 a, f32x16 c, int sb, int sa) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, c, 0, 0, 0, sb, 0, sa);
}

// LDS image of a [rows][128] byte tile: 16-byte chunk c of row r at position c ^ ((r >> 1) & 7) - 16 consecutive rows then hit every bank once
__device__ __forceinline__ int swz(int r, int c) { return c ^ ((r >> 1) & 7); }

struct Fp8Tile {                  // kernel arguments
    const uint8_t *a, *b, *sa, *sb;
    int64_t M, N, Kp;
    int pitch, nk;                // scale pitch in bytes, k blocks
    int tiles, tiles_n, group, splits, k_per_split;      // grid: tiles * splits
    const float* bias;
    int act;
    void* out;
    int out_type, accumulate;
    int64_t ldc;
    float* part;                  // splits > 1: fp32 [splits][tiles][BM * BN / 1024][256 threads][4], the accumulators as they lie
};

// ---- epilogue: `cnt` of eight consecutive columns n .. n + 7 of row m, from fp32 sums
template <int CNT>
__device__ __forceinline__ void fp8_bias(const Fp8Tile& p, int64_t n, int cnt, float (&b)[CNT]) {
#pragma unroll
    for (int e = 0; e < CNT; ++e) b[e] = 0.f;
    if (!p.bias) return;
    struct __attribute__((packed, aligned(4))) Row { float v[CNT]; };
    if (cnt >= CNT) {
        const Row r = *(const Row*)(p.bias + n);
#pragma unroll
        for (int e = 0; e < CNT; ++e) b[e] = r.v[e];
    } else {
#pragma unroll
        for (int e = 0; e < CNT - 1; ++e)
            if (e < cnt) b[e] = p.bias[n + e];
    }
}
template <int CNT>
__device__ __forceinline__ void fp8_bias_act(const Fp8Tile& p, const float (&bias)[CNT], float (&v)[CNT]) {
#pragma unroll
    for (int e = 0; e < CNT; ++e) v[e] += bias[e];
    if (p.act == ACT_QUICKGELU) {
#pragma unroll
        for (int e = 0; e < CNT; ++e) v[e] = quick_gelu_f(v[e]);
    } else if (p.act == ACT_GELU_ERF) {
#pragma unroll
        for (int e = 0; e < CNT; ++e) v[e] = gelu_erf_f(v[e]);
    }
}
__device__ __forceinline__ void fp8_store_f32(const Fp8Tile& p, int64_t o, int cnt, float (&v)[8]) {
    if (p.accumulate) {
        float c[8];
        load8((const float*)p.out + o, cnt, c);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += c[e];
    }
    store8((float*)p.out + o, cnt, v);
}

// The accumulators of a BM x BN tile leave through LDS in fp32, CHUNK rows at a time, so that a wave writes whole rows: 16-byte unit u of
// row r sits at a slot that makes both the writers (16 rows, one unit) and the readers (one row, units 2 u and 2 u + 1) hit all banks.
template <int BN>
__device__ __forceinline__ int fp8_slot(int unit, int r) {
    return ((unit >> 1) | ((unit & 1) * (BN / 8))) ^ (r & (BN / 8 < 16 ? BN / 8 - 1 : 15));
}

template <int BM, int BN, int TM, int TN, int CHUNK, int THREADS, int MI, int NJ>
__device__ __forceinline__ void fp8_epilogue(const Fp8Tile& p, f32x16 (&acc)[MI][NJ], char* smem, int64_t m0, int64_t n0, int wr, int wc, bool writer) {
    constexpr int LPR = BN / 8;                                      // lanes per row of the read-back
    const int lane = threadIdx.x & 63;
    float* sC = (float*)smem;
    const int u = threadIdx.x % LPR;
    const int64_t n = n0 + u * 8, left = p.N - n;
    const int cnt = left >= 8 ? 8 : left > 0 ? (int)left : 0;
    float bias[8];                                                   // this thread's columns: the same for all its rows
    fp8_bias<8>(p, n, cnt, bias);
#pragma unroll
    for (int ch = 0; ch < BM / CHUNK; ++ch) {
        __syncthreads();                                             // the operand tiles, or the previous rows, have been read
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int rl = wr * TM + i * 32;
            if (rl / CHUNK != ch || !writer) continue;               // wave-uniform
            const int r = rl % CHUNK + (lane & 31);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int unit = (wc * TN + j * 32 + 8 * g) / 4 + (lane >> 5);
                    *(f32x4*)(sC + r * BN + fp8_slot<BN>(unit, r) * 4) =
                        f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                }
        }
        __syncthreads();
#pragma unroll 4
        for (int r = threadIdx.x / LPR; r < CHUNK; r += THREADS / LPR) {
            const int64_t m = m0 + ch * CHUNK + r;
            if (m >= p.M) break;
            const f32x4 lo = *(const f32x4*)(sC + r * BN + fp8_slot<BN>(2 * u, r) * 4), hi = *(const f32x4*)(sC + r * BN + fp8_slot<BN>(2 * u + 1, r) * 4);
            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            fp8_bias_act<8>(p, bias, v);
            fp8_store_f32(p, m * p.ldc + n, cnt, v);
        }
    }
}

// The same for 16-bit outputs: bias and activation on the registers, then the tile goes through LDS as it will be stored - half the LDS bytes
// and one pass of two barriers.  16-byte unit u of row r sits at u ^ (r mod units).  Type and activation are compile-time and the bias
// comes from LDS (`bias`: this thread's column's value, loaded before the k loop): with the branches in every group of columns the code was larger than
// the instruction cache (256 x 256 tile: 40 000 cycles instead of 9 900).
template <typename T, int ACT, int BM, int BN, int TM, int TN, int THREADS, int MI, int NJ>
__device__ __forceinline__ void fp8_epilogue16(const Fp8Tile& p, f32x16 (&acc)[MI][NJ], char* smem, float bias, int64_t m0, int64_t n0, int wr, int wc, bool writer) {
    constexpr int UNITS = BN / 8;
    const int lane = threadIdx.x & 63;
    float* const sBias = (float*)(smem + BM * BN * 2);
    __syncthreads();                                                 // the operand tiles have been read
    if (threadIdx.x < BN) sBias[threadIdx.x] = bias;
    __syncthreads();
    if (writer) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            f32x4 bj[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) bj[g] = *(const f32x4*)(sBias + wc * TN + j * 32 + 8 * g + 4 * (lane >> 5));
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = wc * TN + j * 32 + 8 * g;              // this lane's columns: c + 4 (lane >> 5) + 0..3
                const f32x4 b = bj[g];
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    const int r = wr * TM + i * 32 + (lane & 31);
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = acc[i][j][4 * g + e] + b[e];
                        if constexpr (ACT == ACT_QUICKGELU) x[e] = quick_gelu_f(x[e]);
                        if constexpr (ACT == ACT_GELU_ERF) x[e] = gelu_erf_f(x[e]);
                    }
                    *(u32x2*)(smem + (r * UNITS + ((c / 8) ^ (r & (UNITS < 32 ? UNITS - 1 : 31)))) * 16 + (lane >> 5) * 8) =
                        u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
                }
            }
            __builtin_amdgcn_sched_barrier(0);                       // one column tile at a time: hoisted together they spill
        }
    }
    __syncthreads();
    const int u = threadIdx.x % UNITS, r0 = threadIdx.x / UNITS;
    const int64_t n = n0 + u * 8, left = p.N - n;
    const int rows = p.M - m0 < BM ? (int)(p.M - m0) : BM;
    T* o = (T*)p.out + m0 * p.ldc + n;
    auto at = [&](int r) { return *(const u32x4*)(smem + (r * UNITS + (u ^ (r & (UNITS < 32 ? UNITS - 1 : 31)))) * 16); };
    if (left >= 8) {
        T* w = o + r0 * p.ldc;
#pragma unroll 4
        for (int r = r0; r < rows; r += THREADS / UNITS, w += THREADS / UNITS * p.ldc) *(Vec8<T>*)w = __builtin_bit_cast(Vec8<T>, at(r));
    } else if (left > 0) {
#pragma unroll 1
        for (int r = r0; r < rows; r += THREADS / UNITS) {
            const u32x4 v = at(r);
#pragma unroll
            for (int e = 0; e < 7; ++e)
                if (e < left) o[r * p.ldc + e] = __builtin_bit_cast(T, (uint16_t)(v[e >> 1] >> (16 * (e & 1))));
        }
    }
}

// What leaves a tile kernel: 16 bits with a compile-time activation, fp32 (with any activation), or the partial sums of a k slice
template <typename T, int ACT_>
struct Fp8Out { using type = T; static constexpr int ACT = ACT_; };
using Fp8Wide = Fp8Out<float, ACT_NONE>;
using Fp8Part = Fp8Out<void, ACT_NONE>;
// the bias of this thread's column of the tile, loaded before the k loop (16-bit outputs)
template <typename OUT, int BN>
__device__ __forceinline__ float fp8_bias_of(const Fp8Tile& p, int64_t n0) {
    if constexpr (__is_same(typename OUT::type, float) || __is_same(typename OUT::type, void)) return 0.f;
    else return p.bias && threadIdx.x < BN && n0 + threadIdx.x < p.N ? p.bias[n0 + threadIdx.x] : 0.f;
}

// 16-byte chunks of an operand row that lane holds for half h of a k block: 32 consecutive bytes
__device__ __forceinline__ i32x8 fp8_frag(const char* tile, int r, int h, int lane) {
    const int c = h * 4 + (lane >> 5) * 2;
    const u32x4 lo = *(const u32x4*)(tile + r * 128 + swz(r, c) * 16), hi = *(const u32x4*)(tile + r * 128 + swz(r, c + 1) * 16);
    return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// Partial sums: 16 bytes per thread and instruction straight from the accumulators, whole lines and no LDS - the join reads them the same way
template <int BM, int BN, int MI, int NJ>
__device__ __forceinline__ void fp8_partial(const Fp8Tile& p, f32x16 (&acc)[MI][NJ], int slice, int64_t m0, int64_t n0, bool writer) {
    if (!writer) return;
    const int64_t tile = (m0 / BM) * p.tiles_n + n0 / BN;
    f32x4* o = (f32x4*)p.part + ((int64_t)slice * p.tiles + tile) * (BM * BN / 4) + (threadIdx.x & 255);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                o[((i * NJ + j) * 4 + g) * 256] = f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
}

template <typename OUT, int BM, int BN, int TM, int TN, int CHUNK, int THREADS, int MI, int NJ>
__device__ __forceinline__ void fp8_finish_tile(const Fp8Tile& p, f32x16 (&acc)[MI][NJ], char* smem, float bias, int slice, int64_t m0, int64_t n0, int wr, int wc,
                                                bool writer) {
    if constexpr (__is_same(typename OUT::type, void)) fp8_partial<BM, BN>(p, acc, slice, m0, n0, writer);
    else if constexpr (__is_same(typename OUT::type, float)) fp8_epilogue<BM, BN, TM, TN, CHUNK, THREADS>(p, acc, smem, m0, n0, wr, wc, writer);
    else fp8_epilogue16<typename OUT::type, OUT::ACT, BM, BN, TM, TN, THREADS>(p, acc, smem, bias, m0, n0, wr, wc, writer);
}

// workgroup -> k slice and (m0, n0).  An XCD works on consecutive logical ids: first the tiles of one slice, which share its operands in that XCD's L2
// (2304 x 768 x 19712 in 8 slices, tiles dealt to XCDs regardless of their slice: 50.7 us, so: 50.2), and in groups of `group` column tiles, so that the
// B rows of a group stay there
__device__ __forceinline__ int fp8_tile_of(const Fp8Tile& p, int bm, int bn, int64_t& m0, int64_t& n0) {
    int bid = xcd_remap(blockIdx.x, gridDim.x);
    const int slice = p.splits > 1 ? bid / p.tiles : 0, tiles_m = p.tiles / p.tiles_n;
    bid -= slice * p.tiles;
    int c0 = 0, wg = p.group < p.tiles_n ? p.group : p.tiles_n;
    while (bid >= tiles_m * wg) {
        bid -= tiles_m * wg;
        c0 += wg;
        wg = p.group < p.tiles_n - c0 ? p.group : p.tiles_n - c0;
    }
    m0 = (int64_t)(bid / wg) * bm;
    n0 = (int64_t)(c0 + bid % wg) * bn;
    return slice;
}

// Large products: 256 x 256 tile, 4 waves (2 x 2), wave tile 128 x 128: one workgroup per CU, one wave per SIMD.  Such a wave tile reads the least
// LDS per product (64 KB of DMA in, 128 KB out per k block of 2048 matrix cycles).
// Phase 2 kt multiplies the upper two row tiles of A with all of B of k block kt, phase 2 kt + 1 the lower two: 16 MFMA each, from registers,
// the first half of the k block before the second; between them the wave reads what comes next from LDS, where two k blocks of the chunks Y0 / Y1
// (A rows of the even / odd phase, 16 KB) and B (32 KB) lie, whole 128-byte rows:
//   phase 2 kt reads B(kt) second half, Y1(kt);  phase 2 kt + 1 reads Y0(kt + 1) and, behind its barrier, B(kt + 1) first half
// One barrier per phase, four MFMA before its end (they run while the waves meet).  Behind the even one B(kt) and Y1(kt) are in registers
// everywhere and their places take the DMA of k block kt + 2, behind the odd one Y0(kt + 1) is and Y0(kt + 3) follows: everything is needed three
// barriers later, 16 DMA stay in flight behind each counted wait.
// Measured cycles per k block (2048 of them matrix): 2 256; with stages of 64-byte half rows, where every 128-byte line is asked for twice,
// 2 400-2 620; with 8 waves of 128 x 64 (192 KB out of LDS per k block) taking turns on the SIMDs, 2 720.  The epilogue takes 9 900 when one round of
// tiles is all there is and up to 22 000 between rounds: all CUs store 33 MB at once, at the 4.6 TB/s a fill of that size reaches.
// Bound by the power limit: 8192 x 8192 x 4096 in 217-222 us, 2.5 PFLOP/s, at 1.8 GHz (zeros as data: 20 % faster; in the first milliseconds of a load, while
// the power management settles, up to 284).  fp32 outputs 248, with accumulate 310: twice the bytes stored, then as many read, behind the k loop.
// Chunks behind the last k block are issued with an empty descriptor (zeros, no fetch), so the counts hold to the end.
// Scales: two 4-byte DMA per lane and four k blocks bring the scale dwords of all 512 rows into one of two 2 KB buffers, four k blocks ahead; the
// counted waits do not know of them, which makes the few that see them stricter, never laxer.
template <typename OUT>
__global__ __launch_bounds__(256, 1) void gemm_fp8_256_kernel(const Fp8Tile p) {
    constexpr int CH = 128 * 128;                           // bytes of a chunk; LDS: Y0 Y0' Y1 Y1' B0 B0' B1 B1' scales
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char* const sS = smem + 8 * CH;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = wid >> 1, wc = wid & 1;
    int64_t m0, n0;
    const int slice = fp8_tile_of(p, 256, 256, m0, n0);
    const float bias = fp8_bias_of<OUT, 256>(p, n0);
    const int k_begin = slice * p.k_per_split;
    const int nk = (k_begin + p.k_per_split < p.nk ? k_begin + p.k_per_split : p.nk) - k_begin;
    const int64_t ma = p.M - m0 < 256 ? p.M - m0 : 256, nb = p.N - n0 < 256 ? p.N - n0 : 256;
    const uint32_t ld = (uint32_t)p.Kp, kofs = (uint32_t)k_begin * 128u, bytesA = (uint32_t)ma * ld, bytesB = (uint32_t)nb * ld;
    const uint8_t *baseA = p.a + m0 * p.Kp, *baseB = p.b + n0 * p.Kp;
    const __amdgpu_buffer_rsrc_t rsSA = make_rsrc(p.sa + m0 * p.pitch, (uint32_t)ma * (uint32_t)p.pitch);
    const __amdgpu_buffer_rsrc_t rsSB = make_rsrc(p.sb + n0 * p.pitch, (uint32_t)nb * (uint32_t)p.pitch);
    const uint32_t soff = (uint32_t)(wid * 64 + lane) * (uint32_t)p.pitch + (uint32_t)k_begin;          // k_begin % 4 == 0
    // chunk row c = wid * 32 + t * 8 + (lane >> 3) is tile row (c >> 6) * 128 + half * 64 + (c & 63); 16-byte unit u of it lies at swz(c, u)
    uint32_t vo[2][4];
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int t = 0; t < 4; ++t)
            vo[f][t] = (uint32_t)((wid >> 1) * 128 + f * 64 + (wid & 1) * 32 + t * 8 + (lane >> 3)) * ld + (uint32_t)swz(t * 8 + (lane >> 3), lane & 7) * 16u;
    auto dma = [&](bool isB, int half, int t, int kt, int par) {       // par = kt & 1
        const bool on = kt < nk;
        char* d = smem + (isB ? 4 : 0) * CH + (half * 2 + par) * CH + (wid * 32 + t * 8) * 128;
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(isB ? baseB : baseA, on ? (isB ? bytesB : bytesA) : 0u);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LDS_PTR(d), 16, vo[half][t], on ? kofs + (uint32_t)kt * 128u : 0u, 0, 0);
    };
    auto scales = [&](int g) {
        char* d = sS + (g & 1) * 2048 + wid * 256;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsSA, LDS_PTR(d), 4, soff + (uint32_t)g * 4u, 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsSB, LDS_PTR(d + 1024), 4, soff + (uint32_t)g * 4u, 0, 0, 0);
    };
    f32x16 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    const int arow = wr * 128 + (lane & 31), brow = wc * 128 + (lane & 31);
    uint32_t fa[2][2], fb[2][2];                            // [half of the k block][16-byte unit]: first tile of a chunk, of the k block's parity
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int u = swz(lane & 31, h * 4 + (lane >> 5) * 2 + q) * 16;
            fa[h][q] = (uint32_t)((wr * 64 + (lane & 31)) * 128 + u);
            fb[h][q] = (uint32_t)(4 * CH + (wc * 64 + (lane & 31)) * 128 + u);
        }
    u32x4 A[2][2][2][2], B[4][2][2];                        // A: [phase][tile][h][unit], B: [tile][h][unit]
    auto read_a = [&](int half, int n) {           // n 0..7
        const int i = n >> 2, h = (n >> 1) & 1, q = n & 1;
        A[half][i][h][q] = *(const u32x4*)(smem + fa[h][q] + half * 2 * CH + i * 4096);
    };
    auto read_b = [&](int h, int j) {
#pragma unroll
        for (int q = 0; q < 2; ++q) B[j][h][q] = *(const u32x4*)(smem + fb[h][q] + (j >> 1) * 2 * CH + (j & 1) * 4096);
    };
    auto join = [](const u32x4 (&t)[2]) {
        return i32x8{(int)t[0][0], (int)t[0][1], (int)t[0][2], (int)t[0][3], (int)t[1][0], (int)t[1][1], (int)t[1][2], (int)t[1][3]};
    };
    int sa[4], sb[4], na[4], nb_[4];
    // DMA d of a k block: B, then Y1
    auto dma_by1 = [&](int d, int kt, int par) {
        if (d < 8) dma(true, d >> 2, d & 3, kt, par);
        else dma(false, 1, d & 3, kt, par);
    };
    auto dma_y0 = [&](int d, int kt, int par) { dma(false, 0, d, kt, par); };
    scales(0);
#pragma unroll
    for (int d = 0; d < 8; ++d) dma_by1(d, 0, 0);
#pragma unroll
    for (int d = 0; d < 4; ++d) dma_y0(d, 0, 0);
#pragma unroll
    for (int d = 8; d < 12; ++d) dma_by1(d, 0, 0);
#pragma unroll
    for (int d = 0; d < 4; ++d) dma_y0(d, 1, 1);
#pragma unroll
    for (int d = 0; d < 12; ++d) dma_by1(d, 1, 1);
    wait_vmcnt<16>();
    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int n = 0; n < 8; ++n) read_a(0, n);
#pragma unroll
    for (int j = 0; j < 4; ++j) read_b(0, j);
#pragma unroll
    for (int i = 0; i < 4; ++i) { sa[i] = *(const int*)(sS + (arow + i * 32) * 4); sb[i] = *(const int*)(sS + 1024 + (brow + i * 32) * 4); }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    dma_y0(0, 2, 0);
    dma_y0(1, 2, 0);
    // phase H of k block kt
#define SPN_FP8_PHASE(H)                                                                                                                              \
    _Pragma("unroll") for (int x = 0; x < 16; ++x) {                                                                                                  \
        const int h = x >> 3, i = x & 1, j = (x >> 1) & 3;                                                                                            \
        acc[2 * H + i][j] = mfma_fp8(join(B[j][h]), join(A[H][i][h]), acc[2 * H + i][j], sb[j], sa[2 * H + i]);                                       \
        asm volatile("" : "+a"(acc[2 * H + i][j]) :: "memory");                                                                                       \
        __builtin_amdgcn_sched_barrier(0);                                                                                                            \
        if (H == 0) {                                                                                                                                 \
            if (x < 4) read_b(1, x);                                                                                                                 \
            if (x >= 4 && x < 8) { read_a(1, 2 * (x - 4)); read_a(1, 2 * (x - 4) + 1); }                                                              \
        } else {                                                                                                                                      \
            if (x < 8) read_a(0, x);                                                                                                                  \
            if (x >= 12) read_b(0, x - 12);                                                                                                           \
            if (x == 8 || x == 9) {                                                                                                                   \
                _Pragma("unroll") for (int e = 0; e < 4; ++e) {                                                                                       \
                    if (x == 8) na[e] = *(const int*)(s + (arow + e * 32) * 4);                                                                       \
                    else nb_[e] = *(const int*)(s + 1024 + (brow + e * 32) * 4);                                                                      \
                }                                                                                                                                     \
            }                                                                                                                                         \
        }                                                                                                                                             \
        if (x == 11) asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)\n\ts_barrier" ::: "memory");                                                        \
        if (H == 0) {                                                                                                                                 \
            if (x == 8 || x == 10) dma_y0(x == 8 ? 2 : 3, kt + 2, kt & 1);                                                                            \
            if (x >= 12 && x < 15) dma_by1(x - 12, kt + 2, kt & 1);                                                                                             \
        } else {                                                                                                                                      \
            if (x < 11 && (x & 3) != 3) dma_by1(3 + x - (x >> 2), kt + 2, kt & 1);                                                                    \
            if (x == 13 || x == 15) dma_y0(x == 13 ? 0 : 1, kt + 3, ~kt & 1);                                                                         \
        }                                                                                                                                             \
        asm volatile("" ::: "memory");                                                                                                                \
        __builtin_amdgcn_sched_barrier(0);                                                                                                            \
    }
#pragma unroll 1
    for (int kt = 0; kt < nk; ++kt) {
        const char* s = sS + (((kt + 1) >> 2) & 1) * 2048;          // the next k block's scales
        SPN_FP8_PHASE(0)
        if ((kt & 3) == 0) scales((kt >> 2) + 1);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < 2; ++q) { fa[h][q] ^= CH; fb[h][q] ^= CH; }     // the other k block of each chunk
        SPN_FP8_PHASE(1)
        const int sh = ((kt + 1) & 3) * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) { sa[i] = na[i] >> sh; sb[i] = nb_[i] >> sh; }
    }
#undef SPN_FP8_PHASE
    wait_vmcnt<0>();                                        // the empty chunks too: the epilogue uses their place
    fp8_finish_tile<OUT, 256, 256, 128, 128, 128, 256>(p, acc, smem, bias, slice, m0, n0, wr, wc, true);
}

// Smaller products: BM x BN tile by KG groups of 2 x 2 waves that take every KG-th k block, S LDS buffers per group.  Stage i + S - 1 is issued
// behind the barrier that ends the reading of stage i - 1, so S - 2 whole stages stay in flight behind each wait.  The groups' sums meet in LDS in
// group order.
template <typename OUT, int BM, int BN, int KG, int S>
__global__ __launch_bounds__(256 * KG, 2) void gemm_fp8_tile_kernel(const Fp8Tile p) {
    constexpr int MI = BM / 64, NJ = BN / 64, ROWS = BM + BN, DMA = ROWS / 32 + 1;           // DMA instructions per wave and stage
    constexpr int SC = ROWS * 128, STAGE = SC + 1024;
    constexpr int SROWS = ROWS <= 128 ? 32 : 64;                                             // rows whose scales one wave brings (256 bytes each)
    static_assert(ROWS <= 256 && BM % SROWS == 0 && BN % SROWS == 0, "a wave brings the scales of one operand");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave >> 2, wid = wave & 3, wr = wid >> 1, wc = wid & 1;
    int64_t m0, n0;
    const int slice = fp8_tile_of(p, BM, BN, m0, n0);
    const float bias = fp8_bias_of<OUT, BN>(p, n0);
    const int k_begin = slice * p.k_per_split;
    const int nk = (k_begin + p.k_per_split < p.nk ? k_begin + p.k_per_split : p.nk) - k_begin;
    const int steps = (nk + KG - 1) / KG, mine = nk > kg ? (nk - kg + KG - 1) / KG : 0;       // this group's k blocks: k_begin + kg + KG i
    const int64_t ma = p.M - m0 < BM ? p.M - m0 : BM, nb = p.N - n0 < BN ? p.N - n0 : BN;
    const uint32_t ld = (uint32_t)p.Kp, pitch = (uint32_t)p.pitch;
    const __amdgpu_buffer_rsrc_t rsA = make_rsrc(p.a + m0 * p.Kp, (uint32_t)ma * ld), rsB = make_rsrc(p.b + n0 * p.Kp, (uint32_t)nb * ld);
    const int s0 = wid * SROWS < ROWS ? wid * SROWS : ROWS - SROWS;                          // a wave too many brings the last rows again, to a place of its own
    const int srow = s0 + lane % SROWS;
    const bool sA = s0 < BM;
    const __amdgpu_buffer_rsrc_t rsS = sA ? make_rsrc(p.sa + m0 * p.pitch, (uint32_t)ma * pitch) : make_rsrc(p.sb + n0 * p.pitch, (uint32_t)nb * pitch);
    const uint32_t soff = (uint32_t)(sA ? srow : srow - BM) * pitch;
    char* const ring = smem + kg * S * STAGE;
    auto stage = [&](int i) {
        char* s = ring + (i % S) * STAGE;
        const int kb = k_begin + kg + KG * i;
#pragma unroll
        for (int t = 0; t < ROWS / 32; ++t) {
            const int R0 = (t * 4 + wid) * 8, r = R0 + (lane >> 3), c = swz(r, lane & 7);     // 8 rows of 128 bytes per instruction
            const bool isA = t * 32 < BM;
            glds16(isA ? rsA : rsB, s + R0 * 128, (uint32_t)(isA ? r : r - BM) * ld + (uint32_t)(kb * 128 + c * 16));
        }
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsS, LDS_PTR(s + SC + wid * 256), 4, soff + (uint32_t)(kb & ~3), 0, 0, 0);
    };
    f32x16 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
        if (i < mine) stage(i);
    const int arow = wr * (BM / 2) + (lane & 31), brow = BM + wc * (BN / 2) + (lane & 31);
    auto scale_at = [&](const char* s, int row, int sh) { return *(const int*)(s + SC + row / SROWS * 256 + row % SROWS * 4) >> sh; };
    for (int i = 0; i < steps; ++i) {
        if (mine - 1 - i >= S - 2) wait_vmcnt<(S - 2) * DMA>();
        else wait_vmcnt<0>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (i + S - 1 < mine) stage(i + S - 1);
        if (i < mine) {
            const char* s = ring + (i % S) * STAGE;
            const int sh = ((k_begin + kg + KG * i) & 3) * 8;
            int sa[MI], sb[NJ];
#pragma unroll
            for (int q = 0; q < MI; ++q) sa[q] = scale_at(s, arow + q * 32, sh);
#pragma unroll
            for (int q = 0; q < NJ; ++q) sb[q] = scale_at(s, brow + q * 32, sh);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                i32x8 fa[MI], fb[NJ];
#pragma unroll
                for (int q = 0; q < MI; ++q) fa[q] = fp8_frag(s, arow + q * 32, h, lane);
#pragma unroll
                for (int q = 0; q < NJ; ++q) fb[q] = fp8_frag(s, brow + q * 32, h, lane);
#pragma unroll
                for (int q = 0; q < MI; ++q)
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[q][j] = mfma_fp8(fb[j], fa[q], acc[q][j], sb[j], sa[q]);
            }
        }
    }
    if constexpr (KG > 1) {
        f32x4* red = (f32x4*)smem;
        __syncthreads();
        if (kg > 0) {
#pragma unroll
            for (int q = 0; q < MI * NJ; ++q)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    red[((kg - 1) * MI * NJ * 4 + q * 4 + g) * 256 + (threadIdx.x & 255)] =
                        f32x4{acc[q / NJ][q % NJ][4 * g], acc[q / NJ][q % NJ][4 * g + 1], acc[q / NJ][q % NJ][4 * g + 2], acc[q / NJ][q % NJ][4 * g + 3]};
        }
        __syncthreads();
        if (kg == 0) {
#pragma unroll
            for (int k = 0; k < KG - 1; ++k)
#pragma unroll
                for (int q = 0; q < MI * NJ; ++q)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 v = red[(k * MI * NJ * 4 + q * 4 + g) * 256 + threadIdx.x];
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[q / NJ][q % NJ][4 * g + e] += v[e];
                    }
        }
    }
    fp8_finish_tile<OUT, BM, BN, BM / 2, BN / 2, BM, 256 * KG>(p, acc, smem, bias, slice, m0, n0, wr, wc, kg == 0);
}
template <int BM, int BN, int KG, int S>
constexpr int fp8_tile_lds() {
    constexpr int ring = KG * S * ((BM + BN) * 128 + 1024), red = KG > 1 ? (KG - 1) * BM * BN * 4 : 0, out = BM * BN * 4;
    return ring > red ? (ring > out ? ring : out) : (red > out ? red : out);
}

// Few rows: no shared staging.  A workgroup owns 16 columns and all rows, its waves take groups of four k blocks in turn and load their
// operand fragments straight into registers (each operand byte is used by one wave only, so LDS would not save a load); the waves' sums meet in
// LDS in wave order, once, at the end.  Bound by bytes in flight: the weights stream once.

// 16 MT rows (MT 1, 2) x 16 columns, v_mfma_scale_f32_16x16x128_f8f6f4: lane -> row lane & 15, 32 bytes at (lane >> 4) * 32 of a k block; C: row m = lane & 15,
// columns 4 (lane >> 4) + 0..3
template <int MT>
__global__ __launch_bounds__(1024) void gemm_fp8_rows_kernel(const Fp8Tile p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const uint32_t ld = (uint32_t)p.Kp, pitch = (uint32_t)p.pitch;
    const int64_t nb = p.N - n0 < 16 ? p.N - n0 : 16;
    const __amdgpu_buffer_rsrc_t rsA = make_rsrc(p.a, (uint32_t)p.M * ld), rsB = make_rsrc(p.b + n0 * p.Kp, (uint32_t)nb * ld);
    const __amdgpu_buffer_rsrc_t rsSA = make_rsrc(p.sa, (uint32_t)p.M * pitch), rsSB = make_rsrc(p.sb + n0 * p.pitch, (uint32_t)nb * pitch);
    const int r = lane & 15;
    const uint32_t off = (uint32_t)r * ld + (uint32_t)(lane >> 4) * 32u;
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto load = [&](const __amdgpu_buffer_rsrc_t& rs, uint32_t o) {
        const u32x4 lo = __builtin_amdgcn_raw_buffer_load_b128(rs, o, 0, 0), hi = __builtin_amdgcn_raw_buffer_load_b128(rs, o + 16u, 0, 0);
        return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    };
    const int groups = (p.nk + 3) >> 2;
    for (int g = wid; g < groups; g += waves) {
        int sa[MT];
        int sb = __builtin_amdgcn_raw_buffer_load_b32(rsSB, (uint32_t)r * pitch + (uint32_t)g * 4u, 0, 0);
#pragma unroll
        for (int i = 0; i < MT; ++i) sa[i] = __builtin_amdgcn_raw_buffer_load_b32(rsSA, (uint32_t)(r + i * 16) * pitch + (uint32_t)g * 4u, 0, 0);
        i32x8 b[4], a[MT][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (g * 4 + q >= p.nk) continue;                          // wave-uniform
            b[q] = load(rsB, off + (uint32_t)(g * 4 + q) * 128u);
#pragma unroll
            for (int i = 0; i < MT; ++i) a[i][q] = load(rsA, off + (uint32_t)(i * 16) * ld + (uint32_t)(g * 4 + q) * 128u);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (g * 4 + q >= p.nk) continue;
#pragma unroll
            for (int i = 0; i < MT; ++i)
                acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[q], a[i][q], acc[i], 0, 0, 0, sb >> (8 * q), 0, sa[i] >> (8 * q));
        }
    }
    f32x4* red = (f32x4*)smem;
#pragma unroll
    for (int i = 0; i < MT; ++i) red[(wid * MT + i) * 64 + lane] = acc[i];
    __syncthreads();
    for (int t = threadIdx.x; t < MT * 64; t += blockDim.x) {
        f32x4 s = red[t];
        for (int w = 1; w < waves; ++w) s += red[w * MT * 64 + t];
        const int64_t m = (t >> 6) * 16 + (t & 15), n = n0 + ((t & 63) >> 4) * 4;
        if (m >= p.M || n >= p.N) continue;
        const int cnt = p.N - n >= 4 ? 4 : (int)(p.N - n);
        float bias[4], v[4] = {s[0], s[1], s[2], s[3]};
        fp8_bias<4>(p, n, cnt, bias);
        fp8_bias_act<4>(p, bias, v);
        const int64_t o = m * p.ldc + n;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (e >= cnt) continue;
            if (p.out_type == ET_BF16) ((bf16_t*)p.out)[o + e] = f2bf(v[e]);
            else if (p.out_type == ET_F16) ((f16_t*)p.out)[o + e] = (f16_t)v[e];
            else ((float*)p.out)[o + e] = v[e] + (p.accumulate ? ((float*)p.out)[o + e] : 0.f);
        }
    }
}

// Sum of the k slices in their order, then bias, activation and the output's type.  One workgroup per 32 x 32 accumulator tile position of a tile (blockIdx.y):
// a thread reads the 4 x 4 values it had as a thread of the product, from every slice; then the two halves of the wave exchange every second group of
// four columns, so that a lane writes eight consecutive ones.
__global__ __launch_bounds__(256) void gemm_fp8_join_kernel(const Fp8Tile p, int bm, int bn) {
    const int nj = bn / 64, i = blockIdx.y / nj, j = blockIdx.y % nj, lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int64_t quads = (int64_t)bm * bn / 4, slice = (int64_t)gridDim.x * quads;
    const f32x4* o = (const f32x4*)p.part + (int64_t)blockIdx.x * quads + (int64_t)blockIdx.y * 1024 + threadIdx.x;
    f32x4 v[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) v[g] = o[g * 256];
#pragma unroll 4
    for (int s = 1; s < p.splits; ++s)
#pragma unroll
        for (int g = 0; g < 4; ++g) v[g] += o[s * slice + g * 256];
    const int64_t m = (int64_t)(blockIdx.x / p.tiles_n) * bm + (wid >> 1) * (bm / 2) + i * 32 + (lane & 31);
    const int64_t n0 = (int64_t)(blockIdx.x % p.tiles_n) * bn + (wid & 1) * (bn / 2) + j * 32;
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[g][e]), __float_as_uint(v[g + 1][e]), false, false);
            x[e] = __uint_as_float(t[0]);
            x[4 + e] = __uint_as_float(t[1]);
        }
        const int64_t n = n0 + 8 * (g + (lane >> 5)), left = p.N - n;
        if (m >= p.M || left <= 0) continue;
        const int cnt = left >= 8 ? 8 : (int)left;
        float bias[8];
        fp8_bias<8>(p, n, cnt, bias);
        fp8_bias_act<8>(p, bias, x);
        if (p.out_type == ET_BF16) store8((bf16_t*)p.out + m * p.ldc + n, cnt, x);
        else if (p.out_type == ET_F16) store8((f16_t*)p.out + m * p.ldc + n, cnt, x);
        else fp8_store_f32(p, m * p.ldc + n, cnt, x);
    }
}

// Which kernel, and over how many k slices: the least estimated time  rounds * (fixed + step * k blocks)  [+ the join of the slices].  fixed and
// step are fitted to the measured times (us, M x N x K, no slices; * = what the rule takes; last column: in k slices):
//                          64 x 64   128 x 64   128 x 128   128 x 128   256 x 256   slices
//                         2 groups   2 groups    2 groups    2 per CU
//   385 x 1000 x 1160        7.6*      7.8         8.8         9.8        17.2
//   256 x 4096 x 4096       12.2*     15.7        22.4        25.8        37.8
//   512 x 4096 x 4096       22.7      17.2*       22.8        26.6        38.9
//   1024 x 4096 x 4096      43.2      32.1        25.6*       29.5        40.2
//   2048 x 2048 x 2048      26.5      19.6        15.3*       17.0        25.3
//   4096 x 2048 x 768       29.5      21.1        16.7        12.2*       17.1
//   8192 x 1024 x 4096      79.0      58.4        47.6        38.1*       52.5
//   3000 x 3000 x 3000      66.9      58.4        52.4        46.4        37.7*
//   19712 x 2304 x 768     146         99.4        74.5        53.5        53.2*
//   4096 x 4096 x 4096     156        113          91.5        75.3        55.9*
//   2048 x 2048 x 8192        -         -          46.4*        -           -           49.2 (256 x 256, 4)
//   768 x 768 x 19712       50.8      72.0       106         111         159         33.2* (128 x 128, 8)
//   2304 x 768 x 19712     101         75.3        99.8       112         165         49.2* (256 x 256, 8)
// Up to 32 rows the rows kernel competes: every group of 16 columns reads all of A again, through L2 at 7.5 TB/s.  Weights from HBM, us
// (rows kernel / tiles; * = taken), N x K:
//                      1 row    8 rows   16 rows          32 rows         33 rows
//   4096 x 4096         6.5*     7.0*     7.4*             9.4*           12.0
//   8192 x 8192        16.2*    18.6*    21.6 / 21.2*     29.4 / 21.6*    21.8
//   14336 x 4096       14.9*    17.0*    20.2 / 16.0*     27.8 / 16.3*    16.3
//   4096 x 14336       12.9*    14.8*    17.3*            23.7 / 20.1*    20.2
enum { FP8_64, FP8_128X64, FP8_128G2, FP8_128, FP8_256, FP8_ROWS };
struct Fp8Plan { int kind, threads, tiles_n, splits, k_per_split, bm, bn; int64_t tiles; };
static Fp8Plan fp8_plan(int64_t M, int64_t N, int64_t Kp) {
    static const struct { int bm, bn, threads, per_cu; float fixed, step; } shape[] = {
        {64, 64, 512, 1, 3.5f, 0.265f}, {128, 64, 512, 1, 1.5f, 0.50f}, {128, 128, 512, 1, 5.4f, 0.65f}, {128, 128, 256, 2, 7.0f, 1.05f},
        {256, 256, 256, 1, 9.5f, 1.40f}};
    Fp8Plan q;
    const int nk = (int)(Kp / 128), cus = device_cu_count();
    const float bytes = (float)Kp * (float)(M + N);
    float best = 0.f;
    q.kind = -1;
    if (M <= 32) {
        q.kind = FP8_ROWS;
        q.tiles = q.tiles_n = (int)((N + 15) / 16);
        int w = 4;
        while (w < 16 && w * 4 < nk) w *= 2;
        q.threads = w * 64;
        q.splits = 1;
        q.k_per_split = nk;
        q.bm = q.bn = 0;
        const float l2 = (float)Kp * (float)(16 + M) * (float)q.tiles / 7.5e6f, hbm = bytes / 5.0e6f;
        best = 2.5f + (l2 > hbm ? l2 : hbm);
    }
    for (int k = FP8_64; k <= FP8_256; ++k) {
        if (k != FP8_64 && M <= shape[k].bm / 2) continue;           // half of the rows empty
        const int64_t tn = (N + shape[k].bn - 1) / shape[k].bn, tiles = ((M + shape[k].bm - 1) / shape[k].bm) * tn;
        for (int s = 1; s <= 16; s *= 2) {
            const int per = ((nk + s - 1) / s + 3) & ~3;             // whole scale dwords
            if (s > 1 && (per * (s - 1) >= nk || tiles * s > (int64_t)cus * shape[k].per_cu)) break;      // a slice more only fills a round
            const float rounds = (float)((tiles * s + cus * shape[k].per_cu - 1) / (cus * shape[k].per_cu));
            // one row of tiles: nobody else brings its part of B near, and a CU pulls 8 KB from HBM in 0.325 us
            const float step = M <= shape[k].bm && shape[k].step < 0.325f ? 0.325f : shape[k].step;
            float t = rounds * (shape[k].fixed + step * (float)(s > 1 ? per : nk));
            // the partial sums' stores and the join: 11.6-20 us measured for 14-17 M of them
            if (s > 1) t += 6.0f + 0.65e-6f * (float)s * (float)M * (float)N;
            if (t < 3.5f + bytes / 4.5e6f) t = 3.5f + bytes / 4.5e6f;         // the operands' bytes
            if (q.kind < 0 || t < best) {
                best = t;
                q.kind = k; q.threads = shape[k].threads; q.tiles_n = (int)tn; q.tiles = tiles; q.splits = s; q.k_per_split = s > 1 ? per : nk;
                q.bm = shape[k].bm; q.bn = shape[k].bn;
            }
        }
    }
    return q;
}
size_t gemm_nt_fp8_ws_bytes(int64_t M, int64_t N, int64_t Kp) {
    if (M <= 0 || N <= 0 || Kp <= 0) return 0;
    const Fp8Plan q = fp8_plan(M, N, Kp);
    return q.splits > 1 ? (size_t)q.splits * q.tiles * q.bm * q.bn * sizeof(float) : 0;
}

// more than 64 KB of dynamic LDS has to be asked for, once per kernel and device
static constexpr int FP8_256_LDS = 4 * 256 * 128 + 2 * 2048;
static int fp8_lds(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return (int)e;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return SPN_OK;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return (int)e;
    done.fetch_or(bit, std::memory_order_relaxed);
    return SPN_OK;
}

template <typename OUT>
static int fp8_launch(const Fp8Tile& p, const Fp8Plan& q, hipStream_t st) {
    static std::atomic<uint64_t> done[FP8_ROWS];
    const dim3 grid((unsigned)(q.tiles * p.splits));
#define SPN_FP8_LAUNCH(LDS_, ...)                                                                                   \
    do {                                                                                                            \
        const int rc = fp8_lds((const void*)__VA_ARGS__, LDS_, done[q.kind]);                                       \
        if (rc) return rc;                                                                                          \
        hipLaunchKernelGGL((__VA_ARGS__), grid, dim3(q.threads), LDS_, st, p);                                      \
    } while (0)
    switch (q.kind) {
        case FP8_64: SPN_FP8_LAUNCH((fp8_tile_lds<64, 64, 2, 4>()), gemm_fp8_tile_kernel<OUT, 64, 64, 2, 4>); break;
        case FP8_128X64: SPN_FP8_LAUNCH((fp8_tile_lds<128, 64, 2, 3>()), gemm_fp8_tile_kernel<OUT, 128, 64, 2, 3>); break;
        case FP8_128G2: SPN_FP8_LAUNCH((fp8_tile_lds<128, 128, 2, 2>()), gemm_fp8_tile_kernel<OUT, 128, 128, 2, 2>); break;
        case FP8_128: SPN_FP8_LAUNCH((fp8_tile_lds<128, 128, 1, 2>()), gemm_fp8_tile_kernel<OUT, 128, 128, 1, 2>); break;
        default: SPN_FP8_LAUNCH(FP8_256_LDS, gemm_fp8_256_kernel<OUT>); break;
    }
#undef SPN_FP8_LAUNCH
    return SPN_OK;
}
template <typename T>
static int fp8_launch_act(const Fp8Tile& p, const Fp8Plan& q, hipStream_t st) {
    if (p.act == ACT_QUICKGELU) return fp8_launch<Fp8Out<T, ACT_QUICKGELU>>(p, q, st);
    if (p.act == ACT_GELU_ERF) return fp8_launch<Fp8Out<T, ACT_GELU_ERF>>(p, q, st);
    return fp8_launch<Fp8Out<T, ACT_NONE>>(p, q, st);
}

int gemm_nt_fp8(const Fp8Gemm& g, hipStream_t st) {
    if (!g.a || !g.b || !g.sa || !g.sb || !g.out || g.M < 0 || g.N <= 0 || g.Kp <= 0) return SPN_ERR_ARG;
    if (g.M == 0) return SPN_OK;
    if (g.Kp % 128 || g.Kp >= (1ll << 24) || g.ldc < g.N || g.M >= (1ll << 31) || g.N >= (1ll << 31)) return SPN_ERR_SHAPE;
    if ((uintptr_t)g.a % 16 || (uintptr_t)g.b % 16 || (uintptr_t)g.sa % 4 || (uintptr_t)g.sb % 4) return SPN_ERR_SHAPE;
    if (g.out_type < ET_F32 || g.out_type > ET_F16 || (g.accumulate && (g.out_type != ET_F32 || g.act != ACT_NONE))) return SPN_ERR_ARG;
    if (g.act < ACT_NONE || g.act > ACT_GELU_ERF) return SPN_ERR_ARG;
    const size_t need = gemm_nt_fp8_ws_bytes(g.M, g.N, g.Kp);
    if (need && (!g.ws || g.ws_bytes < need || (uintptr_t)g.ws % 16)) return SPN_ERR_WORKSPACE;
    Fp8Tile p;
    p.a = g.a; p.b = g.b; p.sa = g.sa; p.sb = g.sb; p.M = g.M; p.N = g.N; p.Kp = g.Kp;
    p.pitch = qscale_pitch(g.Kp); p.nk = (int)(g.Kp / 128);
    p.bias = g.bias; p.act = g.act; p.out = g.out; p.out_type = g.out_type; p.accumulate = g.accumulate; p.ldc = g.ldc; p.part = g.ws;
    const Fp8Plan q = fp8_plan(g.M, g.N, g.Kp);
    p.splits = q.splits; p.k_per_split = q.k_per_split; p.tiles = (int)q.tiles; p.tiles_n = q.tiles_n;
    p.group = 8;
    if (q.tiles * q.threads >= (1ll << 32)) return SPN_ERR_SHAPE;      // what a launch can hold
    if (q.kind == FP8_ROWS) {
        const int mt = (int)((g.M + 15) / 16);
        const size_t lds = (size_t)(q.threads / 64) * mt * 1024;
        if (mt == 1) hipLaunchKernelGGL(gemm_fp8_rows_kernel<1>, dim3((unsigned)q.tiles), dim3(q.threads), lds, st, p);
        else hipLaunchKernelGGL(gemm_fp8_rows_kernel<2>, dim3((unsigned)q.tiles), dim3(q.threads), lds, st, p);
    } else {
        int rc;
        if (p.splits > 1) rc = fp8_launch<Fp8Part>(p, q, st);
        else if (p.out_type == ET_F32) rc = fp8_launch<Fp8Wide>(p, q, st);
        else if (p.out_type == ET_BF16) rc = fp8_launch_act<bf16_t>(p, q, st);
        else rc = fp8_launch_act<f16_t>(p, q, st);
        if (rc) return rc;
    }
    SPN_CHECK_LAUNCH();
    if (p.splits > 1) {
        hipLaunchKernelGGL(gemm_fp8_join_kernel, dim3((unsigned)q.tiles, (unsigned)(q.bm / 64 * (q.bn / 64))), dim3(256), 0, st, p, q.bm, q.bn);
        SPN_CHECK_LAUNCH();
    }
    return SPN_OK;
}

}  // namespace spn
