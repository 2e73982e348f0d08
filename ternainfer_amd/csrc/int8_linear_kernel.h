// Matrix product in 8-bit integers with a scale for every row of both sides:
//
//   out[m][n] = float(sum_k x[m][k] w[n][k]) * x_scale[m] * w_scale[n],   x_scale[m] = max_k |x[m][k]| / 127
//
// Both sides lie in blocks of 16 rows by 64 columns, 1 KB in the order in which the matrix cores' operands are read: a lane's 16 columns of a row are 16
// bytes, 16 rows beside each other.  A block goes global -> LDS as it is, one load a wave, and a 32x32x32 operand is one conflict-free 16-byte read a lane.
#pragma once

#include "norm_quant_kernel.h"

namespace terna {

constexpr int kInt8Threads = 256;
constexpr int kInt8MaxK = 131056;              // 128 * 128 * K < 2^31

__host__ __device__ constexpr int int8_k_blocks(int K) { return 2 * ((K + 127) / 128); }
constexpr long long int8_bands(long long rows) { return (rows + 15) / 16; }

// ---- rows into blocks ------------------------------------------------------------------------------------------------------------------

// 16 columns from k on, zeros behind the last
template <typename E>
__device__ __forceinline__ void int8_load(const E* row, int k, int K, bool wide, float (&f)[16])
{
    if (wide && k + 16 <= K) {
        if constexpr (sizeof(E) == 2) {
            unpack_bf16x8(*reinterpret_cast<const u32x4*>(row + k), f);
            unpack_bf16x8(*reinterpret_cast<const u32x4*>(row + k + 8), f + 8);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(row + k + 4 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) f[4 * i + e] = x[e];
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            if constexpr (sizeof(E) == 2) f[e] = k + e < K ? bf16_bits_to_float(row[k + e]) : 0.0f;
            else f[e] = k + e < K ? row[k + e] : 0.0f;
        }
    }
}
__device__ __forceinline__ size_t int8_piece(int row, int piece, int k_blocks)     // byte of columns 16 * piece .. + 15 of a row
{
    return ((static_cast<size_t>(row >> 4) * k_blocks + (piece >> 2)) << 10) + (((piece & 3) * 16 + (row & 15)) << 4);
}

// ROWS rows a workgroup, 256 / ROWS threads each; the rows are read twice (the second time from the caches): their maximum, then their integers.
template <typename E, int ROWS>
__global__ __launch_bounds__(kInt8Threads) void terna_int8_quantise_kernel(const E* __restrict__ x, long long row_stride, uint8_t* __restrict__ packed,
                                                                           float* __restrict__ scale, int R, int K, int wide)
{
// the product is rounded before it is rounded to an integer
#pragma clang fp contract(off)
    constexpr int EACH = kInt8Threads / ROWS;
    __shared__ float tops[kInt8Threads / 64][ROWS];
    const int tid = threadIdx.x, wave = tid >> 6, mine = tid % ROWS, part = tid / ROWS;
    const int r = blockIdx.x * ROWS + mine, k_blocks = int8_k_blocks(K), pieces = 4 * k_blocks;
    const E* const row = x + static_cast<size_t>(min(r, R - 1)) * row_stride;
    float top = 0.0f;
    for (int p = part; p < pieces; p += EACH) {
        float f[16];
        int8_load(row, 16 * p, K, wide, f);
#pragma unroll
        for (int e = 0; e < 16; ++e) top = max_keep_nan(top, fabsf(f[e]));
    }
#pragma unroll
    for (int off = 32; off >= ROWS; off >>= 1) top = max_keep_nan(top, __shfl_xor(top, off));
    if ((tid & 63) < ROWS) tops[wave][mine] = top;
    __syncthreads();
    top = tops[0][mine];
#pragma unroll
    for (int w = 1; w < kInt8Threads / 64; ++w) top = max_keep_nan(top, tops[w][mine]);
    if (r >= R) return;
    const bool finite = top < INFINITY, zero = top < 0x1p-120f;
    const float by = !finite || zero ? 0.0f : __fdiv_rn(127.0f, top);
    if (part == 0) scale[r] = !finite ? NAN : zero ? 0.0f : __fdiv_rn(top, 127.0f);
    const float magic = 12582912.0f;           // 1.5 * 2^23: a sum's low byte is the integer
    for (int p = part; p < pieces; p += EACH) {
        float f[16];
        int8_load(row, 16 * p, K, wide, f);
        u32x4 q;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(f[4 * i + e] * by + magic);
            q[i] = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
        }
        if (!finite) q = u32x4{0u, 0u, 0u, 0u};
        *reinterpret_cast<u32x4*>(packed + int8_piece(r, p, k_blocks)) = q;
    }
}

// int8 rows as they are: 16 rows a workgroup
__global__ __launch_bounds__(kInt8Threads) void terna_int8_pack_kernel(const uint8_t* __restrict__ x, long long row_stride, uint8_t* __restrict__ packed, int R, int K, int wide)
{
    const int r = blockIdx.x * 16 + (threadIdx.x & 15), k_blocks = int8_k_blocks(K);
    if (r >= R) return;
    const uint8_t* const row = x + static_cast<size_t>(r) * row_stride;
    for (int p = threadIdx.x >> 4; p < 4 * k_blocks; p += kInt8Threads / 16) {
        u32x4 q{0u, 0u, 0u, 0u};
        if (wide && 16 * p + 16 <= K) q = *reinterpret_cast<const u32x4*>(row + 16 * p);
        else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (16 * p + e < K) q[e >> 2] |= static_cast<uint32_t>(row[16 * p + e]) << (8 * (e & 3));
        }
        *reinterpret_cast<u32x4*>(packed + int8_piece(r, p, k_blocks)) = q;
    }
}

// ---- the product ------------------------------------------------------------------------------------------------------------------

struct Int8Linear {
    const uint8_t *x, *w;
    const float *x_scale, *w_scale;
    void* out;
    int M, N, K, tiles_m, tiles_n;
};

// A workgroup's tile: WN x WM waves of NA x MB products of 32 x 32 -- features x rows --, SK blocks of 64 columns a stage, ST stages in LDS.
template <int WN, int WM, int NA, int MB, int SK, int ST>
struct Int8Tile {
    static constexpr int BN = 32 * NA * WN, BM = 32 * MB * WM;
    static constexpr int kBlocks = (BN + BM) / 16 * SK, kLoads = kBlocks / 4, kStage = kBlocks * 1024, kBytes = ST * kStage;
    static_assert(WN * WM == 4 && kBlocks % 4 == 0);
};

template <typename Out, int WN, int WM, int NA, int MB, int SK, int ST>
__global__ __launch_bounds__(256, (NA * MB > 8 ? 1 : 2)) void terna_int8_linear_kernel(Int8Linear a)
{
    using Tile = Int8Tile<WN, WM, NA, MB, SK, ST>;
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int wn = wave % WN, wm = wave / WN;
    const int tile_m = blockIdx.x % a.tiles_m, tile_n = blockIdx.x / a.tiles_m;
    const int k_blocks = int8_k_blocks(a.K), steps = k_blocks / SK;
    const int bands_w = (a.N + 15) >> 4, bands_x = (a.M + 15) >> 4;
    // ---- blocks that this wave fetches: block wave + 4 i of a stage (bands behind the last are read from it)
    const uint8_t* from[Tile::kLoads];
#pragma unroll
    for (int i = 0; i < Tile::kLoads; ++i) {
        const int l = wave + 4 * i, band = l / SK, kb = l % SK;
        const bool weight = band < Tile::BN / 16;
        const int at = weight ? min(tile_n * (Tile::BN / 16) + band, bands_w - 1) : min(tile_m * (Tile::BM / 16) + band - Tile::BN / 16, bands_x - 1);
        from[i] = (weight ? a.w : a.x) + ((static_cast<size_t>(at) * k_blocks + kb) << 10);
    }
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem)) + wave * 1024;
    auto load = [&](int step, int at) __attribute__((always_inline)) {     // (behind the last step its blocks again, which nobody reads)
        const size_t off = static_cast<size_t>(min(step, steps - 1)) * (SK * 1024);
#pragma unroll
        for (int i = 0; i < Tile::kLoads; ++i) lds_dma_b128(from[i] + off, lane * 16, lds0 + at * Tile::kStage + i * 4096);
    };
    // operand of 32 rows (two bands), 32 columns
    const int lane_at = ((lane >> 4) & 1) * (SK * 1024) + ((half * 16 + (lane & 15)) << 4);
    auto operand = [&](const uint8_t* stage, int band, int kb, int s) __attribute__((always_inline)) {
        return __builtin_bit_cast(i32x4, *reinterpret_cast<const u32x4*>(stage + (band * SK + kb) * 1024 + lane_at + s * 512));
    };
    i32x16 acc[NA][MB];
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) load(i, i);
    int at = 0;
    for (int step = 0; step < steps; ++step) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((ST - 2) * Tile::kLoads) : "memory");
        load(step + ST - 1, at == 0 ? ST - 1 : at - 1);
        const uint8_t* const stage = smem + at * Tile::kStage;
        at = at + 1 == ST ? 0 : at + 1;
#pragma unroll
        for (int kb = 0; kb < SK; ++kb)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                i32x4 w[NA], x[MB];
#pragma unroll
                for (int i = 0; i < NA; ++i) w[i] = operand(stage, (wn * NA + i) * 2, kb, s);
#pragma unroll
                for (int j = 0; j < MB; ++j) x[j] = operand(stage, Tile::BN / 16 + (wm * MB + j) * 2, kb, s);
#pragma unroll
                for (int i = 0; i < NA; ++i)
#pragma unroll
                    for (int j = 0; j < MB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[i], x[j], acc[i][j], 0, 0, 0);
            }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");

    // lane: row m of its 32, features 8 i + 4 half .. + 3
    Out* const out = static_cast<Out*>(a.out);
    const bool wide = (a.N & 3) == 0;
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        const int m = tile_m * Tile::BM + (wm * MB + j) * 32 + (lane & 31);
        if (m >= a.M) continue;
        const float xs = a.x_scale[m];
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int v = 0; v < 16; v += 4) {
                const int n = tile_n * Tile::BN + (wn * NA + i) * 32 + 2 * v + 4 * half;
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = static_cast<float>(acc[i][j][v + e]) * xs * (n + e < a.N ? a.w_scale[n + e] : 0.0f);
                Out* const to = out + static_cast<size_t>(m) * a.N + n;
                if (wide && n + 4 <= a.N) {
                    if constexpr (sizeof(Out) == 2) *reinterpret_cast<u32x2*>(to) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
                    else *reinterpret_cast<f32x4*>(to) = f32x4{y[0], y[1], y[2], y[3]};
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (n + e >= a.N) continue;
                        if constexpr (sizeof(Out) == 2) to[e] = float_to_bf16_bits(y[e]);
                        else to[e] = y[e];
                    }
                }
            }
    }
}

}  // namespace terna
