// Matrix product in 8-bit integers with a scale for every row of both sides:
//
//   out[m][n] = float(sum_k x[m][k] w[n][k]) * x_scale[m] * w_scale[n],   x_scale[m] = max_k |x[m][k]| / 127
//
// Both sides lie in blocks of 16 rows by 64 columns, 1 KB in the order in which the matrix cores' operands are read: a lane's 16 columns of a row are 16
// bytes, 16 rows beside each other.  A block goes global -> LDS as it is, one load a wave, and a 32x32x32 operand is one conflict-free 16-byte read a lane.
//
// What bounds the product: of few rows the weights' bytes (a vocabulary of 128256 by 2560 and one row 58 us, 5.7 TB/s; a library's product in bf16 119), of many
// the matrix instructions, whose pipes are busy half of the clocks at 1.9 GHz (8192 x 8192 x 8192 460 us, 2390 Tera-operations a second, a library's own product in
// 8-bit integers 480 to 500; 4096 x 13824 x 2560 147 us, 1980, of whose tiles the last round is a third full).  Between them it is a CU's reads: a stage of a
// 64 x 64 tile is 16 KB for 0.18 us with four stages under way -- 40 bytes a clock, or a read's 0.7 us: not told apart (333 x 2501 x 6912, 240 workgroups: 14.4 to 14.8 us
// replayed, 15.3 and more under a profiler; a second group of four waves for half of a stage's columns changes nothing there, nor do two parts with a launch that joins
// them, 19.6).
#pragma once

#include "int8_plan.h"
#include "norm_quant_kernel.h"

namespace terna {

constexpr int kInt8Threads = 256;
constexpr int kInt8MaxK = 131056;              // 128 * 128 * K < 2^31

constexpr long long int8_bands(long long rows) { return (rows + 15) / 16; }

// ---- rows into blocks ------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ size_t int8_piece(int row, int piece, int k_blocks)     // byte of columns 16 * piece .. + 15 of a row
{
    return ((static_cast<size_t>(row >> 4) * k_blocks + (piece >> 2)) << 10) + (((piece & 3) * 16 + (row & 15)) << 4);
}

// 16 columns of a row as they are, zeros behind the last
template <typename E>
struct Int8Piece {
    static constexpr int WORDS = sizeof(E);                                // of 16 bytes
    u32x4 of[WORDS];

    __device__ __forceinline__ void load(const E* row, int k, int K, bool wide)
    {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) of[i] = u32x4{0u, 0u, 0u, 0u};
        if (k >= K) return;
        if (wide && k + 16 <= K) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) of[i] = *reinterpret_cast<const u32x4*>(row + k + i * (16 / WORDS));
            return;
        }
        constexpr int PER = 4 / sizeof(E);                                 // elements of a 32-bit word
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            uint32_t bits = 0;
            if (k + e < K) {
                if constexpr (sizeof(E) == 4) bits = __float_as_uint(row[k + e]);
                else bits = row[k + e];
            }
            const int w = e / PER;
            of[w >> 2][w & 3] |= bits << (8 * sizeof(E) * (e % PER));
        }
    }
    __device__ __forceinline__ void values(float (&f)[16]) const
    {
        if constexpr (sizeof(E) == 2) {
            unpack_bf16x8(of[0], f);
            unpack_bf16x8(of[1], f + 8);
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) f[e] = __uint_as_float(of[e >> 2][e & 3]);
        }
    }
};

// A wave a row, HELD pieces of 16 columns a lane in registers; longer rows are read again for their integers.  2048 rows of 2560 take 5.6 us, 13 where
// sixteen threads took a row, read twice; 8192 of 6912 43 us, 4 TB/s.
template <typename E, int HELD>
__global__ __launch_bounds__(kInt8Threads) void terna_int8_quantise_kernel(const E* __restrict__ x, long long row_stride, uint8_t* __restrict__ packed,
                                                                           float* __restrict__ scale, int R, int K, int wide)
{
// the product is rounded before it is rounded to an integer
#pragma clang fp contract(off)
    // Workgroups go to the XCDs round robin: each XCD takes a run of the rows, whose pieces -- eight rows' to a line of memory -- meet in its L2 (8192 x 6912: 46 us without)
    const int lane = threadIdx.x & 63, group = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int r = group * (kInt8Threads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (r >= R) return;
    const int k_blocks = int8_k_blocks(K), pieces = 4 * k_blocks;
    const E* const row = x + static_cast<size_t>(r) * row_stride;
    Int8Piece<E> held[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) held[i].load(row, 16 * (lane + 64 * i), K, wide);
    float top = 0.0f;
    auto measure = [&](const Int8Piece<E>& piece) __attribute__((always_inline)) {
        float f[16];
        piece.values(f);
#pragma unroll
        for (int e = 0; e < 16; ++e) top = max_keep_nan(top, fabsf(f[e]));
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i) measure(held[i]);
    for (int p = lane + 64 * HELD; p < pieces; p += 64) {
        Int8Piece<E> piece;
        piece.load(row, 16 * p, K, wide);
        measure(piece);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = max_keep_nan(top, __shfl_xor(top, off));
    const bool finite = top < INFINITY, zero = top < 0x1p-120f;
    const float by = !finite || zero ? 0.0f : __fdiv_rn(127.0f, top);
    if (lane == 0) scale[r] = !finite ? NAN : zero ? 0.0f : __fdiv_rn(top, 127.0f);
    const float magic = 12582912.0f;           // 1.5 * 2^23: a sum's low byte is the integer
    auto write = [&](const Int8Piece<E>& piece, int p) __attribute__((always_inline)) {
        float f[16];
        piece.values(f);
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
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (lane + 64 * i < pieces) write(held[i], lane + 64 * i);
    for (int p = lane + 64 * HELD; p < pieces; p += 64) {
        Int8Piece<E> piece;
        piece.load(row, 16 * p, K, wide);
        write(piece, p);
    }
}

// int8 rows as they are: a wave four blocks of a band, whole kilobytes out: 8192 x 6912 20 us, 38 with a wave a row, whose pieces go out one by one
constexpr int kInt8PackBlocks = 4;
__global__ __launch_bounds__(kInt8Threads) void terna_int8_pack_kernel(const uint8_t* __restrict__ x, long long row_stride, uint8_t* __restrict__ packed, int R, int K, int wide)
{
    const int lane = threadIdx.x & 63, k_blocks = int8_k_blocks(K), each = (k_blocks + kInt8PackBlocks - 1) / kInt8PackBlocks;
    const long long unit = static_cast<long long>(blockIdx.x) * (kInt8Threads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int band = static_cast<int>(unit / each), b0 = static_cast<int>(unit - static_cast<long long>(band) * each) * kInt8PackBlocks, r = 16 * band + (lane & 15);
    if (r >= R) return;
    const uint8_t* const row = x + static_cast<size_t>(r) * row_stride;
    Int8Piece<uint8_t> piece[kInt8PackBlocks];
#pragma unroll
    for (int i = 0; i < kInt8PackBlocks; ++i) piece[i].load(row, 64 * (b0 + i) + 16 * (lane >> 4), K, wide);
#pragma unroll
    for (int i = 0; i < kInt8PackBlocks; ++i)
        if (b0 + i < k_blocks) *reinterpret_cast<u32x4*>(packed + ((static_cast<size_t>(band) * k_blocks + b0 + i) << 10) + lane * 16) = piece[i].of[0];
}

// ---- the product ------------------------------------------------------------------------------------------------------------------

struct Int8Linear {
    const uint8_t *x, *w;
    const float *x_scale, *w_scale;
    void* out;
    int32_t* partial;                          // more than one split: sums [tile][split][wave][product][4][lane][4]
    int M, N, K, tiles_m, tiles_n, splits;
};

// A workgroup's tile: WN x WM waves of NA x MB products of 32 x 32 -- features x rows --, SK blocks of 64 columns a stage, ST stages in LDS.
template <int WN, int WM, int NA, int MB, int SK, int ST>
struct Int8Tile {
    static constexpr int BN = 32 * NA * WN, BM = 32 * MB * WM;
    static constexpr int kBlocks = (BN + BM) / 16 * SK, kLoads = kBlocks / 4, kStage = kBlocks * 1024, kRing = ST * kStage;
    static_assert(WN * WM == 4 && kBlocks % 4 == 0 && ST >= 3);
    // results on their way out: 32 rows of each of the WM waves at a time, 16 bytes apart in the banks
    template <typename Out>
    static constexpr int pitch() { return BN * static_cast<int>(sizeof(Out)) + 16; }
    template <typename Out>
    static constexpr int bytes() { return kRing > 32 * WM * pitch<Out>() ? kRing : 32 * WM * pitch<Out>(); }
};

// Where a workgroup works.  Workgroups go to the XCDs round robin: each XCD takes a run of the tiles, which go down bands of up to four tiles of rows, so that
// what is under way on an XCD at a time is about as many tiles wide as high and its reads meet in its L2.
struct Int8Place {
    int tile, tile_m, tile_n, split;
    bool real;
};
__device__ __forceinline__ Int8Place int8_place(const Int8Linear& a, int splits)
{
    const int tiles = a.tiles_m * a.tiles_n, units = tiles * splits, per_xcd = (units + 7) / 8;
    const int in_xcd = blockIdx.x >> 3, unit = (blockIdx.x & 7) * per_xcd + in_xcd;
    Int8Place p;
    p.real = unit < units && in_xcd < per_xcd;
    p.tile = splits == 1 ? unit : unit / splits;
    p.split = unit - p.tile * splits;
    const int band = p.tile / (4 * a.tiles_n), high = min(4, a.tiles_m - 4 * band), in_band = p.tile - band * (4 * a.tiles_n);
    p.tile_n = in_band / high;
    p.tile_m = 4 * band + in_band - p.tile_n * high;
    return p;
}

// Sums -> results, out by whole rows: lane (m, half) has features 8 i + 4 half .. + 3 of row m of its 32.
template <typename Out, typename Tile, int WN, int WM, int NA, int MB>
__device__ __forceinline__ void int8_finish(const Int8Linear& a, const Int8Place& place, const i32x16 (&acc)[NA][MB], uint8_t* smem)
{
    constexpr int BN = Tile::BN, BM = Tile::BM;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int wn = wave % WN, wm = wave / WN, tile_m = place.tile_m, tile_n = place.tile_n;
    constexpr int PITCH = Tile::template pitch<Out>(), SIZE = sizeof(Out), EACH = 16 / SIZE, ROW = BN / EACH;      // 16-byte pieces of a row
    Out* const out = static_cast<Out*>(a.out);
    const bool whole = static_cast<long long>(a.N) * SIZE % 16 == 0;
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        const int m = tile_m * BM + (wm * MB + j) * 32 + (lane & 31);
        const float xs = a.x_scale[min(m, a.M - 1)];
        const float* w_scale = a.w_scale;
        asm volatile("" : "+s"(w_scale));                                  // read again every time: kept, they were registers that the tile does not leave
        uint8_t* const row = smem + (wm * 32 + (lane & 31)) * PITCH + (wn * NA * 32 + 4 * half) * SIZE;
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int n = tile_n * BN + (wn * NA + i) * 32 + 8 * v + 4 * half;
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = static_cast<float>(acc[i][j][4 * v + e]) * xs * w_scale[min(n + e, a.N - 1)];
                uint8_t* const to = row + (32 * i + 8 * v) * SIZE;
                if constexpr (SIZE == 2) *reinterpret_cast<u32x2*>(to) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
                else *reinterpret_cast<f32x4*>(to) = f32x4{y[0], y[1], y[2], y[3]};
            }
        __syncthreads();
        const int m0 = tile_m * BM + j * 32;                               // of the first wave's rows; the next wave's MB * 32 further
        if (whole) {
            for (int x = tid; x < 32 * WM * ROW; x += 256) {
                const int r = x / ROW, piece = x % ROW, mm = m0 + (r >> 5) * (MB * 32) + (r & 31), n = tile_n * BN + piece * EACH;
                if (mm < a.M && n < a.N) *reinterpret_cast<u32x4*>(out + static_cast<size_t>(mm) * a.N + n) = *reinterpret_cast<const u32x4*>(smem + r * PITCH + piece * 16);
            }
        } else {
            // rows that begin anywhere: the pieces that memory has aligned, then the elements in front of and behind them (650 x 50021 x 272: 47 us, element by element 68; with
            // 50024 features, all aligned, 40)
            const int count = min(BN, a.N - tile_n * BN);
            auto row_at = [&](int r) { return m0 + (r >> 5) * (MB * 32) + (r & 31); };
            auto head_of = [&](const Out* to) { return min(count, -static_cast<int>(reinterpret_cast<uintptr_t>(to) / SIZE) & (EACH - 1)); };
            for (int x = tid; x < 32 * WM * ROW; x += 256) {
                const int r = x / ROW, mm = row_at(r);
                if (mm >= a.M) continue;
                Out* const to = out + static_cast<size_t>(mm) * a.N + tile_n * BN;
                const int from = head_of(to) + x % ROW * EACH;
                if (from + EACH > count) continue;
                const uint32_t* const words = reinterpret_cast<const uint32_t*>(smem + r * PITCH + (from * SIZE & ~3));
                u32x4 y{words[0], words[1], words[2], words[3]};
                if constexpr (SIZE == 2) {
                    const uint32_t last = words[4], by = (from & 1) * 2;
                    y = u32x4{__builtin_amdgcn_alignbyte(y.y, y.x, by), __builtin_amdgcn_alignbyte(y.z, y.y, by), __builtin_amdgcn_alignbyte(y.w, y.z, by), __builtin_amdgcn_alignbyte(last, y.w, by)};
                }
                *reinterpret_cast<u32x4*>(to + from) = y;
            }
            for (int x = tid; x < 32 * WM * 2 * EACH; x += 256) {
                const int r = x / (2 * EACH), e = x % (2 * EACH), mm = row_at(r);
                if (mm >= a.M) continue;
                Out* const to = out + static_cast<size_t>(mm) * a.N + tile_n * BN;
                const int head = head_of(to), c = e < EACH ? e : head + (count - head) / EACH * EACH + e - EACH;
                if (c < (e < EACH ? head : count)) to[c] = *reinterpret_cast<const Out*>(smem + r * PITCH + c * SIZE);
            }
        }
        if (j + 1 < MB) __syncthreads();
    }
}

template <typename Out, int WN, int WM, int NA, int MB, int SK, int ST>
__global__ __launch_bounds__(256, 2) void terna_int8_linear_kernel(Int8Linear a)
{
    using Tile = Int8Tile<WN, WM, NA, MB, SK, ST>;
    constexpr int BN = Tile::BN, BM = Tile::BM, LOADS = Tile::kLoads;
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int wn = wave % WN, wm = wave / WN;
    const Int8Place place = int8_place(a, a.splits);
    if (!place.real) return;
    const int tile_m = place.tile_m, tile_n = place.tile_n;
    const int k_blocks = int8_k_blocks(a.K), all_steps = k_blocks / SK, share = (all_steps + a.splits - 1) / a.splits;
    const int first = place.split * share, steps = min(share, all_steps - first);
    const int bands_w = (a.N + 15) >> 4, bands_x = (a.M + 15) >> 4;
    // ---- blocks that this wave fetches: block wave + 4 i of a stage (bands behind the last are read from it)
    const uint8_t* from[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int l = wave + 4 * i, b = l / SK, kb = l % SK;
        const bool weight = b < BN / 16;
        const int at = weight ? min(tile_n * (BN / 16) + b, bands_w - 1) : min(tile_m * (BM / 16) + b - BN / 16, bands_x - 1);
        from[i] = (weight ? a.w : a.x) + ((static_cast<size_t>(at) * k_blocks + first * SK + kb) << 10);
    }
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem)) + wave * 1024;
    auto load = [&](int step, int at, int i) __attribute__((always_inline)) {          // (behind the last step its blocks again, which nobody reads)
        lds_dma_b128(from[i] + static_cast<uint32_t>(min(step, steps - 1)) * (SK * 1024), lane * 16, lds0 + at * Tile::kStage + i * 4096);
    };
    // operand of 32 rows (two bands), 32 columns
    const int lane_at = ((lane >> 4) & 1) * (SK * 1024) + ((half * 16 + (lane & 15)) << 4);
    constexpr int HALVES = 2 * SK, OPERANDS = NA + MB, PRODUCTS = NA * MB;
    struct Operands {
        i32x4 of[OPERANDS];                                                // features, then rows
    };
    auto operand = [&](const uint8_t* stage, int h, int i) __attribute__((always_inline)) {
        const int two = i < NA ? wn * NA + i : BN / 32 + wm * MB + i - NA;
        return __builtin_bit_cast(i32x4, *reinterpret_cast<const u32x4*>(stage + (two * 2 * SK + (h >> 1)) * 1024 + lane_at + (h & 1) * 512));
    };
    // (a product that waits for the one before it, its own sum, stands still for longer than it takes: few have two sums in turns)
    constexpr int SUMS = PRODUCTS <= 2 ? 2 : 1;
    i32x16 sums[SUMS][NA][MB];
#pragma unroll
    for (int u = 0; u < SUMS; ++u)
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int j = 0; j < MB; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) sums[u][i][j][v] = 0;
    i32x16 (&acc)[NA][MB] = sums[0];
#pragma unroll
    for (int s = 0; s < ST - 1; ++s)
#pragma unroll
        for (int i = 0; i < LOADS; ++i) load(s, s, i);
    Operands cur;
    int at = 0;
    for (int step = 0; step < steps; ++step) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((ST - 2) * LOADS) : "memory");
        const int behind = at == 0 ? ST - 1 : at - 1, ahead = at + 1 == ST ? 0 : at + 1;
        const uint8_t* const stage = smem + at * Tile::kStage;
#pragma unroll
        for (int i = 0; i < OPERANDS; ++i) cur.of[i] = operand(stage, 0, i);
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            Operands next;
            // the next operands' reads and the requests, spread over the products
#pragma unroll
            for (int p = 0; p < PRODUCTS; ++p) {
                const int i = p / MB, j = p % MB;
                i32x16& sum = sums[h % SUMS][i][j];
                sum = __builtin_amdgcn_mfma_i32_32x32x32_i8(cur.of[i], cur.of[NA + j], sum, 0, 0, 0);
#pragma unroll
                for (int r = p * OPERANDS / PRODUCTS; r < (p + 1) * OPERANDS / PRODUCTS; ++r)
                    if (h + 1 < HALVES) next.of[r] = operand(stage, h + 1, r);
                const int q = h * PRODUCTS + p;
#pragma unroll
                for (int r = q * LOADS / (HALVES * PRODUCTS); r < (q + 1) * LOADS / (HALVES * PRODUCTS); ++r) load(step + ST - 1, behind, r);
                if (PRODUCTS > 4) __builtin_amdgcn_sched_barrier(0);
            }
            if (h + 1 < HALVES) cur = next;
        }
        at = ahead;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if constexpr (SUMS == 2) {
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int j = 0; j < MB; ++j) acc[i][j] += sums[1][i][j];
    }
    if (a.splits > 1) {                                                    // (integers: in whatever order they are added)
        int32_t* const to = a.partial + (static_cast<size_t>(place.tile) * a.splits + place.split) * (BN * BM) + wave * (NA * MB * 1024) + lane * 4;
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int j = 0; j < MB; ++j)
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    *reinterpret_cast<i32x4*>(to + ((i * MB + j) * 4 + v) * 256) = i32x4{acc[i][j][4 * v], acc[i][j][4 * v + 1], acc[i][j][4 * v + 2], acc[i][j][4 * v + 3]};
        return;
    }
    int8_finish<Out, Tile, WN, WM, NA, MB>(a, place, acc, smem);
}

// The splits' sums of a tile, and its results.
template <typename Out, int WN, int WM, int NA, int MB, int SK, int ST>
__global__ __launch_bounds__(256, 1) void terna_int8_join_kernel(Int8Linear a)
{
    using Tile = Int8Tile<WN, WM, NA, MB, SK, ST>;
    extern __shared__ __align__(16) uint8_t smem[];
    const Int8Place place = int8_place(a, 1);
    if (!place.real) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int32_t* from = a.partial + static_cast<size_t>(place.tile) * a.splits * (Tile::BN * Tile::BM) + wave * (NA * MB * 1024) + lane * 4;
    i32x16 acc[NA][MB];
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;
    for (int s = 0; s < a.splits; ++s, from += Tile::BN * Tile::BM) {
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int j = 0; j < MB; ++j)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const i32x4 x = *reinterpret_cast<const i32x4*>(from + ((i * MB + j) * 4 + v) * 256);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][4 * v + e] += x[e];
                }
    }
    int8_finish<Out, Tile, WN, WM, NA, MB>(a, place, acc, smem);
}

}  // namespace terna
