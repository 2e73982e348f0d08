// Attention of a tree of drafted tokens over the cache: node i of a sequence sees the slots in front of the tree and, of the tree's own (node j in slot
// start + j), those of its mask.
//
//   out[row] = sum_s p_s v_s / sum_s p_s,  p_s = exp(scale q . k_s - max)
//
// The rows of a kv head -- its G = H / KV query heads times the nodes, row r = node * G + head -- are the columns of 32x32x16 products, 32 a wave: the scores
// (slots x rows) come out of the matrix cores in the layout in which their exponentials go back in as the second product's operand, and a row's maximum
// and sum are one exchange between two lanes.
//   * A workgroup is four waves: RW of them share the slots, 32 rows each, and 4 / RW groups of those take turns of 32 slots, so that a few rows still
//     read a cache with four waves.  The groups' numerators are joined in LDS at the end, the splits' by a second launch.
//   * Keys and values go global -> LDS directly, ST - 1 steps ahead; 16-byte pieces are XOR-swizzled on the way, so that neither the keys' 16-byte operand reads
//     nor the values' transposing ones conflict.  A wave that shares its slots with nobody waits for its own requests only.
//   * Probabilities are two bf16, high and low part: 16 bits of them count.  The running maximum is raised, and the output rescaled, only where it grows by
//     more than 2^3 -- a row's own.
//   * Only the last tiles have slots of the tree.  There the mask's bits select the scores, and values that are not finite are taken out -- a slot that
//     one node sees and another does not must not reach the other through 0 * NaN; the rows that do see them get them back at the end.
// What bounds it: see the launch's side (abi_tree.hip) and the times there.
#pragma once

#include "draft_tree_kernel.h"
#include "tree_plan.h"

namespace terna {

typedef short tree_s16x4 __attribute__((ext_vector_type(4)));

constexpr float kTreeGrowth = 3.0f;

struct TreeAttention {
    const uint16_t *q, *k, *v;
    const long long *start, *mask;
    uint16_t* out;                             // [B * T][H * D], or
    float* partial;                            // more than one split: fp32 [rows][splits][D] numerators, then [rows][splits][2] maximum, sum
    long long q_seq, q_head, q_node;           // strides, elements
    long long k_seq, k_head, v_seq, v_head;
    int k_slot, v_slot;                        // ... of a slot, bytes
    int B, T, H, KV, S, W, splits, tiles, per_seq;
    float scale;                               // times log2(e)
};

template <int D, int RW, int ST>
struct TreeShape {
    static constexpr int KW = 4 / RW;
    static constexpr int kTile = kTreeTile * D * 2;                        // bytes of a tile's keys, or values
    static constexpr int kRing = KW * ST * 2 * kTile;
    static constexpr int kRow = D + 4;                                     // floats of a row of numerators in LDS
    static constexpr int kJoin = 4 * 32 * kRow * 4;
    static constexpr int kBytes = kRing > kJoin ? kRing : kJoin;
};

// Layout of a tile's values: rows of 2 D bytes, conflict-free for transposing reads.
template <int D>
__device__ __forceinline__ int tree_value_piece(int row, int piece) { return piece ^ (D == 128 ? (row & 7) << 1 : (row & 6)); }
template <int D>
__device__ __forceinline__ int tree_key_piece(int row, int piece) { return piece ^ (D == 128 ? row & 15 : (row >> 1) & 7); }

// NaN where one of them is
__device__ __forceinline__ float tree_max3(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }

// max / sum over the lanes L, L ^ 32
template <bool IS_MAX>
__device__ __forceinline__ float tree_halves(float v)
{
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return IS_MAX ? max_keep_nan(a, b) : a + b;
}

template <int D, int RW, int ST>
__global__ __launch_bounds__(256, RW == 1 ? 1 : 2) void terna_tree_attention_kernel(TreeAttention a)
{
    using Shape = TreeShape<D, RW, ST>;
    constexpr int KW = Shape::KW, KS = D / 16, DT = D / 32, TILE = Shape::kTile;
    constexpr int PIECES = D / 8, PER_LOAD = 64 / PIECES, LOADS = kTreeTile / RW / PER_LOAD;      // rows of a 1 KB load; loads of a wave and tile
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float2 stat[4][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = wave / RW, rw = wave % RW, qi = lane & 31, half = lane >> 5;
    // Workgroups go to the XCDs round robin: the row tiles of one (sequence, kv head, split) -- which read the same slots -- eight apart, on one XCD.
    const int G = a.H / a.KV, units = a.B * a.KV * a.splits;
    const int block = blockIdx.x / (8 * a.tiles), within = blockIdx.x - block * (8 * a.tiles);
    const int unit = 8 * block + (within & 7), tile = within >> 3;
    if (unit >= units) return;
    const int split = unit % a.splits, bk = unit / a.splits, kvh = bk % a.KV, b = bk / a.KV;

    // ---- rows
    const int rows = a.T * G, r = (tile * RW + rw) * 32 + qi;
    const bool real = r < rows;
    const int node = real ? r / G : 0, h = kvh * G + (real ? r - node * G : 0);
    const long long st64 = a.start[b];
    const unsigned long long* const mask = reinterpret_cast<const unsigned long long*>(a.mask) + (static_cast<size_t>(a.per_seq ? b : 0) * a.T + node) * a.W;
    const uint16_t* const qrow = a.q + b * a.q_seq + h * a.q_head + node * a.q_node;
    u32x4 q[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = *reinterpret_cast<const u32x4*>(qrow + 16 * ks + 8 * half);
    const int start = static_cast<int>(min(max(st64, 0ll), static_cast<long long>(a.S)));
    const int inside = min(a.T, a.S - start);                              // nodes that have a slot
    const unsigned long long first_word = mask[0];
    bool active = false, outside = false;                                  // the row has a node; sees a slot behind the cache
    for (int w = 0; w < a.W; ++w) {
        const unsigned long long bits = w == 0 ? first_word : mask[w];
        const int has = min(max(inside - 64 * w, 0), 64), in_tree = min(a.T - 64 * w, 64);
        const unsigned long long fit = has == 64 ? ~0ull : (1ull << has) - 1, valid = in_tree == 64 ? ~0ull : (1ull << in_tree) - 1;
        active |= (bits & valid) != 0;
        outside |= (bits & valid & ~fit) != 0;
    }
    active = active && real && st64 >= 0;
    outside = active && (outside || st64 > a.S);
    const int n = __syncthreads_or(active) ? start + inside : 0;           // slots that the workgroup reads
    const int all_tiles = (n + kTreeTile - 1) / kTreeTile, share = (all_tiles + a.splits - 1) / a.splits;
    const int begin = split * share, end = min(begin + share, all_tiles);
    const int steps = end > begin ? (end - begin + KW - 1) / KW : 0;       // of every group: a tile behind the end has no slot that counts

    // a negative scale's sign, and a scale of zero (0 * -inf would unmask a slot), go into the queries
    const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        if (a.scale < 0.0f) q[ks] ^= u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
        if (a.scale == 0.0f) {
            float x[8];
            unpack_bf16x8(q[ks], x);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= 0.0f;
            q[ks] = pack_bf16x8(x);
        }
        pin_registers(q[ks]);                                              // landed before the first hand-issued request
    }

    // ---- the cache's tiles
    const uint8_t* const kb = reinterpret_cast<const uint8_t*>(a.k + b * a.k_seq + kvh * a.k_head);
    const uint8_t* const vb = reinterpret_cast<const uint8_t*>(a.v + b * a.v_seq + kvh * a.v_head);
    uint8_t* const ring = smem + group * (ST * 2 * TILE);
    const uint32_t ring0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ring)) + rw * (LOADS * 1024);
    const int load_row = rw * (kTreeTile / RW) + lane / PIECES, piece = lane & (PIECES - 1);
    uint32_t k_at[LOADS], v_at[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        k_at[i] = tree_key_piece<D>(load_row + i * PER_LOAD, piece) << 4;
        v_at[i] = tree_value_piece<D>(load_row + i * PER_LOAD, piece) << 4;
    }
    auto slot_of = [&](int step) __attribute__((always_inline)) { return (begin + KW * step + group) * kTreeTile; };
    auto load = [&](int step, int at) __attribute__((always_inline)) {     // slots behind the last are read from its row
        const int k0 = min(slot_of(step), n - 1), left = n - 1 - k0;
        const uint8_t *const kt = kb + static_cast<long long>(k0) * a.k_slot, *const vt = vb + static_cast<long long>(k0) * a.v_slot;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t row = min(load_row + i * PER_LOAD, left);
            lds_dma_b128(kt, row * a.k_slot + k_at[i], ring0 + at * (2 * TILE) + i * 1024);
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t row = min(load_row + i * PER_LOAD, left);
            lds_dma_b128(vt, row * a.v_slot + v_at[i], ring0 + at * (2 * TILE) + TILE + i * 1024);
        }
    };
    int va[DT];
    const int vrow = 4 * half + ((lane & 15) >> 2);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) va[dt] = vrow * (2 * D) + (tree_value_piece<D>(vrow, 4 * dt + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) << 4) + 8 * (lane & 1);
    auto key_operand = [&](const uint8_t* keys, int ks) __attribute__((always_inline)) {
        return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(keys + qi * (2 * D) + (tree_key_piece<D>(qi, 2 * ks + half) << 4)));
    };
    auto value_operand = [&](const uint8_t* vals, int i, int dt) __attribute__((always_inline)) {       // 16 slots, 32 dimensions
        using Tr = tree_s16x4 __attribute__((address_space(3)))*;
        const u32x2 a0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(vals + va[dt] + i * 16 * 2 * D)));
        const u32x2 a1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(vals + va[dt] + (i * 16 + 8) * 2 * D)));
        return u32x4{a0.x, a0.y, a1.x, a1.y};
    };
    // bits of this row's mask for the 32 slots from k0 on: those in front of the tree are seen
    auto seen_bits = [&](int k0) __attribute__((always_inline)) {
        const int first = k0 - start;                                      // node of the tile's first slot
        uint32_t bits = 0;
        if (first < 0) bits = first <= -32 ? ~0u : (1u << -first) - 1;
        auto word = [&](int w) { return w < 0 || w >= a.W ? 0ull : w == 0 ? first_word : mask[w]; };
        if (first > -32 && first < inside) {
            const int w = first >> 6, by = first & 63;
            unsigned long long window = word(w) >> by;
            if (by != 0) window |= word(w + 1) << (64 - by);
            if (first < 0) window &= ~static_cast<unsigned long long>(bits);
            else window &= inside - first >= 32 ? ~0ull : (1ull << (inside - first)) - 1;
            if (first < 0 && inside - first < 32) window &= (1ull << (inside - first)) - 1;
            bits |= static_cast<uint32_t>(window);
        }
        return bits;
    };

    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[dt][v] = 0.0f;
    float m_run = -INFINITY, l_run = 0.0f;
    bool taken_out = false;                                                // a value that is not finite, among the tree's

    if (steps > 0) {
#pragma unroll
        for (int i = 0; i < ST - 1; ++i) load(i, i);
    }
    int at = 0;
    for (int step = 0; step < steps; ++step) {
        if constexpr (RW == 1) {
            // (this wave's reads of the tile that is overwritten have returned: the products took them)
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            load(step + ST - 1, at == 0 ? ST - 1 : at - 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 1) * 2 * LOADS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((ST - 2) * 2 * LOADS) : "memory");
            load(step + ST - 1, at == 0 ? ST - 1 : at - 1);
        }
        const uint8_t *const keys = ring + at * (2 * TILE), *const vals = keys + TILE;
        at = at + 1 == ST ? 0 : at + 1;
        const int k0 = slot_of(step);
        f32x16 s;
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(key_operand(keys, ks), __builtin_bit_cast(bf16x8, q[ks]), s, 0, 0, 0);
        const bool last_tiles = k0 + kTreeTile > start || k0 >= end * kTreeTile;
        if (last_tiles) {
            const uint32_t bits = k0 >= end * kTreeTile ? 0u : seen_bits(k0);
#pragma unroll
            for (int v = 0; v < 16; ++v)
                if (!(bits >> (8 * (v >> 2) + 4 * half + (v & 3)) & 1u)) s[v] = -INFINITY;
        }
        float top = tree_max3(tree_max3(s[0], s[1], s[2]), s[3], s[4]);
#pragma unroll
        for (int v = 5; v < 15; v += 2) top = tree_max3(top, s[v], s[v + 1]);
        top = tree_halves<true>(max_keep_nan(top, s[15])) * scale;
        if (__any(top > m_run + kTreeGrowth)) {
            const float m_new = top > m_run + kTreeGrowth ? top : m_run;   // a row by its own growth alone: its bits do not hang on the rows beside it
            const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
        }
        const float shift = m_run == -INFINITY ? 0.0f : -m_run;
        u32x4 p_hi[2], p_lo[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float p[8], high[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(__fmaf_rn(s[8 * i + e], scale, shift));
                l_run += p[e];
            }
            p_hi[i] = pack_bf16x8(p);
            unpack_bf16x8(p_hi[i], high);
#pragma unroll
            for (int e = 0; e < 8; ++e) high[e] = p[e] - high[e];
            p_lo[i] = pack_bf16x8(high);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                u32x4 x = value_operand(vals, i, dt);
                if (last_tiles) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {                          // exponents of ones: infinity or NaN
                        const bool low = (x[e] & 0x7f80u) == 0x7f80u, upper = (x[e] & 0x7f800000u) == 0x7f800000u;
                        taken_out |= low || upper;
                        x[e] &= (low ? 0u : 0xffffu) | (upper ? 0u : 0xffff0000u);
                    }
                }
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, p_hi[i]), o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, p_lo[i]), o[dt], 0, 0, 0);
            }
    }
    l_run = tree_halves<false>(l_run);
    if (__any(taken_out)) {                                                // rare: they are added where they are seen
        const int from = max(start / kTreeTile, begin);
        for (int k_tile = from; k_tile < end; ++k_tile) {
            if ((k_tile - begin) % KW != group) continue;
            const uint32_t bits = seen_bits(k_tile * kTreeTile);
            for (int j = 0; j < kTreeTile; ++j) {
                if (!(bits >> j & 1u)) continue;
                const uint16_t* const value = reinterpret_cast<const uint16_t*>(vb + static_cast<long long>(k_tile * kTreeTile + j) * a.v_slot);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int v = 0; v < 16; ++v) {
                        const uint16_t x = value[32 * dt + 8 * (v >> 2) + 4 * half + (v & 3)];
                        if ((x & 0x7f80u) == 0x7f80u) o[dt][v] += bf16_bits_to_float(x);
                    }
            }
        }
    }

    // ---- the groups' numerators, over their largest maximum
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");                // (requests behind the end too)
    float* const join = reinterpret_cast<float*>(smem);
    if (half == 0) stat[wave][qi] = float2{m_run, l_run};
    constexpr int ROW = Shape::kRow;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f32x4*>(join + (wave * 32 + qi) * ROW + 32 * dt + 8 * i + 4 * half) = f32x4{o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]};
    // (flags of a row, from the lane that has them to the threads that write it)
    const unsigned long long rows_outside = __ballot(outside), rows_active = __ballot(active);
    __shared__ uint32_t flags[RW][2];
    if (group == 0 && lane == 0) flags[rw][0] = static_cast<uint32_t>(rows_active), flags[rw][1] = static_cast<uint32_t>(rows_outside);
    __syncthreads();
    constexpr int STEP = 256 / PIECES;                                     // rows of the workgroup at a time, eight dimensions a thread
    const int dim = (tid & (PIECES - 1)) * 8;
#pragma unroll
    for (int row0 = 0; row0 < 32 * RW; row0 += STEP) {
        const int row = row0 + tid / PIECES, row_at = tile * 32 * RW + row, rwave = row >> 5, in_wave = row & 31;
        if (row_at >= rows) continue;
        const bool is_active = flags[rwave][0] >> in_wave & 1u, is_outside = flags[rwave][1] >> in_wave & 1u;
        float m = -INFINITY, l = 0.0f, weight[KW], x[8];
#pragma unroll
        for (int g = 0; g < KW; ++g) m = fmaxf(m, stat[g * RW + rwave][in_wave].x);
        const float m_use = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int g = 0; g < KW; ++g) {
            const float2 one = stat[g * RW + rwave][in_wave];
            weight[g] = KW == 1 ? 1.0f : __builtin_amdgcn_exp2f(one.x - m_use);
            l += one.y * weight[g];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.0f;
#pragma unroll
        for (int g = 0; g < KW; ++g) {
            const float* const from = join + ((g * RW + rwave) * 32 + in_wave) * ROW + dim;
            const f32x4 lower = *reinterpret_cast<const f32x4*>(from), upper = *reinterpret_cast<const f32x4*>(from + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += lower[e] * weight[g], x[4 + e] += upper[e] * weight[g];
        }
        const int of_node = row_at / G;
        const size_t out_row = (static_cast<size_t>(b) * a.T + of_node) * a.H + kvh * G + row_at - of_node * G;
        // nothing seen: zeros
        const float factor = is_outside ? NAN : !is_active || l == 0.0f ? 0.0f : a.splits > 1 ? 1.0f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = factor == 0.0f ? 0.0f : x[e] * factor;
        if (a.splits > 1) {
            float* const to = a.partial + (out_row * a.splits + split) * D + dim;
            *reinterpret_cast<f32x4*>(to) = f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4*>(to + 4) = f32x4{x[4], x[5], x[6], x[7]};
            if (dim == 0)
                *reinterpret_cast<float2*>(a.partial + static_cast<size_t>(a.B) * a.T * a.H * a.splits * D + (out_row * a.splits + split) * 2) =
                    is_outside ? float2{0.0f, 1.0f} : is_active ? float2{m, l} : float2{-INFINITY, 0.0f};
        } else {
            *reinterpret_cast<u32x4*>(a.out + out_row * D + dim) = pack_bf16x8(x);
        }
    }
}

// The splits' numerators over their largest maximum: a wave a row, D / 64 dimensions a lane.
template <int D>
__global__ __launch_bounds__(256) void terna_tree_merge_kernel(const float* __restrict__ partial, uint16_t* __restrict__ out, int rows, int splits)
{
    constexpr int E = D / 64, AHEAD = 8;
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= rows) return;
    const float* const x = partial + static_cast<size_t>(row) * splits * D + E * lane;
    const float2 one = lane < splits ? reinterpret_cast<const float2*>(partial + static_cast<size_t>(rows) * splits * D)[static_cast<size_t>(row) * splits + lane]
                                     : float2{-INFINITY, 0.0f};
    float m = one.x;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    const float weight = __builtin_amdgcn_exp2f(one.x - (m == -INFINITY ? 0.0f : m));
    float l = one.y * weight;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) l += __shfl_xor(l, off);
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.0f;
    for (int s0 = 0; s0 < splits; s0 += AHEAD) {
        float y[AHEAD][E];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) y[i][e] = x[static_cast<size_t>(min(s0 + i, splits - 1)) * D + e];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const float w = s0 + i < splits ? __shfl(weight, s0 + i) : 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] += w == 0.0f && s0 + i >= splits ? 0.0f : y[i][e] * w;
        }
    }
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
    if constexpr (E == 2) {
        *reinterpret_cast<uint32_t*>(out + static_cast<size_t>(row) * D + 2 * lane) = l == 0.0f ? 0u : pack_bf16x2(sum[0] * inverse, sum[1] * inverse);
    } else {
        out[static_cast<size_t>(row) * D + lane] = l == 0.0f ? static_cast<uint16_t>(0) : float_to_bf16_bits(sum[0] * inverse);
    }
}

}  // namespace terna
