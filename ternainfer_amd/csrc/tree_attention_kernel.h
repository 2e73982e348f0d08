// Attention of a tree of drafted tokens over the cache: node i of a sequence sees the slots in front of the tree and, of the tree's own (node j in slot
// start + j), those of its mask.
//
//   out[row] = sum_s p_s v_s / sum_s p_s,  p_s = exp(scale q . k_s - max)
//
// The rows of a kv head -- its G = H / KV query heads times the nodes, row r = node * G + head -- are the columns of 32x32x16 products, 32 a wave: the scores
// (slots x rows) come out of the matrix cores in the layout in which their exponentials go back in as the second product's operand, and a row's maximum
// and sum are one exchange between two lanes.
//   * RW waves of a workgroup share the slots, 32 rows each, and KW groups of those take turns of 32 slots, so that a few rows still read a cache with four waves
//     and many leave few numerators to join.  The groups' are joined in LDS at the end, the splits' by a second launch (which groups, how many splits: tree_plan.h).
//   * Keys and values go global -> LDS directly, ST - 1 steps ahead; 16-byte pieces are XOR-swizzled on the way, so that neither the keys' 16-byte operand reads
//     nor the values' transposing ones conflict.  A wave that shares its slots with nobody waits for its own requests only.
//     With 128 rows a workgroup the next step's keys are read ahead of this one's exponentials (measured with probabilities in one bf16: 800 rows over 8300 slots 65.2 us, so 63.6; now 76).
//   * Probabilities are two bf16, high and low part: 15 bits of them count.  One bf16 is 2^-9 of every term, which shows where large values nearly cancel: two slots
//     with half of the weight each and values of 200 and -200 came out 0.3 off, for 10 % less time with more than 64 rows a kv head (60 nodes of 4 heads over 32001 slots 40.0 us, so 43.3 to 45.4).
//     The running maximum is raised, and the output rescaled, only where it grows by more than 2^3 -- a row's own.
//   * Only the last tiles have slots of the tree.  There the mask's bits select the scores, and values that are not finite are taken out -- a slot that
//     one node sees and another does not must not reach the other through 0 * NaN; the rows that do see them get them back at the end.
// What bounds it: of few rows a sequence and many sequences the cache's bytes (64 sequences of one token over 8000 slots 229 us, 5.7 TB/s; 32 of 13 nodes over
// 7500 119 us, 4.9), of many rows the steps -- 64 slots of 128 rows in two groups: 1536 clocks of a SIMD's matrix instructions, 1450 of its vector
// instructions, 128 KB of LDS reads; 1.0 to 1.15 us where nothing comes from memory, 1.5 to 1.6 where all does, of which two workgroups that share their slots need 0.9 for
// the memory alone -- and with little to read what surrounds the steps: 3 us until the first tile is there, 3.5 for the join in LDS and the rows' way out, 4 to 5 for the
// second launch.
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
    float* partial;                            // more than one part a sequence: fp32 [parts][T * H][D] numerators, [parts][T * H][2] maximum and sum, then TreeShare [B]
    long long q_seq, q_head, q_node;           // strides, elements
    long long k_seq, k_head, v_seq, v_head;
    int k_slot, v_slot;                        // ... of a slot, bytes
    int B, T, H, KV, S, W, parts, tiles, per_seq;       // parts: of all sequences together, 0 where none is split
    float scale;                               // times log2(e)
};

// A sequence's parts: the first of them, and how many.
struct TreeShare {
    int first, count;
};

// A workgroup's shape: KW groups of RW waves that share the slots, 32 query rows each; ST tiles of keys and values in each group's ring.
template <int D, int RW, int KW, int ST>
struct TreeShape {
    static constexpr int kWaves = RW * KW, kThreads = 64 * kWaves;
    static constexpr int kTile = kTreeTile * D * 2;                        // bytes of a tile's keys, or values
    static constexpr int kRing = KW * ST * 2 * kTile;
    static constexpr int kRow = D + 4;                                     // floats of a row of numerators in LDS
    static constexpr int kJoin = kWaves * 32 * kRow * 4;
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

// Which part of which sequence a workgroup takes.  The parts that the launch has room for are dealt out by the sequences' lengths, all at most `longest` tiles long, the
// shortest such length within an eighth: with as many for each, the longest sequence's would last longest (8 sequences of 1670 to 4001 slots: 33 us, so 30).
// Every wave works it out, a sequence a lane.
struct TreePart {
    int b, start, split;                       // b < 0: none; start: -1 for a sequence without a tree, S + 1 for one behind the cache
    TreeShare share;
};
__device__ __forceinline__ uint32_t tree_wave_sum(uint32_t x)
{
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off);
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ TreePart tree_part(const TreeAttention& a, int part)
{
    const int lane = threadIdx.x & 63;
    auto start_of = [&](int b) { return static_cast<int>(min(max(a.start[b], -1ll), a.S + 1ll)); };
    auto tiles_of = [&](int start) { return start < 0 ? 0u : static_cast<uint32_t>(min(start + a.T, a.S) + kTreeTile - 1) / kTreeTile; };
    TreePart p;
    if (a.parts == 0) {
        p.b = part, p.start = start_of(part), p.split = 0, p.share = TreeShare{part, 1};
        return p;
    }
    if (a.B == 1) {
        p.b = part < kTreeMaxSplits ? 0 : -1, p.start = start_of(0), p.split = part, p.share = TreeShare{0, min(a.parts, kTreeMaxSplits)};
        return p;
    }
    int start = lane < a.B ? start_of(lane) : -1;
    auto start_at = [&](int b0) { return b0 == 0 && a.B <= 64 ? start : b0 + lane < a.B ? start_of(b0 + lane) : -1; };
    auto count_of = [&](int b, int start, uint32_t longest) {              // (a sequence has one at least)
        return b < a.B ? min(max((tiles_of(start) + longest - 1) / longest, 1u), static_cast<uint32_t>(kTreeMaxSplits)) : 0u;
    };
    uint32_t all = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) all += tree_wave_sum(tiles_of(start_at(b0)));
    const uint32_t parts = static_cast<uint32_t>(a.parts);
    // (at all / (parts - B), rounded up, they certainly fit)
    for (uint32_t longest = max((all + parts - 1) / parts, 1u);; longest += max(longest / 8, 1u)) {
        uint32_t total = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) total += tree_wave_sum(count_of(b0 + lane, start_at(b0), longest));
        if (total > parts) continue;
        int before = 0;
        p.b = -1;
        for (int b0 = 0; b0 < a.B && p.b < 0; b0 += 64) {
            const int at = start_at(b0), count = count_of(b0 + lane, at, longest);
            int upto = count;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int x = __shfl_up(upto, off);
                if (lane >= off) upto += x;
            }
            const int first = before + upto - count;
            const unsigned long long found = __ballot(part >= first && part < first + count);
            if (found != 0) {
                const int who = __builtin_ctzll(found);
                p.b = b0 + who, p.start = __builtin_amdgcn_readlane(at, who);
                p.share = TreeShare{__builtin_amdgcn_readlane(first, who), __builtin_amdgcn_readlane(count, who)};
                p.split = part - p.share.first;
            }
            before += __builtin_amdgcn_readlane(upto, 63);
        }
        return p;
    }
}

template <int D, int RW, int KW, int ST, int PER_SIMD>
__global__ __launch_bounds__(64 * RW * KW, PER_SIMD) void terna_tree_attention_kernel(TreeAttention a)
{
    static_assert(ST == 2 || ST == 4);
    using Shape = TreeShape<D, RW, KW, ST>;
    constexpr int KS = D / 16, DT = D / 32, TILE = Shape::kTile;
    constexpr int PIECES = D / 8, PER_LOAD = 64 / PIECES, PER_TILE = TILE / 1024, LOADS = 2 * PER_TILE / RW;       // rows of a 1 KB load; loads of a tile's keys; of a wave and step
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float2 stat[Shape::kWaves][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = wave / RW, rw = wave % RW, qi = lane & 31, half = lane >> 5;
    const int G = a.H / a.KV;
    const TreePlace place_of = tree_place(blockIdx.x, (a.parts == 0 ? a.B : a.parts) * a.KV, a.tiles);
    if (place_of.unit < 0) return;
    const int unit = place_of.unit, tile = place_of.tile;
    const int kvh = unit % a.KV;
    const TreePart part = tree_part(a, unit / a.KV);
    if (part.b < 0) return;
    const int b = part.b, splits = part.share.count;

    // ---- rows
    const int rows = a.T * G, start = min(max(part.start, 0), a.S), inside = min(a.T, a.S - start);        // inside: nodes that have a slot
    const int r = (tile * RW + rw) * 32 + qi, node = r < rows ? r / G : 0, h = kvh * G + (r < rows ? r - node * G : 0);
    const unsigned long long* const mask = reinterpret_cast<const unsigned long long*>(a.mask) + (static_cast<size_t>(a.per_seq ? b : 0) * a.T + node) * a.W;
    const unsigned long long first_word = mask[0];
    u32x4 q[KS];
    {
        const uint16_t* const row = a.q + b * a.q_seq + h * a.q_head + node * a.q_node;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) q[ks] = *reinterpret_cast<const u32x4*>(row + 16 * ks + 8 * half);
    }
    // ---- the cache's tiles
    const int n = part.start < 0 ? 0 : start + inside;                     // slots that the workgroup reads
    const int all_tiles = (n + kTreeTile - 1) / kTreeTile, share = (all_tiles + splits - 1) / splits;
    const int begin = part.split * share, end = min(begin + share, all_tiles);
    const int all_steps = end > begin ? (end - begin + KW - 1) / KW : 0;   // of every group: a tile behind the end has no slot that counts
    const uint8_t* const kb = reinterpret_cast<const uint8_t*>(a.k + b * a.k_seq + kvh * a.k_head);
    const uint8_t* const vb = reinterpret_cast<const uint8_t*>(a.v + b * a.v_seq + kvh * a.v_head);
    uint8_t* const ring = smem + group * (ST * 2 * TILE);
    const uint32_t ring0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ring)) + rw * 1024;
    // Of a step's loads a wave has those rw, rw + RW, ...: first the keys', then the values'.
    int load_row[LOADS];
    uint32_t load_piece[LOADS], load_at[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int l = rw + RW * i;
        load_row[i] = (l % PER_TILE) * PER_LOAD + lane / PIECES;
        load_piece[i] = (l < PER_TILE ? tree_key_piece<D>(load_row[i], lane & (PIECES - 1)) : tree_value_piece<D>(load_row[i], lane & (PIECES - 1))) << 4;
        load_at[i] = static_cast<uint32_t>(load_row[i] * (l < PER_TILE ? a.k_slot : a.v_slot)) + load_piece[i];
    }
    auto slot_of = [&](int step) __attribute__((always_inline)) { return (begin + KW * step + group) * kTreeTile; };
    // a step's keys and values into their place of the ring; slots behind the last are read from its row
    auto load = [&](int step, int at) __attribute__((always_inline)) {
        const int k0 = min(slot_of(step), n - 1), left = n - 1 - k0;
        const uint8_t *const kt = kb + static_cast<long long>(k0) * a.k_slot, *const vt = vb + static_cast<long long>(k0) * a.v_slot;
        const uint32_t to = ring0 + at * (2 * TILE);
        if (left >= kTreeTile - 1) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) lds_dma_b128(rw + RW * i < PER_TILE ? kt : vt, load_at[i], to + i * (RW * 1024));
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const bool keys = rw + RW * i < PER_TILE;
                lds_dma_b128(keys ? kt : vt, static_cast<uint32_t>(min(load_row[i], left) * (keys ? a.k_slot : a.v_slot)) + load_piece[i], to + i * (RW * 1024));
            }
        }
    };
    if (all_steps > 0) load(0, 0);                                         // on its way while the masks are looked at

    bool active = false, outside = part.start > a.S;                       // the row has a node; sees a slot behind the cache
    for (int w = 0; w < a.W; ++w) {
        const unsigned long long bits = w == 0 ? first_word : mask[w];
        const int has = min(max(inside - 64 * w, 0), 64), in_tree = min(a.T - 64 * w, 64);
        const unsigned long long fit = has == 64 ? ~0ull : (1ull << has) - 1, valid = in_tree == 64 ? ~0ull : (1ull << in_tree) - 1;
        active |= (bits & valid) != 0;
        outside |= (bits & valid & ~fit) != 0;
    }
    active = active && r < rows && part.start >= 0;
    outside = outside && active;
    const bool needed = __syncthreads_or(active);
    const int steps = !needed ? 0 : RW == 1 ? max(end - begin - group + KW - 1, 0) / KW : all_steps;      // (groups that wait for each other make as many)

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
        pin_registers(q[ks]);                                              // landed before the next hand-issued request
    }

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
    // bits of a row's mask for the 32 slots from k0 on: those in front of the tree are seen
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
    bool taken_out = false;                                                // a value that is not finite, among the tree's

    // Infinities and NaN -- exponents of ones -- out of pieces of values, remembered.  There are hardly ever any: one look at all of them.
    auto finite = [&](u32x4* x, int pieces) __attribute__((always_inline)) {
        typedef unsigned short two __attribute__((ext_vector_type(2)));
        two most{0, 0};
#pragma unroll
        for (int i = 0; i < pieces; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) most = __builtin_elementwise_max(most, __builtin_bit_cast(two, x[i][e] & 0x7fff7fffu));
        const bool broken = most.x >= 0x7f80u || most.y >= 0x7f80u;
        if (!__any(broken)) return;
        taken_out |= broken;
#pragma unroll
        for (int i = 0; i < pieces; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[i][e] &= ((x[i][e] & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) | ((x[i][e] & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u);
    };
    auto unseen = [&](f32x16& s, int k0) __attribute__((always_inline)) {
        const uint32_t bits = k0 >= end * kTreeTile ? 0u : seen_bits(k0);
#pragma unroll
        for (int v = 0; v < 16; ++v)
            if (!(bits >> (8 * (v >> 2) + 4 * half + (v & 3)) & 1u)) s[v] = -INFINITY;
    };
    auto largest = [&](const f32x16& s) __attribute__((always_inline)) {
        float tops[2] = {tree_max3(s[0], s[1], s[2]), tree_max3(s[3], s[4], s[5])};
#pragma unroll
        for (int v = 6; v < 14; v += 4) {
            tops[0] = tree_max3(tops[0], s[v], s[v + 1]);
            tops[1] = tree_max3(tops[1], s[v + 2], s[v + 3]);
        }
        return tree_max3(tree_max3(tops[0], tops[1], s[14]), s[15], s[15]);
    };
    float l_run = 0.0f, m_run = -INFINITY;
    // this group's steps whose tiles lie in front of the tree
    const int plain = needed ? max(min(start / kTreeTile, end) - begin - group + KW - 1, 0) / KW : 0;
    int at = 0;                                                            // place in the ring
    bf16x8 key[KS];
    auto take = [&](int step, auto last_tiles, auto place) __attribute__((always_inline)) {
        constexpr bool LAST = decltype(last_tiles)::value;                 // may have slots of the tree, or behind the end
        constexpr int PLACE = decltype(place)::value;                      // known: offsets that instructions carry; -1: `at`
        const int here = PLACE < 0 ? at : PLACE, behind = PLACE < 0 ? (at == 0 ? ST - 1 : at - 1) : (PLACE + ST - 1) % ST;
        if constexpr (RW == 1) {
            // (this wave's reads of the tile that is overwritten have returned: the products took them)
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            load(step + ST - 1, behind);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 1) * LOADS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((RW == 4 ? ST - 3 : ST - 2) * LOADS) : "memory");
            load(step + ST - 1, behind);
        }
        const uint8_t *const keys = ring + here * (2 * TILE), *const vals = keys + TILE;
        if constexpr (PLACE < 0) at = at + 1 == ST ? 0 : at + 1;
        f32x16 s;
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(RW == 4 ? key[ks] : key_operand(keys, ks), __builtin_bit_cast(bf16x8, q[ks]), s, 0, 0, 0);
        if constexpr (RW == 4) {
            const uint8_t* const ahead = ring + (PLACE < 0 ? at : (PLACE + 1) % ST) * (2 * TILE);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) key[ks] = key_operand(ahead, ks);
        }
        if constexpr (LAST) unseen(s, slot_of(step));
        const float top = tree_halves<true>(largest(s)) * scale;
        const bool more = top > m_run + kTreeGrowth;                // a row by its own growth alone: its bits do not hang on the rows beside it
        if (__any(more)) {
            const float m_new = more ? top : m_run;
            const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
        }
        const float shift = m_run == -INFINITY ? 0.0f : -m_run;
        float sum[2] = {0.0f, 0.0f};
        u32x4 high[2], low[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(__fmaf_rn(s[8 * i + e], scale, shift));
            // high: the upper 16 bits as they are; low: the rest and 2^-20 of the whole, so that it is positive and an infinite value stays one in both products
            float rest[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sum[e & 1] += p[e];
                rest[e] = __fmaf_rn(p[e], 1.0f + 0x1p-20f, -__uint_as_float(__float_as_uint(p[e]) & 0xffff0000u));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) high[i][e] = __builtin_amdgcn_perm(__float_as_uint(p[2 * e + 1]), __float_as_uint(p[2 * e]), 0x07060302u);
            low[i] = pack_bf16x8(rest);
        }
        l_run += sum[0] + sum[1];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            u32x4 x[DT];
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) x[dt] = value_operand(vals, i, dt);
            if constexpr (LAST) finite(x, DT);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const bf16x8 y = __builtin_bit_cast(bf16x8, x[dt]);
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y, __builtin_bit_cast(bf16x8, high[i]), o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y, __builtin_bit_cast(bf16x8, low[i]), o[dt], 0, 0, 0);
            }
        }
    };
    if (steps > 0) {
#pragma unroll
        for (int i = 1; i < ST - 1; ++i) load(i, i);
    }
    if constexpr (RW == 4) {
        if (steps > 0) {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((ST - 2) * LOADS) : "memory");
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) key[ks] = key_operand(ring, ks);
        }
    }
    using Anywhere = std::integral_constant<int, -1>;
    int step = 0;
    for (; step + ST <= plain; step += ST) {
        take(step, std::false_type{}, std::integral_constant<int, 0>{});
        take(step + 1, std::false_type{}, std::integral_constant<int, 1>{});
        if constexpr (ST > 2) {
            take(step + 2, std::false_type{}, std::integral_constant<int, 2>{});
            take(step + 3, std::false_type{}, std::integral_constant<int, 3>{});
        }
    }
    for (; step < plain; ++step) take(step, std::false_type{}, Anywhere{});
    for (; step < steps; ++step) take(step, std::true_type{}, Anywhere{});
    l_run = tree_halves<false>(l_run);
    if (m_run == INFINITY) l_run = NAN;                                    // a score above what fp32 holds: NaN, not a row that sees nothing
    if (__any(taken_out)) {                                                // rare: they are added where they are seen
        const int from = max(min(start / kTreeTile, end) - KW, begin);     // (whatever tile it can have been; added twice, they are what they were)
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

    if (a.parts != 0 && part.split == 0 && kvh == 0 && tile == 0 && tid == 0)
        reinterpret_cast<TreeShare*>(a.partial + static_cast<size_t>(a.parts) * a.T * a.H * (D + 2))[b] = part.share;

    // ---- the groups' numerators, over their largest maximum
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");                // (requests behind the end too)
    float* const join = reinterpret_cast<float*>(smem);
    constexpr int ROW = Shape::kRow;
    __shared__ uint32_t flags[RW][2];                                      // of a row, from the lane that has them to the threads that write it
    if (half == 0) stat[wave][qi] = float2{m_run, l_run};
    const unsigned long long rows_outside = __ballot(outside), rows_active = __ballot(active);
    if (group == 0 && lane == 0) flags[rw][0] = static_cast<uint32_t>(rows_active), flags[rw][1] = static_cast<uint32_t>(rows_outside);
    constexpr int EIGHTS = D / 8, STEP = Shape::kThreads / EIGHTS;               // of a row; rows of the workgroup at a time, eight dimensions a thread
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x16& x = o[dt];
            *reinterpret_cast<f32x4*>(join + (wave * 32 + qi) * ROW + 32 * dt + 8 * i + 4 * half) = f32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
        }
    __syncthreads();
    const int dim = (tid & (EIGHTS - 1)) * 8;
#pragma unroll
    for (int row0 = 0; row0 < 32 * RW; row0 += STEP) {
        const int row = row0 + tid / EIGHTS, row_at = tile * (32 * RW) + row, rwave = row >> 5, in_wave = row & 31;
        if ((STEP > 32 * RW && row >= 32 * RW) || row_at >= rows) continue;
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
        const float factor = is_outside ? NAN : !is_active || l == 0.0f ? 0.0f : splits > 1 ? 1.0f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = factor == 0.0f ? 0.0f : x[e] * factor;
        if (splits > 1) {
            const size_t all = static_cast<size_t>(a.T) * a.H, at = (part.share.first + part.split) * all + (out_row - b * all);
            float* const to = a.partial + at * D + dim;
            *reinterpret_cast<f32x4*>(to) = f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4*>(to + 4) = f32x4{x[4], x[5], x[6], x[7]};
            if (dim == 0)
                reinterpret_cast<float2*>(a.partial + a.parts * all * D)[at] = is_outside ? float2{0.0f, 1.0f} : is_active ? float2{m, l} : float2{-INFINITY, 0.0f};
        } else {
            *reinterpret_cast<u32x4*>(a.out + out_row * D + dim) = pack_bf16x8(x);
        }
    }
}

// The parts' numerators of the sequences that have several, over their largest maximum: a wave a row, four dimensions a lane, so that two or four parts are read side by
// side; the first of them on their way before their weights are known.
template <int D>
__global__ __launch_bounds__(256) void terna_tree_merge_kernel(const float* __restrict__ partial, uint16_t* __restrict__ out, int B, int rows, int parts)
{
    constexpr int LANES = D / 4, BESIDE = 64 / LANES, AHEAD = 8;           // lanes of a part; parts side by side; of a lane, in flight
    const int lane = threadIdx.x & 63, at = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (at >= B * rows) return;
    const int b = at / rows, row = at - b * rows;                          // rows: of a sequence
    const size_t all = static_cast<size_t>(parts) * rows;
    const TreeShare share = B == 1 ? TreeShare{0, min(parts, kTreeMaxSplits)} : reinterpret_cast<const TreeShare*>(partial + all * (D + 2))[b];
    if (share.count == 1) return;                                          // written by its workgroups
    const int which = lane / LANES, piece = lane & (LANES - 1);
    const float* const x = partial + (static_cast<size_t>(share.first) * rows + row) * D + 4 * piece;
    f32x4 y[AHEAD];
    auto fetch = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) y[i] = *reinterpret_cast<const f32x4*>(x + static_cast<size_t>(min(s0 + i * BESIDE + which, share.count - 1)) * rows * D);
    };
    const float2 one = lane < share.count ? reinterpret_cast<const float2*>(partial + all * D)[static_cast<size_t>(share.first + lane) * rows + row] : float2{-INFINITY, 0.0f};
    fetch(0);
    float m = one.x;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    const float weight = __builtin_amdgcn_exp2f(one.x - (m == -INFINITY ? 0.0f : m));
    float l = one.y * weight;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) l += __shfl_xor(l, off);
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0;;) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int part = s0 + i * BESIDE + which;
            const float w = __shfl(weight, min(part, share.count - 1));
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += part < share.count ? y[i][e] * w : 0.0f;
        }
        s0 += AHEAD * BESIDE;
        if (s0 >= share.count) break;
        fetch(s0);
    }
#pragma unroll
    for (int off = LANES; off < 64; off *= 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], off);
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
    if (which != 0) return;
    *reinterpret_cast<u32x2*>(out + static_cast<size_t>(at) * D + 4 * piece) =
        l == 0.0f ? u32x2{0u, 0u} : u32x2{pack_bf16x2(sum[0] * inverse, sum[1] * inverse), pack_bf16x2(sum[2] * inverse, sum[3] * inverse)};
}

}  // namespace terna
