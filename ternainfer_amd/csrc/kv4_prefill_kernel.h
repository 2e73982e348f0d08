// Attention of many query rows over the 4-bit cache (kv4_format.h): prompts and chunks of them.  The result of kv4_attention_kernel.h, laid out for the
// matrix cores' rate instead of memory's.
//
// A workgroup takes 128 rows of a kv head (row r = t * G + head) and all slots they see: eight waves, two groups of four; a wave has 32 rows, as the columns
// of 32x32x16 products, and every second tile of 64 slots; the two groups' halves are joined at the end.  (Two groups of four and not eight waves over 256
// rows, nor two workgroups of four: a causal triangle's longest rows last half as long, and a launch is as long as its last workgroup.)
//   * Matrix and vector work take turns: a group's turn of products -- the values of tile i, the scores of tile i + 1 -- falls into the other's turn of
//     softmax and conversions (a barrier a turn; every SIMD has a wave of each group).  In step, both groups wanted the same unit at the same time, and
//     the times of the two added up (3 x 500 tokens behind 8001 slots: 147 us, so 133).
//   * Values: converted (two an instruction, exact) into LDS by the group's four waves together and read back transposed; pieces of 16 bytes are
//     XOR-swizzled by row.  Keys: every wave converts its own from registers while products run -- through LDS they took as many of its clocks as the
//     values, more than there are.
//   * Values and probabilities are fp16: a value is a code times a power of two, exact in fp16 for scale bytes 104 .. 140 (2^-23 .. 2^13); probabilities keep 11 bits,
//     held at 2^12 for a row's maximum (up to 2^15 by what follows) so that those 2^-26 of it are still normal numbers.  A tile with any other scale
//     marks its workgroup, which starts again with bf16 values and probabilities in two bf16 -- the products twice.
//   * A row's running maximum is raised, and the output rescaled, only where it grows by more than 2^3 itself.
// Scales that stand for NaN and slots that a row does not see: as in kv4_attention_kernel.h.
#pragma once

#include "kv4_attention_kernel.h"

namespace terna {

constexpr int kKv4Tile = 64;                   // slots of a tile

template <int D>
struct Kv4PrefillLds {
    static constexpr int kTile = kKv4Tile * D * 2;                         // bytes of a tile's values
    static constexpr int kQueryStep = 64 * 16 + 32;                        // bytes from a piece of 64 half rows to the next: neither written nor read in conflict
    static constexpr int kNumerators = 2 * kKv4Rows * (D / 2) * 4, kOutRow = 2 * D + 16;
    static constexpr int kWork = 2 * kTile + 4 * (D / 16) * kQueryStep;    // the two groups' tiles and the queries; then half of the groups' numerators, then outputs
    static constexpr int kBytes = kWork > kNumerators ? kWork : kNumerators;
    static_assert(kBytes >= kKv4Rows * kOutRow, "outputs fit");
};

// max / sum over the lanes L, L ^ 32
template <bool IS_MAX>
__device__ __forceinline__ float halves_reduce(float v)
{
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return IS_MAX ? fmaxf(a, b) : a + b;
}

struct Kv4PrefillShared {
    float2 stat[2][kKv4Rows];
    int first_broken[4], wide_scales;
};

// The work of a workgroup; false where a value's scale does not fit fp16 (HALF), in every thread, with nothing written.
template <int D, bool HALF>
__device__ __forceinline__ bool kv4_prefill(const Kv4Attention& a, uint8_t* smem, Kv4PrefillShared& shared)
{
    constexpr float HELD = HALF ? kKv4HeldHalf : kKv4Held, GROWTH = HALF ? kKv4Growth : 0.0f;
    constexpr int KS = D / 16, DT = D / 32, GROUPS = D / kKv4Group, TILE = Kv4PrefillLds<D>::kTile;
    constexpr int WORDS = D / 32;                                          // words of codes of a thread: 8 * WORDS dimensions of a row
    auto& stat = shared.stat;
    auto& first_broken = shared.first_broken;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = wave >> 2, qi = lane & 31, half = lane >> 5;
    const int G = a.H / a.KV, rows = a.T * G;
    // Workgroups go to the XCDs round robin.  The row blocks of a (sequence, kv head, split) are dealt out in a.parts parts -- part c: c, c + parts, ... from
    // the last one down -- and an XCD takes a run of all parts, so that it reads few caches, from its L2, and walks them longest rows first.
    // (a.parts divides the blocks as evenly as eight or fewer can: a workgroup without work still takes a CU's place for a microsecond or two.)
    const int pairs = a.B * a.KV * a.splits, per_xcd = (pairs * a.parts + 7) / 8;
    const int slot = blockIdx.x >> 3, round = slot / per_xcd;
    const int unit = (blockIdx.x & 7) * per_xcd + slot - round * per_xcd, pair = unit / a.parts;
    const int from_last = a.parts * round + unit - pair * a.parts;
    if (pair >= pairs || from_last >= a.tiles) return true;
    const int first_row = (a.tiles - 1 - from_last) * kKv4Rows;
    const int split = pair % a.splits, bk = pair / a.splits, kvh = bk % a.KV, b = bk / a.KV;

    // ---- rows
    const int r = first_row + (wave & 3) * 32 + qi;
    const bool real = r < rows;
    const int t = real ? r / G : 0, h = kvh * G + (real ? r - t * G : 0);
    const long long p64 = a.pos[(a.per_seq ? b * a.T : 0) + t];

    // ---- cache
    const size_t base = (static_cast<size_t>(b) * a.KV + kvh) * a.S;
    const uint8_t *kb = a.k + base * (D / 2), *ksb = a.k_scale + base * GROUPS, *vb = a.v + base * (D / 2), *vsb = a.v_scale + base * GROUPS;
    const int tg = tid & 255, my_row = tg >> 2, part = tg & 3, my_group = part * GROUPS / 4;
    constexpr int KW = D / 16;                                             // words of key codes of a lane: half a row
    uint32_t k_codes[2][KW], k_bytes[2], v_codes[WORDS], v_byte;
    int begin = 0, end = 0;                                                // tiles of this split
    auto slot_of = [&](int step) __attribute__((always_inline)) { return (begin + 2 * step + group) * kKv4Tile; };
    auto load_keys = [&](int step, int i) __attribute__((always_inline)) { // a quarter of a row; the last with the scales
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t at = min(slot_of(step) + 32 * j + qi, a.S - 1);
            const u32x4 c = *reinterpret_cast<const u32x4*>(kb + static_cast<uint32_t>(at * (D / 2) + half * (D / 4) + 16 * i));
#pragma unroll
            for (int n = 0; n < 4; ++n) k_codes[j][4 * i + n] = c[n];
            if (i != KW / 4 - 1) continue;
            if constexpr (GROUPS == 4) k_bytes[j] = *reinterpret_cast<const uint16_t*>(ksb + static_cast<uint32_t>(at * GROUPS + 2 * half));
            else k_bytes[j] = ksb[static_cast<uint32_t>(at * GROUPS + half)];
        }
    };
    auto load_values = [&](int step) __attribute__((always_inline)) {
        const uint32_t at = min(slot_of(step) + my_row, a.S - 1);
        if constexpr (WORDS == 4) {
            const u32x4 c = *reinterpret_cast<const u32x4*>(vb + static_cast<uint32_t>(at * (D / 2) + part * 16));
#pragma unroll
            for (int i = 0; i < WORDS; ++i) v_codes[i] = c[i];
        } else {
            const u32x2 c = *reinterpret_cast<const u32x2*>(vb + static_cast<uint32_t>(at * (D / 2) + part * 8));
            v_codes[0] = c.x, v_codes[1] = c.y;
        }
        // (the row's four at once: of a byte the compiler wants to clear the rest, and waits for it too early)
        if constexpr (GROUPS == 4) v_byte = *reinterpret_cast<const uint32_t*>(vsb + static_cast<uint32_t>(at * GROUPS));
        else v_byte = vsb[static_cast<uint32_t>(at * GROUPS + my_group)];
    };
    // (in one piece, the first tile is known before the positions are)
    auto load_first = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KW / 4; ++i) load_keys(0, i);
        load_values(0);
    };
    if (a.splits == 1) load_first();
    // Queries of both groups in LDS, in the products' order: piece i of every row's half, then i + 1 32 bytes further than that (registers are short,
    // LDS's clocks are not).  Read as whole rows, 16 bytes a lane: a row at a lane took 5000 clocks of a workgroup's 8000 before its first product.
    uint8_t* const queries = smem + 2 * TILE + (wave & 3) * (KS * Kv4PrefillLds<D>::kQueryStep);
    {
        constexpr int LANES = D / 8, AT_ONCE = 64 / LANES, LOADS = 32 / AT_ONCE / 2;       // lanes of a row, rows of a load; the groups take a half each
        const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
        u32x4 x[LOADS];
#pragma unroll
        for (int n = 0; n < LOADS; ++n) {
            const int row = min(first_row + (wave & 3) * 32 + (group * LOADS + n) * AT_ONCE + lane / LANES, rows - 1), token = row / G;
            x[n] = *reinterpret_cast<const u32x4*>(a.q + ((static_cast<size_t>(b) * a.H + kvh * G + row - token * G) * a.T + token) * D + (lane & (LANES - 1)) * 8);
        }
#pragma unroll
        for (int n = 0; n < LOADS; ++n) {
            x[n] ^= u32x4{sign, sign, sign, sign};
            if (a.scale == 0.0f) {                                         // 0 * -inf would unmask a slot: the zero into the queries
                float y[8];
                RotaryVector<uint16_t>::unpack(x[n], y);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] *= 0.0f;
                x[n] = RotaryVector<uint16_t>::pack(y);
            }
            const int piece = lane & (LANES - 1), row = (group * LOADS + n) * AT_ONCE + lane / LANES;
            *reinterpret_cast<u32x4*>(queries + (piece & (KS - 1)) * Kv4PrefillLds<D>::kQueryStep + (piece / KS * 32 + row) * 16) = x[n];
        }
    }

    const bool outside = p64 >= a.S;
    const int my_last = !real || p64 < 0 ? -1 : outside ? a.S - 1 : static_cast<int>(p64);
    int n_keys = my_last + 1, n_full = real ? my_last + 1 : a.S;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        n_keys = max(n_keys, __shfl_xor(n_keys, off));
        n_full = min(n_full, __shfl_xor(n_full, off));
    }
    n_keys = __builtin_amdgcn_readfirstlane(n_keys);                       // of the wave
    n_full = __builtin_amdgcn_readfirstlane(n_full);
    if (lane == 0) stat[group][wave & 3] = float2{__int_as_float(n_keys), 0.0f};
    if (tid < GROUPS) first_broken[tid] = 0x7fffffff;
    if (tid == 0) shared.wide_scales = 0;
    __syncthreads();
    int all_keys = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) all_keys = max(all_keys, __float_as_int(stat[0][w].x));
    all_keys = __builtin_amdgcn_readfirstlane(all_keys);                   // of the workgroup
    const int all_tiles = (all_keys + kKv4Tile - 1) / kKv4Tile, share = (all_tiles + a.splits - 1) / a.splits;
    begin = split * share;
    end = min(begin + share, all_tiles);
    const int steps = (end - begin + 1) / 2;
    if (a.splits > 1) load_first();

    const int last = min(my_last, end * kKv4Tile - 1);                     // of this split
    n_full = min(n_full, end * kKv4Tile);

    const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale);

    uint8_t* const vals = smem + group * TILE;
    int va[DT];
    const int vrow = 4 * half + ((lane & 15) >> 2);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) va[dt] = kv4_piece<D>(vrow, 4 * dt + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 8 * (lane & 1);
    int broken = 0x7fffffff;
    bool wide = false;

    f32x16 o[DT];
    float m_run, l_run;
    auto write_values = [&](int step) __attribute__((always_inline)) {
        const int at = slot_of(step) + my_row;
        uint32_t byte = GROUPS == 4 ? v_byte >> (8 * my_group) & 255u : v_byte;
        if (at >= all_keys) byte = 127u;
        if (byte == kKv4Broken) {
            broken = min(broken, at);
            byte = 127u;
        }
        if (HALF) {
            uint32_t codes = v_codes[0];
#pragma unroll
            for (int i = 1; i < WORDS; ++i) codes |= v_codes[i];
            wide |= (byte < kKv4HalfLow || byte > kKv4HalfHigh) && (codes & kKv4Magnitudes) != 0;
            byte = min(byte, kKv4HalfHigh);
        } else {
            byte = min(byte, kKv4MaxByte);
        }
        const float vs = __uint_as_float(byte << 23);
#pragma unroll
        for (int i = 0; i < WORDS; ++i)
            *reinterpret_cast<u32x4*>(vals + kv4_piece<D>(my_row, part * WORDS + i)) = HALF ? kv4_values_half(v_codes[i], vs) : kv4_values(v_codes[i], vs);
    };
    f32x16 s[2];
    u32x4 p_hi[4], p_lo[4];
    auto key_operand = [&](int k) __attribute__((always_inline)) {         // k = 2 i + j: 32 slots, eight dimensions of each half
        const int j = k & 1, i = k >> 1;
        const float ks = __uint_as_float((GROUPS == 4 ? (i < KS / 2 ? k_bytes[j] & 255u : k_bytes[j] >> 8) : k_bytes[j]) << 23);
        return __builtin_bit_cast(bf16x8, kv4_values(k_codes[j][i], ks));
    };
    auto query_operand = [&](int i) __attribute__((always_inline)) {
        return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(queries + i * Kv4PrefillLds<D>::kQueryStep + lane * 16));
    };
    auto value_operand = [&](int k) __attribute__((always_inline)) {   // k = DT * n + dt: 16 slots, 32 dimensions
        using Tr = s16x4 __attribute__((address_space(3)))*;
        const int n = k / DT, dt = k & (DT - 1);
        const u32x2 a0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(vals + va[dt] + n * 16 * 2 * D)));
        const u32x2 a1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(vals + va[dt] + (n * 16 + 8) * 2 * D)));
        return u32x4{a0.x, a0.y, a1.x, a1.y};
    };
    // A turn of products in 2 KS (= 4 DT) slices, each a product of scores and one of outputs; operands are read two slices ahead, converted one
    // ahead, and the order is held: left to the compiler they were all read first, into more registers than there are.
    constexpr int SLICES = 2 * KS, AHEAD = 2;
    auto products = [&](auto with_outputs, int next) __attribute__((always_inline)) {   // next: the tile whose keys are requested in place of those used up
        constexpr bool OUT = decltype(with_outputs)::value;
        u32x4 vop[AHEAD + 1];
        bf16x8 kop[2], qop[2];
        if constexpr (OUT) {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) vop[k] = value_operand(k);
        }
        qop[0] = query_operand(0);
        qop[1] = query_operand(1);
        kop[0] = key_operand(0);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) s[j][v] = 0.0f;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < SLICES; ++k) {
            s[k & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kop[k & 1], qop[(k >> 1) & 1], s[k & 1], 0, 0, 0);
            if ((k & 1) && k / 2 + 2 < KS) qop[(k >> 1) & 1] = query_operand(k / 2 + 2);
            if constexpr (OUT) {
                if (k + AHEAD < SLICES) vop[(k + AHEAD) % (AHEAD + 1)] = value_operand(k + AHEAD);
            }
            if (k + 1 < SLICES) kop[(k + 1) & 1] = key_operand(k + 1);
            if constexpr (OUT) {
                const int n = k / DT, dt = k & (DT - 1);
                const u32x4 values = vop[k % (AHEAD + 1)];
                if constexpr (HALF) {
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, values), __builtin_bit_cast(f16x8, p_hi[n]), o[dt], 0, 0, 0);
                } else {
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, values), __builtin_bit_cast(bf16x8, p_hi[n]), o[dt], 0, 0, 0);
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, values), __builtin_bit_cast(bf16x8, p_lo[n]), o[dt], 0, 0, 0);
                }
            }
            if (KW == 8 && k == SLICES / 2) load_keys(next, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        load_keys(next, KW / 4 - 1);
    };
    auto softmax = [&](int k0) __attribute__((always_inline)) {
        if (k0 + kKv4Tile > n_full) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (k0 + 32 * j + 8 * (v >> 2) + 4 * half + (v & 3) > last) s[j][v] = -INFINITY;
        }
        float tops[4];                                                     // four chains: one would be sixteen instructions that wait for each other
#pragma unroll
        for (int c = 0; c < 4; ++c) tops[c] = kv4_max3(s[0][c], s[1][c], s[0][4 + c]);
#pragma unroll
        for (int v = 4; v < 12; v += 4)
#pragma unroll
            for (int c = 0; c < 4; ++c) tops[c] = kv4_max3(tops[c], s[1][v + c], s[0][v + 4 + c]);
#pragma unroll
        for (int c = 0; c < 4; c += 2) tops[c] = kv4_max3(tops[c], s[1][12 + c], s[1][13 + c]);
        float top = kv4_max3(kv4_max3(tops[0], tops[1], tops[2]), tops[3], -INFINITY);
        top = halves_reduce<true>(top) * scale;
        if (__any(top > m_run + GROWTH)) {
            const float m_new = top > m_run + GROWTH ? top : m_run;            // a row by its own growth alone: its bits do not hang on the rows beside it
            const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
        }
        const float shift = HELD - (m_run == -INFINITY ? 0.0f : m_run);
        float sum[2] = {0.0f, 0.0f};                                       // fp16: of the probabilities as the products take them, two an instruction
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                s[j][v] = __builtin_amdgcn_exp2f(__fmaf_rn(s[j][v], scale, shift));
                if constexpr (!HALF) sum[v & 1] += s[j][v];
            }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = s[n >> 1][8 * (n & 1) + e];
            if constexpr (HALF) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f16x2 pair = __builtin_convertvector((f32x2{p[2 * e], p[2 * e + 1]}), f16x2);
                    p_hi[n][e] = __builtin_bit_cast(uint32_t, pair);
                    sum[e & 1] = __builtin_amdgcn_fdot2(pair, f16x2{1, 1}, sum[e & 1], false);
                }
            } else {
                float back[8];
                p_hi[n] = RotaryVector<uint16_t>::pack(p);
                RotaryVector<uint16_t>::unpack(p_hi[n], back);
#pragma unroll
                for (int e = 0; e < 8; ++e) back[e] = p[e] - back[e];
                p_lo[n] = RotaryVector<uint16_t>::pack(back);
            }
        }
        l_run += sum[0] + sum[1];
    };
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[dt][v] = 0.0f;
    m_run = -INFINITY;
    l_run = 0.0f;
    // The end of a turn: what it has computed is computed here, not behind the barrier in the other group's turn of the same kind.
    auto turn_of_products_ends = [&]() __attribute__((always_inline)) {
        asm volatile("" : "+v"(s[0]), "+v"(s[1]));
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
    };
    auto turn_of_softmax_ends = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < 4; ++n) asm volatile("" : "+v"(p_hi[n]));
        if constexpr (!HALF) {
#pragma unroll
            for (int n = 0; n < 4; ++n) asm volatile("" : "+v"(p_lo[n]));
        }
        asm volatile("" : "+v"(l_run));
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
    };
    if (group == 1) __syncthreads();                                       // half a step behind
    products(std::false_type{}, 1);
    turn_of_products_ends();
    write_values(0);
    load_values(1);
    softmax(slot_of(0));
    turn_of_softmax_ends();
    for (int step = 1; step < steps; ++step) {
        __builtin_amdgcn_s_setprio(1);
        products(std::true_type{}, step + 1);
        __builtin_amdgcn_s_setprio(0);
        turn_of_products_ends();
        write_values(step);
        load_values(step + 1);
        softmax(slot_of(step));
        turn_of_softmax_ends();
    }
    products(std::true_type{}, steps);                                     // (and scores of a tile behind the end, which nobody reads)
    __syncthreads();
    if (group == 0) __syncthreads();
    l_run = halves_reduce<false>(l_run);
    m_run -= HELD;                                                     // what the probabilities are relative to: the splits of a row may differ in it
    if (HALF && wide) shared.wide_scales = 1;
    __syncthreads();
    if (HALF && shared.wide_scales) return false;                          // (all have read it behind the barrier; nobody writes it before the next)

    // ---- the two groups: each finishes half of the dimensions, with the other's numerators from LDS
    if (broken != 0x7fffffff) atomicMin(&first_broken[my_group], broken);
    const int row_at = (wave & 3) * 32 + qi;
    if (half == 0) stat[group][row_at] = float2{m_run, l_run};
    f32x4* const given = reinterpret_cast<f32x4*>(smem) + group * (kKv4Rows * D / 8);       // [piece of 4 dimensions][row]: D / 8 pieces
    const int keep = group == 0 ? 0 : DT / 2;
#pragma unroll
    for (int dt = 0; dt < DT / 2; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f32x4 x;
#pragma unroll
            for (int v = 0; v < 4; ++v) x[v] = group == 0 ? o[DT / 2 + dt][4 * i + v] : o[dt][4 * i + v];
            given[(8 * dt + 2 * i + half) * kKv4Rows + row_at] = x;
        }
    __syncthreads();
    const f32x4* const got = reinterpret_cast<const f32x4*>(smem) + (1 - group) * (kKv4Rows * D / 8);
    const float2 one = stat[0][row_at], two = stat[1][row_at];
    const float m = fmaxf(one.x, two.x), m_use = m == -INFINITY ? 0.0f : m;
    const float w0 = __builtin_amdgcn_exp2f(one.x - m_use), w1 = __builtin_amdgcn_exp2f(two.x - m_use);
    const float l = one.y * w0 + two.y * w1, w_mine = group == 0 ? w0 : w1, w_other = group == 0 ? w1 : w0;
    const size_t out_row = (static_cast<size_t>(b) * a.T + t) * a.H + h;
    const float inverse = a.splits > 1 ? 1.0f : p64 < 0 ? 0.0f : 1.0f / l;
    auto numerators = [&](int dt, int i) __attribute__((always_inline)) {  // 32 dimensions share a scale: one NaN for all of them
        const bool nan = outside || (p64 >= 0 && p64 >= first_broken[keep + dt]);
        const float mine = nan ? NAN : w_mine * inverse, others = w_other * inverse;
        const f32x4 other = got[(8 * dt + 2 * i + half) * kKv4Rows + row_at];
        f32x4 x;
#pragma unroll
        for (int v = 0; v < 4; ++v) x[v] = (group == 0 ? o[dt][4 * i + v] : o[DT / 2 + dt][4 * i + v]) * mine + other[v] * others;
        return x;
    };
    if (a.splits > 1) {
        if (!real) return true;
        if (group == 0 && half == 0)
            *reinterpret_cast<float2*>(a.partial + static_cast<size_t>(a.B) * a.T * a.H * a.splits * D + (out_row * a.splits + split) * 2) = float2{m, l};
#pragma unroll
        for (int dt = 0; dt < DT / 2; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(a.partial + (out_row * a.splits + split) * D + 32 * (keep + dt) + 8 * i + 4 * half) = numerators(dt, i);
        return true;
    }
    u32x2 rounded[DT / 2][4];
#pragma unroll
    for (int dt = 0; dt < DT / 2; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 x = numerators(dt, i);
            rounded[dt][i] = u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
        }
    // through LDS into whole rows, 16 bytes a lane
    __syncthreads();
    uint8_t* const out_rows = smem + (wave & 3) * (32 * Kv4PrefillLds<D>::kOutRow);
#pragma unroll
    for (int dt = 0; dt < DT / 2; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x2*>(out_rows + qi * Kv4PrefillLds<D>::kOutRow + (32 * (keep + dt) + 8 * i + 4 * half) * 2) = rounded[dt][i];
    __syncthreads();
    constexpr int LANES = D / 8, AT_ONCE = 64 / LANES, STORES = 32 / AT_ONCE / 2;
#pragma unroll
    for (int n = 0; n < STORES; ++n) {
        const int in_wave = (group * STORES + n) * AT_ONCE + lane / LANES, row = first_row + (wave & 3) * 32 + in_wave;
        if (row < rows) {
            const int token = row / G;
            *reinterpret_cast<u32x4*>(a.out + ((static_cast<size_t>(b) * a.T + token) * a.H + kvh * G + row - token * G) * D + (lane & (LANES - 1)) * 8) =
                *reinterpret_cast<const u32x4*>(out_rows + in_wave * Kv4PrefillLds<D>::kOutRow + (lane & (LANES - 1)) * 16);
        }
    }
    return true;
}

// (a function of its own: its registers are not the other's)
template <int D>
__device__ __attribute__((noinline)) void kv4_prefill_any_scale(Kv4Attention a, uint8_t* smem, Kv4PrefillShared& shared)
{
    __syncthreads();
    kv4_prefill<D, false>(a, smem, shared);
}

template <int D>
__global__ __launch_bounds__(512, 2) void terna_kv4_prefill_kernel(Kv4Attention a)
{
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Kv4PrefillShared shared;
    if (!kv4_prefill<D, true>(a, smem, shared)) kv4_prefill_any_scale<D>(a, smem, shared);
}

}  // namespace terna
