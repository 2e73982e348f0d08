// Attention of many query rows over the 4-bit cache (kv4_format.h): prompts and chunks of them.  The result of kv4_attention_kernel.h, laid out for the
// matrix cores' rate instead of memory's.
//
// A workgroup takes 128 rows of a kv head (row r = t * G + head) and all slots they see: eight waves, two groups of four; a wave has 32 rows, as the columns
// of 32x32x16 products, and every second tile of 64 slots; the two groups' halves are joined at the end.  (Two groups of four and not eight waves over 256
// rows, nor two workgroups of four: a causal triangle's longest rows last half as long, and a launch is as long as its last workgroup.)
//   * Codes go to registers two tiles ahead, converted (two values an instruction, exact) into LDS one tile ahead, where the four waves of the group share
//     them: keys as bf16, 16-byte pieces XOR-swizzled by row; values swizzled for transposing reads.  One barrier a tile.
//   * Values and probabilities are fp16: a value is a code times a power of two, exact in fp16 for scale bytes 104 .. 140 (2^-23 .. 2^13); probabilities keep 11 bits,
//     held at 2^12 for a row's maximum (up to 2^15 by what follows) so that those 2^-26 of it are still normal numbers.  A tile with any other scale
//     marks its workgroup, which starts again with bf16 values and probabilities in two bf16 -- the products twice.
//   * A row's running maximum is raised, and the output rescaled, only where it grows by more than 2^3.
// Scales that stand for NaN and slots that a row does not see: as in kv4_attention_kernel.h.
#pragma once

#include "kv4_attention_kernel.h"

namespace terna {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kKv4Rows = 128;                  // query rows of a workgroup
constexpr int kKv4Tile = 64;                   // slots of a tile
constexpr uint32_t kKv4HalfLow = 104, kKv4HalfHigh = 140;

template <int D>
struct Kv4PrefillLds {
    static constexpr int kTile = kKv4Tile * D * 2;                         // bytes of a tile's keys, or values
    static constexpr int kBytes = 2 * 2 * 2 * kTile;                       // groups, buffers, keys and values
};

// Byte offset of a key tile's 16-byte piece: 16 rows that are read together lie in different banks.
template <int D>
__device__ __forceinline__ int kv4_key_piece(int row, int piece)
{
    return row * (2 * D) + ((piece ^ (D == 128 ? row & 15 : (row >> 1) & 7)) << 4);
}

__device__ __forceinline__ u32x4 kv4_values_half(uint32_t codes, float scale)
{
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3))};
}

// max / sum over the lanes L, L ^ 32
template <bool IS_MAX>
__device__ __forceinline__ float halves_reduce(float v)
{
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return IS_MAX ? fmaxf(a, b) : a + b;
}

template <int D>
__global__ __launch_bounds__(512, 2) void terna_kv4_prefill_kernel(Kv4Attention a)
{
    constexpr int KS = D / 16, DT = D / 32, GROUPS = D / kKv4Group, TILE = Kv4PrefillLds<D>::kTile;
    constexpr int WORDS = D / 32;                                          // words of codes of a thread: 8 * WORDS dimensions of a row
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float2 stat[2][kKv4Rows];
    __shared__ int first_broken[GROUPS], wide_scales;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = wave >> 2, qi = lane & 31, half = lane >> 5;
    const int G = a.H / a.KV, rows = a.T * G;
    // Workgroups go to the XCDs round robin.  An XCD takes a run of the (sequence, kv head, split)s' eighths -- eighth c: the row blocks c, c + 8, ... from the
    // last one down -- so that it reads few of them, from its L2, and walks them longest rows first.
    const int pairs = a.B * a.KV * a.splits;
    const int slot = blockIdx.x >> 3, round8 = slot / pairs;
    const int eighth = pairs * (blockIdx.x & 7) + slot - round8 * pairs;
    const int from_last = 8 * round8 + (eighth & 7);
    if (from_last >= a.tiles) return;
    const int first_row = (a.tiles - 1 - from_last) * kKv4Rows;
    const int split = (eighth >> 3) % a.splits, bk = (eighth >> 3) / a.splits, kvh = bk % a.KV, b = bk / a.KV;

    // ---- rows
    const int r = first_row + (wave & 3) * 32 + qi;
    const bool real = r < rows;
    const int t = real ? r / G : 0, h = kvh * G + (real ? r - t * G : 0);
    const long long p64 = a.pos[(a.per_seq ? b * a.T : 0) + t];
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
    if (tid == 0) wide_scales = 0;
    __syncthreads();
    int all_keys = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) all_keys = max(all_keys, __float_as_int(stat[0][w].x));
    all_keys = __builtin_amdgcn_readfirstlane(all_keys);                   // of the workgroup
    const int all_tiles = (all_keys + kKv4Tile - 1) / kKv4Tile, share = (all_tiles + a.splits - 1) / a.splits;
    const int begin = split * share, end = min(begin + share, all_tiles), steps = (end - begin + 1) / 2;

    bf16x8 bq[KS];
    {
        const uint16_t* qrow = a.q + ((static_cast<size_t>(b) * a.H + h) * a.T + t) * D + 8 * half;
        const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
        for (int i = 0; i < KS; ++i) bq[i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(qrow + 16 * i) ^ u32x4{sign, sign, sign, sign});
        if (a.scale == 0.0f) {                                             // 0 * -inf would unmask a slot: the zero into the queries
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                float x[8];
                RotaryVector<uint16_t>::unpack(__builtin_bit_cast(u32x4, bq[i]), x);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= 0.0f;
                bq[i] = __builtin_bit_cast(bf16x8, RotaryVector<uint16_t>::pack(x));
            }
        }
    }
    const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale);

    // ---- cache
    const size_t base = (static_cast<size_t>(b) * a.KV + kvh) * a.S;
    const uint8_t *kb = a.k + base * (D / 2), *ksb = a.k_scale + base * GROUPS, *vb = a.v + base * (D / 2), *vsb = a.v_scale + base * GROUPS;
    const int tg = tid & 255, my_row = tg >> 2, part = tg & 3, my_group = part * GROUPS / 4;
    struct Codes {
        uint32_t k[WORDS], v[WORDS], ks, vs;
    } ahead;
    auto load = [&](int step) __attribute__((always_inline)) {
        const uint32_t at = min((begin + 2 * step + group) * kKv4Tile + my_row, a.S - 1);
        if constexpr (WORDS == 4) {
            const u32x4 kc = *reinterpret_cast<const u32x4*>(kb + at * (D / 2) + part * 16), vc = *reinterpret_cast<const u32x4*>(vb + at * (D / 2) + part * 16);
#pragma unroll
            for (int i = 0; i < WORDS; ++i) ahead.k[i] = kc[i], ahead.v[i] = vc[i];
        } else {
            const u32x2 kc = *reinterpret_cast<const u32x2*>(kb + at * (D / 2) + part * 8), vc = *reinterpret_cast<const u32x2*>(vb + at * (D / 2) + part * 8);
            ahead.k[0] = kc.x, ahead.k[1] = kc.y, ahead.v[0] = vc.x, ahead.v[1] = vc.y;
        }
        ahead.ks = ksb[at * GROUPS + my_group];
        ahead.vs = vsb[at * GROUPS + my_group];
    };
    uint8_t* const tiles = smem + group * 4 * TILE;                        // [buffer][keys, values]
    int broken = 0x7fffffff;
    bool wide = false;

    f32x16 o[DT];
    float m_run, l_run;
    auto pass = [&](auto in_half) __attribute__((always_inline)) {
        constexpr bool HALF = decltype(in_half)::value;
        constexpr float HELD = HALF ? 12.0f : kKv4Held, GROWTH = HALF ? 3.0f : 0.0f;
        auto convert = [&](int step) __attribute__((always_inline)) {
            uint8_t* const to = tiles + (step & 1) * 2 * TILE;
            const int at = (begin + 2 * step + group) * kKv4Tile + my_row;
            const float ks = __uint_as_float(ahead.ks << 23);
            uint32_t byte = at < all_keys ? ahead.vs : 127u;
            if (byte == kKv4Broken) {
                broken = min(broken, at);
                byte = 127u;
            }
            if (HALF) {
                wide |= byte < kKv4HalfLow || byte > kKv4HalfHigh;
                byte = min(byte, kKv4HalfHigh);
            } else {
                byte = min(byte, kKv4MaxByte);
            }
            const float vs = __uint_as_float(byte << 23);
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                *reinterpret_cast<u32x4*>(to + kv4_key_piece<D>(my_row, part * WORDS + i)) = kv4_values(ahead.k[i], ks);
                *reinterpret_cast<u32x4*>(to + TILE + kv4_piece<D>(my_row, part * WORDS + i)) = HALF ? kv4_values_half(ahead.v[i], vs) : kv4_values(ahead.v[i], vs);
            }
        };
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[dt][v] = 0.0f;
        m_run = -INFINITY;
        l_run = 0.0f;
        if (steps > 0) {
            load(0);
            convert(0);
            if (steps > 1) load(1);
        }
        int ka[KS], va[DT];
#pragma unroll
        for (int i = 0; i < KS; ++i) ka[i] = kv4_key_piece<D>(qi, 2 * i + half);
        const int vrow = 4 * half + ((lane & 15) >> 2);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) va[dt] = kv4_piece<D>(vrow, 4 * dt + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 8 * (lane & 1);
        for (int step = 0; step < steps; ++step) {
            __syncthreads();
            if (step + 1 < steps) {
                convert(step + 1);
                if (step + 2 < steps) load(step + 2);
            }
            const int k0 = (begin + 2 * step + group) * kKv4Tile;
            if (k0 >= n_keys || begin + 2 * step + group >= end) continue;     // nothing that this wave's rows see (uniform)
            const uint8_t* const keys = tiles + (step & 1) * 2 * TILE;
            const uint8_t* const vals = keys + TILE;
            f32x16 s[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int v = 0; v < 16; ++v) s[j][v] = 0.0f;
#pragma unroll
                for (int i = 0; i < KS; ++i)
                    s[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(keys + ka[i] + j * 32 * 2 * D)), bq[i], s[j], 0, 0, 0);
            }
            if (k0 + kKv4Tile > n_full) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (k0 + 32 * j + 8 * (v >> 2) + 4 * half + (v & 3) > my_last) s[j][v] = -INFINITY;
            }
            float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
            for (int v = 1; v < 16; ++v) top = fmaxf(top, fmaxf(s[0][v], s[1][v]));
            top = halves_reduce<true>(top) * scale;
            if (__any(top > m_run + GROWTH)) {
                const float m_new = fmaxf(m_run, top);
                const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));
                m_run = m_new;
                l_run *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
            }
            const float shift = HELD - (m_run == -INFINITY ? 0.0f : m_run);
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    s[j][v] = __builtin_amdgcn_exp2f(__fmaf_rn(s[j][v], scale, shift));
                    sum[v & 3] += s[j][v];
                }
            }
            l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
            for (int n = 0; n < 4; ++n) {                                  // 16 slots
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = s[n >> 1][8 * (n & 1) + e];
                u32x4 p_hi, p_lo;
                if constexpr (HALF) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) p_hi[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{p[2 * e], p[2 * e + 1]}), f16x2));
                } else {
                    float back[8];
                    p_hi = RotaryVector<uint16_t>::pack(p);
                    RotaryVector<uint16_t>::unpack(p_hi, back);
#pragma unroll
                    for (int e = 0; e < 8; ++e) back[e] = p[e] - back[e];
                    p_lo = RotaryVector<uint16_t>::pack(back);
                }
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    using Tr = s16x4 __attribute__((address_space(3)))*;
                    const u32x2 a0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(vals + va[dt] + n * 16 * 2 * D)));
                    const u32x2 a1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(vals + va[dt] + (n * 16 + 8) * 2 * D)));
                    const u32x4 values{a0.x, a0.y, a1.x, a1.y};
                    if constexpr (HALF) {
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, values), __builtin_bit_cast(f16x8, p_hi), o[dt], 0, 0, 0);
                    } else {
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, values), __builtin_bit_cast(bf16x8, p_hi), o[dt], 0, 0, 0);
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, values), __builtin_bit_cast(bf16x8, p_lo), o[dt], 0, 0, 0);
                    }
                }
            }
        }
        l_run = halves_reduce<false>(l_run);
        m_run -= HELD;                                                     // what the probabilities are relative to: the splits of a row may differ in it
    };
    pass(std::true_type{});
    if (wide) wide_scales = 1;
    __syncthreads();
    if (wide_scales) {                                                     // (all have read it behind the barrier; nobody writes it again)
        pass(std::false_type{});
        __syncthreads();
    }

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
    if (!real) return;
    const size_t out_row = (static_cast<size_t>(b) * a.T + t) * a.H + h;
    const float inverse = p64 < 0 ? 0.0f : 1.0f / l;
    if (a.splits > 1 && group == 0 && half == 0)
        *reinterpret_cast<float2*>(a.partial + static_cast<size_t>(a.B) * a.T * a.H * a.splits * D + (out_row * a.splits + split) * 2) = float2{m, l};
#pragma unroll
    for (int dt = 0; dt < DT / 2; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 32 * (keep + dt) + 8 * i + 4 * half;
            const f32x4 other = got[(8 * dt + 2 * i + half) * kKv4Rows + row_at];
            f32x4 x;
#pragma unroll
            for (int v = 0; v < 4; ++v) x[v] = (group == 0 ? o[dt][4 * i + v] : o[DT / 2 + dt][4 * i + v]) * w_mine + other[v] * w_other;
            if (outside || (p64 >= 0 && p64 >= first_broken[d / kKv4Group])) x = f32x4{NAN, NAN, NAN, NAN};
            if (a.splits == 1) {
                if (p64 < 0) x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                else x *= inverse;
                *reinterpret_cast<u32x2*>(a.out + out_row * D + d) = u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
            } else {
                *reinterpret_cast<f32x4*>(a.partial + (out_row * a.splits + split) * D + d) = x;
            }
        }
}

}  // namespace terna
