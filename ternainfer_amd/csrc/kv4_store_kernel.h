// New rows into the 4-bit cache (kv4_format.h), rotary positions applied on the way, and rows of it back as bf16.
//
// What bounds the store: memory -- a token's fused projection row is read once, its queries are written once in bf16, its keys and values once in
// 4.25 bits.  A workgroup takes a few tokens whole: their angles once into LDS (rotary_common.h), then eight dimensions a thread and step; the
// 32 values that share a scale are a quad's, whose maximum takes two quad permutations.
#pragma once

#include "kv4_format.h"
#include "rotary_kernel.h"

namespace terna {

// max over the four lanes of a quad, of bits without a sign
__device__ __forceinline__ uint32_t kv4_quad_max(uint32_t v)
{
    const uint32_t a = __builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, true);        // lanes 1 0 3 2
    v = v > a ? v : a;
    const uint32_t b = __builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, true);        // lanes 2 3 0 1
    return v > b ? v : b;
}
__device__ __forceinline__ uint32_t kv4_amax_bits(const float x[8])
{
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t b = __float_as_uint(x[e]) & 0x7fffffffu;
        m = m > b ? m : b;
    }
    return kv4_quad_max(m);
}

// The dimensions d .. d + 7 of a head (16 bytes at `own`) turned: the pairs' other halves from `head` where they are not in the piece.
template <bool ADJACENT>
__device__ __forceinline__ void kv4_turn8(const uint16_t* __restrict__ head, const u32x4& own, int d, const float2* cs, int pairs, float x[8])
{
    using V = RotaryVector<uint16_t>;
    V::unpack(own, x);
    if constexpr (ADJACENT) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (d / 2 + e < pairs) {
                const float2 y = rotary_turn(x[2 * e], x[2 * e + 1], cs[d / 2 + e]);
                x[2 * e] = y.x;
                x[2 * e + 1] = y.y;
            }
        }
    } else if ((pairs & 7) == 0) {
        if (d >= 2 * pairs) return;
        const bool lower = d < pairs;
        float o[8];
        V::unpack(*reinterpret_cast<const u32x4*>(head + (lower ? d + pairs : d - pairs)), o);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = lower ? rotary_turn(x[e], o[e], cs[d + e]).x : rotary_turn(o[e], x[e], cs[d - pairs + e]).y;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int at = d + e;
            if (at < pairs) x[e] = rotary_turn(x[e], bf16_bits_to_float(head[at + pairs]), cs[at]).x;
            else if (at < 2 * pairs) x[e] = rotary_turn(bf16_bits_to_float(head[at - pairs]), x[e], cs[at - pairs]).y;
        }
    }
}

// xqkv bf16 rows b * T + t of `row` elements: H query, KV key, KV value heads -> q bf16 [B][H][T][D], rotated; slot pos of the caches
template <int D, bool ADJACENT>
__global__ __launch_bounds__(kRotaryThreads) void terna_kv4_store_kernel(const uint16_t* __restrict__ xqkv, const long long* __restrict__ pos,
                                                                         const double* __restrict__ frequency, uint16_t* __restrict__ q, uint8_t* __restrict__ k,
                                                                         uint8_t* __restrict__ k_scale, uint8_t* __restrict__ v, uint8_t* __restrict__ v_scale,
                                                                         RotaryShape s, int KV, int S, long long row)
{
    constexpr int PIECES = D / 8;
    __shared__ float2 cs[kRotaryMaxAngles];
    const int first = blockIdx.x * s.tokens_a_group;
    const int count = min(s.tokens_a_group, s.tokens - first);
    const RotaryTokens where(first, s.T);
    const int heads = s.H + 2 * KV, total = count * heads * PIECES;
    const int y_step = gridDim.y * kRotaryThreads;
    int i = blockIdx.y * kRotaryThreads + threadIdx.x;
    struct Piece { int n, head, d; const uint16_t* from; u32x4 own; };
    auto fetch = [&](int i) __attribute__((always_inline)) {
        Piece p;
        const int all = i / PIECES;
        p.d = (i & (PIECES - 1)) * 8;
        p.n = all / heads;
        p.head = all - p.n * heads;
        p.from = xqkv + (first + p.n) * row + p.head * D;
        p.own = *reinterpret_cast<const u32x4*>(p.from + p.d);
        return p;
    };
    Piece p{};
    if (i < total) p = fetch(i);
    rotary_angles(cs, pos, frequency, s, first, count, where);
    __syncthreads();
    for (; i < total;) {
        int b, t;
        where.of(p.n, &b, &t);
        float x[8];
        if (p.head < s.H) {
            kv4_turn8<ADJACENT>(p.from, p.own, p.d, cs + p.n * s.pairs, s.pairs, x);
            *reinterpret_cast<u32x4*>(q + ((static_cast<size_t>(b) * s.H + p.head) * s.T + t) * D + p.d) = RotaryVector<uint16_t>::pack(x);
        } else {
            const bool is_key = p.head < s.H + KV;
            if (is_key) kv4_turn8<ADJACENT>(p.from, p.own, p.d, cs + p.n * s.pairs, s.pairs, x);
            else RotaryVector<uint16_t>::unpack(p.own, x);
            const uint32_t byte = kv4_scale_byte(kv4_amax_bits(x)), codes = kv4_codes(x, byte);
            const long long slot = pos[s.per_seq ? first + p.n : t];
            if (slot >= 0 && slot < S) {
                const int kvh = p.head - s.H - (is_key ? 0 : KV);
                const size_t at = (static_cast<size_t>(b) * KV + kvh) * S + static_cast<size_t>(slot);
                *reinterpret_cast<uint32_t*>((is_key ? k : v) + at * (D / 2) + p.d / 2) = codes;
                if ((p.d & (kKv4Group - 1)) == 0) (is_key ? k_scale : v_scale)[at * (D / kKv4Group) + p.d / kKv4Group] = static_cast<uint8_t>(byte);
            }
        }
        i += y_step;
        if (i < total) p = fetch(i);
    }
}

// Keys and values of the slots pos as bf16 [B][T][KV][D]; NaN for a position outside the cache.  32 dimensions a thread.
__global__ __launch_bounds__(256) void terna_kv4_rows_kernel(const uint8_t* __restrict__ k, const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v,
                                                             const uint8_t* __restrict__ v_scale, const long long* __restrict__ pos, uint16_t* __restrict__ k_out,
                                                             uint16_t* __restrict__ v_out, int T, int KV, int S, int D, int per_seq, long long groups)
{
    const long long all = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (all >= 2 * groups) return;
    const bool is_key = all < groups;
    const long long i = is_key ? all : all - groups;
    const int parts = D / kKv4Group;
    const long long head = i / parts;
    const int part = static_cast<int>(i - head * parts);
    const long long token = head / KV;
    const int kvh = static_cast<int>(head - token * KV);
    const long long b = token / T;
    const long long slot = pos[per_seq ? token : token - b * T];
    u32x4 codes{0u, 0u, 0u, 0u};
    uint32_t byte = kKv4Broken;
    if (slot >= 0 && slot < S) {
        const size_t at = (static_cast<size_t>(b) * KV + kvh) * S + static_cast<size_t>(slot);
        codes = *reinterpret_cast<const u32x4*>((is_key ? k : v) + at * (D / 2) + part * 16);
        byte = (is_key ? k_scale : v_scale)[at * parts + part];
    }
    u32x4* to = reinterpret_cast<u32x4*>((is_key ? k_out : v_out) + i * kKv4Group);
    const float scale = __uint_as_float(byte << 23);
#pragma unroll
    for (int n = 0; n < 4; ++n) to[n] = byte == kKv4Broken ? u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u} : kv4_values(codes[n], scale);
}

}  // namespace terna
