// New rows into the 4-bit cache (kv4_format.h), rotary positions applied on the way, and rows of it back as bf16.
//
// What bounds the store: memory -- a token's fused projection row is read once, its queries are written once in bf16, its keys and values once in
// 4.25 bits.  A workgroup takes a few tokens whole: their angles once into LDS (rotary_common.h), then eight dimensions a thread and step; the
// 32 values that share a scale are a quad's, whose maximum takes two quad permutations.  Two steps are under way at a time.  Measured, 30 heads of 128
// dimensions a row: 4 x 8192 tokens 91 us, 4.8 TB/s of the 4.9 that a large copy reaches; 2 x 1920 15.9 us, 52 MB, of which about 5 are the launch and its
// ends (one step under way 17.8; half pairs, which read their partners too, 20.8, and 25.9; four steps slow small calls by 0.4 us).
// Rows back: 4 x 8192 tokens of 5 kv heads 21.9 us, 4.8 TB/s.
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

// Half pairs: the 16 bytes that hold the partners of dimensions d .. d + 7 of `head`, where a piece's partners are one (else what is read is not used).
template <bool ADJACENT>
__device__ __forceinline__ u32x4 kv4_partner(const uint16_t* __restrict__ head, const u32x4& own, int d, int pairs)
{
    if (ADJACENT || (pairs & 7) != 0) return own;
    return *reinterpret_cast<const u32x4*>(head + (d < pairs ? d + pairs : d < 2 * pairs ? d - pairs : d));
}
// The dimensions d .. d + 7 of a head (16 bytes, `own`) turned; half pairs with kv4_partner's, or with single elements of the head.
template <bool ADJACENT>
__device__ __forceinline__ void kv4_turn8(const uint16_t* __restrict__ head, const u32x4& own, const u32x4& partner, int d, const float2* cs, int pairs, float x[8])
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
        V::unpack(partner, o);
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

constexpr int kKv4StoreTokens = 64;            // of a workgroup, at most: tokens double while they have 1024 pieces or fewer, at least 24 each

// xqkv bf16 rows b * T + t of `row` elements: H query, KV key, KV value heads -> q bf16 [B][H][T][D], rotated; slot pos of the caches
template <int D, bool ADJACENT>
__global__ __launch_bounds__(kRotaryThreads) void terna_kv4_store_kernel(const uint16_t* __restrict__ xqkv, const long long* __restrict__ pos,
                                                                         const double* __restrict__ frequency, uint16_t* __restrict__ q, uint8_t* __restrict__ k,
                                                                         uint8_t* __restrict__ k_scale, uint8_t* __restrict__ v, uint8_t* __restrict__ v_scale,
                                                                         RotaryShape s, int KV, int S, long long row)
{
    constexpr int PIECES = D / 8, AHEAD = 2;
    __shared__ float2 cs[kRotaryMaxAngles];
    __shared__ long long slots[kKv4StoreTokens];
    const int first = blockIdx.x * s.tokens_a_group;
    const int count = min(s.tokens_a_group, s.tokens - first);
    const RotaryTokens where(first, s.T);
    const int heads = s.H + 2 * KV, total = count * heads * PIECES;
    const int y_step = gridDim.y * kRotaryThreads;
    int i = blockIdx.y * kRotaryThreads + threadIdx.x;
    struct Piece { int n, head, d; const uint16_t* from; u32x4 own, partner; };
    auto fetch = [&](int i, Piece& p) __attribute__((always_inline)) {     // (behind the last: the last once more, so that no load hangs on a branch)
        i = min(i, total - 1);
        const int all = i / PIECES;
        p.d = (i & (PIECES - 1)) * 8;
        p.n = all / heads;
        p.head = all - p.n * heads;
        p.from = xqkv + (first + p.n) * row + p.head * D;
        p.own = *reinterpret_cast<const u32x4*>(p.from + p.d);
        p.partner = kv4_partner<ADJACENT>(p.from, p.own, p.d, s.pairs);
    };
    Piece ring[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) fetch(i + u * y_step, ring[u]);
    rotary_angles(cs, pos, frequency, s, first, count, where);
    if (threadIdx.x < count) {
        int b, t;
        where.of(threadIdx.x, &b, &t);
        slots[threadIdx.x] = pos[s.per_seq ? first + threadIdx.x : t];
    }
    __syncthreads();
    auto store = [&](const Piece& p) __attribute__((always_inline)) {
        int b, t;
        where.of(p.n, &b, &t);
        float x[8];
        if (p.head < s.H) {
            kv4_turn8<ADJACENT>(p.from, p.own, p.partner, p.d, cs + p.n * s.pairs, s.pairs, x);
            *reinterpret_cast<u32x4*>(q + ((static_cast<size_t>(b) * s.H + p.head) * s.T + t) * D + p.d) = RotaryVector<uint16_t>::pack(x);
        } else {
            const bool is_key = p.head < s.H + KV;
            if (is_key) kv4_turn8<ADJACENT>(p.from, p.own, p.partner, p.d, cs + p.n * s.pairs, s.pairs, x);
            else RotaryVector<uint16_t>::unpack(p.own, x);
            const uint32_t byte = kv4_scale_byte(kv4_amax_bits(x)), codes = kv4_codes(x, byte);
            const long long slot = slots[p.n];
            if (slot >= 0 && slot < S) {
                const int kvh = p.head - s.H - (is_key ? 0 : KV);
                const size_t at = (static_cast<size_t>(b) * KV + kvh) * S + static_cast<size_t>(slot);
                *reinterpret_cast<uint32_t*>((is_key ? k : v) + at * (D / 2) + p.d / 2) = codes;
                if ((p.d & (kKv4Group - 1)) == 0) (is_key ? k_scale : v_scale)[at * (D / kKv4Group) + p.d / kKv4Group] = static_cast<uint8_t>(byte);
            }
        }
    };
    for (; i < total; i += AHEAD * y_step)
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (i + u * y_step < total) store(ring[u]);
            fetch(i + (AHEAD + u) * y_step, ring[u]);
        }
}

// Keys and values of the slots pos as bf16 [B][T][KV][D]; NaN for a position outside the cache.  A workgroup takes a few tokens, a thread eight dimensions a step:
// four bytes of codes to sixteen, neighbours next to each other.
__global__ __launch_bounds__(256) void terna_kv4_rows_kernel(const uint8_t* __restrict__ k, const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v,
                                                             const uint8_t* __restrict__ v_scale, const long long* __restrict__ pos, uint16_t* __restrict__ k_out,
                                                             uint16_t* __restrict__ v_out, int T, int KV, int S, int D, int per_seq, int tokens, int tokens_a_group)
{
    const int first = blockIdx.x * tokens_a_group, count = min(tokens_a_group, tokens - first);
    const RotaryTokens where(first, T);
    const int half = KV * D / 8, total = count * 2 * half;
    for (int i = threadIdx.x; i < total; i += 256) {
        const int n = i / (2 * half), in_token = i - n * (2 * half);
        const bool is_key = in_token < half;
        const int d = (is_key ? in_token : in_token - half) * 8, kvh = d / D, at_d = d & (D - 1);
        int b, t;
        where.of(n, &b, &t);
        const long long slot = pos[per_seq ? first + n : t];
        uint32_t codes = 0, byte = kKv4Broken;
        if (slot >= 0 && slot < S) {
            const size_t at = (static_cast<size_t>(b) * KV + kvh) * S + static_cast<size_t>(slot);
            codes = *reinterpret_cast<const uint32_t*>((is_key ? k : v) + at * (D / 2) + at_d / 2);
            byte = (is_key ? k_scale : v_scale)[at * (D / kKv4Group) + at_d / kKv4Group];
        }
        const u32x4 broken{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
        *reinterpret_cast<u32x4*>((is_key ? k_out : v_out) + static_cast<size_t>(first + n) * (KV * D) + d) =
            byte == kKv4Broken ? broken : kv4_values(codes, __uint_as_float(byte << 23));
    }
}

}  // namespace terna
