// Attention of a few query rows over the 4-bit cache (kv4_format.h): single-token steps, drafted tokens, short chunks.
//
//   out[row] = sum_s p_s v_s / sum_s p_s,  p_s = exp(scale q . k_s - max),  s = 0 .. pos of the row's token
//
// The rows of a kv head -- its G = H / KV query heads times the new tokens, row r = t * G + head -- are taken sixteen at a time, as the columns of the
// matrix cores' 16x16x32 products.  A wave works alone on 32 slots at a time: codes -> bf16 in registers (the hardware conversion, two values an
// instruction, the scale inside it: exact), scores, running maximum and sum, output; no wave waits for another until the end, where the four or
// eight of a workgroup and then the splits are merged.
//   * Keys: a lane holds a quarter of a row (one 16-byte load of a row of 128 dimensions) and its scale byte; the products run over the dimensions in
//     the order in which the lanes hold them, for queries and keys alike.
//   * Values: a lane holds 32 dimensions of a row, which share a scale; converted rows go through LDS (of the wave alone) and come back transposed.
//   * Values and probabilities are fp16 (below), all sums fp32.  The running maximum is raised, and the output rescaled, only where it grows by more than 2^3 -- a row's own, so that a
//     row's bits are the same whatever the rows that share its tile, real or padded, hold (but for value scales that send them all through bf16 values: below).
//     Raising all where one grew, which needs a comparison less, was 1 % faster and gave a step's last tile other bits than store and attention have.
//   * A value scale of 255 (NaN) in a slot that a row does not see must not reach it through 0 * NaN: the first such slot of each 32 dimensions is
//     kept and NaN given to the rows that see it; the products use the largest finite scale in its place.  So also whatever unwritten slots hold.
// What bounds it: a long cache -- memory (4 x 32768 slots, 5 kv heads: 85 MB in 20 us, 4.2 TB/s, then 4 for the splits); a short one -- the launch, two trips to memory (position,
// cache), then 0.63 us a step of a wave, a chain through LDS and two kinds of products (1 x 384 slots 6.4 us, 8 x 384 7.0).
#pragma once

#include "kv4_plan.h"
#include "kv4_store_kernel.h"

namespace terna {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kKv4Held = -26.0f;             // a row's largest probability is held at 2^-26: sums over 2^25 slots of the largest values stay finite

// Values and probabilities in fp16: a value is a code times a power of two, exact in fp16 for scale bytes 104 .. 140 (2^-23 .. 2^13); probabilities keep 11 bits, held
// at 2^12 for a row's running maximum -- up to 2^15 where a larger score has not raised it yet -- so that those 2^-26 of it are still normal numbers.  Any
// other scale of a group that is not all zeros marks the workgroup, which starts again with bf16 values and probabilities in two bf16, the products twice.
constexpr uint32_t kKv4HalfLow = 104, kKv4HalfHigh = 140;
constexpr uint32_t kKv4Magnitudes = 0x77777777u;           // the bits of eight codes that make them no zeros
constexpr float kKv4HeldHalf = 12.0f, kKv4Growth = 3.0f;

__device__ __forceinline__ u32x4 kv4_values_half(uint32_t codes, float scale)
{
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3))};
}

// NaN where one of them is: a row with such a score is NaN, whatever its maximum.  (IEEE 754-2019's maximum, one instruction.  From fmaxf the compiler makes two, each
// behind one that quiets a NaN; and not inline assembly, in front of which it does not wait for the matrix products that are read here.)
__device__ __forceinline__ float kv4_max3(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }

struct Kv4Attention {
    const uint16_t* q;                         // [B][H][T][D]; STEP: rows of `row` elements as terna_kv4_store_kernel takes them
    uint8_t *k, *k_scale, *v, *v_scale;        // (written by STEP only)
    const long long* pos;
    uint16_t* out;                             // [B * T][H * D], or
    float* partial;                            // more than one split: fp32 [rows][splits][D] numerators, then [rows][splits][2] maximum, sum
    const double* frequency;                   // STEP
    double amplitude;
    long long row;
    int B, T, H, KV, S, tiles, splits, per_seq, pairs, parts;
    float scale;                               // times log2(e)
};

// Layout of an 8-row by 16-byte-piece swizzle: rows of 2 D bytes, conflict-free for row-wise 16-byte writes and transposing reads.
template <int D>
__device__ __forceinline__ int kv4_piece(int row, int piece)
{
    return row * (2 * D) + ((piece ^ (D == 128 ? (row & 7) << 1 : (row & 6))) << 4);
}

template <int D, bool STEP, bool ADJACENT, int NW>
__global__ __launch_bounds__(64 * NW, 2) void terna_kv4_attention_kernel(Kv4Attention a)
{
    constexpr int DL = D / 4, KI = DL / 8, DT = D / 16, GROUPS = D / kKv4Group;
    constexpr int STAGE = kKv4Step * D * 2;                    // bytes of a wave's converted values
    __shared__ __align__(16) uint8_t smem[NW * STAGE];
    __shared__ float2 stat[NW][16];
    __shared__ int first_broken[GROUPS], wide_scales;
    __shared__ __align__(16) uint32_t new_codes[2][D / 8];     // STEP: the new token's key and value
    __shared__ uint32_t new_scale[2][GROUPS];
    __shared__ float2 angles[STEP ? D / 2 : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int qi = lane & 15, g = lane >> 4;
    // Workgroups go to the XCDs round robin: the tiles of one (sequence, kv head, split) -- which read the same slots -- eight apart, on one XCD.
    const int G = a.H / a.KV, groups = a.B * a.KV * a.splits;
    const int block = blockIdx.x / (8 * a.tiles), within = blockIdx.x - block * (8 * a.tiles);
    const int group = 8 * block + (within & 7), tile = within >> 3;
    if (group >= groups) return;
    const int split = group % a.splits, bk = group / a.splits, kvh = bk % a.KV, b = bk / a.KV;

    // ---- rows
    const int rows = a.T * G, r = tile * 16 + qi;
    const bool real = r < rows;
    const int t = real ? r / G : 0, h = kvh * G + (real ? r - t * G : 0);
    const long long p64 = a.pos[(a.per_seq ? b * a.T : 0) + t];
    const bool outside = p64 >= a.S;                           // its result is NaN
    const int my_last = !real || p64 < 0 ? -1 : outside ? a.S - 1 : static_cast<int>(p64);
    int n_keys = my_last + 1, n_full = real ? my_last + 1 : a.S;
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
        n_keys = max(n_keys, __shfl_xor(n_keys, off));
        n_full = min(n_full, __shfl_xor(n_full, off));
    }
    n_keys = __builtin_amdgcn_readfirstlane(n_keys);
    n_full = __builtin_amdgcn_readfirstlane(n_full);
    const int all_steps = (n_keys + kKv4Step - 1) / kKv4Step, share = (all_steps + a.splits - 1) / a.splits;
    const int begin = split * share, end = min(begin + share, all_steps);

    // ---- cache rows: this lane's addresses
    const size_t base = (static_cast<size_t>(b) * a.KV + kvh) * a.S;
    const uint8_t *kb = a.k + base * (D / 2), *ksb = a.k_scale + base * GROUPS, *vb = a.v + base * (D / 2), *vsb = a.v_scale + base * GROUPS;
    const int k_group = g * DL / kKv4Group;
    constexpr int VL = GROUPS / 2;                             // value loads of a lane: rows of GROUPS lanes each
    const int v_group = lane & (GROUPS - 1), v_row = lane / GROUPS;
    struct Tile {
        uint32_t k[2][KI], ks[2], vs[VL];
        u32x4 v[VL];
    };
    // Requests end with the split: a step behind it -- two are always under way -- touches no memory and gets zeros.  (Not by a branch: where a load may
    // or may not have been issued, the wait for one in front of it waits for both.)
    const uint32_t in_reach = static_cast<uint32_t>(max(min(end * kKv4Step, a.S), 0));
    const __amdgpu_buffer_rsrc_t rk = make_raw_buffer(kb, in_reach * (D / 2)), rks = make_raw_buffer(ksb, in_reach * GROUPS), rv = make_raw_buffer(vb, in_reach * (D / 2)),
                                 rvs = make_raw_buffer(vsb, in_reach * GROUPS);
    auto load = [&](int step, Tile& x) __attribute__((always_inline)) {
        const uint32_t k0 = static_cast<uint32_t>(step) * kKv4Step;         // (requests behind the longest cache pass 2^31)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t at = (k0 + qi) * (D / 2) + g * (DL / 2) + j * 16 * (D / 2);
            if constexpr (KI == 4) {
                const u32x4 c = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, at, 0, 0));
#pragma unroll
                for (int i = 0; i < KI; ++i) x.k[j][i] = c[i];
            } else {
                const u32x2 c = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rk, at, 0, 0));
                x.k[j][0] = c.x;
                x.k[j][1] = c.y;
            }
            x.ks[j] = __builtin_amdgcn_raw_buffer_load_b8(rks, (k0 + qi) * GROUPS + k_group + j * 16 * GROUPS, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < VL; ++i) {
            x.v[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, (k0 + v_row) * (D / 2) + v_group * 16 + i * (64 / GROUPS) * (D / 2), 0, 0));
            x.vs[i] = __builtin_amdgcn_raw_buffer_load_b8(rvs, k0 * GROUPS + lane + i * 64, 0, 0);
        }
    };
    Tile ring[3];                                              // the next two steps are under way: a trip to memory takes longer than a step
    auto load_first = [&]() __attribute__((always_inline)) {
        load(begin + wave, ring[0]);
        load(begin + wave + NW, ring[1]);
    };
    load_first();

    // ---- queries: a lane's quarter of its row
    bf16x8 bq[KI];
    if constexpr (STEP) {
        const uint16_t* token = a.q + b * a.row;
        const int last = p64 < 0 || outside ? -1 : static_cast<int>(p64);      // one token: the same in every lane
        for (int j = tid; j < a.pairs; j += 64 * NW) angles[j] = rotary_angle(a.pos[a.per_seq ? b : 0], a.frequency[j], a.amplitude);
        if (tid < GROUPS) first_broken[tid] = 0x7fffffff;
        if (tid == 0) wide_scales = 0;
        __syncthreads();
        // the tile's query heads, then the new key and value: eight dimensions a thread; queries through LDS into the products' order
        constexpr int PIECES = D / 8;
        const int heads = min(16, rows - tile * 16);
        for (int i = tid; i < (heads + 2) * PIECES; i += 64 * NW) {
            const int n = i / PIECES, d = (i & (PIECES - 1)) * 8;
            const int head = n < heads ? kvh * G + tile * 16 + n : n == heads ? a.H + kvh : a.H + a.KV + kvh;
            const uint16_t* from = token + head * D;
            const u32x4 own = *reinterpret_cast<const u32x4*>(from + d);
            float x[8];
            if (n <= heads) kv4_turn8<ADJACENT>(from, own, kv4_partner<ADJACENT>(from, own, d, a.pairs), d, angles, a.pairs, x);
            else RotaryVector<uint16_t>::unpack(own, x);
            if (n < heads) {
                *reinterpret_cast<u32x4*>(smem + kv4_piece<D>(n, d / 8)) = RotaryVector<uint16_t>::pack(x);
            } else {
                const uint32_t byte = kv4_scale_byte(kv4_amax_bits(x)), codes = kv4_codes(x, byte);
                new_codes[n - heads][d / 8] = codes;
                if ((d & (kKv4Group - 1)) == 0) new_scale[n - heads][d / kKv4Group] = byte;
                // the split that reads the new slot writes it, once a kv head
                const bool mine = tile == 0 && last >= begin * kKv4Step && last < end * kKv4Step;
                if (mine) {
                    const size_t at = base + last;
                    *reinterpret_cast<uint32_t*>((n == heads ? a.k : a.v) + at * (D / 2) + d / 2) = codes;
                    if ((d & (kKv4Group - 1)) == 0) (n == heads ? a.k_scale : a.v_scale)[at * GROUPS + d / kKv4Group] = static_cast<uint8_t>(byte);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < KI; ++i) bq[i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(smem + kv4_piece<D>(real ? qi : 0, (g * DL) / 8 + i)));
        __syncthreads();
    } else {
        const uint16_t* qrow = a.q + ((static_cast<size_t>(b) * a.H + h) * a.T + t) * D + g * DL;
#pragma unroll
        for (int i = 0; i < KI; ++i) bq[i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(qrow + 8 * i));
        if (tid < GROUPS) first_broken[tid] = 0x7fffffff;
        if (tid == 0) wide_scales = 0;
        __syncthreads();
    }
    // The scale's sign goes into the queries, a scale of 0 too (0 * -inf would unmask a slot): the largest score is then that of the largest product.
    const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale);
    if (a.scale <= 0.0f) {
#pragma unroll
        for (int i = 0; i < KI; ++i) {
            float x[8];
            RotaryVector<uint16_t>::unpack(__builtin_bit_cast(u32x4, bq[i]), x);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= a.scale == 0.0f ? 0.0f : -1.0f;
            bq[i] = __builtin_bit_cast(bf16x8, RotaryVector<uint16_t>::pack(x));
        }
    }
    // STEP: the slot that this launch fills is read from what it was filled with
    auto patch = [&](int step, Tile& x) __attribute__((always_inline)) {
        const int k0 = step * kKv4Step;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (k0 + 16 * j + qi == n_keys - 1) {
#pragma unroll
                for (int i = 0; i < KI; ++i) x.k[j][i] = new_codes[0][g * KI + i];
                x.ks[j] = new_scale[0][k_group];
            }
        }
#pragma unroll
        for (int i = 0; i < VL; ++i) {
            if (k0 + i * (64 / GROUPS) + v_row == n_keys - 1) {
                x.v[i] = *reinterpret_cast<const u32x4*>(&new_codes[1][v_group * 4]);
                x.vs[i] = new_scale[1][v_group];
            }
        }
    };

    uint8_t* stage = smem + wave * STAGE;
    int va[DT];
    const int vrow = 4 * g + (qi >> 2);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) va[dt] = kv4_piece<D>(vrow, 2 * dt + ((qi & 3) >> 1)) + 8 * (qi & 1);
    const int new_step = STEP && n_keys > 0 && !outside ? (n_keys - 1) / kKv4Step : -1;
    f32x4 o[DT];
    float m_run, l_run;
    int broken = 0x7fffffff;                                   // this lane's 32 dimensions
    bool wide = false;
    // All steps of the wave, with values and probabilities in fp16 (HALF) or with bf16 values and probabilities in two bf16.
    auto pass = [&](auto in_half) __attribute__((always_inline)) {
        constexpr bool HALF = decltype(in_half)::value;
        constexpr float HELD = HALF ? kKv4HeldHalf : kKv4Held, GROWTH = HALF ? kKv4Growth : 0.0f;
        auto work = [&](int step, Tile& x) __attribute__((always_inline)) {
            const int k0 = step * kKv4Step;
            // values -> rows in LDS
#pragma unroll
            for (int i = 0; i < VL; ++i) {
                const int row = i * (64 / GROUPS) + v_row;
                uint32_t byte = x.vs[i];
                // one test for what is rare: NaN, slots that nobody sees and what they hold, scales that fp16 has no room for
                if (k0 + kKv4Step > n_keys || __any(byte < kKv4HalfLow || byte > kKv4HalfHigh)) {
                    if (k0 + row >= n_keys) byte = 127u;
                    if (byte == kKv4Broken) {
                        broken = min(broken, k0 + row);
                        byte = 127u;
                    }
                    if (HALF) wide |= (byte < kKv4HalfLow || byte > kKv4HalfHigh) && ((x.v[i][0] | x.v[i][1] | x.v[i][2] | x.v[i][3]) & kKv4Magnitudes) != 0;
                    byte = min(byte, HALF ? kKv4HalfHigh : kKv4MaxByte);
                }
                const float vs = __uint_as_float(byte << 23);
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    *reinterpret_cast<u32x4*>(stage + kv4_piece<D>(row, v_group * 4 + n)) = HALF ? kv4_values_half(x.v[i][n], vs) : kv4_values(x.v[i][n], vs);
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            // scores of keys 16 j + 4 g + v
            f32x4 s[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                s[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                const float ks = __uint_as_float(x.ks[j] << 23);
#pragma unroll
                for (int i = 0; i < KI; ++i)
                    s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kv4_values(x.k[j][i], ks)), bq[i], s[j], 0, 0, 0);
            }
            // the transposed values, requested in front of the softmax: left to itself the compiler reads each where it is used, eight trips to LDS in a row
            u32x4 values[DT];
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                using Tr = s16x4 __attribute__((address_space(3)))*;
                const u32x2 a0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(stage + va[dt])));
                const u32x2 a1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(stage + va[dt] + 16 * 2 * D)));
                values[dt] = u32x4{a0.x, a0.y, a1.x, a1.y};
            }
            __builtin_amdgcn_sched_barrier(0);
            if (k0 + kKv4Step > n_full) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (k0 + 16 * (e >> 2) + 4 * g + (e & 3) > my_last) s[e >> 2][e & 3] = -INFINITY;
            }
            float top = kv4_max3(kv4_max3(s[0][0], s[0][1], s[0][2]), kv4_max3(s[0][3], s[1][0], s[1][1]), kv4_max3(s[1][2], s[1][3], s[1][3]));
            top = cross_row_reduce<true>(top) * scale;
            if (__any(top > m_run + GROWTH)) {
                const float m_new = top > m_run + GROWTH ? top : m_run;            // a row by its own growth alone: its bits do not hang on the rows beside it
                const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));       // (a row that has seen nothing yet: exp(-inf))
                m_run = m_new;
                l_run *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
            }
            const float shift = HELD - (m_run == -INFINITY ? 0.0f : m_run);
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(__fmaf_rn(s[e >> 2][e & 3], scale, shift));
            // outputs: dims 16 dt + 4 g + v of row qi
            if constexpr (HALF) {
                u32x4 packed;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f16x2 pair = __builtin_convertvector((f32x2{p[2 * e], p[2 * e + 1]}), f16x2);
                    packed[e] = __builtin_bit_cast(uint32_t, pair);
                    l_run = __builtin_amdgcn_fdot2(pair, f16x2{1, 1}, l_run, false);
                }
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, values[dt]), __builtin_bit_cast(f16x8, packed), o[dt], 0, 0, 0);
            } else {
                float back[8];
                const u32x4 hi = RotaryVector<uint16_t>::pack(p);
                RotaryVector<uint16_t>::unpack(hi, back);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    l_run += p[e];
                    back[e] = p[e] - back[e];
                }
                const bf16x8 p_hi = __builtin_bit_cast(bf16x8, hi), p_lo = __builtin_bit_cast(bf16x8, RotaryVector<uint16_t>::pack(back));
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, values[dt]), p_hi, o[dt], 0, 0, 0);
                    o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, values[dt]), p_lo, o[dt], 0, 0, 0);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        };
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m_run = -INFINITY;
        l_run = 0.0f;
        int step = begin + wave;
        while (step < end) {
#pragma unroll
            for (int n = 0; n < 3; ++n) {
                load(step + 2 * NW, ring[(n + 2) % 3]);
                if (STEP && step == new_step) patch(step, ring[n]);
                work(step, ring[n]);
                step += NW;
                if (step >= end) break;
            }
        }
        l_run = cross_row_reduce<false>(l_run);
        m_run -= HELD;                                         // what the probabilities are relative to: the splits of a row may differ in it
    };
    pass(std::true_type{});
    if (wide) wide_scales = 1;
    __syncthreads();
    if (wide_scales) {                                         // (all have read it behind the barrier; nobody writes it again)
        load_first();
        pass(std::false_type{});
    }

    // ---- the waves
    if (broken != 0x7fffffff) atomicMin(&first_broken[v_group], broken);      // a minimum: any order
    if (g == 0) stat[wave][qi] = float2{m_run, l_run};
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, stat[w][qi].x);
    const float mine = __builtin_amdgcn_exp2f(m_run - (top == -INFINITY ? 0.0f : top));
    float* numerators = reinterpret_cast<float*>(smem) + wave * 16 * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
        for (int v = 0; v < 4; ++v) o[dt][v] *= mine;
        *reinterpret_cast<f32x4*>(numerators + qi * D + ((16 * dt + 4 * g) ^ ((qi & 7) << 2))) = o[dt];
    }
    __syncthreads();
    // a thread: eight dimensions of a row, the waves' numerators
    constexpr int PIECES = D / 8;
    for (int i = tid; i < 16 * PIECES; i += 64 * NW) {
        const int n = i / PIECES, d = (i & (PIECES - 1)) * 8, rr = tile * 16 + n;
        if (rr >= rows) continue;
        const int tt = rr / G, hh = kvh * G + rr - tt * G;
        const long long q64 = a.pos[(a.per_seq ? b * a.T : 0) + tt];
        float m = -INFINITY, l = 0.0f, x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; ++w) m = fmaxf(m, stat[w][n].x);
        const float m_use = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            l += stat[w][n].y * __builtin_amdgcn_exp2f(stat[w][n].x - m_use);
            const float* from = reinterpret_cast<const float*>(smem) + (w * 16 + n) * D;
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const f32x4 y = *reinterpret_cast<const f32x4*>(from + ((d + e) ^ ((n & 7) << 2)));
#pragma unroll
                for (int v = 0; v < 4; ++v) x[e + v] += y[v];
            }
        }
        if (q64 >= a.S || (q64 >= 0 && q64 >= first_broken[d / kKv4Group])) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = NAN;
        }
        const size_t out_row = (static_cast<size_t>(b) * a.T + tt) * a.H + hh;
        if (a.splits == 1) {
            const float inverse = q64 < 0 ? 0.0f : 1.0f / l;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = q64 < 0 ? 0.0f : x[e] * inverse;
            *reinterpret_cast<u32x4*>(a.out + out_row * D + d) = RotaryVector<uint16_t>::pack(x);
        } else {
            float* to = a.partial + (out_row * a.splits + split) * D + d;
            *reinterpret_cast<f32x4*>(to) = f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4*>(to + 4) = f32x4{x[4], x[5], x[6], x[7]};
            if (d == 0) *reinterpret_cast<float2*>(a.partial + static_cast<size_t>(a.B) * a.T * a.H * a.splits * D + (out_row * a.splits + split) * 2) = float2{m, l};
        }
    }
}

// The splits of a row: four waves, each every fourth split, D / 64 dimensions a lane.  Their order is fixed, so is the result.  What bounds it: the launch and two
// trips to memory -- eight splits are under way at a time (step and merge of 1 x 32768 slots in 43 splits 15.0 us with one, so 13.5; of 1 x 131072 29.0 and 25.5).
template <int D>
__global__ __launch_bounds__(256) void terna_kv4_merge_kernel(const float* __restrict__ partial, const long long* __restrict__ pos, uint16_t* __restrict__ out, int T, int H,
                                                              int splits, int per_seq)
{
    constexpr int V = D / 64;
    __shared__ float part[4][D];
    const int row = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float2* stat = reinterpret_cast<const float2*>(partial + static_cast<size_t>(gridDim.x) * splits * D) + static_cast<size_t>(row) * splits;
    const float2 none{-INFINITY, 0.0f}, s0 = lane < splits ? stat[lane] : none, s1 = lane + 64 < splits ? stat[lane + 64] : none;
    const float* o = partial + static_cast<size_t>(row) * splits * D + V * lane;
    constexpr int AT_ONCE = 8;
    float part_of[AT_ONCE][V];
    auto fetch = [&](int from) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
#pragma unroll
            for (int v = 0; v < V; ++v) part_of[n][v] = 0.0f;
            if (from + 4 * n < splits) {                                   // (the same for the wave)
#pragma unroll
                for (int v = 0; v < V; ++v) part_of[n][v] = o[static_cast<size_t>(from + 4 * n) * D + v];
            }
        }
    };
    fetch(wave);
    const int token = row / H, t = token % T;
    const long long p = pos[per_seq ? token : t];
    float m = fmaxf(s0.x, s1.x);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    const float m_use = m == -INFINITY ? 0.0f : m;
    const float w0 = __builtin_amdgcn_exp2f(s0.x - m_use), w1 = __builtin_amdgcn_exp2f(s1.x - m_use);
    float l = s0.y * w0 + s1.y * w1;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off);
    float x[V];
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = 0.0f;
    for (int i = wave; i < splits; i += 4 * AT_ONCE) {
        if (i != wave) fetch(i);
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
            const int at = i + 4 * n;
            if (at >= splits) break;
            const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(at < 64 ? w0 : w1), at & 63));
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] += part_of[n][v] * w;
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) part[wave][V * lane + v] = x[v];
    __syncthreads();
    const int d = threadIdx.x;
    if (d < D) out[static_cast<size_t>(row) * D + d] = float_to_bf16_bits(p < 0 ? 0.0f : ((part[0][d] + part[1][d]) + (part[2][d] + part[3][d])) / l);
}

}  // namespace terna
