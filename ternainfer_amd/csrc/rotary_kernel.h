// Rotary positions on rows of heads: x [B][T][H][D] with any strides of its first three dimensions -> out, or in place.
//
// out[b][t][h][2j], [2j + 1] (adjacent) or [j], [j + R / 2] (half) = the pair turned by the angle of pos[t] (pos[b][t]), j < R / 2; the
// dimensions from R on are copied.
//
// What bounds it: memory -- a row is read once and written once.  A workgroup takes a few tokens with all their heads: the angles (a 64-bit
// series, about 40 instructions) are computed once a token into LDS and serve every head; its rows are requested before that.  A thread moves
// 16 bytes of a head at a time (half pairs: 16 bytes and their partners); rows that are no whole 16 bytes, or half pairs whose partners lie
// across such a piece, take the kernel of one pair a thread (2 x 1920 x 25 heads of 128 dimensions in bf16: 11.5 us by pieces, 22.5 by pairs).
// Measured: 4 x 8192 tokens of 25 heads of 128 dimensions in bf16 74.9 us, 5.6 TB/s; one token 3.4, which is the launch and two trips to memory.
#pragma once

#include "rotary_common.h"

namespace terna {

struct RotaryRows {
    long long batch, token, head;             // strides, elements
};

struct RotaryShape {
    int T, H, D, pairs, per_seq, tokens, tokens_a_group;      // tokens = B * T; a group has at most T of them where T > 1
    double amplitude;
};

// Token `first + n` of all as (sequence, token): first's by division, once a workgroup, the others from it.
struct RotaryTokens {
    int b0, t0, T;
    __device__ __forceinline__ RotaryTokens(int first, int T_) : b0(T_ > 1 ? first / T_ : first), t0(T_ > 1 ? first - b0 * T_ : 0), T(T_) {}
    __device__ __forceinline__ void of(int n, int* b, int* t) const
    {
        const int next = T > 1 ? t0 + n >= T : n;
        *b = b0 + next;
        *t = T > 1 ? t0 + n - (next ? T : 0) : 0;
    }
};

constexpr int kRotaryThreads = 256;
constexpr int kRotaryMaxAngles = 1024;         // of a workgroup: 8 KB of LDS

template <typename T>
struct RotaryVector;
template <>
struct RotaryVector<uint16_t> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const u32x4& v, float* x)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(v[i] << 16);
            x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float* x)
    {
        return u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
    }
    static __device__ __forceinline__ float load(const uint16_t* p) { return bf16_bits_to_float(*p); }
    static __device__ __forceinline__ void store(uint16_t* p, float v) { *p = float_to_bf16_bits(v); }
};
template <>
struct RotaryVector<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const u32x4& v, float* x)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(v[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float* x)
    {
        return u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    }
    static __device__ __forceinline__ float load(const float* p) { return *p; }
    static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
};

// The angles of a workgroup's tokens into LDS: cs[token][pair].
__device__ __forceinline__ void rotary_angles(float2* cs, const long long* __restrict__ pos, const double* __restrict__ frequency, const RotaryShape& s, int first, int count,
                                              const RotaryTokens& where)
{
    for (int i = threadIdx.x; i < count * s.pairs; i += kRotaryThreads) {
        const int n = i / s.pairs, j = i - n * s.pairs;
        int b, t;
        where.of(n, &b, &t);
        cs[i] = rotary_angle(pos[s.per_seq ? first + n : t], frequency[j], s.amplitude);
    }
}

// One piece of 16 bytes a thread and step.  Half pairs: a step is a piece of the lower half and its partner; pieces from R on follow.
template <typename T, bool ADJACENT>
__global__ __launch_bounds__(kRotaryThreads) void terna_rotary_kernel(const T* x, T* out, const long long* __restrict__ pos,
                                                                      const double* __restrict__ frequency, RotaryRows in, RotaryRows to, RotaryShape s, int in_place)
{
    using V = RotaryVector<T>;
    constexpr int N = V::N;
    __shared__ float2 cs[kRotaryMaxAngles];
    const int first = blockIdx.x * s.tokens_a_group;
    const int count = min(s.tokens_a_group, s.tokens - first);
    const RotaryTokens where(first, s.T);
    // pieces of a head: adjacent -- all D / N (in place: those that hold a pair); half -- R / 2 / N pairs of pieces, then the rest
    const int turning = ADJACENT ? (2 * s.pairs + N - 1) / N : s.pairs / N;
    const int pieces = in_place ? turning : ADJACENT ? s.D / N : s.D / N - turning;
    const int heads = count * s.H, total = heads * pieces;
    const int y_step = gridDim.y * kRotaryThreads;
    int i = blockIdx.y * kRotaryThreads + threadIdx.x;
    struct Piece { const T* from; T* to; int n, at; u32x4 own, other; };
    auto fetch = [&](int i) __attribute__((always_inline)) {
        Piece p;
        const int head = i / pieces;
        p.at = i - head * pieces;
        p.n = head / s.H;
        const int h = head - p.n * s.H;
        int b, t;
        where.of(p.n, &b, &t);
        p.from = x + b * in.batch + t * in.token + h * in.head;
        p.to = out + b * to.batch + t * to.token + h * to.head;
        const bool turns = ADJACENT || p.at < turning;
        const int d = turns ? p.at * N : (p.at + turning) * N;
        p.own = *reinterpret_cast<const u32x4*>(p.from + d);
        p.other = p.own;
        if (!ADJACENT && turns) p.other = *reinterpret_cast<const u32x4*>(p.from + d + s.pairs);
        return p;
    };
    Piece p{};
    if (i < total) p = fetch(i);
    rotary_angles(cs, pos, frequency, s, first, count, where);
    __syncthreads();
    for (; i < total;) {
        const float2* angle = cs + p.n * s.pairs;
        float a[N], b[N];
        V::unpack(p.own, a);
        if constexpr (ADJACENT) {
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
                const int j = p.at * (N / 2) + e;
                if (j < s.pairs) {
                    const float2 y = rotary_turn(a[2 * e], a[2 * e + 1], angle[j]);
                    a[2 * e] = y.x;
                    a[2 * e + 1] = y.y;
                }
            }
            *reinterpret_cast<u32x4*>(p.to + p.at * N) = V::pack(a);
        } else if (p.at < turning) {
            V::unpack(p.other, b);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float2 y = rotary_turn(a[e], b[e], angle[p.at * N + e]);
                a[e] = y.x;
                b[e] = y.y;
            }
            *reinterpret_cast<u32x4*>(p.to + p.at * N) = V::pack(a);
            *reinterpret_cast<u32x4*>(p.to + p.at * N + s.pairs) = V::pack(b);
        } else {
            *reinterpret_cast<u32x4*>(p.to + (p.at + turning) * N) = p.own;
        }
        i += y_step;
        if (i < total) p = fetch(i);
    }
}

// One pair, or one element behind them, a thread and step: any alignment.
template <typename T, bool ADJACENT>
__global__ __launch_bounds__(kRotaryThreads) void terna_rotary_pairs_kernel(const T* x, T* out, const long long* __restrict__ pos,
                                                                            const double* __restrict__ frequency, RotaryRows in, RotaryRows to, RotaryShape s, int in_place)
{
    using V = RotaryVector<T>;
    __shared__ float2 cs[kRotaryMaxAngles];
    const int first = blockIdx.x * s.tokens_a_group;
    const int count = min(s.tokens_a_group, s.tokens - first);
    const RotaryTokens where(first, s.T);
    rotary_angles(cs, pos, frequency, s, first, count, where);
    __syncthreads();
    const int pieces = in_place ? s.pairs : s.D - s.pairs;             // pairs, then single elements
    const int total = count * s.H * pieces;
    for (int i = blockIdx.y * kRotaryThreads + threadIdx.x; i < total; i += gridDim.y * kRotaryThreads) {
        const int head = i / pieces, at = i - head * pieces, n = head / s.H, h = head - n * s.H;
        int b, t;
        where.of(n, &b, &t);
        const T* from = x + b * in.batch + t * in.token + h * in.head;
        T* dest = out + b * to.batch + t * to.token + h * to.head;
        if (at < s.pairs) {
            const int d0 = ADJACENT ? 2 * at : at, d1 = ADJACENT ? 2 * at + 1 : at + s.pairs;
            const float2 y = rotary_turn(V::load(from + d0), V::load(from + d1), cs[n * s.pairs + at]);
            V::store(dest + d0, y.x);
            V::store(dest + d1, y.y);
        } else {
            dest[s.pairs + at] = from[s.pairs + at];
        }
    }
}

}  // namespace terna
