// Log probabilities of given tokens, entropies and the largest alternatives of rows of logits, in one pass over them.
//
//   log p_v = x_v - m - ln s,  H = ln s - t / s,  with m = max x, s = sum exp(x - m), t = sum exp(x - m) (x - m)
//
// A thread keeps (m, s, t) of its pieces of 16 bytes and rescales by exp(m_old - m_new) a piece; threads, then splits of a row, are merged the same
// way, in a fixed order.  fp32 throughout: differences are formed before they are scaled, and the terms of -inf are held to exp(-1e4) = 0 so that
// 0 * inf does not arise.
//
// Alternatives without a second pass over everything.  Elements are in order by (value, lower index first) as 64-bit keys; NaN below all.  Sixteen lanes' pieces
// are a block of 256 contiguous bytes -- a wave's, 1024 bytes, where those would be more than LDS has room for --, whose largest value is kept (four permutations
// and a store for about 80 other instructions).  If T is a bound that k blocks' bests reach, k elements reach T, so the k best elements do, and they lie in
// blocks whose best reaches T: those alone are read again, elements that reach T go to LDS, and the k best of these are found by counting.  The order in
// which they arrive there does not matter.  Where a row is split, the launch that merges its parts does this, once a row (each part finding its own k best
// first: 8 rows of 128256 with 20 alternatives 18.2 us, so 13.5).  Bests and the bound they give are every wave's work: with one wave's, one row took 11.8 us, so 9.3.
// T is the k-th best of 64 (for k > 32: of 256) bests of blocks taken together, by bisection over the keys' bits, a ballot a bit, which ends as soon as exactly
// k reach it (10 - 15 rounds where values differ); about 1.2 k blocks reach it.  Elements go to LDS in one sweep; only where they are more than it holds are
// they taken again in rounds, with the best k kept from each to the next.  (Blocks and not, say, the pieces of a thread: those are 4 KB apart, and the
// second reading of the few that matter took three quarters of the row's lines, 17 us of 70 for 1024 x 128256.)
//
// What bounds it: many rows -- memory (1024 x 128256 in bf16, 263 MB: 49.7 us without alternatives, 5.3 TB/s; the blocks' bests 7 more, 20 alternatives 4 more;
// two pieces a thread ahead: 4 were 3 us slower, 1 12); one row -- two launches (the row split over workgroups, then merged), a trip to memory each (5.1 us)
// and the selection of the alternatives (4.2).
#pragma once

#include <type_traits>

#include "terna_common.h"

namespace terna {

constexpr int kLogprobThreads = 256;
constexpr int kLogprobMaxTop = 64;
constexpr int kLogprobBatch = 2048;            // elements that one round over the pieces can add
constexpr int kLogprobSlack = 512;             // kept between rounds
constexpr int kLogprobKeys = kLogprobBatch + kLogprobSlack;
constexpr int kLogprobBlocks = 2056;           // of a row
constexpr float kLog2e = 1.4426950408889634f;

typedef unsigned long long key64;

__device__ __forceinline__ uint32_t logprob_order(float x)                 // numbers in order, NaN below all
{
    const uint32_t b = __float_as_uint(x + 0.0f);                          // (zeros of both signs are equal)
    return x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logprob_value(uint32_t order)
{
    return order == 0 ? NAN : __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}

struct LogprobStats {
    float m, s, t;
};
// b's terms to a's.  A part without terms has m = -inf and s = t = 0.
__device__ __forceinline__ LogprobStats logprob_join(const LogprobStats& a, const LogprobStats& b)
{
    const float m = fmaxf(a.m, b.m), use = m == -INFINITY ? 0.0f : m;
    const float da = max_keep_nan(a.m - use, -1e4f), db = max_keep_nan(b.m - use, -1e4f);
    const float fa = __builtin_amdgcn_exp2f(da * kLog2e), fb = __builtin_amdgcn_exp2f(db * kLog2e);
    return {m, a.s * fa + b.s * fb, fa * (a.t + a.s * da) + fb * (b.t + b.s * db)};
}

// over the wave, in every lane: quads and rows by permutations within 16 lanes, then rows
template <typename Op>
__device__ __forceinline__ float logprob_row(float v, Op op)
{
    auto dpp = [](float x, auto control) {
        return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), decltype(control)::value, 0xf, 0xf, true));
    };
    v = op(v, dpp(v, std::integral_constant<int, 0xB1>{}));                // lanes 1 0 3 2
    v = op(v, dpp(v, std::integral_constant<int, 0x4E>{}));                // lanes 2 3 0 1
    v = op(v, dpp(v, std::integral_constant<int, 0x141>{}));               // the row's halves mirrored
    return op(v, dpp(v, std::integral_constant<int, 0x140>{}));            // the row mirrored
}
__device__ __forceinline__ float logprob_wave_max(float v) { return cross_row_reduce<true>(logprob_row(v, [](float a, float b) { return fmaxf(a, b); })); }
__device__ __forceinline__ float logprob_wave_sum(float v) { return cross_row_reduce<false>(logprob_row(v, [](float a, float b) { return a + b; })); }

template <typename T>
struct LogprobVector;
template <>
struct LogprobVector<uint16_t> {
    static constexpr int N = 8;
    static __device__ __forceinline__ float at(const u32x4& v, int e) { return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16); }
    static __device__ __forceinline__ float load(const uint16_t* p) { return bf16_bits_to_float(*p); }
};
template <>
struct LogprobVector<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ float at(const u32x4& v, int e) { return __uint_as_float(v[e]); }
    static __device__ __forceinline__ float load(const float* p) { return *p; }
};

struct LogprobArgs {
    const void* logits;
    const long long* targets;                  // or null
    float *logprob, *entropy;                  // [M]
    long long* top_ids;                        // [M][top]
    float* top_logprobs;
    float* partial;                            // splits > 1: LogprobStats [M][splits], then, where top > 0, the blocks' bests fp32 [M][blocks]
    long long ld;
    int M, V, top, splits, blocks, shift;      // a block: 2^shift pieces, 16 or 64
};

// The row as whole 16-byte pieces, its own first and last elements somewhere in the first and last of them: a piece that holds an element of the row lies in
// the allocation that does.
template <typename T>
struct LogprobRow {
    static constexpr int N = LogprobVector<T>::N;
    const u32x4* pieces;
    int lead, all;
    __device__ __forceinline__ LogprobRow(const LogprobArgs& a, int row)
    {
        const T* first = static_cast<const T*>(a.logits) + row * a.ld;
        lead = static_cast<int>((reinterpret_cast<uintptr_t>(first) & 15) / sizeof(T));
        pieces = reinterpret_cast<const u32x4*>(first - lead);
        all = (lead + a.V + N - 1) / N;
    }
};

struct LogprobSelection {
    key64 keys[kLogprobKeys];
    key64 sorted[kLogprobMaxTop], most[kLogprobThreads];
    float best[kLogprobBlocks];
    uint16_t chosen[kLogprobBlocks];
    int count, chosen_count;
};

// How many of `n` keys in LDS reach `bound`: one wave.
__device__ __forceinline__ int logprob_count(const key64* keys, int n, key64 bound, int lane)
{
    int count = 0;
    for (int i = 0; i < n; i += 64) count += __popcll(__ballot(i + lane < n && keys[i + lane] >= bound));
    return count;
}
// A bound that `want` of the wave's keys, one a lane, reach and no more (keys differ); 0 where no more than that are not 0.
__device__ __forceinline__ key64 logprob_bound64(key64 mine, int want)
{
    key64 bound = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const key64 next = bound | 1ull << bit;
        const int count = __popcll(__ballot(mine >= next));
        if (count >= want) bound = next;
        if (count == want) break;
    }
    return bound;
}
// The same for n keys in LDS, or 0 where there are no more than `want`.  One wave.
__device__ __forceinline__ key64 logprob_bound(const key64* keys, int n, int want, int lane)
{
    if (n <= want) return 0;
    key64 bound = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const key64 next = bound | 1ull << bit;
        const int count = logprob_count(keys, n, next, lane);
        if (count >= want) bound = next;
        if (count == want) break;
    }
    return bound;
}
// The keys that reach `bound` to the front, in their order; returns how many.  One wave.
__device__ __forceinline__ int logprob_compact(key64* keys, int n, key64 bound, int lane)
{
    int kept = 0;
    for (int i = 0; i < n; i += 64) {
        const key64 k = i + lane < n ? keys[i + lane] : 0;
        const bool in = i + lane < n && k >= bound;
        const key64 mask = __ballot(in);
        if (in) keys[kept + __popcll(mask & ((1ull << lane) - 1))] = k;     // (at or before where it was read, which all lanes have done)
        kept += __popcll(mask);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    return kept;
}
// The `top` best of n keys, best first, into `sorted` (zeros where there are fewer).  One wave; keys is changed.
__device__ __forceinline__ void logprob_best(key64* keys, int n, int top, key64* sorted, int lane)
{
    if (n > 64) {
        key64 most = 0;                                                    // `top` lanes' best ones reach the bound: so do `top` keys, and few more
        for (int i = lane; i < n; i += 64) most = most > keys[i] ? most : keys[i];
        n = logprob_compact(keys, n, logprob_bound64(most, top), lane);
        if (n > 64) n = logprob_compact(keys, n, logprob_bound(keys, n, top, lane), lane);
    }
    const key64 mine = lane < n ? keys[lane] : 0;
    int rank = 0;
    for (int i = 0; i < n; ++i) {
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(mine), i), hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(mine >> 32), i);
        rank += (static_cast<key64>(hi) << 32 | lo) > mine;
    }
    if (lane < top) sorted[lane] = 0;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (lane < n && rank < top) sorted[rank] = mine;
}

template <typename T>
__device__ __forceinline__ void logprob_results(const LogprobArgs& a, int row, const LogprobStats& s, const key64* sorted)
{
    const int tid = threadIdx.x;
    const bool none = s.m == -INFINITY;                                    // every logit -inf (or NaN): no distribution
    const float log_sum = none ? NAN : logf(s.s);
    if (tid == 0) {
        a.entropy[row] = log_sum - s.t / s.s;
        if (a.targets) {
            const long long v = a.targets[row];
            a.logprob[row] = v >= 0 && v < a.V ? LogprobVector<T>::load(static_cast<const T*>(a.logits) + row * a.ld + v) - s.m - log_sum : NAN;
        }
    }
    if (tid < a.top) {
        const key64 k = sorted[tid];
        a.top_ids[static_cast<size_t>(row) * a.top + tid] = static_cast<uint32_t>(~k);
        a.top_logprobs[static_cast<size_t>(row) * a.top + tid] = logprob_value(static_cast<uint32_t>(k >> 32)) - s.m - log_sum;
    }
}

// (m, s, t) of the workgroup's threads, in every thread
__device__ __forceinline__ LogprobStats logprob_join_all(LogprobStats s, LogprobStats* part)
{
    const float m = logprob_wave_max(s.m), use = m == -INFINITY ? 0.0f : m;
    const float down = max_keep_nan(s.m - use, -1e4f), f = __builtin_amdgcn_exp2f(down * kLog2e);
    const LogprobStats wave{m, logprob_wave_sum(s.s * f), logprob_wave_sum(f * __fmaf_rn(s.s, down, s.t))};
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = wave;
    __syncthreads();
    return logprob_join(logprob_join(part[0], part[1]), logprob_join(part[2], part[3]));
}

// The row's a.top best elements into h.sorted, from the blocks' bests in h.best (behind a barrier).  The whole workgroup.
template <typename T>
__device__ __forceinline__ void logprob_select(const LogprobArgs& a, const LogprobRow<T>& x, LogprobSelection& h)
{
    using Vec = LogprobVector<T>;
    constexpr int N = Vec::N, AHEAD = 2;
    const int tid = threadIdx.x, lane = tid & 63, size = 1 << a.shift, blocks = (x.all + size - 1) >> a.shift;
    if (tid == 0) h.count = 0, h.chosen_count = 0;
    auto block_key = [&](int block) __attribute__((always_inline)) {
        return static_cast<key64>(logprob_order(h.best[block])) << 32 | static_cast<uint32_t>(~block);
    };
    key64 bound = 0;
    for (int i = tid; i < blocks; i += kLogprobThreads) bound = max(bound, block_key(i));
    h.most[tid] = bound;
    __syncthreads();
    key64 most[4];                                                         // (every wave finds the bound for itself)
#pragma unroll
    for (int n = 0; n < 4; ++n) most[n] = h.most[64 * n + lane];
    if (a.top > 32) {
        bound = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const key64 next = bound | 1ull << bit;
            int count = 0;
#pragma unroll
            for (int n = 0; n < 4; ++n) count += __popcll(__ballot(most[n] >= next));
            if (count >= a.top) bound = next;
            if (count == a.top) break;
        }
    } else {
        bound = logprob_bound64(max(max(most[0], most[1]), max(most[2], most[3])), a.top);
    }
    for (int i = tid; i < blocks; i += kLogprobThreads)
        if (block_key(i) >= bound) h.chosen[atomicAdd(&h.chosen_count, 1)] = static_cast<uint16_t>(i);
    __syncthreads();
    int owners = h.chosen_count;
    auto piece_of = [&](int i, bool everybody) __attribute__((always_inline)) {             // -1: none
        const int n = i >> a.shift, piece = n < owners ? (everybody ? n : h.chosen[n]) << a.shift | (i & (size - 1)) : x.all;
        return piece < x.all ? piece : -1;
    };
    auto offer = [&](int piece, const u32x4& v) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int index = piece * N + e - x.lead;
            const uint32_t order = logprob_order(Vec::at(v, e));
            if (index >= 0 && index < a.V && (static_cast<key64>(order) << 32 | static_cast<uint32_t>(~(piece >> a.shift))) >= bound) {
                const int at = atomicAdd(&h.count, 1);
                if (at < kLogprobKeys) h.keys[at] = static_cast<key64>(order) << 32 | static_cast<uint32_t>(~index);
            }
        }
    };
    for (int from = 0; from < owners << a.shift; from += AHEAD * kLogprobThreads) {
        int piece[AHEAD];
        u32x4 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            piece[i] = piece_of(from + i * kLogprobThreads + tid, false);
            v[i] = x.pieces[max(piece[i], 0)];
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (piece[i] >= 0) offer(piece[i], v[i]);
    }
    __syncthreads();
    // Again in rounds where LDS did not hold them, and without a bound where NaN made a block's best no element.
    if (h.count > kLogprobKeys || h.count < a.top) {
        const bool everybody = h.count < a.top;
        __syncthreads();
        if (tid == 0) h.count = 0;
        if (everybody) bound = 0, owners = blocks;
        __syncthreads();
        for (int from = 0; from < owners << a.shift; from += kLogprobThreads) {
            const int piece = piece_of(from + tid, everybody);
            if (piece >= 0) offer(piece, x.pieces[piece]);
            __syncthreads();
            const int have = h.count;
            __syncthreads();                                               // (all have read it before the next round counts on)
            if (have > kLogprobSlack && from + kLogprobThreads < owners << a.shift) {      // room for the next round: only the best stay
                if (tid < 64) {
                    const int n = logprob_compact(h.keys, have, logprob_bound(h.keys, have, a.top, lane), lane);
                    if (lane == 0) h.count = n;
                }
                __syncthreads();
            }
        }
    }
    if (tid < 64) logprob_best(h.keys, h.count, a.top, h.sorted, lane);
    __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(kLogprobThreads) void terna_logprobs_kernel(LogprobArgs a)
{
    using Vec = LogprobVector<T>;
    constexpr int N = Vec::N, AHEAD = 2;
    __shared__ LogprobSelection h;
    __shared__ LogprobStats part[kLogprobThreads / 64];
    const int tid = threadIdx.x;
    const int row = blockIdx.x / a.splits, split = blockIdx.x - row * a.splits;
    const LogprobRow<T> line(a, row);
    const int lead = line.lead, all = line.all;
    const u32x4* pieces = line.pieces;
    const int share = ((all + a.splits - 1) / a.splits + 63) & ~63;        // whole blocks
    const int begin = split * share, end = min(begin + share, all);
    const int inside_from = lead ? 1 : 0, inside_to = (lead + a.V) / N;    // pieces of the row's elements alone
    float* bests = a.partial + 3 * static_cast<size_t>(a.M) * a.splits + static_cast<size_t>(row) * a.blocks;

    const int rounds = max(0, (end - begin + kLogprobThreads - 1) / kLogprobThreads);
    LogprobStats s{-INFINITY, 0.0f, 0.0f};
    auto take = [&](int round, const u32x4& v) __attribute__((always_inline)) {            // (all lanes, for the blocks' sake)
        const int piece = begin + round * kLogprobThreads + tid;
        float x[N];
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = Vec::at(v, e);
        if (piece < inside_from || piece >= min(inside_to, end)) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int at = piece * N + e - lead;
                if (at < 0 || at >= a.V || piece >= end) x[e] = -INFINITY;
            }
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < N; ++e) top = fmaxf(top, x[e]);
        if (a.top > 0) {
            float block = logprob_row(top, [](float p, float q) { return fmaxf(p, q); });
            if (a.shift == 6) block = cross_row_reduce<true>(block);
            if ((tid & ((1 << a.shift) - 1)) == 0 && piece < end) (a.splits > 1 ? bests : h.best)[piece >> a.shift] = block;
        }
        const float m = fmaxf(s.m, top), use = m == -INFINITY ? 0.0f : m;
        const float down = max_keep_nan(s.m - use, -1e4f), f = __builtin_amdgcn_exp2f(down * kLog2e);
        float sum = 0.0f, weighted = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float d = max_keep_nan(x[e] - use, -1e4f), p = __builtin_amdgcn_exp2f(d * kLog2e);
            sum += p;
            weighted = __fmaf_rn(p, d, weighted);
        }
        s.t = __fmaf_rn(f, __fmaf_rn(s.s, down, s.t), weighted);
        s.s = __fmaf_rn(s.s, f, sum);
        s.m = m;
    };
    {
        u32x4 now[AHEAD], next[AHEAD];
        auto fetch = [&](u32x4* to, int round) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) to[i] = pieces[min(begin + (round + i) * kLogprobThreads + tid, all - 1)];
        };
        int round = 0;
        if (rounds > 0) fetch(now, 0);
        for (; round + AHEAD <= rounds; round += AHEAD) {
            fetch(next, round + AHEAD);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) take(round + i, now[i]);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) now[i] = next[i];
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (round + i < rounds) take(round + i, now[i]);
    }
    s = logprob_join_all(s, part);
    if (a.splits > 1) {
        if (tid == 0) reinterpret_cast<LogprobStats*>(a.partial)[static_cast<size_t>(row) * a.splits + split] = s;
        return;
    }
    if (a.top > 0) logprob_select(a, line, h);                             // (h.best is whole behind the barrier in logprob_join_all)
    logprob_results<T>(a, row, s, h.sorted);
}

// The splits of a row, and its alternatives.
template <typename T>
__global__ __launch_bounds__(kLogprobThreads) void terna_logprobs_merge_kernel(LogprobArgs a)
{
    __shared__ LogprobSelection h;
    __shared__ LogprobStats part[kLogprobThreads / 64];
    const int tid = threadIdx.x, row = blockIdx.x;
    const LogprobRow<T> line(a, row);
    LogprobStats s{-INFINITY, 0.0f, 0.0f};
    if (tid < a.splits) s = reinterpret_cast<const LogprobStats*>(a.partial)[static_cast<size_t>(row) * a.splits + tid];
    if (a.top > 0) {
        const float* bests = a.partial + 3 * static_cast<size_t>(a.M) * a.splits + static_cast<size_t>(row) * a.blocks;
        for (int i = tid; i < (line.all + (1 << a.shift) - 1) >> a.shift; i += kLogprobThreads) h.best[i] = bests[i];
    }
    s = logprob_join_all(s, part);
    if (a.top > 0) logprob_select(a, line, h);
    logprob_results<T>(a, row, s, h.sorted);
}

}  // namespace terna
