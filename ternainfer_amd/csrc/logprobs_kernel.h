// Log probabilities of given tokens, entropies and the largest alternatives of rows of logits, in one pass over them.
//
//   log p_v = x_v - m - ln s,  H = ln s - t / s,  with m = max x, s = sum exp(x - m), t = sum exp(x - m) (x - m)
//
// A thread keeps (m, s, t) of its pieces of 16 bytes and rescales by exp(m_old - m_new) a piece; threads, then splits of a row, are merged the same
// way, in a fixed order.  fp32 throughout: differences are formed before they are scaled, and the terms of -inf are held to exp(-1e4) = 0 so that
// 0 * inf does not arise.
//
// Alternatives without a second pass over everything.  Elements are in order by (value, lower index first) as 64-bit keys; NaN below all.  Sixteen lanes' pieces
// are a block of 256 contiguous bytes, whose largest value goes to LDS (four permutations and a store for about 80 other instructions).  If T is a bound that
// k blocks' bests reach, k elements reach T, so the k best elements do, and they lie in blocks whose best reaches T: those alone are read again, elements
// that reach T go to LDS, and the k best of these are found by counting.  The order in which they arrive there does not matter.
// T is the k-th best of 64 (for k > 32: of 256) bests of blocks taken together, by bisection over the keys' bits, a ballot a bit, which ends as soon as exactly
// k reach it (10 - 15 rounds where values differ); about 1.2 k blocks reach it.  Elements go to LDS in one sweep; only where they are more than it holds are
// they taken again in rounds, with the best k kept from each to the next.  (Blocks and not, say, the pieces of a thread: those are 4 KB apart, and the
// second reading of the few that matter took three quarters of the row's lines, 17 us of 70 for 1024 x 128256.)
//
// What bounds it: many rows -- memory (vector work: 11 issue slots an element against 64 a clock and CU); one row -- two launches (the row split over
// workgroups, then merged), a trip to memory each and the selection of the alternatives.
#pragma once

#include <type_traits>

#include "terna_common.h"

namespace terna {

constexpr int kLogprobThreads = 256;
constexpr int kLogprobMaxTop = 64;
constexpr int kLogprobBatch = 2048;            // elements that one round over the pieces can add
constexpr int kLogprobSlack = 512;             // kept between rounds
constexpr int kLogprobKeys = kLogprobBatch + kLogprobSlack;
constexpr int kLogprobBlocks = 2048;           // of a workgroup: 16 pieces each
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
    void* partial;                             // splits > 1: key64 [M][splits][top], then LogprobStats [M][splits]
    long long ld;
    int M, V, top, splits;
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

template <typename T>
__global__ __launch_bounds__(kLogprobThreads) void terna_logprobs_kernel(LogprobArgs a)
{
    using Vec = LogprobVector<T>;
    constexpr int N = Vec::N, AHEAD = 4;
    __shared__ key64 keys[kLogprobKeys];
    __shared__ key64 sorted[kLogprobMaxTop];
    __shared__ LogprobStats part[kLogprobThreads / 64];
    __shared__ float best[kLogprobBlocks];
    __shared__ uint16_t chosen[kLogprobBlocks];
    __shared__ key64 bound_of;
    __shared__ int count_of, chosen_count;
    const int tid = threadIdx.x, lane = tid & 63;
    const int row = blockIdx.x / a.splits, split = blockIdx.x - row * a.splits;
    // The row as whole 16-byte pieces, its own first and last elements somewhere in the first and last of them: a piece that holds an element of the
    // row lies in the allocation that does.
    const T* first = static_cast<const T*>(a.logits) + row * a.ld;
    const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(first) & 15) / sizeof(T));
    const u32x4* pieces = reinterpret_cast<const u32x4*>(first - lead);
    const int all = (lead + a.V + N - 1) / N, share = (all + a.splits - 1) / a.splits;
    const int begin = split * share, end = min(begin + share, all);
    const int inside_from = lead ? 1 : 0, inside_to = (lead + a.V) / N;    // pieces of the row's elements alone

    const int rounds = max(0, (end - begin + kLogprobThreads - 1) / kLogprobThreads), blocks = max(0, (end - begin + 15) / 16);
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
            const float block = logprob_row(top, [](float p, float q) { return fmaxf(p, q); });
            if ((tid & 15) == 0 && piece < end) best[(piece - begin) >> 4] = block;
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

    const int in_range = max(0, min(end * N - lead, a.V) - max(begin * N - lead, 0));       // elements of this split
    const int want = min(a.top, in_range);
    if (a.top > 0) {
        if (tid == 0) count_of = 0;                                        // (`best` is whole behind the barrier in logprob_join_all)
        auto block_key = [&](int block) __attribute__((always_inline)) {
            return static_cast<key64>(logprob_order(best[block])) << 32 | static_cast<uint32_t>(~block);
        };
        if (tid < 64) {
            key64 b = 0;
            if (want > 32) {
                key64 most[4] = {0, 0, 0, 0};
                for (int i = 0; i < blocks; i += 256)
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        if (i + 64 * n + lane < blocks) most[n] = max(most[n], block_key(i + 64 * n + lane));
                for (int bit = 63; bit >= 0; --bit) {
                    const key64 next = b | 1ull << bit;
                    int count = 0;
#pragma unroll
                    for (int n = 0; n < 4; ++n) count += __popcll(__ballot(most[n] >= next));
                    if (count >= want) b = next;
                    if (count == want) break;
                }
            } else if (want > 0) {
                key64 most = 0;
                for (int i = lane; i < blocks; i += 64) most = max(most, block_key(i));
                b = logprob_bound64(most, want);
            }
            int n = 0;
            for (int i = 0; i < blocks; i += 64) {
                const bool in = i + lane < blocks && block_key(i + lane) >= b;
                const key64 mask = __ballot(in);
                if (in) chosen[n + __popcll(mask & ((1ull << lane) - 1))] = static_cast<uint16_t>(i + lane);
                n += __popcll(mask);
            }
            if (lane == 0) bound_of = b, chosen_count = n;
        }
        __syncthreads();
        key64 bound = bound_of;
        int owners = chosen_count;
        auto piece_of = [&](int i, bool everybody) __attribute__((always_inline)) {         // -1: none
            const int n = i >> 4, piece = n < owners ? begin + (everybody ? n : chosen[n]) * 16 + (i & 15) : end;
            return piece < end ? piece : -1;
        };
        auto offer = [&](int piece, const u32x4& v) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int index = piece * N + e - lead;
                const uint32_t order = logprob_order(Vec::at(v, e));
                if (index >= 0 && index < a.V && (static_cast<key64>(order) << 32 | static_cast<uint32_t>(~((piece - begin) >> 4))) >= bound) {
                    const int at = atomicAdd(&count_of, 1);
                    if (at < kLogprobKeys) keys[at] = static_cast<key64>(order) << 32 | static_cast<uint32_t>(~index);
                }
            }
        };
        for (int from = 0; from < owners * 16; from += AHEAD * kLogprobThreads) {
            int piece[AHEAD];
            u32x4 v[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                piece[i] = piece_of(from + i * kLogprobThreads + tid, false);
                v[i] = pieces[max(piece[i], 0)];
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (piece[i] >= 0) offer(piece[i], v[i]);
        }
        __syncthreads();
        // Again in rounds where LDS did not hold them, and without a bound where NaN made a block's best no element.
        if (count_of > kLogprobKeys || count_of < want) {
            const bool everybody = count_of < want;
            __syncthreads();
            if (tid == 0) count_of = 0;
            if (everybody) bound = 0, owners = blocks;
            __syncthreads();
            for (int from = 0; from < owners * 16; from += kLogprobThreads) {
                const int piece = piece_of(from + tid, everybody);
                if (piece >= 0) offer(piece, pieces[piece]);
                __syncthreads();
                const int have = count_of;
                __syncthreads();                                           // (all have read it before the next round counts on)
                if (have > kLogprobSlack && from + kLogprobThreads < owners * 16) {      // room for the next round: only the best stay
                    if (tid < 64) {
                        const int n = logprob_compact(keys, have, logprob_bound(keys, have, want, lane), lane);
                        if (lane == 0) count_of = n;
                    }
                    __syncthreads();
                }
            }
        }
        if (tid < 64) logprob_best(keys, count_of, a.top, sorted, lane);
        __syncthreads();
    }
    if (a.splits == 1) {
        logprob_results<T>(a, row, s, sorted);
    } else {
        const size_t slot = static_cast<size_t>(row) * a.splits + split;
        key64* to = static_cast<key64*>(a.partial);
        if (tid < a.top) to[slot * a.top + tid] = sorted[tid];
        if (tid == 0) reinterpret_cast<LogprobStats*>(to + static_cast<size_t>(a.M) * a.splits * a.top)[slot] = s;
    }
}

// The splits of a row.
template <typename T>
__global__ __launch_bounds__(kLogprobThreads) void terna_logprobs_merge_kernel(LogprobArgs a)
{
    __shared__ key64 keys[kLogprobKeys];
    __shared__ key64 sorted[kLogprobMaxTop];
    __shared__ LogprobStats part[kLogprobThreads / 64];
    const int tid = threadIdx.x, row = blockIdx.x, n = a.splits * a.top;
    const key64* from = static_cast<const key64*>(a.partial) + static_cast<size_t>(row) * n;
    const LogprobStats* stats = reinterpret_cast<const LogprobStats*>(static_cast<const key64*>(a.partial) + static_cast<size_t>(a.M) * n) + static_cast<size_t>(row) * a.splits;
    for (int i = tid; i < n; i += kLogprobThreads) keys[i] = from[i];
    LogprobStats s{-INFINITY, 0.0f, 0.0f};
    if (tid < a.splits) s = stats[tid];
    s = logprob_join_all(s, part);
    if (a.top > 0) {
        if (tid < 64) logprob_best(keys, n, a.top, sorted, tid);
        __syncthreads();
    }
    logprob_results<T>(a, row, s, sorted);
}

}  // namespace terna
