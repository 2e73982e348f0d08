// What stands around the attention of a tree of drafted tokens (tree_attention_kernel.h): masks and depths from the nodes' parents, the branch that greedy
// decoding takes, and its keys and values to where the text ends.
//
// A tree has T nodes, a node's parent before it: parents[i] in 0 .. i - 1, or -1 for a root; with any other parent -- and behind such a node -- it is none
// (padding).  mask[i] has a bit for i and each of its ancestors, 64 nodes a word; none for padding.
#pragma once

#include "norm_quant_kernel.h"

namespace terna {

constexpr int kTreeMaxNodes = 512, kTreeThreads = 256;

// One workgroup a sequence.  Ancestors by doubling: a node takes over what the node that it points at has seen, and points where that one points;
// nine rounds for the longest chain of 512, where walking it node by node is 512 reads of LDS one after the other.  16 nodes 2.5 us, 64 sequences of 512 10.6.
template <int W>
__global__ __launch_bounds__(kTreeThreads) void terna_draft_tree_kernel(const long long* __restrict__ parents, long long* __restrict__ mask,
                                                                        long long* __restrict__ depth, int T)
{
    constexpr int NODES = 64 * W, EACH = (NODES + kTreeThreads - 1) / kTreeThreads;
    __shared__ unsigned long long seen[W][NODES];
    __shared__ int to[NODES];                                  // -1: behind a root; -2: behind padding
    const int tid = threadIdx.x;
    const long long* const of = parents + static_cast<size_t>(blockIdx.x) * T;
    for (int i = tid; i < T; i += kTreeThreads) {
        const long long p = of[i];
        to[i] = p < -1 || p >= i ? -2 : static_cast<int>(p);
#pragma unroll
        for (int w = 0; w < W; ++w) seen[w][i] = i >> 6 == w ? 1ull << (i & 63) : 0ull;
    }
    __syncthreads();
    for (int reach = 1; reach < T; reach *= 2) {
        unsigned long long more[EACH][W];
        int next[EACH];
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int i = tid + e * kTreeThreads, j = i < T ? to[i] : -1;
            next[e] = j < 0 ? j : to[j];
#pragma unroll
            for (int w = 0; w < W; ++w) more[e][w] = j < 0 ? 0ull : seen[w][j];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int i = tid + e * kTreeThreads;
            if (i >= T) continue;
            to[i] = next[e];
#pragma unroll
            for (int w = 0; w < W; ++w) seen[w][i] |= more[e][w];
        }
        __syncthreads();
    }
    for (int i = tid; i < T; i += kTreeThreads) {
        const bool node = to[i] == -1;
        const size_t at = static_cast<size_t>(blockIdx.x) * T + i;
        int above = -1;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const unsigned long long bits = node ? seen[w][i] : 0ull;
            mask[at * W + w] = static_cast<long long>(bits);
            above += __popcll(bits);
        }
        depth[at] = above;
    }
}

// ---- greedy acceptance ------------------------------------------------------------------------------------------------------------------
// Two launches: the largest logit of every node in `parts` parts of its row (index and value; equal values by lower index, NaN never: as the greedy step),
// and a workgroup a sequence that joins them, finds every node's child that carries its token, and follows those from node 0.

constexpr int kAcceptBatch = 8;                // 16-byte loads in flight per thread

struct AcceptBest {
    float value;
    int index;
};

// The larger value, of equal ones the lower index
__device__ __forceinline__ void accept_merge(float& best, int& idx, float v, int i)
{
    if (v > best || (v == best && i < idx)) {
        best = v;
        idx = i;
    }
}

// A row's elements [first, last) -- its start aligned for one element only: those in front of the first 16-byte boundary and behind the last one by one.
template <typename E>
__global__ __launch_bounds__(kTreeThreads) void terna_accept_best_kernel(const E* __restrict__ logits, long long row, AcceptBest* __restrict__ best_of, int V, int parts)
{
    constexpr int VE = 16 / sizeof(E);
    __shared__ AcceptBest of_wave[kTreeThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int node = blockIdx.x / parts, part = blockIdx.x - node * parts;
    const E* const x = logits + static_cast<size_t>(node) * row;
    const int head = min(V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(E)));
    const int pieces = (V - head) / VE, share = (pieces + parts - 1) / parts;
    const int p0 = part * share, p1 = min(p0 + share, pieces);
    const E* const body = x + head;
    float best = -INFINITY;
    int idx = 0x7fffffff;
    auto take = [&](float v, int i) __attribute__((always_inline)) {           // a thread's indices ascend: a strict compare keeps the first
        const bool better = v > best;
        best = better ? v : best;
        idx = better ? i : idx;
    };
    auto value = [](E v) __attribute__((always_inline)) {
        if constexpr (sizeof(E) == 2) return bf16_bits_to_float(v);
        else return v;
    };
    if (part == 0 && tid < head) take(value(x[tid]), tid);
    for (int base = p0; base < p1; base += kTreeThreads * kAcceptBatch) {
        u32x4 raw[kAcceptBatch];
#pragma unroll
        for (int u = 0; u < kAcceptBatch; ++u)
            raw[u] = *reinterpret_cast<const u32x4*>(body + static_cast<size_t>(min(base + u * kTreeThreads + tid, p1 - 1)) * VE);
#pragma unroll
        for (int u = 0; u < kAcceptBatch; ++u) {
            const int p = base + u * kTreeThreads + tid;
            if (p >= p1) continue;
            float f[VE];
            if constexpr (sizeof(E) == 2) unpack_bf16x8(raw[u], f);
            else {
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(raw[u][e]);
            }
#pragma unroll
            for (int e = 0; e < VE; ++e) take(f[e], head + VE * p + e);
        }
    }
    if (part == parts - 1 && head + pieces * VE + tid < V && tid < VE) take(value(x[head + pieces * VE + tid]), head + pieces * VE + tid);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) accept_merge(best, idx, __shfl_xor(best, off), __shfl_xor(idx, off));
    if (lane == 0) of_wave[wave] = AcceptBest{best, idx};
    __syncthreads();
    if (tid != 0) return;
#pragma unroll
    for (int w = 1; w < kTreeThreads / 64; ++w) accept_merge(best, idx, of_wave[w].value, of_wave[w].index);
    best_of[blockIdx.x] = AcceptBest{best, idx};
}

__global__ __launch_bounds__(kTreeThreads) void terna_accept_path_kernel(const AcceptBest* __restrict__ best_of, const long long* __restrict__ tokens,
                                                                         const long long* __restrict__ parents, long long* __restrict__ path,
                                                                         long long* __restrict__ count, long long* __restrict__ behind, int T, int parts)
{
    __shared__ int says[kTreeMaxNodes], child[kTreeMaxNodes], line[kTreeMaxNodes], length;
    const int tid = threadIdx.x;
    const size_t first = static_cast<size_t>(blockIdx.x) * T;
    for (int i = tid; i < T; i += kTreeThreads) {
        float best = -INFINITY;
        int idx = 0x7fffffff;
        for (int c = 0; c < parts; c += kAcceptBatch) {
            AcceptBest b[kAcceptBatch];
#pragma unroll
            for (int u = 0; u < kAcceptBatch; ++u) b[u] = best_of[(first + i) * parts + min(c + u, parts - 1)];
#pragma unroll
            for (int u = 0; u < kAcceptBatch; ++u) accept_merge(best, idx, b[u].value, b[u].index);
        }
        says[i] = idx == 0x7fffffff ? 0 : idx;
        child[i] = kTreeMaxNodes;
    }
    __syncthreads();
    for (int i = tid; i < T; i += kTreeThreads) {
        const long long p = parents[first + i];
        if (p >= 0 && p < i && tokens[first + i] == says[p]) atomicMin(&child[p], i);
    }
    __syncthreads();
    if (tid == 0) {
        int n = 0;
        for (int at = parents[first] == -1 ? 0 : kTreeMaxNodes; at < kTreeMaxNodes; at = child[at]) line[n++] = at;
        length = n;
        count[blockIdx.x] = n;
        behind[blockIdx.x] = n == 0 ? -1 : says[line[n - 1]];
    }
    __syncthreads();
    for (int i = tid; i < T; i += kTreeThreads) path[first + i] = i < length ? line[i] : -1;
}

// ---- moving rows of caches ------------------------------------------------------------------------------------------------------------------
// Rows start + path[i] -> start + i of every cache of a launch, i < count.  A path ascends, so that path[i] >= i and in ascending order no row is
// written before it has been read; a thread has a column of its own (a piece of a head's rows) and reads eight rows at a time.  A row outside the cache
// stays where it is.

constexpr int kMoveCaches = 64;                // of a launch: their descriptions are kernel arguments
constexpr int kMoveAhead = 8;

struct MoveCache {
    uint8_t* rows;
    long long sequence, head, slot;            // strides, bytes
    int heads, slots, pieces, piece_shift;     // pieces of 2^piece_shift bytes in a row
};
struct MoveCaches {
    MoveCache of[kMoveCaches];
};

template <typename P>
__device__ __forceinline__ void move_column(uint8_t* column, long long slot_bytes, long long start, const int* line, int n)
{
    for (int i0 = 0; i0 < n; i0 += kMoveAhead) {
        P x[kMoveAhead];
        const int here = min(n - i0, kMoveAhead);
#pragma unroll
        for (int e = 0; e < kMoveAhead; ++e)
            if (e < here && line[i0 + e] >= 0) x[e] = *reinterpret_cast<const P*>(column + (start + line[i0 + e]) * slot_bytes);
#pragma unroll
        for (int e = 0; e < kMoveAhead; ++e)
            if (e < here && line[i0 + e] >= 0) *reinterpret_cast<P*>(column + (start + i0 + e) * slot_bytes) = x[e];
    }
}

__global__ __launch_bounds__(kTreeThreads) void terna_cache_move_kernel(MoveCaches caches, const long long* __restrict__ starts, const long long* __restrict__ path,
                                                                        const long long* __restrict__ count, int T)
{
    __shared__ int line[kTreeMaxNodes];
    const MoveCache& c = caches.of[blockIdx.x];
    const int b = blockIdx.y, tid = threadIdx.x;
    const long long start = starts[b];
    const int n = static_cast<int>(min(max(count[b], 0ll), static_cast<long long>(T)));
    if (start < 0 || start >= c.slots) return;
    for (int i = tid; i < n; i += kTreeThreads) {              // -1: a row that stays
        const long long p = path[static_cast<size_t>(b) * T + i];
        line[i] = p <= i || p >= c.slots - start ? -1 : static_cast<int>(p);
    }
    __syncthreads();
    for (int x = tid; x < c.heads * c.pieces; x += kTreeThreads) {
        const int head = x / c.pieces, piece = x - head * c.pieces;
        uint8_t* const column = c.rows + b * c.sequence + head * c.head + (static_cast<long long>(piece) << c.piece_shift);
        switch (c.piece_shift) {
        case 4: move_column<u32x4>(column, c.slot, start, line, n); break;
        case 3: move_column<u32x2>(column, c.slot, start, line, n); break;
        case 2: move_column<uint32_t>(column, c.slot, start, line, n); break;
        case 1: move_column<uint16_t>(column, c.slot, start, line, n); break;
        default: move_column<uint8_t>(column, c.slot, start, line, n); break;
        }
    }
}

}  // namespace terna
