// C ABI of decoding with a tree of drafted tokens: masks of a tree, attention over the cache, greedy acceptance, moving cache rows.
// Declarations: include/ternaspmm.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>

#include "../../include/ternaspmm.h"
#include "host_util.h"
#include "tree_attention_kernel.h"

using namespace terna;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool tree_nodes_ok(int B, int T) { return B >= 1 && T >= 1 && T <= kTreeMaxNodes && launch_fits(B, kTreeThreads); }

bool tree_shape_ok(int B, int T, int H, int KV, int D, int S)
{
    if (!tree_nodes_ok(B, T) || H < 1 || KV < 1 || H % KV != 0 || (D != 64 && D != 128) || S < 1 || S > 1 << 25 || H > 4096 || static_cast<long long>(B) * T * H > 1 << 28) return false;
    const TreePlan plan = tree_plan(B, T, H, KV, D, S);
    return launch_fits(tree_blocks(static_cast<long long>(B) * KV * plan.splits, plan.tiles), 512);
}
// Strides in elements of rows that are read 16 bytes at a time.
bool strides_ok(const long long* s, int n)
{
    for (int i = 0; i < n; ++i)
        if (s[i] < 0 || (s[i] & 7)) return false;
    return true;
}

template <int D, int RW, int KW, int ST, int PER_SIMD>
void launch_tree(const TreeAttention& a, long long grid, hipStream_t st)
{
    using Shape = TreeShape<D, RW, KW, ST>;
    auto kernel = terna_tree_attention_kernel<D, RW, KW, ST, PER_SIMD>;
    if (Shape::kBytes > kPlainLds - 4096) allow_dynamic_lds(kernel, Shape::kBytes, "hipFuncSetAttribute(tree attention)", __LINE__);
    launch(kernel, dim3(static_cast<unsigned>(grid)), dim3(Shape::kThreads), Shape::kBytes, st, a);
}
template <int D>
void launch_tree_attention(const TreeAttention& a, const TreePlan& plan, long long grid, hipStream_t st)
{
    if (plan.rows == 32) launch_tree<D, 1, 4, D == 128 ? 2 : 4, 1>(a, grid, st);
    else if (plan.rows == 64) launch_tree<D, 2, 2, D == 128 ? 2 : 4, 2>(a, grid, st);
    else if (plan.groups == 1) launch_tree<D, 4, 1, 4, 2>(a, grid, st);
    else launch_tree<D, 4, 2, 4, 2>(a, grid, st);
    if (a.parts != 0) {
        const int all = a.T * a.H;
        launch(terna_tree_merge_kernel<D>, dim3((a.B * all + 3) / 4), dim3(256), 0, st, a.partial, a.out, a.B, all, a.parts);
    }
}

// Parts of a row of logits: up to eight workgroups a CU, of a round of loads at least (acceptance of
// 16 rows of 128256 with one part each 16.1 us, so 7.0; of 512 28.9, so 28.6).
int accept_parts(long long rows, int V, int fp32)
{
    const int pieces = V / (fp32 ? 4 : 8), round = kTreeThreads * kAcceptBatch;
    int parts = 1;
    while (parts < 64 && 2 * rows * parts <= 2048 && pieces > parts * round) parts *= 2;
    return parts;
}
bool accept_shape_ok(int B, int T, int V, int fp32) { return tree_nodes_ok(B, T) && V >= 1 && V <= 1 << 19 && launch_fits(static_cast<long long>(B) * T * accept_parts(static_cast<long long>(B) * T, V, fp32), kTreeThreads); }

}  // namespace

extern "C" {

int ternaspmm_draft_tree(const long long* parents, long long* mask, long long* depth, int B, int T, terna_stream stream)
{
    if (!tree_nodes_ok(B, T) || !parents || !mask || !depth) return -1;
    void (*const kernels[])(const long long*, long long*, long long*, int) = {terna_draft_tree_kernel<1>, terna_draft_tree_kernel<2>, terna_draft_tree_kernel<3>,
                                                                              terna_draft_tree_kernel<4>, terna_draft_tree_kernel<5>, terna_draft_tree_kernel<6>,
                                                                              terna_draft_tree_kernel<7>, terna_draft_tree_kernel<8>};
    launch(kernels[(T + 63) / 64 - 1], dim3(B), dim3(kTreeThreads), 0, static_cast<hipStream_t>(stream), parents, mask, depth, T);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die("ternaspmm_draft_tree", e, __LINE__);
    return 0;
}

long long ternaspmm_tree_attention_workspace_bytes(int B, int T, int H, int KV, int D, int S)
{
    if (!tree_shape_ok(B, T, H, KV, D, S)) return -1;
    const int splits = tree_plan(B, T, H, KV, D, S).splits;
    return splits == 1 ? 0 : 4ll * B * T * H * splits * (D + 2) + static_cast<long long>(sizeof(TreeShare)) * B;
}

int ternaspmm_tree_attention(const terna_bf16* q, const long long* q_strides, const terna_bf16* k, const long long* k_strides, const terna_bf16* v, const long long* v_strides,
                             const long long* start, const long long* mask, int per_sequence, terna_bf16* out, void* workspace, int B, int T, int H, int KV, int D, int S,
                             float scale, terna_stream stream)
{
    if (!tree_shape_ok(B, T, H, KV, D, S) || !q || !k || !v || !start || !mask || !out || !q_strides || !k_strides || !v_strides || !aligned16(q) || !aligned16(k) || !aligned16(v) ||
        !aligned16(out) || !aligned16(workspace) || !strides_ok(q_strides, 3) || !strides_ok(k_strides, 3) || !strides_ok(v_strides, 3) || !std::isfinite(scale * static_cast<float>(M_LOG2E)) ||
        k_strides[2] >= 1 << 24 || v_strides[2] >= 1 << 24)
        return -1;
    const TreePlan plan = tree_plan(B, T, H, KV, D, S);
    TreeAttention a{};
    a.q = q, a.k = k, a.v = v, a.start = start, a.mask = mask, a.out = out, a.partial = static_cast<float*>(workspace);
    a.q_seq = q_strides[0], a.q_head = q_strides[1], a.q_node = q_strides[2];
    a.k_seq = k_strides[0], a.k_head = k_strides[1], a.k_slot = static_cast<int>(2 * k_strides[2]);
    a.v_seq = v_strides[0], a.v_head = v_strides[1], a.v_slot = static_cast<int>(2 * v_strides[2]);
    a.B = B, a.T = T, a.H = H, a.KV = KV, a.S = S, a.W = (T + 63) / 64, a.per_seq = per_sequence != 0;
    a.parts = workspace && plan.splits > 1 ? B * plan.splits : 0, a.tiles = plan.tiles;
    a.scale = scale * static_cast<float>(M_LOG2E);
    const long long grid = tree_blocks(static_cast<long long>(a.parts == 0 ? B : a.parts) * KV, plan.tiles);
    if (D == 128) launch_tree_attention<128>(a, plan, grid, static_cast<hipStream_t>(stream));
    else launch_tree_attention<64>(a, plan, grid, static_cast<hipStream_t>(stream));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die("ternaspmm_tree_attention", e, __LINE__);
    return 0;
}

long long ternaspmm_tree_accept_workspace_bytes(int B, int T, int V, int fp32)
{
    return accept_shape_ok(B, T, V, fp32) ? static_cast<long long>(sizeof(AcceptBest)) * B * T * accept_parts(static_cast<long long>(B) * T, V, fp32) : -1;
}

int ternaspmm_tree_accept(const void* logits, long long row, int fp32, const long long* tokens, const long long* parents, long long* path, long long* count, long long* next,
                          void* workspace, int B, int T, int V, terna_stream stream)
{
    if (!accept_shape_ok(B, T, V, fp32) || !logits || !tokens || !parents || !path || !count || !next || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 7) || row < 0 ||
        (reinterpret_cast<uintptr_t>(logits) & (fp32 ? 3 : 1)))
        return -1;
    const int parts = accept_parts(static_cast<long long>(B) * T, V, fp32);
    AcceptBest* const best = static_cast<AcceptBest*>(workspace);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (fp32) launch(terna_accept_best_kernel<float>, dim3(B * T * parts), dim3(kTreeThreads), 0, st, static_cast<const float*>(logits), row, best, V, parts);
    else launch(terna_accept_best_kernel<uint16_t>, dim3(B * T * parts), dim3(kTreeThreads), 0, st, static_cast<const uint16_t*>(logits), row, best, V, parts);
    launch(terna_accept_path_kernel, dim3(B), dim3(kTreeThreads), 0, st, best, tokens, parents, path, count, next, T, parts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die("ternaspmm_tree_accept", e, __LINE__);
    return 0;
}

int ternaspmm_cache_move(const ternaspmm_cache_rows* caches, int n, const long long* start, const long long* path, const long long* count, int B, int T, terna_stream stream)
{
    if (n < 0 || !tree_nodes_ok(B, T) || B > 65535 || !start || !path || !count || (n > 0 && !caches)) return -1;
    for (int i = 0; i < n; ++i) {
        const ternaspmm_cache_rows& c = caches[i];
        if (!c.rows || c.heads < 1 || c.slots < 1 || c.bytes < 1 || c.slot < c.bytes || c.head < 0 || c.sequence < 0 || static_cast<long long>(c.heads) * c.bytes > 1ll << 30)
            return -1;
    }
    MoveCaches m{};
    for (int i0 = 0; i0 < n; i0 += kMoveCaches) {
        const int here = std::min(n - i0, kMoveCaches);
        for (int i = 0; i < here; ++i) {
            const ternaspmm_cache_rows& c = caches[i0 + i];
            // the widest access that its addresses and strides allow
            const unsigned long long all = reinterpret_cast<uintptr_t>(c.rows) | c.sequence | c.head | c.slot | static_cast<unsigned long long>(c.bytes);
            const int shift = (all & 15) == 0 ? 4 : (all & 7) == 0 ? 3 : (all & 3) == 0 ? 2 : (all & 1) == 0 ? 1 : 0;
            m.of[i] = MoveCache{static_cast<uint8_t*>(c.rows), c.sequence, c.head, c.slot, c.heads, c.slots, c.bytes >> shift, shift};
        }
        launch(terna_cache_move_kernel, dim3(here, B), dim3(kTreeThreads), 0, static_cast<hipStream_t>(stream), m, start, path, count, T);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) die("ternaspmm_cache_move", e, __LINE__);
    }
    return 0;
}

}  // extern "C"
