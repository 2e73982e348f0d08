// C ABI of the 4-bit key/value cache: store, rows of it, attention of few and of many query rows, the single-token step (kv4_*_kernel.h).
// Declarations: include/ternaspmm.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>

#include "../../include/ternaspmm.h"
#include "host_util.h"
#include "kv4_plan.h"
#include "kv4_prefill_kernel.h"

using namespace terna;

namespace {

bool kv4_shape_ok(int B, int T, int H, int KV, int D, int S)
{
    return B >= 1 && T >= 1 && H >= 1 && KV >= 1 && H % KV == 0 && (D == 64 || D == 128) && S >= 1 && S <= 1 << 25 && H <= 4096 &&
           static_cast<long long>(B) * T <= 1 << 24 && static_cast<long long>(B) * T * H <= 1 << 28;
}
// Workgroups of the attention's launch: a kv head's tiles of rows eight apart (few rows), or its row blocks in `parts` rounds over the XCDs (many).
long long kv4_workgroups(long long heads_and_splits, int tiles, bool many, int* parts)
{
    if (!many) return (heads_and_splits + 7) / 8 * 8 * tiles;
    const int rounds = (tiles + 7) / 8;
    *parts = (tiles + rounds - 1) / rounds;
    return 8 * ((heads_and_splits * *parts + 7) / 8) * rounds;
}
// The attention's shapes: those that a launch of few rows has room for, in one part and by four waves (more parts, or eight, are only taken where all workgroups
// together are a few hundred).  One of many rows, which there are above 32, has fewer threads: 512 for 128 rows, where few take 256 for 16.
bool kv4_attention_ok(int B, int T, int H, int KV, int D, int S)
{
    if (!kv4_shape_ok(B, T, H, KV, D, S)) return false;
    return launch_fits(kv4_workgroups(static_cast<long long>(B) * KV, kv4_tiles(static_cast<long long>(T) * (H / KV), false), false, nullptr), 256);
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool kv4_cache_ok(const ternaspmm_kv4* c) { return c && c->k && c->k_scale && c->v && c->v_scale && aligned16(c->k) && aligned16(c->v) &&
                                                           ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 3) == 0; }

template <int D, bool STEP>
void launch_kv4_few(const Kv4Attention& a, int waves, int adjacent, long long grid, hipStream_t st)
{
    auto kernel = waves == 8 ? terna_kv4_attention_kernel<D, STEP, true, 8> : terna_kv4_attention_kernel<D, STEP, true, 4>;
    if constexpr (STEP) {
        if (!adjacent) kernel = waves == 8 ? terna_kv4_attention_kernel<D, true, false, 8> : terna_kv4_attention_kernel<D, true, false, 4>;
    }
    launch(kernel, dim3(static_cast<unsigned>(grid)), dim3(64 * waves), 0, st, a);
}

template <bool STEP>
void launch_kv4_attention(const char* who, Kv4Attention a, int D, int adjacent, hipStream_t st)
{
    const Kv4Plan plan = kv4_plan(a.B, a.T, a.H, a.KV, D, a.S);
    a.splits = a.partial ? plan.splits : 1;
    // (one token without a workspace by few rows, so that a step, which has no room there for turned queries, is the same)
    const bool many = !STEP && plan.many && (a.T > 1 || a.partial);
    a.tiles = kv4_tiles(static_cast<long long>(a.T) * (a.H / a.KV), many);
    const long long groups = static_cast<long long>(a.B) * a.KV * a.splits;
    const long long grid = kv4_workgroups(groups, a.tiles, many, &a.parts);
    if (many) {
        const int lds = D == 128 ? Kv4PrefillLds<128>::kBytes : Kv4PrefillLds<64>::kBytes;
        auto kernel = D == 128 ? terna_kv4_prefill_kernel<128> : terna_kv4_prefill_kernel<64>;
        if (lds > kPlainLds - 4096) allow_dynamic_lds(kernel, lds, "hipFuncSetAttribute(4-bit attention)", __LINE__);
        launch(kernel, dim3(grid), dim3(512), lds, st, a);
    } else {
        if (D == 128) launch_kv4_few<128, STEP>(a, plan.waves, adjacent, grid, st);
        else launch_kv4_few<64, STEP>(a, plan.waves, adjacent, grid, st);
    }
    if (a.splits > 1)
        launch(D == 128 ? terna_kv4_merge_kernel<128> : terna_kv4_merge_kernel<64>, dim3(a.B * a.T * a.H), dim3(256), 0, st, a.partial, a.pos, a.out, a.T, a.H, a.splits,
               a.per_seq);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die(who, e, __LINE__);
}

// Of the workspace of one new token: the queries that a step by many rows stores in front of the parts.
long long kv4_query_bytes(int B, int T, int H, int KV, int D, int S) { return T == 1 && kv4_plan(B, T, H, KV, D, S).many ? 2ll * B * H * D : 0; }

}  // namespace

extern "C" {

int ternaspmm_kv4_splits(int B, int T, int H, int KV, int D, int S)
{
    if (!kv4_attention_ok(B, T, H, KV, D, S)) return -1;
    return kv4_plan(B, T, H, KV, D, S).splits;
}

long long ternaspmm_kv4_workspace_bytes(int B, int T, int H, int KV, int D, int S)
{
    if (!kv4_attention_ok(B, T, H, KV, D, S)) return -1;
    const int splits = kv4_plan(B, T, H, KV, D, S).splits;
    return kv4_query_bytes(B, T, H, KV, D, S) + (splits == 1 ? 0 : 4ll * B * T * H * splits * (D + 2));
}

int ternaspmm_kv4_store(const terna_bf16* qkv, long long row, const long long* pos, int per_sequence, const double* frequency, int pairs, double amplitude,
                        terna_bf16* q_out, const ternaspmm_kv4* cache, int B, int T, int H, int KV, int D, int S, int adjacent, terna_stream stream)
{
    if (!kv4_shape_ok(B, T, H, KV, D, S) || !kv4_cache_ok(cache) || !qkv || !pos || !frequency || !q_out || pairs < 1 || 2 * pairs > D || row < (H + 2ll * KV) * D || (row & 7) ||
        !aligned16(qkv) || !aligned16(q_out) || KV > 4096)
        return -1;
    RotaryShape s{T, H, D, pairs, per_sequence != 0, B * T, 1, amplitude};
    const int steps = (H + 2 * KV) * (D / 8);
    // Tokens a workgroup: as for ternaspmm_rotary; half pairs, whose pieces are read twice, twice as many (us, 4 x 8192 tokens of 30 heads adjacent 91.2, with
    // twice as many 96.5; 2 x 4096 of 48 half 49.1, with half as many 52.9).
    while (2 * s.tokens_a_group * pairs <= kRotaryMaxAngles && (adjacent ? 2 : 1) * s.tokens_a_group * steps <= 4 * kRotaryThreads && s.tokens / (2 * s.tokens_a_group) >= 512 &&
           (T == 1 || 2 * s.tokens_a_group <= T))
        s.tokens_a_group *= 2;
    const int groups = (s.tokens + s.tokens_a_group - 1) / s.tokens_a_group;
    if (!launch_fits(groups, kRotaryThreads)) return -1;
    int slices = 1;
    while (slices < 64 && groups * slices < 512 && 2 * slices * kRotaryThreads <= s.tokens_a_group * steps) slices *= 2;
    auto kernel = D == 128 ? (adjacent ? terna_kv4_store_kernel<128, true> : terna_kv4_store_kernel<128, false>)
                           : (adjacent ? terna_kv4_store_kernel<64, true> : terna_kv4_store_kernel<64, false>);
    launch(kernel, dim3(groups, slices), dim3(kRotaryThreads), 0, static_cast<hipStream_t>(stream), qkv, pos, frequency, q_out, cache->k, cache->k_scale, cache->v,
           cache->v_scale, s, KV, S, row);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die("ternaspmm_kv4_store", e, __LINE__);
    return 0;
}

int ternaspmm_kv4_rows(const ternaspmm_kv4* cache, const long long* pos, int per_sequence, terna_bf16* k_out, terna_bf16* v_out, int B, int T, int KV, int D, int S,
                       terna_stream stream)
{
    if (!kv4_shape_ok(B, T, KV, KV, D, S) || !kv4_cache_ok(cache) || !pos || !k_out || !v_out || !aligned16(k_out) || !aligned16(v_out)) return -1;
    // two steps a thread, and no fewer workgroups than the CUs; a group has at most T tokens of them where T > 1
    const int tokens = B * T, most = T > 1 ? T : tokens, tokens_a_group = std::max(1, std::min({512 / (2 * KV * (D / 8)), most, tokens / 512}));
    const int groups = (tokens + tokens_a_group - 1) / tokens_a_group;
    if (!launch_fits(groups, 256)) return -1;
    launch(terna_kv4_rows_kernel, dim3(groups), dim3(256), 0, static_cast<hipStream_t>(stream), cache->k, cache->k_scale, cache->v,
           cache->v_scale, pos, k_out, v_out, T, KV, S, D, per_sequence != 0, tokens, tokens_a_group);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die("ternaspmm_kv4_rows", e, __LINE__);
    return 0;
}

int ternaspmm_kv4_attention(const terna_bf16* q, const ternaspmm_kv4* cache, const long long* pos, int per_sequence, terna_bf16* out, void* workspace, int B, int T, int H,
                            int KV, int D, int S, float scale, terna_stream stream)
{
    if (!kv4_attention_ok(B, T, H, KV, D, S) || !kv4_cache_ok(cache) || !q || !pos || !out || !aligned16(q) || !aligned16(out) || !aligned16(workspace)) return -1;
    Kv4Attention a{};
    a.q = q, a.k = cache->k, a.k_scale = cache->k_scale, a.v = cache->v, a.v_scale = cache->v_scale, a.pos = pos, a.out = out, a.partial = static_cast<float*>(workspace);
    a.B = B, a.T = T, a.H = H, a.KV = KV, a.S = S, a.per_seq = per_sequence != 0;
    a.scale = scale * static_cast<float>(M_LOG2E);
    launch_kv4_attention<false>("ternaspmm_kv4_attention", a, D, 1, static_cast<hipStream_t>(stream));
    return 0;
}

int ternaspmm_kv4_step(const terna_bf16* qkv, long long row, const long long* pos, int per_sequence, const double* frequency, int pairs, double amplitude,
                       const ternaspmm_kv4* cache, terna_bf16* out, void* workspace, int B, int H, int KV, int D, int S, float scale, int adjacent, terna_stream stream)
{
    if (!kv4_attention_ok(B, 1, H, KV, D, S) || !kv4_cache_ok(cache) || !qkv || !pos || !frequency || !out || pairs < 1 || 2 * pairs > D || row < (H + 2ll * KV) * D || (row & 7) ||
        !aligned16(qkv) || !aligned16(out) || !aligned16(workspace))
        return -1;
    // The kernel of many rows takes queries that are turned, and keys that lie in the cache: two launches or three, by the plan of the attention whose bits a step
    // has (us, against few rows in one launch: 128 sequences of 128 query heads and a kv head, 512 slots 20.9 / 21.4, 4096 68 / 79; 96 of 48, 6000 58 / 55).
    if (const long long queries = workspace ? kv4_query_bytes(B, 1, H, KV, D, S) : 0; queries > 0) {
        terna_bf16* q = static_cast<terna_bf16*>(workspace);
        if (ternaspmm_kv4_store(qkv, row, pos, per_sequence, frequency, pairs, amplitude, q, cache, B, 1, H, KV, D, S, adjacent, stream) != 0) return -1;
        return ternaspmm_kv4_attention(q, cache, pos, per_sequence, out, static_cast<uint8_t*>(workspace) + queries, B, 1, H, KV, D, S, scale, stream);
    }
    Kv4Attention a{};
    a.q = qkv, a.k = cache->k, a.k_scale = cache->k_scale, a.v = cache->v, a.v_scale = cache->v_scale, a.pos = pos, a.out = out, a.partial = static_cast<float*>(workspace);
    a.frequency = frequency, a.amplitude = amplitude, a.row = row, a.pairs = pairs;
    a.B = B, a.T = 1, a.H = H, a.KV = KV, a.S = S, a.per_seq = per_sequence != 0;
    a.scale = scale * static_cast<float>(M_LOG2E);
    launch_kv4_attention<true>("ternaspmm_kv4_step", a, D, adjacent, static_cast<hipStream_t>(stream));
    return 0;
}

}  // extern "C"
