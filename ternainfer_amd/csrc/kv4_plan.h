// Which kernel takes the attention of a call over the 4-bit cache, and in how many parts.  Host code without HIP: tests/kv4_plan_check.cpp runs it on the CPU.
#pragma once

#include <algorithm>

namespace terna {

constexpr int kKv4Step = 32;                   // slots of a wave's step (few rows)
constexpr int kKv4FewRows = 16;                // query rows of a workgroup of the kernel of few rows (kv4_attention_kernel.h)
constexpr int kKv4Rows = 128;                  // ... of many (kv4_prefill_kernel.h)
constexpr int kKv4MaxSplits = 128;             // parts of a row: two a lane of the launch that joins them

// Workgroups along the rows of a kv head.
inline int kv4_tiles(long long rows, bool many)
{
    const int each = many ? kKv4Rows : kKv4FewRows;
    return static_cast<int>((rows + each - 1) / each);
}

// How the attention of one call is laid out: by 16 rows of a kv head and waves of their own (few rows: memory), or by 128 rows (many: matrix cores), and the
// parts that the slots are read in.  By the times that the two take as a function of the sizes (us, from 110 measured shapes, graphs of 24 launches;
// causal ones included, whose rows see half of what is counted here):
//   few    a workgroup 4.2 + 0.63 a round of its four waves alone on its CU, 4.5 + 1.1 with a second one (64 dimensions: a fourth) beside it; one of eight waves
//          is as two beside each other in half the parts (one token of 32 sequences, 1528 slots: 14.9 in three parts of four waves, 13.3 in one of eight)
//   many   a workgroup 9 + 1.75 a step of its two groups (128 slots), one to a CU
//   parts  2 for the launch that joins them, and their numerators written and read at 3 TB/s
// Measured, few / many: 8 x 16 tokens, 4096 slots 17 / 22; 1 x 32, 32768 31 / 29; 8 x 64, 4096 55 / 41; prompts 1 x 400 14.2 / 14.9, 4 x 200 15.5 / 12.0, 1 x 1024 34.6 / 22.6;
// parts of 1 x 1 token, 1024 slots 9.3 in one, 7.7 in four, 32768 17.2 in 102 of them; 1 x 384 tokens in one 6.1, in three 7.8.
struct Kv4Plan {
    bool many;
    int splits, waves;                         // waves: of few rows
};
inline Kv4Plan kv4_plan(int B, int T, int H, int KV, int D, int S)
{
    const long long rows = static_cast<long long>(T) * (H / KV), heads = static_cast<long long>(B) * KV;
    const float all_rows = static_cast<float>(rows) * static_cast<float>(heads);
    const long long steps = (S + kKv4Step - 1) / kKv4Step, tiles_few = kv4_tiles(rows, false), tiles_many = kv4_tiles(rows, true);
    auto joined = [&](long long n) { return n == 1 ? 0.0f : 2.0f + all_rows * static_cast<float>(8 * D * n) * (1.0f / 3e6f); };
    auto rounds = [&](long long n, int waves) { return static_cast<float>((steps + waves * n - 1) / (waves * n)); };
    auto few = [&](long long n) {
        const float wgs = static_cast<float>(heads * tiles_few * n);
        return std::max(1.0f, wgs / (D == 64 ? 1024.0f : 512.0f)) * (wgs <= 256.0f ? 4.2f + 0.63f * rounds(n, 4) : 4.5f + 1.1f * rounds(n, 4)) + joined(n);
    };
    auto few_of_eight = [&](long long n) { return 4.5f + 1.1f * rounds(n, 8) + joined(n); };
    auto many = [&](long long n) {
        const float wgs = static_cast<float>(heads * tiles_many * n);
        return (wgs <= 256.0f ? 1.0f : wgs / 256.0f + 0.5f) * (9.0f + 1.75f * rounds(n, 4)) + joined(n);
    };
    // the next count of parts that saves a round
    auto next = [&](long long n, int waves) {
        const long long r = (steps + waves * n - 1) / (waves * n);
        return r <= 1 ? kKv4MaxSplits + 1ll : (steps + waves * (r - 1) - 1) / (waves * (r - 1));
    };
    Kv4Plan p{false, 1, 4};
    float best = few(1);
    const long long most = std::min<long long>({kKv4MaxSplits, (steps + 3) / 4, 512 / (heads * tiles_few)}), most_of_eight = std::min(most, 256 / (heads * tiles_few));
    for (long long n = next(1, 4); n <= most; n = next(n, 4))
        if (const float time = few(n); time < best) best = time, p.splits = static_cast<int>(n);
    for (long long n = 1; n <= most_of_eight; n = next(n, 8))
        if (const float time = few_of_eight(n); time < best - 0.25f) best = time, p.splits = static_cast<int>(n), p.waves = 8;
    if (rows <= 32) return p;
    const long long most_many = std::min<long long>({kKv4MaxSplits, steps / 8, 256 / (heads * tiles_many)});
    for (long long n = 1; n <= std::max(1ll, most_many); n = next(n, 4))
        if (const float time = many(n); time < best) best = time, p = Kv4Plan{true, static_cast<int>(n), 4};
    return p;
}

}  // namespace terna
