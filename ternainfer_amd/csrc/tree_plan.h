// How the attention of a tree of drafted tokens over the cache is laid out.  Host code without HIP: tests/draft_plan_check.cpp runs it on the CPU.
#pragma once

#include <algorithm>
#include <cmath>

namespace terna {

constexpr int kTreeTile = 32;                  // slots of a wave's step
constexpr int kTreeMaxSplits = 64;             // parts of a row: one a lane of the launch that joins them

struct TreePlan {
    int rows;                                  // query rows of a workgroup: 32, 64 or 128
    int tiles;                                 // workgroups along the rows of a kv head
    int splits;                                // parts that the slots are read in, of a sequence of the cache's length
};
// The parts by the time they take, us, fitted to 250 measured shapes and numbers of parts (an error of 12 %; the parts chosen by it took 1 % longer than the
// best ones, 11 % at the worst): a step of a workgroup's four waves -- 4, 2 or 1 tiles -- 0.97, 1.03 or 0.75, 1.08 with a second workgroup of
// 128 rows beside it; 8 around a workgroup's steps, 4 for the launch that joins the parts, their numerators written and read at 5.9 TB/s, and the cache
// itself at 5.8, less where workgroups are fewer than the CUs or do not fill their last round.
inline TreePlan tree_plan(int B, int T, int H, int KV, int D, int S)
{
    const long long rows = static_cast<long long>(T) * (H / KV), heads = static_cast<long long>(B) * KV, tiles = (S + kTreeTile - 1) / kTreeTile;
    TreePlan p;
    p.rows = rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    p.tiles = static_cast<int>((rows + p.rows - 1) / p.rows);
    const int together = 128 / p.rows;         // tiles of a workgroup's step
    const float cache = static_cast<float>(heads) * static_cast<float>(S) * static_cast<float>(4 * D) * 0.172e-6f;
    auto time = [&](long long n) {
        const float wgs = static_cast<float>(heads * p.tiles) * static_cast<float>(n), steps = static_cast<float>((tiles + together * n - 1) / (together * n));
        const float places = wgs <= 256.0f || (p.rows == 32 && D == 128) ? 256.0f : 512.0f;        // (32 rows of 128 dimensions: one to a CU)
        const float step = (p.rows == 32 ? 0.97f : p.rows == 64 ? 1.03f : places == 256.0f ? 0.75f : 1.08f) * (D == 64 ? 0.67f : 1.0f);
        const float full = std::max(1.0f, wgs / places), whole = std::ceil(full), rounds = full > 3.0f ? full : 0.5f * (full + whole);
        const float memory = cache * std::pow(std::max(1.0f, 0.9f * places * whole / wgs), 0.6f);
        return std::max(rounds * (8.0f + steps * step), memory + 8.0f) +
               (n == 1 ? 0.0f : 4.0f + static_cast<float>(rows * heads) * static_cast<float>(8 * D * n) * 0.171e-6f);
    };
    p.splits = 1;
    float best = time(1);
    const long long most = std::min<long long>({kTreeMaxSplits, (tiles + 1) / 2, std::max(1ll, 4096 / (heads * p.tiles))});
    for (long long n = 2; n <= most; ++n)
        if (const float t = time(n); t < best) best = t, p.splits = static_cast<int>(n);
    return p;
}

}  // namespace terna
