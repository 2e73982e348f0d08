// How the attention of a tree of drafted tokens over the cache is laid out.  Host code without HIP: tests/tree_plan_check.cpp runs it on the CPU.
#pragma once

#include <algorithm>

namespace terna {

constexpr int kTreeTile = 32;                  // slots of a wave's step
constexpr int kTreeMaxSplits = 64;             // parts of a row: one a lane of the launch that joins them

struct TreePlan {
    int row_waves;                             // waves of a workgroup that share its slots, 32 query rows each; the other 4 / row_waves take other slots
    int tiles;                                 // workgroups along the rows of a kv head
    int splits;                                // parts that the slots are read in
};
inline TreePlan tree_plan(int B, int T, int H, int KV, int D, int S)
{
    const long long rows = static_cast<long long>(T) * (H / KV), heads = static_cast<long long>(B) * KV, steps = (S + kTreeTile - 1) / kTreeTile;
    TreePlan p;
    p.row_waves = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
    p.tiles = static_cast<int>((rows + 32 * p.row_waves - 1) / (32 * p.row_waves));
    const int together = 4 / p.row_waves;      // tiles of a workgroup's step
    const long long groups = heads * p.tiles;
    auto time = [&](long long n) {
        const long long wgs = groups * n, mine = (steps + together * n - 1) / (together * n);
        const float places = p.row_waves == 1 ? 256.0f : 512.0f;
        const float each = p.row_waves == 1 ? 1.0f : 0.8f * (wgs > 256 ? 2.0f : 1.0f);
        return std::max(1.0f, static_cast<float>((wgs + places - 1) / places)) * (4.0f + each * static_cast<float>(mine)) +
               (n == 1 ? 0.0f : 2.0f + static_cast<float>(rows * heads) * static_cast<float>(8 * D * n) * (1.0f / 3e6f));
    };
    p.splits = 1;
    float best = time(1);
    const long long most = std::min<long long>(kTreeMaxSplits, (steps + together - 1) / together);
    for (long long n = 2; n <= most; ++n)
        if (const float t = time(n); t < best) best = t, p.splits = static_cast<int>(n);
    return p;
}

}  // namespace terna
