// How the attention of a tree of drafted tokens over the cache is laid out.  Host code without HIP: tests/draft_plan_check.cpp runs it on the CPU.
#pragma once

#include <algorithm>
#include <cmath>

namespace terna {

constexpr int kTreeTile = 32;                  // slots of a wave's step
constexpr int kTreeMaxSplits = 64;             // parts of a row: one a lane of the launch that joins them

struct TreePlan {
    int rows;                                  // query rows of a workgroup: 32, 64 or 128
    int groups;                                // of its waves, that take turns of the tiles: 4, 2, and for 128 rows 1 or 2
    int tiles;                                 // workgroups along the rows of a kv head
    int splits;                                // parts that the slots are read in, of a sequence of the cache's length
};
// The groups and the parts by the time they take, us: steps of a workgroup and what surrounds them, in rounds of the workgroups that there is room for, or the
// cache's bytes -- at 5.8 TB/s, less where workgroups are fewer than the CUs or do not fill their last round --, and the launch that joins the parts, whose
// numerators are written and read at 5.4 to 5.9.  Fitted to 250 measured shapes and numbers of parts of up to 64 rows (an error of 12 %) and 555 of more (11 %; the
// plan chosen by it took 1.3 % longer than the best one in the mean of 30 shapes, 10 % at the worst; one group alone 3.8 % in the mean, two 4.4).  128 rows in two groups are a
// workgroup of eight waves, one to a CU, with half the numerators that two workgroups of four have: 240 rows over 32768 slots 47 us, with one group 50; where workgroups are many,
// those of one group start and end while others compute: 33 sequences of 720 rows over 399 slots 103 us, with two groups 128.
inline TreePlan tree_plan(int B, int T, int H, int KV, int D, int S)
{
    const long long rows = static_cast<long long>(T) * (H / KV), heads = static_cast<long long>(B) * KV, tiles = (S + kTreeTile - 1) / kTreeTile;
    TreePlan p;
    p.rows = rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    p.tiles = static_cast<int>((rows + p.rows - 1) / p.rows);
    const float cache = static_cast<float>(heads) * static_cast<float>(S) * static_cast<float>(4 * D) * 0.172e-6f;
    auto time = [&](int groups, long long n) {
        const float wgs = static_cast<float>(heads * p.tiles) * static_cast<float>(n), steps = static_cast<float>((tiles + groups * n - 1) / (groups * n));
        // (32 rows of 128 dimensions and eight waves: one to a CU)
        const float places = wgs <= 256.0f || (p.rows == 32 && D == 128) || (p.rows == 128 && groups == 2) ? 256.0f : 512.0f;
        float step, around = 8.0f;
        if (p.rows == 32) step = 0.97f;
        else if (p.rows == 64) step = 1.03f;
        else if (groups == 2) step = 1.09f, around = 7.5f;
        else if (places == 256.0f) step = 0.72f, around = 7.7f;
        else step = 1.31f, around = 3.3f;
        if (D == 64) step *= p.rows == 128 ? 0.66f : 0.67f;
        const float full = std::max(1.0f, wgs / places), whole = std::ceil(full), rounds = full > 3.0f ? full : p.rows == 128 ? whole : 0.5f * (full + whole);
        const float memory = cache * std::pow(std::max(1.0f, 0.9f * places * whole / wgs), 0.6f);
        return std::max(rounds * (around + steps * step), memory + 8.0f) +
               (n == 1 ? 0.0f : (p.rows == 128 ? 6.6f : 4.0f) + static_cast<float>(rows * heads) * static_cast<float>(8 * D * n) * (p.rows == 128 ? 0.193e-6f : 0.171e-6f));
    };
    const int least = 128 / p.rows, widest = std::max(least, 2);
    p.groups = least, p.splits = 1;
    float best = time(least, 1);
    const long long most = std::min<long long>({kTreeMaxSplits, (tiles + 1) / 2, std::max(1ll, 4096 / (heads * p.tiles))});
    for (int groups = least; groups <= widest; ++groups)
        for (long long n = 1; n <= most; ++n)
            if (const float t = time(groups, n); t < best) best = t, p.groups = groups, p.splits = static_cast<int>(n);
    return p;
}

// Where a workgroup works: on which part of a kv head (unit; -1: nowhere), on which of its row tiles.  Workgroups go to the XCDs round robin: the tiles of a unit, which
// read the same slots, are on one XCD, eight units on eight, and those of the last units, fewer than eight, on all in equal shares (20 units of 12 tiles: 36 on four of
// the XCDs and 24 on the others 58 us, 30 on each 39, both with probabilities in one bf16; in two 45).
struct TreePlace {
    int unit, tile;
};
constexpr TreePlace tree_place(int block, int units, int tiles)
{
    const int xcd = block & 7, at = block >> 3, whole = (units >> 3) * tiles, others = (units & 7) * tiles, each = (others + 7) >> 3;
    const int index = at < whole ? at : xcd * each + at - whole;           // of a tile among those of its kind
    if (at >= whole && (at - whole >= each || index >= others)) return TreePlace{-1, 0};
    const int of = index / tiles;
    return TreePlace{at < whole ? 8 * of + xcd : (units & ~7) + of, index - of * tiles};
}
constexpr long long tree_blocks(long long units, int tiles) { return 8 * (units / 8 * tiles + (units % 8 * tiles + 7) / 8); }

}  // namespace terna
