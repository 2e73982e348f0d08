// How a matrix product in 8-bit integers is laid out.  Host code without HIP: tests/draft_plan_check.cpp runs it on the CPU.
#pragma once

#include <algorithm>

namespace terna {

// 64-column blocks of a packed row
constexpr int int8_k_blocks(int K) { return 2 * ((K + 127) / 128); }

// Tiles that a workgroup computes, features x rows; which of them the kernel is instantiated for is the launch's list (abi_int8.hip), in this order.
// Two workgroups share a CU.  Times in us, fitted to 400 measured products (an error of 12 %; of 60 shapes the choice took 8 % longer than the fastest at
// the worst): of a block of 64 columns of a workgroup alone on its CU and of one beside another, and of what surrounds them.
struct Int8TileTime {
    int features, rows;
    float alone, beside, around;
};
constexpr Int8TileTime kInt8Tiles[] = {
    {128, 32, 0.099f, 0.270f, 3.3f}, {64, 64, 0.088f, 0.195f, 3.2f},   {128, 64, 0.132f, 0.328f, 4.1f},  {256, 64, 0.202f, 0.578f, 5.2f},
    {128, 128, 0.211f, 0.514f, 5.5f}, {128, 192, 0.256f, 0.653f, 7.2f}, {128, 256, 0.330f, 0.839f, 9.7f},
};
constexpr int kInt8TileKinds = sizeof(kInt8Tiles) / sizeof(kInt8Tiles[0]), kInt8SplitTile = 1, kInt8MaxSplits = 4;

struct Int8Plan {
    int tile, splits;                          // splits: parts of the columns, joined by a second launch
    long long tiles;
};
// Few tiles of many columns are split (60 x 2560 x 6912, 40 tiles: 12.8 us, in four parts 10.0); only the smallest tile is, the others are not chosen where
// there are few.  `room`: whether there is a workspace for it.
inline Int8Plan int8_plan(int M, int N, int K, bool room)
{
    const int blocks = int8_k_blocks(K);
    const float bytes = static_cast<float>(N) * K + static_cast<float>(M) * K + 2.0f * static_cast<float>(M) * N;
    Int8Plan best{0, 1, 0};
    float least = 0.0f;
    for (int i = 0; i < kInt8TileKinds; ++i) {
        const Int8TileTime& t = kInt8Tiles[i];
        const long long tiles = static_cast<long long>((M + t.rows - 1) / t.rows) * ((N + t.features - 1) / t.features);
        for (int splits = 1; splits <= (room && i == kInt8SplitTile ? kInt8MaxSplits : 1); ++splits) {
            const int share = (blocks / 2 + splits - 1) / splits, steps = 2 * share;    // (whole stages of 128 columns)
            if (splits > 1 && share * (splits - 1) >= blocks / 2) continue;             // a part without a stage
            const float wgs = static_cast<float>(tiles) * splits;
            if (splits > 1 && (wgs > 512.0f || steps < 4)) break;
            float time;
            if (wgs <= 256.0f) {
                time = t.around + steps * t.alone;
            } else {
                // of a few rounds the last counts half as much as if it were full
                const float all = std::max(1.0f, wgs / 512.0f);
                const float rounds = all > 3.0f ? all : 0.5f * (all + static_cast<float>((tiles * splits + 511) / 512));
                time = rounds * (t.around + steps * t.beside);
            }
            time = std::max(time, bytes * 0.246e-6f) + 0.1f * time;        // (what memory bounds, by the tile that computes it in the least time)
            if (splits > 1) time += 0.7f + 0.35f * splits + wgs * static_cast<float>(t.features * t.rows) * (8.0f / 3.5e6f);
            if (least == 0.0f || time < least) least = time, best = Int8Plan{i, splits, tiles};
        }
    }
    return best;
}

}  // namespace terna
