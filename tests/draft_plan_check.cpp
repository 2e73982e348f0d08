// The plans of the tree attention and of the 8-bit product: their workgroups cover every row, their parts fit the launches that join them and hold something.
#include <cstdio>
#include <vector>

#include "../ternainfer_amd/csrc/int8_plan.h"
#include "../ternainfer_amd/csrc/tree_plan.h"

using namespace terna;

int main()
{
    int shapes = 0, split = 0, wrong = 0, groups[5] = {};
    for (int B : {1, 2, 3, 8, 31, 64, 300, 65535})
        for (int T : {1, 2, 7, 16, 33, 64, 65, 512})
            for (int KV : {1, 2, 5, 8})
                for (int G : {1, 4, 5, 8, 17, 64})
                    for (int D : {64, 128})
                        for (int S : {1, 31, 33, 384, 4352, 32768, 1 << 25}) {
                            if (static_cast<long long>(B) * T * G * KV > 1 << 28) continue;
                            const TreePlan p = tree_plan(B, T, G * KV, KV, D, S);
                            const long long rows = static_cast<long long>(T) * G, covered = static_cast<long long>(p.tiles) * p.rows;
                            ++shapes;
                            split += p.splits > 1;
                            ++groups[p.groups < 1 || p.groups > 4 ? 0 : p.groups];
                            if (p.groups * p.rows != 128 && !(p.rows == 128 && p.groups == 2)) std::printf("tree: %d rows in %d groups\n", p.rows, p.groups), ++wrong;
                            if ((p.rows != 32 && p.rows != 64 && p.rows != 128) || covered < rows || covered - rows >= p.rows || p.splits < 1 || p.splits > kTreeMaxSplits ||
                                (p.splits > 1 && (p.splits - 1) * static_cast<long long>(kTreeTile) >= S)) {
                                std::printf("tree: B %d T %d KV %d G %d D %d S %d: rows %d tiles %d splits %d\n", B, T, KV, G, D, S, p.rows, p.tiles, p.splits);
                                ++wrong;
                            }
                        }
    // every row tile of every unit is some workgroup's, and one's alone
    for (int units = 1; units <= 300; units += units < 40 ? 1 : 13)
        for (int tiles : {1, 2, 3, 5, 7, 12, 16, 64}) {
            std::vector<int> taken(units * tiles, 0);
            for (long long block = 0; block < tree_blocks(units, tiles); ++block) {
                const TreePlace p = tree_place(static_cast<int>(block), units, tiles);
                if (p.unit >= 0 && (p.unit >= units || p.tile < 0 || p.tile >= tiles || taken[p.unit * tiles + p.tile]++)) ++wrong;
            }
            for (int x : taken) wrong += x != 1;
        }
    int reached[kInt8TileKinds] = {}, joined = 0;
    for (int M : {1, 2, 16, 17, 32, 33, 60, 64, 65, 128, 200, 333, 512, 1000, 2048, 4096, 8192, 100000})
        for (int N : {1, 16, 100, 254, 1000, 2501, 2560, 3840, 13824, 50021, 128256})
            for (int K : {1, 16, 64, 65, 352, 640, 2560, 6912, 131056})
                for (bool room : {false, true}) {
                    const Int8Plan p = int8_plan(M, N, K, room);
                    const Int8TileTime& t = kInt8Tiles[p.tile];
                    const int steps = int8_k_blocks(K) / 2, share = (steps + p.splits - 1) / p.splits;
                    ++shapes;
                    ++reached[p.tile];
                    joined += p.splits > 1;
                    if (p.tiles * t.rows * t.features < static_cast<long long>(M) * N || p.splits < 1 || p.splits > kInt8MaxSplits || (p.splits > 1 && (!room || p.tile != kInt8SplitTile)) ||
                        share * (p.splits - 1) >= steps + (p.splits == 1)) {
                        std::printf("int8: %d x %d x %d: tile %d splits %d\n", M, N, K, p.tile, p.splits);
                        ++wrong;
                    }
                }
    // few rows and channels of every number of columns: no part is without a stage
    for (int K = 64; K <= 131056; K += 64)
        for (int M : {1, 60}) {
            const Int8Plan p = int8_plan(M, 2560, K, true);
            const int steps = int8_k_blocks(K) / 2, share = (steps + p.splits - 1) / p.splits;
            ++shapes;
            if (share * (p.splits - 1) >= steps) std::printf("int8: %d x 2560 x %d: splits %d\n", M, K, p.splits), ++wrong;
        }
    for (int i = 0; i < kInt8TileKinds; ++i)
        if (!reached[i]) std::printf("int8: no shape takes tile %d\n", i), ++wrong;
    std::printf("%d shapes, %d trees in parts, %d products in parts, %d wrong\n", shapes, split, joined, wrong);
    if (!groups[1] || !groups[2] || !groups[4]) std::printf("tree: no shape has 1, 2 or 4 groups\n"), ++wrong;
    if (wrong || !split || !joined) return 1;
    std::printf("draft plans ok\n");
    return 0;
}
