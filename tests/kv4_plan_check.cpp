// The plan of the attention over the 4-bit cache: the workgroups of the kernel that it names cover every query row, and its parts fit the launch that joins them.
#include <cstdio>

#include "../ternainfer_amd/csrc/kv4_plan.h"

using namespace terna;

int main()
{
    int shapes = 0, steps_of_many = 0, wrong = 0;
    for (int B : {1, 2, 3, 8, 32, 48, 96, 128, 256, 4096})
        for (int T : {1, 2, 5, 33, 129, 2048})
            for (int KV : {1, 2, 5, 8})
                for (int G : {1, 4, 16, 17, 32, 33, 48, 64, 71, 128, 300, 512})
                    for (int D : {64, 128})
                        for (int S : {1, 31, 32, 129, 1528, 6000, 32768, 1 << 25}) {
                            const Kv4Plan p = kv4_plan(B, T, G * KV, KV, D, S);
                            const long long rows = static_cast<long long>(T) * G;
                            const long long covered = static_cast<long long>(kv4_tiles(rows, p.many)) * (p.many ? kKv4Rows : kKv4FewRows);
                            ++shapes;
                            steps_of_many += T == 1 && p.many;
                            if (covered < rows || covered - rows >= kKv4Rows || p.splits < 1 || p.splits > kKv4MaxSplits || (p.waves != 4 && p.waves != 8) || (p.many && rows <= 32)) {
                                std::printf("B %d T %d KV %d G %d D %d S %d: many %d splits %d waves %d\n", B, T, KV, G, D, S, p.many, p.splits, p.waves);
                                ++wrong;
                            }
                        }
    // the shapes of the steps of many query heads in the GPU tests reach the kernel of many rows
    const int reached[][5] = {{128, 128, 1, 128, 40}, {256, 64, 1, 128, 128}, {96, 48, 1, 128, 6000}, {48, 96, 2, 128, 5600}, {8, 71, 1, 64, 32768}, {1, 568, 8, 64, 32768}, {4, 128, 1, 64, 32768}};
    for (const auto& s : reached)
        if (!kv4_plan(s[0], 1, s[1], s[2], s[3], s[4]).many) std::printf("%d x %d / %d heads of %d, %d slots: few\n", s[0], s[1], s[2], s[3], s[4]), ++wrong;
    std::printf("%d shapes, %d steps of many rows, %d wrong\n", shapes, steps_of_many, wrong);
    if (wrong || !steps_of_many) return 1;
    std::printf("kv4 plan ok\n");
    return 0;
}
