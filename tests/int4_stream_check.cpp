// Walks every wavefront of the single-row form of the 4-bit linear layer as the kernel does and counts the
// groups of codes that it would read outside the weights. Arguments: lines "blocks groups grid" on stdin;
// prints a line for each case with a bad index, and the number of cases.
#include <cstdio>

#include "yvmoe_linear_stream.h"

template <int RB, int D>
static bool check(int blocks, int groups, int most) {
    const int sets = (blocks + RB - 1) / RB, grid = sets < most ? sets : most;
    long long bad = 0, worst = 0;
    for (int wg = 0; wg < grid; ++wg)
        for (int wave = 0; wave < 8; ++wave) {
            yvmoe::CodeStream<RB> s(blocks, groups, wave, wg, grid);
            // D - 1 loads before the loop, then one for each group that the wavefront multiplies
            const int own = wave < groups ? (groups - wave + 7) / 8 : 0;
            for (long long i = 0, n = D - 1 + (long long)s.items * own; i < n; ++i, s.next())
                for (int b = 0; b < RB; ++b) {
                    const long long at = s.at(b), over = at - ((long long)blocks * groups - 1);
                    if (at < 0 || over > 0) ++bad, worst = over > worst ? over : worst;
                }
        }
    if (bad) printf("RB %d D %d blocks %d groups %d grid %d: %lld reads, %lld groups past the end\n", RB, D, blocks,
                    groups, grid, bad, worst);
    return bad == 0;
}

int main() {
    int blocks, groups, most, n = 0, failed = 0;
    while (scanf("%d %d %d", &blocks, &groups, &most) == 3) {
        failed += !check<1, 3>(blocks, groups, most) + !check<2, 3>(blocks, groups, most) +
                  !check<4, 2>(blocks, groups, most);
        n += 3;
    }
    printf("%d cases, %d failed\n", n, failed);
    return failed != 0;
}
