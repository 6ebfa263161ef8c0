// Host test of the tile walk and the patch halves of the 8-bit linears' large kernel (crane_b200/csrc/fp8_tiles.h).
//   1. the items of all pairs cover every tile of 256 x 256 once, strips included
//   2. a piece is never put into the half of the patch that the store ahead of it may still be reading (all but the last store have read theirs)
// usage: test_fp8_tiles
#include "../../crane_b200/csrc/fp8_tiles.h"

#include <algorithm>
#include <cstdio>
#include <vector>

using namespace cb;
struct Args { int tiles_m, tiles_n, whole, cut; };

static int check(int M, int N, int esize, int pairs) {
    const F8Turns t = f8_turns(M, N, pairs);
    const Args a = {(M + 255) / 256, (N + 255) / 256, t.whole, t.cut};
    std::vector<int> seen((size_t)a.tiles_m * a.tiles_n, 0);
    for (int i = 0; i < t.items; ++i) {
        const F8Item it = f8_item(a, i);
        if (it.mt < 0 || it.mt >= a.tiles_m || it.n0 < 0 || it.n0 / 256 >= a.tiles_n || it.n0 % it.width) return 1;
        seen[(size_t)it.mt * a.tiles_n + it.n0 / 256] += it.width;
    }
    for (int w : seen) if (w != 256) return 2;
    for (int pair = 0; pair < std::min(t.items, pairs); ++pair)
        for (int warp = 0; warp < 16; ++warp) {                     // two CTAs' eight: 32 rows, half of the columns each
            uint32_t phases = 0;
            int last = -1;
            for (int i = pair; i < t.items; i += pairs) {
                const F8Item it = f8_item(a, i);
                const int C = it.width / 2, m0 = it.mt * 256 + (warp >> 3) * 128 + (warp & 3) * 32, n0 = it.n0 + ((warp >> 2) & 1) * C, end = std::min(N, n0 + C);
                phases ^= 3;                                        // (what the accumulators' turns do to the word's other bits)
                if (C * esize < 128) { last = -1; continue; }       // leaves through registers, behind a wait for all stores
                for (int c = 0; c < C && n0 + c < end && m0 < M; c += 128 / esize) {
                    const int half = f8_half(phases);
                    if (half == last) return 3;
                    last = half;
                    f8_half_stored(phases);
                }
            }
        }
    return 0;
}

int main() {
    const int sizes[][2] = {{8192, 4160}, {8192, 576}, {4096, 4160}, {8192, 24608}, {8192, 4128}, {4459, 11616}, {2304, 17056}, {4900, 4200}, {1111, 12288}, {65, 64}, {8192, 24576}};
    for (const auto& s : sizes)
        for (int pairs : {1, 2, 7, 74})
            for (int esize : {2, 4})
                if (const int e = check(s[0], s[1], esize, pairs)) { printf("%d x %d, %d bytes, %d pairs: fault %d\n", s[0], s[1], esize, pairs, e); return 1; }
    for (int M = 65; M < 3000; M += 211)
        for (int N = 8; N < 6000; N += 136)
            for (int esize : {2, 4})
                if (const int e = check(M, N, esize, 74)) { printf("%d x %d, %d bytes: fault %d\n", M, N, esize, e); return 1; }
    printf("fp8_tiles: ok\n");
    return 0;
}
