// How f8_pair_kernel (fp8_gemm.cu) walks its tiles, and which half of a warp's patch the next piece of results goes through: plain arithmetic, the same on either side
// (a C++ compiler alone takes it too).
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define F8_BOTH __host__ __device__ __forceinline__
#else
#define F8_BOTH inline
#endif

namespace cb {

constexpr int F8_BAND = 8;                         // rows of tiles that are walked together: neighbours in time share weights and activations in L2

// Tiles of 256 x 256; tiles 0 .. whole - 1 as they are, then strips of 256 / cut columns: `items` together
struct F8Turns { int whole, items, cut; };
inline F8Turns f8_turns(int M, int N, int pairs) {       // tiles of a pair, those of the last turn cut into strips where pairs are free for them
    const int tiles = ((M + 255) / 256) * ((N + 255) / 256), left = tiles % pairs;
    F8Turns t;
    t.cut = left == 0 || 2 * left > pairs ? 1 : 4 * left > pairs ? 2 : 4;
    t.whole = tiles - (t.cut > 1 ? left : 0);
    t.items = t.whole + (tiles - t.whole) * t.cut;
    return t;
}

struct F8Item { int mt, n0, width; };
template <typename A>                              // A: tiles_m, tiles_n, whole, cut
F8_BOTH F8Item f8_item(const A& a, int i) {
    int t = i, sub = 0, width = 256;
    if (i >= a.whole) {
        const int j = i - a.whole;
        t = a.whole + j / a.cut; sub = j % a.cut; width = 256 / a.cut;
    }
    const int per = F8_BAND * a.tiles_n, b = t / per, r = t - b * per, left = a.tiles_m - b * F8_BAND, w = left < F8_BAND ? left : F8_BAND, nt = r / w;
    return F8Item{b * F8_BAND + r - nt * w, nt * 256 + sub * width, width};
}

// A warp's pieces of 128 bytes a row leave by TMA from two halves of its patch in turn, and a half is written again when all stores but the last one have read theirs.
// So the turns go on from tile to tile: a ragged tile has an odd number of pieces, and with turns of its own the next one would start in the half that is still being read.
// The turn is the word's highest bit (a register of its own for it is one that the sums' kernel does not have).
F8_BOTH int f8_half(uint32_t phases) { return (int)(phases >> 31); }
F8_BOTH void f8_half_stored(uint32_t& phases) { phases ^= 1u << 31; }

}  // namespace cb
