// How stg_beam_select cuts rows into pieces, a CTA each.  Host arithmetic only.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace stg {

// CTAs of the selection that an SM holds, for all of its kernels: they are compiled for it.  bf16 behind a soft cap, whose tile is
// 32-bit numbers, spills at the 64 registers that leaves, and gains all the same (36 to 512 rows of 50,257 to 256,000 at a cap of 30:
// 10 to 28 % less time than with one CTA of 122 registers; 256 rows of 262,144 behind masks of 20 %: 2 % more).
constexpr int kBeamCtas = 2;

// Pieces that all rows of a call together may be cut into beyond one each.
constexpr int kBeamExtraPieces = 8192;

// Of the cuts into whole tiles the one with the least time: waves of CTAs times
// tiles of each and about two tiles' worth for the rest of a CTA.  (256 rows of 151,936 fp32: one piece 33.6 us, two
// 34.7, ten 49.0; 64 rows of 262,144 bf16 behind masks: four pieces 20.3, three 24.4, eight 22.0; 4 rows of 151,936: nineteen
// pieces 10.3, ten 10.8.)
inline void beam_pieces(int rows, int vocab, int tile, int sms, int &pieces, int &len)
{
    const int tiles = (vocab + tile - 1) / tile, at_once = kBeamCtas * sms;
    const int most = std::max(1, std::min(tiles, kBeamExtraPieces / rows + 1));
    int64_t least = INT64_MAX;
    int each = tiles;
    for (int c = 1; c <= most; c++) {
        const int per = (tiles + c - 1) / c, got = (tiles + per - 1) / per;
        const int64_t cost = (((int64_t)rows * got + at_once - 1) / at_once) * (per + 2);
        if (cost < least) { least = cost; each = per; }
    }
    pieces = (tiles + each - 1) / each;
    len = each * tile;
}

}  // namespace stg
