// The cut of rows into pieces, against the time that it stands for: waves of the CTAs that the kernel in question has resident,
// times what one of them takes.  Prints "beam_pieces: ok".
#include "stg_beam_pieces.h"

#include <cstdio>

int main()
{
    const int sms = 148;
    for (int tile : {8192, 16384})  // fp32 and bf16
        for (int rows : {1, 2, 4, 30, 64, 96, 147, 148, 149, 160, 256, 296, 297, 512, 1000, 66000})
            for (int vocab : {1, 31, 8192, 16385, 50257, 151936, 256000, 262144, 1 << 24}) {
                const int tiles = (vocab + tile - 1) / tile;
                const long long resident = stg::kBeamCtas * sms;  // what the kernels' launch bounds ask for
                int pieces = 0, len = 0;
                stg::beam_pieces(rows, vocab, tile, sms, pieces, len);
                const auto time = [&](long long c) { return ((long long)rows * ((tiles + (tiles + c - 1) / c - 1) / ((tiles + c - 1) / c)) + resident - 1) / resident * ((tiles + c - 1) / c + 2); };
                const bool covers = (long long)pieces * len >= vocab && (long long)(pieces - 1) * len < vocab && len % tile == 0;
                const bool fits = (long long)rows * pieces <= rows + stg::kBeamExtraPieces;
                long long least = time(1);
                for (int c = 2; c <= tiles && c <= stg::kBeamExtraPieces / rows + 1; c++) least = std::min(least, time(c));
                const long long is = ((long long)rows * pieces + resident - 1) / resident * (len / tile + 2);
                if (!covers || !fits || is != least) {
                    std::printf("beam_pieces: tile %d, %d rows of %d: %d pieces of %d take %lld, not %lld\n", tile, rows, vocab, pieces, len, is, least);
                    return 1;
                }
            }
    std::printf("beam_pieces: ok\n");
    return 0;
}
