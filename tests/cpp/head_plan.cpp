// How the head's calls are cut up, over many sizes: pieces of the vocabulary, rings in shared memory, tensor memory, and where a weight's
// codes lie, read back as the kernels read them.  Prints "head_plan: ok".
#include "stg_head_plan.h"

#include <cstdio>
#include <cstdlib>
#include <vector>

using namespace stg;

static int bad(const char *what, long long a = 0, long long b = 0, long long c = 0)
{
    std::printf("head_plan: %s (%lld, %lld, %lld)\n", what, a, b, c);
    return 1;
}

static int losses()
{
    const int sms = 148;
    for (int rows : {1, 2, 7, 8, 9, 100, 127, 128, 129, 255, 256, 257, 1000, 2047, 8192, 65537, 1 << 20})
        for (int vocab : {1, 2, 63, 64, 65, 255, 257, 1000, 32000, 50257, 151936, 262144, 1 << 26})
            for (int width : {8, 72, 512, 4096, 1 << 16}) for (bool backward : {false, true}) {
                const HeadPlan p = head_shape(rows, vocab, width, sms, backward);
                const int all = backward && rows <= kLowRows ? 2 * rows : rows;  // with the remainders'
                if (p.rows_pad < all || p.rows_pad % kHeadTileM != 0) return bad("padded rows", rows);
                if (p.pair != (all > kHeadTileM) || (all != rows && all > p.tile_m)) return bad("remainders in one row of tiles", rows);
                if (p.tile_n % (p.pair ? 32 : 16) != 0 || p.tile_n < 64 || p.tile_n > 256 || (all > p.tile_m && p.tile_n != 256)) return bad("tile width", rows, vocab, p.tile_n);
                if ((int64_t)p.tiles_n * p.tile_n < vocab || (int64_t)(p.tiles_n - 1) * p.tile_n >= vocab) return bad("tiles", rows, vocab);
                // pieces cover the vocabulary; all but the last end with a block of the sums over it
                if ((int64_t)p.pieces * p.piece < vocab || (int64_t)(p.pieces - 1) * p.piece >= vocab || p.piece % 64 != 0) return bad("pieces", rows, vocab, p.piece);
                if (p.grads_stride < p.piece || p.grads_stride % p.tile_n != 0 || p.grads_stride % 8 != 0) return bad("gradients' rows", rows, vocab, p.grads_stride);
                if ((int64_t)p.rows_pad * p.grads_stride * 2 > (int64_t)300 << 20 && p.piece > 2048 + 256) return bad("gradients' size", rows, vocab, p.piece);
                if (p.sums_rows < p.rows_pad) return bad("sums", rows, vocab, width);
                const int a_rows = std::min(kHeadTileM, (all + 7) / 8 * 8);
                for (int mode : {kStats, kGrad, kHidden, kWeight}) {
                    const int n = mode < kHidden ? p.tile_n : 256, a = mode < kHidden ? a_rows : kHeadTileM;
                    const GemmRing r = gemm_ring(mode, p.pair, n, a);
                    const int own = n / (p.pair ? 2 : 1), b_bytes = mode < kHidden ? own * 128 : (own + 63) / 64 * 8192, a_bytes = mode == kWeight ? 16384 : a * 128;
                    if (r.stages < 2 || r.stages > kGemmStages || r.a_at % 1024 != 0 || r.stage_bytes % 1024 != 0) return bad("ring", mode, n, r.stages);
                    if (r.a_at < b_bytes || r.stage_bytes - r.a_at < a_bytes) return bad("stage", mode, n, a);
                    // the tensor cores read 128 rows of the first operand
                    if ((r.stages - 1) * r.stage_bytes + r.a_at + kGemmABytes > kGemmRingBytes) return bad("the last stage ends behind the ring", mode, n, a);
                }
            }
    if (1024 + kGemmRingBytes + kGemmEpiWarps * kGemmOut + 1024 > 232448) return bad("shared memory");
    return 0;
}

// A code of entry row and column col of a unit, as packing puts it and as both kernels read it.
static int codes()
{
    std::vector<uint32_t> unit(kUnitCodes / 4);
    std::vector<int> code(16 * 128);
    for (int &c : code) c = std::rand() & 15;
    auto at = [&](int row, int col) { return (uint32_t)code[row * 128 + col]; };
    for (int block = 0; block < 2; block++)
        for (int lane = 0; lane < 32; lane++)
            for (int s = 0; s < 4; s++) {
                const int g = lane >> 2, t = lane & 3, col = block * 64 + 32 * (s / 2) + 8 * t + 4 * (s % 2);
                const uint32_t w = at(g, col) | at(g + 8, col) << 4 | at(g, col + 2) << 8 | at(g + 8, col + 2) << 12 | at(g, col + 1) << 16 | at(g + 8, col + 1) << 20 | at(g, col + 3) << 24 |
                                   at(g + 8, col + 3) << 28;
                unit[block * 128 + code_place(lane) * 4 + s] = w ^ kCodeSigns;
            }
    // the fragments of mma.m16n8k16: a pair's two halves are neighbours in the sum
    for (int lane = 0; lane < 32; lane++)
        for (int i = 0; i < 8; i++) {
            const int g = lane >> 2, t = lane & 3, block = i / 4, s = i % 4, col = block * 64 + 32 * (s / 2) + 8 * t + 4 * (s % 2);
            const uint32_t w = unit[block * 128 + code_place(lane) * 4 + s] ^ kCodeSigns;
            const int want[8] = {(int)at(g, col), (int)at(g + 8, col), (int)at(g, col + 2), (int)at(g + 8, col + 2), (int)at(g, col + 1), (int)at(g + 8, col + 1), (int)at(g, col + 3), (int)at(g + 8, col + 3)};
            for (int n = 0; n < 8; n++)
                if ((int)(w >> (4 * n) & 15) != want[n]) return bad("fragment", lane, i, n);
        }
    // an entry per thread: 16 columns of 32 bits for 64 columns, two neighbours to each
    for (int row = 0; row < 16; row++)
        for (int block = 0; block < 2; block++)
            for (int t = 0; t < 4; t++)
                for (int k = 0; k < 4; k++) {
                    const int g = row & 7, shift = row & 8 ? 4 : 0;
                    const uint32_t w = unit[block * 128 + (g * 64 + (t ^ (g >> 1)) * 16) / 4 + k] ^ kCodeSigns;
                    const int to = 16 * (k / 2) + 4 * t + 2 * (k % 2);
                    for (int half = 0; half < 2; half++)
                        for (int pair = 0; pair < 2; pair++)
                            if ((w >> (8 * half) >> shift >> (16 * pair) & 15) != at(row, block * 64 + 2 * (to + half) + pair)) return bad("row", row, block, to);
                }
    return 0;
}

static int logits()
{
    const size_t room = 232448 - 4096;
    for (int group : {32, 64, 128})
        for (bool zeros : {false, true})
            for (int vocab : {1, 15, 16, 17, 129, 50257, 151936, 1 << 26})
                for (int width : {group, 3 * group, 512, 896, 2048, 4096, 8192, 1 << 16}) {
                    if (width % group != 0) continue;
                    const Head4 w = head4_shape(vocab, width, group, zeros);
                    if (w.unit_bytes % 32 != 0 || (int64_t)w.tiles * 16 < vocab || w.units_per_tile * 128 < width) return bad("units", group, vocab, width);
                    for (int rows : {1, 2, 3, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 256, 300, 5000}) {
                        if (streams(w, rows, zeros, room)) {
                            for (int some : {rows, std::min(rows, 16), (rows + (rows + 15) / 16 - 1) / ((rows + 15) / 16)}) {
                                if (some > 16) continue;
                                const StreamShape s = stream_shape(w, some, zeros, room);
                                if (s.chunk < 1 || s.chunk > 4 || s.smem > room) return bad("stream", width, some, s.smem);
                                if (s.pitch % 16 != 0 || s.sums % 16 != 0 || s.unscale % 8 != 0 || s.slots % 16 != 0 || s.bars % 8 != 0 || s.ring % 128 != 0) return bad("alignment", width, some);
                            }
                        } else if (rows <= kStreamRows && width <= 4096) {
                            return bad("does not stream", width, rows, group);
                        }
                        const TilesShape a = tiles_shape(w, rows, 148, room);
                        if (a.n * a.blocks < rows || a.slots < 1 || a.slots * a.n + 64 * tiles_buffers(a.n) > 512) return bad("tensor memory", rows, a.n, a.slots);
                        if (a.state_stages < 2 || a.smem > room || a.per_item > kTilesMost || (int64_t)a.items_v * a.per_item < w.tiles) return bad("tiles", rows, a.state_stages, a.per_item);
                    }
                }
    return 0;
}

int main()
{
    if (losses() || codes() || logits()) return 1;
    std::printf("head_plan: ok\n");
    return 0;
}
