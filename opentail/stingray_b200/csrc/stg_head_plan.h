// The head (stg_head_*.cu): sizes, and how calls are cut up.  Host arithmetic without CUDA, tested for itself.
#pragma once
#include <stddef.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>

#ifdef __CUDACC__
#define STG_HD __host__ __device__
#else
#define STG_HD
#endif

namespace stg {

// ---- losses and gradients (stg_head_loss.cu, stg_head_gemm.cuh) ----

constexpr int kHeadTileM = 128;
constexpr int kMostSplits = 64;

enum HeadMode { kStats = 0, kGrad = 1, kHidden = 2, kWeight = 3 };

struct HeadPlan {
    bool pair;              // tiles of 256 rows by two CTAs
    int tile_m, rows_pad;
    int tile_n, tiles_n;    // of the vocabulary
    int piece, pieces;      // backward: vocabulary entries whose gradients are there at a time; a multiple of 64
    int grads_stride, sums_rows;
    size_t bytes;           // of workspace
};

// Rows that the backward pass keeps the remainders of, as rows of their own (k_head_prep): as many fit beside them into one row of tiles (100 rows in
// one of 256: 1607 us in place of 1154, 4096 x 256,000).
constexpr int kLowRows = 64;

// Terms of a sum that the backward pass's products keep in one accumulator (stg_head_gemm.cuh); bf16, whose rounding is eight times as coarse, eight times as
// many.
constexpr int kGradColumns = 1024, kHiddenColumns = 16384, kWeightRows = 16384;
STG_HD constexpr int part_of(int terms, bool bf16) { return bf16 ? 8 * terms : terms; }

inline HeadPlan head_shape(int rows, int vocab, int width, int sms, bool backward)
{
    HeadPlan p;
    memset(&p, 0, sizeof(p));
    if (backward && rows <= kLowRows) rows *= 2;
    p.pair = rows > kHeadTileM;
    p.tile_m = p.pair ? 2 * kHeadTileM : kHeadTileM;
    p.rows_pad = (rows + kHeadTileM - 1) / kHeadTileM * kHeadTileM;
    // One row of tiles reads the weight once, and its time is that of the CTAs with the most of it: the width of a
    // tile is the one whose waves take the fewest vocabulary entries, the widest of those (64 x 4096 x 151,936: 5 waves of 208, 1040
    // entries per CTA, in place of 5 of 256)
    p.tile_n = 256;
    const int step = p.pair ? 32 : 16, workers = p.pair ? std::max(1, sms / 2) : sms;
    if (rows <= p.tile_m)
        for (int64_t n = 256, least = INT64_MAX; n >= 64; n -= step) {
            const int64_t tiles = (vocab + n - 1) / n, most = (tiles + workers - 1) / workers * n;
            if (most < least) { least = most; p.tile_n = (int)n; }
        }
    p.tiles_n = (vocab + p.tile_n - 1) / p.tile_n;
    // a piece of the gradients takes 256 MB at most, or 2048 columns
    const int64_t whole = ((int64_t)vocab + 63) / 64 * 64;
    const int64_t most = std::min<int64_t>(std::max<int64_t>(2048, (int64_t)(1 << 27) / std::max(1, p.rows_pad)), whole);
    p.pieces = (int)((whole + most - 1) / most);
    const int64_t each = ((whole + p.pieces - 1) / p.pieces + 255) / 256 * 256;  // whole tiles
    p.piece = (int)std::min(each, whole);
    p.pieces = (int)((whole + p.piece - 1) / p.piece);
    p.grads_stride = (p.piece + p.tile_n - 1) / p.tile_n * p.tile_n;
    // room for splits: eight tiles per SM (155 MB), which leaves k_head_prep the choice of waves that are nearly full
    p.sums_rows = (int)std::max<int64_t>(p.rows_pad, std::min<int64_t>((int64_t)kMostSplits * p.rows_pad, (int64_t)8 * sms * kHeadTileM * 256 / width));
    return p;
}

// The ring of a product's operands in shared memory: 64 columns of both to a stage, the second operand's boxes ahead of the first's.  Stages
// are as large as their boxes and as many as fit: what is in flight is what hides memory's latency where rows are few (5 x 4096 x
// 256,000: 345 us, 366 with four stages).
constexpr int kGemmK = 64;                                  // columns of a stage: 128 bytes, the swizzle's width
constexpr int kGemmStages = 8;                              // at most
constexpr int kGemmRingBytes = 196608;
constexpr int kGemmABytes = kHeadTileM * kGemmK * 2;        // that the tensor cores read, also where boxes have fewer rows
constexpr int kGemmEpiWarps = 8;
constexpr int kGemmOut = 4096;                              // bytes that each of the eight warps writes its results from: 32 rows of 128 bytes

struct GemmRing {
    int a_at, stage_bytes, stages;
};
inline GemmRing gemm_ring(int mode, bool pair, int tile_n, int a_rows)
{
    // operands whose rows run along M or N come in boxes of 64 by 64
    const int b_cols = tile_n / (pair ? 2 : 1), b_bytes = mode < kHidden ? b_cols * 128 : (b_cols + 63) / 64 * 8192, a_bytes = mode == kWeight ? kGemmABytes : a_rows * 128;
    GemmRing r;
    r.a_at = (b_bytes + 1023) / 1024 * 1024;
    r.stage_bytes = r.a_at + (a_bytes + 1023) / 1024 * 1024;
    // the last stage's first operand is read as 128 rows, whatever its boxes have
    r.stages = std::min(kGemmStages, (kGemmRingBytes - (kGemmABytes - (r.stage_bytes - r.a_at))) / r.stage_bytes);
    return r;
}

// ---- weights in 4 bits (stg_head_logits.cu, stg_head_tiles.cu) ----

// The packed weight: units of 16 vocabulary entries by 128 columns, a tile's units (16 entries, all columns, zeros behind the last)
// next to each other.  A unit: twice 512 bytes of codes, of which a lane of a warp holds 16 - what it needs of 64 columns in four
// steps of mma.m16n8k16 (word s: step s); the columns of a step are chosen such that a lane's share of a hidden state are eight
// neighbours for two steps: step s, columns 32 (s / 2) + 8 t + 4 (s % 2) + 0..3 for t = lane % 4.  Then the scales, and in the same way
// the zero points: for entry g = 0..7 the unit's groups, for each of them entries g and g + 8.  A word's nibbles 0, 2, 4, 6 are four columns of entry
// g, and nibbles 1, 3, 5, 7 those of entry g + 8 (in the order of columns 0, 2, 1, 3), as q - 8 in two's complement.  Lane (g, t)'s 16 bytes
// lie at 64 g + 16 (t ^ g / 2): eight lanes that read those of eight entries g for one t meet in no bank.
constexpr uint32_t kCodeSigns = 0x88888888u;
constexpr int kHeadRows4 = 16, kUnitCols = 128, kUnitCodes = 1024;

STG_HD constexpr int code_place(int lane) { return (lane & ~3) | ((lane & 3) ^ (lane >> 3)); }  // of a lane's 16 bytes among the 32

struct Head4 {
    const unsigned char *units;
    int vocab, width, group, tiles, units_per_tile, unit_bytes, groups_per_unit;
};

inline Head4 head4_shape(int vocab, int width, int group, bool zeros)
{
    Head4 w;
    memset(&w, 0, sizeof(w));
    w.vocab = vocab; w.width = width; w.group = group;
    w.groups_per_unit = kUnitCols / group;
    w.unit_bytes = kUnitCodes + 32 * w.groups_per_unit * (zeros ? 2 : 1);
    w.units_per_tile = (width + kUnitCols - 1) / kUnitCols;
    w.tiles = (vocab + kHeadRows4 - 1) / kHeadRows4;
    return w;
}
inline size_t head4_bytes(const Head4 &w) { return (size_t)w.tiles * w.units_per_tile * w.unit_bytes; }

// The kernel that the weight streams through: hidden states whole in shared memory, and a ring for each warp.
constexpr int kStreamWarps = 16, kStreamStages = 2;
constexpr int kIntRows = 2;      // as integers of four digits
constexpr int kStreamRows = 32;

struct StreamShape {
    int pitch;          // bytes between rows of hidden states
    int chunk;          // units of a stage; 0: it does not fit
    size_t sums, unscale, slots, ring, bars, smem;  // offsets, and bytes in all
};

inline StreamShape stream_shape(const Head4 &w, int rows, bool zeros, size_t most)
{
    const int nt = rows <= 8 ? 1 : 2;
    const bool ints = rows <= kIntRows;
    StreamShape s;
    memset(&s, 0, sizeof(s));
    const size_t cols = (size_t)w.units_per_tile * kUnitCols;
    s.pitch = (int)(ints ? cols + 16 : cols * 2 + 64);  // rows g and g + 1 of a fragment in different banks
    s.sums = (size_t)8 * nt * s.pitch;
    s.unscale = s.sums + (zeros ? cols / w.group * 8 * nt * 4 : 0);
    s.slots = (s.unscale + (size_t)8 * nt * 8 + 15) / 16 * 16;
    s.bars = s.slots + (size_t)kStreamWarps * nt * 512;
    s.ring = (s.bars + kStreamWarps * kStreamStages * 8 + 127) / 128 * 128;
    const size_t unit = (size_t)kStreamWarps * kStreamStages * w.unit_bytes;
    s.chunk = s.ring + unit <= most ? (int)std::min<size_t>(4, (most - s.ring) / unit) : 0;
    s.smem = s.ring + s.chunk * unit;
    return s;
}

// Up to 32 rows stream, where 16 of them fit into shared memory beside the rings; more than 16 in two calls of half of them, each of which reads
// the weight (17 x 4096 x 151,936: 2 x 80 us, stg_head_tiles.cu 207 with groups of 128, 333 with groups of 32).
inline bool streams(const Head4 &w, int rows, bool zeros, size_t smem)
{
    return rows <= kStreamRows && stream_shape(w, std::min(rows, 16), zeros, smem).chunk > 0;
}

// The kernel for more rows.
constexpr int kTilesMost = 8;        // tiles of an item
constexpr int kTilesChunk = 4;       // units of a stage: copies of one unit each kept the copying warp busy for 1400 cycles a unit
constexpr int kTilesStages = 6;      // of either ring at most
constexpr int kTilesSlots = 8;       // accumulators at most
STG_HD constexpr int tiles_buffers(int n) { return n <= 64 ? 4 : 2; }  // of unpacked weights, 64 columns of tensor memory each, behind the accumulators
STG_HD constexpr size_t tiles_code_stage(int unit_bytes, int groups_per_unit, int n)
{
    return ((size_t)kTilesChunk * (kTilesMost * unit_bytes + groups_per_unit * n * 4) + 1023) / 1024 * 1024;
}

struct TilesShape {
    int n, blocks;          // rows of a block (16, 32, 64 or 128) and their number
    int per_item, items_v;  // tiles of an item, and items of the vocabulary
    int code_stages, state_stages, slots;
    size_t smem;
};

inline TilesShape tiles_shape(const Head4 &w, int rows, int sms, size_t room)
{
    TilesShape a;
    memset(&a, 0, sizeof(a));
    a.blocks = (rows + 127) / 128;
    const int each = (rows + a.blocks - 1) / a.blocks;
    a.n = each <= 16 ? 16 : each <= 32 ? 32 : each <= 64 ? 64 : 128;
    // Few rows: the time is that of the CTA with the most of the weight, and smaller items share it out more evenly.  Many: an item takes
    // its time however few tiles it has.
    a.per_item = kTilesMost;
    if (a.n <= 32)
        for (int64_t n = kTilesMost, least = INT64_MAX; n >= 5; n--) {
            const int64_t items = (w.tiles + n - 1) / n, most = (items + sms - 1) / sms * n;
            if (most < least) { least = most; a.per_item = (int)n; }
        }
    a.items_v = (w.tiles + a.per_item - 1) / a.per_item;
    a.slots = std::min(kTilesSlots, (512 - 64 * tiles_buffers(a.n)) / a.n);
    const size_t code = tiles_code_stage(w.unit_bytes, w.groups_per_unit, a.n), state = (size_t)2 * a.n * 128;
    a.code_stages = a.n <= 64 ? 3 : 2;
    a.state_stages = (int)std::min<size_t>(kTilesStages, (room - 1024 - a.code_stages * code) / state);
    a.smem = 1024 + a.code_stages * code + a.state_stages * state;
    return a;
}

}  // namespace stg
