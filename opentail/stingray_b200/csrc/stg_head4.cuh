// A head's weight in 4 bits (stg_head_logits.cu, stg_head_tiles.cu): how it is laid out, and a call's arguments.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "stg_handle.h"

namespace stg {

// The packed weight: units of 16 vocabulary entries by 128 columns, a tile's units (16 entries, all columns, zeros behind the last)
// next to each other.  A unit: twice 512 bytes of codes, of which a lane of a warp holds 16 - what it needs of 64 columns in four
// steps of mma.m16n8k16 (word s: step s); the columns of a step are chosen such that a lane's share of a hidden state are eight
// neighbours for two steps: step s, columns 32 (s / 2) + 8 t + 4 (s % 2) + 0..3 for t = lane % 4.  Then the scales, and in the same way
// the zero points: for entry g = 0..7 the unit's groups, for each of them entries g and g + 8.  A word's nibbles 0, 2, 4, 6 are four columns of entry
// g, and nibbles 1, 3, 5, 7 those of entry g + 8 (in the order of columns 0, 2, 1, 3), as q - 8 in two's complement.  Lane (g, t)'s 16 bytes
// lie at 64 g + 16 (t ^ g / 2): eight lanes that read those of eight entries g for one t meet in no bank.
constexpr uint32_t kCodeSigns = 0x88888888u;
constexpr int kHeadRows4 = 16, kUnitCols = 128, kUnitCodes = 1024;

struct Head4 {
    const unsigned char *units;
    int vocab, width, group, tiles, units_per_tile, unit_bytes, groups_per_unit;
};

static Head4 head4_shape(int vocab, int width, int group, bool zeros)
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
static size_t head4_bytes(const Head4 &w) { return (size_t)w.tiles * w.units_per_tile * w.unit_bytes; }

struct HeadLogits {
    Head4 w;
    const uint16_t *hidden;
    int64_t hidden_stride;
    bool vec;
    int rows;
    void *out;
    int64_t out_stride;
    bool hidden_bf16, out_bf16;
};


template <bool BF16>
__device__ __forceinline__ float half_at(uint16_t x)
{
    return BF16 ? __uint_as_float((uint32_t)x << 16) : __half2float(__ushort_as_half(x));
}

__device__ __forceinline__ int code_place(int lane) { return (lane & ~3) | ((lane & 3) ^ (lane >> 3)); }

// (x & mask) ^ base, in one instruction.
__device__ __forceinline__ uint32_t bits_of(uint32_t x, uint32_t mask, uint32_t base)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(r) : "r"(x), "r"(mask), "r"(base));
    return r;
}

// Eight neighbouring hidden states.
__device__ __forceinline__ uint4 eight_states(const uint16_t *from, bool vec)
{
    if (vec) return __ldg((const uint4 *)from);
    uint32_t e[8];
#pragma unroll
    for (int j = 0; j < 8; j++) e[j] = from[j];
    return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
}

// More rows than the stream takes (stg_head_tiles.cu).
size_t head_tiles_workspace(StgHandle h, const Head4 &w, int rows);
int head_tiles(StgHandle h, const HeadLogits &p, bool scale_bf16, void *workspace, cudaStream_t stream);

}  // namespace stg
