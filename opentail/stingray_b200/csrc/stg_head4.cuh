// A head's weight in 4 bits (stg_head_logits.cu, stg_head_tiles.cu): how it is laid out, and a call's arguments.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "stg_handle.h"
#include "stg_head_plan.h"

namespace stg {

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

// (x & mask) ^ base, in one instruction.
__device__ __forceinline__ uint32_t bits_of(uint32_t x, uint32_t mask, uint32_t base)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(r) : "r"(x), "r"(mask), "r"(base));
    return r;
}

// Eight neighbouring hidden states.  (Not as read-only data: the kernel ahead may still have been writing them when this one began.)
__device__ __forceinline__ uint4 eight_states(const uint16_t *from, bool vec)
{
    if (vec) return *(const uint4 *)from;
    uint32_t e[8];
#pragma unroll
    for (int j = 0; j < 8; j++) e[j] = from[j];
    return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
}

// More rows than the stream takes (stg_head_tiles.cu).
size_t head_tiles_workspace(StgHandle h, const Head4 &w, int rows);
int head_tiles(StgHandle h, const HeadLogits &p, bool scale_bf16, void *workspace, cudaStream_t stream);

}  // namespace stg
