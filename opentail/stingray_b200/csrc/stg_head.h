// The head (stg_head_*.cu): what its kernels share.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../../include/stingray_sampler.h"
#include "stg_handle.h"
#include "stg_head_plan.h"

namespace stg {

// What the preparation of a call finds out, in device memory.
struct HeadInfo {
    int32_t used;       // rows that have a loss, and those of their remainders
    int32_t low;        // backward: how many rows there are ahead of the remainders', or 0: there are none
    int32_t splits;     // backward: parts of a piece of the vocabulary whose gradients of the hidden states are kept apart
    float scale;        // power of two that the logits' gradients are multiplied with where they are rounded to 16 bits
    float unscale;      // its inverse
};

// A row that has a loss, in the order of the rows; behind the last one up to a multiple of kHeadTileM rows of zeros.
struct HeadRow {
    int32_t row, target;
    float norm;         // its normaliser
    float a, b;         // the gradient of logit v is a * softmax[v] - b * [v == target]
    int32_t low;        // != 0: the row of what rounding to 16 bits takes from another one's gradients
};

struct HeadWs {
    HeadInfo *info;
    HeadRow *rows;      // [padded rows]
    int32_t *place;     // [rows]: its place among the used rows, -1: no loss, -2: its target lies outside the vocabulary
    void *hidden;       // [padded rows, width]: hidden states of the used rows
    float *hit;         // [padded rows]: the target's logit; backward, more than 64 rows: its gradient
    int32_t *first;     // backward, more than 64 rows: [vocab]: where the used rows with this target begin in `order`, -1: there are none;
    int32_t *order;     // [padded rows]: the used rows by their targets, those of one target in their order; and
    int32_t *count;     // [padded rows]: where a target's rows begin, their number
    float2 *parts;      // [padded rows, two per tile of the vocabulary]: largest logit and the sum of exp relative to it
    void *grads;        // [padded rows, piece]: gradients of a piece's logits
    float *sums;        // [splits, used rows up to a multiple of kHeadTileM, width]: gradients of the hidden states so far
};

// A tensor map (stg_head_loss.cu): sizes and boxes from the innermost dimension on, strides in bytes between the others; zeros outside.
int head_map_of(StgHandle h, CUtensorMap *map, CUtensorMapDataType type, int dims, const void *p, const cuuint64_t *size, const cuuint64_t *stride, const cuuint32_t *box,
                CUtensorMapSwizzle swizzle);

}  // namespace stg
