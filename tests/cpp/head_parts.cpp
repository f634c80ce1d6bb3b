// Gradients of a weight that are summed in parts: the ring of their tiles of half the width, and from which sizes on sums are taken in parts.  Prints
// "head_parts: ok".
#include "stg_head_plan.h"

#include <cstdio>

using namespace stg;

int main()
{
    const GemmRing r = gemm_ring(kWeight, true, 128, kHeadTileM);
    const int b_bytes = 128 / 2 * kGemmK * 2;  // a CTA of the pair has half of the columns
    bool ok = r.stages >= 2 && r.stages <= kGemmStages && r.a_at >= b_bytes && r.a_at % 1024 == 0 && r.stage_bytes % 1024 == 0 && r.stage_bytes - r.a_at >= kGemmABytes &&
              r.stages * r.stage_bytes <= kGemmRingBytes;
    // parts are whole blocks, and so many rows are always pairs'
    ok = ok && kWeightRows % kGemmK == 0 && kGradColumns % kGemmK == 0 && kWeightRows > 2 * kHeadTileM && kWeightRows > kLowRows;
    for (bool bf16 : {false, true}) {
        const int f = bf16 ? 4 : 1;
        ok = ok && !grad_in_parts(f * kGradColumns, bf16) && grad_in_parts(f * kGradColumns + 8, bf16) && !weight_in_parts(f * kWeightRows, bf16) &&
             weight_in_parts(f * kWeightRows + 1, bf16) && head_shape(f * kWeightRows + 1, 1000, 64, 148, true).pair;
    }
    std::printf(ok ? "head_parts: ok\n" : "head_parts: wrong\n");
    return ok ? 0 : 1;
}
