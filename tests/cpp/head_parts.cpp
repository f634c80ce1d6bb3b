// Gradients of a weight that are summed in parts: the ring of their tiles of half the width, and the parts.  Prints
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
    // parts are whole blocks, and rows that are summed in parts are always pairs'
    for (bool bf16 : {false, true}) {
        ok = ok && part_of(kWeightRows, bf16) == (bf16 ? 8 : 1) * kWeightRows && kLowRows < kWeightRows;
        ok = ok && kWeightRows % kGemmK == 0 && kGradColumns % kGemmK == 0 && kHiddenColumns % kGemmK == 0 && head_shape(part_of(kWeightRows, bf16) + 1, 1000, 64, 148, true).pair;
    }
    std::printf(ok ? "head_parts: ok\n" : "head_parts: wrong\n");
    return ok ? 0 : 1;
}
