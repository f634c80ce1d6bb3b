// The products of a head's loss and of its gradients on the tensor cores, one kernel with four epilogues.
//
//   kStats   logits = hidden weight^T, of which a tile leaves each row's maximum, the sum of exp relative to it and the target's logit
//   kGrad    the same logits again; their gradients, rounded to the operands' 16 bits, for the two products below
//   kHidden  gradients of the hidden states += gradients weight, over a piece of the vocabulary, in fp32
//   kWeight  gradients of the weight = gradients^T hidden, for a piece of the vocabulary, rounded once
//
// A persistent CTA per SM takes tiles of 128 x tile_n.  One warp loads 64 columns of both operands at a time by TMA into a ring of four stages,
// one thread issues tcgen05.mma into one of two accumulators in tensor memory, and eight warps work on the other one meanwhile: a
// thread has one row.  Operands lie in shared memory with their rows along K (hidden, weight, gradients) or along M or N
// (weight and hidden states of the two gradients' products, gradients transposed): nothing is transposed in memory.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "stg_head.h"
#include "stg_pdl.cuh"
#include "stg_tc.cuh"

namespace stg {

enum HeadMode { kStats = 0, kGrad = 1, kHidden = 2, kWeight = 3 };

struct HeadGemm {
    HeadInfo *info;
    const HeadRow *rows;
    int n;              // columns of the product: vocabulary entries of the piece (kStats, kGrad), width
    int m;              // kWeight: vocabulary entries of the piece
    int k;              // width (kStats, kGrad), vocabulary entries of the piece (kHidden)
    int first;          // the piece's first vocabulary entry
    int tile_n;         // a multiple of 16, at most 256
    float cap;
    float2 *parts;      // [rows, pieces]
    int pieces;
    float *hit;
    void *grads;
    int64_t grads_stride;
    float *sums;
    int64_t sums_stride;
    void *out;
    int64_t out_stride;
};

constexpr int kGemmStages = 4;
constexpr int kGemmEpiWarps = 8;
constexpr int kGemmThreads = 64 + 32 * kGemmEpiWarps;
constexpr int kGemmK = 64;                                  // columns of a stage: 128 bytes, the swizzle's width
constexpr int kGemmABytes = kHeadTileM * kGemmK * 2;
constexpr int kGemmBBytes = 256 * kGemmK * 2;
constexpr int kGemmStageBytes = kGemmABytes + kGemmBBytes;
constexpr int kGemmSmem = 1024 + kGemmStages * kGemmStageBytes;
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    uint32_t r;
    if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Sixteen accumulators of a row.
struct HeadCols {
    uint32_t v[16];
    __device__ __forceinline__ float f(int i) const { return __uint_as_float(v[i]); }
};

template <int MODE, bool BF16, bool CAP>
__global__ void __launch_bounds__(kGemmThreads, 1) k_head_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                               const __grid_constant__ HeadGemm g)
{
    constexpr bool kAMn = MODE == kWeight, kBMn = MODE == kHidden || MODE == kWeight;
    extern __shared__ unsigned char raw[];
    __shared__ alignas(8) uint64_t bars[2 * kGemmStages + 4];
    __shared__ uint32_t tmem_slot;
    __shared__ int dead_;
    volatile int *dead = &dead_;
    const uint32_t ring = (smem_at(raw) + 1023u) & ~1023u;
    const uint32_t full = smem_at(bars), empty = full + 8 * kGemmStages, acc_full = empty + 8 * kGemmStages, acc_empty = acc_full + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 0 && one_lane()) {
        tma_prefetch(&map_a);
        tma_prefetch(&map_b);
        for (int i = 0; i < kGemmStages; i++) { bar_init(full + 8 * i, 1); bar_init(empty + 8 * i, 1); }
        for (int i = 0; i < 2; i++) { bar_init(acc_full + 8 * i, 1); bar_init(acc_empty + 8 * i, kGemmEpiWarps); }
        dead_ = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 1) tmem_alloc(smem_at(&tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_release();
    pdl_wait();

    const int used = g.info->used;
    const int tiles_m = ((MODE == kWeight ? g.m : used) + kHeadTileM - 1) / kHeadTileM;
    const int tiles_n = (g.n + g.tile_n - 1) / g.tile_n;
    const int tiles = tiles_m * tiles_n;
    const int blocks = ((MODE == kWeight ? used : g.k) + kGemmK - 1) / kGemmK;

    if (warp == 0) {
        if (one_lane()) {
            uint32_t at = 0;  // stages filled so far
            bool ok = true;
            const int chunks = (g.tile_n + 63) / 64;
            const uint32_t bytes = kGemmABytes + (kBMn ? (uint32_t)chunks * 8192u : (uint32_t)g.tile_n * 128u);
            for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
                const int m0 = (t % tiles_m) * kHeadTileM, n0 = (t / tiles_m) * g.tile_n;
                for (int kb = 0; kb < blocks; kb++, at++) {
                    const uint32_t s = at % kGemmStages, bar = full + 8 * s;
                    ok = bar_wait(empty + 8 * s, ((at / kGemmStages) & 1u) ^ 1u, dead);
                    if (!ok) break;
                    const uint32_t a = ring + s * kGemmStageBytes, b = a + kGemmABytes;
                    const int k0 = kb * kGemmK;
                    bar_expect(bar, bytes);
                    if (kAMn) {
                        tma_load(a, &map_a, m0, k0, bar);
                        tma_load(a + 8192, &map_a, m0 + 64, k0, bar);
                    } else {
                        tma_load(a, &map_a, k0, m0, bar);
                    }
                    if (kBMn) {
                        for (int c = 0; c < chunks; c++) tma_load(b + c * 8192, &map_b, n0 + c * 64, (MODE == kHidden ? g.first : 0) + k0, bar);
                    } else {
                        tma_load(b, &map_b, k0, g.first + n0, bar);
                    }
                }
            }
            // copies in flight end before the CTA does
            for (uint32_t i = at < kGemmStages ? 0 : at - kGemmStages; i < at; i++)
                for (uint32_t j = 0; j < (1u << 20) && !bar_try(full + 8 * (i % kGemmStages), (i / kGemmStages) & 1u); j++) {}
        }
    } else if (warp == 1) {
        if (one_lane()) {
            const uint32_t idesc = tc_idesc(BF16, kAMn, kBMn, kHeadTileM, (uint32_t)g.tile_n);
            const uint64_t da = tc_desc_base(kAMn ? 8192u : 16u), db = tc_desc_base(kBMn ? 8192u : 16u);
            uint32_t at = 0, tile = 0;
            bool ok = true;
            for (int t = blockIdx.x; ok && blocks > 0 && t < tiles; t += gridDim.x, tile++) {
                const uint32_t acc = tile & 1u;
                ok = bar_wait(acc_empty + 8 * acc, ((tile >> 1) & 1u) ^ 1u, dead);
                if (!ok) break;
                tc_fence_after();
                for (int kb = 0; kb < blocks; kb++, at++) {
                    const uint32_t s = at % kGemmStages;
                    ok = bar_wait(full + 8 * s, (at / kGemmStages) & 1u, dead);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t a = ring + s * kGemmStageBytes, b = a + kGemmABytes;
#pragma unroll
                    for (int k = 0; k < kGemmK / 16; k++)
                        tc_mma(tmem + acc * 256, tc_desc(da, a + k * (kAMn ? 2048 : 32)), tc_desc(db, b + k * (kBMn ? 2048 : 32)), idesc, kb > 0 || k > 0);
                    tc_commit(empty + 8 * s);
                }
                if (ok) tc_commit(acc_full + 8 * acc);
            }
            // what was issued ends before tensor memory is given back: the last commits arrive on `empty`
            for (uint32_t i = at < kGemmStages ? 0 : at - kGemmStages; i < at; i++)
                for (uint32_t j = 0; j < (1u << 20) && !bar_try(empty + 8 * (i % kGemmStages), (i / kGemmStages) & 1u); j++) {}
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int chunks = g.tile_n / 16, c_begin = half == 0 ? 0 : (chunks + 1) / 2, c_end = half == 0 ? (chunks + 1) / 2 : chunks;
        const float unscale = g.info->unscale, scale = g.info->scale;
        uint32_t tile = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, tile++) {
            const uint32_t acc = tile & 1u;
            const int m0 = (t % tiles_m) * kHeadTileM, tn = t / tiles_m, n0 = tn * g.tile_n;
            const int r = m0 + quarter * 32 + lane;  // below rows_pad
            const uint32_t from = tmem + acc * 256 + ((uint32_t)(quarter * 32) << 16);
            HeadRow row = {};
            if (MODE == kStats || MODE == kGrad) row = g.rows[r];
            if (blocks > 0) {
                bool ok = bar_wait(acc_full + 8 * acc, (tile >> 1) & 1u, dead);
                if (!__all_sync(0xFFFFFFFFu, ok)) break;
                tc_fence_after();
            }
            float top = -CUDART_INF_F, sum = 0.f;
            for (int c = c_begin; c < c_end; c++) {
                const int col = n0 + c * 16;
                HeadCols x;
                if (blocks > 0) {
                    tmem_load16(from + c * 16, x.v);
                    tmem_loaded();
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++) x.v[i] = 0u;
                }
                if (MODE == kStats) {
                    if (col >= g.n) continue;  // the same for the whole warp
                    float z[16], most = -CUDART_INF_F;
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        z[i] = CAP ? tanhf(x.f(i) / g.cap) * g.cap : x.f(i);
                        if (col + i >= g.n) z[i] = -CUDART_INF_F;
                        most = fmaxf(most, z[i]);
                    }
                    const unsigned at = (unsigned)(row.target - col);
                    if (at < 16u) {
                        float hit = 0.f;
#pragma unroll
                        for (int i = 0; i < 16; i++) hit = at == (unsigned)i ? z[i] : hit;
                        g.hit[r] = hit;
                    }
                    const float next = fmaxf(top, most), ref = next == -CUDART_INF_F ? 0.f : next * kLog2e;
                    float s = sum * exp2_fast(top * kLog2e - ref);
                    if (top == -CUDART_INF_F) s = 0.f;
#pragma unroll
                    for (int i = 0; i < 16; i++) s += exp2_fast(fmaf(z[i], kLog2e, -ref));
                    sum = s;
                    top = next;
                } else if (MODE == kGrad) {
                    uint32_t o[8];
                    float d[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        float slope = scale;
                        float z = x.f(i);
                        if (CAP) {
                            const float th = tanhf(z / g.cap);
                            z = th * g.cap;
                            slope *= 1.f - th * th;
                        }
                        d[i] = row.a * exp2_fast(fmaf(z, kLog2e, -row.norm2));
                        if (g.first + col + i == row.target) d[i] -= row.b;
                        d[i] = col + i < g.n ? d[i] * slope : 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) o[i] = pack2<BF16>(d[2 * i], d[2 * i + 1]);
                    uint4 *to = (uint4 *)((uint16_t *)g.grads + (int64_t)r * g.grads_stride + col);
                    to[0] = make_uint4(o[0], o[1], o[2], o[3]);
                    to[1] = make_uint4(o[4], o[5], o[6], o[7]);
                } else if (MODE == kHidden) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (col + 4 * i >= g.n) break;  // width is a multiple of 8
                        float4 *to = (float4 *)(g.sums + (int64_t)r * g.sums_stride + col + 4 * i);
                        float4 v = make_float4(x.f(4 * i), x.f(4 * i + 1), x.f(4 * i + 2), x.f(4 * i + 3));
                        if (g.first > 0) {
                            const float4 w = *to;
                            v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
                        }
                        *to = v;
                    }
                } else if (r < g.m) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        if (col + 8 * i >= g.n) break;
                        uint32_t o[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) o[j] = pack2<BF16>(x.f(8 * i + 2 * j) * unscale, x.f(8 * i + 2 * j + 1) * unscale);
                        *(uint4 *)((uint16_t *)g.out + (int64_t)(g.first + r) * g.out_stride + col + 8 * i) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                }
            }
            if (MODE == kStats) g.parts[(int64_t)r * g.pieces + 2 * tn + half] = make_float2(top, sum);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(acc_empty + 8 * acc);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_free(tmem, 512);
    if (threadIdx.x == 0 && dead_ != 0) g.info->failed = 1;
}

}  // namespace stg
