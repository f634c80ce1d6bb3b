// The products of a head's loss and of its gradients on the tensor cores, one kernel with four epilogues.
//
//   kStats   logits = hidden weight^T, of which a tile leaves each row's maximum, the sum of exp relative to it and the target's logit
//   kGrad    the same logits again; their gradients, rounded to the operands' 16 bits, for the two products below
//   kHidden  gradients of the hidden states += gradients weight, over a piece of the vocabulary, in fp32
//   kWeight  gradients of the weight = gradients^T hidden, for a piece of the vocabulary, rounded once
//
// Persistent pairs of CTAs take tiles of 256 x 256 (PAIR; up to 128 rows: single CTAs take tiles of 128 x tile_n).  Each CTA loads 64 columns
// of its 128 rows of the one operand and of its half of the other at a time by TMA, into a ring of six stages; one thread of the pair
// issues tcgen05.mma into one of two accumulators in tensor memory, and eight warps of each CTA work on the other one meanwhile: a
// thread has one row.  Operands lie in shared memory with their rows along K (hidden, weight, gradients) or along M or N
// (weight and hidden states of the two gradients' products, gradients transposed): nothing is transposed in memory.
//
// The tensor cores' additions lose up to a step of the running sum each, always towards zero.  For the losses a sum is therefore
// kept for kAccBlocks * 64 columns at most and the parts are added up in registers, which costs nothing next to the products
// (8192 x 4096 x 151,936: the normalisers' error 1.7e-6 without, relative).
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
    const int32_t *targets;  // kStats: the hidden states are the caller's own, `used_rows` of them; else NULL
    int used_rows;
    int rows_pad;
    int n;              // columns of the product: vocabulary entries of the piece (kStats, kGrad), width
    int m;              // kWeight: vocabulary entries of the piece
    int k;              // width (kStats, kGrad), vocabulary entries of the piece (kHidden)
    int first;          // the piece's first vocabulary entry
    int tile_n;         // a multiple of 16, at most 256
    int group;          // tiles are taken in groups of so many rows of tiles, column by column
    float cap;
    float2 *parts;      // [rows, pieces]
    int pieces;
    float *hit;
    void *out;          // where map_out's rows lie, and elements between them
    int64_t out_stride;
    int a_rows;         // rows of the first operand's boxes: fewer than 128 where there are fewer rows
};

constexpr int kGemmEpiWarps = 8;
constexpr int kAccBlocks = 16;
constexpr int kGemmThreads = 64 + 32 * kGemmEpiWarps;
constexpr int kGemmK = 64;                                  // columns of a stage: 128 bytes, the swizzle's width
constexpr int kGemmABytes = kHeadTileM * kGemmK * 2;
template <bool PAIR>
struct GemmRing {
    static constexpr int kStages = PAIR ? 6 : 4;
    static constexpr int kBBytes = (PAIR ? 128 : 256) * kGemmK * 2;
    static constexpr int kStageBytes = kGemmABytes + kBBytes;
    static constexpr int kSmem = 1024 + kStages * kStageBytes;
};
constexpr int kGemmOut = 4096;                              // bytes that each of the eight warps writes its results from: 32 rows of 128 bytes
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

// tanh(x) as 1 - 2 / (exp(2 x) + 1): off by 2^-22 at most, of 1, which a soft cap's logits are looked at in.  (tanhf took longer than the
// products: 1000 x 2560 x 262,144 in 2015 us.)
__device__ __forceinline__ float tanh_fast(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(exp2_fast(x * (2.f * kLog2e)) + 1.f));
    return fmaf(-2.f, y, 1.f);
}
template <bool CAP>
__device__ __forceinline__ float head_capped(float x, float cap, float by_cap) { return CAP ? tanh_fast(x * by_cap) * cap : x; }

// A tile, or the part of one that a split takes: blocks [begin, end) of the sum.
struct HeadTile {
    int m, n, split, begin, end;
    __device__ __forceinline__ HeadTile(int t, int tiles_m, int tiles_n, int group, int splits, int blocks)
    {
        const int each = tiles_m * tiles_n;
        split = splits == 1 ? 0 : t / each;
        t -= split * each;
        const int first = t / (group * tiles_n) * group, rows = min(group, tiles_m - first), in = t - first * tiles_n;
        m = first + in % rows;
        n = in / rows;
        begin = (int)((int64_t)blocks * split / splits);
        end = (int)((int64_t)blocks * (split + 1) / splits);
    }
};

template <int MODE, bool BF16, bool CAP, bool PAIR>
__global__ void __launch_bounds__(kGemmThreads, 1) k_head_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                               const __grid_constant__ CUtensorMap map_out, const __grid_constant__ HeadGemm g)
{
    using Ring = GemmRing<PAIR>;
    constexpr bool kAMn = MODE == kWeight, kBMn = MODE == kHidden || MODE == kWeight;
    constexpr int kStages = Ring::kStages, kCtas = PAIR ? 2 : 1, kTileM = kCtas * kHeadTileM;
    extern __shared__ unsigned char raw[];
    __shared__ alignas(8) uint64_t bars[2 * kStages + 4];
    __shared__ uint32_t tmem_slot;
    __shared__ int dead_;
    volatile int *dead = &dead_;
    const uint32_t ring = (smem_at(raw) + 1023u) & ~1023u;
    const uint32_t full = smem_at(bars), empty = full + 8 * kStages, acc_full = empty + 8 * kStages, acc_empty = acc_full + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0u;

    if (warp == 0 && one_lane()) {
        tma_prefetch(&map_a);
        tma_prefetch(&map_b);
        if (MODE != kStats) tma_prefetch(&map_out);
        for (int i = 0; i < kStages; i++) { bar_init(full + 8 * i, 1); bar_init(empty + 8 * i, 1); }
        for (int i = 0; i < 2; i++) { bar_init(acc_full + 8 * i, 1); bar_init(acc_empty + 8 * i, kCtas * kGemmEpiWarps); }
        dead_ = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 1) tmem_alloc<PAIR>(smem_at(&tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_release();
    pdl_wait();
    asm volatile("fence.proxy.async;" ::: "memory");  // what the kernels ahead have written is read by TMA

    const int used = MODE == kStats && g.targets ? g.used_rows : g.info->used;
    const int tiles_m = ((MODE == kWeight ? g.m : used) + kTileM - 1) / kTileM;
    const int tiles_n = (g.n + g.tile_n - 1) / g.tile_n;
    const int splits = MODE == kHidden ? g.info->splits : 1;
    const int tiles = tiles_m * tiles_n * splits;
    const int blocks = ((MODE == kWeight ? used : g.k) + kGemmK - 1) / kGemmK;
    const int part = MODE == kStats ? kAccBlocks : 1 << 30;  // blocks of an accumulator
    const int first_tile = blockIdx.x / kCtas, step = gridDim.x / kCtas;

    if (warp == 0) {
        if (one_lane()) {
            uint32_t at = 0;  // stages filled so far
            bool ok = true;
            const int own_n = g.tile_n / kCtas, chunks = (own_n + 63) / 64;
            const uint32_t bytes = kCtas * ((kAMn ? kGemmABytes : (uint32_t)g.a_rows * 128u) + (kBMn ? (uint32_t)chunks * 8192u : (uint32_t)own_n * 128u));
            for (int t = first_tile; ok && t < tiles; t += step) {
                const HeadTile tile(t, tiles_m, tiles_n, g.group, splits, blocks);
                const int m0 = tile.m * kTileM + rank * kHeadTileM, n0 = tile.n * g.tile_n + rank * own_n;
                for (int kb = tile.begin; kb < tile.end; kb++, at++) {
                    const uint32_t s = at % kStages;
                    ok = bar_wait(empty + 8 * s, ((at / kStages) & 1u) ^ 1u, dead);
                    if (!ok) break;
                    const uint32_t a = ring + s * Ring::kStageBytes, b = a + kGemmABytes;
                    const uint32_t bar = PAIR ? cluster_at(full + 8 * s, 0) : full + 8 * s;  // both CTAs' bytes count on the first one's barrier
                    const int k0 = kb * kGemmK;
                    if (rank == 0) bar_expect(full + 8 * s, bytes);
                    if (kAMn) {
                        tma_load<PAIR>(a, &map_a, m0, k0, bar);
                        tma_load<PAIR>(a + 8192, &map_a, m0 + 64, k0, bar);
                    } else {
                        tma_load<PAIR>(a, &map_a, k0, m0, bar);
                    }
                    if (kBMn) {
                        for (int c = 0; c < chunks; c++) tma_load<PAIR>(b + c * 8192, &map_b, n0 + c * 64, (MODE == kHidden ? g.first : 0) + k0, bar);
                    } else {
                        tma_load<PAIR>(b, &map_b, k0, g.first + n0, bar);
                    }
                }
            }
            // copies in flight end before the CTA does
            for (uint32_t i = at < kStages ? 0 : at - kStages; rank == 0 && i < at; i++)
                for (uint32_t j = 0; j < (1u << 20) && !bar_try(full + 8 * (i % kStages), (i / kStages) & 1u); j++) {}
        }
    } else if (warp == 1) {
        if (rank == 0 && one_lane()) {
            const uint32_t idesc = tc_idesc(BF16, kAMn, kBMn, kTileM, (uint32_t)g.tile_n);
            const uint64_t da = tc_desc_base(kAMn ? 8192u : 16u), db = tc_desc_base(kBMn ? 8192u : 16u);
            uint32_t at = 0, unit = 0;
            bool ok = true;
            for (int t = first_tile; ok && t < tiles; t += step) {
                const HeadTile tile(t, tiles_m, tiles_n, g.group, splits, blocks);
                for (int k0 = tile.begin, k1; ok && k0 < tile.end; k0 = k1, unit++) {
                    const uint32_t acc = unit & 1u;
                    k1 = min(tile.end - k0, part) + k0;
                    ok = bar_wait(acc_empty + 8 * acc, ((unit >> 1) & 1u) ^ 1u, dead);
                    if (!ok) break;
                    tc_fence_after();
                    for (int kb = k0; kb < k1; kb++, at++) {
                        const uint32_t s = at % kStages;
                        ok = bar_wait(full + 8 * s, (at / kStages) & 1u, dead);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t a = ring + s * Ring::kStageBytes, b = a + kGemmABytes;
#pragma unroll
                        for (int k = 0; k < kGemmK / 16; k++)
                            tc_mma<PAIR>(tmem + acc * 256, tc_desc(da, a + k * (kAMn ? 2048 : 32)), tc_desc(db, b + k * (kBMn ? 2048 : 32)), idesc, kb > k0 || k > 0);
                        tc_commit<PAIR>(empty + 8 * s);
                    }
                    if (ok) tc_commit<PAIR>(acc_full + 8 * acc);
                }
            }
            // what was issued ends before tensor memory is given back: the last commits arrive on `empty`
            for (uint32_t i = at < kStages ? 0 : at - kStages; i < at; i++)
                for (uint32_t j = 0; j < (1u << 20) && !bar_try(empty + 8 * (i % kStages), (i / kStages) & 1u); j++) {}
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int chunks = g.tile_n / 16, c_begin = half == 0 ? 0 : (chunks + 1) / 2, c_end = half == 0 ? (chunks + 1) / 2 : chunks;  // 8 at most
        const float unscale = MODE == kWeight ? g.info->unscale : 1.f, scale = MODE == kGrad ? g.info->scale : 1.f;
        const uint32_t free_bar = PAIR ? cluster_at(acc_empty, 0) : acc_empty;
        const uint32_t out = ring + kStages * Ring::kStageBytes + (warp - 2) * kGemmOut;
        const float by_cap = CAP ? 1.f / g.cap : 0.f;
        uint32_t unit = 0;
        bool ok = true;
        for (int t = first_tile; ok && t < tiles; t += step) {
            const HeadTile tile(t, tiles_m, tiles_n, g.group, splits, blocks);
            const int m0 = tile.m * kTileM + rank * kHeadTileM, tn = tile.n, n0 = tn * g.tile_n;
            const bool some = tile.begin < tile.end;
            const int r = m0 + quarter * 32 + lane;
            // where the unit's accumulator is, once it is full, and the word that it has been read
            auto full_unit = [&]() -> uint32_t {
                const uint32_t acc = unit & 1u;
                ok = __all_sync(0xFFFFFFFFu, bar_wait(acc_full + 8 * acc, (unit >> 1) & 1u, dead));
                tc_fence_after();
                return tmem + acc * 256 + ((uint32_t)(quarter * 32) << 16);
            };
            auto read_unit = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (PAIR) bar_arrive_remote(free_bar + 8 * (unit & 1u));
                    else bar_arrive(free_bar + 8 * (unit & 1u));
                }
                unit++;
            };
            if constexpr (MODE == kStats) {
                const bool rows_here = m0 + quarter * 32 < used;  // of this warp
                const int target = r >= used ? -1 : g.targets ? g.targets[r] : g.rows[r].target;
                float z[8][16];
                for (int k0 = 0; k0 < blocks; k0 += kAccBlocks) {
                    const uint32_t from = full_unit();
                    if (!ok) break;
#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        if (c_begin + c >= c_end || !rows_here) break;
                        HeadCols x;
                        tmem_load16(from + (c_begin + c) * 16, x.v);
                        tmem_loaded();
#pragma unroll
                        for (int i = 0; i < 16; i++) z[c][i] = k0 == 0 ? x.f(i) : z[c][i] + x.f(i);
                    }
                    read_unit();
                }
                if (!ok) break;
                if (!rows_here) continue;
                float top = -CUDART_INF_F;
                float most[4] = {top, top, top, top};
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    const int col = n0 + (c_begin + c) * 16;
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const bool in = c_begin + c < c_end && col + i < g.n;
                        z[c][i] = in ? head_capped<CAP>(z[c][i], g.cap, by_cap) : -CUDART_INF_F;
                        most[i & 3] = fmaxf(most[i & 3], z[c][i]);
                        if (in && col + i == target) g.hit[r] = z[c][i];
                    }
                }
                top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
                const float ref = top == -CUDART_INF_F ? 0.f : top * kLog2e;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 8; c++)
#pragma unroll
                    for (int i = 0; i < 16; i++) sum[i & 3] += exp2_fast(fmaf(z[c][i], kLog2e, -ref));
                if (r < used) g.parts[(int64_t)r * g.pieces + 2 * tn + half] = make_float2(top, (sum[0] + sum[1]) + (sum[2] + sum[3]));
            } else {
                // what 128 bytes of a row hold goes through shared memory and out as a box of the warp's 32 rows
                // (one row of tiles, whose widths are not whole boxes, has few gradients: each thread writes its own)
                constexpr bool kDirect = MODE == kGrad && !PAIR;
                constexpr int kOutCols = MODE == kHidden ? 32 : 64, kOutChunks = kOutCols / 16;
                const int slab = (used + kHeadTileM - 1) / kHeadTileM * kHeadTileM;  // rows of a split
                const int r0 = m0 + quarter * 32;
                const bool rows_here = r0 < (MODE == kWeight ? g.m : MODE == kHidden ? slab : g.rows_pad) && (some || MODE != kHidden || g.first == 0);
                HeadRow row = {};
                if (MODE == kGrad && rows_here) row = g.rows[r];
                const uint32_t from = some ? full_unit() : 0u;
                if (!ok) break;
                for (int c0 = c_begin; c0 < c_end && rows_here; c0 += kOutChunks) {
                    if (n0 + c0 * 16 >= g.n) break;
                    if (!kDirect) {
                        if (lane == 0) store_read();
                        __syncwarp();
                    }
#pragma unroll
                    for (int c = 0; c < kOutChunks; c++) {
                        const int col = n0 + (c0 + c) * 16;
                        if (c0 + c >= c_end) break;
                        HeadCols x;
                        if (some) {
                            tmem_load16(from + (c0 + c) * 16, x.v);
                            tmem_loaded();
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; i++) x.v[i] = 0u;
                        }
                        const uint32_t to = out + lane * 128;  // its 16 bytes are exchanged as a 128-byte swizzle wants them
                        if constexpr (MODE == kHidden) {
#pragma unroll
                            for (int i = 0; i < 4; i++) shared_store(to + (((4 * c + i) ^ (lane & 7)) << 4), x.v[4 * i], x.v[4 * i + 1], x.v[4 * i + 2], x.v[4 * i + 3]);
                        } else {
                            uint32_t o[8];
                            if constexpr (MODE == kGrad) {
                                float d[16];
#pragma unroll
                                for (int i = 0; i < 16; i++) {
                                    float slope = scale, z = x.f(i);
                                    if (CAP) {
                                        const float th = tanh_fast(z * by_cap);
                                        z = th * g.cap;
                                        slope *= 1.f - th * th;
                                    }
                                    d[i] = row.a * exp2_fast(fmaf(z, kLog2e, -row.norm2));
                                    if (g.first + col + i == row.target) d[i] -= row.b;
                                    d[i] = r < used ? d[i] * slope : 0.f;
                                }
#pragma unroll
                                for (int i = 0; i < 8; i++) o[i] = pack2<BF16>(d[2 * i], d[2 * i + 1]);
                            } else {
#pragma unroll
                                for (int i = 0; i < 8; i++) o[i] = pack2<BF16>(x.f(2 * i) * unscale, x.f(2 * i + 1) * unscale);
                            }
                            if constexpr (kDirect) {
                                uint4 *at = (uint4 *)((uint16_t *)g.out + (int64_t)r * g.out_stride + col);
                                at[0] = make_uint4(o[0], o[1], o[2], o[3]);
                                at[1] = make_uint4(o[4], o[5], o[6], o[7]);
                            } else {
                                shared_store(to + (((2 * c) ^ (lane & 7)) << 4), o[0], o[1], o[2], o[3]);
                                shared_store(to + (((2 * c + 1) ^ (lane & 7)) << 4), o[4], o[5], o[6], o[7]);
                            }
                        }
                    }
                    if (kDirect) continue;
                    async_proxy_fence();
                    __syncwarp();
                    if (lane == 0) {
                        const int x = n0 + c0 * 16, y = (MODE == kWeight ? g.first : MODE == kHidden ? tile.split * slab : 0) + r0;
                        if (MODE == kHidden && g.first > 0) tma_store<true>(&map_out, x, y, out);
                        else tma_store<false>(&map_out, x, y, out);
                        store_commit();
                    }
                }
                if (some) read_unit();
            }
        }
        if (MODE != kStats && lane == 0) store_done();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    tc_fence_after();
    if (warp == 1) tmem_free<PAIR>(tmem, 512);
    if (dead_ != 0) {  // a wait has given up: what this CTA should have written is NaN
        for (int t = first_tile; t < tiles; t += step) {
            const HeadTile tile(t, tiles_m, tiles_n, g.group, splits, blocks);
            for (int i = threadIdx.x; i < kHeadTileM * g.tile_n; i += kGemmThreads) {
                const int r = tile.m * kTileM + (int)rank * kHeadTileM + i / g.tile_n, c = tile.n * g.tile_n + i % g.tile_n;
                if (MODE == kStats && r < used && i % g.tile_n < 2) g.parts[(int64_t)r * g.pieces + 2 * tile.n + i % g.tile_n] = make_float2(0.f, CUDART_NAN_F);
                if (MODE == kHidden && r < used && c < g.n) ((float *)g.out)[((int64_t)tile.split * ((used + kHeadTileM - 1) / kHeadTileM * kHeadTileM) + r) * g.out_stride + c] = CUDART_NAN_F;
                if ((MODE == kGrad && r < used && c < g.n) || (MODE == kWeight && r < g.m && c < g.n))
                    ((uint16_t *)g.out)[(int64_t)((MODE == kWeight ? g.first : 0) + r) * g.out_stride + c] = 0x7FFFu;
            }
        }
    }
}

}  // namespace stg
