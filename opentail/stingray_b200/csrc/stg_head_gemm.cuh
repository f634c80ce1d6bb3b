// The products of a head's loss and of its gradients on the tensor cores, one kernel with four epilogues.
//
//   kStats   logits = hidden weight^T, of which a tile leaves each row's maximum, the sum of exp relative to it and the target's logit
//   kGrad    the same logits again; their gradients, rounded to the operands' 16 bits, for the two products below
//   kHidden  gradients of the hidden states += gradients weight, over a piece of the vocabulary, in fp32
//   kWeight  gradients of the weight = gradients^T hidden, for a piece of the vocabulary, rounded once
//
// Persistent pairs of CTAs take tiles of 256 x tile_n (PAIR; up to 128 rows: single CTAs take tiles of 128 x tile_n).  Each CTA loads 64 columns
// of its 128 rows of the one operand and of its half of the other at a time by TMA, into a ring of up to eight stages; one thread of the pair
// issues tcgen05.mma into one of two accumulators in tensor memory, and eight warps of each CTA work on the other one meanwhile: a
// thread has one row.  Operands lie in shared memory with their rows along K (hidden, weight, gradients) or along M or N
// (weight and hidden states of the two gradients' products, gradients transposed): nothing is transposed in memory.
//
// The tensor cores' additions lose up to a step of the running sum each, always towards zero, some 1e-7 of it on average.  For the losses a sum is
// therefore kept for 1024 columns at most and the parts are added up in registers (8192 x 4096 x 151,936: the normalisers are 3.7e-7 off,
// 1.7e-6 without, relative; 512 columns: 7.9 ms in place of 7.3); single CTAs, which wait for memory, take 512 (64 x 4096 x 151,936: 1.8e-7 off).
// The backward pass takes parts where a sum is so long that it would show beside the results' rounding (stg_head_plan.h; bf16, eight times as
// coarse, from eight times as many terms on).  Gradients of logits take the losses' parts, which makes the logits the same, bit for bit, so that probabilities add
// up to 1 whatever the logits are off: 20 rows x 16,384 x 2000 in fp16, a wrong token certain at logits of 65, are 2.3e-4 off, their own rounding, in place
// of 1.0e-3.  It takes more registers than there are: 2 to 5 % of a step (2048 x 8192 x 32,000: 2490 us, 2360 in one accumulator).  Gradients
// of a weight take tiles of half the width for it, 11 % of a step of 32,768 x 2048 x 32,000: 262,144 rows of one sign, fp16, are 2.3e-4 off in place of 1.6e-3.
// Those of the hidden states add their parts in memory.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "stg_head.h"
#include "stg_pdl.cuh"
#include "stg_tc.cuh"

namespace stg {

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
    const int32_t *first_of, *order, *count;  // kWeight: HeadWs, or NULL
    const uint16_t *hidden;       // kWeight: [rows, n]
    int a_rows;         // rows of the first operand's boxes: fewer than 128 where there are fewer rows
    int stages, stage_bytes;  // the second operand's boxes ahead of the first's
    int a_at;
};

// Blocks that an accumulator holds.  LONG: sums that are taken in parts in registers (stg_head_plan.h).
template <int MODE, bool BF16, bool PAIR, bool LONG>
constexpr int kAccBlocks = MODE == kStats || (MODE == kGrad && LONG) ? (PAIR ? 16 : 8)
                         : MODE == kHidden                           ? part_of(kHiddenColumns, BF16) / kGemmK
                         : MODE == kWeight && LONG                   ? part_of(kWeightRows, BF16) / kGemmK
                                                                     : 1 << 30;
constexpr int kGemmThreads = 64 + 32 * kGemmEpiWarps;
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

template <bool BF16>
__device__ __forceinline__ float half_of(uint32_t x)  // its lower half
{
    return BF16 ? __uint_as_float(x << 16) : __half2float(__ushort_as_half((unsigned short)x));
}

// Sixteen accumulators of a row.
struct HeadCols {
    uint32_t v[16];
    __device__ __forceinline__ float f(int i) const { return __uint_as_float(v[i]); }
};

// cap * tanh(z / cap), and tanh itself, 2^-19 of their own size off at most: below |x| = 1/4 by tanh's series around 0 up to x^9, of z and not of x,
// so that a logit far below the cap stays as it is; above as 1 - 2 / (exp(2 x) + 1), which is 2^-22 off, of 1.  (tanhf took longer than the
// products: 1000 x 2560 x 262,144 in 2015 us.)
struct Capped {
    float z, tanh;
};
__device__ __forceinline__ Capped head_cap(float z, float cap, float by_cap)
{
    const float x = z * by_cap, s = x * x;
    float q;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(exp2_fast(x * (2.f * kLog2e)) + 1.f));
    const float series = fmaf(s, fmaf(s, fmaf(s, fmaf(s, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f), th = fmaf(-2.f, q, 1.f);
    return fabsf(x) < 0.25f ? Capped{z * series, x * series} : Capped{th * cap, th};
}

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

// kWeight: the lanes whose entries' rows - `n` of this lane's - the warp goes through together, a lane's after another's.  A lane by itself takes one
// row after another, at kRestAlone cycles each beside the products' traffic, all lanes at the same time; the warp takes kRestLane for a lane's and
// kRestRow more for each row.  So no accumulator is held for longer than a bounded wait lasts, however many rows have one target: 8192 rows x
// 2048 x 32,000 take 2430 us with targets spread evenly, 3150 with the k-th token 1 / k as often as the first (4100 where each lane walked through
// its own) and 4150 with one target (16,840).
constexpr unsigned kRestsAlone = 4, kRestAlone = 2000, kRestLane = 2500, kRestRow = 200;
__device__ __forceinline__ uint32_t rests_together(int n)
{
    const uint32_t many = __ballot_sync(0xFFFFFFFFu, n > (int)kRestsAlone);
    if (many == 0u) return 0u;
    const unsigned most = __reduce_max_sync(0xFFFFFFFFu, (unsigned)n), all = __reduce_add_sync(0xFFFFFFFFu, n > (int)kRestsAlone ? (unsigned)n : 0u);
    return (uint64_t)most * kRestAlone > (uint64_t)__popc(many) * kRestLane + (uint64_t)all * kRestRow ? many : 0u;
}

template <int MODE, bool BF16, bool CAP, bool PAIR, bool LONG>
__global__ void __launch_bounds__(kGemmThreads, 1) k_head_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                               const __grid_constant__ CUtensorMap map_out, const __grid_constant__ HeadGemm g)
{
    constexpr bool kAMn = MODE == kWeight, kBMn = MODE == kHidden || MODE == kWeight;
    constexpr int kCtas = PAIR ? 2 : 1, kTileM = kCtas * kHeadTileM;
    extern __shared__ unsigned char raw[];
    __shared__ alignas(8) uint64_t bars[2 * kGemmStages + 4];
    __shared__ uint32_t tmem_slot;
    __shared__ int dead_;
    volatile int *dead = &dead_;
    const uint32_t ring = (smem_at(raw) + 1023u) & ~1023u;
    const uint32_t full = smem_at(bars), empty = full + 8 * kGemmStages, acc_full = empty + 8 * kGemmStages, acc_empty = acc_full + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0u;

    if (warp == 0 && one_lane()) {
        tma_prefetch(&map_a);
        tma_prefetch(&map_b);
        if (MODE != kStats) tma_prefetch(&map_out);
        for (int i = 0; i < g.stages; i++) { bar_init(full + 8 * i, 1); bar_init(empty + 8 * i, 1); }
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
    async_fence();  // what the kernels ahead have written is read by TMA

    const int used = MODE == kStats && g.targets ? g.used_rows : g.info->used;
    const int tiles_m = ((MODE == kWeight ? g.m : used) + kTileM - 1) / kTileM;
    const int tiles_n = (g.n + g.tile_n - 1) / g.tile_n;
    const int splits = MODE == kHidden ? g.info->splits : 1;
    const int tiles = tiles_m * tiles_n * splits;
    const int blocks = ((MODE == kWeight ? used : g.k) + kGemmK - 1) / kGemmK;
    constexpr int kPart = kAccBlocks<MODE, BF16, PAIR, LONG>;
    const int first_tile = blockIdx.x / kCtas, step = gridDim.x / kCtas;

    if (warp == 0) {
        if (one_lane()) {
            uint32_t loaded = 0, phase = 1;
            int s = 0;
            bool ok = true;
            const int own_n = g.tile_n / kCtas, chunks = (own_n + 63) / 64;
            const uint32_t bytes = kCtas * ((kAMn ? kGemmABytes : (uint32_t)g.a_rows * 128u) + (kBMn ? (uint32_t)chunks * 8192u : (uint32_t)own_n * 128u));
            for (int t = first_tile; ok && t < tiles; t += step) {
                const HeadTile tile(t, tiles_m, tiles_n, g.group, splits, blocks);
                const int m0 = tile.m * kTileM + rank * kHeadTileM, n0 = tile.n * g.tile_n + rank * own_n;
                for (int kb = tile.begin; kb < tile.end; kb++, loaded++) {
                    ok = bar_wait(empty + 8 * s, phase, dead);
                    if (!ok) break;
                    const uint32_t b = ring + s * g.stage_bytes, a = b + g.a_at;
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
                    if (++s == g.stages) { s = 0; phase ^= 1u; }
                }
            }
            // copies in flight end before the CTA does
            const uint32_t n = (uint32_t)g.stages;
            for (uint32_t i = loaded < n ? 0 : loaded - n; rank == 0 && i < loaded; i++)
                for (uint32_t j = 0; j < (1u << 20) && !bar_try(full + 8 * (i % n), (i / n) & 1u); j++) {}
        }
    } else if (warp == 1) {
        if (rank == 0 && one_lane()) {
            const uint32_t idesc = tc_idesc(BF16, kAMn, kBMn, kTileM, (uint32_t)g.tile_n);
            const uint64_t da = tc_desc_base(kAMn ? 8192u : 16u), db = tc_desc_base(kBMn ? 8192u : 16u);
            uint32_t at = 0, unit = 0, phase = 0;
            int s = 0;
            bool ok = true;
            for (int t = first_tile; ok && t < tiles; t += step) {
                const HeadTile tile(t, tiles_m, tiles_n, g.group, splits, blocks);
                for (int k0 = tile.begin, k1; ok && k0 < tile.end; k0 = k1, unit++) {
                    const uint32_t acc = unit & 1u;
                    k1 = min(tile.end - k0, kPart) + k0;
                    ok = bar_wait(acc_empty + 8 * acc, ((unit >> 1) & 1u) ^ 1u, dead);
                    if (!ok) break;
                    tc_fence_after();
                    for (int kb = k0; kb < k1; kb++, at++) {
                        ok = bar_wait(full + 8 * s, phase, dead);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t b = ring + s * g.stage_bytes, a = b + g.a_at;
#pragma unroll
                        for (int k = 0; k < kGemmK / 16; k++)
                            tc_mma<PAIR>(tmem + acc * 256, tc_desc(da, a + k * (kAMn ? 2048 : 32)), tc_desc(db, b + k * (kBMn ? 2048 : 32)), idesc, kb > k0 || k > 0);
                        tc_commit<PAIR>(empty + 8 * s);
                        if (++s == g.stages) { s = 0; phase ^= 1u; }
                    }
                    if (ok) tc_commit<PAIR>(acc_full + 8 * acc);
                }
            }
            // what was issued ends before tensor memory is given back: the last commits arrive on `empty`
            const uint32_t n = (uint32_t)g.stages;
            for (uint32_t i = at < n ? 0 : at - n; i < at; i++)
                for (uint32_t j = 0; j < (1u << 20) && !bar_try(empty + 8 * (i % n), (i / n) & 1u); j++) {}
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int chunks = g.tile_n / 16, c_begin = half == 0 ? 0 : (chunks + 1) / 2, c_end = half == 0 ? (chunks + 1) / 2 : chunks;  // 8 at most
        const float unscale = MODE == kWeight ? g.info->unscale : 1.f, scale = MODE == kGrad ? g.info->scale : 1.f;
        const uint32_t free_bar = PAIR ? cluster_at(acc_empty, 0) : acc_empty;
        const uint32_t out = ring + kGemmRingBytes + (warp - 2) * kGemmOut;
        const float by_cap = CAP ? fminf(1.f / g.cap, 3.0e38f) : 0.f;  // a cap of almost nothing: 0 stays 0
        uint32_t unit = 0;
        bool ok = true;
        // kWeight: the rows whose target this thread's entry of a tile is: where they begin in g.order, and their number
        const bool rests = MODE == kWeight && g.first_of && g.info->low == 0;
        auto rests_of = [&](int t) {
            if (t >= tiles) return make_int2(0, 0);
            const int entry = HeadTile(t, tiles_m, tiles_n, g.group, splits, blocks).m * kTileM + (int)rank * kHeadTileM + quarter * 32 + lane;
            const int first = entry < g.m ? g.first_of[g.first + entry] : -1;
            return first < 0 ? make_int2(0, 0) : make_int2(first, g.count[first]);
        };
        int2 next_rests = rests ? rests_of(first_tile) : make_int2(0, 0);
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
            // adds an accumulator's columns to their sums so far, of which it is the first
            auto add_unit = [&](auto &z, uint32_t from, bool first, bool rows_here) {
#pragma unroll
                for (int c = 0; c < (int)(sizeof(z) / sizeof(z[0])); c++) {
                    if (c_begin + c >= c_end || !rows_here) break;
                    HeadCols x;
                    tmem_load16(from + (c_begin + c) * 16, x.v);
                    tmem_loaded();
#pragma unroll
                    for (int i = 0; i < 16; i++) z[c][i] = first ? x.f(i) : z[c][i] + x.f(i);
                }
                read_unit();
            };
            if constexpr (MODE == kStats) {
                const bool rows_here = m0 + quarter * 32 < used;  // of this warp
                const int target = r >= used ? -1 : g.targets ? g.targets[r] : g.rows[r].target;
                float z[8][16];
                for (int k0 = 0; k0 < blocks; k0 += kPart) {
                    const uint32_t from = full_unit();
                    if (!ok) break;
                    add_unit(z, from, k0 == 0, rows_here);
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
                        z[c][i] = !in ? -CUDART_INF_F : CAP ? head_cap(z[c][i], g.cap, by_cap).z : z[c][i];
                        most[i & 3] = fmaxf(most[i & 3], z[c][i]);
                    }
                    const unsigned at = (unsigned)(target - col);  // (a store that each element decides on: 1398 us in place of 1331 for 1000 x 2560 x 262,144)
                    if (at < 16u && c_begin + c < c_end && target >= 0) {
                        float hit = 0.f;
#pragma unroll
                        for (int i = 0; i < 16; i++) hit = at == (unsigned)i ? z[c][i] : hit;
                        g.hit[r] = hit;
                    }
                }
                top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
                // Relative to the largest logit itself: its own term is 1, so that no sum is below 1 and no loss below 0, at any size of
                // the logits (a product with log2(e) that is taken off afterwards has a rounding, 2^-24 of the logit).
                const float ref = top == -CUDART_INF_F ? 0.f : top;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 8; c++)
#pragma unroll
                    for (int i = 0; i < 16; i++) sum[i & 3] += exp2_fast((z[c][i] - ref) * kLog2e);
                if (r < used) g.parts[(int64_t)r * g.pieces + 2 * tn + half] = make_float2(top, (sum[0] + sum[1]) + (sum[2] + sum[3]));
            } else {
                // what 128 bytes of a row hold goes through shared memory and out as a box of the warp's 32 rows
                // (one row of tiles, whose widths are not whole boxes, has few gradients: each thread writes its own)
                const bool direct = MODE == kGrad && (!PAIR || g.tile_n != 256);
                constexpr int kOutCols = MODE == kHidden ? 32 : 64, kOutChunks = kOutCols / 16;
                const int slab = (used + kHeadTileM - 1) / kHeadTileM * kHeadTileM;  // rows of a split
                const int r0 = m0 + quarter * 32;
                const bool rows_here = r0 < (MODE == kWeight ? g.m : MODE == kHidden ? slab : g.rows_pad) && (some || MODE != kHidden || g.first == 0);
                HeadRow row = {};
                if (MODE == kGrad && rows_here) row = g.rows[r];
                // Beyond 64 rows the target's gradient, the largest of a row mostly, is left out of the products and added where their results are rounded, not
                // rounded itself: in an accumulator it makes the additions of all that follows it coarser, too (1000 x 512 x 131,072 in fp16, weights with a
                // mean of four deviations: 6.2e-4 off in place of 4.3e-4)
                const bool apart = MODE == kGrad && g.info->low == 0;
                row.a *= scale;
                row.b *= scale;
                int2 mine = make_int2(0, 0);
                uint32_t together = 0u;
                if (MODE == kWeight && rests) {  // read a tile ahead
                    mine = next_rests;
                    next_rests = rests_of(t + step);
                    together = rests_together(mine.y);
                }
                const bool any_rests = MODE == kWeight && __any_sync(0xFFFFFFFFu, mine.y > 0);
                // LONG: sums of all parts but the last; kWeight has as many columns as one box, kGrad's boxes are unrolled for them
                float z[MODE == kGrad ? 8 : kOutChunks][16];
                bool more = false;
                for (int k0 = 0; LONG && k0 + kPart < blocks; k0 += kPart) {
                    const uint32_t from = full_unit();
                    if (!ok) break;
                    add_unit(z, from, !more, rows_here);
                    more = true;
                }
                if (LONG && !ok) break;
                // kHidden: a sum's later parts are added to the first in memory, when that has got there
                const int rounds = MODE == kHidden && some ? (tile.end - tile.begin + kPart - 1) / kPart : 1;
                for (int round = 0; round < rounds; round++) {
                    const uint32_t from = some ? full_unit() : 0u;
                    if (!ok) break;
                    if (MODE == kHidden && round > 0 && lane == 0) store_done();
#pragma unroll LONG && MODE == kGrad ? 8 / kOutChunks : 1
                    for (int box = 0; box < 8 / kOutChunks; box++) {
                        const int c0 = c_begin + box * kOutChunks;
                        if (c0 >= c_end || !rows_here || n0 + c0 * 16 >= g.n) break;
                        // all of a box's columns on their way before the first is waited for, and the last box's shared memory waited for last
                        HeadCols x[kOutChunks];
#pragma unroll
                        for (int c = 0; c < kOutChunks; c++) {
                            if (some && c0 + c < c_end) {
                                tmem_load16(from + (c0 + c) * 16, x[c].v);
                            } else {
#pragma unroll
                                for (int i = 0; i < 16; i++) x[c].v[i] = 0u;
                            }
                        }
                        if (some) tmem_loaded();
                        if (LONG && more) {
#pragma unroll
                            for (int c = 0; c < kOutChunks; c++)
#pragma unroll
                                for (int i = 0; i < 16; i++) x[c].v[i] = __float_as_uint(z[MODE == kGrad ? box * kOutChunks + c : c][i] + x[c].f(i));
                        }
                        if (MODE == kWeight && any_rests) {  // the targets' gradients of the rows whose target this is
                            const int own = together >> lane & 1u ? 0 : mine.y;
                            for (int k = 0; k < own; k++) {
                                const int q = g.order[mine.x + k];
                                const float rest = g.hit[q];
                                const uint16_t *h = g.hidden + (int64_t)q * g.n + n0 + c0 * 16;
#pragma unroll
                                for (int c = 0; c < 2 * kOutChunks; c++) {
                                    if (n0 + c0 * 16 + 8 * c >= g.n) break;
                                    const uint4 e = ((const uint4 *)h)[c];
                                    const uint32_t w[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
                                    for (int i = 0; i < 8; i++)
                                        x[c / 2].v[8 * (c & 1) + i] = __float_as_uint(fmaf(rest, half_of<BF16>(w[i / 2] >> (16 * (i & 1))), x[c / 2].f(8 * (c & 1) + i)));
                                }
                            }
                            __syncwarp();
                            for (uint32_t left = together; left != 0u; left &= left - 1u) {  // by the warp: a lane has two columns
                                const int to = __ffs(left) - 1, begin = __shfl_sync(0xFFFFFFFFu, mine.x, to), n = __shfl_sync(0xFFFFFFFFu, mine.y, to), col = n0 + c0 * 16 + 2 * lane;
                                float2 sum = make_float2(0.f, 0.f);
                                for (int k0 = 0; k0 < n; k0 += 32) {  // a lane looks up a row
                                    const int q = k0 + lane < n ? g.order[begin + k0 + lane] : 0;
                                    const float rest = k0 + lane < n ? g.hit[q] : 0.f;
                                    const int here = min(32, n - k0);
#pragma unroll 8
                                    for (int k = 0; k < here; k++) {
                                        const int row = __shfl_sync(0xFFFFFFFFu, q, k);
                                        const float by = __shfl_sync(0xFFFFFFFFu, rest, k);
                                        const uint32_t e = col < g.n ? *(const uint32_t *)(g.hidden + (int64_t)row * g.n + col) : 0u;
                                        sum.x = fmaf(by, half_of<BF16>(e), sum.x);
                                        sum.y = fmaf(by, half_of<BF16>(e >> 16), sum.y);
                                    }
                                }
                                if (lane == 0) store_read();
                                __syncwarp();
                                shared_store2(out + lane * 8, __float_as_uint(sum.x), __float_as_uint(sum.y));
                                __syncwarp();
                                if (lane == to) {
#pragma unroll
                                    for (int i = 0; i < 16 * kOutChunks; i += 4) {
                                        const float4 v = shared_load(out + i * 4);
                                        uint32_t *at = x[i / 16].v + i % 16;
                                        at[0] = __float_as_uint(__uint_as_float(at[0]) + v.x);
                                        at[1] = __float_as_uint(__uint_as_float(at[1]) + v.y);
                                        at[2] = __float_as_uint(__uint_as_float(at[2]) + v.z);
                                        at[3] = __float_as_uint(__uint_as_float(at[3]) + v.w);
                                    }
                                }
                                __syncwarp();
                            }
                        }
                        uint32_t o[kOutChunks][MODE == kHidden ? 1 : 8];
#pragma unroll
                        for (int c = 0; c < kOutChunks; c++) {
                            const int col = n0 + (c0 + c) * 16;
                            if constexpr (MODE == kGrad) {
                                float d[16], slope[16];
#pragma unroll
                                for (int i = 0; i < 16; i++) {
                                    float logit = x[c].f(i);
                                    if (CAP) {
                                        const Capped capped = head_cap(logit, g.cap, by_cap);
                                        logit = capped.z;
                                        slope[i] = 1.f - capped.tanh * capped.tanh;
                                    }
                                    d[i] = row.a * exp2_fast((logit - row.norm) * kLog2e);
                                }
                                const unsigned at = (unsigned)(row.target - g.first - col);
                                if (at < 16u && c0 + c < c_end) {
                                    float hit = 0.f;
#pragma unroll
                                    for (int i = 0; i < 16; i++)
                                        if (at == (unsigned)i) {
                                            d[i] -= row.b;
                                            hit = CAP ? d[i] * slope[i] : d[i];
                                            if (apart) d[i] = 0.f;
                                        }
                                    if (apart && r < used) g.hit[r] = hit;
                                }
#pragma unroll
                                for (int i = 0; i < 16 && CAP; i++) d[i] *= slope[i];
                                if (row.low != 0) {
#pragma unroll
                                    for (int i = 0; i < 16; i++) d[i] -= BF16 ? __bfloat162float(__float2bfloat16_rn(d[i])) : __half2float(__float2half_rn(d[i]));
                                }
#pragma unroll
                                for (int i = 0; i < 8; i++) o[c][i] = r < used ? pack2<BF16>(d[2 * i], d[2 * i + 1]) : 0u;
                            } else if constexpr (MODE == kWeight) {
#pragma unroll
                                for (int i = 0; i < 8; i++) o[c][i] = pack2<BF16>(x[c].f(2 * i) * unscale, x[c].f(2 * i + 1) * unscale);
                            }
                        }
                        if (!direct) {
                            if (lane == 0) store_read();
                            __syncwarp();
                        }
#pragma unroll
                        for (int c = 0; c < kOutChunks; c++) {
                            const uint32_t to = out + lane * 128;  // its 16 bytes are exchanged as a 128-byte swizzle wants them
                            if constexpr (MODE == kHidden) {
#pragma unroll
                                for (int i = 0; i < 4; i++) shared_store(to + (((4 * c + i) ^ (lane & 7)) << 4), x[c].v[4 * i], x[c].v[4 * i + 1], x[c].v[4 * i + 2], x[c].v[4 * i + 3]);
                            } else if (direct) {
                                if (c0 + c < c_end) {
                                    uint4 *at = (uint4 *)((uint16_t *)g.out + (int64_t)r * g.out_stride + n0 + (c0 + c) * 16);
                                    at[0] = make_uint4(o[c][0], o[c][1], o[c][2], o[c][3]);
                                    at[1] = make_uint4(o[c][4], o[c][5], o[c][6], o[c][7]);
                                }
                            } else {
                                shared_store(to + (((2 * c) ^ (lane & 7)) << 4), o[c][0], o[c][1], o[c][2], o[c][3]);
                                shared_store(to + (((2 * c + 1) ^ (lane & 7)) << 4), o[c][4], o[c][5], o[c][6], o[c][7]);
                            }
                        }
                        if (direct) continue;
                        async_proxy_fence();
                        __syncwarp();
                        if (lane == 0) {
                            const int x = n0 + c0 * 16, y = (MODE == kWeight ? g.first : MODE == kHidden ? tile.split * slab : 0) + r0;
                            if (MODE == kHidden && (g.first > 0 || round > 0)) tma_store<true>(&map_out, x, y, out);
                            else tma_store<false>(&map_out, x, y, out);
                            store_commit();
                        }
                    }
                    if (some) read_unit();
                }
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
