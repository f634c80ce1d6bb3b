// stg_head_logits for more rows than the stream takes: weights go to tensor memory, hidden states to shared memory, and tcgen05.mma multiplies
// them, 128 vocabulary entries by up to 128 rows at a time.
//
// A CTA per SM takes items - up to eight tiles of 16 vocabulary entries, for a block of rows - and goes through their units of 128 columns.
// One warp copies four units of every tile at a time into a ring of stages, another the hidden states' columns of a unit into a second ring.  Teams of four warps turn codes into fp16
// numbers q - 8, exactly, each of them the units in turn, a thread one entry, and store them to tensor memory, a few buffers in turn.  One
// thread multiplies, each group of columns into an accumulator of its own (a ring of them), and more warps add them up, scaled by the
// entry's scale: a thread's numbers all have the same.  So the weight is not rounded, and scales meet fp32 sums.
//
// A unit of eight tiles is 32 KB of unpacked weight into tensor memory, and each of its groups 512 bytes of sums per row out of it, which by
// themselves measure as some 30 and 60 bytes a cycle.  64 rows x 4096 x 151,936 take 173 us with groups of 128, bound by the way in (26 bytes a cycle), and 282
// with groups of 32, by the way out.  256 rows take 410 (780 TFLOP/s; the library's bf16 product of that size would be 193 at its best rate), 22 bytes a
// cycle in and 43 out with two thirds of the issue slots taken: nothing is full.  509 with zero points, which move no more but double the adding
// warps' work and halve their number (TilesWarps); 704 with groups of 32.  Zero points with groups of 32 and more than 64 rows spill 96 bytes.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include "stg_head.h"
#include "stg_head4.cuh"
#include "stg_launch.h"
#include "stg_pdl.cuh"
#include "stg_tc.cuh"

namespace stg {

struct HeadTiles {
    HeadLogits p;
    uint16_t *states;       // [blocks * n, padded width] fp16, zeros where there are no rows
    float2 *unscale;        // [blocks * n]: the inverse of what a row was multiplied with, in two factors
    float *sums;            // [blocks][groups of the padded width][n]: sums of groups, for zero points
    int n, blocks, per_item, items_v, code_stages, state_stages, slots;  // TilesShape
    bool scale_bf16;
};

// Hidden states as fp16: bf16 ones times a power of two that takes a row's largest finite one to [2^14, 2^15).  That is exact down to 2^-29 of
// it, and 2^-40 of it off below.
template <bool ZEROS>
__global__ void __launch_bounds__(256) k_head_states(const __grid_constant__ HeadTiles a)
{
    __shared__ uint32_t most;
    const HeadLogits &p = a.p;
    const int row = blockIdx.x, per = p.w.units_per_tile * (kUnitCols / 8);  // a multiple of 16
    pdl_release();
    pdl_wait();
    if (threadIdx.x == 0) most = 0u;
    __syncthreads();
    const uint16_t *from = p.hidden + (int64_t)row * p.hidden_stride;
    const bool there = row < p.rows;
    if (p.hidden_bf16 && there) {
        uint32_t m = 0u;
        for (int i = threadIdx.x; i < per; i += 256) {
            if (8 * i >= p.w.width) break;
            const uint4 v = eight_states(from + 8 * i, p.vec);
            const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t lo = e[j] & 0x7FFFu, hi = e[j] >> 16 & 0x7FFFu;
                m = max(m, max(lo < 0x7F80u ? lo : 0u, hi < 0x7F80u ? hi : 0u));
            }
        }
        m = __reduce_max_sync(0xFFFFFFFFu, m);
        if ((threadIdx.x & 31) == 0) atomicMax(&most, m);
    }
    __syncthreads();
    const float top = __uint_as_float(most << 16);
    const int e = top > 0.f ? 14 - ilogbf(top) : 0, half = e / 2;
    const float s1 = __uint_as_float((uint32_t)(127 + half) << 23), s2 = __uint_as_float((uint32_t)(127 + e - half) << 23);
    if (threadIdx.x == 0) a.unscale[row] = make_float2(__uint_as_float((uint32_t)(127 - half) << 23), __uint_as_float((uint32_t)(127 - (e - half)) << 23));
    const int lanes = p.w.group / 8;  // that have a group
    for (int i = threadIdx.x; i < per; i += 256) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (there && 8 * i < p.w.width) v = eight_states(from + 8 * i, p.vec);
        uint32_t x[4] = {v.x, v.y, v.z, v.w};
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (p.hidden_bf16)
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(x[j]) : "f"(half_at<true>((uint16_t)(x[j] >> 16)) * s1 * s2), "f"(half_at<true>((uint16_t)x[j]) * s1 * s2));
            s += half_at<false>((uint16_t)x[j]) + half_at<false>((uint16_t)(x[j] >> 16));
        }
        ((uint4 *)(a.states + (int64_t)row * per * 8))[i] = make_uint4(x[0], x[1], x[2], x[3]);
        if (ZEROS) {  // half warps are here as a whole
            for (int o = 1; o < lanes; o *= 2) s += __shfl_xor_sync(0xFFFFu << (threadIdx.x & 16), s, o);
            if ((i & (lanes - 1)) == 0) a.sums[((int64_t)(row / a.n) * (per / lanes) + i / lanes) * a.n + row % a.n] = s;
        }
    }
}

// Two warps load, one multiplies; teams of four unpack, and sets of four add up, each some of the columns.  Every warp's waits and
// arrivals cost it about a hundred instructions a unit, so few warps with many columns each take less time than many with few: 128 rows have
// one team, whose registers the sums then get, and two sets - but where a unit is one group without zero points, which leaves the adding
// warps less to do than the unpacking ones, two teams and four sets (4096 x 151,936, 256 rows: 410 us in place of 439; with zero points
// 689 in place of 487, with groups of 64 526 in place of 511).
template <bool ZEROS, int G, int C>
struct TilesWarps {
    static constexpr bool kMany = C == 8 && G == 1 && !ZEROS;
    static constexpr int kTeams = C == 8 && !kMany ? 1 : 2, kSets = kMany ? 4 : 2, kUnpack = 3, kAdd = 3 + 4 * kTeams;
    static constexpr int kThreads = 32 * (3 + 4 * kTeams + 4 * kSets);
};

// a b + c, two at a time.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("{\n.reg .b64 x, y, z, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 w, x, y, z;\nmov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// G groups to a unit; 16 C rows to a block.
template <bool ZEROS, int G, int C>
__global__ void __launch_bounds__(TilesWarps<ZEROS, G, C>::kThreads, 1) k_head_tiles(const __grid_constant__ CUtensorMap states, const __grid_constant__ HeadTiles a)
{
    using Warps = TilesWarps<ZEROS, G, C>;
    constexpr int N = 16 * C, kTeams = Warps::kTeams, kSets = Warps::kSets, kThreads = Warps::kThreads, kCols = N / kSets;
    constexpr int kBuffers = tiles_buffers(N);
    constexpr uint32_t kUnpacked = 512 - 64 * kBuffers, kStateBytes = 2 * N * 128;
    extern __shared__ unsigned char raw[];
    __shared__ alignas(8) uint64_t bars[4 * kTilesStages + 2 * kBuffers + 2 * kTilesSlots];
    __shared__ uint32_t tmem_slot;
    __shared__ int dead_;
    volatile int *dead = &dead_;
    const Head4 &w = a.p.w;
    // the rings: hidden states, then codes, in each stage with the groups' sums ahead
    unsigned char *const states_p = raw + ((1024u - (smem_at(raw) & 1023u)) & 1023u), *const codes_p = states_p + a.state_stages * kStateBytes;
    const uint32_t code_stage = (uint32_t)tiles_code_stage(w.unit_bytes, w.groups_per_unit, N), tile_stage = kTilesChunk * (uint32_t)w.unit_bytes;
    constexpr uint32_t kSumBytes = ZEROS ? G * N * 4 : 0, kCodesAt = kTilesChunk * kSumBytes;
    const uint32_t c_full = smem_at(bars), c_empty = c_full + 8 * kTilesStages, s_full = c_empty + 8 * kTilesStages, s_empty = s_full + 8 * kTilesStages,
                   a_full = s_empty + 8 * kTilesStages, a_empty = a_full + 8 * kBuffers, d_full = a_empty + 8 * kBuffers, d_empty = d_full + 8 * kTilesSlots;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 0 && one_lane()) {
        tma_prefetch(&states);
        for (int i = 0; i < a.code_stages; i++) { bar_init(c_full + 8 * i, 1); bar_init(c_empty + 8 * i, kTilesChunk * (4 + 4 * kSets)); }
        for (int i = 0; i < a.state_stages; i++) { bar_init(s_full + 8 * i, 1); bar_init(s_empty + 8 * i, 1); }
        for (int i = 0; i < kBuffers; i++) { bar_init(a_full + 8 * i, 4); bar_init(a_empty + 8 * i, 1); }
        for (int i = 0; i < a.slots; i++) { bar_init(d_full + 8 * i, 1); bar_init(d_empty + 8 * i, 4 * kSets); }
        dead_ = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 1) tmem_alloc<false>(smem_at(&tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_release();
    pdl_wait();
    async_fence();  // what the kernels ahead have written - hidden states, groups' sums, the packed weight - is read by bulk copies
    const int items = a.items_v * a.blocks, per = w.units_per_tile;

    if (warp == 0) {  // hidden states
        if (one_lane()) {
            int s = 0;
            uint32_t phase = 1, loaded = 0;
            bool ok = true;
            for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
                for (int u = 0; u < per; u++) {
                    ok = bar_wait(s_empty + 8 * s, phase, dead);
                    if (!ok) break;
                    bar_expect(s_full + 8 * s, kStateBytes);
                    tma_load3(smem_at(states_p) + s * kStateBytes, &states, 0, item % a.blocks * N, 2 * u, s_full + 8 * s);
                    loaded++;
                    if (++s == a.state_stages) { s = 0; phase ^= 1u; }
                }
            }
            // copies in flight end before the CTA does
            for (uint32_t i = loaded < (uint32_t)a.state_stages ? 0 : loaded - a.state_stages; i < loaded; i++)
                for (uint32_t j = 0; j < (1u << 20) && !bar_try(s_full + 8 * (i % a.state_stages), (i / a.state_stages) & 1u); j++) {}
        }
    } else if (warp == 2) {  // codes, scales, zero points and groups' sums
        int s = 0;
        uint32_t phase = 1, loaded = 0;
        bool ok = true;
        for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
            const int t0 = item / a.blocks * a.per_item, tiles = min(a.per_item, w.tiles - t0);
            const unsigned char *from = w.units + (int64_t)(t0 + lane) * per * w.unit_bytes;
            const float *sums = a.sums + (int64_t)(item % a.blocks) * per * G * N;
            for (int u = 0; u < per; u += kTilesChunk) {
                const uint32_t n = (uint32_t)min(kTilesChunk, per - u), bar = c_full + 8 * s;
                ok = __all_sync(0xFFFFFFFFu, bar_wait(c_empty + 8 * s, phase, dead));
                if (!ok) break;
                const uint32_t to = smem_at(codes_p) + s * code_stage;
                if (lane == 0) bar_expect(bar, n * (uint32_t)(tiles * w.unit_bytes + kSumBytes));
                __syncwarp();
                if (lane < tiles) bulk_load(to + kCodesAt + lane * tile_stage, from + (int64_t)u * w.unit_bytes, n * (uint32_t)w.unit_bytes, bar);
                if (ZEROS && lane == 31) bulk_load(to, sums + (int64_t)u * G * N, n * kSumBytes, bar);
                loaded++;
                if (++s == a.code_stages) { s = 0; phase ^= 1u; }
            }
        }
        if (lane == 0)
            for (uint32_t i = loaded < (uint32_t)a.code_stages ? 0 : loaded - a.code_stages; i < loaded; i++)
                for (uint32_t j = 0; j < (1u << 20) && !bar_try(c_full + 8 * (i % a.code_stages), (i / a.code_stages) & 1u); j++) {}
    } else if (warp == 1) {
        if (one_lane()) {
            const uint32_t idesc = tc_idesc(false, false, false, 128, N);
            const uint64_t db = tc_desc_base(16);
            int s = 0, slot = 0;
            uint32_t phase = 0, slot_phase = 1, at = 0;
            bool ok = true;
            for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
                for (int u = 0; ok && u < per; u++, at++) {
                    const uint32_t buf = at % kBuffers;
                    ok = bar_wait(s_full + 8 * s, phase, dead) && bar_wait(a_full + 8 * buf, (at / kBuffers) & 1u, dead);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t b = smem_at(states_p) + s * kStateBytes;
#pragma unroll
                    for (int gr = 0; gr < G; gr++) {
                        ok = bar_wait(d_empty + 8 * slot, slot_phase, dead);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int k = gr * (8 / G); k < (gr + 1) * (8 / G); k++)
                            tc_mma_from_tmem(tmem + slot * N, tmem + kUnpacked + buf * 64 + k * 8, tc_desc(db, b + (k / 4) * (N * 128) + (k % 4) * 32), idesc, k > gr * (8 / G));
                        tc_commit<false>(d_full + 8 * slot);
                        if (++slot == a.slots) { slot = 0; slot_phase ^= 1u; }
                    }
                    if (!ok) break;
                    tc_commit<false>(a_empty + 8 * buf);
                    tc_commit<false>(s_empty + 8 * s);
                    if (++s == a.state_stages) { s = 0; phase ^= 1u; }
                }
            }
            // what was issued ends before tensor memory is given back: the last units' commits arrive on a_empty
            for (uint32_t i = at < kBuffers ? 0 : at - kBuffers; i < at; i++)
                for (uint32_t j = 0; j < (1u << 20) && !bar_try(a_empty + 8 * (i % kBuffers), (i / kBuffers) & 1u); j++) {}
        }
    } else if (warp < Warps::kAdd) {
        const int quarter = warp & 3, team = (warp - Warps::kUnpack) >> 2, m = quarter * 32 + lane, g = lane & 7;
        const uint32_t to_lanes = tmem + kUnpacked + ((uint32_t)(quarter * 32) << 16);
        const bool upper = (lane & 8) != 0;
        const uint32_t mask = upper ? 0x00F000F0u : 0x000F000Fu, base = upper ? 0x64806480u : 0x64086408u, by = upper ? 0x2C002C00u : 0x3C003C00u,
                       less = upper ? 0xD480D480u : 0xE408E408u;  // 1/16 and -72, or 1 and -1032
        const unsigned char *codes = codes_p + kCodesAt + (m >> 4) * tile_stage + g * 64;
        int s = 0;
        uint32_t phase = 0, at = 0;
        bool ok = true;
        for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
            for (int u = 0; ok && u < per; u++, at++) {
                const int in = u % kTilesChunk;
                const bool last = in + 1 == kTilesChunk || u + 1 == per;
                if (at % kTeams == (uint32_t)team) {
                    const uint32_t buf = at % kBuffers;
                    ok = __all_sync(0xFFFFFFFFu, bar_wait(c_full + 8 * s, phase, dead));
                    if (!ok) break;
                    const unsigned char *unit = codes + s * code_stage + in * w.unit_bytes;
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        uint32_t x[32];
#pragma unroll
                        for (int t = 0; t < 4; t++) {
                            const uint4 q = *(const uint4 *)(unit + half * 512 + ((t ^ (g >> 1)) * 16));
                            const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const int to = 16 * (k / 2) + 4 * t + 2 * (k % 2);
                                asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(x[to]) : "r"(bits_of(word[k], mask, base)), "r"(by), "r"(less));
                                asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(x[to + 1]) : "r"(bits_of(word[k] >> 8, mask, base)), "r"(by), "r"(less));
                            }
                        }
                        if (half == 0) {
                            ok = __all_sync(0xFFFFFFFFu, bar_wait(a_empty + 8 * buf, ((at / kBuffers) & 1u) ^ 1u, dead));
                            if (!ok) break;
                            tc_fence_after();
                        }
                        tmem_store32(to_lanes + buf * 64 + half * 32, x);
                    }
                    if (!ok) break;
                    tmem_stored();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        bar_arrive(a_full + 8 * buf);
                        bar_arrive_times(c_empty + 8 * s, last ? kTilesChunk - in : 1);  // a shorter stage's last unit counts for the missing ones
                    }
                }
                if (last && ++s == a.code_stages) { s = 0; phase ^= 1u; }
            }
        }
    } else {
        const int quarter = warp & 3, set = (warp - Warps::kAdd) >> 2, m = quarter * 32 + lane, g = lane & 7;
        const uint32_t from_lanes = tmem + ((uint32_t)(quarter * 32) << 16) + set * kCols;
        const unsigned char *words = codes_p + kCodesAt + (m >> 4) * tile_stage + kUnitCodes + g * G * 4 + ((lane & 8) ? 2 : 0);
        const float *sums_at = (const float *)codes_p + set * kCols;
        float2 acc[kCols / 2];
#pragma unroll
        for (int i = 0; i < kCols / 2; i++) acc[i] = make_float2(0.f, 0.f);
        int s = 0, slot = 0;
        uint32_t phase = 0, slot_phase = 0;
        bool ok = true;
        for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
            for (int u = 0; u < per; u++) {
                const int in = u % kTilesChunk;
                const bool last = in + 1 == kTilesChunk || u + 1 == per;
                ok = __all_sync(0xFFFFFFFFu, bar_wait(c_full + 8 * s, phase, dead));
                if (!ok) break;
                float scale[G], zero[G];
#pragma unroll
                for (int gr = 0; gr < G; gr++) {
                    const unsigned char *word = words + s * code_stage + in * w.unit_bytes + gr * 4;
                    const uint16_t sw = *(const uint16_t *)word;
                    scale[gr] = a.scale_bf16 ? half_at<true>(sw) : half_at<false>(sw);
                    if (ZEROS) {
                        const uint16_t zw = *(const uint16_t *)(word + 32 * G);
                        zero[gr] = 8.f - (a.scale_bf16 ? half_at<true>(zw) : half_at<false>(zw));
                    }
                }
                const float *sums = (const float *)((const unsigned char *)sums_at + s * code_stage + in * kSumBytes);
#pragma unroll
                for (int gr = 0; gr < G; gr++) {
                    ok = __all_sync(0xFFFFFFFFu, bar_wait(d_full + 8 * slot, slot_phase, dead));
                    if (!ok) break;
                    tc_fence_after();
                    constexpr int kLoad = kCols < 32 ? kCols : 32;
#pragma unroll
                    for (int c = 0; c < kCols; c += kLoad) {
                        uint32_t x[kLoad];
                        if constexpr (kLoad == 8) {
                            tmem_load8(from_lanes + slot * N, x);
                        } else {
#pragma unroll
                            for (int i = 0; i < kLoad; i += 16) tmem_load16(from_lanes + slot * N + c + i, *(uint32_t(*)[16])(x + i));
                        }
                        tmem_loaded();
                        if (c + kLoad == kCols) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) bar_arrive(d_empty + 8 * slot);
                            if (++slot == a.slots) { slot = 0; slot_phase ^= 1u; }
                        }
#pragma unroll
                        for (int i = 0; i < kLoad; i += 4) {
                            float2 v = make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), y = make_float2(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
                            if (ZEROS) {
                                const float4 u = *(const float4 *)(sums + gr * N + c + i);
                                v = fma2(make_float2(zero[gr], zero[gr]), make_float2(u.x, u.y), v);
                                y = fma2(make_float2(zero[gr], zero[gr]), make_float2(u.z, u.w), y);
                            }
                            acc[(c + i) / 2] = fma2(make_float2(scale[gr], scale[gr]), v, acc[(c + i) / 2]);
                            acc[(c + i) / 2 + 1] = fma2(make_float2(scale[gr], scale[gr]), y, acc[(c + i) / 2 + 1]);
                        }
                    }
                }
                if (!ok) break;
                __syncwarp();
                if (lane == 0) bar_arrive_times(c_empty + 8 * s, last ? kTilesChunk - in : 1);
                if (last && ++s == a.code_stages) { s = 0; phase ^= 1u; }
            }
            if (!ok) break;
            const int t0 = item / a.blocks * a.per_item, tiles = min(a.per_item, w.tiles - t0), r0 = item % a.blocks * N + set * kCols;
            const int64_t v = (int64_t)t0 * kHeadRows4 + m;
            const bool mine = m < tiles * kHeadRows4 && v < w.vocab;
#pragma unroll
            for (int i = 0; i < kCols; i++) {
                const int r = r0 + i;
                if (mine && r < a.p.rows) {
                    const float2 un = a.unscale[r];
                    const float x = ((i & 1) ? acc[i / 2].y : acc[i / 2].x) * un.x * un.y;
                    if (a.p.out_bf16) ((__nv_bfloat16 *)a.p.out)[r * a.p.out_stride + v] = __float2bfloat16_rn(x);
                    else ((float *)a.p.out)[r * a.p.out_stride + v] = x;
                }
            }
#pragma unroll
            for (int i = 0; i < kCols / 2; i++) acc[i] = make_float2(0.f, 0.f);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_free<false>(tmem, 512);
    if (dead_ != 0) {  // a wait has given up: the CTA's logits are NaN
        for (int item = blockIdx.x; item < items; item += gridDim.x) {
            const int64_t v0 = (int64_t)(item / a.blocks) * a.per_item * kHeadRows4, v1 = min((int64_t)w.vocab, v0 + a.per_item * kHeadRows4);
            const int r0 = item % a.blocks * N, r1 = min(a.p.rows, r0 + N);
            for (int64_t i = threadIdx.x; i < (v1 - v0) * (r1 - r0); i += kThreads) {
                const int64_t to = (r0 + i / (v1 - v0)) * a.p.out_stride + v0 + i % (v1 - v0);
                if (a.p.out_bf16) ((uint16_t *)a.p.out)[to] = 0x7FFFu;
                else ((float *)a.p.out)[to] = CUDART_NAN_F;
            }
        }
    }
}

// ---- host ----

static HeadTiles tiles_args(StgHandle h, const Head4 &w, int rows)
{
    const TilesShape s = tiles_shape(w, rows, h->sm_count, h->smem_optin);
    HeadTiles a;
    memset(&a, 0, sizeof(a));
    a.n = s.n; a.blocks = s.blocks; a.per_item = s.per_item; a.items_v = s.items_v;
    a.code_stages = s.code_stages; a.state_stages = s.state_stages; a.slots = s.slots;
    return a;
}

static size_t tiles_layout(const Head4 &w, HeadTiles &a, char *base)
{
    size_t at = 0;
    auto take = [&](size_t bytes) { char *x = base ? base + at : nullptr; at += round_up(bytes, 256); return x; };
    const size_t rows = (size_t)a.blocks * a.n, units = (size_t)w.units_per_tile;
    a.states = (uint16_t *)take(rows * units * kUnitCols * 2);
    a.unscale = (float2 *)take(rows * sizeof(float2));
    a.sums = (float *)take(rows * units * w.groups_per_unit * 4);
    return at;
}

size_t head_tiles_workspace(StgHandle h, const Head4 &w, int rows)
{
    HeadTiles a = tiles_args(h, w, rows);
    return tiles_layout(w, a, nullptr);
}

template <bool ZEROS, int G>
static cudaError_t launch_tiles(const HeadTiles &a, const CUtensorMap &states, int sms, cudaStream_t stream)
{
    void (*fn)(CUtensorMap, HeadTiles) = a.n == 16 ? k_head_tiles<ZEROS, G, 1> : a.n == 32 ? k_head_tiles<ZEROS, G, 2> : a.n == 64 ? k_head_tiles<ZEROS, G, 4> : k_head_tiles<ZEROS, G, 8>;
    const int threads = a.n == 128 ? TilesWarps<ZEROS, G, 8>::kThreads : TilesWarps<ZEROS, G, 1>::kThreads;
    const size_t smem = 1024 + a.code_stages * tiles_code_stage(a.p.w.unit_bytes, a.p.w.groups_per_unit, a.n) + (size_t)a.state_stages * 2 * a.n * 128;
    const cudaError_t e = ensure_dynamic_smem((const void *)fn, smem);
    return e != cudaSuccess ? e : launch_behind(fn, dim3((unsigned)std::min(sms, a.items_v * a.blocks)), threads, smem, stream, states, a);
}

int head_tiles(StgHandle h, const HeadLogits &p, bool scale_bf16, void *workspace, cudaStream_t stream)
{
    HeadTiles a = tiles_args(h, p.w, p.rows);
    tiles_layout(p.w, a, (char *)workspace);
    a.p = p;
    a.scale_bf16 = scale_bf16;
    const bool zeros = p.w.unit_bytes != kUnitCodes + 32 * p.w.groups_per_unit;
    const int64_t width = (int64_t)p.w.units_per_tile * kUnitCols;
    // 128 columns of a block's rows as two boxes of 64
    CUtensorMap states;
    const cuuint64_t s_size[3] = {64, (cuuint64_t)a.blocks * a.n, (cuuint64_t)width / 64}, s_stride[2] = {(cuuint64_t)width * 2, 128};
    const cuuint32_t s_box[3] = {64, (cuuint32_t)a.n, 2};
    const int rc = head_map_of(h, &states, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, a.states, s_size, s_stride, s_box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    CK(launch_behind(zeros ? k_head_states<true> : k_head_states<false>, dim3((unsigned)(a.blocks * a.n)), 256, 0, stream, a));
    using Launch = cudaError_t (*)(const HeadTiles &, const CUtensorMap &, int, cudaStream_t);
    static const Launch launch[2][3] = {{launch_tiles<false, 1>, launch_tiles<false, 2>, launch_tiles<false, 4>}, {launch_tiles<true, 1>, launch_tiles<true, 2>, launch_tiles<true, 4>}};
    CK(launch[zeros][p.w.groups_per_unit == 1 ? 0 : p.w.groups_per_unit == 2 ? 1 : 2](a, states, h->sm_count, stream));
    h->stats.kernel_launches += 2;
    return STG_OK;
}

}  // namespace stg
