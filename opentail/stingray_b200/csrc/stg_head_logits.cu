// stg_head_pack, stg_head_logits: a decode step's logits from a weight in 4 bits with a scale, and a zero point, per group of columns.
//
// logit[r][v] = sum over groups g of  scale[v][g] * (sum of (q - 8) h  -  (zero[v][g] - 8) * sum of h)  over the group's columns.
// q - 8 is exact in the hidden states' 16 bits and its products with them are exact in fp32, so a group's sum comes from the
// tensor cores without a rounding of the weight, and scales are applied to fp32 sums.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <new>

#include "stg_beam.h"
#include "stg_head.h"
#include "stg_launch.h"
#include "stg_pdl.cuh"
#include "stg_tc.cuh"

namespace stg {

// The packed weight: units of 16 vocabulary entries by 128 columns, a tile's units (16 entries, all columns, zeros behind the last)
// next to each other.  A unit: twice 512 bytes of codes, of which a lane of a warp holds 16 - what it needs of 64 columns in four
// steps of mma.m16n8k16 (word s: step s); the columns of a step are chosen such that a lane's share of a hidden state are eight
// neighbours for two steps: step s, columns 32 (s / 2) + 8 t + 4 (s % 2) + 0..3 for t = lane % 4.  Then the scales, and in the same way
// the zero points: for entry g = 0..7 the unit's groups, for each of them entries g and g + 8.
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

struct HeadPack {
    Head4 w;
    const uint8_t *codes;
    int64_t codes_stride;
    const uint16_t *scales, *zeros;
    unsigned char *out;
};

// One warp per unit.
__global__ void __launch_bounds__(256) k_head_pack(const __grid_constant__ HeadPack p)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const Head4 &w = p.w;
    const int64_t units = (int64_t)w.tiles * w.units_per_tile;
    pdl_release();
    pdl_wait();
    for (int64_t unit = blockIdx.x * 8ll + (threadIdx.x >> 5); unit < units; unit += gridDim.x * 8ll) {
        const int64_t v0 = unit / w.units_per_tile * kHeadRows4;
        const int k0 = (int)(unit % w.units_per_tile) * kUnitCols;
        unsigned char *out = p.out + unit * w.unit_bytes;
        auto code = [&](int row, int col) -> uint32_t {  // col is even: two codes of a byte; 8 where there is no weight
            return v0 + row < w.vocab && col < w.width ? p.codes[(v0 + row) * p.codes_stride + col / 2] : 0x88u;
        };
#pragma unroll
        for (int block = 0; block < 2; block++) {
            uint32_t word[4];
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const int col = k0 + block * 64 + 32 * (s / 2) + 8 * t + 4 * (s % 2);
                const uint32_t a = code(g, col), b = code(g + 8, col), c = code(g, col + 2), d = code(g + 8, col + 2);
                word[s] = (a & 15u) | (b & 15u) << 4 | (c & 15u) << 8 | (d & 15u) << 12 | (a >> 4) << 16 | (b >> 4) << 20 | (c >> 4) << 24 | (d >> 4) << 28;
            }
            ((uint4 *)(out + block * 512))[lane] = make_uint4(word[0], word[1], word[2], word[3]);
        }
        const int n = 16 * w.groups_per_unit, groups = w.width / w.group;
        for (int i = lane; i < n; i += 32) {
            const int64_t v = v0 + i / (2 * w.groups_per_unit) + 8 * (i & 1);
            const int group = k0 / w.group + i / 2 % w.groups_per_unit;
            const bool on = v < w.vocab && group < groups;  // else scale 0
            ((uint16_t *)(out + kUnitCodes))[i] = on ? p.scales[v * groups + group] : 0;
            if (p.zeros) ((uint16_t *)(out + kUnitCodes))[n + i] = on ? p.zeros[v * groups + group] : 0;
        }
    }
}

struct HeadLogits {
    Head4 w;
    const uint16_t *hidden;
    int64_t hidden_stride;
    bool vec;
    int rows;
    void *out;
    int64_t out_stride;
    bool out_bf16;
};

template <bool BF16>
__device__ __forceinline__ float half_at(uint16_t x)
{
    return BF16 ? __uint_as_float((uint32_t)x << 16) : __half2float(__ushort_as_half(x));
}

// Eight codes of a word as the four registers of an A fragment, q - 8 each.  A code is put below the bits of a number
// whose last bits count in ones (fp16: 1024, or 1024 with the code times 16; bf16: 128), and that number is taken off; both are exact.
template <bool BF16>
__device__ __forceinline__ void codes_to_a(uint32_t w, uint32_t (&a)[4])
{
    if (BF16) {
        const uint32_t one = 0x3F803F80u, less = 0xC308C308u;  // 1, -136
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t v = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
            asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(a[i]) : "r"(v), "r"(one), "r"(less));
        }
    } else {
        const uint32_t sixteenth = 0x2C002C00u, low = 0xE408E408u, high = 0xD480D480u;  // 1/16, -1032, -72
        const uint32_t u = w >> 8;
        const uint32_t v0 = (w & 0x000F000Fu) | 0x64006400u, v1 = (w & 0x00F000F0u) | 0x64006400u;
        const uint32_t v2 = (u & 0x000F000Fu) | 0x64006400u, v3 = (u & 0x00F000F0u) | 0x64006400u;
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(a[0]) : "r"(v0), "r"(low));
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(a[1]) : "r"(v1), "r"(sixteenth), "r"(high));
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(a[2]) : "r"(v2), "r"(low));
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(a[3]) : "r"(v3), "r"(sixteenth), "r"(high));
    }
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

// A unit's part of 16 logits for 8 NT rows of hidden states.  x: this lane's share of the first row group's row lane / 4 at the unit's first
// column; sums: of the unit's first group, per group 8 NT of them.
template <bool BF16, bool SBF16, bool ZEROS, int G, int NT>
__device__ __forceinline__ void unit_logits(float (&acc)[NT][4], const unsigned char *unit, const unsigned char *x, int pitch, const float *sums)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint4 q[2] = {((const uint4 *)unit)[lane], ((const uint4 *)(unit + 512))[lane]};
    const uint32_t word[8] = {q[0].x, q[0].y, q[0].z, q[0].w, q[1].x, q[1].y, q[1].z, q[1].w};
    uint32_t scale[G], zero[G];
    auto words = [&](uint32_t (&to)[G], const unsigned char *from) {
        if constexpr (G == 4) { const uint4 v = ((const uint4 *)from)[g]; to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w; }
        else if constexpr (G == 2) { const uint2 v = ((const uint2 *)from)[g]; to[0] = v.x; to[1] = v.y; }
        else to[0] = ((const uint32_t *)from)[g];
    };
    words(scale, unit + kUnitCodes);
    if (ZEROS) words(zero, unit + kUnitCodes + 32 * G);
#pragma unroll
    for (int gr = 0; gr < G; gr++) {
        float part[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) part[n][i] = 0.f;
#pragma unroll
        for (int h = gr * (4 / G); h < (gr + 1) * (4 / G); h++) {  // 32 columns each
            uint32_t a0[4], a1[4];
            codes_to_a<BF16>(word[2 * h], a0);
            codes_to_a<BF16>(word[2 * h + 1], a1);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint4 v = *(const uint4 *)(x + n * 8 * pitch + h * 64);
                mma16816<BF16>(part[n], a0, v.x, v.y);
                mma16816<BF16>(part[n], a1, v.z, v.w);
            }
        }
        const float s0 = half_at<SBF16>((uint16_t)scale[gr]), s1 = half_at<SBF16>((uint16_t)(scale[gr] >> 16));
#pragma unroll
        for (int n = 0; n < NT; n++) {
            if (ZEROS) {
                const float z0 = 8.f - half_at<SBF16>((uint16_t)zero[gr]), z1 = 8.f - half_at<SBF16>((uint16_t)(zero[gr] >> 16));
                const float2 u = *(const float2 *)(sums + gr * 8 * NT + n * 8 + 2 * t);
                part[n][0] = fmaf(z0, u.x, part[n][0]);
                part[n][1] = fmaf(z0, u.y, part[n][1]);
                part[n][2] = fmaf(z1, u.x, part[n][2]);
                part[n][3] = fmaf(z1, u.y, part[n][3]);
            }
            acc[n][0] = fmaf(s0, part[n][0], acc[n][0]);
            acc[n][1] = fmaf(s0, part[n][1], acc[n][1]);
            acc[n][2] = fmaf(s1, part[n][2], acc[n][2]);
            acc[n][3] = fmaf(s1, part[n][3], acc[n][3]);
        }
    }
}

template <int NT>
__device__ __forceinline__ void write_logits(const HeadLogits &p, const float (&acc)[NT][4], int64_t tile, int r0)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t v = tile * kHeadRows4 + g + (i >= 2 ? 8 : 0);
            const int r = r0 + n * 8 + 2 * t + (i & 1);
            if (v >= p.w.vocab || r >= p.rows) continue;
            if (p.out_bf16) ((__nv_bfloat16 *)p.out)[r * p.out_stride + v] = __float2bfloat16_rn(acc[n][i]);
            else ((float *)p.out)[r * p.out_stride + v] = acc[n][i];
        }
}

// Hidden states of rows [r0, r0 + 8 NT) and columns [k0, k0 + cols) into shared memory, zeros where there are none; `cols` whole units.
// The sums of their groups too, for zero points.
template <bool BF16, bool ZEROS, int G, int NT>
__device__ __forceinline__ void stage_states(const HeadLogits &p, int r0, int k0, int cols, unsigned char *xs, int pitch, float *sums)
{
    for (int i = threadIdx.x; i < 8 * NT * (cols / 8); i += blockDim.x) {
        const int n = i / (cols / 8), k = (i - n * (cols / 8)) * 8;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (r0 + n < p.rows && k0 + k < p.w.width) v = eight_states(p.hidden + (int64_t)(r0 + n) * p.hidden_stride + k0 + k, p.vec);
        *(uint4 *)(xs + n * pitch + k * 2) = v;
    }
    if (ZEROS) {
        __syncthreads();
        constexpr int kGroup = kUnitCols / G;
        for (int i = threadIdx.x; i < cols / kGroup * 8 * NT; i += blockDim.x) {
            const int n = i % (8 * NT), gr = i / (8 * NT);
            float s = 0.f;
            for (int k = 0; k < kGroup; k += 8) {
                const uint4 v = *(const uint4 *)(xs + n * pitch + (gr * kGroup + k) * 2);
                const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; j++) s += half_at<BF16>((uint16_t)e[j]) + half_at<BF16>((uint16_t)(e[j] >> 16));
            }
            sums[i] = s;
        }
    }
    __syncthreads();
}

// Up to 16 rows: the weight streams through, once.  Hidden states lie in shared memory whole.  A CTA per SM has a run of tiles, whose
// units its 16 warps share out evenly, each a run of neighbours that it copies into a ring of its own (bulk copies, one per stage), so no
// warp waits for another before the end.  A tile that several warps have units of is added up there, by the warp that has its first.
constexpr int kStreamWarps = 16, kStreamStages = 2;

struct StreamShape {
    int pitch;          // bytes between rows of hidden states
    int chunk;          // units of a stage
    size_t sums, slots, ring, bars, smem;  // offsets, and bytes in all
};

template <bool BF16, bool SBF16, bool ZEROS, int G, int NT>
__global__ void __launch_bounds__(kStreamWarps * 32, 1) k_head_stream(const __grid_constant__ HeadLogits p, const __grid_constant__ StreamShape s)
{
    extern __shared__ __align__(128) unsigned char sm[];
    __shared__ int dead_;
    volatile int *dead = &dead_;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Head4 &w = p.w;
    const int per = w.units_per_tile;
    const int64_t t0 = (int64_t)w.tiles * blockIdx.x / gridDim.x, t1 = (int64_t)w.tiles * (blockIdx.x + 1) / gridDim.x;
    const int units = (int)(t1 - t0) * per;  // of the CTA
    auto first_of = [&](int i) { return (int)((int64_t)units * i / kStreamWarps); };
    const int u0 = first_of(warp), u1 = first_of(warp + 1);
    const unsigned char *from = w.units + (t0 * per + u0) * w.unit_bytes;
    const uint32_t ring_bytes = (uint32_t)(s.chunk * w.unit_bytes), bar = smem_at(sm + s.bars) + warp * kStreamStages * 8;
    const unsigned char *ring = sm + s.ring + (size_t)warp * kStreamStages * ring_bytes;
    const int chunks = (u1 - u0 + s.chunk - 1) / s.chunk;
    if (threadIdx.x == 0) dead_ = 0;
    if (lane == 0) {
        for (int i = 0; i < kStreamStages; i++) bar_init(bar + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_release();
    pdl_wait();
    auto load = [&](int c) {  // lane 0
        const int n = min(s.chunk, u1 - u0 - c * s.chunk), stage = c % kStreamStages;
        bar_expect(bar + 8 * stage, (uint32_t)(n * w.unit_bytes));
        bulk_load(smem_at(ring) + stage * ring_bytes, from + (int64_t)c * ring_bytes, (uint32_t)(n * w.unit_bytes), bar + 8 * stage);
    };
    if (lane == 0)
        for (int c = 0; c < kStreamStages && c < chunks; c++) load(c);
    float *sums = (float *)(sm + s.sums);
    stage_states<BF16, ZEROS, G, NT>(p, 0, 0, per * kUnitCols, sm, s.pitch, sums);

    const unsigned char *x = sm + (lane >> 2) * s.pitch + (lane & 3) * 16;
    float *slot = (float *)(sm + s.slots) + (size_t)warp * NT * 128;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] = 0.f;
    int ku = u0 % per, tile = u0 / per;      // the next unit's place
    bool own = ku == 0;                      // this warp has the tile's first unit
    bool left = false;                       // what is in acc belongs to a tile that is not at its end
    int c = 0;
    for (; c < chunks; c++) {
        const int stage = c % kStreamStages;
        if (!__all_sync(0xFFFFFFFFu, bar_wait(bar + 8 * stage, (c / kStreamStages) & 1, dead))) break;
        const int n = min(s.chunk, u1 - u0 - c * s.chunk);
        for (int j = 0; j < n; j++) {
            unit_logits<BF16, SBF16, ZEROS, G, NT>(acc, ring + stage * ring_bytes + j * w.unit_bytes, x + ku * (kUnitCols * 2), s.pitch, sums + ku * G * 8 * NT);
            left = true;
            if (++ku == per) {
                if (own) {
                    write_logits<NT>(p, acc, t0 + tile, 0);
                } else {
#pragma unroll
                    for (int m = 0; m < NT; m++) ((float4 *)slot)[m * 32 + lane] = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
                }
#pragma unroll
                for (int m = 0; m < NT; m++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[m][i] = 0.f;
                ku = 0;
                tile++;
                own = true;
                left = false;
            }
        }
        __syncwarp();
        if (lane == 0 && c + kStreamStages < chunks) load(c + kStreamStages);
    }
    if (left && !own) {
#pragma unroll
        for (int m = 0; m < NT; m++) ((float4 *)slot)[m * 32 + lane] = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
    }
    __syncthreads();
    if (left && own) {
        for (int i = warp + 1; i < kStreamWarps && first_of(i) < (tile + 1) * per; i++) {
            if (first_of(i) == first_of(i + 1)) continue;
            const float4 *other = (const float4 *)((float *)(sm + s.slots) + (size_t)i * NT * 128);
#pragma unroll
            for (int m = 0; m < NT; m++) {
                const float4 v = other[m * 32 + lane];
                acc[m][0] += v.x; acc[m][1] += v.y; acc[m][2] += v.z; acc[m][3] += v.w;
            }
        }
        write_logits<NT>(p, acc, t0 + tile, 0);
    }
    if (dead_ != 0) {  // a wait has given up: the copies under way end, and the CTA's logits are NaN
        if (lane == 0)
            for (int i = c; i < chunks && i < c + kStreamStages; i++)
                for (uint32_t j = 0; j < (1u << 20) && !bar_try(bar + 8 * (i % kStreamStages), (i / kStreamStages) & 1); j++) {}
        __syncthreads();
        for (int64_t i = threadIdx.x; i < (t1 - t0) * kHeadRows4 * p.rows; i += blockDim.x) {
            const int64_t v = t0 * kHeadRows4 + i / p.rows, r = i % p.rows;
            if (v >= w.vocab) break;
            if (p.out_bf16) ((uint16_t *)p.out)[r * p.out_stride + v] = 0x7FFFu;
            else ((float *)p.out)[r * p.out_stride + v] = __uint_as_float(0x7FFFFFFFu);
        }
    }
}

// More rows than the stream takes: blocks of 16 rows, each of which reads the weight.
constexpr int kLogitsCols = 2048;  // columns of the hidden states that a CTA has in shared memory at a time
constexpr int kLogitsPitch = kLogitsCols * 2 + 64;

template <bool BF16, bool SBF16, bool ZEROS, int G, int NT>
__global__ void __launch_bounds__(256) k_head_logits(const __grid_constant__ HeadLogits p)
{
    extern __shared__ __align__(128) unsigned char sm[];
    float *sums = (float *)(sm + 8 * NT * kLogitsPitch);
    const int lane = threadIdx.x & 31, tile = blockIdx.x * 8 + (threadIdx.x >> 5), r0 = blockIdx.y * 8 * NT;
    const Head4 &w = p.w;
    pdl_release();
    pdl_wait();
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] = 0.f;
    const unsigned char *x = sm + (lane >> 2) * kLogitsPitch + (lane & 3) * 16;
    for (int k0 = 0; k0 < w.width; k0 += kLogitsCols) {
        const int cols = min(kLogitsCols, w.units_per_tile * kUnitCols - k0);
        __syncthreads();
        stage_states<BF16, ZEROS, G, NT>(p, r0, k0, cols, sm, kLogitsPitch, sums);
        if (tile >= w.tiles) continue;
        const unsigned char *from = w.units + ((int64_t)tile * w.units_per_tile + k0 / kUnitCols) * w.unit_bytes;
#pragma unroll 2
        for (int u = 0; u < cols / kUnitCols; u++)
            unit_logits<BF16, SBF16, ZEROS, G, NT>(acc, from + (int64_t)u * w.unit_bytes, x + u * kUnitCols * 2, kLogitsPitch, sums + u * G * 8 * NT);
    }
    if (tile < w.tiles) write_logits<NT>(p, acc, tile, r0);
}

// ---- host ----

static int head4_check(StgHandle h, const char *who, int32_t vocab, int32_t width, int32_t group, int32_t scale_dtype)
{
    const std::string at = std::string(who) + ": ";
    if (vocab <= 0 || width <= 0) return fail(h, STG_ERR_INVALID_ARGUMENT, at + "vocab and width must be > 0");
    if (vocab > (1 << 26) || width > (1 << 16)) return fail(h, STG_ERR_CAPACITY, at + "more than 2^26 vocabulary entries or a width of 2^16");
    if (group != 32 && group != 64 && group != 128) return fail(h, STG_ERR_UNSUPPORTED, at + "group must be 32, 64 or 128");
    if (width % group != 0) return fail(h, STG_ERR_UNSUPPORTED, at + "width must be a multiple of group");
    if (scale_dtype != STG_DTYPE_BF16 && scale_dtype != STG_DTYPE_F16) return fail(h, STG_ERR_INVALID_ARGUMENT, at + "scale_dtype must be STG_DTYPE_BF16 or STG_DTYPE_F16");
    return STG_OK;
}

static int head_pack(StgHandle h, const StgHeadPack *b, cudaStream_t stream)
{
    if (!b || b->struct_size != (int32_t)sizeof(StgHeadPack)) return fail(h, STG_ERR_INVALID_ARGUMENT, "bad StgHeadPack");
    int rc = head4_check(h, "stg_head_pack", b->vocab, b->width, b->group, b->scale_dtype);
    if (rc) return rc;
    if (!b->codes || !b->scales || !b->packed) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_pack: codes, scales and packed are required");
    if (b->codes_stride < b->width / 2) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_pack: codes_stride smaller than width / 2");
    if (misaligned(b->scales, 2) || misaligned(b->zeros, 2) || misaligned(b->packed, 256))
        return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_pack: scales or zeros not aligned to their elements, or packed not to 256 bytes");
    HeadPack p;
    memset(&p, 0, sizeof(p));
    p.w = head4_shape(b->vocab, b->width, b->group, b->zeros != nullptr);
    if (b->packed_bytes < head4_bytes(p.w)) return fail(h, STG_ERR_CAPACITY, "stg_head_pack: packed is smaller than stg_head_pack_bytes says");
    const OnDevice on(h->cfg.device);
    CK(on.error);
    p.codes = (const uint8_t *)b->codes; p.codes_stride = b->codes_stride;
    p.scales = (const uint16_t *)b->scales; p.zeros = (const uint16_t *)b->zeros;
    p.out = (unsigned char *)b->packed;
    CK(launch_behind(k_head_pack, dim3((unsigned)h->sm_count * 8), 256, 0, stream, p));
    h->stats.kernel_launches++;
    return STG_OK;
}

static StreamShape stream_shape(const HeadLogits &p, int nt, bool zeros, size_t most)
{
    StreamShape s;
    memset(&s, 0, sizeof(s));
    const size_t cols = (size_t)p.w.units_per_tile * kUnitCols;
    s.pitch = (int)(cols * 2 + 64);  // rows g and g + 1 of a fragment in different banks
    s.sums = (size_t)8 * nt * s.pitch;
    s.slots = s.sums + (zeros ? cols / p.w.group * 8 * nt * 4 : 0);
    s.bars = s.slots + (size_t)kStreamWarps * nt * 512;
    s.ring = round_up(s.bars + kStreamWarps * kStreamStages * 8, 128);
    const size_t unit = (size_t)kStreamWarps * kStreamStages * p.w.unit_bytes;
    s.chunk = s.ring + unit <= most ? (int)std::min<size_t>(4, (most - s.ring) / unit) : 0;
    s.smem = s.ring + s.chunk * unit;
    return s;
}

template <bool BF16, bool SBF16, bool ZEROS, int G>
static cudaError_t launch_logits(StgHandle h, const HeadLogits &p, cudaStream_t stream)
{
    const int nt = p.rows <= 8 ? 1 : 2;
    const StreamShape s = stream_shape(p, nt, ZEROS, h->smem_optin);
    if (p.rows <= 16 && s.chunk > 0) {
        void (*fn)(HeadLogits, StreamShape) = nt == 1 ? k_head_stream<BF16, SBF16, ZEROS, G, 1> : k_head_stream<BF16, SBF16, ZEROS, G, 2>;
        const cudaError_t e = ensure_dynamic_smem((const void *)fn, s.smem);
        return e != cudaSuccess ? e : launch_behind(fn, dim3((unsigned)std::min(h->sm_count, p.w.tiles)), kStreamWarps * 32, s.smem, stream, p, s);
    }
    const size_t smem = (size_t)8 * nt * (kLogitsPitch + (ZEROS ? kLogitsCols / 32 * 4 : 0));
    void (*fn)(HeadLogits) = nt == 1 ? k_head_logits<BF16, SBF16, ZEROS, G, 1> : k_head_logits<BF16, SBF16, ZEROS, G, 2>;
    const cudaError_t e = ensure_dynamic_smem((const void *)fn, smem);
    return e != cudaSuccess ? e : launch_behind(fn, dim3((unsigned)(p.w.tiles + 7) / 8, (unsigned)(p.rows + 8 * nt - 1) / (8 * nt)), 256, smem, stream, p);
}

template <bool BF16, bool SBF16, bool ZEROS>
static cudaError_t launch_logits_of(StgHandle h, const HeadLogits &p, cudaStream_t stream)
{
    return p.w.group == 32 ? launch_logits<BF16, SBF16, ZEROS, 4>(h, p, stream) : p.w.group == 64 ? launch_logits<BF16, SBF16, ZEROS, 2>(h, p, stream)
                                                                                : launch_logits<BF16, SBF16, ZEROS, 1>(h, p, stream);
}

static int head_logits(StgHandle h, const StgHeadLogits *b, cudaStream_t stream)
{
    if (!b || b->struct_size != (int32_t)sizeof(StgHeadLogits)) return fail(h, STG_ERR_INVALID_ARGUMENT, "bad StgHeadLogits");
    int rc = head4_check(h, "stg_head_logits", b->vocab, b->width, b->group, b->scale_dtype);
    if (rc) return rc;
    if (b->rows < 0) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_logits: rows must be >= 0");
    if (b->rows > (1 << 20)) return fail(h, STG_ERR_CAPACITY, "stg_head_logits: more than 2^20 rows");
    if (b->hidden_dtype != STG_DTYPE_BF16 && b->hidden_dtype != STG_DTYPE_F16) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_logits: hidden_dtype must be STG_DTYPE_BF16 or STG_DTYPE_F16");
    if (b->logits_dtype != STG_DTYPE_F32 && b->logits_dtype != STG_DTYPE_BF16) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_logits: logits_dtype must be STG_DTYPE_F32 or STG_DTYPE_BF16");
    if (b->hidden_stride < b->width || b->row_stride < b->vocab) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_logits: a row stride smaller than the row");
    if (b->rows == 0) return STG_OK;
    if (!b->packed || !b->hidden || !b->logits) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_logits: packed, hidden and logits are required");
    if (misaligned(b->packed, 256) || misaligned(b->hidden, 2) || misaligned(b->logits, b->logits_dtype == STG_DTYPE_F32 ? 4 : 2))
        return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_logits: packed is not aligned to 256 bytes, or an array not to its elements");
    HeadLogits p;
    memset(&p, 0, sizeof(p));
    p.w = head4_shape(b->vocab, b->width, b->group, b->has_zeros != 0);
    if (b->packed_bytes != head4_bytes(p.w)) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_logits: packed_bytes is not what stg_head_pack_bytes says for these sizes");
    p.w.units = (const unsigned char *)b->packed;
    p.hidden = (const uint16_t *)b->hidden; p.hidden_stride = b->hidden_stride;
    p.vec = !misaligned(b->hidden, 16) && (b->rows == 1 || b->hidden_stride % 8 == 0);
    p.rows = b->rows; p.out = b->logits; p.out_stride = b->row_stride; p.out_bf16 = b->logits_dtype == STG_DTYPE_BF16;
    const OnDevice on(h->cfg.device);
    CK(on.error);
    using Launch = cudaError_t (*)(StgHandle, const HeadLogits &, cudaStream_t);
    static const Launch launch[2][2][2] = {{{launch_logits_of<false, false, false>, launch_logits_of<false, false, true>}, {launch_logits_of<false, true, false>, launch_logits_of<false, true, true>}},
                                           {{launch_logits_of<true, false, false>, launch_logits_of<true, false, true>}, {launch_logits_of<true, true, false>, launch_logits_of<true, true, true>}}};
    CK(launch[b->hidden_dtype == STG_DTYPE_BF16][b->scale_dtype == STG_DTYPE_BF16][b->has_zeros != 0](h, p, stream));
    h->stats.kernel_launches++;
    h->stats.calls++;
    return STG_OK;
}

}  // namespace stg

extern "C" {

int stg_head_pack_bytes(StgHandle h, int32_t vocab, int32_t width, int32_t group, int32_t has_zeros, uint64_t *out_bytes)
try {
    if (!h) return STG_ERR_INVALID_ARGUMENT;
    const int rc = stg::head4_check(h, "stg_head_pack_bytes", vocab, width, group, STG_DTYPE_F16);
    if (rc) return rc;
    if (!out_bytes) return stg::fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_pack_bytes: out_bytes is required");
    *out_bytes = stg::head4_bytes(stg::head4_shape(vocab, width, group, has_zeros != 0));
    return STG_OK;
} catch (const std::bad_alloc &) {
    return STG_ERR_CAPACITY;
}

int stg_head_pack(StgHandle h, const StgHeadPack *pack, void *stream)
try {
    return h ? stg::head_pack(h, pack, (cudaStream_t)stream) : STG_ERR_INVALID_ARGUMENT;
} catch (const std::bad_alloc &) {
    return STG_ERR_CAPACITY;
}

int stg_head_logits(StgHandle h, const StgHeadLogits *logits, void *stream)
try {
    return h ? stg::head_logits(h, logits, (cudaStream_t)stream) : STG_ERR_INVALID_ARGUMENT;
} catch (const std::bad_alloc &) {
    return STG_ERR_CAPACITY;
}

}  // extern "C"
