// stg_head_pack, stg_head_logits: a decode step's logits from a weight in 4 bits with a scale, and a zero point, per group of columns.
//
// logit[r][v] = sum over groups g of  scale[v][g] * (sum of (q - 8) h  -  (zero[v][g] - 8) * sum of h)  over the group's columns.
// q - 8 is exact in the hidden states' 16 bits and its products with them are exact in fp32, so a group's sum comes from the
// tensor cores without a rounding of the weight, and scales are applied to fp32 sums.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>
#include <string.h>

#include <new>

#include "stg_beam.h"
#include "stg_head4.cuh"
#include "stg_launch.h"
#include "stg_pdl.cuh"
#include "stg_tc.cuh"

namespace stg {

struct HeadPack {
    Head4 w;
    const uint8_t *codes;
    int64_t codes_stride;
    const uint16_t *scales, *zeros;
    unsigned char *out;
    bool vec;           // rows of codes begin at 16 bytes
};

// One warp per unit, whose codes - 64 bytes of each of 16 rows - it brings into shared memory first: 16 bytes at a time where rows begin at 16
// bytes (4096 x 151,936: 256 us, 378 with bytes read where they are needed).
__global__ void __launch_bounds__(256) k_head_pack(const __grid_constant__ HeadPack p)
{
    __shared__ uint4 codes[8][16][5];  // a row's 64 bytes, and 16 that keep rows out of each other's banks
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warp = threadIdx.x >> 5;
    const Head4 &w = p.w;
    const int64_t units = (int64_t)w.tiles * w.units_per_tile;
    pdl_release();
    pdl_wait();
    for (int64_t unit = blockIdx.x * 8ll + warp; unit < units; unit += gridDim.x * 8ll) {
        const int64_t v0 = unit / w.units_per_tile * kHeadRows4;
        const int k0 = (int)(unit % w.units_per_tile) * kUnitCols;
        unsigned char *out = p.out + unit * w.unit_bytes;
        __syncwarp();
#pragma unroll
        for (int i = lane; i < 64; i += 32) {
            const int row = i >> 2, part = i & 3;
            uint4 x = make_uint4(kCodeSigns, kCodeSigns, kCodeSigns, kCodeSigns);  // codes of 8 where there is no weight
            if (v0 + row < w.vocab && k0 + part * 32 < w.width) {  // the width is a multiple of 32
                const uint8_t *from = p.codes + (v0 + row) * p.codes_stride + k0 / 2 + part * 16;
                if (p.vec) {
                    x = __ldcs((const uint4 *)from);
                } else {
                    uint32_t e[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) e[j] = from[4 * j] | from[4 * j + 1] << 8 | from[4 * j + 2] << 16 | (uint32_t)from[4 * j + 3] << 24;
                    x = make_uint4(e[0], e[1], e[2], e[3]);
                }
            }
            codes[warp][row][part] = x;
        }
        __syncwarp();
        auto code = [&](int row, int col) -> uint32_t { return ((const uint8_t *)codes[warp][row])[col / 2]; };  // col is even: two codes of a byte
#pragma unroll
        for (int block = 0; block < 2; block++) {
            uint32_t word[4];
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const int col = block * 64 + 32 * (s / 2) + 8 * t + 4 * (s % 2);
                const uint32_t a = code(g, col), b = code(g + 8, col), c = code(g, col + 2), d = code(g + 8, col + 2);
                word[s] = (a & 15u) | (b & 15u) << 4 | (c & 15u) << 8 | (d & 15u) << 12 | (a >> 4) << 16 | (b >> 4) << 20 | (c >> 4) << 24 | (d >> 4) << 28;
            }
            ((uint4 *)(out + block * 512))[code_place(lane)] = make_uint4(word[0] ^ kCodeSigns, word[1] ^ kCodeSigns, word[2] ^ kCodeSigns, word[3] ^ kCodeSigns);
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

// Eight codes of a word as the four registers of an fp16 A fragment, q - 8 each.  A code, its highest bit turned back, is put below
// the bits of 1024, plain or times 16, and what is too much is taken off; all of it is exact.
struct CodeBits {  // held in registers: an instruction has room for one constant at most
    uint32_t low, high, low_base, high_base, low_less, high_less, sixteenth;
    __device__ __forceinline__ CodeBits()
    {
        asm volatile("mov.b32 %0, 0x000F000F;\nmov.b32 %1, 0x00F000F0;\nmov.b32 %2, 0x64086408;\nmov.b32 %3, 0x64806480;" : "=r"(low), "=r"(high), "=r"(low_base), "=r"(high_base));
        asm volatile("mov.b32 %0, 0xE408E408;\nmov.b32 %1, 0xD480D480;\nmov.b32 %2, 0x2C002C00;" : "=r"(low_less), "=r"(high_less), "=r"(sixteenth));  // -1032, -72, 1/16
    }
};
__device__ __forceinline__ void codes_to_a(const CodeBits &k, uint32_t w, uint32_t (&a)[4])
{
    const uint32_t u = w >> 8;
    const uint32_t v0 = bits_of(w, k.low, k.low_base), v1 = bits_of(w, k.high, k.high_base), v2 = bits_of(u, k.low, k.low_base), v3 = bits_of(u, k.high, k.high_base);
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(a[0]) : "r"(v0), "r"(k.low_less));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(a[1]) : "r"(v1), "r"(k.sixteenth), "r"(k.high_less));
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(a[2]) : "r"(v2), "r"(k.low_less));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(a[3]) : "r"(v3), "r"(k.sixteenth), "r"(k.high_less));
}

// d = a b + c
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// Entry g's and g + 8's scales or zero points of a unit's groups.
template <int G>
__device__ __forceinline__ void group_words(uint32_t (&to)[G], const unsigned char *from, int g)
{
    if constexpr (G == 4) {
        const uint4 v = ((const uint4 *)from)[g];
        to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
    } else if constexpr (G == 2) {
        const uint2 v = ((const uint2 *)from)[g];
        to[0] = v.x; to[1] = v.y;
    } else {
        to[0] = ((const uint32_t *)from)[g];
    }
}

// A unit's part of 16 logits for 8 NT rows of hidden states.  x: this lane's share of the first row group's row lane / 4 at the unit's first
// column; sums: of the unit's first group, per group 8 NT of them.
template <bool SBF16, bool ZEROS, int G, int NT>
__device__ __forceinline__ void unit_logits(const CodeBits &bits, float (&acc)[NT][4], const unsigned char *unit, const unsigned char *x, int pitch, const float *sums)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint4 q[2] = {((const uint4 *)unit)[code_place(lane)], ((const uint4 *)(unit + 512))[code_place(lane)]};
    const uint32_t word[8] = {q[0].x, q[0].y, q[0].z, q[0].w, q[1].x, q[1].y, q[1].z, q[1].w};
    uint32_t scale[G], zero[G];
    group_words<G>(scale, unit + kUnitCodes, g);
    if (ZEROS) group_words<G>(zero, unit + kUnitCodes + 32 * G, g);
#pragma unroll
    for (int gr = 0; gr < G; gr++) {
        float part[NT][4];
#pragma unroll
        for (int h = gr * (4 / G); h < (gr + 1) * (4 / G); h++) {  // 32 columns each
            uint32_t a0[4], a1[4];
            codes_to_a(bits, word[2 * h], a0);
            codes_to_a(bits, word[2 * h + 1], a1);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint4 v = *(const uint4 *)(x + n * 8 * pitch + h * 64);
                if (h == gr * (4 / G)) mma16816(part[n], a0, v.x, v.y, 0.f, 0.f, 0.f, 0.f);
                else mma16816(part[n], a0, v.x, v.y, part[n][0], part[n][1], part[n][2], part[n][3]);
                mma16816(part[n], a1, v.z, v.w, part[n][0], part[n][1], part[n][2], part[n][3]);
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

// The same for two rows of hidden states as integers of four digits, base 256, which are eight columns of mma.m16n8k32 over 8-bit integers:
// 16 (q - 8) of eight codes takes three instructions, where fp16 takes nine.  Sums of a group are exact; they come out on top of
// 1.5 * 2^23, as whose last bits they can be read in fp32 (below 2^21 each).
template <bool SBF16, bool ZEROS, int G>
__device__ __forceinline__ void unit_logits_int(float (&acc)[4], const unsigned char *unit, const unsigned char *x, const float *sums)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint4 q[2] = {((const uint4 *)unit)[code_place(lane)], ((const uint4 *)(unit + 512))[code_place(lane)]};
    const uint32_t word[8] = {q[0].x, q[0].y, q[0].z, q[0].w, q[1].x, q[1].y, q[1].z, q[1].w};
    const uint4 b[2] = {((const uint4 *)x)[0], ((const uint4 *)x)[1]};
    const uint32_t digits[8] = {b[0].x, b[0].y, b[0].z, b[0].w, b[1].x, b[1].y, b[1].z, b[1].w};
    uint32_t scale[G], zero[G];
    group_words<G>(scale, unit + kUnitCodes, g);
    if (ZEROS) group_words<G>(zero, unit + kUnitCodes + 32 * G, g);
    constexpr int kTop = 0x4B400000;
#pragma unroll
    for (int gr = 0; gr < G; gr++) {
        int part[4] = {kTop, kTop, kTop, kTop};
#pragma unroll
        for (int h = gr * (4 / G); h < (gr + 1) * (4 / G); h++) {
            const uint32_t a0 = (word[2 * h] * 16u) & 0xF0F0F0F0u, a1 = word[2 * h] & 0xF0F0F0F0u;
            const uint32_t a2 = (word[2 * h + 1] * 16u) & 0xF0F0F0F0u, a3 = word[2 * h + 1] & 0xF0F0F0F0u;
            asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                : "=r"(part[0]), "=r"(part[1]), "=r"(part[2]), "=r"(part[3])
                : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(digits[2 * h]), "r"(digits[2 * h + 1]), "r"(part[0]), "r"(part[1]), "r"(part[2]), "r"(part[3]));
        }
        const float s0 = half_at<SBF16>((uint16_t)scale[gr]), s1 = half_at<SBF16>((uint16_t)(scale[gr] >> 16));
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = __int_as_float(part[i]) - 12582912.f;
        if (ZEROS) {
            const float z0 = 8.f - half_at<SBF16>((uint16_t)zero[gr]), z1 = 8.f - half_at<SBF16>((uint16_t)(zero[gr] >> 16));
            const float2 u = *(const float2 *)(sums + gr * 8 + 2 * t);
            f[0] = fmaf(z0, u.x, f[0]);
            f[1] = fmaf(z0, u.y, f[1]);
            f[2] = fmaf(z1, u.x, f[2]);
            f[3] = fmaf(z1, u.y, f[3]);
        }
        acc[0] = fmaf(s0, f[0], acc[0]);
        acc[1] = fmaf(s0, f[1], acc[1]);
        acc[2] = fmaf(s1, f[2], acc[2]);
        acc[3] = fmaf(s1, f[3], acc[3]);
    }
}

template <int NT>
__device__ __forceinline__ void write_logits(const HeadLogits &p, const float (&acc)[NT][4], int64_t tile, const float2 *unscale)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t v = tile * kHeadRows4 + g + (i >= 2 ? 8 : 0);
            const int r = n * 8 + 2 * t + (i & 1);
            if (v >= p.w.vocab || r >= p.rows) continue;
            const float2 u = unscale[r];
            const float x = acc[n][i] * u.x * u.y;
            if (p.out_bf16) ((__nv_bfloat16 *)p.out)[r * p.out_stride + v] = __float2bfloat16_rn(x);
            else ((float *)p.out)[r * p.out_stride + v] = x;
        }
}

// The sums of groups of hidden states that lie in shared memory, for zero points; `cols` whole units.
template <int G, int NT>
__device__ __forceinline__ void sum_groups(int cols, const unsigned char *xs, int pitch, float *sums)
{
    constexpr int kGroup = kUnitCols / G;
    for (int i = threadIdx.x; i < cols / kGroup * 8 * NT; i += blockDim.x) {
        const int n = i % (8 * NT), gr = i / (8 * NT);
        float s = 0.f;
        for (int k = 0; k < kGroup; k += 8) {
            const uint4 v = *(const uint4 *)(xs + n * pitch + (gr * kGroup + k) * 2);
            const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; j++) s += half_at<false>((uint16_t)e[j]) + half_at<false>((uint16_t)(e[j] >> 16));
        }
        sums[i] = s;
    }
}

// Hidden states of up to 8 NT rows into shared memory in fp16, zeros where there are none, `cols` whole units: bf16 ones times a power of two that
// takes a row's largest finite one to [2^14, 2^15).  That is exact down to 2^-29 of it, and 2^-40 of it off below.  `unscale`: the
// inverse, in two factors.
template <bool ZEROS, int G, int NT>
__device__ __forceinline__ void stage_rows(const HeadLogits &p, int cols, unsigned char *xs, int pitch, float *sums, float2 *unscale, uint32_t *most)
{
    const int per = cols / 8;  // a multiple of 16
    if (threadIdx.x < 8 * NT) most[threadIdx.x] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * NT * per; i += blockDim.x) {
        const int n = i / per, k = (i - n * per) * 8;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (n < p.rows && k < p.w.width) v = eight_states(p.hidden + (int64_t)n * p.hidden_stride + k, p.vec);
        *(uint4 *)(xs + n * pitch + k * 2) = v;
        if (p.hidden_bf16 && n < p.rows) {  // half warps have one row
            const uint32_t e[4] = {v.x, v.y, v.z, v.w};
            uint32_t m = 0u;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t lo = e[j] & 0x7FFFu, hi = e[j] >> 16 & 0x7FFFu;
                m = max(m, max(lo < 0x7F80u ? lo : 0u, hi < 0x7F80u ? hi : 0u));
            }
            m = __reduce_max_sync(0xFFFFu << (threadIdx.x & 16), m);
            if ((threadIdx.x & 15) == 0) atomicMax(&most[n], m);
        }
    }
    __syncthreads();
    if (p.hidden_bf16) {
        for (int i = threadIdx.x; i < min(8 * NT, p.rows) * per; i += blockDim.x) {
            const int n = i / per;
            const float top = __uint_as_float(most[n] << 16);
            const int e = top > 0.f ? 14 - ilogbf(top) : 0, half = e / 2;
            const float s1 = __uint_as_float((uint32_t)(127 + half) << 23), s2 = __uint_as_float((uint32_t)(127 + e - half) << 23);
            uint4 *at = (uint4 *)(xs + n * pitch + (i - n * per) * 16);
            const uint4 v = *at;
            uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; j++)
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(x[j]) : "f"(half_at<true>((uint16_t)(x[j] >> 16)) * s1 * s2), "f"(half_at<true>((uint16_t)x[j]) * s1 * s2));
            *at = make_uint4(x[0], x[1], x[2], x[3]);
        }
    }
    if (threadIdx.x < 8 * NT) {
        const float top = __uint_as_float(most[threadIdx.x] << 16);
        const int e = top > 0.f ? 14 - ilogbf(top) : 0, half = e / 2;
        unscale[threadIdx.x] = make_float2(__uint_as_float((uint32_t)(127 - half) << 23), __uint_as_float((uint32_t)(127 - (e - half)) << 23));
    }
    __syncthreads();
    if (ZEROS) {
        sum_groups<G, NT>(cols, xs, pitch, sums);
        __syncthreads();
    }
}

// Up to two rows as integers: hidden state x is X * 2^(e - 30), e the exponent above the row's largest finite one, X rounded - exact down to
// 2^-22 of the largest, 2^-31 of it off below - and X four digits of -128 .. 127.  Column 4 r + d of `xs` (pitch bytes between columns) has
// digit d of row r, the highest first; of a unit's 128 columns a lane's are next to each other: byte 32 t + 8 h + i is column
// 32 h + 8 t + i, the middle two of every four exchanged.  A row with a hidden state that is not finite comes out NaN: `bad` says
// so, and the inverse that its logits are multiplied with at the end is NaN.
template <bool ZEROS, int G>
__device__ __forceinline__ void stage_digits(const HeadLogits &p, int cols, unsigned char *xs, int pitch, float *sums, float2 *unscale, uint32_t *most)
{
    const int per = cols / 8;
    if (threadIdx.x < 8) most[threadIdx.x] = 0u;
    __syncthreads();
    float bad[2] = {0.f, 0.f};
    // twice over the rows, which are in L2 or L1: for the largest, and for the digits
    for (int pass = 0; pass < 2; pass++) {
        for (int i = threadIdx.x; i < 2 * per; i += blockDim.x) {
            const int r = i >= per ? 1 : 0, k = (i - r * per) * 8;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (r < p.rows && k < p.w.width) v = eight_states(p.hidden + (int64_t)r * p.hidden_stride + k, p.vec);
            const uint32_t e[4] = {v.x, v.y, v.z, v.w};
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint16_t h = (uint16_t)(e[j / 2] >> (16 * (j & 1)));
                x[j] = p.hidden_bf16 ? half_at<true>(h) : half_at<false>(h);
                if (!(fabsf(x[j]) < CUDART_INF_F)) {
                    bad[r] += x[j] * 0.f;
                    x[j] = 0.f;
                }
            }
            if (pass == 0) {
                float m = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(x[j]));
                const uint32_t u = __reduce_max_sync(0xFFFFu << (threadIdx.x & 16), __float_as_uint(m));
                if ((threadIdx.x & 15) == 0) atomicMax(&most[r], u);
            } else {
                const float top = __uint_as_float(most[r]);
                const int e2 = top > 0.f ? 29 - ilogbf(top) : 0, half = e2 / 2;  // |X| < 2^30
                const float s1 = __uint_as_float((uint32_t)(127 + half) << 23), s2 = __uint_as_float((uint32_t)(127 + e2 - half) << 23);
                uint32_t d[4][2] = {};
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    int X = __float2int_rn(x[j] * s1 * s2);
                    const int byte = (j & 3) == 1 ? 2 : (j & 3) == 2 ? 1 : (j & 3);
#pragma unroll
                    for (int n = 3; n >= 0; n--) {
                        const int digit = (int)(int8_t)X;
                        d[n][j / 4] |= (uint32_t)(uint8_t)digit << (8 * byte);
                        X = (X - digit) >> 8;
                    }
                }
                const int in = k & 127, at = (k & ~127) + (in >> 3 & 3) * 32 + (in >> 5) * 8;
#pragma unroll
                for (int n = 0; n < 4; n++) *(uint2 *)(xs + (4 * r + n) * pitch + at) = make_uint2(d[n][0], d[n][1]);
            }
        }
        __syncthreads();
    }
    // (most[4 + r], behind the rows' largest: what is added to a row's logits)
#pragma unroll
    for (int r = 0; r < 2; r++)
        if (bad[r] != 0.f) ((volatile uint32_t *)most)[4 + r] = 0x7FC00000u;  // NaN: times zero, so is an infinity
    __syncthreads();
    if (threadIdx.x < 2) {
        const float top = __uint_as_float(most[threadIdx.x]);
        const int e2 = top > 0.f ? 29 - ilogbf(top) + 4 : 4, half = e2 / 2;  // 16 (q - 8)
        const float nan = __uint_as_float(most[4 + threadIdx.x]);
        unscale[threadIdx.x] = make_float2(__uint_as_float((uint32_t)(127 - half) << 23) + nan, __uint_as_float((uint32_t)(127 - (e2 - half)) << 23));
    }
    if (ZEROS) {
        constexpr int kGroup = kUnitCols / G;
        for (int i = threadIdx.x; i < cols / kGroup * 8; i += blockDim.x) {  // column n of group gr: a group is bytes 8 h .. of every 32
            const int n = i % 8, gr = i / 8;
            const unsigned char *from = xs + n * pitch + gr / G * kUnitCols + (gr % G) * (32 / G);
            int sum = 0;
            for (int t = 0; t < 4; t++)
                for (int j = 0; j < 32 / G; j += 4) sum = __dp4a(*(const int *)(from + 32 * t + j), 0x01010101, sum);
            sums[i] = 16.f * (float)sum;
        }
    }
    __syncthreads();
}

// Up to 16 rows at a time: the weight streams through, once.  Hidden states lie in shared memory whole.  A CTA per SM has a run of tiles, whose
// units its 16 warps share out evenly, each a run of neighbours that it copies into a ring of its own (bulk copies, one per stage), so no
// warp waits for another before the end.  A tile that several warps have units of is added up there, by the warp that has its first.
//
// One row x 4096 x 151,936, groups of 32: 60 us for 351 MB (5.9 TB/s, 89 % of the copy rate; 84 as fp16, 250 with plain loads and fp16);
// groups of 128: 56.  Three to eight rows 65 to 73, bound by instructions (154 for a unit of 2048 weights, of which unpacking is 72 and
// the products 8); 16 rows 98 to 104, where the products' pipe and the unpacking's share the time.
template <int NT, bool INT>
__device__ __forceinline__ void stream_write(const HeadLogits &p, const float (&acc)[NT][4], int64_t tile, const float2 *unscale)
{
    if constexpr (INT) {  // two lanes have a row's digits: columns 2 t and 2 t + 1
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, r = t >> 1;
        const float s1 = (t & 1) ? 256.f : 16777216.f, s2 = (t & 1) ? 1.f : 65536.f;
        float low = acc[0][0] * s1 + acc[0][1] * s2, high = acc[0][2] * s1 + acc[0][3] * s2;
        low += __shfl_xor_sync(0xFFFFFFFFu, low, 1);
        high += __shfl_xor_sync(0xFFFFFFFFu, high, 1);
        const int64_t v = tile * kHeadRows4 + g + 8 * (t & 1);
        if (r < p.rows && v < p.w.vocab) {
            const float2 u = unscale[r];
            const float x = ((t & 1) ? high : low) * u.x * u.y;
            if (p.out_bf16) ((__nv_bfloat16 *)p.out)[r * p.out_stride + v] = __float2bfloat16_rn(x);
            else ((float *)p.out)[r * p.out_stride + v] = x;
        }
    } else {
        write_logits<NT>(p, acc, tile, unscale);
    }
}

// INT: up to two rows as integers, NT 1.
template <bool SBF16, bool ZEROS, int G, int NT, bool INT>
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
    async_fence();  // the weight may have been packed by the kernel ahead
    auto load = [&](int c) {  // lane 0
        const int n = min(s.chunk, u1 - u0 - c * s.chunk), stage = c % kStreamStages;
        bar_expect(bar + 8 * stage, (uint32_t)(n * w.unit_bytes));
        bulk_load(smem_at(ring) + stage * ring_bytes, from + (int64_t)c * ring_bytes, (uint32_t)(n * w.unit_bytes), bar + 8 * stage);
    };
    if (lane == 0)
        for (int c = 0; c < kStreamStages && c < chunks; c++) load(c);
    float *sums = (float *)(sm + s.sums);
    const float2 *unscale = (const float2 *)(sm + s.unscale);
    __shared__ uint32_t most[8 * NT];
    if (INT) stage_digits<ZEROS, G>(p, per * kUnitCols, sm, s.pitch, sums, (float2 *)(sm + s.unscale), most);
    else stage_rows<ZEROS, G, NT>(p, per * kUnitCols, sm, s.pitch, sums, (float2 *)(sm + s.unscale), most);

    const unsigned char *x = sm + (lane >> 2) * s.pitch + (lane & 3) * (INT ? 32 : 16);
    float *slot = (float *)(sm + s.slots) + (size_t)warp * NT * 128;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] = 0.f;
    const CodeBits bits;
    int ku = u0 % per, tile = u0 / per;      // the next unit's place
    bool own = ku == 0;                      // this warp has the tile's first unit
    bool left = false;                       // what is in acc belongs to a tile that is not at its end
    int c = 0;
    for (; c < chunks; c++) {
        const int stage = c % kStreamStages;
        if (!__all_sync(0xFFFFFFFFu, bar_wait(bar + 8 * stage, (c / kStreamStages) & 1, dead))) break;
        const int n = min(s.chunk, u1 - u0 - c * s.chunk);
        for (int j = 0; j < n; j++) {
            const unsigned char *unit = ring + stage * ring_bytes + j * w.unit_bytes;
            if constexpr (INT) unit_logits_int<SBF16, ZEROS, G>(acc[0], unit, x + ku * kUnitCols, sums + ku * G * 8);
            else unit_logits<SBF16, ZEROS, G, NT>(bits, acc, unit, x + ku * (kUnitCols * 2), s.pitch, sums + ku * G * 8 * NT);
            left = true;
            if (++ku == per) {
                if (own) {
                    stream_write<NT, INT>(p, acc, t0 + tile, unscale);
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
        stream_write<NT, INT>(p, acc, t0 + tile, unscale);
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
    p.vec = !misaligned(b->codes, 16) && b->codes_stride % 16 == 0;
    p.scales = (const uint16_t *)b->scales; p.zeros = (const uint16_t *)b->zeros;
    p.out = (unsigned char *)b->packed;
    CK(launch_behind(k_head_pack, dim3((unsigned)h->sm_count * 8), 256, 0, stream, p));
    h->stats.kernel_launches++;
    return STG_OK;
}

template <bool SBF16, bool ZEROS, int G>
static cudaError_t launch_stream(StgHandle h, const HeadLogits &p, cudaStream_t stream)
{
    const StreamShape s = stream_shape(p.w, p.rows, ZEROS, h->smem_optin);
    void (*fn)(HeadLogits, StreamShape) = p.rows <= kIntRows ? k_head_stream<SBF16, ZEROS, G, 1, true> : p.rows <= 8 ? k_head_stream<SBF16, ZEROS, G, 1, false>
                                                                                                                    : k_head_stream<SBF16, ZEROS, G, 2, false>;
    const cudaError_t e = ensure_dynamic_smem((const void *)fn, s.smem);
    return e != cudaSuccess ? e : launch_behind(fn, dim3((unsigned)std::min(h->sm_count, p.w.tiles)), kStreamWarps * 32, s.smem, stream, p, s);
}

template <bool SBF16, bool ZEROS>
static cudaError_t launch_stream_of(StgHandle h, const HeadLogits &p, cudaStream_t stream)
{
    return p.w.group == 32 ? launch_stream<SBF16, ZEROS, 4>(h, p, stream) : p.w.group == 64 ? launch_stream<SBF16, ZEROS, 2>(h, p, stream)
                                                                                : launch_stream<SBF16, ZEROS, 1>(h, p, stream);
}

static int head_logits_check(StgHandle h, const StgHeadLogits *b, const char *who)
{
    const std::string at = std::string(who) + ": ";
    if (!b || b->struct_size != (int32_t)sizeof(StgHeadLogits)) return fail(h, STG_ERR_INVALID_ARGUMENT, "bad StgHeadLogits");
    const int rc = head4_check(h, who, b->vocab, b->width, b->group, b->scale_dtype);
    if (rc) return rc;
    if (b->rows < 0) return fail(h, STG_ERR_INVALID_ARGUMENT, at + "rows must be >= 0");
    if (b->rows > (1 << 20)) return fail(h, STG_ERR_CAPACITY, at + "more than 2^20 rows");
    if (b->hidden_dtype != STG_DTYPE_BF16 && b->hidden_dtype != STG_DTYPE_F16) return fail(h, STG_ERR_INVALID_ARGUMENT, at + "hidden_dtype must be STG_DTYPE_BF16 or STG_DTYPE_F16");
    if (b->logits_dtype != STG_DTYPE_F32 && b->logits_dtype != STG_DTYPE_BF16) return fail(h, STG_ERR_INVALID_ARGUMENT, at + "logits_dtype must be STG_DTYPE_F32 or STG_DTYPE_BF16");
    return STG_OK;
}

static size_t head_logits_workspace(StgHandle h, const StgHeadLogits *b)
{
    const Head4 w = head4_shape(b->vocab, b->width, b->group, b->has_zeros != 0);
    return b->rows == 0 || streams(w, b->rows, b->has_zeros != 0, h->smem_optin) ? 0 : head_tiles_workspace(h, w, b->rows);
}

static int head_logits(StgHandle h, const StgHeadLogits *b, cudaStream_t stream)
{
    const int rc = head_logits_check(h, b, "stg_head_logits");
    if (rc) return rc;
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
    p.rows = b->rows; p.hidden_bf16 = b->hidden_dtype == STG_DTYPE_BF16; p.out = b->logits; p.out_stride = b->row_stride; p.out_bf16 = b->logits_dtype == STG_DTYPE_BF16;
    const OnDevice on(h->cfg.device);
    CK(on.error);
    if (!streams(p.w, p.rows, b->has_zeros != 0, h->smem_optin)) {
        if (!b->workspace || misaligned(b->workspace, 256) || b->workspace_bytes < head_tiles_workspace(h, p.w, p.rows))
            return fail(h, STG_ERR_CAPACITY, "stg_head_logits: workspace missing, not aligned to 256 bytes or smaller than stg_head_logits_workspace says");
        const int rc2 = head_tiles(h, p, b->scale_dtype == STG_DTYPE_BF16, b->workspace, stream);
        if (rc2) return rc2;
    } else {
        using Launch = cudaError_t (*)(StgHandle, const HeadLogits &, cudaStream_t);
        static const Launch launch[2][2] = {{launch_stream_of<false, false>, launch_stream_of<false, true>}, {launch_stream_of<true, false>, launch_stream_of<true, true>}};
        const int calls = (p.rows + 15) / 16, rows = p.rows, each = (rows + calls - 1) / calls;
        for (int r = 0; r < rows; r += each) {
            HeadLogits q = p;
            q.rows = std::min(each, rows - r);
            q.hidden += (int64_t)r * p.hidden_stride;
            q.out = (char *)p.out + (int64_t)r * p.out_stride * (p.out_bf16 ? 2 : 4);
            CK(launch[b->scale_dtype == STG_DTYPE_BF16][b->has_zeros != 0](h, q, stream));
            h->stats.kernel_launches++;
        }
    }
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

int stg_head_logits_workspace(StgHandle h, const StgHeadLogits *logits, uint64_t *out_bytes)
try {
    if (!h) return STG_ERR_INVALID_ARGUMENT;
    const int rc = stg::head_logits_check(h, logits, "stg_head_logits_workspace");
    if (rc) return rc;
    if (!out_bytes) return stg::fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_logits_workspace: out_bytes is required");
    *out_bytes = stg::head_logits_workspace(h, logits);
    return STG_OK;
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
