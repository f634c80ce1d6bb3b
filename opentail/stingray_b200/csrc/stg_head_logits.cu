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

namespace stg {

// The packed weight: tiles of 16 vocabulary entries by blocks of 64 columns, 512 bytes each, a tile's blocks next to each other; then
// per tile and group the 16 scales, then in the same way the zero points.  A lane of a warp holds 16 bytes of a block, which are what
// it needs of the weight in four steps of mma.m16n8k16 (word s: step s); the columns of a step are chosen such that a lane's share
// of a hidden state are eight neighbours for two steps: step s, columns 32 (s / 2) + 8 t + 4 (s % 2) + 0..3 for t = lane % 4.
constexpr int kHeadRows4 = 16, kHeadCols4 = 64, kHeadBlock4 = 512;

struct Head4 {
    const unsigned char *codes, *scales, *zeros;
    int vocab, width, group, blocks, groups, tiles;  // groups: of the padded width
};

static void head4_shape(int vocab, int width, int group, bool zeros, Head4 &w, size_t &bytes)
{
    w.vocab = vocab; w.width = width; w.group = group;
    w.blocks = (width + kHeadCols4 - 1) / kHeadCols4;
    w.groups = std::max(1, (w.blocks * kHeadCols4 + group - 1) / group);
    w.tiles = (vocab + kHeadRows4 - 1) / kHeadRows4;
    const size_t codes = (size_t)w.tiles * w.blocks * kHeadBlock4, scales = round_up((size_t)w.tiles * w.groups * 32, 256);
    w.codes = nullptr;
    w.scales = w.codes + codes;
    w.zeros = zeros ? w.scales + scales : nullptr;
    bytes = codes + scales * (zeros ? 2 : 1);
}

struct HeadPack {
    const uint8_t *codes;
    int64_t codes_stride;
    const uint16_t *scales, *zeros;
    unsigned char *out_codes;
    uint16_t *out_scales, *out_zeros;
    int vocab, width, group, blocks, groups, true_groups;
};

// One warp per tile and block.
__global__ void __launch_bounds__(256) k_head_pack(const __grid_constant__ HeadPack p)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, block = blockIdx.x * 8 + (threadIdx.x >> 5), tile = blockIdx.y;
    pdl_release();
    pdl_wait();
    if (block >= p.blocks) return;
    auto code = [&](int row, int col) -> uint32_t {  // col is even: two codes of a byte
        const int v = tile * kHeadRows4 + row;
        return v < p.vocab && col < p.width ? p.codes[(int64_t)v * p.codes_stride + col / 2] : 0x88u;
    };
    uint32_t word[4];
#pragma unroll
    for (int s = 0; s < 4; s++) {
        const int col = block * kHeadCols4 + 32 * (s / 2) + 8 * t + 4 * (s % 2);
        const uint32_t a = code(g, col), b = code(g + 8, col), c = code(g, col + 2), d = code(g + 8, col + 2);
        word[s] = (a & 15u) | (b & 15u) << 4 | (c & 15u) << 8 | (d & 15u) << 12 | (a >> 4) << 16 | (b >> 4) << 20 | (c >> 4) << 24 | (d >> 4) << 28;
    }
    ((uint4 *)(p.out_codes + ((int64_t)tile * p.blocks + block) * kHeadBlock4))[lane] = make_uint4(word[0], word[1], word[2], word[3]);
}

// Scales and zero points: per tile and group eight pairs of entries g and g + 8.  Where there is no weight: scale 0.
__global__ void __launch_bounds__(256) k_head_pack_scales(const __grid_constant__ HeadPack p)
{
    pdl_release();
    pdl_wait();
    const int64_t n = (int64_t)((p.vocab + kHeadRows4 - 1) / kHeadRows4) * p.groups * 16;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const int pair = (int)(i & 15), group = (int)((i >> 4) % p.groups);
        const int64_t v = (i >> 4) / p.groups * kHeadRows4 + (pair >> 1) + 8 * (pair & 1);
        const bool on = v < p.vocab && group < p.true_groups;
        p.out_scales[i] = on ? p.scales[v * p.true_groups + group] : 0;
        if (p.zeros) p.out_zeros[i] = on ? p.zeros[v * p.true_groups + group] : 0;
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

constexpr int kLogitsCols = 2048;  // columns of the hidden states that a CTA has in shared memory at a time
constexpr int kLogitsPitch = kLogitsCols * 2 + 64;

// A warp has a tile of 16 vocabulary entries and NT times eight rows of hidden states.
template <bool BF16, bool SBF16, bool ZEROS, int NT>
__global__ void __launch_bounds__(256) k_head_logits(const __grid_constant__ HeadLogits p, bool out_bf16)
{
    extern __shared__ uint4 smem4[];
    unsigned char *xs = (unsigned char *)smem4;                    // [8 NT][kLogitsPitch]
    float *sums = (float *)(xs + 8 * NT * kLogitsPitch);           // [groups of a chunk][8 NT]
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, tile = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int r0 = blockIdx.y * 8 * NT, rows = min(8 * NT, p.rows - r0);
    const Head4 &w = p.w;
    pdl_release();
    pdl_wait();
    float acc[NT][4], part[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] = part[n][i] = 0.f;
    const uint32_t *scales = (const uint32_t *)w.scales + (int64_t)tile * w.groups * 8 + g;
    const uint32_t *zeros = (const uint32_t *)w.zeros + (int64_t)tile * w.groups * 8 + g;
    for (int k0 = 0; k0 < w.width; k0 += kLogitsCols) {
        const int cols = min(kLogitsCols, w.blocks * kHeadCols4 - k0);
        __syncthreads();
        for (int i = threadIdx.x; i < 8 * NT * (cols / 8); i += 256) {
            const int n = i / (cols / 8), k = (i - n * (cols / 8)) * 8;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            const uint16_t *from = p.hidden + (int64_t)(r0 + n) * p.hidden_stride + k0 + k;
            if (n < rows && k0 + k < w.width) {  // the width is a multiple of 32
                if (p.vec) {
                    v = __ldg((const uint4 *)from);
                } else {
                    uint32_t e[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) e[j] = from[j];
                    v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
                }
            }
            *(uint4 *)(xs + n * kLogitsPitch + k * 2) = v;
        }
        __syncthreads();
        const int groups = (cols + w.group - 1) / w.group;
        if (ZEROS) {
            for (int i = threadIdx.x; i < groups * 8 * NT; i += 256) {
                const int n = i % (8 * NT), gr = i / (8 * NT);
                float s = 0.f;
                for (int k = gr * w.group; k < min(cols, (gr + 1) * w.group); k++) s += half_at<BF16>(*(const uint16_t *)(xs + n * kLogitsPitch + k * 2));
                sums[gr * 8 * NT + n] = s;
            }
            __syncthreads();
        }
        if (tile >= w.tiles) continue;
        const uint4 *codes = (const uint4 *)(w.codes + ((int64_t)tile * w.blocks + k0 / kHeadCols4) * kHeadBlock4) + lane;
        const int steps_per_group = w.group / 16;
        int step = 0;
#pragma unroll 4
        for (int b = 0; b < cols / kHeadCols4; b++) {
            const uint4 q = __ldcs(codes + b * 32);
            const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t a0[4], a1[4];
                codes_to_a<BF16>(word[2 * h], a0);
                codes_to_a<BF16>(word[2 * h + 1], a1);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const uint4 x = *(const uint4 *)(xs + (n * 8 + g) * kLogitsPitch + (b * kHeadCols4 + h * 32 + 8 * t) * 2);
                    mma16816<BF16>(part[n], a0, x.x, x.y);
                    mma16816<BF16>(part[n], a1, x.z, x.w);
                }
                step += 2;
                if (step % steps_per_group == 0) {
                    const int gr = step / steps_per_group - 1;
                    const uint32_t s2 = __ldg(scales + (k0 / w.group + gr) * 8);
                    const float s0 = half_at<SBF16>((uint16_t)s2), s1 = half_at<SBF16>((uint16_t)(s2 >> 16));
                    float z0 = 0.f, z1 = 0.f;
                    if (ZEROS) {
                        const uint32_t z2 = __ldg(zeros + (k0 / w.group + gr) * 8);
                        z0 = 8.f - half_at<SBF16>((uint16_t)z2);
                        z1 = 8.f - half_at<SBF16>((uint16_t)(z2 >> 16));
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        if (ZEROS) {
                            const float2 x = *(const float2 *)(sums + gr * 8 * NT + n * 8 + 2 * t);
                            part[n][0] = fmaf(z0, x.x, part[n][0]);
                            part[n][1] = fmaf(z0, x.y, part[n][1]);
                            part[n][2] = fmaf(z1, x.x, part[n][2]);
                            part[n][3] = fmaf(z1, x.y, part[n][3]);
                        }
                        acc[n][0] = fmaf(s0, part[n][0], acc[n][0]);
                        acc[n][1] = fmaf(s0, part[n][1], acc[n][1]);
                        acc[n][2] = fmaf(s1, part[n][2], acc[n][2]);
                        acc[n][3] = fmaf(s1, part[n][3], acc[n][3]);
#pragma unroll
                        for (int i = 0; i < 4; i++) part[n][i] = 0.f;
                    }
                }
            }
        }
    }
    if (tile >= w.tiles) return;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int v = tile * kHeadRows4 + g + (i >= 2 ? 8 : 0), r = n * 8 + 2 * t + (i & 1);
            if (v >= w.vocab || r >= rows) continue;
            const int64_t at = (int64_t)(r0 + r) * p.out_stride + v;
            if (out_bf16) ((__nv_bfloat16 *)p.out)[at] = __float2bfloat16_rn(acc[n][i]);
            else ((float *)p.out)[at] = acc[n][i];
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
    Head4 w;
    size_t bytes;
    head4_shape(b->vocab, b->width, b->group, b->zeros != nullptr, w, bytes);
    if (b->packed_bytes < bytes) return fail(h, STG_ERR_CAPACITY, "stg_head_pack: packed is smaller than stg_head_pack_bytes says");
    const OnDevice on(h->cfg.device);
    CK(on.error);
    HeadPack p;
    memset(&p, 0, sizeof(p));
    unsigned char *base = (unsigned char *)b->packed;
    p.codes = (const uint8_t *)b->codes; p.codes_stride = b->codes_stride;
    p.scales = (const uint16_t *)b->scales; p.zeros = (const uint16_t *)b->zeros;
    p.out_codes = base;
    p.out_scales = (uint16_t *)(base + (size_t)w.scales);
    p.out_zeros = b->zeros ? (uint16_t *)(base + (size_t)w.zeros) : nullptr;
    p.vocab = b->vocab; p.width = b->width; p.group = b->group; p.blocks = w.blocks; p.groups = w.groups; p.true_groups = b->width / b->group;
    const int most = 65535;
    for (int t = 0; t < w.tiles; t += most) {
        HeadPack q = p;
        const int n = std::min(most, w.tiles - t);
        q.codes += (int64_t)t * kHeadRows4 * p.codes_stride;
        q.vocab -= t * kHeadRows4;
        q.out_codes += (int64_t)t * w.blocks * kHeadBlock4;
        CK(launch_behind(k_head_pack, dim3((unsigned)(w.blocks + 7) / 8, (unsigned)n), 256, 0, stream, q));
        h->stats.kernel_launches++;
    }
    CK(launch_behind(k_head_pack_scales, dim3((unsigned)h->sm_count * 4), 256, 0, stream, p));
    h->stats.kernel_launches++;
    return STG_OK;
}

template <bool BF16, bool SBF16, bool ZEROS>
static cudaError_t launch_logits(const HeadLogits &p, bool out_bf16, cudaStream_t stream)
{
    const dim3 grid((unsigned)(p.w.tiles + 7) / 8, (unsigned)(p.rows <= 8 ? 1 : (p.rows + 15) / 16));
    const int nt = p.rows <= 8 ? 1 : 2;
    const size_t smem = (size_t)8 * nt * (kLogitsPitch + (ZEROS ? kLogitsCols / 32 * 4 : 0));
    void (*fn)(HeadLogits, bool) = nt == 1 ? k_head_logits<BF16, SBF16, ZEROS, 1> : k_head_logits<BF16, SBF16, ZEROS, 2>;
    const cudaError_t e = ensure_dynamic_smem((const void *)fn, smem);
    return e != cudaSuccess ? e : launch_behind(fn, grid, 256, smem, stream, p, out_bf16);
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
    size_t bytes;
    head4_shape(b->vocab, b->width, b->group, b->has_zeros != 0, p.w, bytes);
    if (b->packed_bytes != bytes) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_logits: packed_bytes is not what stg_head_pack_bytes says for these sizes");
    const unsigned char *base = (const unsigned char *)b->packed;
    p.w.codes = base;
    p.w.scales = base + (size_t)p.w.scales;
    if (b->has_zeros) p.w.zeros = base + (size_t)p.w.zeros;
    p.hidden = (const uint16_t *)b->hidden; p.hidden_stride = b->hidden_stride;
    p.vec = !misaligned(b->hidden, 16) && (b->rows == 1 || b->hidden_stride % 8 == 0);
    p.rows = b->rows; p.out = b->logits; p.out_stride = b->row_stride;
    const OnDevice on(h->cfg.device);
    CK(on.error);
    using Launch = cudaError_t (*)(const HeadLogits &, bool, cudaStream_t);
    static const Launch launch[2][2][2] = {{{launch_logits<false, false, false>, launch_logits<false, false, true>}, {launch_logits<false, true, false>, launch_logits<false, true, true>}},
                                           {{launch_logits<true, false, false>, launch_logits<true, false, true>}, {launch_logits<true, true, false>, launch_logits<true, true, true>}}};
    CK(launch[b->hidden_dtype == STG_DTYPE_BF16][b->scale_dtype == STG_DTYPE_BF16][b->has_zeros != 0](p, b->logits_dtype == STG_DTYPE_BF16, stream));
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
    stg::Head4 w;
    size_t bytes;
    stg::head4_shape(vocab, width, group, has_zeros != 0, w, bytes);
    *out_bytes = bytes;
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
