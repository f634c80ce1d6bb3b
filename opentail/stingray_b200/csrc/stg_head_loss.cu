// stg_head_loss, stg_head_loss_backward: softmax cross entropy of hidden states and a head's weight, in pieces of the vocabulary.
//
// With z = cap(hidden weight^T), a row's normaliser is log(sum(exp(z))), its loss the normaliser minus z[target], and the gradient of
// z[v] is (dl + dn) exp(z[v] - normaliser) - dl [v == target], for gradients dl of the loss and dn of the normaliser.  Rows without a
// loss take no part: the others are gathered first, so that nothing is computed for them and what their hidden states
// hold reaches nothing.  The forward product keeps a maximum and a sum per row and tile; the backward forms a piece's logits
// again, rounds their gradients to the operands' 16 bits (they are probabilities times a factor: a relative error of half a step
// each, and the products' sums are fp32) and multiplies them with weight and hidden states.
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>
#include <string.h>

#include <new>

#include "stg_beam.h"
#include "stg_head.h"
#include "stg_head_gemm.cuh"
#include "stg_launch.h"

namespace stg {

// ---- which rows have a loss ----

struct HeadPrep {
    HeadWs ws;
    int rows, vocab;
    const int32_t *targets;
    const float *norms, *grad_loss, *grad_norms;  // NULL in the forward pass (grad_norms: also where there are none)
    int width, tile_m, workers, blocks, sums_rows;  // backward: for the number of splits
};

constexpr int kPrepThreads = 1024;

__global__ void __launch_bounds__(kPrepThreads) k_head_prep(const __grid_constant__ HeadPrep p)
{
    __shared__ int warp_sum[32];
    __shared__ float warp_most[32];
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    pdl_release();
    pdl_wait();
    int before = 0;
    float most = 0.f;
    for (int base = 0; base < p.rows; base += kPrepThreads) {
        const int r = base + tid;
        const int t = r < p.rows ? p.targets[r] : -1;
        const bool on = t >= 0 && t < p.vocab;
        const unsigned ballot = __ballot_sync(0xFFFFFFFFu, on);
        if (lane == 0) warp_sum[w] = __popc(ballot);
        __syncthreads();
        int ahead = 0, all = 0;
        for (int i = 0; i < 32; i++) {
            if (i < w) ahead += warp_sum[i];
            all += warp_sum[i];
        }
        const int at = before + ahead + __popc(ballot & ((1u << lane) - 1u));
        if (r < p.rows) p.ws.place[r] = on ? at : t < 0 ? -1 : -2;
        if (on) {
            HeadRow row = {r, t, 0.f, 0.f, 0.f, 0};
            if (p.norms) {
                row.b = p.grad_loss[r];
                row.a = row.b + (p.grad_norms ? p.grad_norms[r] : 0.f);
                row.norm = p.norms[r];
                most = fmaxf(most, fmaxf(fabsf(row.a), fabsf(row.b)));
            }
            p.ws.rows[at] = row;
        }
        before += all;
        __syncthreads();
    }
    // Up to 64 rows have room for as many more in the one row of tiles that they take.  They get what the rounding of the logits' gradients
    // leaves, as rows of their own, at no cost: a row's largest gradient is its target's, and its rounding shows in both results
    // (one row: up to 2^-8 of them).
    const int low = p.norms && p.rows <= kLowRows ? before : 0;
    if (low > 0) {
        __syncthreads();
        if (tid < low) {
            HeadRow row = p.ws.rows[tid];
            row.low = 1;
            p.ws.rows[low + tid] = row;
        }
        before += low;
    }
    for (int i = before + tid; i < (before + kHeadTileM - 1) / kHeadTileM * kHeadTileM; i += kPrepThreads) p.ws.rows[i] = HeadRow{-1, -1, 0.f, 0.f, 0.f, 0};
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
    if (lane == 0) warp_most[w] = most;
    __syncthreads();
    if (w == 1 && p.norms) {
        // few tiles of the hidden states' gradients: pieces of the vocabulary are split, so that the tiles' parts fill the chip
        const int tiles = (before + p.tile_m - 1) / p.tile_m * ((p.width + 255) / 256), slab = (before + kHeadTileM - 1) / kHeadTileM * kHeadTileM;
        uint64_t least = ~0ull;
        for (int n = lane + 1; n <= kMostSplits; n += 32)
            if (n == 1 || (n <= p.blocks && (int64_t)n * slab <= p.sums_rows)) {
                // waves of tiles times their blocks, and some sixteen blocks' time for a tile's sums to be written and read (with six, 819 rows of
                // 2048 x 151,936 were split in nine in place of two: fuller waves, but 1.59 ms in place of 1.55 at the card's power limit)
                const uint32_t cost = (uint32_t)((tiles * n + p.workers - 1) / p.workers) * (uint32_t)((p.blocks + n - 1) / n + 16);
                least = min(least, (uint64_t)cost << 32 | (uint32_t)n);
            }
        for (int o = 16; o > 0; o >>= 1) least = min(least, __shfl_xor_sync(0xFFFFFFFFu, least, o));
        if (lane == 0) p.ws.info->splits = (int)(uint32_t)least;
    }
    if (tid == 0) {
        for (int i = 1; i < 32; i++) most = fmaxf(most, warp_most[i]);
        // the largest factor comes to lie in [2^13, 2^14): a gradient of a logit is at most the sum of two, and fits
        // fp16, of whose range the small ones then use as much as there is
        int e = 0;
        if (most > 0.f && most < CUDART_INF_F) e = max(-110, min(110, 13 - ilogbf(most)));
        p.ws.info->used = before;
        p.ws.info->low = low;
        p.ws.info->scale = exp2f((float)e);
        p.ws.info->unscale = exp2f((float)-e);
    }
}

// Hidden states of the rows that have a loss, next to each other, zeros behind them up to whole tiles.
__global__ void __launch_bounds__(128) k_head_gather(const __grid_constant__ HeadWs ws, const uint16_t *hidden, int64_t stride, int width, bool vec, bool order, int vocab)
{
    pdl_release();
    pdl_wait();
    const int c = blockIdx.x, used = ws.info->used;
    if (order)  // no row has a target yet (k_head_order)
        for (int64_t i = (int64_t)c * 128 + threadIdx.x; i < vocab; i += (int64_t)gridDim.x * 128) ws.first[i] = -1;
    if (c >= (used + kHeadTileM - 1) / kHeadTileM * kHeadTileM) return;
    uint4 *to = (uint4 *)((uint16_t *)ws.hidden + (int64_t)c * width);
    const uint16_t *from = c < used ? hidden + (int64_t)ws.rows[c].row * stride : nullptr;
    for (int i = threadIdx.x; i < width / 8; i += 128) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (from && vec) {
            v = ((const uint4 *)from)[i];  // (not as read-only data: a kernel ahead may still have been writing it when this one began)
        } else if (from) {
            uint32_t e[8];
#pragma unroll
            for (int j = 0; j < 8; j++) e[j] = from[8 * i + j];
            v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        }
        to[i] = v;
    }
}

// The used rows by their targets, whose gradients are added to the weight's apart: a row's place is the number of rows with a smaller target and of those
// ahead of it with its own.  Four threads to a row look through all rows, 4096 at a time in shared memory.
constexpr int kOrderThreads = 256, kOrderRows = 4096;

__global__ void __launch_bounds__(kOrderThreads) k_head_order(const __grid_constant__ HeadWs ws)
{
    __shared__ int4 targets[kOrderRows / 4];
    pdl_release();
    pdl_wait();
    const int used = ws.info->used, first = blockIdx.x * (kOrderThreads / 4), r = first + threadIdx.x / 4, part = threadIdx.x & 3;
    if (ws.info->low > 0 || first >= used) return;
    const int mine = r < used ? ws.rows[r].target : -1;
    int smaller = 0, ahead = 0, behind = 0;  // rows with a smaller target, and those with this one ahead of the row and behind it
    for (int from = 0; from < used; from += kOrderRows) {
        __syncthreads();
        for (int i = threadIdx.x; i < kOrderRows; i += kOrderThreads) ((int *)targets)[i] = from + i < used ? ws.rows[from + i].target : 0x7FFFFFFF;
        __syncthreads();
        const int n = (min(kOrderRows, used - from) + 3) / 4, at = r - from, own = at >> 2;  // the row itself is number `at`, if it is among these
        auto count = [&](int begin, int end, int &same) {
            int less[4] = {0, 0, 0, 0}, equal[4] = {0, 0, 0, 0};
#pragma unroll 4
            for (int i = begin + ((part - begin) & 3); i < end; i += 4) {
                const int4 t = targets[i];
                less[0] += t.x < mine; equal[0] += t.x == mine;
                less[1] += t.y < mine; equal[1] += t.y == mine;
                less[2] += t.z < mine; equal[2] += t.z == mine;
                less[3] += t.w < mine; equal[3] += t.w == mine;
            }
            smaller += (less[0] + less[1]) + (less[2] + less[3]);
            same += (equal[0] + equal[1]) + (equal[2] + equal[3]);
        };
        count(0, min(max(own, 0), n), ahead);
        count(max(own + 1, 0), n, behind);
        if (own >= 0 && own < n) {
            const int i = 4 * own + part, t = ((const int *)targets)[i];
            smaller += t < mine;
            ahead += t == mine && i < at;
            behind += t == mine && i > at;
        }
    }
    for (int o = 1; o < 4; o *= 2) {
        smaller += __shfl_xor_sync(0xFFFFFFFFu, smaller, o);
        ahead += __shfl_xor_sync(0xFFFFFFFFu, ahead, o);
        behind += __shfl_xor_sync(0xFFFFFFFFu, behind, o);
    }
    if (r >= used || part != 0) return;
    ws.order[smaller + ahead] = r;
    if (ahead > 0) return;
    ws.first[mine] = smaller;
    ws.count[smaller] = 1 + behind;
}

// A row's maxima and sums joined: its normaliser and loss.  `targets`: the rows are the caller's own, else they have been gathered.
__global__ void __launch_bounds__(128) k_head_join(const __grid_constant__ HeadWs ws, int pieces, const int32_t *targets, int vocab, float *loss, float *norms)
{
    __shared__ float tops[4];
    __shared__ double sums[4];
    pdl_release();
    pdl_wait();
    const int r = blockIdx.x, tid = threadIdx.x, at = !targets ? ws.place[r] : targets[r] < 0 ? -1 : targets[r] >= vocab ? -2 : r;
    if (at < 0) {
        if (tid == 0) loss[r] = norms[r] = at == -1 ? 0.f : CUDART_NAN_F;
        return;
    }
    const float2 *parts = ws.parts + (int64_t)at * pieces;
    // each thread joins its own as they come, eight at a time; they are joined relative to the largest of all then.  A NaN sum stays.
    float top = -CUDART_INF_F;
    double sum = 0.0;
    for (int base = tid; base < pieces; base += 8 * 128) {
        float2 v[8];
        float most = top;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = base + i * 128 < pieces ? parts[base + i * 128] : make_float2(-CUDART_INF_F, 0.f);
#pragma unroll
        for (int i = 0; i < 8; i++) most = fmaxf(most, v[i].x);
        const float ref = most > -CUDART_INF_F ? most : 0.f;
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) part += v[i].y * expf(v[i].x - ref);
        sum = (top > -CUDART_INF_F ? sum * (double)expf(top - ref) : sum) + (double)part;
        top = most;
    }
    float all = top;
    for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, o));
    if ((tid & 31) == 0) tops[tid >> 5] = all;
    __syncthreads();
    all = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    if (top > -CUDART_INF_F) sum *= (double)expf(top - all);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if ((tid & 31) == 0) sums[tid >> 5] = sum;
    __syncthreads();
    if (tid == 0) {
        const double rest = log(sums[0] + sums[1] + sums[2] + sums[3]);
        norms[r] = (float)((double)all + rest);
        loss[r] = (float)((double)all - (double)ws.hit[at] + rest);  // what the target lacks to the largest logit, exactly, and nothing of either's size
    }
}

// Gradients of the hidden states: the splits' sums added up and rounded, back in their rows; zeros where a row has no loss.  Where the logits'
// gradients have no remainders of their own, the target's - the largest of a row, mostly - is multiplied here (rounded like the others it made a bf16
// gradient 2.4e-3 off in place of 1.7e-3, which is its own rounding).  A CTA has 256 columns
// of a row, and eight threads share out the splits of each eight columns.
template <bool BF16>
__global__ void __launch_bounds__(256) k_head_spread(const __grid_constant__ HeadWs ws, int width, const uint16_t *weight, int64_t weight_stride,
                                                              uint16_t *out)
{
    __shared__ float4 parts[8][32][2];
    pdl_release();
    pdl_wait();
    const int r = blockIdx.x, at = ws.place[r], splits = ws.info->splits, tid = threadIdx.x & 31, w = threadIdx.x >> 5, col = blockIdx.y * 256 + tid * 8;
    const float unscale = ws.info->unscale;
    const int64_t slab = (int64_t)((ws.info->used + kHeadTileM - 1) / kHeadTileM * kHeadTileM) * width;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
    const int low = ws.info->low;
    for (int part = 0; at >= 0 && col < width && part < (low > 0 ? 2 : 1); part++) {  // the row's, and its remainders'
        const float *from = ws.sums + (int64_t)(at + part * low) * width + col;
#pragma unroll 4
        for (int s = w; s < splits; s += 8) {
            const float4 u = *(const float4 *)(from + s * slab), v = *(const float4 *)(from + s * slab + 4);
            x.x += u.x; x.y += u.y; x.z += u.z; x.w += u.w;
            y.x += v.x; y.y += v.y; y.z += v.z; y.w += v.w;
        }
    }
    if (splits > 1) {
        parts[w][tid][0] = x;
        parts[w][tid][1] = y;
        __syncthreads();
        for (int i = 1; w == 0 && i < min(8, splits); i++) {
            const float4 u = parts[i][tid][0], v = parts[i][tid][1];
            x.x += u.x; x.y += u.y; x.z += u.z; x.w += u.w;
            y.x += v.x; y.y += v.y; y.z += v.z; y.w += v.w;
        }
    }
    if (w == 0 && at >= 0 && low == 0 && col < width) {
        const float rest = ws.hit[at];
        const uint4 t = *(const uint4 *)(weight + (int64_t)ws.rows[at].target * weight_stride + col);
        x.x = fmaf(rest, half_of<BF16>(t.x), x.x); x.y = fmaf(rest, half_of<BF16>(t.x >> 16), x.y);
        x.z = fmaf(rest, half_of<BF16>(t.y), x.z); x.w = fmaf(rest, half_of<BF16>(t.y >> 16), x.w);
        y.x = fmaf(rest, half_of<BF16>(t.z), y.x); y.y = fmaf(rest, half_of<BF16>(t.z >> 16), y.y);
        y.z = fmaf(rest, half_of<BF16>(t.w), y.z); y.w = fmaf(rest, half_of<BF16>(t.w >> 16), y.w);
    }
    if (w == 0 && col < width)
        *(uint4 *)(out + (int64_t)r * width + col) = make_uint4(pack2<BF16>(x.x * unscale, x.y * unscale), pack2<BF16>(x.z * unscale, x.w * unscale),
                                                                pack2<BF16>(y.x * unscale, y.y * unscale), pack2<BF16>(y.z * unscale, y.w * unscale));
}

// ---- host ----

// Offsets of the workspace; `base` NULL: only its size.
static HeadWs head_layout(const StgHeadLoss *b, bool backward, HeadPlan &p, char *base)
{
    HeadWs ws;
    memset(&ws, 0, sizeof(ws));
    size_t at = 0;
    auto take = [&](size_t bytes) { char *x = base ? base + at : nullptr; at += round_up(bytes, 256); return x; };
    const size_t R = (size_t)p.rows_pad;
    ws.info = (HeadInfo *)take(sizeof(HeadInfo));
    ws.rows = (HeadRow *)take(R * sizeof(HeadRow));
    ws.place = (int32_t *)take(R * 4);
    ws.hidden = take(R * (size_t)b->width * 2);
    ws.hit = (float *)take(R * 4);
    if (backward) {
        ws.grads = take(R * (size_t)p.grads_stride * 2);
        ws.sums = (float *)take((size_t)p.sums_rows * (size_t)b->width * 4);
        if (b->rows > kLowRows) {
            ws.first = (int32_t *)take((size_t)b->vocab * 4);
            ws.order = (int32_t *)take(R * 4);
            ws.count = (int32_t *)take(R * 4);
        }
    } else {
        ws.parts = (float2 *)take(R * 2 * (size_t)p.tiles_n * sizeof(float2));
    }
    p.bytes = at;
    return ws;
}

static HeadPlan head_plan(StgHandle h, const StgHeadLoss *b, bool backward)
{
    HeadPlan p = head_shape(b->rows, b->vocab, b->width, h->sm_count, backward);
    head_layout(b, backward, p, nullptr);
    return p;
}

static int head_check(StgHandle h, const StgHeadLoss *b, const char *who)
{
    const std::string at = std::string(who) + ": ";
    if (!b || b->struct_size != (int32_t)sizeof(StgHeadLoss)) return fail(h, STG_ERR_INVALID_ARGUMENT, "bad StgHeadLoss");
    if (b->rows < 0 || b->vocab <= 0 || b->width <= 0) return fail(h, STG_ERR_INVALID_ARGUMENT, at + "rows must be >= 0, vocab and width > 0");
    if (b->rows > (1 << 20) || b->vocab > (1 << 26) || b->width > (1 << 16)) return fail(h, STG_ERR_CAPACITY, at + "more than 2^20 rows, 2^26 vocabulary entries or a width of 2^16");
    if (b->dtype != STG_DTYPE_BF16 && b->dtype != STG_DTYPE_F16) return fail(h, STG_ERR_INVALID_ARGUMENT, at + "dtype must be STG_DTYPE_BF16 or STG_DTYPE_F16");
    if (b->width % 8 != 0) return fail(h, STG_ERR_UNSUPPORTED, at + "width must be a multiple of 8");
    if (b->hidden_stride < b->width || b->weight_stride < b->width) return fail(h, STG_ERR_INVALID_ARGUMENT, at + "a row stride smaller than width");
    if (!(b->logit_softcap >= 0.f) || b->logit_softcap > 3.0e38f) return fail(h, STG_ERR_INVALID_ARGUMENT, at + "logit_softcap must be 0 (off) or a finite positive cap");
    return STG_OK;
}

static int head_check_arrays(StgHandle h, const StgHeadLoss *b, const char *who, bool backward, const HeadPlan &p)
{
    const std::string at = std::string(who) + ": ";
    if (!b->hidden || !b->weight || !b->targets || !b->log_norms || (!backward && !b->loss) || (backward && !b->grad_loss))
        return fail(h, STG_ERR_INVALID_ARGUMENT, at + "hidden, weight, targets, log_norms and loss (backward: grad_loss) are required");
    if (misaligned(b->hidden, 2) || misaligned(b->targets, 4) || misaligned(b->log_norms, 4) || misaligned(b->loss, 4) || misaligned(b->grad_loss, 4) ||
        misaligned(b->grad_log_norms, 4) || misaligned(b->grad_hidden, 16) || misaligned(b->grad_weight, 16))
        return fail(h, STG_ERR_INVALID_ARGUMENT, at + "an array is not aligned to its elements, or a gradient not to 16 bytes");
    if (misaligned(b->weight, 16) || b->weight_stride % 8 != 0) return fail(h, STG_ERR_UNSUPPORTED, at + "the weight's rows must begin at 16 bytes");
    if (!b->workspace || misaligned(b->workspace, 256) || b->workspace_bytes < p.bytes)
        return fail(h, STG_ERR_CAPACITY, at + "workspace missing, not aligned to 256 bytes or smaller than stg_head_loss_workspace says");
    return STG_OK;
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                 const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int head_map_of(StgHandle h, CUtensorMap *map, CUtensorMapDataType type, int dims, const void *p, const cuuint64_t *size, const cuuint64_t *stride, const cuuint32_t *box,
                CUtensorMapSwizzle swizzle)
{
    static const EncodeTiled encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) fn = nullptr;
        return (EncodeTiled)fn;
    }();
    if (!encode) return fail(h, STG_ERR_CUDA, "cuTensorMapEncodeTiled is not there");
    const cuuint32_t step[3] = {1, 1, 1};
    const CUresult e = encode(map, type, (cuuint32_t)dims, (void *)p, size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return e == CUDA_SUCCESS ? STG_OK : fail(h, STG_ERR_CUDA, "cuTensorMapEncodeTiled failed with " + std::to_string((int)e));
}

// A map of 16-bit rows: boxes of 64 columns (128 bytes, swizzled) by `box_rows` rows.
static int head_map(StgHandle h, CUtensorMap *map, bool bf16, const void *p, int64_t columns, int64_t rows, int64_t stride, int box_rows)
{
    const cuuint64_t size[2] = {(cuuint64_t)columns, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
    return head_map_of(h, map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, p, size, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int MODE, bool LONG>
static cudaError_t head_gemm(StgHandle h, bool bf16, bool pair, cudaStream_t stream, const CUtensorMap &a, const CUtensorMap &b, const CUtensorMap &out,
                             HeadGemm g, int64_t tiles)
{
    using Kernel = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, HeadGemm);
    constexpr bool C = MODE == kStats || MODE == kGrad;  // the others have no soft cap
    constexpr bool S = !(MODE == kWeight && LONG);       // so many rows are pairs'
    static const Kernel kernels[2][2][2] = {
        {{k_head_gemm<MODE, false, false, !S, LONG>, k_head_gemm<MODE, false, false, true, LONG>}, {k_head_gemm<MODE, false, C, !S, LONG>, k_head_gemm<MODE, false, C, true, LONG>}},
        {{k_head_gemm<MODE, true, false, !S, LONG>, k_head_gemm<MODE, true, false, true, LONG>}, {k_head_gemm<MODE, true, C, !S, LONG>, k_head_gemm<MODE, true, C, true, LONG>}}};
    const Kernel fn = kernels[bf16][g.cap != 0.f][pair];
    const GemmRing ring = gemm_ring(MODE, pair, g.tile_n, g.a_rows);
    g.a_at = ring.a_at; g.stage_bytes = ring.stage_bytes; g.stages = ring.stages;
    const size_t smem = 1024 + kGemmRingBytes + (MODE == kStats ? 0 : kGemmEpiWarps * kGemmOut);
    const cudaError_t e = ensure_dynamic_smem((const void *)fn, smem);
    if (e != cudaSuccess) return e;
    h->stats.kernel_launches++;
    const int ctas = pair ? 2 : 1;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = 2;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(ctas * std::max<int64_t>(1, std::min<int64_t>(tiles, h->sm_count / ctas))));
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = at;
    cfg.numAttrs = pair ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, fn, a, b, out, g);
}

static bool head_rows_aligned(const StgHeadLoss *b) { return !misaligned(b->hidden, 16) && (b->rows == 1 || b->hidden_stride % 8 == 0); }

static int head_begin(StgHandle h, const StgHeadLoss *b, const HeadWs &ws, const HeadPlan &p, bool backward, bool order, cudaStream_t stream)
{
    const HeadPrep prep = {ws, b->rows, b->vocab, b->targets, backward ? b->log_norms : nullptr, b->grad_loss, b->grad_log_norms,
                           b->width, p.tile_m, h->sm_count * kHeadTileM / p.tile_m, (p.piece + kGemmK - 1) / kGemmK, p.sums_rows};
    CK(launch_behind(k_head_prep, dim3(1), kPrepThreads, 0, stream, prep));
    CK(launch_behind(k_head_gather, dim3((unsigned)p.rows_pad), 128, 0, stream, ws, (const uint16_t *)b->hidden, b->hidden_stride, b->width, head_rows_aligned(b), order,
                     b->vocab));
    h->stats.kernel_launches += 2;
    if (order) {
        CK(launch_behind(k_head_order, dim3((unsigned)(p.rows_pad + kOrderThreads / 4 - 1) / (kOrderThreads / 4)), kOrderThreads, 0, stream, ws));
        h->stats.kernel_launches++;
    }
    return STG_OK;
}

// Tiles are taken in groups of rows, so that what runs at a time reads few rows and columns over and over in L2: 8192 x 4096 x 151,936 in
// 7.9 ms with groups of 16 x 256 rows, 8.3 with all rows, 8.5 with 6; its gradients' products over pieces of 15,360 with groups of 8 in
// 24.5 ms, 27.6 with all rows.
constexpr int kGroupLogits = 16, kGroupGrads = 8;

static int head_box_rows(int rows) { return std::min(kHeadTileM, (rows + 7) / 8 * 8); }

static HeadGemm head_args(const StgHeadLoss *b, const HeadWs &ws, const HeadPlan &p)
{
    HeadGemm g;
    memset(&g, 0, sizeof(g));
    g.info = ws.info; g.rows = ws.rows; g.rows_pad = p.rows_pad; g.tile_n = p.tile_n; g.group = kGroupLogits; g.cap = b->logit_softcap;
    g.a_rows = head_box_rows(b->rows);  // backward: twice as many, below
    return g;
}

static int head_forward(StgHandle h, const StgHeadLoss *b, cudaStream_t stream)
{
    int rc = head_check(h, b, "stg_head_loss");
    if (rc || b->rows == 0) return rc;
    HeadPlan p = head_plan(h, b, false);
    rc = head_check_arrays(h, b, "stg_head_loss", false, p);
    if (rc) return rc;
    const OnDevice on(h->cfg.device);
    CK(on.error);
    const HeadWs ws = head_layout(b, false, p, (char *)b->workspace);
    const bool bf16 = b->dtype == STG_DTYPE_BF16;
    // one row of tiles takes no less time for fewer rows: they are read where they are
    const bool direct = !p.pair && head_rows_aligned(b);
    CUtensorMap rows, weight;
    if ((rc = direct ? head_map(h, &rows, bf16, b->hidden, b->width, b->rows, b->rows == 1 ? b->width : b->hidden_stride, head_box_rows(b->rows))
                     : head_map(h, &rows, bf16, ws.hidden, b->width, p.rows_pad, b->width, head_box_rows(b->rows)))) return rc;
    if ((rc = head_map(h, &weight, bf16, b->weight, b->width, b->vocab, b->weight_stride, p.pair ? p.tile_n / 2 : p.tile_n))) return rc;
    if (!direct && (rc = head_begin(h, b, ws, p, false, false, stream))) return rc;
    HeadGemm g = head_args(b, ws, p);
    g.targets = direct ? b->targets : nullptr; g.used_rows = b->rows;
    g.n = b->vocab; g.k = b->width;
    g.parts = ws.parts; g.hit = ws.hit; g.pieces = 2 * p.tiles_n;
    CK((head_gemm<kStats, false>(h, bf16, p.pair, stream, rows, weight, rows, g, (int64_t)((b->rows + p.tile_m - 1) / p.tile_m) * p.tiles_n)));
    CK(launch_behind(k_head_join, dim3((unsigned)b->rows), 128, 0, stream, ws, 2 * p.tiles_n, g.targets, b->vocab, b->loss, b->log_norms));
    h->stats.kernel_launches++;
    h->stats.calls++;
    return STG_OK;
}

static int head_backward(StgHandle h, const StgHeadLoss *b, cudaStream_t stream)
{
    int rc = head_check(h, b, "stg_head_loss_backward");
    if (rc) return rc;
    if (!b->grad_hidden && !b->grad_weight) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_loss_backward: neither grad_hidden nor grad_weight");
    const OnDevice on(h->cfg.device);
    CK(on.error);
    const size_t weight_bytes = (size_t)b->vocab * b->width * 2;
    if (b->rows == 0) {
        if (b->grad_weight) CK(cudaMemsetAsync(b->grad_weight, 0, weight_bytes, stream));
        return STG_OK;
    }
    HeadPlan p = head_plan(h, b, true);
    rc = head_check_arrays(h, b, "stg_head_loss_backward", true, p);
    if (rc) return rc;
    const HeadWs ws = head_layout(b, true, p, (char *)b->workspace);
    const bool bf16 = b->dtype == STG_DTYPE_BF16;
    CUtensorMap rows_k, weight_k, grads_k, weight_mn, grads_mn, rows_mn;  // how the operands' boxes of 64 columns are cut
    CUtensorMap grads_out, sums_out, weight_out;                          // results: boxes of 32 rows
    const int box_rows = head_box_rows(2 * b->rows);  // with the remainders'
    if ((rc = head_map(h, &rows_k, bf16, ws.hidden, b->width, p.rows_pad, b->width, box_rows))) return rc;
    if ((rc = head_map(h, &weight_k, bf16, b->weight, b->width, b->vocab, b->weight_stride, p.pair ? p.tile_n / 2 : p.tile_n))) return rc;
    if ((rc = head_map(h, &weight_mn, bf16, b->weight, b->width, b->vocab, b->weight_stride, kGemmK))) return rc;
    if ((rc = head_map(h, &rows_mn, bf16, ws.hidden, b->width, p.rows_pad, b->width, kGemmK))) return rc;
    if (b->grad_hidden) {
        const cuuint64_t size[2] = {(cuuint64_t)b->width, (cuuint64_t)p.sums_rows}, stride[1] = {(cuuint64_t)b->width * 4};
        const cuuint32_t box[2] = {32, 32};
        if ((rc = head_map_of(h, &sums_out, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, ws.sums, size, stride, box, CU_TENSOR_MAP_SWIZZLE_128B))) return rc;
    }
    const bool order = b->grad_weight && ws.first;
    if ((rc = head_begin(h, b, ws, p, true, order, stream))) return rc;
    const int64_t tiles_m = (p.rows_pad + p.tile_m - 1) / p.tile_m, tiles_w = (b->width + 255) / 256;
    for (int i = 0; i < p.pieces; i++) {
        const int first = i * p.piece, count = std::min(p.piece, b->vocab - first);
        // what lies behind the piece's columns is read as zeros
        if ((rc = head_map(h, &grads_k, bf16, ws.grads, count, p.rows_pad, p.grads_stride, kHeadTileM))) return rc;
        if ((rc = head_map(h, &grads_mn, bf16, ws.grads, count, p.rows_pad, p.grads_stride, kGemmK))) return rc;
        if ((rc = head_map(h, &grads_out, bf16, ws.grads, count, p.rows_pad, p.grads_stride, 32))) return rc;
        HeadGemm g = head_args(b, ws, p);
        g.first = first;
        g.n = count; g.k = b->width; g.a_rows = box_rows;
        g.out = ws.grads; g.out_stride = p.grads_stride; g.hit = ws.hit;
        CK(((b->width > part_of(kGradColumns, bf16) ? head_gemm<kGrad, true> : head_gemm<kGrad, false>)(h, bf16, p.pair, stream, rows_k, weight_k, grads_out, g, tiles_m * ((count + p.tile_n - 1) / p.tile_n))));
        g.n = b->width; g.tile_n = 256; g.group = kGroupGrads; g.cap = 0.f;
        if (b->grad_hidden) {
            g.k = count; g.a_rows = kHeadTileM;
            g.out = ws.sums; g.out_stride = b->width;
            CK((head_gemm<kHidden, false>(h, bf16, p.pair, stream, grads_k, weight_mn, sums_out, g, tiles_m * tiles_w * 64)));
        }
        if (b->grad_weight) {
            g.m = count;
            g.first_of = order ? ws.first : nullptr; g.order = ws.order; g.count = ws.count; g.hidden = (const uint16_t *)ws.hidden;
            g.out = b->grad_weight; g.out_stride = b->width;
            if ((rc = head_map(h, &weight_out, bf16, b->grad_weight, b->width, first + count, b->width, 32))) return rc;
            const bool in_parts = b->rows > part_of(kWeightRows, bf16);
            if (in_parts) g.tile_n = 128;
            CK(((in_parts ? head_gemm<kWeight, true> : head_gemm<kWeight, false>)(h, bf16, p.pair, stream, grads_mn, rows_mn, weight_out, g,
                                                                                 (int64_t)((count + p.tile_m - 1) / p.tile_m) * ((b->width + g.tile_n - 1) / g.tile_n))));
        }
    }
    if (b->grad_hidden) {
        CK(launch_behind(bf16 ? k_head_spread<true> : k_head_spread<false>, dim3((unsigned)b->rows, (unsigned)(b->width + 255) / 256), 256, 0, stream, ws, b->width, (const uint16_t *)b->weight, b->weight_stride,
                         (uint16_t *)b->grad_hidden));
        h->stats.kernel_launches++;
    }
    h->stats.calls++;
    return STG_OK;
}

}  // namespace stg

extern "C" {

int stg_head_loss_workspace(StgHandle h, const StgHeadLoss *loss, int32_t backward, uint64_t *out_bytes)
try {
    if (!h) return STG_ERR_INVALID_ARGUMENT;
    const int rc = stg::head_check(h, loss, "stg_head_loss_workspace");
    if (rc) return rc;
    if (!out_bytes) return stg::fail(h, STG_ERR_INVALID_ARGUMENT, "stg_head_loss_workspace: out_bytes is required");
    *out_bytes = stg::head_plan(h, loss, backward != 0).bytes;
    return STG_OK;
} catch (const std::bad_alloc &) {
    return STG_ERR_CAPACITY;
}

int stg_head_loss(StgHandle h, const StgHeadLoss *loss, void *stream)
try {
    return h ? stg::head_forward(h, loss, (cudaStream_t)stream) : STG_ERR_INVALID_ARGUMENT;
} catch (const std::bad_alloc &) {
    return STG_ERR_CAPACITY;
}

int stg_head_loss_backward(StgHandle h, const StgHeadLoss *loss, void *stream)
try {
    return h ? stg::head_backward(h, loss, (cudaStream_t)stream) : STG_ERR_INVALID_ARGUMENT;
} catch (const std::bad_alloc &) {
    return STG_ERR_CAPACITY;
}

}  // extern "C"
