// stg_beam_select: the best continuations of every sequence over its beams and the vocabulary.
//
// With x the logits of beam k, m their maximum and S = sum exp(x - m), candidate (k, v) scores
//     score[k] + ((x[v] - m) - log S)
// in 64 bits.  Within a beam the order is that of the logits alone, so a row is read once: a running maximum, a
// running sum, and the list of its best logits as 64-bit keys (stg_select.cuh); the scores are made for the few
// that are left when a sequence's rows come together.  The terms of S are computed and added up in 32 bits over the 16 or
// 32 elements that a thread holds, in 64 beyond: their roundings (1e-7 each, either way) leave about 1e-8 of S, so two
// beams' candidates change places only if they lie closer than that.
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>
#include <string.h>

#include <new>

#include "stg_beam.h"
#include "stg_select.cuh"
#include "stg_types.h"

namespace stg {

constexpr int kBeamThreads = 256;
constexpr int kBeamList = 1024;  // entries of a list in shared memory, a power of two
// the key of -infinity at token 0 .. : what is no candidate lies at or below it
constexpr u64 kNoKey = ((u64)0x007FFFFFu << 32) | 0xFFFFFFFFu;

struct BeamSelect {
    const void *logits;
    int64_t row_stride;
    const float *scores;
    const uint32_t *mask;
    int64_t mask_stride;
    const uint8_t *uses_mask;
    float softcap;
    int32_t n_seq, beams, vocab, n;
    int32_t pieces, piece_len;
    BeamWs ws;
    int32_t *tokens, *parents;
    float *out_scores, *log_norms;
    uint32_t *flags;
};

// How a thread reads its share of a tile: U loads of E elements.  VEC: 16 bytes each, element e of load u is
// (u * 256 + thread) * E + e of the tile; else single elements, (u * E + e) * 256 + thread.
template <bool BF16, bool VEC>
struct BeamTile {
    static constexpr int E = BF16 ? 8 : 4;
    static constexpr int U = 4;
    static constexpr int kLen = kBeamThreads * U * E;
    static __device__ __forceinline__ int at(int u, int e)
    {
        return VEC ? (u * kBeamThreads + (int)threadIdx.x) * E + e : (u * E + e) * kBeamThreads + (int)threadIdx.x;
    }
};

// elements at(u, 0 ..) of the tile that starts at `base`; masked ones and those at or beyond `end` read as -infinity
template <bool BF16, bool VEC>
static __device__ __forceinline__ void beam_load(const LogitRow row, const uint32_t *mrow, int base, int end, int u, float *v)
{
    typedef BeamTile<BF16, VEC> T;
    const int i = base + T::at(u, 0);
    if (VEC && i + T::E <= end) {
        if constexpr (BF16) {
            const uint4 t = __ldcs((const uint4 *)((const uint16_t *)row.p + i));
            v[0] = bf16_lo(t.x); v[1] = bf16_hi(t.x); v[2] = bf16_lo(t.y); v[3] = bf16_hi(t.y);
            v[4] = bf16_lo(t.z); v[5] = bf16_hi(t.z); v[6] = bf16_lo(t.w); v[7] = bf16_hi(t.w);
        } else {
            const float4 t = __ldcs((const float4 *)((const float *)row.p + i));
            v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        }
        if (row.cap != 0.f)
#pragma unroll
            for (int e = 0; e < T::E; e++) v[e] = soft_cap(v[e], row.cap);
    } else {
#pragma unroll
        for (int e = 0; e < T::E; e++) {
            const int j = base + T::at(u, e);
            v[e] = j < end ? load_one<BF16>(row, j) : -CUDART_INF_F;
        }
    }
    if (mrow != nullptr)
#pragma unroll
        for (int e = 0; e < T::E; e++) {
            const int j = base + T::at(u, e);
            if (j < end && !mask_bit(mrow, j)) v[e] = -CUDART_INF_F;
        }
}

// Sorts the first `cnt` entries of `list` descending (bitonic, padded with zeros: no key is 0).  All threads.
static __device__ void sort_list(u64 *list, int cnt)
{
    int len = 32;
    while (len < cnt) len <<= 1;
    for (int i = cnt + threadIdx.x; i < len; i += kBeamThreads) list[i] = 0ull;
    __syncthreads();
    for (int k = 2; k <= len; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int t = threadIdx.x; t < len / 2; t += kBeamThreads) {
                const int a = 2 * j * (t / j) + t % j, b = a + j;
                const u64 x = list[a], y = list[b];
                if ((x < y) == ((a & k) == 0)) { list[a] = y; list[b] = x; }
            }
            __syncthreads();
        }
}

// One piece of a row: its maximum, its sum and its n best logits.
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(kBeamThreads) k_beam_rows(const __grid_constant__ BeamSelect a)
{
    typedef BeamTile<BF16, VEC> T;
    __shared__ u64 list[kBeamList];
    __shared__ int cnt, want;
    __shared__ u64 thr;                       // later elements belong to the n best only above this key
    __shared__ uint32_t tops[kBeamThreads];   // the threads' largest logits of the first tile
    __shared__ float red_m[kBeamThreads / 32];
    __shared__ double red_s[kBeamThreads / 32];
    const int row = blockIdx.y, piece = blockIdx.x, tid = threadIdx.x;
    const float score = a.scores[row];
    if (!(score > -CUDART_INF_F && score < CUDART_INF_F)) return;  // a dead beam
    const LogitRow lr{(const char *)a.logits + (int64_t)row * a.row_stride * (BF16 ? 2 : 4), a.softcap};
    const uint32_t *mrow = a.mask != nullptr && (a.uses_mask == nullptr || a.uses_mask[row]) ? a.mask + (int64_t)row * a.mask_stride : nullptr;
    const int begin = piece * a.piece_len, end = min(a.vocab, begin + a.piece_len);
    const int n = a.n;
    if (tid == 0) { cnt = 0; want = 0; thr = kNoKey; }
    __syncthreads();
    float m = -CUDART_INF_F;
    double s = 0.0;

    for (int base = begin; base < end; base += T::kLen) {
        float v[T::U][T::E];
#pragma unroll
        for (int u = 0; u < T::U; u++) beam_load<BF16, VEC>(lr, mrow, base, end, u, v[u]);
        float top = -CUDART_INF_F;
#pragma unroll
        for (int u = 0; u < T::U; u++)
#pragma unroll
            for (int e = 0; e < T::E; e++) top = fmaxf(top, v[u][e]);
        if (top > m) {
            s *= exp((double)m - (double)top);
            m = top;
        }
        // a thread that has seen nothing but -infinity (and NaN, which the sum has to show)
        const float ref = m == -CUDART_INF_F ? 0.f : m;
        float part = 0.f;
#pragma unroll
        for (int u = 0; u < T::U; u++)
#pragma unroll
            for (int e = 0; e < T::E; e++) part += expf(v[u][e] - ref);
        s += (double)part;

        if (base == begin) {
            // At least n elements are as large as the n-th largest of the threads' maxima.
            tops[tid] = ord32(top);
            __syncthreads();
            int above = 0;
            for (int t = 0; t < kBeamThreads; t++) above += tops[t] > tops[tid] || (tops[t] == tops[tid] && t < tid);
            if (above == n - 1 && top > -CUDART_INF_F) thr = (u64)tops[tid] << 32;
        }
        __syncthreads();
        u64 bound = thr;
        float low = key_val(bound);
        int hits = 0;
        if (top >= low) {
#pragma unroll
            for (int u = 0; u < T::U; u++)
#pragma unroll
                for (int e = 0; e < T::E; e++)
                    if (v[u][e] >= low && make_key(v[u][e], base + T::at(u, e)) > bound) hits++;
        }
        if (!__syncthreads_or(hits)) continue;
        if (hits) atomicAdd(&want, hits);
        __syncthreads();
        const bool fits = cnt + want <= kBeamList;
        __syncthreads();
        if (tid == 0) want = 0;
        if (fits) {
            if (hits)
#pragma unroll
                for (int u = 0; u < T::U; u++)
#pragma unroll
                    for (int e = 0; e < T::E; e++) {
                        const u64 key = make_key(v[u][e], base + T::at(u, e));
                        if (v[u][e] >= low && key > bound) list[atomicAdd(&cnt, 1)] = key;
                    }
        } else {
            // More than there is room for (a row that ascends, or one of equal logits): one element of every thread at a time.
#pragma unroll
            for (int u = 0; u < T::U; u++)
#pragma unroll
                for (int e = 0; e < T::E; e++) {
                    __syncthreads();
                    const int c = cnt;
                    __syncthreads();  // read by all before anyone appends
                    if (c > kBeamList - kBeamThreads) {
                        sort_list(list, c);
                        if (tid == 0) { cnt = min(c, n); if (c >= n) thr = list[n - 1]; }
                        __syncthreads();
                        bound = thr;
                    }
                    const u64 key = make_key(v[u][e], base + T::at(u, e));
                    if (v[u][e] >= key_val(bound) && key > bound) list[atomicAdd(&cnt, 1)] = key;
                }
        }
        __syncthreads();
        if (cnt >= n + n / 2 || cnt > kBeamList / 2) {
            const int c = cnt;
            sort_list(list, c);
            if (tid == 0) { cnt = min(c, n); if (c >= n) thr = list[n - 1]; }
        }
        __syncthreads();
    }

    const int c = cnt;
    sort_list(list, c);
    float wm = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xFFFFFFFFu, wm, o));
    if ((tid & 31) == 0) red_m[tid >> 5] = wm;
    __syncthreads();
    for (int w = 0; w < kBeamThreads / 32; w++) wm = fmaxf(wm, red_m[w]);
    // exp(-infinity - finite) is 0; a NaN sum stays NaN whatever it is multiplied by
    if (m != wm) s *= exp((double)(m == -CUDART_INF_F && wm == -CUDART_INF_F ? 0.f : m) - (double)wm);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if ((tid & 31) == 0) red_s[tid >> 5] = s;
    __syncthreads();
    const int64_t at = (int64_t)row * a.pieces + piece;
    if (tid == 0) {
        s = 0.0;
        for (int w = 0; w < kBeamThreads / 32; w++) s += red_s[w];
        a.ws.parts[at] = BeamPart{s, wm, min(c, n)};
    }
    for (int i = tid; i < min(c, n); i += kBeamThreads) a.ws.keys[at * n + i] = list[i];
}

static __device__ __forceinline__ u64 ord64(double v)
{
    const u64 b = (u64)__double_as_longlong(v + 0.0);
    return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
static __device__ __forceinline__ double unord64(u64 k)
{
    return __longlong_as_double((long long)((k >> 63) ? (k & 0x7FFFFFFFFFFFFFFFull) : ~k));
}

// The candidates of one sequence: its beams' pieces come together.
__global__ void __launch_bounds__(kBeamThreads) k_beam_merge(const __grid_constant__ BeamSelect a)
{
    __shared__ double base[STG_BEAM_MAX_BEAMS];   // score - log S of a beam, -infinity: it has no candidates
    __shared__ float top[STG_BEAM_MAX_BEAMS];     // m
    __shared__ u64 best[kBeamList], what[kBeamList];  // score and key of a candidate
    __shared__ int8_t whose[kBeamList];
    __shared__ int cnt;
    __shared__ u64 bound;                          // candidates below this score are not among the n best
    __shared__ uint32_t flags;
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
    const int K = a.beams, n = a.n, C = a.pieces;
    if (tid == 0) { cnt = 0; bound = 0ull; flags = 0u; }
    __syncthreads();
    for (int k = tid >> 5; k < K; k += kBeamThreads / 32) {
        const int row = seq * K + k;
        const float score = a.scores[row];
        const bool alive = score > -CUDART_INF_F && score < CUDART_INF_F;
        const BeamPart *parts = a.ws.parts + (int64_t)row * C;
        float m = -CUDART_INF_F;
        double s = 0.0;
        if (alive) {
            for (int c = lane; c < C; c += 32) m = fmaxf(m, parts[c].m);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            for (int c = lane; c < C; c += 32) {
                const BeamPart p = parts[c];
                s += p.m == m ? p.s : p.s * exp((double)p.m - (double)m);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        }
        if (lane == 0) {
            const bool none = m == -CUDART_INF_F && s == 0.0;        // dead, or nothing in the row
            const bool bad = !none && !(s > 0.0 && s < CUDART_INF);  // NaN or +infinity among the logits
            const double logs = log(s);
            base[k] = none || bad ? -CUDART_INF : (double)score - logs;
            top[k] = m;
            if (bad) atomicOr(&flags, STG_BEAM_BAD_ROW);
            if (alive && none) atomicOr(&flags, STG_ROW_FULLY_MASKED);
            if (a.log_norms) a.log_norms[row] = none ? -CUDART_INF_F : (float)((double)m + logs);
        }
    }
    __syncthreads();
    const int total = K * C * n;
    for (int first = 0; first < total; first += kBeamThreads) {
        const int i = first + tid;
        if (i < total) {
            const int part = i / n, j = i % n, k = part / C;
            if (base[k] > -CUDART_INF && j < a.ws.parts[(int64_t)seq * K * C + part].count) {
                const u64 key = a.ws.keys[((int64_t)seq * K * C + part) * n + j];
                const u64 s = ord64(((double)key_val(key) - (double)top[k]) + base[k]);
                if (s >= bound) {
                    const int at = atomicAdd(&cnt, 1);
                    best[at] = s; what[at] = key; whose[at] = (int8_t)k;
                }
            }
        }
        __syncthreads();
        const bool last = first + kBeamThreads >= total;
        if (cnt <= kBeamList - kBeamThreads && !last) { __syncthreads(); continue; }
        // keep the n best: every entry counts those ahead of it
        const int c = cnt;
        u64 s[kBeamList / kBeamThreads], w[kBeamList / kBeamThreads];
        int8_t k[kBeamList / kBeamThreads];
        int rank[kBeamList / kBeamThreads];
#pragma unroll
        for (int r = 0; r < kBeamList / kBeamThreads; r++) {
            const int e = r * kBeamThreads + tid;
            rank[r] = kBeamList;
            if (e >= c) continue;
            s[r] = best[e]; w[r] = what[e]; k[r] = whose[e];
            int ahead = 0;
            for (int o = 0; o < c; o++)
                ahead += best[o] > s[r] || (best[o] == s[r] && (whose[o] < k[r] || (whose[o] == k[r] && what[o] > w[r])));
            rank[r] = ahead;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kBeamList / kBeamThreads; r++)
            if (rank[r] < n) { best[rank[r]] = s[r]; what[rank[r]] = w[r]; whose[rank[r]] = k[r]; }
        __syncthreads();
        if (tid == 0) { cnt = min(c, n); if (c >= n) bound = best[n - 1]; }
        __syncthreads();
    }
    const int c = cnt;
    for (int i = tid; i < n; i += kBeamThreads) {
        const int64_t o = (int64_t)seq * n + i;
        a.tokens[o] = i < c ? key_idx(what[i]) : -1;
        a.parents[o] = i < c ? whose[i] : -1;
        a.out_scores[o] = i < c ? (float)unord64(best[i]) : -CUDART_INF_F;
    }
    if (tid == 0 && a.flags) a.flags[seq] = flags | (c < n ? (uint32_t)STG_BEAM_SHORT : 0u);
}

int beam_check_rows(StgHandle h, const char *who, int32_t n_seq, int32_t n_beams)
{
    if (n_seq < 0 || n_beams < 1) return fail(h, STG_ERR_INVALID_ARGUMENT, std::string(who) + ": n_seq must be >= 0 and n_beams >= 1");
    if (n_beams > STG_BEAM_MAX_BEAMS) return fail(h, STG_ERR_CAPACITY, std::string(who) + ": at most 32 beams per sequence");
    if ((int64_t)n_seq * n_beams > h->cfg.max_rows) return fail(h, STG_ERR_CAPACITY, std::string(who) + ": n_seq * n_beams exceeds max_rows");
    return STG_OK;
}

// Workspace of a call on a stream that is being captured: its own, since the graph may run beside anything else the handle does.
static int captured_workspace(StgHandle h, size_t bytes, void **out)
{
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // an allocation is no work of the capture
    CK(cudaThreadExchangeStreamCaptureMode(&mode));
    DevBuf b;
    const int rc = dev_alloc(nullptr, b, bytes);  // without guard bytes: they are set on a stream that cannot be used now
    const cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
    if (rc) return fail(h, rc, "stg_beam_select: no memory for a captured call's workspace");
    h->bm_captured.push_back(b);
    if (e != cudaSuccess) return cuda_fail(h, e, "cudaThreadExchangeStreamCaptureMode");
    *out = b.p;
    return STG_OK;
}

static int beam_select(StgHandle h, const StgBeamBatch *b, cudaStream_t stream)
{
    if (!b || b->struct_size != (int32_t)sizeof(StgBeamBatch)) return fail(h, STG_ERR_INVALID_ARGUMENT, "bad StgBeamBatch");
    int rc = beam_check_rows(h, "stg_beam_select", b->n_seq, b->n_beams);
    if (rc) return rc;
    if (b->vocab <= 0) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_select: vocab must be > 0");
    if (b->vocab > h->cfg.max_vocab) return fail(h, STG_ERR_CAPACITY, "vocab exceeds max_vocab");
    if (b->n_candidates < 1) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_select: n_candidates must be >= 1");
    if (b->n_candidates > STG_BEAM_MAX_CANDIDATES) return fail(h, STG_ERR_CAPACITY, "stg_beam_select: at most 128 candidates per sequence");
    if (b->logits_dtype != STG_DTYPE_F32 && b->logits_dtype != STG_DTYPE_BF16) return fail(h, STG_ERR_INVALID_ARGUMENT, "unknown logits_dtype");
    if (b->row_stride < b->vocab) return fail(h, STG_ERR_INVALID_ARGUMENT, "row_stride smaller than vocab");
    if (b->mask && b->mask_row_stride < ((int64_t)b->vocab + 31) / 32) return fail(h, STG_ERR_INVALID_ARGUMENT, "mask_row_stride too small");
    if (!(b->logit_softcap >= 0.f) || b->logit_softcap > 3.0e38f)
        return fail(h, STG_ERR_INVALID_ARGUMENT, "logit_softcap must be 0 (off) or a finite positive cap");
    if (b->n_seq == 0) return STG_OK;
    if (!b->logits || !b->scores || !b->tokens || !b->parents || !b->candidate_scores)
        return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_select: logits, scores, tokens, parents and candidate_scores are required");
    const size_t esz = b->logits_dtype == STG_DTYPE_BF16 ? 2 : 4;
    if (misaligned(b->logits, esz) || misaligned(b->scores, 4) || misaligned(b->mask, 4) || misaligned(b->tokens, 4) || misaligned(b->parents, 4) ||
        misaligned(b->candidate_scores, 4) || misaligned(b->log_norms, 4) || misaligned(b->seq_flags, 4))
        return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_select: an array is not aligned to its elements");
    CK(cudaSetDevice(h->cfg.device));
    BeamSelect a;
    memset(&a, 0, sizeof(a));
    a.logits = b->logits; a.row_stride = b->row_stride; a.scores = b->scores;
    a.mask = b->mask; a.mask_stride = b->mask_row_stride; a.uses_mask = b->row_uses_mask;
    a.softcap = b->logit_softcap;
    a.n_seq = b->n_seq; a.beams = b->n_beams; a.vocab = b->vocab; a.n = b->n_candidates;
    a.tokens = b->tokens; a.parents = b->parents; a.out_scores = b->candidate_scores; a.log_norms = b->log_norms; a.flags = b->seq_flags;
    const int rows = b->n_seq * b->n_beams;
    a.pieces = 1;
    a.piece_len = b->vocab;

    const size_t b_parts = round_up((size_t)rows * a.pieces * sizeof(BeamPart), 256), b_keys = (size_t)rows * a.pieces * a.n * 8;
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    CK(cudaStreamIsCapturing(stream, &cap));
    void *ws = h->bm_ws.p;
    if (cap != cudaStreamCaptureStatusNone) {
        rc = captured_workspace(h, b_parts + b_keys, &ws);
    } else {
        if (b_parts + b_keys > h->bm_ws.bytes) return fail(h, STG_ERR_CAPACITY, "stg_beam_select: workspace too small");
        rc = order_behind_last(h, stream);
    }
    if (rc) return rc;
    a.ws.parts = (BeamPart *)ws;
    a.ws.keys = (u64 *)((char *)ws + b_parts);
    const bool vec = !misaligned(b->logits, 16) && (rows == 1 || (size_t)b->row_stride * esz % 16 == 0);
    const dim3 grid((unsigned)a.pieces, (unsigned)rows);
    if (b->logits_dtype == STG_DTYPE_BF16) {
        if (vec) k_beam_rows<true, true><<<grid, kBeamThreads, 0, stream>>>(a);
        else k_beam_rows<true, false><<<grid, kBeamThreads, 0, stream>>>(a);
    } else {
        if (vec) k_beam_rows<false, true><<<grid, kBeamThreads, 0, stream>>>(a);
        else k_beam_rows<false, false><<<grid, kBeamThreads, 0, stream>>>(a);
    }
    CK(cudaGetLastError());
    k_beam_merge<<<b->n_seq, kBeamThreads, 0, stream>>>(a);
    CK(cudaGetLastError());
    h->stats.calls++;
    h->stats.kernel_launches += 2;
    return STG_OK;
}

}  // namespace stg

extern "C" int stg_beam_select(StgHandle h, const StgBeamBatch *batch, void *stream)
{
    if (!h) return STG_ERR_INVALID_ARGUMENT;
    try {
        return stg::beam_select(h, batch, (cudaStream_t)stream);
    } catch (const std::bad_alloc &) {
        return STG_ERR_CAPACITY;
    }
}
