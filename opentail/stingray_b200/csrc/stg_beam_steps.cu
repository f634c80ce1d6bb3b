// stg_beam_start, stg_beam_advance, stg_beam_backtrace: a search's bookkeeping on the device.
//
// One warp per sequence: lane k holds beam k and entry k of the pool, which is sorted, so a hypothesis finds its place by
// one ballot and the entries behind it move up by one shuffle.  Nothing here moves more than a few hundred bytes per
// sequence; what bounds these kernels is the chain of dependent loads and the launch.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>
#include <string.h>

#include "stg_beam.h"
#include "stg_pdl.cuh"
#include "stg_types.h"

namespace stg {

constexpr int kStepWarps = 4;  // sequences per CTA

struct EosSet {
    int32_t n;
    int32_t id[STG_BEAM_MAX_EOS];
};

__global__ void __launch_bounds__(kStepWarps * 32) k_beam_start(const __grid_constant__ StgBeamSearch s, int first, int count)
{
    const int lane = threadIdx.x & 31, i = blockIdx.x * kStepWarps + (threadIdx.x >> 5);
    pdl_release();
    pdl_wait();
    if (i >= count) return;
    const int seq = first + i, K = s.n_beams;
    if (lane < K) {
        const int o = seq * K + lane;
        s.tokens[o] = s.pad_token;
        s.parents[o] = lane;
        s.scores[o] = lane == 0 ? 0.f : -CUDART_INF_F;
        s.pool_scores[o] = -CUDART_INF_F;
        s.pool_steps[o] = s.pool_parents[o] = s.pool_tokens[o] = -1;
    }
    if (lane == 0) s.steps[seq] = s.done[seq] = 0;
}

// Entry `lane` of a sequence's pool, best first.
struct PoolEntry {
    float score;
    int32_t step, parent, token;

    // All lanes offer the same hypothesis; an equal one stands behind the older.
    __device__ __forceinline__ void offer(int lane, int K, float sc, int t, int par, int tok)
    {
        const int pos = __popc(__ballot_sync(0xFFFFFFFFu, lane < K && score >= sc));
        const float us = __shfl_up_sync(0xFFFFFFFFu, score, 1);
        const int ut = __shfl_up_sync(0xFFFFFFFFu, step, 1), up = __shfl_up_sync(0xFFFFFFFFu, parent, 1), uk = __shfl_up_sync(0xFFFFFFFFu, token, 1);
        if (!(sc > -CUDART_INF_F)) return;  // the quotient has left the range of 32 bits
        if (lane > pos) { score = us; step = ut; parent = up; token = uk; }
        if (lane == pos) { score = sc; step = t; parent = par; token = tok; }
    }
};

__global__ void __launch_bounds__(kStepWarps * 32) k_beam_advance(const __grid_constant__ StgBeamSearch s, const __grid_constant__ EosSet eos, int n,
                                                                 const int32_t *cand_tokens, const int32_t *cand_parents, const float *cand_scores,
                                                                 int finish)
{
    __shared__ int32_t next_tok[kStepWarps][32], next_par[kStepWarps][32];
    __shared__ float next_sc[kStepWarps][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, seq = blockIdx.x * kStepWarps + w;
    pdl_release();
    pdl_wait();
    if (seq >= s.n_seq) return;  // whole warps
    const int K = s.n_beams, o = seq * K + lane;
    const int t = s.steps[seq];
    bool over = s.done[seq] != 0 || t < 0 || t >= s.max_steps;
    if (!over) {
        PoolEntry pool{-CUDART_INF_F, -1, -1, -1};
        if (lane < K) pool = PoolEntry{s.pool_scores[o], s.pool_steps[o], s.pool_parents[o], s.pool_tokens[o]};
        const double norm = s.norms[t];
        int alive = 0;
        for (int first = 0; first < n; first += 32) {
            const int i = first + lane;
            const int64_t c = (int64_t)seq * n + i;
            int tok = -1, par = -1;
            float sc = -CUDART_INF_F;
            if (i < n) { tok = cand_tokens[c]; par = cand_parents[c]; sc = cand_scores[c]; }
            const bool valid = tok >= 0 && par >= 0 && par < K && sc > -CUDART_INF_F;
            bool end = false;
            for (int e = 0; e < eos.n; e++) end |= tok == eos.id[e];
            const unsigned on = __ballot_sync(0xFFFFFFFFu, valid && !end);
            const int slot = alive + __popc(on & ((1u << lane) - 1u));
            if (valid && !end && slot < K) { next_tok[w][slot] = tok; next_par[w][slot] = par; next_sc[w][slot] = sc; }
            alive += __popc(on);
            for (unsigned ended = __ballot_sync(0xFFFFFFFFu, valid && end && i < K); ended != 0u; ended &= ended - 1u) {
                const int l = __ffs(ended) - 1;
                pool.offer(lane, K, (float)((double)__shfl_sync(0xFFFFFFFFu, sc, l) / norm), t, __shfl_sync(0xFFFFFFFFu, par, l),
                           __shfl_sync(0xFFFFFFFFu, tok, l));
            }
        }
        alive = min(alive, K);
        __syncwarp();
        int tok = s.pad_token, par = lane;
        float sc = -CUDART_INF_F;
        if (lane < alive) { tok = next_tok[w][lane]; par = next_par[w][lane]; sc = next_sc[w][lane]; }
        if (lane < K) {
            const int64_t at = ((int64_t)t * s.n_seq + seq) * K + lane;
            s.trail_tokens[at] = tok;
            s.trail_parents[at] = par;
        }
        const bool last = finish != 0 || t + 1 == s.max_steps;
        if (last)
            for (int l = 0; l < alive; l++)
                pool.offer(lane, K, (float)((double)__shfl_sync(0xFFFFFFFFu, sc, l) / norm), t, __shfl_sync(0xFFFFFFFFu, par, l),
                           __shfl_sync(0xFFFFFFFFu, tok, l));
        const float worst = __shfl_sync(0xFFFFFFFFu, pool.score, K - 1), best = __shfl_sync(0xFFFFFFFFu, sc, 0);
        over = last || alive == 0 || (worst > -CUDART_INF_F && (s.early_stopping != 0 || worst >= (float)((double)best / norm)));
        if (lane < K) {
            s.pool_scores[o] = pool.score;
            s.pool_steps[o] = pool.step;
            s.pool_parents[o] = pool.parent;
            s.pool_tokens[o] = pool.token;
            if (!over) { s.tokens[o] = tok; s.parents[o] = par; s.scores[o] = sc; }
        }
        if (lane == 0) {
            s.steps[seq] = t + 1;
            if (over) s.done[seq] = 1;
        }
    }
    if (over && lane < K) { s.tokens[o] = s.pad_token; s.parents[o] = lane; s.scores[o] = -CUDART_INF_F; }
}

struct Backtrace {
    const int32_t *tokens, *parents, *ends, *end_parents, *end_tokens;
    int32_t T, n_seq, beams, hyps, pad;
    int32_t *out, *lengths;
    int64_t stride;
};

// A walk back through the trail is a chain of dependent loads, one per step.  But a step is a map of the beams into the
// beams, and maps can be joined in any grouping: so the trail of a sequence is cut into pieces of 16 steps, whose maps are
// found side by side in shared memory; the pieces of a CTA's segment are joined by one lookup each, the segments of a
// cluster of CTAs by one lookup each through distributed shared memory, and then every piece is walked by every hypothesis at once.  A
// trail longer than a cluster's segments is done from its end on, one span after the other.  (64 sequences of eight beams and 4096
// steps: 15.7 us, 1390 with one thread per hypothesis, a load of parent and token per step.  The 25 MB read and written are 3.9
// us; the rest are the chains within a CTA, about 150 lookups one after the other, and two cluster barriers.)
constexpr int kTraceThreads = 256;
constexpr int kPiece = 16;          // steps
constexpr int kMaxSegment = 512;    // steps of a CTA
constexpr int kMaxPieces = kMaxSegment / kPiece;
constexpr int kTraceHyps = 32;      // walked at a time

static int trace_segment(int beams) { return beams <= 16 ? kMaxSegment : kMaxSegment / 2; }
static size_t trace_smem(int beams) { return (size_t)trace_segment(beams) * (beams * 4 + beams + 1); }

__global__ void __launch_bounds__(kTraceThreads) k_beam_backtrace(const __grid_constant__ Backtrace a, int segment)
{
    namespace cg = cooperative_groups;
    extern __shared__ int32_t tok[];                         // [segment, beams]
    uint8_t *par = (uint8_t *)(tok + segment * a.beams);     // [segment, beams + 1]: the last beam is nobody, whose parent is nobody
    __shared__ uint8_t map[kMaxPieces][STG_BEAM_MAX_BEAMS + 1];        // beam behind a piece -> beam ahead of it
    __shared__ uint8_t seg_map[STG_BEAM_MAX_BEAMS + 1];                // the same for the segment
    __shared__ uint8_t all_maps[8][STG_BEAM_MAX_BEAMS + 1];
    __shared__ int32_t ends[STG_BEAM_MAX_CANDIDATES], end_token[STG_BEAM_MAX_CANDIDATES];  // the hypotheses; -1: none
    __shared__ uint8_t from[STG_BEAM_MAX_CANDIDATES];
    __shared__ uint8_t ahead[STG_BEAM_MAX_CANDIDATES];                 // of a hypothesis that starts in this segment
    __shared__ uint8_t carry[STG_BEAM_MAX_CANDIDATES];                 // ... that started in a later span: its beam behind this one
    __shared__ uint8_t enter[kTraceHyps][kMaxPieces];                  // beam behind a piece
    __shared__ uint8_t walked[kTraceHyps][kMaxSegment];
    const cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int seq = blockIdx.x / C, tid = threadIdx.x, K = a.beams, N = a.hyps, W = K + 1;
    const int64_t row = (int64_t)a.n_seq * K;  // of the trail
    const int span = C * segment;
    pdl_release();
    pdl_wait();
    const uint32_t over_k = 0xFFFFFFFFu / (uint32_t)K + 1u;  // i / K is the upper half of i * over_k, for the i below and K > 1
    for (int n = tid; n < N; n += kTraceThreads) {
        const int64_t hyp = (int64_t)seq * N + n;
        const int e = a.ends[hyp];
        ends[n] = e >= 0 && e < a.T ? e : -1;
        from[n] = (uint8_t)min((uint32_t)a.end_parents[hyp], (uint32_t)K);
        end_token[n] = a.end_tokens[hyp];
        if (rank == 0 && a.lengths) a.lengths[hyp] = ends[n] + 1;
    }
    for (int span_begin = (a.T - 1) / span * span; span_begin >= 0; span_begin -= span) {
        const int begin = span_begin + rank * segment, len = max(0, min(segment, a.T - begin));
        const int pieces = (len + kPiece - 1) / kPiece;
        const int64_t at = begin * row + (int64_t)seq * K;
        __syncthreads();
        // eight loads of each array in flight: one after the other they were half of a call's time
        for (int first = tid; first < len * K; first += 8 * kTraceThreads) {
            uint32_t p[8];
            int32_t v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int i = first + j * kTraceThreads, t = K == 1 ? i : (int)__umulhi((uint32_t)i, over_k), k = i - t * K;
                if (i < len * K) {
                    p[j] = (uint32_t)__ldcs(a.parents + at + t * row + k);
                    v[j] = __ldcs(a.tokens + at + t * row + k);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int i = first + j * kTraceThreads, t = K == 1 ? i : (int)__umulhi((uint32_t)i, over_k), k = i - t * K;
                if (i < len * K) {
                    tok[i] = v[j];
                    par[t * W + k] = (uint8_t)min(p[j], (uint32_t)K);
                }
            }
        }
        for (int t = tid; t < len; t += kTraceThreads) par[t * W + K] = (uint8_t)K;
        __syncthreads();
        for (int i = tid; i < pieces * W; i += kTraceThreads) {
            const int p = i / W, k = i - p * W;
            int b = k;
            for (int t = min(len, (p + 1) * kPiece) - 1; t >= p * kPiece; t--) b = par[t * W + b];
            map[p][k] = (uint8_t)b;
        }
        __syncthreads();
        // the first warps join the segment's pieces, the others take the hypotheses that start in it back to its beginning
        if (tid < W) {
            int b = tid;
            for (int p = pieces - 1; p >= 0; p--) b = map[p][b];
            seg_map[tid] = (uint8_t)b;
        }
        for (int n = tid - 64; n >= 0 && n < N; n += kTraceThreads - 64) {
            const int last = ends[n] - 1 - begin;  // its first step back, in the segment
            if (last < 0 || last >= len) continue;
            int b = from[n];
            const int p = last / kPiece;
            for (int t = last; t >= p * kPiece; t--) b = par[t * W + b];
            for (int q = p - 1; q >= 0; q--) b = map[q][b];
            ahead[n] = (uint8_t)b;
        }
        cluster.sync();
        for (int i = tid; i < C * W; i += kTraceThreads) {
            const int c = i / W, k = i - c * W;
            all_maps[c][k] = *cluster.map_shared_rank(&seg_map[k], c);
        }
        __syncthreads();
        for (int n0 = 0; n0 < N; n0 += kTraceHyps) {
            const int some = min(kTraceHyps, N - n0);
            if (tid < some) {
                const int n = n0 + tid, last = ends[n] - 1 - span_begin;
                if (last >= 0) {
                    int c = C, b = 0;  // the segment it starts in; behind all: it is carried along
                    if (last < span) {
                        c = last / segment;
                        b = *cluster.map_shared_rank(&ahead[n], c);
                    } else {
                        b = carry[n];
                    }
                    int here = c == rank ? -1 : K;  // its beam behind this segment
                    for (int q = c - 1; q >= 0; q--) {
                        if (q == rank) here = b;
                        b = all_maps[q][b];
                    }
                    carry[n] = (uint8_t)b;
                    int p = pieces - 1;
                    if (here < 0) {  // starts here: pieces behind its own are not walked, its own from `last` on
                        here = from[n];
                        p = (last - rank * segment) / kPiece;
                        enter[tid][p] = (uint8_t)here;
                        for (int t = last - rank * segment; t >= p * kPiece; t--) here = par[t * W + here];
                        p--;
                    }
                    for (; p >= 0; p--) {
                        enter[tid][p] = (uint8_t)here;
                        here = map[p][here];
                    }
                }
            }
            __syncthreads();
            for (int i = tid; i < some * kMaxPieces; i += kTraceThreads) {
                const int h = i / kMaxPieces, p = i % kMaxPieces;
                if (p >= pieces) continue;
                const int last = ends[n0 + h] - 1 - begin;
                int b = enter[h][p];
                if (last >= p * kPiece)
                    for (int t = min(min(len, (p + 1) * kPiece) - 1, last); t >= p * kPiece; t--) {
                        walked[h][t] = (uint8_t)b;
                        b = par[t * W + b];
                    }
            }
            __syncthreads();
            for (int h = 0; h < some; h++) {
                const int end = ends[n0 + h] - begin;
                int32_t *out = a.out + ((int64_t)seq * N + n0 + h) * a.stride + begin;
#pragma unroll
                for (int j = 0; j < kMaxSegment / kTraceThreads; j++) {
                    const int t = tid + j * kTraceThreads;
                    if (t >= len) break;
                    int v = t == end ? end_token[n0 + h] : a.pad;
                    if (t < end) {
                        const int b = walked[h][t];
                        if (b < K) v = tok[t * K + b];
                    }
                    __stcs(out + t, v);
                }
            }
            __syncthreads();
        }
        cluster.sync();  // the next span overwrites what other CTAs read, and nobody leaves while they do
    }
}

static int check_search(StgHandle h, const char *who, const StgBeamSearch *s)
{
    const std::string w(who);
    if (!s || s->struct_size != (int32_t)sizeof(StgBeamSearch)) return fail(h, STG_ERR_INVALID_ARGUMENT, "bad StgBeamSearch");
    int rc = beam_check_rows(h, who, s->n_seq, s->n_beams);
    if (rc) return rc;
    if (s->max_steps < 1) return fail(h, STG_ERR_INVALID_ARGUMENT, w + ": max_steps must be >= 1");
    if (s->n_eos < 0 || (s->n_eos > 0 && !s->eos_tokens)) return fail(h, STG_ERR_INVALID_ARGUMENT, w + ": bad end tokens");
    if (s->n_eos > STG_BEAM_MAX_EOS) return fail(h, STG_ERR_CAPACITY, w + ": at most 8 end tokens");
    if (s->n_seq == 0) return STG_OK;
    const void *arrays[] = {s->tokens, s->parents, s->scores, s->steps, s->done, s->pool_scores, s->pool_steps, s->pool_parents, s->pool_tokens,
                            s->trail_tokens, s->trail_parents};
    for (const void *p : arrays)
        if (!p || misaligned(p, 4)) return fail(h, STG_ERR_INVALID_ARGUMENT, w + ": an array of the search is missing or not aligned to its elements");
    if (!s->norms || misaligned(s->norms, 8)) return fail(h, STG_ERR_INVALID_ARGUMENT, w + ": norms is missing or not aligned to its elements");
    return STG_OK;
}

}  // namespace stg

using namespace stg;

extern "C" {

int stg_beam_start(StgHandle h, const StgBeamSearch *search, int32_t first_seq, int32_t count, void *stream)
try {
    if (!h) return STG_ERR_INVALID_ARGUMENT;
    int rc = check_search(h, "stg_beam_start", search);
    if (rc) return rc;
    if (first_seq < 0 || count < 0 || (int64_t)first_seq + count > search->n_seq)
        return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_start: sequences outside [0, n_seq)");
    if (count == 0) return STG_OK;
    const OnDevice on(h->cfg.device);
    CK(on.error);
    CK(launch_behind(k_beam_start, dim3((unsigned)(count + kStepWarps - 1) / kStepWarps), kStepWarps * 32, 0, (cudaStream_t)stream, *search, first_seq, count));
    h->stats.kernel_launches++;
    return STG_OK;
} catch (const std::bad_alloc &) {
    return STG_ERR_CAPACITY;
}

int stg_beam_advance(StgHandle h, const StgBeamSearch *search, int32_t n_candidates, const int32_t *cand_tokens,
                     const int32_t *cand_parents, const float *cand_scores, int32_t finish, void *stream)
try {
    if (!h) return STG_ERR_INVALID_ARGUMENT;
    int rc = check_search(h, "stg_beam_advance", search);
    if (rc) return rc;
    if (n_candidates < 1) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_advance: n_candidates must be >= 1");
    if (n_candidates > STG_BEAM_MAX_CANDIDATES) return fail(h, STG_ERR_CAPACITY, "stg_beam_advance: at most 128 candidates per sequence");
    if (search->n_seq == 0) return STG_OK;
    if (!cand_tokens || !cand_parents || !cand_scores || misaligned(cand_tokens, 4) || misaligned(cand_parents, 4) || misaligned(cand_scores, 4))
        return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_advance: an array of the candidates is missing or not aligned to its elements");
    EosSet eos;
    memset(&eos, 0, sizeof(eos));
    eos.n = search->n_eos;
    for (int i = 0; i < eos.n; i++) eos.id[i] = search->eos_tokens[i];
    const OnDevice on(h->cfg.device);
    CK(on.error);
    CK(launch_behind(k_beam_advance, dim3((unsigned)(search->n_seq + kStepWarps - 1) / kStepWarps), kStepWarps * 32, 0, (cudaStream_t)stream, *search, eos,
                     n_candidates, cand_tokens, cand_parents, cand_scores, finish));
    h->stats.kernel_launches++;
    return STG_OK;
} catch (const std::bad_alloc &) {
    return STG_ERR_CAPACITY;
}

int stg_beam_backtrace(StgHandle h, const int32_t *trail_tokens, const int32_t *trail_parents, int32_t n_steps, int32_t n_seq,
                       int32_t n_beams, int32_t n_hyps, const int32_t *hyp_steps, const int32_t *hyp_parents,
                       const int32_t *hyp_tokens, int32_t pad_token, int32_t *sequences, int64_t out_stride, int32_t *lengths,
                       void *stream)
try {
    if (!h) return STG_ERR_INVALID_ARGUMENT;
    int rc = beam_check_rows(h, "stg_beam_backtrace", n_seq, n_beams);
    if (rc) return rc;
    if (n_steps < 0 || n_hyps < 0 || out_stride < n_steps) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_backtrace: negative size, or out_stride smaller than n_steps");
    if (n_hyps > STG_BEAM_MAX_CANDIDATES) return fail(h, STG_ERR_CAPACITY, "stg_beam_backtrace: at most 128 hypotheses per sequence");
    if (n_seq == 0 || n_hyps == 0) return STG_OK;
    const void *arrays[] = {hyp_steps, hyp_parents, hyp_tokens};
    for (const void *p : arrays)
        if (!p || misaligned(p, 4)) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_backtrace: an array of the hypotheses is missing or not aligned to its elements");
    const void *trail[] = {trail_tokens, trail_parents, sequences};
    for (const void *p : trail)
        if ((!p && n_steps > 0) || misaligned(p, 4)) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_backtrace: trail or sequences missing or not aligned to their elements");
    if (misaligned(lengths, 4)) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_backtrace: lengths is not aligned to its elements");
    const OnDevice on(h->cfg.device);
    CK(on.error);
    Backtrace a;
    memset(&a, 0, sizeof(a));
    a.tokens = trail_tokens; a.parents = trail_parents;
    a.ends = hyp_steps; a.end_parents = hyp_parents; a.end_tokens = hyp_tokens;
    a.T = n_steps; a.n_seq = n_seq; a.beams = n_beams; a.hyps = n_hyps; a.pad = pad_token;
    a.out = sequences; a.lengths = lengths; a.stride = out_stride;
    const int segment = trace_segment(n_beams);
    int cluster = 1;
    while (cluster < 8 && cluster * segment < n_steps) cluster *= 2;
    const size_t smem = trace_smem(n_beams);
    // the limit is every thread's and handle's: only ever raised (20 KB are static, so 24 are below what needs no raising)
    if (smem > 24 * 1024) CK(ensure_dynamic_smem((const void *)k_beam_backtrace, smem));
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n_seq * (unsigned)cluster);
    cfg.blockDim = dim3(kTraceThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    CK(cudaLaunchKernelEx(&cfg, k_beam_backtrace, a, segment));
    h->stats.kernel_launches++;
    return STG_OK;
} catch (const std::bad_alloc &) {
    return STG_ERR_CAPACITY;
}

}  // extern "C"
