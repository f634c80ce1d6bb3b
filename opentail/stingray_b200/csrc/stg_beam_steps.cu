// stg_beam_start, stg_beam_advance, stg_beam_backtrace: a search's bookkeeping on the device.
//
// One warp per sequence: lane k holds beam k and entry k of the pool, which is sorted, so a hypothesis finds its place by
// one ballot and the entries behind it move up by one shuffle.  Nothing here moves more than a few hundred bytes per
// sequence; what bounds these kernels is the chain of dependent loads and the launch.
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>
#include <string.h>

#include "stg_beam.h"
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

// One thread per hypothesis walks its way back.
__global__ void __launch_bounds__(128) k_beam_backtrace(const __grid_constant__ Backtrace a)
{
    const int seq = blockIdx.x, n = threadIdx.x;
    if (n >= a.hyps) return;
    const int64_t h = (int64_t)seq * a.hyps + n;
    int32_t *out = a.out + h * a.stride;
    int end = a.ends[h], k = a.end_parents[h];
    if (end < 0 || end >= a.T) end = -1;
    if (a.lengths) a.lengths[h] = end + 1;
    for (int t = end + 1; t < a.T; t++) out[t] = a.pad;
    if (end < 0) return;
    out[end] = a.end_tokens[h];
    for (int t = end - 1; t >= 0; t--) {
        const bool on = k >= 0 && k < a.beams;
        const int64_t at = ((int64_t)t * a.n_seq + seq) * a.beams + k;
        out[t] = on ? a.tokens[at] : a.pad;
        if (on) k = a.parents[at];
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
    CK(cudaSetDevice(h->cfg.device));
    k_beam_start<<<(count + kStepWarps - 1) / kStepWarps, kStepWarps * 32, 0, (cudaStream_t)stream>>>(*search, first_seq, count);
    CK(cudaGetLastError());
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
    CK(cudaSetDevice(h->cfg.device));
    k_beam_advance<<<(search->n_seq + kStepWarps - 1) / kStepWarps, kStepWarps * 32, 0, (cudaStream_t)stream>>>(
        *search, eos, n_candidates, cand_tokens, cand_parents, cand_scores, finish);
    CK(cudaGetLastError());
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
    CK(cudaSetDevice(h->cfg.device));
    Backtrace a;
    memset(&a, 0, sizeof(a));
    a.tokens = trail_tokens; a.parents = trail_parents;
    a.ends = hyp_steps; a.end_parents = hyp_parents; a.end_tokens = hyp_tokens;
    a.T = n_steps; a.n_seq = n_seq; a.beams = n_beams; a.hyps = n_hyps; a.pad = pad_token;
    a.out = sequences; a.lengths = lengths; a.stride = out_stride;
    k_beam_backtrace<<<n_seq, 128, 0, (cudaStream_t)stream>>>(a);
    CK(cudaGetLastError());
    h->stats.kernel_launches++;
    return STG_OK;
} catch (const std::bad_alloc &) {
    return STG_ERR_CAPACITY;
}

}  // extern "C"
