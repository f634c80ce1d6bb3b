// The beam calls through the C++ wrapper: one sequence of two beams decodes three tokens of a vocabulary of four, whose
// logits are known by heart.  Without a CUDA device creation has to be refused.  Prints "beam_check: <result>".
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "stingray_sampler.hpp"

#define REQUIRE(c)                                                        \
    do {                                                                  \
        if (!(c)) {                                                       \
            std::printf("beam_check: FAILED %s (line %d)\n", #c, __LINE__); \
            return 1;                                                     \
        }                                                                 \
    } while (0)

template <class T>
static T *device(const std::vector<T> &v)
{
    T *p = nullptr;
    if (cudaMalloc((void **)&p, v.size() * sizeof(T)) != cudaSuccess) std::exit(1);
    if (cudaMemcpy(p, v.data(), v.size() * sizeof(T), cudaMemcpyHostToDevice) != cudaSuccess) std::exit(1);
    return p;
}
template <class T>
static std::vector<T> host(const T *p, size_t n)
{
    std::vector<T> v(n);
    if (cudaMemcpy(v.data(), p, n * sizeof(T), cudaMemcpyDeviceToHost) != cudaSuccess) std::exit(1);
    return v;
}

int main()
{
    const int K = 2, V = 4, T = 3, n = 4;
    stingray::BatchSampler s = [&]() -> stingray::BatchSampler {
        try {
            return stingray::BatchSampler(0, K, V, 4, 4);
        } catch (const stingray::Error &e) {
            if (e.status() != STG_ERR_NO_DEVICE) throw;
            std::printf("beam_check: no device, creation refused\n");
            std::exit(0);
        }
    }();
    // probabilities 1/2, 1/4, 1/8, 1/8 in every row: token 0 best, token 1 next, 2 and 3 alike
    const std::vector<float> row = {std::log(4.f), std::log(2.f), 0.f, 0.f};
    std::vector<float> logits;
    for (int k = 0; k < K; k++) logits.insert(logits.end(), row.begin(), row.end());

    StgBeamSearch search;
    std::memset(&search, 0, sizeof search);
    const int32_t eos[1] = {3};
    search.n_seq = 1; search.n_beams = K; search.max_steps = T; search.n_eos = 1; search.pad_token = 9; search.eos_tokens = eos;
    search.norms = device(std::vector<double>{1.0, 2.0, 3.0});
    search.tokens = device(std::vector<int32_t>(K)); search.parents = device(std::vector<int32_t>(K)); search.scores = device(std::vector<float>(K));
    search.steps = device(std::vector<int32_t>(1)); search.done = device(std::vector<int32_t>(1));
    search.pool_scores = device(std::vector<float>(K)); search.pool_steps = device(std::vector<int32_t>(K));
    search.pool_parents = device(std::vector<int32_t>(K)); search.pool_tokens = device(std::vector<int32_t>(K));
    search.trail_tokens = device(std::vector<int32_t>(T * K)); search.trail_parents = device(std::vector<int32_t>(T * K));

    StgBeamBatch b;
    std::memset(&b, 0, sizeof b);
    b.n_seq = 1; b.n_beams = K; b.vocab = V; b.logits_dtype = STG_DTYPE_F32; b.n_candidates = n;
    b.logits = device(logits); b.row_stride = V; b.scores = search.scores;
    b.tokens = device(std::vector<int32_t>(n)); b.parents = device(std::vector<int32_t>(n)); b.candidate_scores = device(std::vector<float>(n));

    StgBeamState state;
    std::memset(&state, 0, sizeof state);
    int32_t *const marks = device(std::vector<int32_t>{7, 8});
    state.data = marks; state.row_stride = state.inner_bytes = 4; state.size[0] = state.size[1] = state.size[2] = 1; state.position_dim = -1;
    StgBeamReorder reorder;
    std::memset(&reorder, 0, sizeof reorder);
    reorder.n_seq = 1; reorder.n_beams = K; reorder.n_states = 1; reorder.states = &state; reorder.parents = search.parents; reorder.n_positions = -1;

    s.beam_start(search, 0, 1);
    for (int t = 0; t < T; t++) {
        s.beam_select(b);
        s.beam_advance(search, n, b.tokens, b.parents, b.candidate_scores);
        if (t == 0) s.beam_reorder(reorder);
    }
    // the first step continues beam 0 twice; the best hypotheses of three tokens are 0 0 0 and 0 0 1
    REQUIRE(host(marks, 2) == (std::vector<int32_t>{7, 7}));
    REQUIRE(host(search.done, 1)[0] == 1 && host(search.steps, 1)[0] == 3);
    const std::vector<float> pool = host(search.pool_scores, K);
    REQUIRE(std::fabs(pool[0] + std::log(2.f)) < 1e-5f && std::fabs(pool[1] + 4.f * std::log(2.f) / 3.f) < 1e-5f);
    int32_t *const sequences = device(std::vector<int32_t>(K * T)), *const lengths = device(std::vector<int32_t>(K));
    s.beam_backtrace(search, K, search.pool_steps, search.pool_parents, search.pool_tokens, sequences, lengths);
    REQUIRE(host(lengths, K) == (std::vector<int32_t>{3, 3}));
    const std::vector<int32_t> found = host(sequences, K * T);
    REQUIRE(found[0] == 0 && found[1] == 0 && found[2] == 0);
    REQUIRE(found[3] + found[4] + found[5] == 1);
    // refused, not read: more candidates than there may be
    b.n_candidates = STG_BEAM_MAX_CANDIDATES + 1;
    try {
        s.beam_select(b);
        REQUIRE(!"expected an error");
    } catch (const stingray::Error &e) {
        REQUIRE(e.status() == STG_ERR_CAPACITY);
    }
    std::printf("beam_check: ok\n");
    return 0;
}
