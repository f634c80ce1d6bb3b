// Backtraces of searches with different numbers of beams, each in a thread with a handle and a stream of its own: no call may
// fail for what another thread's call asks of the device.  Prints "beam_threads: <result>".
#include <cuda_runtime.h>

#include <atomic>
#include <cstdio>
#include <string>
#include <thread>
#include <vector>

#include "stingray_sampler.hpp"

static std::atomic<int> failed{0}, started{0};

static std::string why(StgHandle h)
{
    char text[256] = "";
    stg_last_error(h, text, sizeof text);
    return text;
}

static void calls(int K, int threads, int times)
{
    const int T = 24;
    StgHandle h = nullptr;
    StgConfig cfg{};
    cfg.struct_size = (int32_t)sizeof cfg;
    cfg.max_rows = K;
    cfg.max_vocab = 64;
    cfg.max_history = 1;
    cfg.max_top_k = 1;
    if (stg_create(&cfg, &h) != STG_OK) {
        failed = 1;
        std::printf("stg_create: %s\n", why(nullptr).c_str());
        return;
    }
    cudaStream_t stream = nullptr;
    int32_t *p = nullptr;
    const size_t trail = (size_t)T * K, hyps = (size_t)K;
    if (cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking) != cudaSuccess || cudaMalloc((void **)&p, (2 * trail + 4 * hyps + hyps * T) * 4) != cudaSuccess ||
        cudaMemset(p, 0, (2 * trail + 4 * hyps + hyps * T) * 4) != cudaSuccess)
        failed = 1;
    int32_t *const tokens = p, *const parents = p + trail, *const ends = parents + trail, *const end_parents = ends + hyps, *const end_tokens = end_parents + hyps,
                  *const lengths = end_tokens + hyps, *const out = lengths + hyps;
    const std::vector<int32_t> last(hyps, T - 1);
    if (cudaMemcpy(ends, last.data(), hyps * 4, cudaMemcpyHostToDevice) != cudaSuccess) failed = 1;
    started++;
    while (started < threads && !failed) std::this_thread::yield();
    for (int i = 0; i < times && !failed; i++) {
        if (stg_beam_backtrace(h, tokens, parents, T, 1, K, K, ends, end_parents, end_tokens, 0, out, T, lengths, stream) != STG_OK) {
            failed = 1;
            std::printf("%d beams, call %d: %s\n", K, i, why(h).c_str());
        }
        if (i % 256 == 255 && cudaStreamSynchronize(stream) != cudaSuccess) failed = 1;
    }
    if (stream && cudaStreamSynchronize(stream) != cudaSuccess) failed = 1;
    std::vector<int32_t> got(hyps);
    if (!failed && (cudaMemcpy(got.data(), lengths, hyps * 4, cudaMemcpyDeviceToHost) != cudaSuccess || got != std::vector<int32_t>(hyps, T))) failed = 1;
    if (p) cudaFree(p);
    if (stream) cudaStreamDestroy(stream);
    stg_destroy(h);
}

int main()
{
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
        std::printf("beam_threads: no device\n");
        return 0;
    }
    std::vector<std::thread> all;
    const int beams[] = {16, 10, 32, 12};
    for (int K : beams) all.emplace_back(calls, K, 4, 20000);
    for (auto &t : all) t.join();
    std::printf("beam_threads: %s\n", failed ? "FAILED" : "ok");
    return failed ? 1 : 0;
}
