// The head's calls through the C++ wrapper: a weight of whole numbers in 4 bits, whose logits are known by heart, sampled from, and
// the loss of the tokens under a uniform head.  Without a CUDA device creation has to be refused.  Prints "head_check: <result>".
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
            std::printf("head_check: FAILED %s (line %d)\n", #c, __LINE__); \
            return 1;                                                     \
        }                                                                 \
    } while (0)

template <class T>
static T *device(const std::vector<T> &v)
{
    T *p = nullptr;
    if (cudaMalloc((void **)&p, v.size() * sizeof(T) + 1) != cudaSuccess) std::exit(1);
    if (cudaMemcpy(p, v.data(), v.size() * sizeof(T), cudaMemcpyHostToDevice) != cudaSuccess) std::exit(1);
    return p;
}
template <class T>
static std::vector<T> host(const void *p, size_t n)
{
    std::vector<T> v(n);
    if (cudaMemcpy(v.data(), p, n * sizeof(T), cudaMemcpyDeviceToHost) != cudaSuccess) std::exit(1);
    return v;
}

int main()
{
    const int V = 40, D = 64, R = 40;
    stingray::BatchSampler s = [&]() -> stingray::BatchSampler {
        try {
            return stingray::BatchSampler(0, R, V, 4, 4);
        } catch (const stingray::Error &e) {
            if (e.status() != STG_ERR_NO_DEVICE) throw;
            std::printf("head_check: no device, creation refused\n");
            std::exit(0);
        }
    }();
    const uint16_t one = 0x3F80;  // bf16
    // entry v has code 8 + 1 in column v and 8 elsewhere; hidden state r is 2 in column r: logit 2 at r, 0 elsewhere
    std::vector<uint8_t> codes(V * D / 2, 0x88);
    for (int v = 0; v < V; v++) codes[v * D / 2 + v / 2] = v % 2 ? 0x98 : 0x89;
    std::vector<uint16_t> hidden(R * D, 0), scales(V * D / 32, one), weight(V * D, 0);
    for (int r = 0; r < R; r++) hidden[r * D + r] = 0x4000;

    for (int rows : {1, 7, 40}) {
        StgHeadPack pack;
        std::memset(&pack, 0, sizeof pack);
        pack.vocab = V; pack.width = D; pack.group = 32; pack.scale_dtype = STG_DTYPE_BF16;
        pack.codes = device(codes); pack.codes_stride = D / 2; pack.scales = device(scales);
        pack.packed_bytes = s.head_pack_bytes(V, D, 32, false);
        pack.packed = device(std::vector<uint8_t>(pack.packed_bytes));
        s.head_pack(pack);
        StgHeadLogits l;
        std::memset(&l, 0, sizeof l);
        l.rows = rows; l.vocab = V; l.width = D; l.group = 32; l.scale_dtype = STG_DTYPE_BF16; l.hidden_dtype = STG_DTYPE_BF16; l.logits_dtype = STG_DTYPE_F32;
        l.packed = pack.packed; l.packed_bytes = pack.packed_bytes; l.hidden = device(hidden); l.hidden_stride = D;
        l.logits = device(std::vector<float>(rows * V, -1.f)); l.row_stride = V;
        l.workspace_bytes = s.head_logits_workspace(l);
        l.workspace = device(std::vector<uint8_t>(l.workspace_bytes));
        s.head_logits(l);
        const std::vector<float> got = host<float>(l.logits, rows * V);
        for (int r = 0; r < rows; r++)
            for (int v = 0; v < V; v++) REQUIRE(got[r * V + v] == (v == r ? 2.f : 0.f));
    }

    // a weight of zeros: every token has probability 1 / V, and the hidden states' gradients are 0
    StgHeadLoss a;
    std::memset(&a, 0, sizeof a);
    std::vector<int32_t> targets(R);
    for (int r = 0; r < R; r++) targets[r] = r % 3 == 2 ? -1 : r;
    a.rows = R; a.vocab = V; a.width = D; a.dtype = STG_DTYPE_BF16;
    a.hidden = device(hidden); a.hidden_stride = D; a.weight = device(weight); a.weight_stride = D; a.targets = device(targets);
    a.loss = device(std::vector<float>(R)); a.log_norms = device(std::vector<float>(R)); a.grad_loss = device(std::vector<float>(R, 1.f));
    a.grad_hidden = device(std::vector<uint16_t>(R * D, 1)); a.grad_weight = device(std::vector<uint16_t>(V * D, 1));
    for (int backward = 0; backward < 2; backward++) {
        a.workspace_bytes = s.head_loss_workspace(a, backward != 0);
        a.workspace = device(std::vector<uint8_t>(a.workspace_bytes));
        if (backward) s.head_loss_backward(a);
        else s.head_loss(a);
    }
    const std::vector<float> loss = host<float>(a.loss, R);
    for (int r = 0; r < R; r++) REQUIRE(std::fabs(loss[r] - (targets[r] < 0 ? 0.f : std::log((float)V))) < 1e-5f);
    for (uint16_t g : host<uint16_t>(a.grad_hidden, R * D)) REQUIRE((g & 0x7FFF) == 0);
    const std::vector<uint16_t> gw = host<uint16_t>(a.grad_weight, V * D);
    for (int v = 0; v < V; v++)
        for (int d = 0; d < D; d++) {
            // row d has hidden state 2 in column d: 2 (1 / V - [v == d]), where it has a loss
            uint32_t bits = (uint32_t)gw[v * D + d] << 16;
            float g;
            std::memcpy(&g, &bits, 4);
            const float want = d < R && targets[d] >= 0 ? 2.f * (1.f / V - (v == d)) : 0.f;
            REQUIRE(std::fabs(g - want) <= std::fabs(want) / 256.f + 1e-6f);
        }
    a.width = 60;
    try {
        s.head_loss(a);
        REQUIRE(false);
    } catch (const stingray::Error &e) {
        REQUIRE(e.status() == STG_ERR_UNSUPPORTED);
    }
    std::printf("head_check: ok\n");
    return 0;
}
