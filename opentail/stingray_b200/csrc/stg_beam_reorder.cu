// stg_beam_reorder: rows of per-beam state follow the beams that go on, in place.
//
// A column of a state - the same 16 bytes of every beam of a sequence - belongs to one thread, which reads
// all the rows that move before it writes any: beams may swap, and no second buffer is needed.  What is moved is what
// has to be: each row that another one continues is read once, rows that stay are not touched.
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>

#include "stg_beam.h"
#include "stg_types.h"

namespace stg {

constexpr int kMoveThreads = 256;
constexpr int kMoveStates = 48;  // states of one launch

struct MoveState {
    char *data;
    int64_t row_stride, inner, pos_bytes;
    int64_t stride[3];
    int32_t size[3];
    int32_t pos_dim;
    int32_t vec;          // bytes a thread moves at a time: 16, 8, 4, 2 or 1
    int32_t cols;         // vectors of a run, the last one possibly cut off
    int64_t first_tile;   // of this state; a tile is kMoveThreads columns of one sequence
    int64_t seq_tiles;    // tiles of one sequence
};

struct MoveArgs {
    MoveState st[kMoveStates];
    int32_t n_states, beams;
    const int32_t *parents, *positions;
};

template <int MOVES, class V>
__device__ __forceinline__ void move_column(char *col, int64_t row_stride, const int *src, const uint32_t *dst, int n)
{
    V v[MOVES];
#pragma unroll
    for (int i = 0; i < MOVES; i++)
        if (i < n) v[i] = *(const V *)(col + src[i] * row_stride);
#pragma unroll
    for (int i = 0; i < MOVES; i++)
        if (i < n)
            for (uint32_t d = dst[i]; d != 0u; d &= d - 1u) *(V *)(col + (__ffs(d) - 1) * row_stride) = v[i];
}

template <int MOVES>
__global__ void __launch_bounds__(kMoveThreads) k_beam_move(const __grid_constant__ MoveArgs a)
{
    __shared__ int src[STG_BEAM_MAX_BEAMS];        // rows that others continue
    __shared__ uint32_t dst[STG_BEAM_MAX_BEAMS];   // ... and which those are, one bit each
    __shared__ int n_src;
    const int tid = threadIdx.x, K = a.beams;
    int lo = 0, hi = a.n_states - 1;  // the last state whose first tile is not behind this one
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if ((int64_t)blockIdx.x >= a.st[mid].first_tile) lo = mid; else hi = mid - 1;
    }
    const MoveState &st = a.st[lo];
    const int64_t tile = (int64_t)blockIdx.x - st.first_tile;
    const int seq = (int)(tile / st.seq_tiles);
    const int64_t col0 = (tile - seq * st.seq_tiles) * kMoveThreads;
    if (tid < 32) {
        const int p = tid < K ? a.parents[(int64_t)seq * K + tid] : -1;
        const bool moves = p >= 0 && p < K && p != tid;
        uint32_t followers = 0u;
        for (int k = 0; k < K; k++) {
            const int pk = __shfl_sync(0xFFFFFFFFu, moves ? p : -1, k);
            if (pk == tid) followers |= 1u << k;
        }
        const unsigned on = __ballot_sync(0xFFFFFFFFu, followers != 0u);
        const int at = __popc(on & ((1u << tid) - 1u));
        if (followers != 0u) { src[at] = tid; dst[at] = followers; }
        if (tid == 0) n_src = __popc(on);
    }
    __syncthreads();
    const int n = n_src;
    if (n == 0) return;
    const int64_t pos = a.positions ? (int64_t)max(a.positions[seq], 0) : 0;
    const int64_t o0 = col0 / st.cols;
    const int rest = (int)(col0 - o0 * st.cols) + tid;
    const int64_t outer = o0 + rest / st.cols;
    const int col = rest % st.cols;
    const int64_t i0 = outer % st.size[0], o1 = outer / st.size[0], i1 = o1 % st.size[1], i2 = o1 / st.size[1];
    if (i2 >= st.size[2]) return;
    int64_t limit = st.inner;
    if (a.positions) {
        if (st.pos_dim == 0 && i0 >= pos) return;
        if (st.pos_dim == 1 && i1 >= pos) return;
        if (st.pos_dim == 2 && i2 >= pos) return;
        if (st.pos_dim == 3) limit = min(limit, pos * st.pos_bytes);
    }
    const int64_t off = (int64_t)col * st.vec;
    const int64_t left = limit - off;
    if (left <= 0) return;
    char *p = st.data + (int64_t)seq * K * st.row_stride + i0 * st.stride[0] + i1 * st.stride[1] + i2 * st.stride[2] + off;
    if (left >= st.vec) {
        switch (st.vec) {
            case 16: move_column<MOVES, uint4>(p, st.row_stride, src, dst, n); break;
            case 8: move_column<MOVES, uint2>(p, st.row_stride, src, dst, n); break;
            case 4: move_column<MOVES, uint32_t>(p, st.row_stride, src, dst, n); break;
            case 2: move_column<MOVES, uint16_t>(p, st.row_stride, src, dst, n); break;
            default: move_column<MOVES, uint8_t>(p, st.row_stride, src, dst, n); break;
        }
    } else {
        for (int b = 0; b < (int)left; b++) move_column<MOVES, uint8_t>(p + b, st.row_stride, src, dst, n);
    }
}

// Whether rows and runs of the state lie apart: every dimension's stride reaches past all that the smaller ones span.
static bool nested(const StgBeamState &s, int64_t rows)
{
    int64_t span = s.inner_bytes;
    std::pair<int64_t, int64_t> d[4] = {{s.row_stride, rows}, {s.stride[0], s.size[0]}, {s.stride[1], s.size[1]}, {s.stride[2], s.size[2]}};
    std::sort(d, d + 4);
    for (auto &x : d) {
        if (x.second == 1) continue;
        if (x.first < span || x.first > INT64_MAX / 4 / x.second) return false;
        span += x.first * (x.second - 1);
    }
    return true;
}

// `b` split into what the kernel works on; false: nothing of it is to be moved
static bool move_state(const StgBeamState &b, int n_positions, MoveState &m)
{
    memset(&m, 0, sizeof(m));
    m.data = (char *)b.data;
    m.row_stride = b.row_stride;
    m.inner = b.inner_bytes;
    m.pos_bytes = b.position_bytes;
    m.pos_dim = b.position_dim;
    for (int i = 0; i < 3; i++) { m.stride[i] = b.stride[i]; m.size[i] = b.size[i]; }
    if (n_positions >= 0 && b.position_dim == 3) m.inner = std::min(m.inner, (int64_t)n_positions * b.position_bytes);
    if (n_positions >= 0 && b.position_dim >= 0 && b.position_dim < 3) m.size[b.position_dim] = std::min(m.size[b.position_dim], n_positions);
    if (m.inner <= 0 || m.size[0] <= 0 || m.size[1] <= 0 || m.size[2] <= 0) return false;
    uint64_t bits = (uint64_t)(uintptr_t)m.data | (uint64_t)m.row_stride;
    for (int i = 0; i < 3; i++)
        if (m.size[i] > 1) bits |= (uint64_t)m.stride[i];
    m.vec = 16;
    while (bits % (uint64_t)m.vec != 0) m.vec >>= 1;
    while (m.vec > 1 && m.vec > m.inner) m.vec >>= 1;
    return true;
}

static int reorder(StgHandle h, const StgBeamReorder *r, cudaStream_t stream)
{
    if (!r || r->struct_size != (int32_t)sizeof(StgBeamReorder)) return fail(h, STG_ERR_INVALID_ARGUMENT, "bad StgBeamReorder");
    int rc = beam_check_rows(h, "stg_beam_reorder", r->n_seq, r->n_beams);
    if (rc) return rc;
    if (r->n_states < 0 || (r->n_states > 0 && !r->states)) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_reorder: states are missing");
    if (r->mem_flags & ~(uint32_t)STG_MEM_HISTORY_RING) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_reorder: mem_flags knows STG_MEM_HISTORY_RING only");
    const int64_t rows = (int64_t)r->n_seq * r->n_beams;
    for (int i = 0; i < r->n_states; i++) {
        const StgBeamState &s = r->states[i];
        if (s.inner_bytes < 0 || s.size[0] < 0 || s.size[1] < 0 || s.size[2] < 0 || s.position_dim < -1 || s.position_dim > 3 ||
            (s.position_dim == 3 && s.position_bytes <= 0))
            return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_reorder: state " + std::to_string(i) + " has a bad size or position dimension");
        if (rows == 0 || s.inner_bytes == 0 || s.size[0] == 0 || s.size[1] == 0 || s.size[2] == 0) continue;
        if (!s.data) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_reorder: state " + std::to_string(i) + " has no data");
        if (!nested(s, rows)) return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_reorder: rows or runs of state " + std::to_string(i) + " overlap");
    }
    std::vector<StgBeamState> ring;
    if (rows > 0 && (r->mem_flags & STG_MEM_HISTORY_RING)) {
        int longest = 0;
        for (int64_t x = 0; x < rows; x++) {
            const int64_t first = x - x % r->n_beams;
            if (h->ring_len[x] != h->ring_len[first] || h->ring_dropped[x] != h->ring_dropped[first])
                return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_reorder: the histories of a sequence's beams differ in length");
            longest = std::max(longest, h->ring_len[x]);
        }
        StgBeamState s;
        memset(&s, 0, sizeof(s));
        s.data = h->ring_ids.p;
        s.row_stride = (int64_t)std::max(h->cfg.max_history, 1) * 4;
        s.inner_bytes = (int64_t)longest * 4;
        s.size[0] = s.size[1] = s.size[2] = 1;
        s.position_dim = -1;
        ring.push_back(s);
    }
    if (rows == 0 || r->n_beams == 1) return STG_OK;
    if (!r->parents || misaligned(r->parents, 4) || misaligned(r->positions, 4))
        return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_reorder: parents are missing, or an array is not aligned to its elements");
    CK(cudaSetDevice(h->cfg.device));
    const int total = r->n_states + (int)ring.size();
    std::vector<MoveState> moves;  // all of it is checked before any of it is moved
    for (int i = 0; i < total; i++) {
        MoveState m;
        if (!move_state(i < r->n_states ? r->states[i] : ring[0], r->positions ? -1 : r->n_positions, m)) continue;
        const int64_t cols = (m.inner + m.vec - 1) / m.vec;
        const int64_t runs = (int64_t)m.size[0] * m.size[1];
        if (cols > INT32_MAX / 2 || runs > INT64_MAX / 8 / cols / m.size[2])
            return fail(h, STG_ERR_UNSUPPORTED, "stg_beam_reorder: state " + std::to_string(i) + " is too large");
        m.cols = (int32_t)cols;
        m.seq_tiles = (cols * runs * m.size[2] + kMoveThreads - 1) / kMoveThreads;
        if (m.seq_tiles > INT32_MAX / r->n_seq) return fail(h, STG_ERR_UNSUPPORTED, "stg_beam_reorder: state " + std::to_string(i) + " is too large");
        moves.push_back(m);
    }
    MoveArgs a;
    a.n_states = 0;
    a.beams = r->n_beams;
    a.parents = r->parents;
    a.positions = r->positions;
    int64_t tiles = 0;
    auto launch = [&]() -> int {
        if (a.n_states == 0) return STG_OK;
        const unsigned grid = (unsigned)tiles;
        if (r->n_beams <= 4) k_beam_move<4><<<grid, kMoveThreads, 0, stream>>>(a);
        else if (r->n_beams <= 8) k_beam_move<8><<<grid, kMoveThreads, 0, stream>>>(a);
        else if (r->n_beams <= 16) k_beam_move<16><<<grid, kMoveThreads, 0, stream>>>(a);
        else k_beam_move<32><<<grid, kMoveThreads, 0, stream>>>(a);
        CK(cudaGetLastError());
        h->stats.kernel_launches++;
        a.n_states = 0;
        tiles = 0;
        return STG_OK;
    };
    for (MoveState &m : moves) {
        if (a.n_states == kMoveStates || tiles + m.seq_tiles * r->n_seq > INT32_MAX) {
            rc = launch();
            if (rc) return rc;
        }
        m.first_tile = tiles;
        tiles += m.seq_tiles * r->n_seq;
        a.st[a.n_states++] = m;
    }
    return launch();
}

}  // namespace stg

extern "C" int stg_beam_reorder(StgHandle h, const StgBeamReorder *r, void *stream)
{
    if (!h) return STG_ERR_INVALID_ARGUMENT;
    try {
        return stg::reorder(h, r, (cudaStream_t)stream);
    } catch (const std::bad_alloc &) {
        return STG_ERR_CAPACITY;
    }
}
