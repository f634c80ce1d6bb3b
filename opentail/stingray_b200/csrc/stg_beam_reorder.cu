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
#include "stg_pdl.cuh"
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
    int32_t cols;         // vectors that a run can touch; the first and the last may be in part another run's
    int32_t run_tiles;    // tiles of a run; 0: a tile's columns go on from run to run
    int32_t seq_tiles;    // tiles of one sequence
    int32_t first_tile;   // of this state
    const int32_t *used;  // [n_seq * beams]: positions in use of every row, for which a sequence moves if they are one number; null: MoveArgs::positions
};

struct MoveArgs {
    MoveState st[kMoveStates];
    int32_t n_states, beams;
    const int32_t *parents, *positions;
};

// What the beams of a sequence move: rows that others continue, and where to
struct Moves {
    int64_t src[STG_BEAM_MAX_BEAMS], dst[STG_BEAM_MAX_BEAMS];  // offsets of rows
    int first[STG_BEAM_MAX_BEAMS + 1];                          // row src[i] goes to dst[first[i] .. first[i + 1])
    int n;
};

template <int MOVES, class V>
static __device__ __forceinline__ void load_rows(V (&v)[MOVES], const char *at, const Moves &m, int n)
{
#pragma unroll
    for (int i = 0; i < MOVES; i++)
        if (i < n) v[i] = *(const V *)(at + m.src[i]);
}
template <int MOVES, class V>
static __device__ __forceinline__ void store_rows(const V (&v)[MOVES], char *at, const Moves &m, int n)
{
#pragma unroll
    for (int i = 0; i < MOVES; i++)
        if (i < n)
            for (int d = m.first[i]; d < m.first[i + 1]; d++) *(V *)(at + m.dst[d]) = v[i];
}
template <int MOVES, class V>
static __device__ __forceinline__ void move_column(char *at, const Moves &m, int n)
{
    V v[MOVES];
    load_rows(v, at, m, n);
    store_rows(v, at, m, n);
}

// Fewer bytes than a vector, in pieces as large as they are aligned.  Where one end is a vector's, a size occurs once at most,
// and few rows' pieces are all loaded before any is stored.
template <int MOVES>
static __device__ __noinline__ void move_part(char *at, int bytes, int vec, const Moves &m, int n)
{
    const bool tail = ((uintptr_t)at & (unsigned)(vec - 1)) == 0, head = (((uintptr_t)at + bytes) & (unsigned)(vec - 1)) == 0;
    if (MOVES <= 8 && (tail || head)) {
        // where the pieces of 8, 4, 2 and 1 begin: large ones first behind an aligned beginning, last ahead of an aligned end
        char *const p8 = at + (tail ? 0 : bytes & 7), *const p4 = at + (tail ? bytes & 8 : bytes & 3), *const p2 = at + (tail ? bytes & 12 : bytes & 1),
             *const p1 = at + (tail ? bytes & 14 : 0);
        uint2 v8[MOVES];
        uint32_t v4[MOVES];
        uint16_t v2[MOVES];
        uint8_t v1[MOVES];
        if (bytes & 8) load_rows(v8, p8, m, n);
        if (bytes & 4) load_rows(v4, p4, m, n);
        if (bytes & 2) load_rows(v2, p2, m, n);
        if (bytes & 1) load_rows(v1, p1, m, n);
        if (bytes & 8) store_rows(v8, p8, m, n);
        if (bytes & 4) store_rows(v4, p4, m, n);
        if (bytes & 2) store_rows(v2, p2, m, n);
        if (bytes & 1) store_rows(v1, p1, m, n);
        return;
    }
#pragma unroll 1
    while (bytes > 0) {
        int by = 8;
        while (by > bytes || ((uintptr_t)at & (unsigned)(by - 1)) != 0) by >>= 1;
        switch (by) {
            case 8: move_column<MOVES, uint2>(at, m, n); break;
            case 4: move_column<MOVES, uint32_t>(at, m, n); break;
            case 2: move_column<MOVES, uint16_t>(at, m, n); break;
            default: move_column<MOVES, uint8_t>(at, m, n); break;
        }
        at += by;
        bytes -= by;
    }
}

// A tile is kMoveThreads columns of one sequence, one to a thread (two of two beams): occupancy is worth more than several columns' loads in flight
// (four beams, eight layers' caches of 1000 positions: 35.5 us with eight CTAs an SM, 40.9 with five, 43.2 with four columns
// a thread and three CTAs; 32 sequences of eight beams, 3.2 GB moved: 511 us with five CTAs, 568 with four).  More than 16
// beams move 8 bytes a thread: 199 us against 263 with 16 and one CTA an SM.  Two beams move one row or swap: two columns fit
// where four beams have one, and half the CTAs (63 sequences' caches of 1445 positions, 0.2 GB: 77.7 us, 91.8 with one column).
// Where runs are shorter than four tiles a tile's columns go on from run to run, at a division each.
constexpr int move_blocks(int moves) { return moves <= 4 ? 8 : moves <= 8 ? 5 : 3; }
__host__ __device__ constexpr int move_bytes(int beams) { return beams <= 16 ? 16 : 8; }
__host__ __device__ constexpr int move_cols(int beams) { return beams <= 2 ? 2 : 1; }  // of a thread
__host__ __device__ constexpr int tile_cols(int beams) { return move_cols(beams) * kMoveThreads; }

template <int MOVES>
__global__ void __launch_bounds__(kMoveThreads, move_blocks(MOVES)) k_beam_move(const __grid_constant__ MoveArgs a)
{
    __shared__ Moves moves;
    const int tid = threadIdx.x, K = a.beams;
    int lo = 0, hi = a.n_states - 1;  // the last state whose first tile is not behind this one
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if ((int)blockIdx.x >= a.st[mid].first_tile) lo = mid; else hi = mid - 1;
    }
    const MoveState &st = a.st[lo];
    const unsigned tile = blockIdx.x - (unsigned)st.first_tile, seq = tile / (unsigned)st.seq_tiles, in_seq = tile - seq * (unsigned)st.seq_tiles;
    pdl_release();
    pdl_wait();
    const int32_t *const used = st.used ? st.used + (int64_t)seq * K : a.positions ? a.positions + seq : nullptr;
    const int64_t pos = used ? (int64_t)max(*used, 0) : 0;
    if (tid < 32) {
        const bool alike = __all_sync(0xFFFFFFFFu, st.used == nullptr || tid >= K || used[tid] == *used);
        const int p = tid < K && alike ? a.parents[(int64_t)seq * K + tid] : -1;
        const int parent = p >= 0 && p < K && p != tid ? p : -1;
        uint32_t followers = 0u;
        for (int k = 0; k < K; k++)
            if (__shfl_sync(0xFFFFFFFFu, parent, k) == tid) followers |= 1u << k;
        const unsigned on = __ballot_sync(0xFFFFFFFFu, followers != 0u), before = (1u << tid) - 1u;
        int first = 0;  // followers of the rows ahead
        for (int k = 0; k < K; k++) {
            const int f = __popc(__shfl_sync(0xFFFFFFFFu, followers, k));
            first += k < tid ? f : 0;
        }
        if (followers != 0u) {
            const int at = __popc(on & before);
            moves.src[at] = tid * st.row_stride;
            moves.first[at] = first;
            for (uint32_t f = followers; f != 0u; f &= f - 1u) moves.dst[first++] = (__ffs(f) - 1) * st.row_stride;
            if ((on & ~before & ~(1u << tid)) == 0u) moves.first[at + 1] = first;  // the last one
        }
        if (tid == 0) moves.n = __popc(on);
    }
    __syncthreads();
    if (moves.n == 0) return;
    char *const row = st.data + (int64_t)(seq * (unsigned)K) * st.row_stride;
    const int64_t limit = used && st.pos_dim == 3 ? min(st.inner, pos * st.pos_bytes) : st.inner;
    // the run `outer`, or null where it is not to be moved
    auto run = [&](unsigned outer) -> char * {
        unsigned i0 = outer, i1 = 0u, i2 = 0u;
        if (st.size[1] > 1 || st.size[2] > 1) {
            i1 = outer / (unsigned)st.size[0]; i0 = outer - i1 * (unsigned)st.size[0];
            i2 = i1 / (unsigned)st.size[1]; i1 -= i2 * (unsigned)st.size[1];
        }
        if (i2 >= (unsigned)st.size[2] || i1 >= (unsigned)st.size[1] || i0 >= (unsigned)st.size[0]) return nullptr;
        if (used && st.pos_dim >= 0 && st.pos_dim < 3 && (int64_t)(st.pos_dim == 0 ? i0 : st.pos_dim == 1 ? i1 : i2) >= pos) return nullptr;
        return row + i0 * st.stride[0] + i1 * st.stride[1] + i2 * st.stride[2];
    };
    constexpr int kCols = move_cols(MOVES), kTile = tile_cols(MOVES);
    const int n = moves.n;
    // Columns begin at multiples of `vec` in memory, which are the same for all rows: a run's first may begin ahead of it.
    auto column = [&](int q, int64_t &begin) -> char * {
        char *r;
        unsigned c = tid + q * kMoveThreads;
        if (st.run_tiles > 0) {
            const unsigned outer = in_seq / (unsigned)st.run_tiles;
            r = run(outer);
            c += (in_seq - outer * (unsigned)st.run_tiles) * kTile;
        } else {
            const unsigned g = in_seq * kTile + c, outer = g / (unsigned)st.cols;
            r = run(outer);
            c = g - outer * (unsigned)st.cols;
        }
        begin = (int64_t)c * st.vec - (int64_t)((uintptr_t)r & (unsigned)(st.vec - 1));
        return r == nullptr || begin >= limit ? nullptr : r;
    };
    auto move = [&](char *r, int64_t begin) {
        const int64_t end = begin + st.vec;
        if (begin < 0 || end > limit) {
            move_part<MOVES>(r + max(begin, (int64_t)0), (int)(min(end, limit) - max(begin, (int64_t)0)), st.vec, moves, n);
            return;
        }
        switch (st.vec) {
            case 16:
                if constexpr (move_bytes(MOVES) == 16) move_column<MOVES, uint4>(r + begin, moves, n);
                break;
            case 8: move_column<MOVES, uint2>(r + begin, moves, n); break;
            case 4: move_column<MOVES, uint32_t>(r + begin, moves, n); break;
            case 2: move_column<MOVES, uint16_t>(r + begin, moves, n); break;
            default: move_column<MOVES, uint8_t>(r + begin, moves, n); break;
        }
    };
    if constexpr (kCols == 1) {
        int64_t begin;
        char *const r = column(0, begin);
        if (r != nullptr) move(r, begin);
    } else {
        int64_t b0, b1;
        char *const r0 = column(0, b0), *const r1 = column(1, b1);
        const bool in0 = r0 != nullptr && b0 >= 0 && b0 + 16 <= limit, in1 = r1 != nullptr && b1 >= 0 && b1 + 16 <= limit;
        if (st.vec == 16 && in0 && in1) {
            uint4 v0[MOVES], v1[MOVES];
            load_rows(v0, r0 + b0, moves, n);
            load_rows(v1, r1 + b1, moves, n);
            store_rows(v0, r0 + b0, moves, n);
            store_rows(v1, r1 + b1, moves, n);
        } else {
            if (r0 != nullptr) move(r0, b0);
            if (r1 != nullptr) move(r1, b1);
        }
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
static bool move_state(const StgBeamState &b, int beams, int n_positions, MoveState &m)
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
    m.vec = move_bytes(beams);  // as rows are apart: a run's bytes then lie alike in all of them
    while (m.row_stride % m.vec != 0) m.vec >>= 1;
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
    if (rows == 0 || r->n_beams == 1) return STG_OK;
    if (!r->parents || misaligned(r->parents, 4) || misaligned(r->positions, 4))
        return fail(h, STG_ERR_INVALID_ARGUMENT, "stg_beam_reorder: parents are missing, or an array is not aligned to its elements");
    const OnDevice on(h->cfg.device);
    CK(on.error);
    // The tokens in use of a history are read where they are appended, on the device: a captured call finds those of its replay.  The
    // host's lengths say how many there can be, and refuse beams that differ; a captured call makes room for all there ever are.
    std::vector<StgBeamState> ring;
    bool ordered = false;  // the histories are the handle's: what it has enqueued on another stream may read them still
    if (r->mem_flags & STG_MEM_HISTORY_RING) {
        cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
        CK(cudaStreamIsCapturing(stream, &cap));
        const bool captured = cap != cudaStreamCaptureStatusNone;
        int longest = captured ? h->cfg.max_history : 0;
        for (int64_t x = 0; x < rows && !captured; x++) {
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
        s.position_dim = 3;
        s.position_bytes = 4;
        ring.push_back(s);
        ordered = !captured;
    }
    const int total = r->n_states + (int)ring.size();
    std::vector<MoveState> moves;  // all of it is checked before any of it is moved
    for (int i = 0; i < total; i++) {
        MoveState m;
        const bool own = i >= r->n_states;
        if (!move_state(own ? ring[0] : r->states[i], r->n_beams, own || r->positions ? -1 : r->n_positions, m)) continue;
        if (own) m.used = (const int32_t *)h->ring_len_dev.p;
        uint64_t where = (uint64_t)(uintptr_t)m.data;
        for (int j = 0; j < 3; j++)
            if (m.size[j] > 1) where |= (uint64_t)m.stride[j];
        const int64_t cols = (m.inner + m.vec - 1) / m.vec + (where % (uint64_t)m.vec != 0 ? 1 : 0), runs = (int64_t)m.size[0] * m.size[1];
        const int64_t tile = tile_cols(r->n_beams);
        const bool too_many = cols > INT32_MAX / 2 || runs > INT32_MAX / m.size[2];
        int64_t per_seq = INT64_MAX;
        if (!too_many) {
            const bool joined = cols < 4 * tile && cols * (runs * m.size[2]) < INT32_MAX - tile;
            m.cols = (int32_t)cols;
            m.run_tiles = joined ? 0 : (int32_t)((cols + tile - 1) / tile);
            per_seq = joined ? (cols * (runs * m.size[2]) + tile - 1) / tile : m.run_tiles * (runs * m.size[2]);
        }
        if (per_seq > INT32_MAX / r->n_seq) return fail(h, STG_ERR_UNSUPPORTED, "stg_beam_reorder: state " + std::to_string(i) + " is too large");
        m.seq_tiles = (int32_t)per_seq;
        moves.push_back(m);
    }
    if (ordered) {
        rc = order_behind_last(h, stream);
        if (rc) return rc;
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
        const auto fn = r->n_beams <= 2 ? k_beam_move<2> : r->n_beams <= 4 ? k_beam_move<4> : r->n_beams <= 8 ? k_beam_move<8> : r->n_beams <= 16 ? k_beam_move<16> : k_beam_move<32>;
        CK(launch_behind(fn, dim3(grid), kMoveThreads, 0, stream, a));
        h->stats.kernel_launches++;
        a.n_states = 0;
        tiles = 0;
        return STG_OK;
    };
    for (MoveState &m : moves) {
        if (a.n_states == kMoveStates || tiles + (int64_t)m.seq_tiles * r->n_seq > INT32_MAX) {
            rc = launch();
            if (rc) return rc;
        }
        m.first_tile = (int32_t)tiles;
        tiles += (int64_t)m.seq_tiles * r->n_seq;
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
