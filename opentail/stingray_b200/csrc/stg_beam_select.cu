// stg_beam_select: the best continuations of every sequence over its beams and the vocabulary.
//
// With x the logits of beam k, m their maximum and S = sum exp(x - m), candidate (k, v) scores
//     score[k] + ((x[v] - m) - log S)
// in 64 bits.  Within a beam the order is that of the logits alone, so a row is read once: a running maximum, a
// running sum, and the list of its best logits as 64-bit keys (stg_select.cuh); the scores are made for the few
// that are left when a sequence's rows come together.  The terms of S are computed and added up in 32 bits over the 16 or
// 32 elements that a thread holds, in 64 beyond: their roundings (1e-7 each, either way) leave about 1e-8 of S, so two
// beams' candidates change places only if they lie closer than that.
//
// A row is cut into pieces, one CTA each, and the CTA that ends last joins a sequence's pieces: one launch.
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
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamList = 1024;    // a piece's list in shared memory, a power of two
constexpr int kMergeList = 512;    // a sequence's
constexpr int kMergeParts = 2048;  // pieces of a sequence's rows together
// What is no candidate - -infinity - lies at or below this key.
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

// A thread's share of a tile, U loads of E elements, kept as it was read: bf16 stays packed, two to a word, unless a soft
// cap makes other numbers of it.  VEC: loads of 16 bytes, element e of load u is (u * 256 + thread) * E + e of the tile; else
// single elements, (u * E + e) * 256 + thread: the same for every row, so that equal rows have equal sums.
template <bool BF16, bool VEC, bool CAP>
struct BeamTile {
    static constexpr int E = BF16 ? 8 : 4;
    static constexpr int U = 4;
    static constexpr int kLen = kBeamThreads * U * E;
    static constexpr bool kPacked = BF16 && !CAP;
    static constexpr uint32_t kLow = kPacked ? 0xFF80FF80u : 0xFF800000u;  // -infinity
    uint32_t w[U][kPacked ? E / 2 : E];

    static __device__ __forceinline__ int at(int u, int e)
    {
        return VEC ? (u * kBeamThreads + (int)threadIdx.x) * E + e : (u * E + e) * kBeamThreads + (int)threadIdx.x;
    }
    __device__ __forceinline__ float get(int u, int e) const
    {
        if constexpr (kPacked) return (e & 1) ? bf16_hi(w[u][e / 2]) : bf16_lo(w[u][e / 2]);
        else return __uint_as_float(w[u][e]);
    }
    __device__ __forceinline__ void set_low(int u, int e)
    {
        if constexpr (kPacked) w[u][e / 2] = (e & 1) ? (w[u][e / 2] & 0xFFFFu) | 0xFF800000u : (w[u][e / 2] & 0xFFFF0000u) | 0xFF80u;
        else w[u][e] = 0xFF800000u;
    }
    __device__ __forceinline__ void one(const LogitRow row, int u, int e, int j)
    {
        if constexpr (kPacked) {
            const uint32_t x = __ldg((const uint16_t *)row.p + j);
            w[u][e / 2] = (e & 1) ? (w[u][e / 2] & 0xFFFFu) | (x << 16) : (w[u][e / 2] & 0xFFFF0000u) | x;
        } else {
            w[u][e] = __float_as_uint(load_one<BF16>(row, j));
        }
    }

    // The tile that starts at `base`; masked elements and those at or beyond `end` read as -infinity.  A vector without an
    // allowed element is not read.
    __device__ __forceinline__ void load(const LogitRow row, const uint32_t *mrow, int base, int end)
    {
        uint32_t allowed[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            allowed[u] = 0xFFu;
            if (mrow == nullptr) continue;
            const int i = base + at(u, 0);
            if constexpr (VEC) {
                allowed[u] = i < end ? (uint32_t)__ldg((const uint8_t *)mrow + (i >> 3)) >> (i & 7) : 0u;
                if (!BF16) allowed[u] &= 0xFu;
            } else {
                allowed[u] = 0u;
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (base + at(u, e) < end && mask_bit(mrow, base + at(u, e))) allowed[u] |= 1u << e;
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = base + at(u, 0);
#pragma unroll
            for (int x = 0; x < (kPacked ? E / 2 : E); x++) w[u][x] = kLow;
            if (VEC && i + E <= end) {
                if (allowed[u] == 0u) continue;
                if constexpr (BF16) {
                    const uint4 t = __ldcs((const uint4 *)((const uint16_t *)row.p + i));
                    if constexpr (kPacked) {
                        w[u][0] = t.x; w[u][1] = t.y; w[u][2] = t.z; w[u][3] = t.w;
                    } else {
                        const uint32_t p[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
                        for (int e = 0; e < E; e++) w[u][e] = (e & 1) ? p[e / 2] & 0xFFFF0000u : p[e / 2] << 16;
                    }
                } else {
                    const uint4 t = __ldcs((const uint4 *)((const float *)row.p + i));
                    w[u][0] = t.x; w[u][1] = t.y; w[u][2] = t.z; w[u][3] = t.w;
                }
                if constexpr (CAP)
#pragma unroll
                    for (int e = 0; e < E; e++) w[u][e] = __float_as_uint(soft_cap(get(u, e), row.cap));
            } else {
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (base + at(u, e) < end && (allowed[u] >> e & 1u)) one(row, u, e, base + at(u, e));
            }
        }
        if (VEC && mrow != nullptr)
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (!(allowed[u] >> e & 1u)) set_low(u, e);
    }
};

// exp(d), d <= 0 or little above it: 2 to the power of d * log2(e), whose low bits log2(e) needs two floats for
static __device__ __forceinline__ float beam_exp(float d)
{
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(d, 1.9259629e-8f, d * 1.44269502f)));
    return e;
}

struct RowShared {
    u64 list[kBeamList];
    uint32_t tops[kBeamThreads];  // largest logits of the first tile
    float ref[kBeamWarps], top[kBeamWarps];
    double sum[kBeamWarps];
    u64 thr;                      // later elements are among the n best only above this key
    int cnt;
};

struct MergeShared {
    u64 score[kMergeList], key[kMergeList];  // candidates: score, and logit and token
    uint8_t beam[kMergeList];
    float top[kMergeParts];                  // largest logit of a piece
    uint16_t open[kMergeParts];              // pieces that hold a candidate
    uint32_t tops[kBeamThreads];
    double base[STG_BEAM_MAX_BEAMS];         // a beam's candidates score base + (logit - ref); -infinity: it has none
    float ref[STG_BEAM_MAX_BEAMS];
    u64 bound;                               // candidates with a lower score are not among the n best
    uint32_t head;                           // ... the same, as a float rounded down
    uint32_t flags;
    int cnt, n_open;
};

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

// Leaves the n best of the list, sorted, and the n-th as the bound.  All threads; the list has settled.
static __device__ void keep_best(RowShared &sh, int n)
{
    const int c = sh.cnt, tid = threadIdx.x;
    if (c > kBeamThreads) {
        sort_list(sh.list, c);
    } else {  // every entry counts those ahead of it: the keys are distinct
        const u64 mine = tid < c ? sh.list[tid] : 0ull;
        int ahead = kBeamThreads;
        if (tid < c) {
            ahead = 0;
            for (int i = 0; i < c; i++) ahead += sh.list[i] > mine;
        }
        __syncthreads();
        if (ahead < n) sh.list[ahead] = mine;
        __syncthreads();
    }
    if (tid == 0) {
        sh.cnt = min(c, n);
        if (c >= n) sh.thr = sh.list[n - 1];
    }
    __syncthreads();
}

// The n-th largest of `tops` (`len` entries, a multiple of 32), found by counting; published by the thread that holds it.
static __device__ __forceinline__ bool is_nth(const uint32_t *tops, int len, int n)
{
    const int tid = threadIdx.x;
    if (tid >= len) return false;
    const uint32_t mine = tops[tid];
    int ahead = 0;
    for (int i = 0; i < len; i += 4) {
        const uint4 t = *(const uint4 *)(tops + i);
        ahead += (t.x > mine || (t.x == mine && i < tid)) + (t.y > mine || (t.y == mine && i + 1 < tid)) +
                 (t.z > mine || (t.z == mine && i + 2 < tid)) + (t.w > mine || (t.w == mine && i + 3 < tid));
    }
    return ahead == n - 1;
}

// One piece of a row: its sum and its n best logits, into the workspace.
template <bool BF16, bool VEC, bool CAP>
static __device__ __forceinline__ void beam_piece(const BeamSelect &a, RowShared &sh, int row, int piece)
{
    typedef BeamTile<BF16, VEC, CAP> T;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n;
    const LogitRow lr{(const char *)a.logits + (int64_t)row * a.row_stride * (BF16 ? 2 : 4), CAP ? a.softcap : 0.f};
    const uint32_t *mrow = a.mask != nullptr && (a.uses_mask == nullptr || a.uses_mask[row]) ? a.mask + (int64_t)row * a.mask_stride : nullptr;
    const int begin = piece * a.piece_len, end = min(a.vocab, begin + a.piece_len);
    if (tid == 0) { sh.cnt = 0; sh.thr = kNoKey; }
    __syncthreads();
    float ref = -CUDART_INF_F;  // the sum's terms are exp(x - ref); the same for a warp
    float best = -CUDART_INF_F;
    double s = 0.0;

    for (int base = begin; base < end; base += T::kLen) {
        T t;
        t.load(lr, mrow, base, end);
        float top = -CUDART_INF_F;
#pragma unroll
        for (int u = 0; u < T::U; u++)
#pragma unroll
            for (int e = 0; e < T::E; e++) top = fmaxf(top, t.get(u, e));
        best = fmaxf(best, top);
        // The reference need not be the maximum: it follows when a logit is so far above it that terms grow large.
        if (__any_sync(0xFFFFFFFFu, top > ref + 16.f)) {
            const float now = unord32(__reduce_max_sync(0xFFFFFFFFu, ord32(fmaxf(top, ref))));
            s *= exp((double)ref - (double)now);
            ref = now;
        }
        const float r = ref == -CUDART_INF_F ? 0.f : ref;  // nothing yet but -infinity, and NaN, which the sum has to show
        float part = 0.f;
#pragma unroll
        for (int u = 0; u < T::U; u++)
#pragma unroll
            for (int e = 0; e < T::E; e++) part += beam_exp(t.get(u, e) - r);
        s += (double)part;

        if (base == begin) {
            // At least n elements are as large as the n-th largest of the maxima of disjoint groups of them: 64 groups
            // bound it well for up to 32, and are counted through in a quarter of the time of 256.
            const int groups = n <= 32 ? 64 : kBeamThreads;
            float g = top;
            if (n <= 32) {
                g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, 1));
                g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, 2));
                if ((tid & 3) == 0) sh.tops[tid >> 2] = ord32(g);
            } else {
                sh.tops[tid] = ord32(g);
            }
            __syncthreads();
            if (is_nth(sh.tops, groups, n) && sh.tops[tid] > (uint32_t)(kNoKey >> 32)) sh.thr = (u64)sh.tops[tid] << 32;
            __syncthreads();
        }
        u64 bound = sh.thr;
        const float low = key_val(bound);
        const int before = sh.cnt;
        if (!__syncthreads_or(top >= low && top > -CUDART_INF_F)) continue;
        if (top >= low) {
#pragma unroll
            for (int u = 0; u < T::U; u++)
#pragma unroll
                for (int e = 0; e < T::E; e++) {
                    const float x = t.get(u, e);
                    if (x >= low) {
                        const u64 key = make_key(x, base + T::at(u, e));
                        if (key > bound) {
                            const int slot = atomicAdd(&sh.cnt, 1);
                            if (slot < kBeamList) sh.list[slot] = key;
                        }
                    }
                }
        }
        __syncthreads();
        const int c = sh.cnt;
        if (c > kBeamList) {
            // More than there is room for (a row that ascends, or one of equal logits): once more, one element of every
            // thread at a time.
            __syncthreads();
            if (tid == 0) sh.cnt = before;
#pragma unroll
            for (int u = 0; u < T::U; u++)
#pragma unroll
                for (int e = 0; e < T::E; e++) {
                    __syncthreads();
                    const int now = sh.cnt;
                    __syncthreads();  // read by all before anyone appends
                    if (now > kBeamList - kBeamThreads) {
                        keep_best(sh, n);
                        bound = sh.thr;
                    }
                    const float x = t.get(u, e);
                    const u64 key = make_key(x, base + T::at(u, e));
                    if (x >= key_val(bound) && key > bound) sh.list[atomicAdd(&sh.cnt, 1)] = key;
                }
            __syncthreads();
            keep_best(sh, n);
        } else if (c >= 2 * n) {
            keep_best(sh, n);
        }
    }

    keep_best(sh, n);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        best = fmaxf(best, __shfl_xor_sync(0xFFFFFFFFu, best, o));
    }
    if (lane == 0) { sh.sum[warp] = s; sh.ref[warp] = ref; sh.top[warp] = best; }
    __syncthreads();
    const int64_t at = (int64_t)row * a.pieces + piece;
    for (int i = tid; i < n; i += kBeamThreads) a.ws.keys[at * n + i] = i < sh.cnt ? sh.list[i] : 0ull;
    if (warp == 0) {
        const float wr = sh.ref[lane & 7];
        float r = wr, b = sh.top[lane & 7];
        double ws = sh.sum[lane & 7];
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            r = fmaxf(r, __shfl_xor_sync(0xFFFFFFFFu, r, o));
            b = fmaxf(b, __shfl_xor_sync(0xFFFFFFFFu, b, o));
        }
        if (wr != r) ws *= exp((double)wr - (double)r);  // 0 for a warp that has read -infinity alone
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) ws += __shfl_xor_sync(0xFFFFFFFFu, ws, o);
        if (lane == 0) a.ws.parts[at] = BeamPart{ws, r, b};
    }
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

static __device__ __forceinline__ double beam_score(const MergeShared &sh, int k, float x)
{
    return ((double)x - (double)sh.ref[k]) + sh.base[k];
}

// Leaves the n best candidates of the list, in order.  All threads; the list has settled.
static __device__ void keep_candidates(MergeShared &sh, int n)
{
    constexpr int kOwn = kMergeList / kBeamThreads;
    const int c = sh.cnt, tid = threadIdx.x;
    u64 s[kOwn], w[kOwn];
    uint8_t k[kOwn];
    int rank[kOwn];
#pragma unroll
    for (int r = 0; r < kOwn; r++) {
        const int e = r * kBeamThreads + tid;
        rank[r] = kMergeList;
        if (e >= c) continue;
        s[r] = sh.score[e]; w[r] = sh.key[e]; k[r] = sh.beam[e];
        int ahead = 0;
        for (int o = 0; o < c; o++) {
            const u64 x = sh.score[o];
            if (x < s[r]) continue;
            ahead += x > s[r] || sh.beam[o] < k[r] || (sh.beam[o] == k[r] && sh.key[o] > w[r]);
        }
        rank[r] = ahead;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kOwn; r++)
        if (rank[r] < n) { sh.score[rank[r]] = s[r]; sh.key[rank[r]] = w[r]; sh.beam[rank[r]] = k[r]; }
    __syncthreads();
    if (tid == 0) {
        sh.cnt = min(c, n);
        if (c >= n) sh.bound = sh.score[n - 1];
    }
    __syncthreads();
}

// The candidates of one sequence out of its rows' pieces, which other CTAs have written: read past the first-level cache.
static __device__ __forceinline__ void beam_merge(const BeamSelect &a, MergeShared &sh, int seq)
{
    const int tid = threadIdx.x, lane = tid & 31;
    const int K = a.beams, n = a.n, C = a.pieces, P = K * C;
    const BeamPart *parts = a.ws.parts + (int64_t)seq * P;
    const u64 *keys = a.ws.keys + (int64_t)seq * P * n;
    if (tid == 0) { sh.cnt = 0; sh.n_open = 0; sh.bound = 0ull; sh.head = 0u; sh.flags = 0u; }
    __syncthreads();
    for (int k = tid >> 5; k < K; k += kBeamWarps) {
        const int row = seq * K + k;
        const float score = a.scores[row];
        const bool alive = score > -CUDART_INF_F && score < CUDART_INF_F;
        float r = -CUDART_INF_F;
        double s = 0.0;
        for (int c = lane; c < C; c += 32) {
            BeamPart p{0.0, -CUDART_INF_F, -CUDART_INF_F};
            if (alive) {
                const uint4 raw = __ldcg((const uint4 *)(parts + k * C + c));
                p.s = __hiloint2double((int)raw.y, (int)raw.x);
                p.ref = __uint_as_float(raw.z);
                p.top = __uint_as_float(raw.w);
            }
            sh.top[k * C + c] = p.top;
            const float now = fmaxf(r, p.ref);
            if (now != r) s *= exp((double)r - (double)now);
            s += p.ref == now ? p.s : p.s * exp((double)p.ref - (double)now);
            r = now;
        }
        float m = r;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        if (r != m) s *= exp((double)r - (double)m);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        if (lane == 0) {
            const bool none = m == -CUDART_INF_F && s == 0.0;        // dead, or nothing in the row
            const bool bad = !none && !(s > 0.0 && s < CUDART_INF);  // NaN or +infinity among the logits
            const double logs = log(s);
            sh.base[k] = none || bad ? -CUDART_INF : (double)score - logs;
            sh.ref[k] = m;
            if (bad) atomicOr(&sh.flags, STG_BEAM_BAD_ROW);
            if (alive && none) atomicOr(&sh.flags, STG_ROW_FULLY_MASKED);
            if (a.log_norms) a.log_norms[row] = none ? -CUDART_INF_F : (float)((double)m + logs);
        }
    }
    __syncthreads();
    // The n-th largest of the pieces' best candidates (of groups of pieces, one per thread) bounds all others from below.
    // Rounded down to 32 bits, which keeps their order.
    uint32_t mine = 0u;
    for (int p = tid; p < P; p += kBeamThreads) {
        const int k = p / C;
        if (sh.base[k] > -CUDART_INF && sh.top[p] > -CUDART_INF_F) mine = max(mine, ord32(__double2float_rd(beam_score(sh, k, sh.top[p]))));
    }
    sh.tops[tid] = mine;
    __syncthreads();
    const int groups = min(kBeamThreads, (P + 31) & ~31);
    if (n <= groups && is_nth(sh.tops, groups, n)) sh.head = mine;
    __syncthreads();
    const uint32_t head = sh.head;
    for (int p = tid; p < P; p += kBeamThreads) {
        const int k = p / C;
        if (sh.base[k] > -CUDART_INF && sh.top[p] > -CUDART_INF_F && ord32(__double2float_rd(beam_score(sh, k, sh.top[p]))) >= head)
            sh.open[atomicAdd(&sh.n_open, 1)] = (uint16_t)p;
    }
    __syncthreads();
    const int total = sh.n_open * n;
    for (int first = 0; first < total; first += kBeamThreads) {
        const int i = first + tid;
        if (i < total) {
            const int p = sh.open[i / n], k = p / C;
            const u64 key = __ldcg(keys + (int64_t)p * n + i % n);
            if (key != 0ull) {
                const double v = beam_score(sh, k, key_val(key));
                const u64 s = ord64(v);
                if (ord32(__double2float_rd(v)) >= head && s >= sh.bound) {
                    const int at = atomicAdd(&sh.cnt, 1);
                    sh.score[at] = s; sh.key[at] = key; sh.beam[at] = (uint8_t)k;
                }
            }
        }
        __syncthreads();
        const bool full = sh.cnt > kMergeList - kBeamThreads;
        __syncthreads();  // read by all before anyone appends
        if (full) keep_candidates(sh, n);
    }
    keep_candidates(sh, n);
    const int c = sh.cnt;
    for (int i = tid; i < n; i += kBeamThreads) {
        const int64_t o = (int64_t)seq * n + i;
        a.tokens[o] = i < c ? key_idx(sh.key[i]) : -1;
        a.parents[o] = i < c ? (int)sh.beam[i] : -1;
        a.out_scores[o] = i < c ? (float)unord64(sh.score[i]) : -CUDART_INF_F;
    }
    if (tid == 0 && a.flags) a.flags[seq] = sh.flags | (c < n ? (uint32_t)STG_BEAM_SHORT : 0u);
}

// grid (pieces, rows).  The CTA that arrives last at its sequence's ticket joins the sequence's pieces and leaves the ticket
// at zero, as it was found.
template <bool BF16, bool VEC, bool CAP>
__global__ void __launch_bounds__(kBeamThreads, BF16 && CAP ? 3 : 5) k_beam_select(const __grid_constant__ BeamSelect a)
{
    __shared__ union { RowShared row; MergeShared merge; } sh;
    __shared__ bool last;
    const int row = blockIdx.y, seq = row / a.beams;
    const float score = a.scores[row];
    if (score > -CUDART_INF_F && score < CUDART_INF_F) beam_piece<BF16, VEC, CAP>(a, sh.row, row, blockIdx.x);  // else a dead beam
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        last = atomicAdd(a.ws.tickets + seq, 1u) == (uint32_t)(a.beams * a.pieces - 1);
        if (last) a.ws.tickets[seq] = 0u;
        __threadfence();
    }
    __syncthreads();
    if (last) beam_merge(a, sh.merge, seq);
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

// How many CTAs share a row: the cut that gives the busiest SM the least, where a CTA's first tile costs about half a tile more
// than the others.  A tile of a CTA by itself takes about three times as long as one of a full SM, so few rows are
// cut into single tiles.
static void beam_pieces(int rows, int beams, int vocab, int tile, int sms, int &pieces, int &len)
{
    const int tiles = (vocab + tile - 1) / tile;
    const int most = std::max(1, std::min({tiles, kMergeParts / beams, kBeamExtraPieces / rows + 1}));
    double least = 0.0;
    pieces = 1;
    for (int c = 1; c <= most; c++) {
        const int per = (tiles + c - 1) / c, got = (tiles + per - 1) / per;
        if (got != c) continue;
        const double cost = std::max((double)(((int64_t)rows * c + sms - 1) / sms) * (per + 0.5) * 0.3, per + 1.0);
        if (c == 1 || cost < least) { least = cost; pieces = c; }
    }
    len = (tiles + pieces - 1) / pieces * tile;
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
    const int tile = 4096 * (b->logits_dtype == STG_DTYPE_BF16 ? 2 : 1);
    beam_pieces(rows, b->n_beams, b->vocab, tile, h->sm_count, a.pieces, a.piece_len);

    const size_t b_parts = round_up((size_t)rows * a.pieces * sizeof(BeamPart), 256), b_keys = round_up((size_t)rows * a.pieces * a.n * 8, 256);
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    CK(cudaStreamIsCapturing(stream, &cap));
    const bool captured = cap != cudaStreamCaptureStatusNone;
    char *ws = (char *)h->bm_ws.p;
    a.ws.tickets = (uint32_t *)h->bm_tickets.p;
    if (captured) {
        void *own = nullptr;
        rc = captured_workspace(h, b_parts + b_keys + (size_t)b->n_seq * 4, &own);
        ws = (char *)own;
        a.ws.tickets = (uint32_t *)(ws + b_parts + b_keys);
    } else {
        if (b_parts + b_keys > h->bm_ws.bytes) return fail(h, STG_ERR_CAPACITY, "stg_beam_select: workspace too small");
        rc = order_behind_last(h, stream);
    }
    if (rc) return rc;
    a.ws.parts = (BeamPart *)ws;
    a.ws.keys = (u64 *)(ws + b_parts);
    if (captured) CK(cudaMemsetAsync(a.ws.tickets, 0, (size_t)b->n_seq * 4, stream));  // part of the graph
    const bool vec = !misaligned(b->logits, 16) && (rows == 1 || (size_t)b->row_stride * esz % 16 == 0);
    const bool capped = b->logit_softcap != 0.f;
    void (*fn)(BeamSelect);
    if (b->logits_dtype == STG_DTYPE_BF16) fn = vec ? (capped ? k_beam_select<true, true, true> : k_beam_select<true, true, false>)
                                                    : (capped ? k_beam_select<true, false, true> : k_beam_select<true, false, false>);
    else fn = vec ? (capped ? k_beam_select<false, true, true> : k_beam_select<false, true, false>)
                  : (capped ? k_beam_select<false, false, true> : k_beam_select<false, false, false>);
    fn<<<dim3((unsigned)a.pieces, (unsigned)rows), kBeamThreads, 0, stream>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(h, e, "k_beam_select launch");
    h->stats.calls++;
    h->stats.kernel_launches++;
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
