// stg_beam_select: the best continuations of every sequence over its beams and the vocabulary.
//
// With x the logits of beam k, S = sum exp(x - r) for any r near their maximum, candidate (k, v) scores
//     score[k] + ((x[v] - r) - log S)
// in 64 bits.  Within a beam the order is that of the logits alone, and S is not known before the row has been read, so
// the pass over the logits selects nothing: it adds up S and keeps the maximum of every group of 512 (fp32) or 1024 (bf16)
// neighbouring logits.  Order the groups of all beams of a sequence by the score of their best candidate, equal ones as
// candidates are: n groups have n candidates that are ahead of everything in the groups behind them, so the n best
// candidates lie in the n best groups, whatever ties.  The CTA that ends last with a sequence finds those groups and
// reads them once more.  One launch, no barrier and no list in the pass.
//
// The terms of S are computed in 32 bits.  The 16 or 32 that a thread holds are added up in 32 bits, halves to one another, and
// in 64 beyond.  Where one of them makes next to nothing of the others - a logit far above the rest, as of a model that is sure -
// 64 bits add them up from the first on, and every warp's largest term is put right in 64.  What that leaves of S: 1.0e-8 in the mean
// square on rows of N(0, 2.5^2), up to 4.8e-8 with one logit 8 to 21 above a rest of N(0, 0.5^2) to N(0, 6^2), 5.9e-8 at most
// (256 rows each of 50,257, 151,936 and 262,144, both types); the exponential's own error, 2^-22 at most, where most of S is
// equal logits (1.4e-7 at most over flat rows).  Two beams' candidates change places only if they lie closer than that.
//
// What bounds it: the pass by HBM, 95 % of the copy rate on 256 rows of 151,936 fp32 (155 MB in 25 us); the join by latency,
// 7 us for four beams and 13 for sixteen, of which only the last sequences' shows.
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>
#include <string.h>

#include <new>

#include "stg_beam.h"
#include "stg_pdl.cuh"
#include "stg_select.cuh"
#include "stg_types.h"

namespace stg {

constexpr int kBeamThreads = 512;
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamList = 512;  // candidates in shared memory

struct BeamSelect {
    const void *logits;
    int64_t row_stride;
    const float *scores;
    const uint32_t *mask;
    int64_t mask_stride;
    const uint8_t *uses_mask;
    float softcap;
    int32_t n_seq, beams, vocab, n;
    int32_t pieces, piece_len, groups;  // CTAs of a row, their elements, and the row's groups
    BeamWs ws;
    int32_t *tokens, *parents;
    float *out_scores, *log_norms;
    uint32_t *flags;
};

// A thread's share of a tile, U loads of E elements, kept as it was read: bf16 stays packed, two to a word, unless a soft
// cap makes other numbers of it.  A warp's share is a group, kGroup neighbouring elements.  VEC: loads of 16 bytes, element e of
// load u is (u * 32 + lane) * E + e of the group.  Else fp32 (u * E + e) * 32 + lane, one at a time, and bf16 (u * E + (e & ~1)) * 32 +
// 2 * lane + (e & 1), two at a time in rows that begin at 4 bytes (304 rows of 192,782: 37.6 us, one at a time 47.5; 43.8 of 192,783,
// where every other row does).  The same for every row of a call, so that equal rows have equal sums.
template <bool BF16, bool VEC, bool CAP>
struct BeamTile {
    static constexpr int E = BF16 ? 8 : 4;
    static constexpr int U = 4;
    static constexpr int kGroup = 32 * U * E;
    static constexpr int kLen = kBeamWarps * kGroup;
    static constexpr bool kPacked = BF16 && !CAP;
    uint32_t w[U][kPacked ? E / 2 : E];

    static __device__ __forceinline__ int at(int u, int e)
    {
        const int lane = threadIdx.x & 31;
        return VEC ? (u * 32 + lane) * E + e : BF16 ? (u * E + (e & ~1)) * 32 + 2 * lane + (e & 1) : (u * E + e) * 32 + lane;
    }
    __device__ __forceinline__ float get(int u, int e) const
    {
        if constexpr (kPacked) return (e & 1) ? bf16_hi(w[u][e / 2]) : bf16_lo(w[u][e / 2]);
        else return __uint_as_float(w[u][e]);
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
    __device__ __forceinline__ void two(const LogitRow row, int u, int e, int j)
    {
        const uint32_t x = __ldcs((const uint32_t *)((const uint16_t *)row.p + j));
        if constexpr (kPacked) {
            w[u][e / 2] = x;
        } else {
            w[u][e] = x << 16;
            w[u][e + 1] = x & 0xFFFF0000u;
            if constexpr (CAP) {
                w[u][e] = __float_as_uint(soft_cap(get(u, e), row.cap));
                w[u][e + 1] = __float_as_uint(soft_cap(get(u, e + 1), row.cap));
            }
        }
    }
    __device__ __forceinline__ void whole(const LogitRow row, int i, int u)
    {
        const uint4 t = BF16 ? __ldcs((const uint4 *)((const uint16_t *)row.p + i)) : __ldcs((const uint4 *)((const float *)row.p + i));
        if constexpr (kPacked || !BF16) {
            w[u][0] = t.x; w[u][1] = t.y; w[u][2] = t.z; w[u][3] = t.w;
        } else {
            const uint32_t p[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
            for (int e = 0; e < E; e++) w[u][e] = (e & 1) ? p[e / 2] & 0xFFFF0000u : p[e / 2] << 16;
        }
        if constexpr (CAP)
#pragma unroll
            for (int e = 0; e < E; e++) w[u][e] = __float_as_uint(soft_cap(get(u, e), row.cap));
    }

    __device__ __forceinline__ float top() const
    {
        if constexpr (kPacked) {
            uint32_t m = w[0][0];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int x = 0; x < E / 2; x++) asm("max.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[u][x]));
            return fmaxf(fmaxf(-CUDART_INF_F, bf16_lo(m)), bf16_hi(m));
        } else {
            float m = -CUDART_INF_F;
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int e = 0; e < E; e += 2) asm("max.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(get(u, e)), "f"(get(u, e + 1)));
            return m;
        }
    }

    // Which elements of the thread's share of the group at `base` are allowed, bit u * E + e.  Behind `end` a mask's bits say nothing.
    static __device__ __forceinline__ uint32_t allowed(const uint32_t *mrow, int base, int end)
    {
        if (mrow == nullptr) return 0xFFFFFFFFu;
        uint32_t ok = 0u;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = base + at(u, 0);
            if constexpr (VEC) {
                const uint32_t b = i < end ? (uint32_t)__ldg((const uint8_t *)mrow + (i >> 3)) >> (i & 7) : 0u;
                ok |= (b & (BF16 ? 0xFFu : 0xFu)) << (u * E);
            } else if constexpr (BF16) {
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const int j = base + at(u, e);
                    const uint32_t b = j < end ? __ldg(mrow + (j >> 5)) >> (j & 31) : 0u;
                    ok |= (b & (j + 1 < end ? 3u : 1u)) << (u * E + e);
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; e++) {  // a word for all lanes, of which each has one bit
                    const int j = base + at(u, e);
                    const uint32_t b = j < end ? __ldg(mrow + (j >> 5)) >> (j & 31) : 0u;
                    ok |= (b & 1u) << (u * E + e);
                }
            }
        }
        return ok;
    }
    // The group that starts at `base`; elements that are not `ok` and those at or beyond `end` read as -infinity.  A vector
    // without an allowed element is not read.
    __device__ __forceinline__ void load(const LogitRow row, bool masked, uint32_t ok, int base, int end)
    {
        if (!masked && base + kGroup <= end) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                if constexpr (VEC) {
                    whole(row, base + at(u, 0), u);
                } else if (BF16 && ((uintptr_t)row.p & 3) == 0) {
#pragma unroll
                    for (int e = 0; e < E; e += 2) two(row, u, e, base + at(u, e));
                } else {
#pragma unroll
                    for (int e = 0; e < E; e++) one(row, u, e, base + at(u, e));
                }
            }
            return;
        }
        constexpr uint32_t kAll = BF16 ? 0xFFu : 0xFu;
#pragma unroll
        for (int u = 0; u < U; u++) {
#pragma unroll
            for (int x = 0; x < (kPacked ? E / 2 : E); x++) w[u][x] = kPacked ? 0xFF80FF80u : 0xFF800000u;
            if (VEC && base + at(u, 0) + E <= end) {
                if (ok >> (u * E) & kAll) whole(row, base + at(u, 0), u);
            } else if (!VEC && BF16 && ((uintptr_t)row.p & 3) == 0 && base + kGroup <= end) {
#pragma unroll
                for (int e = 0; e < E; e += 2)
                    if (ok >> (u * E + e) & 3u) two(row, u, e, base + at(u, e));
            } else {
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (base + at(u, e) < end && (ok >> (u * E + e) & 1u)) one(row, u, e, base + at(u, e));
            }
        }
    }
    // The allowed elements where a mask leaves a thread no more than `some`, kLeast or kFew, each by a load of its own, as numbers; of
    // a group that does not reach beyond the row
    static constexpr int kFew = 8, kLeast = 4, kWords = kPacked ? E / 2 : E;
    __device__ __forceinline__ void load_few(const LogitRow row, uint32_t ok, int some, int base)
    {
#pragma unroll
        for (int q = 0; q < kFew; q++) {
            if (q == kLeast && some == kLeast) break;
            const int b = __ffs(ok) - 1;
            ok &= ok - 1u;
            uint32_t x = 0xFF800000u;
            if (b >= 0) {
                const int j = base + at(b / E, b % E);
                x = BF16 ? (uint32_t)__ldg((const uint16_t *)row.p + j) << 16 : __ldg((const uint32_t *)row.p + j);
            }
            w[q / kWords][q % kWords] = x;
        }
    }
    __device__ __forceinline__ void cap_few(uint32_t ok, float cap)
    {
        if constexpr (CAP)
#pragma unroll
            for (int q = 0; q < kFew; q++)
                if (q < __popc(ok)) w[q / kWords][q % kWords] = __float_as_uint(soft_cap(few(q), cap));
    }
    __device__ __forceinline__ float few(int q) const { return __uint_as_float(w[q / kWords][q % kWords]); }

    // ... once the loads are back
    __device__ __forceinline__ void mask(uint32_t ok)
    {
        if (ok == 0xFFFFFFFFu || (!VEC && !BF16)) return;  // fp32 elements that are read one by one are read if allowed
#pragma unroll
        for (int u = 0; u < U; u++)
            if constexpr (kPacked) {
#pragma unroll
                for (int x = 0; x < E / 2; x++) {  // a byte permutation takes each half from the word or from -infinity
                    const uint32_t two = ok >> (u * E + 2 * x) & 3u;
                    w[u][x] = __byte_perm(0xFF80FF80u, w[u][x], 0x3210u + ((two | two << 7) & 0x101u) * 0x44u);
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (!(ok >> (u * E + e) & 1u)) w[u][e] = 0xFF800000u;
            }
    }
};

typedef unsigned long long f32x2;
static __device__ __forceinline__ f32x2 pair(float a, float b)
{
    f32x2 p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
static __device__ __forceinline__ void unpair(f32x2 p, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
static __device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b)
{
    f32x2 c;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(c) : "l"(a), "l"(b));
    return c;
}
static __device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c)
{
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// exp(x) / 2^c of two numbers, as 2^(x log2(e) - c), for which log2(e) takes two floats: one alone is off by 1.3e-8, which a
// row's sum would be off by times its logits' distance from zero.  The product with the first is not rounded before
// c is taken off.
static __device__ __forceinline__ f32x2 exp_pair(f32x2 x, f32x2 minus_c)
{
    float a, b;
    unpair(fma2(x, pair(1.9259629e-8f, 1.9259629e-8f), fma2(x, pair(1.44269502f, 1.44269502f), minus_c)), a, b);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    return pair(a, b);
}

static __device__ __forceinline__ float warp_max(float v)
{
    asm("redux.sync.max.f32 %0, %0, 0xFFFFFFFF;" : "+f"(v));
    return v;
}
static __device__ __forceinline__ float warp_min(float v)
{
    asm("redux.sync.min.f32 %0, %0, 0xFFFFFFFF;" : "+f"(v));
    return v;
}

// The sum of term(FIRST) .. term(FIRST + N - 1), halves added to one another: a large term takes part in log2(N) additions, not N, and
// terms that are small beside it have been added to one another by then
template <int FIRST, int N, class Term>
static __device__ __forceinline__ f32x2 halves(const Term &term)
{
    if constexpr (N == 1) return term(FIRST);
    else return add2(halves<FIRST, N / 2>(term), halves<FIRST + N / 2, N / 2>(term));
}
template <int N, class Term>
static __device__ __forceinline__ double sum64(const Term &term)
{
    double a = 0.0, b = 0.0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        float x, y;
        unpair(term(i), x, y);
        a += (double)x;
        b += (double)y;
    }
    return a + b;
}

constexpr double kLn2 = 0.69314718055994530942;
constexpr float kHuge = 1e6f;  // logits beyond take the slow way: c could not tell them apart
// How far a thread's largest logit lies below the warp's where small terms may be lost beside large ones: what is less than
// 2^-24 = e^-16.6 of a sum is, what a sum's own rounding can hide starts earlier.  At 10 a single logit 12 above a rest of
// N(0, 0.5^2) leaves 2.5e-8 of S; at 12 it would 7e-8.  Rows of N(0, 2.5^2) never come here; of those of N(0, 4^2) 9 in 100 groups do, of N(0, 6^2) 30:
// 512 bf16 rows of 256,000 take 62.3, 65.2 and 69.5 us, without this 62 all three; 256 fp32 rows of 151,936 36 to 36.4 us.
constexpr float kApart = 10.f;

// What a sum's terms are relative to: 2^c, c a whole number; or exp(logit) where that is not 0, -infinity as long as there
// are none.
struct BeamRef {
    float c, logit;
    __device__ __forceinline__ double natural() const { return logit != 0.f ? (double)logit : (double)c * kLn2; }
};
static __device__ __noinline__ double exp64(double x) { return exp(x); }

// What a sum relative to `from` is multiplied by to be relative to `to`: without rounding where both are powers of two
static __device__ __noinline__ double scale(BeamRef from, BeamRef to)
{
    if (from.logit == 0.f && to.logit == 0.f) {
        const int by = (int)(from.c - to.c);
        return by < -1022 ? 0.0 : __hiloint2double((1023 + min(by, 1023)) << 20, 0);
    }
    return from.logit == -CUDART_INF_F ? 0.0 : exp(from.natural() - to.natural());
}

// The largest reference of a warp, or one that 32 bits do not tell from it
static __device__ __forceinline__ BeamRef warp_ref(BeamRef r)
{
    const float f = (float)r.natural();
    const int lane = __ffs(__ballot_sync(0xFFFFFFFFu, f == warp_max(f))) - 1;
    return BeamRef{__shfl_sync(0xFFFFFFFFu, r.c, lane), __shfl_sync(0xFFFFFFFFu, r.logit, lane)};
}

// The sum of exp(x - top) over a group with logits beyond kHuge, element by element, eight loads in flight (64 rows of 151,936
// logits of some 1e6: 17.5 us, 27.9 one load after the other).
template <bool BF16, bool VEC, bool CAP>
static __device__ __noinline__ double huge_group(const LogitRow lr, const uint32_t *mrow, int base, int end, float top)
{
    double part = 0.0;
#pragma unroll 8
    for (int j = 0; j < BeamTile<BF16, VEC, CAP>::kGroup / 32; j++) {
        const int i = base + 32 * j + (int)(threadIdx.x & 31);
        if (i < end && (mrow == nullptr || mask_bit(mrow, i))) part += (double)expf(load_one<BF16>(lr, i) - top);
    }
    return part;
}

// One piece of a row: its part of the sum and the maxima of its groups.
template <bool BF16, bool VEC, bool CAP, bool MASK>
static __device__ __forceinline__ void beam_piece(const BeamSelect &a, int row, int piece)
{
    typedef BeamTile<BF16, VEC, CAP> T;
    __shared__ double sums[kBeamWarps];
    __shared__ BeamRef refs[kBeamWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const LogitRow lr{(const char *)a.logits + (int64_t)row * a.row_stride * (BF16 ? 2 : 4), CAP ? a.softcap : 0.f};
    const uint32_t *mrow = MASK && (a.uses_mask == nullptr || a.uses_mask[row]) ? a.mask + (int64_t)row * a.mask_stride : nullptr;
    const int begin = piece * a.piece_len + warp * T::kGroup, end = min(a.vocab, (piece + 1) * a.piece_len);
    float *tops = a.ws.tops + (int64_t)row * a.groups;
    // The sum's terms are exp(x) / 2^c; the same c for a warp.  2^c lies near the largest, as the exponent's rounding goes with
    // its size, and follows when a logit is `limit` or more.
    BeamRef ref{0.f, -CUDART_INF_F};
    float limit = -CUDART_INF_F, best = -CUDART_INF_F;
    double s = 0.0;
    // A group's loads are in flight while the one ahead of it is added up, its mask's a group earlier still.  Behind a mask that leaves
    // no thread more than four or eight elements of its 32 bf16 ones - densities up to about a tenth - these alone are read and added up
    // (256 rows of 262,144, densities of 0.1, 1, 5, 10 and 20 %: 29, 32, 41, 45 and 50 us, all in the long way 46, 46, 47, 47 and 47).
    // Of the 16 fp32 ones that a thread has it is no gain: 41, 49, 57, 62 and 64 against 53, 56, 58, 59 and 59.
    constexpr int kDense = 32;
    const auto most = [&](uint32_t bits, int at) {
        if (!MASK || !BF16 || mrow == nullptr || at + T::kGroup > end) return kDense;
        const int m = (int)__reduce_max_sync(0xFFFFFFFFu, (unsigned)__popc(bits));
        return m > T::kFew ? kDense : m > T::kLeast ? T::kFew : T::kLeast;
    };
    uint32_t ok = T::allowed(mrow, begin, end), next_ok = T::allowed(mrow, begin + T::kLen, end);
    int some = most(ok, begin);
    T next;
    if (begin < end) {
        if (some < kDense) next.load_few(lr, ok, some, begin);
        else next.load(lr, mrow != nullptr, ok, begin, end);
    }
#pragma unroll 1
    for (int base = begin; base < end; base += T::kLen) {
        T t = next;
        const int few = some;
        if (few < kDense) t.cap_few(ok, lr.cap); else t.mask(ok);
        ok = next_ok;
        if (base + T::kLen < end) {
            some = most(ok, base + T::kLen);
            if (some < kDense) next.load_few(lr, ok, some, base + T::kLen);
            else next.load(lr, mrow != nullptr, ok, base + T::kLen, end);
            next_ok = T::allowed(mrow, base + 2 * T::kLen, end);
        }
        float own = -CUDART_INF_F;
        if (few < kDense) {
#pragma unroll
            for (int q = 0; q < T::kFew; q += 2) {
                if (q == T::kLeast && few == T::kLeast) break;
                own = fmaxf(own, fmaxf(t.few(q), t.few(q + 1)));
            }
        } else {
            own = t.top();
        }
        const float top = warp_max(own);
        if (lane == 0) tops[base / T::kGroup] = top;
        if ((fabsf(top) > kHuge || ref.logit > kHuge) && top > -CUDART_INF_F) {
            if ((double)top > ref.natural()) {
                const BeamRef now{0.f, top};
                s *= scale(ref, now);
                ref = now;
                limit = -CUDART_INF_F;  // no c any more
            }
            s += huge_group<BF16, VEC, CAP>(lr, mrow, base, end, top) * exp64((double)top - ref.natural());
            continue;
        }
        // Terms that are next to nothing beside another of the same thread are lost in a sum of 32 bits, one after the other.  Where that
        // is in sight and counts - the warp's largest so far is here, and some thread's largest lies far below it - 64 bits add up.
        const bool apart = top >= best && top - warp_min(own > -CUDART_INF_F ? own : CUDART_INF_F) > kApart;
        best = fmaxf(best, top);
        if (top > limit) {
            const BeamRef now{floorf(top * 1.44269502f), 0.f};
            s *= scale(ref, now);
            ref = now;
            limit = (now.c + 4.f) * 0.693147181f;
        }
        const f32x2 minus_c = pair(-ref.c, -ref.c);
        const auto few_term = [&](int i) { return exp_pair(pair(t.few(2 * i), t.few(2 * i + 1)), minus_c); };
        const auto term = [&](int i) {
            const int u = i / (T::E / 2), e = i % (T::E / 2) * 2;
            return exp_pair(pair(t.get(u, e), t.get(u, e + 1)), minus_c);
        };
        constexpr int kPairs = T::U * T::E / 2;
        if (apart) {
            s += few == kDense ? sum64<kPairs>(term) : few == T::kFew ? sum64<T::kFew / 2>(few_term) : sum64<T::kLeast / 2>(few_term);
            continue;
        }
        float p0, p1;
        unpair(few == kDense ? halves<0, kPairs>(term) : few == T::kFew ? halves<0, T::kFew / 2>(few_term) : halves<0, T::kLeast / 2>(few_term), p0, p1);
        s += (double)(p0 + p1);
    }
    // The largest term was made with the c that there is now.  Where a row's sum is little more than its largest term, that one's
    // error is the sum's, so the warps' largest are put right: 64 bits in place of what was added.
    if (lane == 0 && ref.logit == 0.f && best > -CUDART_INF_F) {
        float was, unused;
        unpair(exp_pair(pair(best, best), pair(-ref.c, -ref.c)), was, unused);
        s += exp64((double)best - ref.natural()) - (double)was;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (lane == 0) { sums[warp] = s; refs[warp] = ref; }
    __syncthreads();
    if (warp == 0) {
        const BeamRef wr = refs[lane % kBeamWarps], r = warp_ref(wr);
        double ws = sums[lane % kBeamWarps] * scale(wr, r);  // 0 for a warp that has read -infinity alone
#pragma unroll
        for (int o = kBeamWarps / 2; o > 0; o >>= 1) ws += __shfl_xor_sync(0xFFFFFFFFu, ws, o);
        if (lane == 0) a.ws.parts[(int64_t)row * a.pieces + piece] = BeamPart{ws, r.c, r.logit};
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

// What is ordered: groups, by their best candidate, and candidates.  `score` is the score as ord64; `rest` decides between equal
// ones: the lower beam, then the larger logit, then the lower group or token.
struct BeamItem {
    u64 score, rest;
};
constexpr int kPosBits = 27;  // 5 bits for the beam, 32 for the logit
constexpr u64 kPosMask = (1ull << kPosBits) - 1ull;
static __device__ __forceinline__ u64 item_rest(float x, int k, int pos)
{
    return (u64)(STG_BEAM_MAX_BEAMS - 1 - k) << 59 | (u64)ord32(x) << kPosBits | (kPosMask - (u64)pos);
}
static __device__ __forceinline__ int item_beam(u64 rest) { return STG_BEAM_MAX_BEAMS - 1 - (int)(rest >> 59); }
static __device__ __forceinline__ float item_logit(u64 rest) { return unord32((uint32_t)(rest >> kPosBits)); }
static __device__ __forceinline__ int item_pos(u64 rest) { return (int)(kPosMask - (rest & kPosMask)); }
static __device__ __forceinline__ bool ahead_of(const BeamItem a, const BeamItem b)
{
    return a.score > b.score || (a.score == b.score && a.rest > b.rest);
}

constexpr int kStage = 8;  // loads of a thread in flight, 8 of 4 bytes or 4 of 16
struct MergeShared {
    union {
        float head[kStage][kBeamThreads];
        uint4 vec[kStage / 2][kBeamThreads];
    } stage;
    BeamItem list[kBeamList];
    uint32_t tops[256];
    double sum[STG_BEAM_MAX_BEAMS];    // S of a beam, relative to ref
    double ref[STG_BEAM_MAX_BEAMS];
    double base[STG_BEAM_MAX_BEAMS];   // a beam's candidates score base + (logit - ref)
    float about[STG_BEAM_MAX_BEAMS];   // ... about that + logit
    float least[STG_BEAM_MAX_BEAMS];   // no smaller logit reaches `low`; NaN: the beam has no candidates
    int group[STG_BEAM_MAX_CANDIDATES];          // the groups that are read again
    uint8_t group_beam[STG_BEAM_MAX_CANDIDATES];
    float size;                        // the largest |about| + |ref| of the beams
    uint32_t low;                      // a float, as ord32, that n candidates reach in `about`; 0: none
    uint32_t masked;                   // bit k: beam k's row goes by its mask
    uint32_t flags;
    int cnt;

    __device__ __forceinline__ u64 score_of(int k, float x) const { return ord64(((double)x - ref[k]) + base[k]); }
    // x + about is off by a few roundings (2^-24) of x, of what `about` was made of - the normaliser's logarithm, at most 46
    // beside `ref`, among it - and of the sum.
    __device__ __forceinline__ void set_least(int k)
    {
        if (low == 0u || !(about[k] > -CUDART_INF_F)) return;  // no bound, or a beam without candidates
        const float l = unord32(low), x = l - about[k];
        least[k] = x - (1e-6f * (fabsf(x) + fabsf(l)) + 2e-6f * size + 2e-5f);
    }
    // More than the list takes have come: nothing of it will be used, so nobody need come any more
    __device__ __forceinline__ bool full() const { return *(const volatile int *)&cnt > kBeamList; }
    // x has reached `least`: it may be one of the n best.  Its score is made when all have come.
    __device__ __forceinline__ void offer(float x, int k, int pos)
    {
        if (full()) return;
        const int at = atomicAdd(&cnt, 1);
        if (at < kBeamList) list[at].rest = item_rest(x, k, pos);
    }
    // The same with its score at once, unless it is behind `bound`
    __device__ __noinline__ void offer_from(float x, int k, int pos, const BeamItem bound)
    {
        const BeamItem item{score_of(k, x), item_rest(x, k, pos)};
        if (ahead_of(bound, item)) return;
        const int at = atomicAdd(&cnt, 1);
        if (at < kBeamList) list[at] = item;
    }
};

// The code below runs once per call and sequence, so what it takes is latency, that of fetching its instructions
// included: loops are left rolled and what is used twice is a function, while loads are issued several at a time.

// `low` out of every thread's best item (its x + about; -infinity: none), such that n of them reach it.  Up to 32: the n-th
// largest of 64 groups of threads, made distinct by their last six bits, for each of which four threads count those above
// it.  Beyond: the upper 20 bits of the n-th largest of 256, found two by two, which takes longer.  0 where there are no n.
// Meanwhile `aside` is called by a warp that has nothing to do with it.  All threads.
template <class Aside>
static __device__ __forceinline__ void find_low(MergeShared &sh, int K, int n, float best, Aside aside)
{
    const int tid = threadIdx.x;
    uint32_t mine = best > -CUDART_INF_F ? ord32(best) : 0u;
    const int per = n <= 32 ? kBeamThreads / 64 : kBeamThreads / 256;
#pragma unroll
    for (int o = 1; o < kBeamThreads / 64; o *= 2)
        if (o < per) mine = max(mine, __shfl_xor_sync(0xFFFFFFFFu, mine, o));
    if (n <= 32) mine = mine >= 64u ? (mine & ~63u) | (63u - (unsigned)(tid / per)) : 0u;
    if (tid % per == 0) sh.tops[tid / per] = mine;
    __syncthreads();
    if (tid >= 256) {
        if (tid < 288) aside(tid - 256);
        if (tid >= 288 && tid < 320) {
            const int k = tid - 288;
            const float size = warp_max(k < K && sh.about[k] > -CUDART_INF_F ? fabsf(sh.about[k]) + fabsf((float)sh.ref[k]) : 0.f);
            if (k == 0) sh.size = size;
        }
    } else if (n <= 32) {
        mine = sh.tops[tid / 4];
        int ahead = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint4 v = *(const uint4 *)(sh.tops + (tid % 4 + 4 * i) * 4);
            ahead += (v.x > mine) + (v.y > mine) + (v.z > mine) + (v.w > mine);
        }
        ahead += __shfl_xor_sync(0xFFFFFFFFu, ahead, 1);
        ahead += __shfl_xor_sync(0xFFFFFFFFu, ahead, 2);
        if (ahead == n - 1 && tid % 4 == 0) sh.low = max(sh.low, mine & ~63u);
    } else if (tid < 32) {
        uint32_t v[8], found = 0u;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = sh.tops[tid + 32 * i];
#pragma unroll 1
        for (int shift = 30; shift >= 12; shift -= 2) {
            const uint32_t t1 = found | (1u << shift), t2 = found | (2u << shift), t3 = found | (3u << shift);
            uint32_t reach = 0u;  // three counts of up to 256
#pragma unroll
            for (int i = 0; i < 8; i++) reach += (v[i] >= t1 ? 1u : 0u) + (v[i] >= t2 ? 1u << 10 : 0u) + (v[i] >= t3 ? 1u << 20 : 0u);
            reach = __reduce_add_sync(0xFFFFFFFFu, reach);
            if ((reach >> 20) >= (uint32_t)n) found = t3;
            else if ((reach >> 10 & 1023u) >= (uint32_t)n) found = t2;
            else if ((reach & 1023u) >= (uint32_t)n) found = t1;
        }
        if (tid == 0) sh.low = max(sh.low, found);
    }
    __syncthreads();
    if (tid < K) sh.set_least(tid);
    __syncthreads();
}

// Sorts the first c entries of the list, best first (bitonic; what it is filled up with is behind everything).  All threads.
static __device__ __noinline__ void sort_list(MergeShared &sh, int c)
{
    int len = 32;
    while (len < c) len <<= 1;
    for (int i = c + (int)threadIdx.x; i < len; i += kBeamThreads) sh.list[i] = BeamItem{0ull, 0ull};
    __syncthreads();
    for (int k = 2; k <= len; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int t = threadIdx.x; t < len / 2; t += kBeamThreads) {
                const int a = 2 * j * (t / j) + t % j, b = a + j;
                const BeamItem x = sh.list[a], y = sh.list[b];
                if (ahead_of(y, x) == ((a & k) == 0)) { sh.list[a] = y; sh.list[b] = x; }
            }
            __syncthreads();
        }
}

// Hands the n best of a list of c entries to emit(place, rest, score), in whatever order.  Few: eight threads per entry count
// those ahead of it, no two being the same.  All threads; the list has settled.
template <class Emit>
static __device__ __forceinline__ void rank_list(MergeShared &sh, int c, int n, Emit emit)
{
    constexpr int kPer = 8;
    const int tid = threadIdx.x, sub = tid % kPer;
    if (c > 4 * (kBeamThreads / kPer)) {  // 512 entries: 45 steps of the sort against 8 rounds of 64
        sort_list(sh, c);
        if (tid < min(c, n)) emit(tid, sh.list[tid].rest, sh.list[tid].score);
        return;
    }
#pragma unroll 1
    for (int first = 0; first < c; first += kBeamThreads / kPer) {
        const int e = first + tid / kPer;
        BeamItem mine{0ull, 0ull};
        int ahead = 0;
        if (e < c) {
            mine = sh.list[e];
#pragma unroll 4
            for (int o = sub; o < c; o += kPer) ahead += ahead_of(sh.list[o], mine);
        }
#pragma unroll
        for (int o = kPer / 2; o > 0; o >>= 1) ahead += __shfl_xor_sync(0xFFFFFFFFu, ahead, o);
        if (e < c && sub == 0 && ahead < n) emit(ahead, mine.rest, mine.score);
    }
}

// After items have been offered: the list holds the n best of them and perhaps more; how many.  Where more were offered than
// it takes - equal ones, a row that ascends - get(i, x, k, pos) for i below `total` is gone through again, every thread a stretch
// of its own, until the list is full; the n-th best of what it holds then is a bound for the next time.  As the list is
// an even sample, that leaves about n of kBeamList.
template <class Get>
static __device__ __forceinline__ int settle(MergeShared &sh, int total, int n, Get get)
{
    const int tid = threadIdx.x;
    __syncthreads();
    int c = sh.cnt;
    if (c <= kBeamList) {
#pragma unroll 1
        for (int i = tid; i < c; i += kBeamThreads) sh.list[i].score = sh.score_of(item_beam(sh.list[i].rest), item_logit(sh.list[i].rest));
        __syncthreads();
        return c;
    }
    const int stretch = (total + kBeamThreads - 1) / kBeamThreads;
    BeamItem bound{0ull, 0ull};
    for (;;) {  // ends: of a full list all but n entries are behind the next bound
        __syncthreads();  // cnt and the list have been read by all
        if (tid == 0) sh.cnt = 0;
        __syncthreads();
#pragma unroll 1
        for (int i = tid * stretch; i < min(total, (tid + 1) * stretch) && !sh.full(); i++) {
            float x;
            int k, pos;
            if (get(i, x, k, pos) && x >= sh.least[k] && x > -CUDART_INF_F) sh.offer_from(x, k, pos, bound);
        }
        __syncthreads();
        c = sh.cnt;
        if (c <= kBeamList) return c;
        __syncthreads();
        sort_list(sh, kBeamList);
        bound = sh.list[n - 1];
    }
}

// The candidates of one sequence out of its rows' sums and group maxima, which other CTAs have written: read past the
// first-level cache.
template <bool BF16, bool VEC, bool CAP, bool MASK>
static __device__ __forceinline__ void beam_merge(const BeamSelect &a, MergeShared &sh, int seq)
{
    typedef BeamTile<BF16, VEC, CAP> T;
    const int tid = threadIdx.x, lane = tid & 31;
    const int K = a.beams, n = a.n, C = a.pieces, G = a.groups, heads = K * G;
    const float *tops = a.ws.tops + (int64_t)seq * heads;
    float head[kStage];
    auto load_heads = [&](int from) {
#pragma unroll
        for (int j = 0; j < kStage; j++) head[j] = from + j * kBeamThreads + tid < heads ? __ldcg(tops + from + j * kBeamThreads + tid) : -CUDART_INF_F;
    };
    auto stage_heads = [&]() {
#pragma unroll
        for (int j = 0; j < kStage; j++) sh.stage.head[j][tid] = head[j];  // a thread reads what it wrote
    };
    load_heads(0);
    if (tid == 0) { sh.cnt = 0; sh.low = 0u; sh.flags = 0u; }
    if (MASK && tid < 32) {
        const unsigned on = __ballot_sync(0xFFFFFFFFu, a.mask != nullptr && tid < K && (a.uses_mask == nullptr || a.uses_mask[seq * K + tid]));
        if (tid == 0) sh.masked = on;
    }
    __syncthreads();
#pragma unroll 1
    for (int k = tid >> 5; k < K; k += kBeamWarps) {
        const int row = seq * K + k;
        const float score = a.scores[row];
        const bool alive = score > -CUDART_INF_F && score < CUDART_INF_F;
        BeamRef r{0.f, -CUDART_INF_F};
        double s = 0.0;
#pragma unroll 1
        for (int c = lane; c < C; c += 32) {
            const uint4 raw = __ldcg((const uint4 *)(a.ws.parts + (int64_t)row * C + c));  // of a dead beam: not written, not used
            const BeamRef p{__uint_as_float(raw.z), __uint_as_float(raw.w)};
            const double ps = __hiloint2double((int)raw.y, (int)raw.x);
            if (c < 32) {  // the only one as a rule
                s = ps;
                r = p;
            } else {
                const BeamRef now = p.natural() > r.natural() ? p : r;
                s = s * scale(r, now) + ps * scale(p, now);
                r = now;
            }
        }
        if (!alive) { r = BeamRef{0.f, -CUDART_INF_F}; s = 0.0; }
        const BeamRef row_ref = warp_ref(r);
        const double m = row_ref.natural();
        s *= scale(r, row_ref);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        if (lane == 0) {
            const bool none = m == -CUDART_INF && s == 0.0;          // dead, or nothing in the row
            const bool bad = !none && !(s > 0.0 && s < CUDART_INF);  // NaN or +infinity among the logits
            sh.sum[k] = s;
            sh.ref[k] = m;
            sh.about[k] = none || bad ? -CUDART_INF_F : (score - logf((float)s)) - (float)m;
            sh.least[k] = none || bad ? CUDART_NAN_F : -CUDART_INF_F;
            if (bad) atomicOr(&sh.flags, STG_BEAM_BAD_ROW);
            if (alive && none) atomicOr(&sh.flags, STG_ROW_FULLY_MASKED);
        }
    }
    stage_heads();
    __syncthreads();

    // ---- the n best groups.  First a bound: the n-th of the threads' best, of which 32 bits are enough. ----
    float best = -CUDART_INF_F;
    auto norms = [&](int k) {  // what takes 64
        if (k >= K) return;
        const double logs = log(sh.sum[k]);
        sh.base[k] = (double)a.scores[seq * K + k] - logs;
        if (a.log_norms) a.log_norms[seq * K + k] = sh.sum[k] == 0.0 ? -CUDART_INF_F : (float)(sh.ref[k] + logs);
    };
#pragma unroll 1
    for (int pass = 0; pass < 2; pass++) {
        int k = (int)((unsigned)tid / (unsigned)G), g = tid - k * G;  // of head i, which goes up by kBeamThreads
#pragma unroll 1
        for (int from = 0; from < heads; from += kStage * kBeamThreads) {
            if (heads > kStage * kBeamThreads) {
                load_heads(from);
                stage_heads();
            }
#pragma unroll 2
            for (int j = 0; j < kStage; j++) {
                const int i = from + j * kBeamThreads + tid;
                if (i >= heads) break;
                const float x = sh.stage.head[j][tid];
                if (x >= sh.least[k] && x > -CUDART_INF_F) {
                    if (pass == 0) best = fmaxf(best, x + sh.about[k]); else sh.offer(x, k, g);
                }
                if (i + kBeamThreads >= heads) break;
                for (g += kBeamThreads; g >= G; g -= G) k++;
            }
        }
        if (pass == 0) find_low(sh, K, n, best, norms);
    }
    int c = settle(sh, heads, n, [&](int i, float &x, int &k, int &g) {
        k = (int)((unsigned)i / (unsigned)G);
        g = i - k * G;
        x = __ldcg(tops + i);
        return true;
    });
    rank_list(sh, c, n, [&](int to, u64 rest, u64) {
        const int k = item_beam(rest);
        sh.group[to] = item_pos(rest);
        sh.group_beam[to] = (uint8_t)k;
        if (to == n - 1) sh.low = max(sh.low, ord32(item_logit(rest) + sh.about[k]));  // a candidate of each of n groups reaches it
    });
    __syncthreads();

    // ---- the n best candidates, which lie in them ----
    const int open = min(c, n);
    if (tid < K) sh.set_least(tid);
    if (tid == 0) sh.cnt = 0;
    __syncthreads();
    constexpr int E = T::E, kVecs = T::kGroup / E, kBatch = kStage / 2;
    const int vecs = open * kVecs;
    auto row_of = [&](int k) { return LogitRow{(const char *)a.logits + (int64_t)(seq * K + k) * a.row_stride * (BF16 ? 2 : 4), CAP ? a.softcap : 0.f}; };
    auto mask_of = [&](int k) { return MASK && (sh.masked >> k & 1u) ? a.mask + (int64_t)(seq * K + k) * a.mask_stride : nullptr; };
    auto first_of = [&](int i) { return sh.group[i / kVecs] * T::kGroup + i % kVecs * E; };
    // Of m groups that compete about n log(m / (m - n)) candidates of the n best reach the n-th group's best.  Where there are hardly
    // more than n, or the others' beams are far behind, that is no close bound: then the threads' best elements give one, at once
    // where it can be told, otherwise when the list has overflown.  (15 sequences of eight beams about two apart, 39,168 bf16
    // tokens, 24 candidates: 18.8 us; with the bound that found the groups, and `settle` for what overflows, 99.)
    best = -CUDART_INF_F;
    bool close = c < n || heads < 2 * n;
#pragma unroll 1
    for (int pass = close ? 0 : 1; pass < 2;) {
#pragma unroll 1
        for (int from = tid; from < vecs; from += kBatch * kBeamThreads) {
            uint4 raw[kBatch];
            uint32_t ok = MASK ? 0u : 0xFFFFFFFFu;  // bit j * E + e: the mask allows that element
#pragma unroll
            for (int j = 0; j < kBatch; j++) {
                const int i = from + j * kBeamThreads;
                raw[j] = make_uint4(0u, 0u, 0u, 0u);
                if (i >= vecs) continue;
                const int v = first_of(i), k = sh.group_beam[i / kVecs];
                const void *p = row_of(k).p;
                const uint32_t *mrow = mask_of(k);
                if (MASK && v < a.vocab) {
                    const uint32_t all = (1u << E) - 1u, some = mrow == nullptr ? all : (uint32_t)__ldg((const uint8_t *)mrow + (v >> 3)) >> (v & 7) & all;
                    ok |= some << (j * E);
                }
                if (VEC && v + E <= a.vocab) {
                    raw[j] = BF16 ? __ldg((const uint4 *)((const uint16_t *)p + v)) : __ldg((const uint4 *)((const float *)p + v));
                } else {
                    uint32_t w[4];
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        if constexpr (BF16) {
                            w[q] = v + 2 * q < a.vocab ? __ldg((const uint16_t *)p + v + 2 * q) : 0u;
                            if (v + 2 * q + 1 < a.vocab) w[q] |= (uint32_t)__ldg((const uint16_t *)p + v + 2 * q + 1) << 16;
                        } else {
                            w[q] = v + q < a.vocab ? __ldg((const uint32_t *)p + v + q) : 0u;
                        }
                    }
                    raw[j] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            uint32_t passed = 0u;  // bit j * E + e: that element reaches `least`
#pragma unroll
            for (int j = 0; j < kBatch; j++) {
                sh.stage.vec[j][tid] = raw[j];  // a thread reads what it wrote
                const int i = from + j * kBeamThreads;
                if (i >= vecs) continue;
                const int k = sh.group_beam[i / kVecs];
                float least = sh.least[k];
                // a capped logit is no further from 0 than the logit, but for roundings
                if constexpr (CAP) least = least > 0.f ? least * (1.f - 1e-6f) : -CUDART_INF_F;
                const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
                if (pass == 0) {
                    float top = -CUDART_INF_F;
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const float x = BF16 ? ((e & 1) ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2])) : __uint_as_float(w[e]);
                        if ((ok >> (j * E + e) & 1u) != 0u && first_of(i) + e < a.vocab) top = fmaxf(top, x);
                    }
                    if (top > -CUDART_INF_F) best = fmaxf(best, (CAP ? soft_cap(top, a.softcap) : top) + sh.about[k]);
                    continue;
                }
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const float x = BF16 ? ((e & 1) ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2])) : __uint_as_float(w[e]);
                    passed |= x >= least ? 1u << (j * E + e) : 0u;
                }
            }
            if (MASK) passed &= ok;
            if (pass == 0) continue;
#pragma unroll 1
            for (; passed != 0u; passed &= passed - 1u) {
                const int b = __ffs(passed) - 1, j = b / E, e = b % E, i = from + j * kBeamThreads;
                const int k = sh.group_beam[i / kVecs], v = first_of(i) + e;
                float x = BF16 ? __uint_as_float((uint32_t)((const uint16_t *)&sh.stage.vec[j][tid])[e] << 16) : ((const float *)&sh.stage.vec[j][tid])[e];
                if constexpr (CAP) x = soft_cap(x, a.softcap);
                if (x >= sh.least[k] && x > -CUDART_INF_F && v < a.vocab) sh.offer(x, k, v);
            }
        }
        if (pass == 0) {
            find_low(sh, K, n, best, [](int) {});
            pass = 1;
            continue;
        }
        __syncthreads();
        if (close || sh.cnt <= kBeamList) break;
        __syncthreads();  // all have seen that it is full
        if (tid == 0) sh.cnt = 0;
        close = true;
        pass = 0;
    }
    c = settle(sh, open * T::kGroup, n, [&](int i, float &x, int &k, int &v) {
        const int g = i / T::kGroup;
        k = sh.group_beam[g];
        v = sh.group[g] * T::kGroup + i % T::kGroup;
        const uint32_t *mrow = mask_of(k);
        if (v >= a.vocab || (mrow != nullptr && !mask_bit(mrow, v))) return false;
        x = load_one<BF16>(row_of(k), v);
        return true;
    });
    rank_list(sh, c, n, [&](int to, u64 rest, u64 score) {
        const int64_t o = (int64_t)seq * n + to;
        a.tokens[o] = item_pos(rest);
        a.parents[o] = item_beam(rest);
        a.out_scores[o] = (float)unord64(score);
    });
    if (tid >= c && tid < n) {
        const int64_t o = (int64_t)seq * n + tid;
        a.tokens[o] = a.parents[o] = -1;
        a.out_scores[o] = -CUDART_INF_F;
    }
    if (tid == 0 && a.flags) a.flags[seq] = sh.flags | (c < n ? (uint32_t)STG_BEAM_SHORT : 0u);
}
static_assert(STG_BEAM_MAX_BEAMS == 32 && STG_BEAM_MAX_CANDIDATES <= kBeamThreads && 2 * STG_BEAM_MAX_CANDIDATES <= kBeamList, "bits of an item, room in the list");

// A CTA per piece of a row; like all kernels of a search launched while the one ahead of it ends.  The CTA that arrives last at
// its sequence's ticket joins the sequence's rows and leaves the ticket at zero, as it was found.
template <bool BF16, bool VEC, bool CAP, bool MASK>
__global__ void __launch_bounds__(kBeamThreads, kBeamCtas) k_beam_select(const __grid_constant__ BeamSelect a)
{
    __shared__ MergeShared sh;
    __shared__ bool last;
    const int row = (int)(blockIdx.x / (unsigned)a.pieces), piece = (int)(blockIdx.x % (unsigned)a.pieces), seq = row / a.beams;
    pdl_release();
    pdl_wait();
    const float score = a.scores[row];
    if (score > -CUDART_INF_F && score < CUDART_INF_F) beam_piece<BF16, VEC, CAP, MASK>(a, row, piece);  // else a dead beam
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t before;  // behind the barrier: for what the whole CTA has written, and what the others have
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.ws.tickets + seq) : "memory");
        last = before == (uint32_t)(a.beams * a.pieces - 1);
        if (last) a.ws.tickets[seq] = 0u;
    }
    __syncthreads();
    if (last) beam_merge<BF16, VEC, CAP, MASK>(a, sh, seq);
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
    if ((int64_t)b->vocab > (int64_t)kPosMask) return fail(h, STG_ERR_UNSUPPORTED, "stg_beam_select: vocab beyond 2^27");
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
    const OnDevice on(h->cfg.device);
    CK(on.error);
    BeamSelect a;
    memset(&a, 0, sizeof(a));
    a.logits = b->logits; a.row_stride = b->row_stride; a.scores = b->scores;
    a.mask = b->mask; a.mask_stride = b->mask_row_stride; a.uses_mask = b->row_uses_mask;
    a.softcap = b->logit_softcap;
    a.n_seq = b->n_seq; a.beams = b->n_beams; a.vocab = b->vocab; a.n = b->n_candidates;
    a.tokens = b->tokens; a.parents = b->parents; a.out_scores = b->candidate_scores; a.log_norms = b->log_norms; a.flags = b->seq_flags;
    const int rows = b->n_seq * b->n_beams;
    const bool bf16 = b->logits_dtype == STG_DTYPE_BF16, capped = b->logit_softcap != 0.f;
    const int group = bf16 ? 1024 : 512, tile = group * kBeamWarps;
    a.groups = (b->vocab + group - 1) / group;
    beam_pieces(rows, b->vocab, tile, h->sm_count, a.pieces, a.piece_len);

    const size_t b_parts = round_up((size_t)rows * a.pieces * sizeof(BeamPart), 256), b_tops = round_up((size_t)rows * a.groups * 4, 256),
                 bytes = b_parts + b_tops;
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    CK(cudaStreamIsCapturing(stream, &cap));
    const bool captured = cap != cudaStreamCaptureStatusNone;
    char *ws = (char *)h->bm_ws.p;
    a.ws.tickets = (uint32_t *)h->bm_tickets.p;
    if (captured) {
        void *own = nullptr;
        rc = captured_workspace(h, bytes + (size_t)b->n_seq * 4, &own);
        ws = (char *)own;
        a.ws.tickets = (uint32_t *)(ws + bytes);
    } else {
        if (bytes > h->bm_ws.bytes) return fail(h, STG_ERR_CAPACITY, "stg_beam_select: workspace too small");
        rc = order_behind_last(h, stream);
    }
    if (rc) return rc;
    a.ws.parts = (BeamPart *)ws;
    a.ws.tops = (float *)(ws + b_parts);
    if (captured) CK(cudaMemsetAsync(a.ws.tickets, 0, (size_t)b->n_seq * 4, stream));  // part of the graph
    const bool vec = !misaligned(b->logits, 16) && (rows == 1 || (size_t)b->row_stride * esz % 16 == 0);
    using Kernel = void (*)(BeamSelect);
    // [bf16][vec][capped][masked]
    static const Kernel kernels[2][2][2][2] = {
        {{{k_beam_select<false, false, false, false>, k_beam_select<false, false, false, true>}, {k_beam_select<false, false, true, false>, k_beam_select<false, false, true, true>}},
         {{k_beam_select<false, true, false, false>, k_beam_select<false, true, false, true>}, {k_beam_select<false, true, true, false>, k_beam_select<false, true, true, true>}}},
        {{{k_beam_select<true, false, false, false>, k_beam_select<true, false, false, true>}, {k_beam_select<true, false, true, false>, k_beam_select<true, false, true, true>}},
         {{k_beam_select<true, true, false, false>, k_beam_select<true, true, false, true>}, {k_beam_select<true, true, true, false>, k_beam_select<true, true, true, true>}}}};
    const Kernel fn = kernels[bf16][vec][capped][b->mask != nullptr];
    const cudaError_t e = launch_behind(fn, dim3((unsigned)a.pieces * (unsigned)rows), kBeamThreads, 0, stream, a);
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
