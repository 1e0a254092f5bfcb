// Log probabilities of given tokens, entropies and the most likely alternatives, from logits, in one pass over them.
//
//   m = max x,  l = sum e^(c (x - m)),  t = sum (x - m) e^(c (x - m))          c = inv_temperature
//   lse = c m + log l,  logprob(i) = c x_i - lse,  entropy = log l - c t / l  (neither term is negative: nothing cancels)
//
// Kept per thread with a running maximum: when it grows by d, l -> l e^(-c d) and t -> (t - d l) e^(-c d).  (The maximum
// is taken off before the change to base 2: logits as low as the type goes, a common mask, stay finite.)
//
// A warp takes a row, or a part of one where there are few rows, on its own: nothing waits for a CTA, and what a unit
// costs beyond its elements (merging lanes, ranking candidates) is paid by one warp, not by eight.  The warp that finishes the
// last part of a row joins them in the order of the parts, so the result does not depend on which one that is.
//
// Alternatives ride along.  The elements a lane takes in one step of its loop are a cell; the softmax needs their maximum
// anyway.  A warp keeps, in shared memory, cells that can hold one of the best `top`: `top` or some more that come
// before all others by (maximum, step).  A cell has to exceed the least maximum kept to enter, which soon is rare
// (the n-th of a row is among the best k with probability k / n).  What is to be kept is found by bisection over the keys, which
// a few more than `top` end early, and not by sorting.  At the end the elements of the kept cells are looked at one by one.
//
// What bounds it: memory, 2 bytes an element, with the special-function unit (one exponential an element, 16 a cycle
// and SM) close behind; what it waits for is loads, two kilobytes a warp of which are under way.  4 096 rows of 50 257 fp16: 85 us
// (4.8 TB/s), 92 with one alternative, 110 with twenty (registers: 16 warps an SM instead of 24; with fewer registers the
// loop spills, 118 and 138).  64 rows of 131 072 bf16: 11 us, with twenty alternatives 21.
#include "act_layout.h"
#include "lm.h"

#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace gpx {

constexpr int kScoreThreads = 128, kScoreWarps = kScoreThreads / 32;
constexpr int kMaxTop = 32;
constexpr float kLog2e = 1.4426950408889634f;

struct ScoreParams {
    const void *logits;
    const int *targets;
    float *logprob, *entropy, *lse, *top_logprob;
    int *top_ids;
    long long ld;
    int rows, vocab, top, parts, part_len;  // part_len: a multiple of 8
    float inv_temperature;
    int *counters;
    float *partials;  // [row][part]: kScorePartFloats
};
constexpr int kScorePartFloats = 4 + 2 * kMaxTop;  // m, l, t, -; keys

typedef unsigned long long score_key;

// Pairs are ordered by value, then by lowest index; NaN is above everything.
__device__ __forceinline__ score_key make_key(float x, int index) {
    unsigned u = __float_as_uint(x + 0.f);  // (-0 and 0 are equal)
    u = x != x ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return (score_key)u << 32 | (0xffffffffu - (unsigned)index);
}
__device__ __forceinline__ float key_value(score_key k) {
    const unsigned u = (unsigned)(k >> 32);
    if (u == 0xffffffffu) return __uint_as_float(0x7fffffffu);
    return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int key_index(score_key k) { return (int)(0xffffffffu - (unsigned)k); }
constexpr score_key kNoKey = 0;  // below every key of a number
// The value below x (what is above it is x or more); of -infinity NaN, which nothing is below or equal to.
__device__ __forceinline__ float value_below(float x) {
    const unsigned u = __float_as_uint(x + 0.f);
    if (x != x || u == 0xff800000u) return __uint_as_float(0x7fffffffu);
    return __uint_as_float((u & 0x80000000u) ? u + 1 : u == 0 ? 0x80000001u : u - 1);
}

struct Sums {
    float m, l, t;
};
__device__ __forceinline__ float reference_of(float m) { return m == -INFINITY ? 0.f : m; }
// (c2: inv_temperature log2 e)
__device__ __forceinline__ Sums join(const Sums &a, const Sums &b, float c2) {
    const float m = fmaxf(a.m, b.m), r = reference_of(m);
    // (of a side without a finite logit l and t are zero: its distance may be anything finite)
    const float da = fmaxf(a.m - r, -1e30f), db = fmaxf(b.m - r, -1e30f);
    const float fa = lm_ex2(da * c2), fb = lm_ex2(db * c2);
    auto shifted = [](float t, float d, float l, float f) { return f == 0.f ? 0.f * l : fmaf(d, l, t) * f; };
    return {m, a.l * fa + b.l * fb, shifted(a.t, da, a.l, fa) + shifted(b.t, db, b.l, fb)};
}
__device__ __forceinline__ Sums join_warp(Sums s, float c2) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1)
        s = join(s, {__shfl_xor_sync(0xffffffffu, s.m, d), __shfl_xor_sync(0xffffffffu, s.l, d), __shfl_xor_sync(0xffffffffu, s.t, d)}, c2);
    return s;
}

template <int ELEM>
struct Vec {
    static constexpr int N = ELEM == LM_F32 ? 4 : 8;  // elements of 16 bytes
};
template <int ELEM>
__device__ __forceinline__ float load1(const void *p, size_t i) {
    if (ELEM == LM_F32) return static_cast<const float *>(p)[i];
    if (ELEM == LM_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
template <int ELEM>
__device__ __forceinline__ float2 unpack(unsigned w) {
    if (ELEM == LM_F16) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <int ELEM>
__device__ __forceinline__ void decode(const uint4 &r, float (&x)[Vec<ELEM>::N]) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (ELEM == LM_F32) {
            x[i] = __uint_as_float(w[i]);
        } else {
            const float2 f = unpack<ELEM>(w[i]);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// The largest element of the vectors of a lane, NaN if one is; 16-bit formats are compared in pairs.
template <int ELEM, int V>
__device__ __forceinline__ float largest_of(const uint4 (&r)[V]) {
    auto both = [](unsigned a, unsigned b) {
        unsigned d;
        if (ELEM == LM_F32) d = __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
        else if (ELEM == LM_F16) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    };
    unsigned m[V];
#pragma unroll
    for (int i = 0; i < V; ++i) m[i] = both(both(r[i].x, r[i].y), both(r[i].z, r[i].w));
#pragma unroll
    for (int i = 1; i < V; ++i) m[0] = both(m[0], m[i]);
    if (ELEM == LM_F32) return __uint_as_float(m[0]);
    const float2 f = unpack<ELEM>(m[0]);
    return max_nan(f.x, f.y);
}

// What a warp keeps, in shared memory: `n` keys, thr the value that a new one has to exceed.
struct Candidates {
    int n;
    float thr;
};
constexpr int kSlots = 3, kBuffer = 32 * kSlots;
__device__ __forceinline__ score_key lds_key(const score_key *p) { return *(volatile const score_key *)p; }
// (None of what follows is inlined: the loop over a row has to fit the instruction cache.)
// Sorts keys that differ and keeps the best `top`; the last of them is the new threshold.
__device__ __noinline__ Candidates keep_best(score_key *keys, Candidates c, int top) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    score_key mine[kSlots];
    int rank[kSlots];
#pragma unroll
    for (int i = 0; i < kSlots; ++i) mine[i] = lane + 32 * i < c.n ? lds_key(keys + lane + 32 * i) : kNoKey, rank[i] = 0;
    if (c.n <= 32) {
#pragma unroll 4
        for (int i = 0; i < c.n; ++i) rank[0] += lds_key(keys + i) > mine[0];
    } else {
#pragma unroll 2
        for (int i = 0; i < c.n; ++i) {
            const score_key k = lds_key(keys + i);
#pragma unroll
            for (int j = 0; j < kSlots; ++j) rank[j] += k > mine[j];
        }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kSlots; ++i)
        if (mine[i] != kNoKey && rank[i] < top) keys[rank[i]] = mine[i];
    __syncwarp();
    c.n = min(c.n, top);
    if (c.n == top) c.thr = key_value(lds_key(keys + top - 1));
    return c;
}

// A cell by its maximum, then the earliest step; lanes of one step are not told apart (their elements' indices interleave).
constexpr int kLaneBits = 5;
__device__ __forceinline__ score_key cell_key(float x, int step, int lane) {
    return (make_key(x, 0) & ~0xffffffffull) | ((0x7ffffffu - (unsigned)step) << kLaneBits) | (unsigned)lane;
}
__device__ __forceinline__ int cell_step(score_key k) { return (int)(0x7ffffffu - ((unsigned)k >> kLaneBits)); }
// Drops cells that `top` others come before.  A bisection over the maxima ends at top + top / 4 + 2 cells; cells of the
// same maximum are told apart by step only where more of them stay than fit (then `top` + 31 at most stay).  What
// comes later has a later step: it has to exceed the least maximum kept.
__device__ __noinline__ Candidates thin(score_key *keys, Candidates c, int top) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    score_key mine[kSlots];
    unsigned value[kSlots], stay[kSlots];
    unsigned to = 0, from = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
        mine[i] = lane + 32 * i < c.n ? lds_key(keys + lane + 32 * i) : kNoKey;
        value[i] = (unsigned)(mine[i] >> 32);
        if (mine[i] != kNoKey) to = max(to, value[i]), from = min(from, value[i]);
    }
    // count(>= from) >= top > count(> to)
    to = __reduce_max_sync(0xffffffffu, to), from = __reduce_min_sync(0xffffffffu, from);
    const int enough = top + top / 4 + 2;
    int n = c.n;
    while (from < to && n > enough) {
        const unsigned mid = from + (to - from + 1) / 2;
        int count = 0;
#pragma unroll
        for (int i = 0; i < kSlots; ++i) count += __popc(__ballot_sync(0xffffffffu, value[i] >= mid));
        if (count >= top) from = mid, n = count;
        else to = mid - 1;
    }
#pragma unroll
    for (int i = 0; i < kSlots; ++i) stay[i] = __ballot_sync(0xffffffffu, mine[i] != kNoKey && value[i] >= from);
    if (n > kBuffer - 32) {
        int rank[kSlots] = {};
        for (int i = 0; i < c.n; ++i) {
            const score_key k = lds_key(keys + i) >> kLaneBits;
#pragma unroll
            for (int j = 0; j < kSlots; ++j) rank[j] += k > mine[j] >> kLaneBits;
        }
#pragma unroll
        for (int i = 0; i < kSlots; ++i) stay[i] = __ballot_sync(0xffffffffu, mine[i] != kNoKey && rank[i] < top);
    }
    __syncwarp();
    c.n = 0;
    unsigned least = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
        if (stay[i] >> lane & 1) {
            keys[c.n + __popc(stay[i] & ((1u << lane) - 1))] = mine[i];
            least = min(least, value[i]);
        }
        c.n += __popc(stay[i]);
    }
    c.thr = key_value((score_key)__reduce_min_sync(0xffffffffu, least) << 32);
    __syncwarp();
    return c;
}
// The cells of a step (of lanes that have one) whose maxima exceed the threshold; all lanes of the warp call together.
__device__ __noinline__ Candidates offer_cells(score_key *keys, Candidates c, float x, int step, bool live, int top) {
    const int lane = threadIdx.x & 31;
    const bool in = live && !(x <= c.thr);
    const unsigned who = __ballot_sync(0xffffffffu, in);
    if (in) keys[c.n + __popc(who & ((1u << lane) - 1))] = cell_key(x, step, lane);
    c.n += __popc(who);
    // (thinned before the buffer is full - it has to hold another 32 -: a stale threshold lets too many pass)
    return c.n > min(top + top / 2 + 6, kBuffer - 32) ? thin(keys, c, top) : c;
}
// The first `count` elements of a vector of each lane that has one (`live`), numbered from index0, where they exceed the
// threshold, in any order; all lanes of the warp call together.
template <int ELEM>
__device__ __noinline__ Candidates offer(score_key *keys, Candidates c, uint4 r, int index0, int count, bool live, float scale, int top) {
    constexpr int N = Vec<ELEM>::N;
    const int lane = threadIdx.x & 31;
    unsigned hits = 0;
    float x[N];
    decode<ELEM>(r, x);
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (!(x[j] * scale <= c.thr)) hits |= 1u << j;
    hits &= live ? (1u << count) - 1 : 0u;
    unsigned who;
    while ((who = __ballot_sync(0xffffffffu, hits != 0)) != 0) {
        if (c.n + __popc(who) > kBuffer) {
            c = keep_best(keys, c, top);
            c.thr = value_below(c.thr);  // (lower indices may come yet)
        }
        const int j = __ffs(hits) - 1;
        float v = x[0];
#pragma unroll
        for (int i = 1; i < N; ++i)
            if (j == i) v = x[i];
        v *= scale;
        const bool in = hits && !(v <= c.thr);
        hits &= hits - 1;
        who = __ballot_sync(0xffffffffu, in);
        if (in) keys[c.n + __popc(who & ((1u << lane) - 1))] = make_key(v, index0 + j);
        c.n += __popc(who);
    }
    return c;
}

constexpr int kAhead = 4;  // vectors a lane works on together, while as many are on their way

struct Outside {
    int head0, heads, tail0, tails;  // elements before and behind the vectors
};
// The best elements of the cells kept, and of those outside any.  Vectors are counted from element index0; steps before
// `whole` have kAhead vectors a lane, the others one.
template <int ELEM>
__device__ __noinline__ Candidates cell_elements(score_key *keys, Candidates c, const unsigned char *row, int index0, int whole, Outside o,
                                                 float scale, int top) {
    constexpr int N = Vec<ELEM>::N, kEsize = ELEM == LM_F32 ? 4 : 2, kBatch = 4;
    const int lane = threadIdx.x & 31;
    __syncwarp();
    if (c.n > top + top / 4 + 2) c = thin(keys, c, top);
    // elements below the least maximum of `top` cells are not among the best
    const int kept = c.n;
    unsigned least = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kSlots; ++i)
        if (lane + 32 * i < kept) least = min(least, (unsigned)(lds_key(keys + lane + 32 * i) >> 32));
    least = __reduce_min_sync(0xffffffffu, least);
    c.thr = kept >= top ? value_below(key_value((score_key)least << 32)) : __uint_as_float(0x7fffffffu);
    // (the cells go to registers, their elements gather in the buffer) a lane takes a vector of a cell
    score_key cell[kSlots];
#pragma unroll
    for (int i = 0; i < kSlots; ++i) cell[i] = lane + 32 * i < kept ? lds_key(keys + lane + 32 * i) : kNoKey;
    __syncwarp();
    c.n = 0;
    const uint4 *vectors = reinterpret_cast<const uint4 *>(row + (size_t)index0 * kEsize);
#pragma unroll 1
    for (int i0 = 0; i0 < kept * kAhead; i0 += 32 * kBatch) {
        uint4 w[kBatch];
        int at[kBatch];  // the vector's number, or -1
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int of = (i0 + 32 * i + lane) / kAhead, a = lane % kAhead;
            score_key k = kNoKey;
#pragma unroll
            for (int j = 0; j < kSlots; ++j) {
                const score_key from = __shfl_sync(0xffffffffu, cell[j], of & 31);
                if (of >> 5 == j) k = from;
            }
            at[i] = cell_step(k) * 32 + (int)((unsigned)k & 31u);
            const bool live = of < kept && (a == 0 || at[i] < whole);
            at[i] = live ? at[i] + a * 32 : -1;
            w[i] = make_uint4(0, 0, 0, 0);
            if (live) w[i] = vectors[at[i]];
        }
#pragma unroll 1
        for (int i = 0; i < kBatch && i0 + 32 * i < kept * kAhead; ++i) {
            c = offer<ELEM>(keys, c, w[0], index0 + at[0] * N, N, at[0] >= 0, scale, top);
#pragma unroll
            for (int e = 1; e < kBatch; ++e) w[e - 1] = w[e], at[e - 1] = at[e];
        }
    }
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
        const int from = i ? o.tail0 : o.head0, count = i ? o.tails : o.heads;
        if (count == 0) continue;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (lane < count)
            w.x = ELEM == LM_F32 ? reinterpret_cast<const unsigned *>(row)[from + lane] : reinterpret_cast<const unsigned short *>(row)[from + lane];
        c = offer<ELEM>(keys, c, w, from + lane, 1, lane < count, scale, top);
    }
    return keep_best(keys, c, top);
}

// The parts of a row joined: their sums, and (lists of 32 keys, the best first) their alternatives.
struct Joined {
    Sums sums;
    Candidates cand;
};
template <bool TOP>
__device__ __noinline__ Joined join_parts(const float *from, int parts, score_key *keys, float c2, int top) {
    const int lane = threadIdx.x & 31;
    Sums sums = {-INFINITY, 0.f, 0.f};
    // lane i joins parts i, i + 32, ..., the warp joins the lanes
    for (int q = lane; q < parts; q += 32) {
        const float4 f = __ldcg(reinterpret_cast<const float4 *>(from + (size_t)q * kScorePartFloats));
        sums = join(sums, {f.x, f.y, f.z}, c2);
    }
    sums = join_warp(sums, c2);
    Candidates cand = {0, 0.f};
    if (TOP) {
        // no key below the last one of any part's list is among the best
        auto list = [&](int q) { return reinterpret_cast<const score_key *>(from + (size_t)q * kScorePartFloats + 4); };
        score_key bound = kNoKey;
        for (int q = lane; q < parts; q += 32) bound = max(bound, __ldcg(list(q) + top - 1));
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) bound = max(bound, __shfl_xor_sync(0xffffffffu, bound, d));
        // the lists' first keys of 32 parts, their second ones, and so on: few reach far
        for (int q0 = 0; q0 < parts; q0 += 32) {
            const bool has = q0 + lane < parts;
            bool more = true;
            for (int j0 = 0; more && j0 < top; j0 += 4) {
                score_key k[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) k[j] = has && j0 + j < top ? __ldcg(list(q0 + lane) + j0 + j) : kNoKey;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool in = k[j] != kNoKey && k[j] >= bound;
                    const unsigned who = __ballot_sync(0xffffffffu, in);
                    more = who != 0;
                    if (!more) break;
                    if (in) keys[cand.n + __popc(who & ((1u << lane) - 1))] = k[j];
                    cand.n += __popc(who);
                    if (cand.n > kBuffer - 32) {
                        cand = keep_best(keys, cand, top);
                        bound = max(bound, lds_key(keys + top - 1));
                    }
                }
            }
        }
        cand = keep_best(keys, cand, top);
    }
    return {sums, cand};
}

template <int ELEM, bool TOP>
__global__ void __launch_bounds__(kScoreThreads, TOP ? 4 : 6)
token_scores_kernel(const __grid_constant__ ScoreParams p, BlpArgs blp) {
    constexpr int N = Vec<ELEM>::N, kEsize = ELEM == LM_F32 ? 4 : 2;
    __shared__ score_key s_keys[TOP ? kScoreWarps * kBuffer : 1];
    pdl_enter();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    if (threadIdx.x == 0) trace_begin(blp);
    const float scale = p.inv_temperature, c2 = p.inv_temperature * kLog2e;
    score_key *const keys = s_keys + (TOP ? wid * kBuffer : 0);
    int iter = 0;
    for (;; ++iter) {
        // a unit a warp: warps claim by themselves, and a launch without a word deals units to them in turn
        int unit;
        if (blp.preempted) {
            if (lane == 0) unit = blp_claim(blp, iter);
            unit = __shfl_sync(0xffffffffu, unit, 0);
        } else {
            const long long u = (long long)iter * gridDim.x * kScoreWarps + wid * gridDim.x + blockIdx.x;
            unit = u < blp.total_tiles ? (int)u : -1;
        }
        if (unit < 0) break;
        const int row = unit / p.parts, part = unit - row * p.parts;
        const unsigned char *base = static_cast<const unsigned char *>(p.logits) + (size_t)row * p.ld * kEsize;
        const int begin = part * p.part_len, end = min(p.vocab, begin + p.part_len);
        Sums sums = {-INFINITY, 0.f, 0.f};
        Candidates cand = {0, __uint_as_float(0x7fffffffu)};

        auto raise = [&](float top) {
            const float m = fmaxf(sums.m, top);
            if (m > sums.m) {
                const float d = sums.m == -INFINITY ? 0.f : sums.m - m, f = lm_ex2(d * c2);
                sums.t = f == 0.f ? 0.f * sums.l : fmaf(d, sums.l, sums.t) * f;
                sums.l *= f;
                sums.m = m;
            }
        };
        // some vectors of this lane; returns their maximum
        auto take = [&](auto &r) {
            constexpr int V = sizeof(r) / sizeof(uint4);
            const float top = largest_of<ELEM, V>(r);
            raise(top);
            const float ref = reference_of(sums.m);
            const float2 cc = make_float2(c2, c2), r2 = make_float2(-ref, -ref);
            float2 l2 = make_float2(0.f, 0.f), t2 = make_float2(0.f, 0.f);
#pragma unroll
            for (int a = 0; a < V; ++a) {
                float x[N];
                decode<ELEM>(r[a], x);
#pragma unroll
                for (int j = 0; j < N; j += 2) {
                    const float2 y = add2(make_float2(x[j], x[j + 1]), r2), b = mul2(y, cc);
                    const float2 e = make_float2(lm_ex2(b.x), lm_ex2(b.y));
                    l2 = add2(l2, e);
                    t2 = fma2(y, e, t2);
                }
            }
            float t = t2.x + t2.y;
            if (t != t) {
                // logits of -infinity (or NaN): no probability times minus infinity is zero
                t = 0.f;
#pragma unroll 1
                for (int a = 0; a < V; ++a) {
                    float x[N];
                    uint4 w = r[0];
#pragma unroll
                    for (int i = 1; i < V; ++i)
                        if (a == i) w = r[i];
                    decode<ELEM>(w, x);
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float y = x[j] - ref;
                        t = fmaf(fmaxf(y, -1e30f), lm_ex2(y * c2), t);
                    }
                }
            }
            sums.l += l2.x + l2.y, sums.t += t;
            return top;
        };

        const int head = min(end - begin, (int)((16 - ((uintptr_t)(base + (size_t)begin * kEsize) & 15)) & 15) / kEsize);
        const int vecs = (end - begin - head) / N;
        const uint4 *v = reinterpret_cast<const uint4 *>(base + (size_t)(begin + head) * kEsize);
        // elements before the first 16-byte boundary and behind the last vector: one a lane
        auto take_single = [&](int index, bool live) {
            if (live) {
                const float x = load1<ELEM>(base, index);
                raise(x);
                const float y = x - reference_of(sums.m), e = lm_ex2(y * c2);
                sums.l += e, sums.t = fmaf(fmaxf(y, -1e30f), e, sums.t);
            }
        };
        if (head) take_single(begin + lane, lane < head);
        constexpr int kStep = 32 * kAhead;
        const int whole = vecs / kStep * kStep;
        uint4 r[kAhead], ahead[kAhead];
        auto fetch = [&](uint4 (&to)[kAhead], int i0) {
#pragma unroll
            for (int a = 0; a < kAhead; ++a) to[a] = __ldcs(v + i0 + a * 32 + lane);
        };
        if (whole) fetch(r, 0);
#pragma unroll 1
        for (int i0 = 0; i0 < whole; i0 += kStep) {
            if (i0 + kStep < whole) fetch(ahead, i0 + kStep);
            const float top = take(r);
            if (TOP && __any_sync(0xffffffffu, !(top * scale <= cand.thr))) cand = offer_cells(keys, cand, top * scale, i0 / 32, true, p.top);
#pragma unroll
            for (int a = 0; a < kAhead; ++a) r[a] = ahead[a];
        }
#pragma unroll 1
        for (int i0 = whole; i0 < vecs; i0 += 32) {
            const bool live = i0 + lane < vecs;
            float top = -INFINITY;
            if (live) {
                uint4 one[1] = {__ldcs(v + i0 + lane)};
                top = take(one);
            }
            if (TOP && __any_sync(0xffffffffu, live && !(top * scale <= cand.thr)))
                cand = offer_cells(keys, cand, top * scale, i0 / 32, live, p.top);
        }
        const int tail0 = begin + head + vecs * N;
        if (tail0 < end) take_single(tail0 + lane, tail0 + lane < end);

        sums = join_warp(sums, c2);
        if (TOP) {
            const Outside outside = {begin, head, tail0, end - tail0};
            cand = cell_elements<ELEM>(keys, cand, base, begin + head, whole, outside, scale, p.top);
            if (lane >= cand.n) keys[lane] = kNoKey;
            __syncwarp();
        }
        if (p.parts > 1) {
            // ---- a part: left in the context; the warp that brings the last one joins them
            float *to = p.partials + (size_t)unit * kScorePartFloats;
            if (lane == 0) to[0] = sums.m, to[1] = sums.l, to[2] = sums.t;
            if (TOP) reinterpret_cast<score_key *>(to + 4)[lane] = keys[lane];
            __threadfence();
            __syncwarp();
            int last = 0;
            if (lane == 0) last = atomicAdd(&p.counters[row], 1) == p.parts - 1;
            if (!__shfl_sync(0xffffffffu, last, 0)) continue;
            __threadfence();
            const float *from = p.partials + (size_t)row * p.parts * kScorePartFloats;
            sums = join_parts<TOP>(from, p.parts, keys, c2, p.top).sums;
            if (lane == 0) p.counters[row] = 0;
        }
        const float logl = logf(sums.l), lse = fmaf(sums.m, scale, logl);
        if (lane == 0) {
            if (p.lse) p.lse[row] = lse;
            if (p.entropy) p.entropy[row] = logl - scale * (sums.t / sums.l);
            if (p.logprob) {
                const int target = p.targets[row];
                float lp = 0.f;
                if (target >= p.vocab) lp = __uint_as_float(0x7fffffffu);
                else if (target >= 0) lp = load1<ELEM>(base, target) * scale - lse;
                p.logprob[row] = lp;
            }
        }
        if (TOP && lane < p.top) {
            const score_key best = lds_key(keys + lane);
            if (p.top_ids) p.top_ids[(size_t)row * p.top + lane] = key_index(best);
            if (p.top_logprob) p.top_logprob[(size_t)row * p.top + lane] = key_value(best) - lse;
        }
        __syncwarp();
    }
    // (units run, counted for the CTA as a whole where somebody asks)
    if (blp.trace && lane == 0) trace_end(blp, iter);
}

template <typename F>
static auto scores_instance(int elem, bool top, F &&f) {
    if (elem == LM_F32) return top ? f(token_scores_kernel<LM_F32, true>) : f(token_scores_kernel<LM_F32, false>);
    if (elem == LM_F16) return top ? f(token_scores_kernel<LM_F16, true>) : f(token_scores_kernel<LM_F16, false>);
    return top ? f(token_scores_kernel<LM_BF16, true>) : f(token_scores_kernel<LM_BF16, false>);
}

}  // namespace gpx

using namespace gpx;

extern "C" int gpx_token_scores(const gpx_token_scores_args *args, void *ctx, const gpx_blp *blp, gpx_stream stream) {
    GPX_REQUIRE(args && ctx, GPX_FAIL, "args or ctx is NULL");
    GPX_REQUIRE((uintptr_t)ctx % 256 == 0, GPX_FAIL, "ctx must be 256-byte aligned");
    const gpx_token_scores_args &a = *args;
    ScoreParams p{};
    BlpArgs b;
    int elem;
    GPX_TRY(lm_check_blp(blp, &b));
    GPX_TRY(lm_elem(a.dtype, true, &elem));
    GPX_REQUIRE(a.rows >= 0 && a.vocab > 0 && a.vocab <= 0x7fffffff - 4096, GPX_OUT_OF_RANGE, "%d rows of %d logits", a.rows, a.vocab);
    GPX_REQUIRE(a.top >= 0 && a.top <= kMaxTop && a.top <= a.vocab, GPX_OUT_OF_RANGE, "top is 0 to %d and at most vocab, not %d", kMaxTop, a.top);
    GPX_REQUIRE(a.top > 0 || (!a.top_ids && !a.top_logprob), GPX_OUT_OF_RANGE, "top is 0, but its outputs are given");
    GPX_REQUIRE(!a.logprob || a.targets, GPX_FAIL, "logprob needs targets");
    GPX_REQUIRE(a.inv_temperature > 0.f && a.inv_temperature <= 3.4e38f, GPX_OUT_OF_RANGE, "inv_temperature must be positive and finite");
    GPX_REQUIRE(((uintptr_t)a.targets | (uintptr_t)a.logprob | (uintptr_t)a.entropy | (uintptr_t)a.lse | (uintptr_t)a.top_ids |
                 (uintptr_t)a.top_logprob) % 4 == 0, GPX_FAIL, "targets and the outputs must be 4-byte aligned");
    p.ld = a.ld ? a.ld : a.vocab;
    GPX_REQUIRE(p.ld >= a.vocab, GPX_OUT_OF_RANGE, "a row of %d is longer than the distance to the next, %lld", a.vocab, p.ld);
    const DeviceInfo &d = device_info();
    GPX_REQUIRE(d.device >= 0, GPX_FAIL, "gpx_init was not called");
    if (a.rows == 0) return GPX_SUCC;
    const int esize = elem == LM_F32 ? 4 : 2;
    GPX_REQUIRE(a.logits && (uintptr_t)a.logits % esize == 0, GPX_FAIL, "logits is NULL or not aligned to its type");
    p.logits = a.logits, p.targets = (const int *)a.targets;
    p.logprob = (float *)a.logprob, p.entropy = (float *)a.entropy, p.lse = (float *)a.lse;
    p.top_logprob = (float *)a.top_logprob, p.top_ids = (int *)a.top_ids;
    p.rows = a.rows, p.vocab = a.vocab, p.top = a.top, p.inv_temperature = a.inv_temperature;
    const LmCtx c = lm_ctx(ctx);
    p.counters = c.counters, p.partials = c.parts;
    const bool top = a.top_ids || a.top_logprob;
    int per_sm = 0;
    GPX_CUDA(scores_instance(elem, top, [&](auto kernel) {
        return lm_resident((const void *)kernel, kScoreThreads, 0, 0, d.device, &per_sm);
    }));
    // Few rows are cut so that two thirds of the warps have a part, of a vector a lane at least.  From half as many rows
    // as warps on they are left whole: a unit costs ~4 us beside its elements, and memory is busy with fewer warps, too
    // (rows of 50 257 fp16, one alternative, whole / in two: 2 000 rows 57 / 72 us, 4 096 rows 109 / 120, with an earlier loop).
    const long long resident = (long long)d.sm_count * per_sm * kScoreWarps;
    long long parts = 1;
    if (a.rows <= kLmCounters) {
        const long long most = std::max(1ll, std::min((long long)a.vocab * esize / (16 * 32),
                                                      (long long)(kLmPartsBytes / (kScorePartFloats * sizeof(float))) / a.rows));
        if (2ll * a.rows < resident) parts = 2 * resident / 3 / a.rows;
        // (a launch that can be preempted drains at the end of a unit; with 8 192 elements, 4 096 rows of 50 257 fp16 with one
        // alternative drain in 17 us at the median, 20 at most, and take 172 us on the device, 94 without a word)
        if (b.preempted) parts = std::max(parts, (a.vocab + 8191ll) / 8192);
        parts = std::max(1ll, std::min({parts, most, (a.vocab + 1023ll) / 1024}));
    }
    p.part_len = (int)(((a.vocab + parts - 1) / parts + 7) / 8 * 8);
    p.parts = (a.vocab + p.part_len - 1) / p.part_len;
    b.total_tiles = a.rows * p.parts;
    const int grid = (int)std::min<long long>((long long)d.sm_count * per_sm, b.total_tiles);
    GPX_CUDA(scores_instance(elem, top, [&](auto kernel) { return launch_layer(kernel, grid, kScoreThreads, 0, as_stream(stream), p, b); }));
    return GPX_SUCC;
}
