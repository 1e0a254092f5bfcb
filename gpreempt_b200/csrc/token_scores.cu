// Log probabilities of given tokens, entropies and the most likely alternatives, from logits, in one pass over them.
//
//   m = max x,  l = sum e^(x - m),  t = sum (x - m) e^(x - m)          x = logit * inv_temperature
//   lse = m + log l,  logprob(i) = x_i - lse,  entropy = log l - t / l  (neither term is negative: nothing cancels)
//
// Kept per thread with a running maximum: when it grows by d, l -> l e^-d and t -> (t - d l) e^-d.  (The maximum is
// taken off before the change to base 2: logits as low as the type goes, a common mask, stay finite.)
// Alternatives ride along: a warp keeps its best `top` (value, index) pairs one a lane, sorted, and looks at its
// vectors more closely only where their maximum, which the softmax needs anyway, reaches the worst of them or of any
// other warp's of the row.  After the first vectors that is rare (the n-th element is among the best k with
// probability k / n).
//
// A tile is a row, or a part of one where there are few rows; the CTA that finishes the last part of a row joins them in
// the order of the parts, so the result does not depend on which one that is.
#include "act_layout.h"
#include "lm.h"

#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace gpx {

constexpr int kScoreThreads = 256, kScoreWarps = kScoreThreads / 32;
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

// Inserts a key into the sorted list of a warp (lane i holds the i-th best).
__device__ __forceinline__ void insert_key(score_key &mine, score_key key, int lane) {
    const int at = __popc(__ballot_sync(0xffffffffu, mine > key));
    const score_key up = __shfl_up_sync(0xffffffffu, mine, 1);
    if (lane == at) mine = key;
    else if (lane > at) mine = up;
}

struct Sums {
    float m, l, t;
};
__device__ __forceinline__ float reference_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ Sums join(const Sums &a, const Sums &b) {
    const float m = fmaxf(a.m, b.m), r = reference_of(m);
    // (of a side without a finite logit l and t are zero: its distance may be anything finite)
    const float da = fmaxf(a.m - r, -1e30f), db = fmaxf(b.m - r, -1e30f);
    const float fa = lm_ex2(da * kLog2e), fb = lm_ex2(db * kLog2e);
    auto shifted = [](float t, float d, float l, float f) { return f == 0.f ? 0.f * l : fmaf(d, l, t) * f; };
    return {m, a.l * fa + b.l * fb, shifted(a.t, da, a.l, fa) + shifted(b.t, db, b.l, fb)};
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
__device__ __forceinline__ void decode(const uint4 &r, float (&x)[Vec<ELEM>::N]) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (ELEM == LM_F32) {
            x[i] = __uint_as_float(w[i]);
        } else {
            float2 f;
            if (ELEM == LM_F16) f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            else f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

template <int ELEM, bool TOP>
__global__ void __launch_bounds__(kScoreThreads)
token_scores_kernel(const __grid_constant__ ScoreParams p, BlpArgs blp) {
    constexpr int N = Vec<ELEM>::N, kAhead = 4;
    __shared__ int s_tile, s_last;
    __shared__ Sums s_sums[kScoreWarps];
    __shared__ score_key s_keys[kScoreWarps][kMaxTop];
    __shared__ float s_worst;  // the largest of the warps' worst kept values: what is below it is not among the best
    pdl_enter();
    const bool dynamic = blp.preempted != nullptr;
    if (threadIdx.x == 0) trace_begin(blp);
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    volatile float *const worst = &s_worst;
    int iter = 0;
    for (;; ++iter) {
        int tile;
        if (threadIdx.x == 0) s_worst = -INFINITY;
        if (dynamic) {
            if (threadIdx.x == 0) s_tile = blp_claim(blp, iter);
            __syncthreads();
            tile = s_tile;
        } else {
            tile = blp_claim(blp, iter);
            __syncthreads();
        }
        if (tile < 0) break;
        const int row = tile / p.parts, part = tile - row * p.parts;
        const unsigned char *base = static_cast<const unsigned char *>(p.logits) + (size_t)row * p.ld * (ELEM == LM_F32 ? 4 : 2);
        const int begin = part * p.part_len, end = min(p.vocab, begin + p.part_len);
        Sums sums = {-INFINITY, 0.f, 0.f};
        score_key mine = kNoKey;
        float thr = -INFINITY;  // values below it are not among the best

        // `count` elements of this lane from index0 on; all lanes of the warp call together
        auto take = [&](const float (&raw)[N], int index0, int count) {
            float x[N];
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                x[j] = j < count ? raw[j] * p.inv_temperature : -INFINITY;
                top = max_nan(top, x[j]);
            }
            const float m = fmaxf(sums.m, top);
            if (m > sums.m) {
                const float d = sums.m == -INFINITY ? 0.f : sums.m - m, f = lm_ex2(d * kLog2e);
                sums.t = f == 0.f ? 0.f * sums.l : fmaf(d, sums.l, sums.t) * f;
                sums.l *= f;
                sums.m = m;
            }
            const float ref = reference_of(sums.m);
            const float2 c2 = make_float2(kLog2e, kLog2e), r2 = make_float2(-ref, -ref);
            float2 l2 = make_float2(0.f, 0.f), t2 = make_float2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const float2 y = add2(make_float2(x[j], x[j + 1]), r2), b = mul2(y, c2);
                const float2 e = make_float2(lm_ex2(b.x), lm_ex2(b.y));
                l2 = add2(l2, e);
                // (no probability times minus infinity is zero)
                t2 = fma2(make_float2(fmaxf(y.x, -1000.f), fmaxf(y.y, -1000.f)), e, t2);
            }
            sums.l += l2.x + l2.y, sums.t += t2.x + t2.y;
            if (TOP) {
                if (!__any_sync(0xffffffffu, count > 0 && !(top < thr))) return;
                thr = fmaxf(thr, *worst);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    unsigned who = __ballot_sync(0xffffffffu, j < count && !(x[j] < thr));
                    while (who) {
                        const int src = __ffs(who) - 1;
                        const float v = __shfl_sync(0xffffffffu, x[j], src);
                        insert_key(mine, make_key(v, __shfl_sync(0xffffffffu, index0, src) + j), lane);
                        const score_key last = __shfl_sync(0xffffffffu, mine, p.top - 1);
                        if (last != kNoKey) thr = fmaxf(thr, key_value(last));
                        who &= who - 1;
                        who &= __ballot_sync(0xffffffffu, !(x[j] < thr));
                    }
                }
                if (thr > *worst && lane == 0) *worst = thr;  // (a lost race leaves a smaller one: nothing is dropped that counts)
            }
        };

        // elements before the first 16-byte boundary and behind the last: one a lane of the first warp
        const int esize = ELEM == LM_F32 ? 4 : 2;
        const int head = min(end - begin, (int)((16 - ((uintptr_t)(base + (size_t)begin * esize) & 15)) & 15) / esize);
        const int vecs = (end - begin - head) / N;
        const uint4 *v = reinterpret_cast<const uint4 *>(base + (size_t)(begin + head) * esize);
        if (wid == 0) {
            const int tail0 = begin + head + vecs * N, tail = end - tail0;
            const int index = lane < head ? begin + lane : tail0 + lane - head;
            float x[N];
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = 0.f;
            const bool live = lane < head + tail;
            if (live) x[0] = load1<ELEM>(base, index);
            if (head + tail) take(x, index, live ? 1 : 0);
        }
        // (whole warps: every lane of a warp takes part in what it keeps)
        for (int i0 = wid * 32; i0 < vecs; i0 += kScoreThreads * kAhead) {
            uint4 r[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const int i = i0 + a * kScoreThreads + lane;
                if (i < vecs) r[a] = __ldcs(v + i);
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const int w0 = i0 + a * kScoreThreads;
                if (w0 >= vecs) break;
                float x[N];
                decode<ELEM>(r[a], x);
                take(x, begin + head + (w0 + lane) * N, w0 + lane < vecs ? N : 0);
            }
        }

        // the warp's sums, the CTA's, and the best of all warps
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1)
            sums = join(sums, {__shfl_xor_sync(0xffffffffu, sums.m, d), __shfl_xor_sync(0xffffffffu, sums.l, d),
                               __shfl_xor_sync(0xffffffffu, sums.t, d)});
        if (lane == 0) s_sums[wid] = sums;
        if (TOP) s_keys[wid][lane] = mine;
        __syncthreads();
        auto merge = [&](const score_key *keys, int stride, int lists) {  // warp 0: further sorted lists into its own
            for (int w = 0; w < lists; ++w) {
                const score_key theirs = lane < p.top ? keys[w * stride + lane] : kNoKey;
                for (int j = 0; j < p.top; ++j) {
                    const score_key key = __shfl_sync(0xffffffffu, theirs, j);
                    if (key <= __shfl_sync(0xffffffffu, mine, p.top - 1)) break;
                    insert_key(mine, key, lane);
                }
            }
        };
        bool finish = p.parts == 1;
        if (wid == 0) {
            for (int w = 1; w < kScoreWarps; ++w) sums = join(sums, s_sums[w]);
            if (TOP) merge(&s_keys[1][0], kMaxTop, kScoreWarps - 1);
            if (!finish) {
                float *to = p.partials + (size_t)tile * kScorePartFloats;
                if (lane == 0) to[0] = sums.m, to[1] = sums.l, to[2] = sums.t;
                if (TOP) reinterpret_cast<score_key *>(to + 4)[lane] = mine;
                __threadfence();
                __syncwarp();
                if (lane == 0) s_last = atomicAdd(&p.counters[row], 1) == p.parts - 1;
                __syncwarp();
                finish = s_last;
                if (finish) {
                    __threadfence();
                    const float *from = p.partials + (size_t)row * p.parts * kScorePartFloats;
                    sums = {-INFINITY, 0.f, 0.f};
                    // lane i joins parts i, i + 32, ..., the warp joins the lanes
                    for (int q = lane; q < p.parts; q += 32) {
                        const float *f = from + (size_t)q * kScorePartFloats;
                        sums = join(sums, {__ldcg(f), __ldcg(f + 1), __ldcg(f + 2)});
                    }
#pragma unroll
                    for (int d = 16; d >= 1; d >>= 1)
                        sums = join(sums, {__shfl_xor_sync(0xffffffffu, sums.m, d), __shfl_xor_sync(0xffffffffu, sums.l, d),
                                           __shfl_xor_sync(0xffffffffu, sums.t, d)});
                    if (TOP) {
                        mine = kNoKey;
                        for (int q = 0; q < p.parts; ++q) {
                            const score_key *keys = reinterpret_cast<const score_key *>(from + (size_t)q * kScorePartFloats + 4);
                            const score_key theirs = lane < p.top ? __ldcg(keys + lane) : kNoKey;
                            for (int j = 0; j < p.top; ++j) {
                                const score_key key = __shfl_sync(0xffffffffu, theirs, j);
                                if (key <= __shfl_sync(0xffffffffu, mine, p.top - 1)) break;
                                insert_key(mine, key, lane);
                            }
                        }
                    }
                    if (lane == 0) p.counters[row] = 0;
                }
            }
            if (finish) {
                const float logl = logf(sums.l);
                const float lse = sums.m + logl;
                if (lane == 0) {
                    if (p.lse) p.lse[row] = lse;
                    if (p.entropy) p.entropy[row] = logl - sums.t / sums.l;
                    if (p.logprob) {
                        const int target = p.targets[row];
                        float lp = 0.f;
                        if (target >= p.vocab) lp = __uint_as_float(0x7fffffffu);
                        else if (target >= 0) lp = load1<ELEM>(base, target) * p.inv_temperature - lse;
                        p.logprob[row] = lp;
                    }
                }
                if (TOP && lane < p.top) {
                    if (p.top_ids) p.top_ids[(size_t)row * p.top + lane] = key_index(mine);
                    if (p.top_logprob) p.top_logprob[(size_t)row * p.top + lane] = key_value(mine) - lse;
                }
            }
        }
        __syncthreads();  // the tile number and the warps' results are rewritten
    }
    if (threadIdx.x == 0) trace_end(blp, iter);
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
        return lm_resident((const void *)kernel, kScoreThreads, 0, d.device, &per_sm);
    }));
    // Few rows are cut so that every resident CTA has a part, of 1024 elements at least.
    const long long resident = (long long)d.sm_count * per_sm;
    long long parts = 1;
    if (a.rows < resident && a.rows <= kLmCounters)
        parts = std::max(1ll, std::min({resident / a.rows, (a.vocab + 1023ll) / 1024,
                                        (long long)(kLmPartsBytes / (kScorePartFloats * sizeof(float))) / a.rows}));
    p.part_len = (int)(((a.vocab + parts - 1) / parts + 7) / 8 * 8);
    p.parts = (a.vocab + p.part_len - 1) / p.part_len;
    b.total_tiles = a.rows * p.parts;
    const int grid = (int)std::min<long long>(resident, b.total_tiles);
    GPX_CUDA(scores_instance(elem, top, [&](auto kernel) { return launch_layer(kernel, grid, kScoreThreads, 0, as_stream(stream), p, b); }));
    return GPX_SUCC;
}
