// Appending keys and values to a paged 8-bit cache, with the position rotation of queries and keys on the way.
//
//   a' = a cos - b sin,  b' = b cos + a sin        for the pairs (a, b) of a head's first `rotated` elements
//   scale' = max(scale of what the page holds, 2^ceil(log2(amax / 448)) of what is new to it)
//   code = e4m3(x / scale');  codes the page holds already: e4m3(code * scale / scale')
//
// Scales are powers of two: a quotient by one is exact, so that a page whose scale grows rounds its older codes again
// only where they leave the normal range, and a tiny difference of an amax hardly ever changes a scale.  (e4m3
// keeps four significant bits wherever the scale puts them; a scale of amax / 448 would gain nothing but the last
// binade above the underflow.)  All arithmetic is float, with the products of a rotation rounded on their own, so that the codes do not
// depend on which instance computes them.
//
// A lane holds eight elements of a row as two groups of four, such that both elements of a pair are its own.
#include "lm.h"

#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace gpx {

struct AppendParams {
    LmBatch batch;
    unsigned char *k_codes, *v_codes;
    float *k_scale, *v_scale;
    int pages, page_shift, kv_heads, heads;
    const unsigned short *q, *k, *v;
    unsigned short *q_out;
    long long q_ld, k_ld, v_ld, q_out_ld;
    const float *cos, *sin;
    int rotated, positions, paired;
    int *error;
};

template <bool HALF>
__device__ __forceinline__ float2 unpack16(unsigned w) {
    if (HALF) return __half22float2(*reinterpret_cast<__half2 *>(&w));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <bool HALF>
__device__ __forceinline__ unsigned pack16(float a, float b) {
    if (HALF) {
        __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<unsigned *>(&h);
    }
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<unsigned *>(&h);
}

// How rows are turned: all of them in the one order or the other, or as the arguments say.
enum TurnMode { TURN_HALVES, TURN_PAIRS, TURN_ANY };

// Where lane i of a row keeps its elements: four from a, four from b, and the first of their angles.
struct Place {
    int a, b;
    bool turned;
};
__device__ __forceinline__ Place place_of(const AppendParams &p, int i, bool rotates) {
    if (!rotates || 8 * i >= p.rotated) return {8 * i, 8 * i + 4, false};
    if (p.paired) return {8 * i, 8 * i + 4, true};
    return {4 * i, 4 * i + p.rotated / 2, true};
}

struct Raw8 {
    uint2 a, b;
};
__device__ __forceinline__ Raw8 fetch8(const unsigned short *row, const Place &at) {
    return {*reinterpret_cast<const uint2 *>(row + at.a), *reinterpret_cast<const uint2 *>(row + at.b)};  // (may be turned in place)
}
template <bool HALF>
__device__ __forceinline__ void decode8(const Raw8 &r, float (&x)[8]) {
    const float2 a0 = unpack16<HALF>(r.a.x), a1 = unpack16<HALF>(r.a.y), b0 = unpack16<HALF>(r.b.x), b1 = unpack16<HALF>(r.b.y);
    x[0] = a0.x, x[1] = a0.y, x[2] = a1.x, x[3] = a1.y, x[4] = b0.x, x[5] = b0.y, x[6] = b1.x, x[7] = b1.y;
}
struct Angles {
    float4 c, s;
};
__device__ __forceinline__ Angles angles_of(const AppendParams &p, int pos, int i, bool turned) {
    if (!turned) return {};
    const size_t at = (size_t)pos * (p.rotated / 2) + 4 * i;
    return {__ldg(reinterpret_cast<const float4 *>(p.cos + at)), __ldg(reinterpret_cast<const float4 *>(p.sin + at))};
}
// (the products are rounded on their own; as pairs of packed instructions the compiler fuses them with the sums)
__device__ __forceinline__ void turn_pair(float &a, float &b, float c, float s) {
    const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    a = x;
}
template <int MODE>
__device__ __forceinline__ void turn8(float (&x)[8], const Angles &t, const Place &at, bool paired) {
    if (MODE == TURN_ANY && !at.turned) return;
    if (MODE == TURN_PAIRS || (MODE == TURN_ANY && paired)) {
        turn_pair(x[0], x[1], t.c.x, t.s.x), turn_pair(x[2], x[3], t.c.y, t.s.y);
        turn_pair(x[4], x[5], t.c.z, t.s.z), turn_pair(x[6], x[7], t.c.w, t.s.w);
    } else {
        turn_pair(x[0], x[4], t.c.x, t.s.x), turn_pair(x[1], x[5], t.c.y, t.s.y);
        turn_pair(x[2], x[6], t.c.z, t.s.z), turn_pair(x[3], x[7], t.c.w, t.s.w);
    }
}

// The bits of the largest magnitude (as unsigned they are ordered as the numbers are), of which NaN is none; where it
// is infinite, that of the finite ones, and `wild` is set.
__device__ __forceinline__ unsigned amax8(const float (&x)[8], bool &wild) {
    float a = fmaxf(fabsf(x[0]), fabsf(x[1])), b = fmaxf(fabsf(x[2]), fabsf(x[3]));
    a = fmaxf(a, fmaxf(fabsf(x[4]), fabsf(x[5]))), b = fmaxf(b, fmaxf(fabsf(x[6]), fabsf(x[7])));
    unsigned m = __float_as_uint(fmaxf(a, b));
    if (m >= 0x7f800000u) {
        wild = true;
        m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned u = __float_as_uint(x[j]) & 0x7fffffffu;
            if (u < 0x7f800000u) m = max(m, u);
        }
    }
    return m;
}
// 2^ceil(log2(amax / 448)), 448 = 1.75 * 2^8: a mantissa above .75 carries into the exponent.
__device__ __forceinline__ float scale_for(unsigned amax_bits) {
    const int e = (int)((amax_bits + 0x1fffffu) >> 23) - 8;
    return __uint_as_float((unsigned)max(e, 1) << 23);
}
// (the conversion turns NaN into NaN, but an infinity into the largest code: it is made NaN before)
__device__ __forceinline__ unsigned codes4(const float *x, float inv, bool wild) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        y[j] = x[j] * inv;
        if (wild && (__float_as_uint(x[j]) & 0x7fffffffu) >= 0x7f800000u) y[j] = __uint_as_float(0x7fffffffu);
    }
    return e4m3x2(y[0], y[1]) | e4m3x2(y[2], y[3]) << 16;
}
__device__ __forceinline__ void store8(unsigned char *row, const Place &at, const float (&x)[8], float inv, bool wild) {
    const unsigned a = codes4(x, inv, wild), b = codes4(x + 4, inv, wild);
    if (at.b == at.a + 4) {
        *reinterpret_cast<uint2 *>(row + at.a) = make_uint2(a, b);
    } else {
        *reinterpret_cast<unsigned *>(row + at.a) = a;
        *reinterpret_cast<unsigned *>(row + at.b) = b;
    }
}
// Codes of a smaller scale under a larger one (ratio: smaller / larger, a power of two).
__device__ __forceinline__ unsigned again4(unsigned w, float ratio) {
    const unsigned lo = e4m3x2_to_f16x2((unsigned short)w), hi = e4m3x2_to_f16x2((unsigned short)(w >> 16));
    const float2 a = unpack16<true>(lo), b = unpack16<true>(hi);
    return e4m3x2(a.x * ratio, a.y * ratio) | e4m3x2(b.x * ratio, b.y * ratio) << 16;
}

__device__ __forceinline__ int page_of(const AppendParams &p, int s, int index) {
    const int page = p.batch.table[(size_t)s * p.batch.table_ld + index];
    if ((unsigned)page < (unsigned)p.pages) return page;
    lm_fail(p.error, LM_BAD_PAGE, s);
    return -1;
}
__device__ __forceinline__ LmSpan append_span(const AppendParams &p, int s) {
    LmSpan span = lm_span(p.batch, s, 1 << p.page_shift, true, p.error);
    if (p.rotated && span.n && span.context > p.positions) {
        lm_fail(p.error, LM_BAD_POSITION, s);
        span.n = 0;
    }
    return span;
}

// One new token a sequence at most: every row (a head of keys, values or queries) is on its own, D / 8 lanes to a
// row, and the amax of a row is all there is of a page that is new.  A request of one token is a chain of reads
// (span, page and angles, scale); the element loads do not wait for it.
constexpr int kAppendOneThreads = 128;
template <int D, bool HALF>
__global__ void __launch_bounds__(kAppendOneThreads)
kv_append_one_kernel(const __grid_constant__ AppendParams p, BlpArgs blp) {
    constexpr int kLanes = D / 8, kRows = kAppendOneThreads / kLanes;
    __shared__ int s_tile;
    pdl_enter();
    const bool dynamic = blp.preempted != nullptr;
    if (threadIdx.x == 0) trace_begin(blp);
    const int i = threadIdx.x % kLanes, r = threadIdx.x / kLanes;
    const unsigned mask = (kLanes == 8 ? 0xffu : 0xffffu) << (threadIdx.x & 31 & ~(kLanes - 1));
    const int page_tokens = 1 << p.page_shift;
    const int rows_a_seq = 2 * p.kv_heads + (p.q ? p.heads : 0);
    int iter = 0;
    for (;; ++iter) {
        int tile;
        if (dynamic) {
            if (threadIdx.x == 0) s_tile = blp_claim(blp, iter);
            __syncthreads();
            tile = s_tile;
            __syncthreads();
        } else {
            tile = blp_claim(blp, iter);
        }
        if (tile < 0) break;
        const long long row = (long long)tile * kRows + r;
        const int s = (int)(row / rows_a_seq);
        if (s >= p.batch.seqs) continue;
        const int role = (int)(row - (long long)s * rows_a_seq);
        const LmSpan span = append_span(p, s);
        if (span.n == 0) continue;
        const int pos = span.context - 1;
        const bool is_v = role >= p.kv_heads && role < 2 * p.kv_heads;
        const Place at = place_of(p, i, !is_v);
        float x[8];
        if (role >= 2 * p.kv_heads) {
            const int h = role - 2 * p.kv_heads;
            const Angles t = angles_of(p, pos, i, at.turned);
            decode8<HALF>(fetch8(p.q + span.first * p.q_ld + h * D, at), x);
            turn8<TURN_ANY>(x, t, at, p.paired);
            unsigned short *out = p.q_out + span.first * p.q_out_ld + h * D;
            *reinterpret_cast<uint2 *>(out + at.a) = make_uint2(pack16<HALF>(x[0], x[1]), pack16<HALF>(x[2], x[3]));
            *reinterpret_cast<uint2 *>(out + at.b) = make_uint2(pack16<HALF>(x[4], x[5]), pack16<HALF>(x[6], x[7]));
            continue;
        }
        const int h = is_v ? role - p.kv_heads : role;
        const int page = page_of(p, s, pos >> p.page_shift);
        const Raw8 raw = fetch8(is_v ? p.v + span.first * p.v_ld + h * D : p.k + span.first * p.k_ld + h * D, at);
        const Angles t = angles_of(p, pos, i, at.turned);
        if (page < 0) continue;
        const int slot = pos & (page_tokens - 1);
        float *scale_at = (is_v ? p.v_scale : p.k_scale) + (size_t)page * p.kv_heads + h;
        const float old = slot ? *scale_at : 0.f;
        decode8<HALF>(raw, x);
        turn8<TURN_ANY>(x, t, at, p.paired);
        bool wild = false;
        unsigned m = amax8(x, wild);
#pragma unroll
        for (int d = kLanes / 2; d >= 1; d >>= 1) m = max(m, __shfl_xor_sync(mask, m, d));
        const float want = scale_for(m), scale = fmaxf(old, want);
        unsigned char *block = (is_v ? p.v_codes : p.k_codes) + ((size_t)page * p.kv_heads + h) * page_tokens * D;
        store8(block + slot * D, at, x, 1.0f / scale, wild);
        if (scale > old) {
            __syncwarp(mask);  // every lane has read the old scale
            if (i == 0) *scale_at = scale;
            const float ratio = old / scale;
            unsigned *w = reinterpret_cast<unsigned *>(block);
            for (int e = i; e < slot * (D / 4); e += kLanes) w[e] = again4(w[e], ratio);
        }
    }
    if (threadIdx.x == 0) trace_end(blp, iter);
}

// Any number of new tokens: a tile is what a sequence adds to one page of one head of keys and values, and the
// queries of that head's group.  Keys and values of the tile wait in shared memory between the reduction of their
// amax and their rounding.  The queries ride along because they turn by the same angles, which are twice their bytes to read
// (as tiles of their own, in the order of memory, the whole took 147 us against 126 at the time).
// What bounds it is latency: loads of a row, a barrier, stores, with 24 warps an SM, and 48 million instructions, which fill 46 %
// of the issue slots.  Eight prompts of 21 700 tokens in all, 32 heads of 128 on 8: 100 us (533 MB, 5.3 TB/s); with 16 warps 117, with
// 32 (64 registers) 116, with the rotation's order looked up for each row 119.
constexpr int kAppendThreads = 256;
template <int D, bool HALF, int MODE>
__global__ void __launch_bounds__(kAppendThreads, 3)
kv_append_kernel(const __grid_constant__ AppendParams p, BlpArgs blp) {
    constexpr int kLanes = D / 8, kRows = kAppendThreads / kLanes, kHeads = 4;
    // keys of the tile, turned, and values as they came, each thread's for itself; sums over the sequences [seqs + 1]
    extern __shared__ float4 keys[];
    uint4 *const values = reinterpret_cast<uint4 *>(keys + (D / 4 << p.page_shift));
    int *const s_prefix = reinterpret_cast<int *>(values + (kLanes << p.page_shift));
    __shared__ int s_tile;
    __shared__ unsigned s_amax[2];
    pdl_enter();
    const bool dynamic = blp.preempted != nullptr;
    if (threadIdx.x == 0) trace_begin(blp);
    const int i = threadIdx.x % kLanes, r0 = threadIdx.x / kLanes;
    const int page_tokens = 1 << p.page_shift;
    const int group = p.q ? p.heads / p.kv_heads : 0;
    blp.total_tiles = lm_prefix(s_prefix, p.batch.seqs, p.error, [&](int s) {
        const LmSpan span = append_span(p, s);
        return span.n ? (((span.context - 1) >> p.page_shift) - ((span.context - span.n) >> p.page_shift) + 1) * p.kv_heads : 0;
    });
    int iter = 0;
    for (;; ++iter) {
        int tile;
        if (threadIdx.x == 0) s_amax[0] = s_amax[1] = 0;
        if (dynamic) {
            if (threadIdx.x == 0) s_tile = blp_claim(blp, iter);
            __syncthreads();
            tile = s_tile;
        } else {
            tile = blp_claim(blp, iter);
            __syncthreads();
        }
        if (tile < 0) break;
        const int s = lm_find(s_prefix, p.batch.seqs, tile);
        const LmSpan span = {p.batch.first[s], p.batch.first[s + 1] - p.batch.first[s], p.batch.context[s]};
        const int within = tile - s_prefix[s];
        const int index = ((span.context - span.n) >> p.page_shift) + within / p.kv_heads, h = within % p.kv_heads;
        // tokens [pos0, pos1) of the sequence go to the slots from `begin` of the page
        const int pos0 = max(span.context - span.n, index << p.page_shift), pos1 = min(span.context, (index + 1) << p.page_shift);
        const int begin = pos0 & (page_tokens - 1), count = pos1 - pos0;
        const int token0 = span.first + pos0 - (span.context - span.n);
        const int page = page_of(p, s, index);  // (the same for the whole CTA)
        const Place at_k = place_of(p, i, true), at_v = place_of(p, i, false);
        // the queries of the group for a token
        auto queries = [&](int row, const Angles &t) {
            const unsigned short *from_a = p.q + (token0 + row) * p.q_ld + h * group * D + at_k.a, *from_b = from_a + (at_k.b - at_k.a);
            unsigned short *to_a = p.q_out + (token0 + row) * p.q_out_ld + h * group * D + at_k.a, *to_b = to_a + (at_k.b - at_k.a);
            auto some = [&](auto heads) {
                constexpr int N = decltype(heads)::value;
                Raw8 raw[N];
#pragma unroll
                for (int e = 0; e < N; ++e)
                    raw[e] = Raw8{*reinterpret_cast<const uint2 *>(from_a + e * D), *reinterpret_cast<const uint2 *>(from_b + e * D)};
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    float x[8];
                    decode8<HALF>(raw[e], x);
                    turn8<MODE>(x, t, at_k, p.paired);
                    *reinterpret_cast<uint2 *>(to_a + e * D) = make_uint2(pack16<HALF>(x[0], x[1]), pack16<HALF>(x[2], x[3]));
                    *reinterpret_cast<uint2 *>(to_b + e * D) = make_uint2(pack16<HALF>(x[4], x[5]), pack16<HALF>(x[6], x[7]));
                }
                from_a += N * D, from_b += N * D, to_a += N * D, to_b += N * D;
            };
            int left = group;
#pragma unroll 1
            for (; left >= kHeads; left -= kHeads) some(std::integral_constant<int, kHeads>());
#pragma unroll 1
            for (; left > 0; --left) some(std::integral_constant<int, 1>());
        };
        if (page < 0)
            for (int row = r0; row < count; row += kRows) queries(row, angles_of(p, pos0 + row, i, at_k.turned));
        if (page >= 0) {
            const size_t block = (size_t)page * p.kv_heads + h;
            const float old_k = begin ? p.k_scale[block] : 0.f, old_v = begin ? p.v_scale[block] : 0.f;
            unsigned mk = 0, mv = 0;
            bool wild = false;
#pragma unroll 1
            for (int row = r0; row < count; row += kRows) {
                const Raw8 v = fetch8(p.v + (token0 + row) * p.v_ld + h * D, at_v);
                const Angles t = angles_of(p, pos0 + row, i, at_k.turned);
                const Raw8 k = fetch8(p.k + (token0 + row) * p.k_ld + h * D, at_k);
                queries(row, t);
                float x[8];
                decode8<HALF>(k, x);
                turn8<MODE>(x, t, at_k, p.paired);
                mk = max(mk, amax8(x, wild));
                float4 *at = keys + row * (D / 4) + i;  // (sixteen bytes a lane, twice: no two lanes of a phase in a bank)
                at[0] = make_float4(x[0], x[1], x[2], x[3]), at[kLanes] = make_float4(x[4], x[5], x[6], x[7]);
                values[row * kLanes + i] = make_uint4(v.a.x, v.a.y, v.b.x, v.b.y);
                decode8<HALF>(v, x);
                mv = max(mv, amax8(x, wild));
            }
            mk = __reduce_max_sync(0xffffffffu, mk), mv = __reduce_max_sync(0xffffffffu, mv);
            if ((threadIdx.x & 31) == 0) atomicMax(&s_amax[0], mk), atomicMax(&s_amax[1], mv);
            __syncthreads();
            const float scale_k = fmaxf(old_k, scale_for(s_amax[0])), scale_v = fmaxf(old_v, scale_for(s_amax[1]));
            const float inv_k = 1.0f / scale_k, inv_v = 1.0f / scale_v;
            unsigned char *to_k = p.k_codes + block * page_tokens * D, *to_v = p.v_codes + block * page_tokens * D;
#pragma unroll 2
            for (int row = r0; row < count; row += kRows) {
                const float4 *at = keys + row * (D / 4) + i;
                const float4 a = at[0], b = at[kLanes];
                const uint4 v = values[row * kLanes + i];
                float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                store8(to_k + (begin + row) * D, at_k, x, inv_k, wild);
                decode8<HALF>(Raw8{make_uint2(v.x, v.y), make_uint2(v.z, v.w)}, x);
                store8(to_v + (begin + row) * D, at_v, x, inv_v, wild);
            }
            if (scale_k > old_k && begin)
                for (int e = threadIdx.x; e < begin * (D / 4); e += kAppendThreads) {
                    unsigned *w = reinterpret_cast<unsigned *>(to_k) + e;
                    *w = again4(*w, old_k / scale_k);
                }
            if (scale_v > old_v && begin)
                for (int e = threadIdx.x; e < begin * (D / 4); e += kAppendThreads) {
                    unsigned *w = reinterpret_cast<unsigned *>(to_v) + e;
                    *w = again4(*w, old_v / scale_v);
                }
            if (threadIdx.x == 0) p.k_scale[block] = scale_k, p.v_scale[block] = scale_v;
        }
        __syncthreads();  // the tile number and the amaxes are rewritten
    }
    if (threadIdx.x == 0) trace_end(blp, iter);
}

template <typename F>
static auto append_instance(int dim, bool half, int mode, F &&f) {
    auto modes = [&](auto d, auto hf) {
        constexpr int D = decltype(d)::value;
        constexpr bool H = decltype(hf)::value;
        if (mode == TURN_HALVES) return f(kv_append_one_kernel<D, H>, kv_append_kernel<D, H, TURN_HALVES>);
        if (mode == TURN_PAIRS) return f(kv_append_one_kernel<D, H>, kv_append_kernel<D, H, TURN_PAIRS>);
        return f(kv_append_one_kernel<D, H>, kv_append_kernel<D, H, TURN_ANY>);
    };
    using D64 = std::integral_constant<int, 64>;
    using D128 = std::integral_constant<int, 128>;
    if (dim == 64) return half ? modes(D64(), std::true_type()) : modes(D64(), std::false_type());
    return half ? modes(D128(), std::true_type()) : modes(D128(), std::false_type());
}

static cudaError_t append_launch(const AppendParams &p, int dim, bool half, const DeviceInfo &d, BlpArgs blp, cudaStream_t s) {
    const int sm_count = d.sm_count, device = d.device;
    const int page_tokens = 1 << p.page_shift;
    const int mode = p.rotated != dim ? TURN_ANY : p.paired ? TURN_PAIRS : TURN_HALVES;
    return append_instance(dim, half, mode, [&](auto one, auto any) {
        int per_sm;
        // One token a sequence at most: rows are independent, a group of lanes takes each.  (Device time with this kernel and with the
        // general one, 32 heads of 128 on 8: one sequence 4.4 and 6.1 us, 64 of them 4.9 and 10.8.)
        if (p.batch.most_new == 1) {
            const long long rows = (long long)p.batch.seqs * (2 * p.kv_heads + (p.q ? p.heads : 0));
            const int a_tile = kAppendOneThreads / (dim / 8);
            blp.total_tiles = (int)((rows + a_tile - 1) / a_tile);
            const cudaError_t e = lm_resident((const void *)one, kAppendOneThreads, 0, 0, device, &per_sm);
            if (e != cudaSuccess) return e;
            const int grid = (int)std::min<long long>(blp.total_tiles, (long long)sm_count * per_sm);
            return launch_layer(one, grid, kAppendOneThreads, 0, s, p, blp);
        }
        const size_t smem = (size_t)page_tokens * dim * 6 + lm_prefix_bytes(p.batch.seqs);
        const size_t most = (size_t)kMostPageTokens * dim * 6 + lm_prefix_bytes(kLmMaxSeqs);
        const cudaError_t e = lm_resident((const void *)any, kAppendThreads, smem, most, device, &per_sm);
        if (e != cudaSuccess) return e;
        // (pages that new tokens can touch: full ones, and two parts of one a sequence)
        const long long tiles = ((long long)p.batch.tokens / page_tokens + 2ll * std::min(p.batch.seqs, p.batch.tokens)) * p.kv_heads;
        const int grid = (int)std::min<long long>(tiles, (long long)sm_count * per_sm);
        return launch_layer(any, grid, kAppendThreads, smem, s, p, blp);
    });
}

}  // namespace gpx

using namespace gpx;

extern "C" int gpx_kv_append(const gpx_kv_cache *cache, const gpx_kv_batch *batch, const gpx_kv_append_args *args, void *ctx,
                             const gpx_blp *blp, gpx_stream stream) {
    GPX_REQUIRE(cache && args && ctx, GPX_FAIL, "cache, args or ctx is NULL");
    GPX_REQUIRE((uintptr_t)ctx % 256 == 0, GPX_FAIL, "ctx must be 256-byte aligned");
    AppendParams p{};
    BlpArgs b;
    int elem;
    GPX_TRY(lm_check_batch(batch, &p.batch));
    GPX_TRY(lm_check_blp(blp, &b));
    GPX_TRY(lm_elem(args->dtype, false, &elem));
    const gpx_kv_append_args &a = *args;
    GPX_REQUIRE(a.k && a.v && !a.q == !a.q_out, GPX_FAIL, "k or v is NULL, or one of q and q_out");
    GPX_REQUIRE(a.heads > 0 && a.heads % cache->kv_heads == 0, GPX_OUT_OF_RANGE, "%d heads are not a multiple of the cache's %d",
                a.heads, cache->kv_heads);
    GPX_REQUIRE(a.rotated >= 0 && a.rotated <= cache->dim && a.rotated % 8 == 0, GPX_OUT_OF_RANGE,
                "rotated is a multiple of 8 up to %d, not %d", cache->dim, a.rotated);
    GPX_REQUIRE(!a.rotated || (a.cos && a.sin && (uintptr_t)a.cos % 16 == 0 && (uintptr_t)a.sin % 16 == 0 && a.positions > 0), GPX_FAIL,
                "a rotation needs cos and sin tables, 16-byte aligned, of at least one position");
    const long long q_row = (long long)a.heads * cache->dim, kv_row = (long long)cache->kv_heads * cache->dim;
    p.q_ld = a.q_ld ? a.q_ld : q_row, p.q_out_ld = a.q_out_ld ? a.q_out_ld : q_row;
    p.k_ld = a.k_ld ? a.k_ld : kv_row, p.v_ld = a.v_ld ? a.v_ld : kv_row;
    GPX_REQUIRE(p.q_ld >= q_row && p.q_out_ld >= q_row && p.k_ld >= kv_row && p.v_ld >= kv_row, GPX_OUT_OF_RANGE,
                "a token's row is longer than the distance to the next");
    GPX_REQUIRE((p.q_ld | p.q_out_ld | p.k_ld | p.v_ld) % 4 == 0 &&
                    ((uintptr_t)a.q | (uintptr_t)a.q_out | (uintptr_t)a.k | (uintptr_t)a.v) % 8 == 0,
                GPX_FAIL, "q, k, v and q_out must be 8-byte aligned, their distances multiples of 4 elements");
    GPX_REQUIRE(a.q != a.q_out || p.q_ld == p.q_out_ld, GPX_FAIL, "queries turned in place keep their distance");
    GPX_REQUIRE(((long long)p.batch.tokens / cache->page_tokens + 2ll * p.batch.seqs) * cache->kv_heads <= 0x7fffffffll &&
                    (long long)p.batch.seqs * (2ll * cache->kv_heads + a.heads) <= 0x7fffffffll,
                GPX_OUT_OF_RANGE, "too many rows");
    const DeviceInfo &d = device_info();
    GPX_REQUIRE(d.device >= 0, GPX_FAIL, "gpx_init was not called");
    if (p.batch.most_new == 0) return GPX_SUCC;
    p.k_codes = cache->k, p.v_codes = cache->v, p.k_scale = cache->k_scale, p.v_scale = cache->v_scale;
    p.pages = cache->pages, p.page_shift = __builtin_ctz((unsigned)cache->page_tokens), p.kv_heads = cache->kv_heads, p.heads = a.heads;
    p.q = (const unsigned short *)a.q, p.k = (const unsigned short *)a.k, p.v = (const unsigned short *)a.v;
    p.q_out = (unsigned short *)a.q_out;
    p.cos = (const float *)a.cos, p.sin = (const float *)a.sin;
    p.rotated = a.rotated, p.positions = a.positions, p.paired = a.paired != 0;
    p.error = lm_ctx(ctx).error;
    GPX_CUDA(append_launch(p, cache->dim, elem == LM_F16, d, b, as_stream(stream)));
    return GPX_SUCC;
}
