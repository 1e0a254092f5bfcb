// What the operators of a decoder's serving step share: the paged cache, the description of a ragged batch, the
// scratch context, and the search for a tile's sequence.
#pragma once

#include "blp.cuh"
#include "common.h"

#include <cuda.h>
#include <cuda_runtime.h>

struct gpx_kv_cache {
    unsigned char *k, *v;      // e4m3 codes [page][kv head][slot][element]
    float *k_scale, *v_scale;  // [page][kv head]
    int pages, page_tokens, kv_heads, dim;
    CUtensorMap map_k, map_v;  // rows of `dim` bytes, boxes of min(page_tokens, 64) rows, swizzled
};

namespace gpx {

// ---- scratch context ------------------------------------------------------------------------------

// Header, arrival counters (zero between launches: whoever joins the parts of a result puts its counter back), and
// what CTAs have in common: sums over the sequences of a batch, parts of results.
constexpr int kLmCounters = 65536;
constexpr int kLmMaxSeqs = 4096;
constexpr int kMostPageTokens = 128;
constexpr int kMostContext = 0x7fffffff - 4096;  // of a sequence: the ends of its last page and of the blocks fetched ahead are still an int
constexpr size_t kLmResetBytes = 256 + kLmCounters * sizeof(int);
constexpr size_t kLmPartsOffset = kLmResetBytes + (kLmMaxSeqs + 64) * sizeof(int);
constexpr size_t kLmPartsBytes = (size_t)64 << 20;
constexpr size_t kLmCtxBytes = kLmPartsOffset + kLmPartsBytes;

enum LmError {
    LM_BAD_SPAN = 1,      // first[] / context[] of a sequence contradict each other or the limits given
    LM_BAD_PAGE = 2,      // a page number outside the cache
    LM_BAD_POSITION = 3,  // a position past the rotation table
    LM_GAVE_UP = 4,       // a bounded wait ran out
    LM_TOO_LONG = 5,      // more blocks of work than 31 bits count
};

struct LmCtx {
    int *error;  // {code, sequence or CTA}
    int *counters;
    int *prefix;  // [kLmMaxSeqs + 1]
    float *parts;
};

inline LmCtx lm_ctx(void *ctx) {
    unsigned char *p = static_cast<unsigned char *>(ctx);
    return {reinterpret_cast<int *>(p), reinterpret_cast<int *>(p + 256), reinterpret_cast<int *>(p + kLmResetBytes), reinterpret_cast<float *>(p + kLmPartsOffset)};
}

// ---- batch ----------------------------------------------------------------------------------------

struct LmBatch {
    const int *table;    // [seqs][table_ld] page numbers
    const int *context;  // [seqs] tokens of a sequence, the new ones among them
    const int *first;    // [seqs + 1] offsets of the sequences' new tokens
    int table_ld, seqs, tokens, most_new;
};

int lm_check_batch(const gpx_kv_batch *b, LmBatch *out);
int lm_check_blp(const gpx_blp *blp, BlpArgs *out);
int lm_elem(const char *dtype, bool f32_too, int *elem);  // dtype name -> GPX_LM_*

enum { LM_F32 = 0, LM_BF16 = 1, LM_F16 = 2 };

#if defined(__CUDACC__)

// CTAs of a kernel that an SM holds with `smem` bytes of dynamic shared memory, of which no launch of it asks for more than
// `most`.  Asked for once a thread, device and KiB (the question costs more than a small launch).  The limit of a kernel's
// shared memory belongs to the process: it is only ever set to `most`, so that no thread takes it from under another's launch.
cudaError_t lm_resident(const void *kernel, int threads, size_t smem, size_t most, int device, int *per_sm);
// Shared memory for the sums over the sequences of a batch, in steps of a KiB (as an SM deals it out): batches of about
// the same size are of one size here.
constexpr size_t lm_prefix_bytes(int seqs) { return ((size_t)(seqs + 1) * sizeof(int) + 1023) / 1024 * 1024; }

__device__ __forceinline__ void lm_fail(int *error, int code, int where) {
    if (atomicCAS(error, 0, code) == 0) error[1] = where;
}

struct LmSpan {
    int first, n, context;  // new tokens [first, first + n) of a sequence of `context` tokens
};

// A span that contradicts itself or the limits of the batch counts as empty, and is reported.
__device__ __forceinline__ LmSpan lm_span(const LmBatch &b, int s, int page_tokens, bool new_in_context, int *error) {
    const int f = b.first[s], e = b.first[s + 1], c = b.context[s];
    const bool fine = f >= 0 && e >= f && e <= b.tokens && e - f <= b.most_new && c >= 0 &&
                      c <= kMostContext && c <= (long long)b.table_ld * page_tokens && (!new_in_context || c >= e - f);
    if (!fine) {
        lm_fail(error, LM_BAD_SPAN, s);
        return {0, 0, 0};
    }
    return {f, e - f, c};
}

// prefix[s] = sum of count(0 .. s-1), prefix[seqs] = the total, for all threads of the CTA together.  A total of
// 2^31 - 1 and more is reported, and nothing is to be done; a count of 2^31 - 1 may stand for one beyond.
template <typename F>
__device__ __forceinline__ int lm_prefix(int *prefix, int seqs, int *error, F &&count) {
    __shared__ unsigned s_sums[32];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
    long long before_all = 0;
    for (int s0 = 0; s0 < seqs; s0 += blockDim.x) {
        const int s = s0 + threadIdx.x;
        const int own = s < seqs ? count(s) : 0;
        unsigned sum = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const unsigned up = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum = min(sum + up, 0x7fffffffu);
        }
        if (s0 > 0) __syncthreads();  // the sums of the round before have been read
        if (lane == 31) s_sums[wid] = sum;
        __syncthreads();
        long long before = before_all;
        for (int w = 0; w < warps; ++w) {
            if (w < wid) before += s_sums[w];
            before_all += s_sums[w];
        }
        if (s < seqs) prefix[s] = (int)(before + sum - own);
    }
    const bool fits = before_all < 0x7fffffff;
    if (threadIdx.x == 0) {
        if (!fits) lm_fail(error, LM_TOO_LONG, 0);
        prefix[seqs] = (int)before_all;
    }
    __syncthreads();
    return fits ? (int)before_all : 0;
}

// An even cut of a line of blocks into tiles: tile t begins at t line / tiles, rounded down, without divisions of 64 bits, which
// are a tenth of a small launch.  The step is rounded up, so that the place is exact: where units are of one length, their ends
// are ends of tiles whenever they can be (a cache of 131 071 tokens takes 54.8 us, 57.5 with a step rounded down, and 58.5 with the
// longer tiles first).
struct LmCut {
    int line, tiles;
    unsigned long long step;  // blocks a tile, times 2^32, rounded up
    float a_block;            // tiles a block
    __device__ __forceinline__ LmCut(int n, int t) : line(n), tiles(t), step(0), a_block(n ? (float)t / (float)n : 0.f) {
        if (t <= 0) return;
        const unsigned long long whole = (unsigned long long)n << 32;
        step = (unsigned long long)((double)n / t * 4294967296.0);
        while (step * t < whole) ++step;
        while (step > 0 && (step - 1) * t >= whole) --step;
    }
    __device__ __forceinline__ int begin(int tile) const { return tile >= tiles ? line : (int)(tile * step >> 32); }
    __device__ __forceinline__ int tile_of(int block) const {
        int tile = min((int)((float)block * a_block), tiles - 1);
        while (tile > 0 && begin(tile) > block) --tile;
        while (begin(tile + 1) <= block) ++tile;
        return tile;
    }
};

// The sequence whose share of [0, prefix[seqs]) holds i.
__device__ __forceinline__ int lm_find(const int *prefix, int seqs, int i) {
    int lo = 0, hi = seqs;  // prefix[lo] <= i < prefix[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

// 2^x, the hardware approximation (relative error ~2^-22; -inf gives 0).
__device__ __forceinline__ float lm_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two e4m3 codes (the lower byte is the lower element) as a pair of halves: exact.
__device__ __forceinline__ unsigned e4m3x2_to_f16x2(unsigned short codes) {
    unsigned d;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(codes));
    return d;
}

// Rounded to nearest even; beyond 448 the largest code, NaN stays NaN.
__device__ __forceinline__ unsigned e4m3x2(float lower, float upper) {
    unsigned short d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(upper), "f"(lower));
    return d;
}

#endif  // __CUDACC__

}  // namespace gpx
