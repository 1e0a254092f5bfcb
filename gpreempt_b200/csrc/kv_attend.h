// What the two kernels of attention over a paged cache share: parameters, a unit of work, formats.
#pragma once

#include "lm.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace gpx {

struct AttendParams {
    CUtensorMap map_k, map_v;
    LmBatch batch;
    const unsigned char *v_codes;
    const float *k_scale, *v_scale;
    int pages, page_shift, kv_heads, heads;
    const unsigned short *q;
    unsigned short *out;
    float *lse;
    long long q_ld, out_ld;
    float scale;
    int causal, window;
    int max_tiles;
    int blocks_a_tile;  // of a preemptible launch; 0: as many tiles as CTAs
    int *error, *counters, *prefix;
    float *parts;
};

// Few rows a head of keys (kv_attend.cu), and many of them (kv_attend_tcgen05.cu).
cudaError_t kv_attend_few_launch(AttendParams &p, int dim, bool half, const DeviceInfo &d, const BlpArgs &blp, cudaStream_t s);
cudaError_t kv_attend_many_launch(AttendParams &p, int dim, bool half, const DeviceInfo &d, const BlpArgs &blp, cudaStream_t s);

#if defined(__CUDACC__)

__device__ __forceinline__ uint32_t pack_halves(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_halves(uint32_t w) { return __half22float2(*reinterpret_cast<__half2 *>(&w)); }
template <bool HALF>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
    if (HALF) return pack_halves(a, b);
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// The power of two below a row's largest query (bits of its magnitude), which brings the row's queries into the range of halves; at
// least 2^-126 and at most 2^125, so that it and its reciprocal are normal numbers (halves have room for what is left of larger ones).
__device__ __forceinline__ float query_factor(uint32_t most) { return __uint_as_float(min(max(most >> 23, 1u), 252u) << 23); }
// 0xff in every byte that is e4m3's NaN (all bits but the sign)
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }

// The first key that a row at a position sees (which is negative where there are more new tokens than keys).
__device__ __forceinline__ int first_seen(const AttendParams &p, int position) {
    return p.window && position >= p.window ? position - p.window + 1 : 0;
}

// A unit's place on the line of blocks, and what it covers.
struct Unit {
    int s, head, row0, rows;      // sequence, head of keys, first of its rows and how many
    int first, n, context;
    int key0;                     // of its first block (a multiple of a block)
    int low, high;                // keys that some row sees: [low, high)
};

// How a sequence falls into units of ROWS rows and blocks of KEYS keys.  Where line() is used, all units of a sequence
// count as many blocks as the longest, so that the place of a block can be computed.
template <int ROWS, int KEYS>
struct Layout {
    const AttendParams &p;
    int group;
    __device__ Layout(const AttendParams &p_) : p(p_), group(p_.heads / p_.kv_heads) {}
    __device__ int row_blocks(int n) const { return (n * group + ROWS - 1) / ROWS; }
    // blocks of keys of each unit of a sequence: the most that one of its blocks of rows can see, one at least
    __device__ int key_blocks(const LmSpan &span) const {
        int keys = span.context;
        // (rows of a block span so many tokens; the first key need not start a block)
        if (p.window) keys = min((long long)keys, (long long)p.window + (ROWS - 1 + group - 1) / group + KEYS - 1);
        return max(1, (keys + KEYS - 1) / KEYS);
    }
    __device__ int line(const LmSpan &span) const {
        const long long all = (long long)row_blocks(span.n) * p.kv_heads * key_blocks(span);
        return all > 0x7fffffff ? 0x7fffffff : (int)all;
    }
    __device__ Unit unit(int s, int index) const {
        Unit u;
        u.s = s;
        u.first = p.batch.first[s], u.n = p.batch.first[s + 1] - u.first, u.context = p.batch.context[s];
        const int blocks = row_blocks(u.n);
        u.head = index / blocks, u.row0 = (index - u.head * blocks) * ROWS;
        u.rows = min(ROWS, u.n * group - u.row0);
        u.low = 0, u.high = u.context;
        if (p.causal) {
            u.high = max(0, u.context - u.n + (u.row0 + u.rows - 1) / group + 1);
            u.low = first_seen(p, u.context - u.n + u.row0 / group);
        }
        u.low = min(u.low, u.high);
        u.key0 = u.low & ~(KEYS - 1);
        return u;
    }
};

#endif  // __CUDACC__

}  // namespace gpx
