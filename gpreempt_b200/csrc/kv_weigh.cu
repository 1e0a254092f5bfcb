// What each key of a paged 8-bit cache has weighed in the attention of new tokens, added to its account.
//
//   w_j = decay w_j (0 for a key of this step) + sum over rows r that see j of e^(scale q_r . k_j k_scale(page of j) - lse_r)
//
// The normalisers are known, so that keys need no look at one another: a key is read once, multiplied by all rows, and its row of
// exponentials summed.  The floor is memory for few rows (D bytes of codes a key and head, 4 read and 4 written of its account, against
// 2 D operations a row); from some eight rows on it is instructions, which for 64 rows, where keys are read twice, take five times as long
// (the table below).  As in the attention of few rows, keys are the M side of the tensor instructions and rows the N side,
// codes become halves in registers, and queries are halves of their row's power of two.  Nothing is shared between warps but the
// queries, and codes go from memory to the registers where they are operands: a lane's elements of a key are 16-byte pieces.
//
// A warp takes sixteen keys of a block of 64; the sum over a key's rows stays in one warp, in the order of the rows, so that the
// result does not depend on the launch.  Rows beyond what an instance holds go over the keys again; the page of a key that any row
// sees is looked up by every pass, so that all agree which keys have none.
//
// Measured, 32 heads of 128 on 8, bf16: single tokens of 64 sequences over 16 384 keys at most 125 us (608 MB, 4.9 TB/s; 116 where a part of
// the keys is in L2 already), of one over 517 a launch.  238 instructions for sixteen keys and eight rows (their codes' conversions are
// 32, the products 8) fill 56 % of the slots with 16 warps an SM: dependent ones, which more warps do not have registers to hide (five
// CTAs an SM, at 96 registers, took 138 us, three, at 168, 138 too, with the operands of the rows in registers 120 against 119).
#include "kv_weigh.h"

#include <algorithm>

namespace gpx {

constexpr int kWeighWarps = 4, kWeighThreads = 32 * kWeighWarps;
constexpr int kWeighKeys = 64;

__device__ __forceinline__ uint4 load_codes(const unsigned char *at) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at));
    return v;
}

template <int D, int NT, bool HALF>
__global__ void __launch_bounds__(kWeighThreads, NT == 1 ? 4 : 3)
kv_weigh_kernel(const __grid_constant__ WeighParams p, BlpArgs blp) {
    constexpr int KS = D / 16, ROWS = 8 * NT, P = D / 64;  // steps of a product; 16-byte pieces of a key that a lane holds
    extern __shared__ int prefix[];  // [seqs + 1]
    __shared__ uint2 q_frag[NT * KS * 32];
    __shared__ float s_factor[ROWS], s_lse[ROWS];
    __shared__ int s_tile;
    const int tid = threadIdx.x, lane = tid & 31, wid = __shfl_sync(0xffffffffu, tid >> 5, 0), g = lane >> 2, t = lane & 3;
    pdl_enter();
    const bool dynamic = blp.preempted != nullptr;
    if (tid == 0) trace_begin(blp);
    const int group = p.heads / p.kv_heads, page_tokens = 1 << p.page_shift;
    const int n_line = lm_prefix(prefix, p.batch.seqs, p.error, [&](int s) {
        const LmSpan span = weigh_span(p, s);
        const long long all = span.n ? (long long)p.kv_heads * ((span.context + kWeighKeys - 1) / kWeighKeys) : 0;
        return all > 0x7fffffff ? 0x7fffffff : (int)all;
    });
    int tiles = dynamic ? max((n_line + p.blocks_a_tile - 1) / p.blocks_a_tile, (int)gridDim.x) : (int)gridDim.x;
    tiles = min(tiles, n_line);
    blp.total_tiles = tiles;
    const LmCut cut(n_line, tiles);

    int iter = 0;
    for (;; ++iter) {
        int tile;
        if (dynamic) {
            if (tid == 0) s_tile = blp_claim(blp, iter);
            __syncthreads();
            tile = s_tile;
            __syncthreads();
        } else {
            tile = blp_claim(blp, iter);
        }
        if (tile < 0) break;
        int begin = cut.begin(tile);
        const int end = cut.begin(tile + 1);
        while (begin < end) {
            // ---- a piece of a unit: some blocks of one head of a sequence
            const int s = lm_find(prefix, p.batch.seqs, begin);
            const int first = p.batch.first[s], n = p.batch.first[s + 1] - first, context = p.batch.context[s];
            const int unit_blocks = (context + kWeighKeys - 1) / kWeighKeys;
            const int head = (begin - prefix[s]) / unit_blocks, block0 = begin - prefix[s] - head * unit_blocks;
            const int blocks = min(end - begin, unit_blocks - block0);
            begin += blocks;
            const int votes = p.observed ? min(n, p.observed) : n, rows = votes * group;
            const int slot = p.account.slots ? p.account.slots[s] : s;
            float *const account = p.account.weights + ((long long)slot * p.kv_heads + head) * p.account.ld;
            const int fresh = p.causal ? max(0, context - n) : context;  // keys from here on begin their account
            // the first key that a row sees (from there on some row sees each)
            const int seen = p.window && context - votes >= p.window ? context - votes - p.window + 1 : 0;
            for (int row0 = 0; row0 < rows; row0 += ROWS) {
                const int some_rows = min(ROWS, rows - row0);
                auto position = [&](int r) { return context - votes + (row0 + r) / group; };  // (of the rows r of this pass)
                auto upto = [&](int pos) { return p.causal ? min(context, max(pos + 1, 0)) : context; };
                auto from = [&](int pos) { return p.window && pos >= p.window ? pos - p.window + 1 : 0; };
                // keys that some row sees, and those that every row sees
                const int pos0 = position(0), pos1 = position(some_rows - 1);
                const int low = from(pos0), high = upto(pos1), all_low = from(pos1), all_high = upto(pos0);
                // what a lane knows of the sixteen keys of its warp in block b0 + lane: row of the cache's codes (-1: no row of this pass
                // sees them, -2: of no page, and the accounts of those that a row of any pass sees stay as they are)
                int at_row = -2;
                float at_scale = 0.f;
                auto look_up = [&](int b0) {
                    at_row = -2;
                    const int key = (block0 + b0 + lane) * kWeighKeys + wid * 16;
                    if (b0 + lane >= blocks || key >= context) return;
                    at_row = -1;
                    if (key + 16 <= seen) return;  // (what ends below may be anybody's by now: its page is not looked up)
                    const int page = p.batch.table[(size_t)s * p.batch.table_ld + (key >> p.page_shift)];
                    if ((unsigned)page >= (unsigned)p.pages) {
                        lm_fail(p.error, LM_BAD_PAGE, s);
                        at_row = -2;
                    } else if (key < high && key + 16 > low) {
                        const long long block = (long long)page * p.kv_heads + head;
                        at_row = (int)((block << p.page_shift) + (key & (page_tokens - 1)));
                        at_scale = p.k_scale[block];
                    }
                };
                struct Keys {
                    uint4 a[P], b[P];  // of keys g and g + 8
                    float old;         // account of key g + 8 t (t < 2)
                };
                auto fetch = [&](int b0, int b) {
                    Keys k;
                    const int row = __shfl_sync(0xffffffffu, at_row, b & 31);
                    const unsigned char *codes = p.k_codes + (size_t)max(row, 0) * D + g * D + 16 * t;
#pragma unroll
                    for (int c = 0; c < P; ++c) {
                        k.a[c] = row >= 0 && b < 32 ? load_codes(codes + 64 * c) : make_uint4(0, 0, 0, 0);
                        k.b[c] = row >= 0 && b < 32 ? load_codes(codes + 8 * D + 64 * c) : make_uint4(0, 0, 0, 0);
                    }
                    const int key = (block0 + b0 + b) * kWeighKeys + wid * 16 + g + 8 * t;
                    k.old = t < 2 && b < 32 && (row != -2 || key < seen) && key < context && (key < fresh || row0 > 0) ? account[key] : 0.f;
                    return k;
                };
                look_up(0);
                Keys k0 = fetch(0, 0), k1 = fetch(0, 1);
                // ---- the rows' queries as operands
                for (int nt = wid; nt < NT; nt += kWeighWarps) {
                    const int r = nt * 8 + g, at = row0 + r;
                    const bool live = r < some_rows;
                    const long long token = first + n - votes + at / group;
                    const int h = head * group + at % group;
                    uint32_t q[KS][2];
                    const float factor = query_operand<KS, HALF>(p.q + (live ? token * p.q_ld + h * D : 0), live, t, q);
#pragma unroll
                    for (int k = 0; k < KS; ++k) q_frag[(nt * KS + k) * 32 + lane] = make_uint2(q[k][0], q[k][1]);
                    if (t == 0) s_factor[r] = factor, s_lse[r] = live ? p.lse[token * p.heads + h] : 0.f;
                }
                __syncthreads();
                // this lane's columns: rows 8 nt + 2 t and the next
                float mult[NT][2], lse[NT][2];
                int lo[NT][2], hi[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int r = 8 * nt + 2 * t + c, pos = position(r);
                        mult[nt][c] = s_factor[r] * p.scale, lse[nt][c] = s_lse[r];
                        lo[nt][c] = from(pos), hi[nt][c] = r < some_rows ? upto(pos) : 0;
                    }
                auto weigh = [&](int b0, int b, Keys &k) {
                    const int row = __shfl_sync(0xffffffffu, at_row, b);
                    const float ks = __shfl_sync(0xffffffffu, at_scale, b);
                    const int key0 = (block0 + b0 + b) * kWeighKeys + wid * 16;
                    float sum[2] = {0.f, 0.f};  // of keys g and g + 8
                    const float old = k.old;
                    if (row >= 0) {
                        float sc[NT][4];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 4; ++c) sc[nt][c] = 0.f;
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            const uint4 &A = k.a[i >> 2], &B = k.b[i >> 2];
                            const uint32_t wa = (i & 3) == 0 ? A.x : (i & 3) == 1 ? A.y : (i & 3) == 2 ? A.z : A.w;
                            const uint32_t wb = (i & 3) == 0 ? B.x : (i & 3) == 1 ? B.y : (i & 3) == 2 ? B.z : B.w;
                            const uint32_t a0 = e4m3x2_to_f16x2((unsigned short)wa), a2 = e4m3x2_to_f16x2((unsigned short)(wa >> 16));
                            const uint32_t a1 = e4m3x2_to_f16x2((unsigned short)wb), a3 = e4m3x2_to_f16x2((unsigned short)(wb >> 16));
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                const uint2 q = q_frag[(nt * KS + i) * 32 + lane];
                                mma_16816(sc[nt], a0, a1, a2, a3, q.x, q.y);
                            }
                        }
                        const bool border = key0 + 16 > all_high || key0 < all_low;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                // (in the units of the normaliser: the difference is rounded once, however large the two are)
                                float e = lm_ex2(fmaf(sc[nt][c], mult[nt][c & 1] * ks, -lse[nt][c & 1]) * 1.4426950408889634f);
                                if (border) {
                                    const int key = key0 + g + (c & 2) * 4;
                                    if (key >= hi[nt][c & 1] || key < lo[nt][c & 1]) e = 0.f;
                                } else if (hi[nt][c & 1] == 0) {  // (a column without a row, whose products may be no numbers)
                                    e = 0.f;
                                }
                                sum[c >> 1] += e;
                            }
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], 1);
                            sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], 2);
                        }
                    }
                    const int key = key0 + g + 8 * t;
                    if (t >= 2 || key >= context || (row == -2 && key >= seen)) return;
                    const float add = t ? sum[1] : sum[0];
                    if (row0 > 0) {
                        if (row >= 0) account[key] = old + add;
                    } else if (row >= 0 || key >= fresh || p.decay != 1.f) {
                        account[key] = key < fresh ? fmaf(p.decay, old, add) : add;
                    }
                };
                for (int b0 = 0;;) {
                    const int some = min(32, blocks - b0);
                    for (int b = 0; b < some; b += 2) {
                        Keys now = k0;
                        if (b + 2 < some) k0 = fetch(b0, b + 2);
                        weigh(b0, b, now);
                        if (b + 1 >= some) break;
                        now = k1;
                        if (b + 3 < some) k1 = fetch(b0, b + 3);
                        weigh(b0, b + 1, now);
                    }
                    b0 += 32;
                    if (b0 >= blocks) break;
                    look_up(b0);
                    k0 = fetch(b0, 0), k1 = fetch(b0, 1);
                }
                __syncthreads();  // the queries are rewritten
            }
            if (head == 0 && block0 == 0) lm_slot_twice(p.account, s, tid, kWeighThreads, p.error);
        }
    }
    if (tid == 0) trace_end(blp, iter);
}

template <typename F>
static auto weigh_instance(int dim, int rows, bool half, F &&f) {
    auto by_rows = [&](auto d, auto hf) {
        constexpr int D = decltype(d)::value;
        constexpr bool H = decltype(hf)::value;
        if (rows <= 8) return f(kv_weigh_kernel<D, 1, H>, 8);
        if (rows <= 16) return f(kv_weigh_kernel<D, 2, H>, 16);
        return f(kv_weigh_kernel<D, 4, H>, 32);
    };
    using D64 = std::integral_constant<int, 64>;
    using D128 = std::integral_constant<int, 128>;
    if (dim == 64) return half ? by_rows(D64(), std::true_type()) : by_rows(D64(), std::false_type());
    return half ? by_rows(D128(), std::true_type()) : by_rows(D128(), std::false_type());
}

// Rows of a head of keys from which on the other kernel takes over.  This and the other, us, 32 heads of 128 on 8, bf16:
//   rows                           64           96          128          256          1 024
//    4 sequences over  2 000   17.5         23.6         29.7 17.6    46.0 24.0    169  48.9
//   16 sequences over  2 000   30.8         43.0         50.2 37.3    90.7 51.5    339 117
//    2 sequences over 20 000   32.8         46.3         59.9 37.1   111   52.8    415 135
//    8 sequences over  8 000   44.2         59.4         77.1 54.1   140   74.0    532 171
// (a chunk of 64 rows is the same work for the other, whatever it holds)
constexpr int kManyVotes = 64;

static cudaError_t weigh_launch(WeighParams &p, int dim, bool half, const DeviceInfo &d, const BlpArgs &blp, cudaStream_t s) {
    const int votes = p.observed ? std::min(p.observed, p.batch.most_new) : p.batch.most_new;
    const long long rows = (long long)votes * (p.heads / p.kv_heads);
    return weigh_instance(dim, (int)std::min<long long>(rows, 1 << 20), half, [&](auto kernel, int a_pass) {
        int per_sm;
        const size_t smem = lm_prefix_bytes(p.batch.seqs), most = lm_prefix_bytes(kLmMaxSeqs);
        const cudaError_t e = lm_resident((const void *)kernel, kWeighThreads, smem, most, d.device, &per_sm);
        if (e != cudaSuccess) return e;
        p.blocks_a_tile = (int)std::max<long long>(1, 16 / ((rows + a_pass - 1) / a_pass));
        return launch_layer(kernel, d.sm_count * per_sm, kWeighThreads, smem, s, p, blp);
    });
}

}  // namespace gpx

using namespace gpx;

extern "C" int gpx_kv_weigh(const gpx_kv_cache *cache, const gpx_kv_batch *batch, const gpx_kv_weights *account, const gpx_kv_weigh_args *args,
                            void *ctx, const gpx_blp *blp, gpx_stream stream) {
    GPX_REQUIRE(cache && args && ctx, GPX_FAIL, "cache, args or ctx is NULL");
    GPX_REQUIRE((uintptr_t)ctx % 256 == 0, GPX_FAIL, "ctx must be 256-byte aligned");
    const gpx_kv_weigh_args &a = *args;
    WeighParams p{};
    BlpArgs b;
    int elem;
    GPX_TRY(lm_check_batch(batch, &p.batch));
    GPX_TRY(lm_check_account(account, p.batch, &p.account));
    GPX_TRY(lm_check_blp(blp, &b));
    GPX_TRY(lm_elem(a.dtype, false, &elem));
    GPX_REQUIRE(a.q && a.lse, GPX_FAIL, "q or lse is NULL");
    GPX_REQUIRE(p.account.kv_heads == cache->kv_heads, GPX_OUT_OF_RANGE, "accounts of %d heads for a cache of %d", p.account.kv_heads,
                cache->kv_heads);
    GPX_REQUIRE(a.heads > 0 && a.heads % cache->kv_heads == 0, GPX_OUT_OF_RANGE, "%d heads are not a multiple of the cache's %d",
                a.heads, cache->kv_heads);
    GPX_REQUIRE(a.window >= 0 && (!a.window || a.causal), GPX_OUT_OF_RANGE, "a window of %d, causal %d", a.window, a.causal);
    GPX_REQUIRE(a.observed >= 0, GPX_OUT_OF_RANGE, "%d tokens observed", a.observed);
    GPX_REQUIRE(a.scale == a.scale && a.scale >= 0.f && a.scale <= 3.4e38f, GPX_OUT_OF_RANGE, "scale must be positive and finite, or 0");
    GPX_REQUIRE(a.decay > 0.f && a.decay <= 1.f, GPX_OUT_OF_RANGE, "decay must be above 0 and at most 1");
    const long long row = (long long)a.heads * cache->dim;
    p.q_ld = a.q_ld ? a.q_ld : row;
    GPX_REQUIRE(p.q_ld >= row, GPX_OUT_OF_RANGE, "a token's row is longer than the distance to the next");
    GPX_REQUIRE(p.q_ld % 8 == 0 && (uintptr_t)a.q % 16 == 0 && (uintptr_t)a.lse % 4 == 0, GPX_FAIL,
                "q must be 16-byte aligned, its distance a multiple of 8 elements, lse 4-byte aligned");
    GPX_REQUIRE((long long)p.batch.most_new * a.heads <= 0x7fffffff - 256, GPX_OUT_OF_RANGE, "too many rows");
    const DeviceInfo &d = device_info();
    GPX_REQUIRE(d.device >= 0, GPX_FAIL, "gpx_init was not called");
    if (p.batch.most_new == 0) return GPX_SUCC;
    p.k_codes = cache->k, p.k_scale = cache->k_scale;
    p.pages = cache->pages, p.page_shift = __builtin_ctz((unsigned)cache->page_tokens), p.kv_heads = cache->kv_heads, p.heads = a.heads;
    p.q = (const unsigned short *)a.q, p.lse = (const float *)a.lse;
    p.scale = a.scale != 0.f ? a.scale : 1.0f / sqrtf((float)cache->dim);
    p.decay = a.decay, p.causal = a.causal != 0, p.window = a.window, p.observed = a.observed;
    const LmCtx c = lm_ctx(ctx);
    p.error = c.error, p.counters = c.counters, p.parts = c.parts;
    const long long votes = p.observed ? std::min(p.observed, p.batch.most_new) : p.batch.most_new;
    const bool many = votes * (a.heads / cache->kv_heads) > kManyVotes;
    GPX_CUDA((many ? kv_weigh_many_launch : weigh_launch)(p, cache->dim, elem == LM_F16, d, b, as_stream(stream)));
    return GPX_SUCC;
}
