// What a conversation keeps of its cache: choosing the tokens that weigh most in each head's account, and moving them to fresh pages.
#include "lm.h"
#include "sm100.cuh"

#include <algorithm>
#include <cuda_fp16.h>

namespace gpx {

constexpr long long kMostKept = 1ll << 31;  // from one head's kept tokens to the next one's

// ---- choosing -------------------------------------------------------------------------------------

struct ChooseParams {
    LmAccount account;
    const int *context;
    int *kept, *counts;
    long long kept_ld;
    int keep, first, last;
    int chunk;  // weights that shared memory has room for
    int *error;
};

constexpr int kChooseHeld = 32, kChooseBatch = 8;  // weights that a thread has room for, and how many it reads at a time
constexpr int kChooseBins = 2048;

// Numbers in their order as unsigned ones: negative, zeros (of either sign), positive, infinity, NaN.
__device__ __forceinline__ unsigned rank_of(float w) {
    const unsigned u = __float_as_uint(w);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    if ((u & 0x7fffffffu) == 0) return 0x80000000u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The least rank that is kept is found digit by digit (11, 11 and 10 bits) from counts of the digits: whole bins above it are
// kept, the bin in which the count is reached is looked at again.  Then every warp counts what it keeps of its share, and
// writes it behind what the warps before it keep.
//
// The ranks of up to 16 384 tokens (32 768 with 1 024 threads) stay in shared memory, 32 a thread, a warp's in one stretch; longer
// accounts are read again for every pass.  What bounds it is instructions, 70 % of the slots: 64 sequences of up to 16 384 tokens, 8 heads, 2 048 of them kept, 26.6 us (21 MB,
// 0.8 TB/s); with every pass reading memory 57, with one load at a time 46, with a place for each ballot 48.
template <int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 3 : 1)
kv_choose_kernel(const __grid_constant__ ChooseParams p, BlpArgs blp) {
    constexpr int kChooseThreads = THREADS, kChooseWarps = THREADS / 32, kOwn = kChooseBins / THREADS;  // (bins of a thread)
    extern __shared__ unsigned ranks[];  // [room of a thread][thread]
    __shared__ int bins[kChooseBins];
    __shared__ int s_sum[kChooseWarps], s_above[kChooseWarps], s_equal[kChooseWarps];
    __shared__ int s_tile, s_bin, s_left, s_all;
    static_assert(kChooseHeld <= 32, "a lane for every step");
    const int tid = threadIdx.x, lane = tid & 31, wid = __shfl_sync(0xffffffffu, tid >> 5, 0);
    pdl_enter();
    const bool dynamic = blp.preempted != nullptr;
    if (tid == 0) trace_begin(blp);
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
        const int s = tile / p.account.kv_heads, head = tile - s * p.account.kv_heads;
        int context = p.context[s];
        const int slot = lm_slot(p.account, s, p.error);
        if (context < 0 || context > kMostContext || context > p.account.ld) {
            if (tid == 0) lm_fail(p.error, LM_BAD_SPAN, s);
            context = 0;
        }
        if (slot < 0) context = 0;
        const int count = min(context, p.keep);
        int *const out = p.kept + ((long long)s * p.account.kv_heads + head) * p.kept_ld;
        if (head == 0 && tid == 0) p.counts[s] = count;
        if (context <= p.keep) {
            for (int j = tid; j < count; j += kChooseThreads) out[j] = j;
            continue;
        }
        for (int j = tid; j < p.first; j += kChooseThreads) out[j] = j;
        for (int j = tid; j < p.last; j += kChooseThreads) out[count - p.last + j] = context - p.last + j;
        // `need` of the `most` weights between them, one at least fewer than there are
        const int most = context - p.first - p.last, need = count - p.first - p.last;
        if (need == 0) continue;
        const float *const weights = p.account.weights + ((long long)slot * p.account.kv_heads + head) * p.account.ld + p.first;
        // chunks of even length; a warp has `a_warp` weights of one, a multiple of 32, from `begin`
        const int chunks = (most - 1) / p.chunk + 1;
        const int a_warp = (((most - 1) / chunks + 1 + kChooseThreads - 1) / kChooseThreads) * 32;
        const int begin = wid * a_warp + lane;
        unsigned *const mine = ranks + tid;
        const int held = a_warp / 32;  // ranks of a thread; places at or past `most` have the rank 0, which no weight has (it would be a NaN's)
        auto load = [&](int chunk, auto &&f) {
            const unsigned from = (unsigned)chunk * a_warp * kChooseWarps + begin;  // (the places behind the last may pass 31 bits)
            for (int e0 = 0; e0 < held; e0 += kChooseBatch) {
                float w[kChooseBatch];
#pragma unroll
                for (int j = 0; j < kChooseBatch; ++j) w[j] = e0 + j < held && from + 32 * (e0 + j) < (unsigned)most ? __ldg(weights + from + 32 * (e0 + j)) : 0.f;
#pragma unroll
                for (int j = 0; j < kChooseBatch; ++j) {
                    if (e0 + j >= held) break;
                    const unsigned r = from + 32 * (e0 + j) < (unsigned)most ? rank_of(w[j]) : 0;
                    mine[(e0 + j) * kChooseThreads] = r;
                    f(r);
                }
            }
        };
        unsigned prefix = 0, mask = 0;  // of the ranks that are still looked at
        int left = need;
        bool all = false;
        for (int digit = 0; digit < 3 && !all; ++digit) {
            const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
            const unsigned of = digit == 2 ? 1023u : 2047u;
#pragma unroll
            for (int j = 0; j < kOwn; ++j) bins[tid + j * kChooseThreads] = 0;
            __syncthreads();
            for (int chunk = 0; chunk < chunks; ++chunk) {
                auto count = [&](unsigned r) {
                    if ((r & mask) == prefix && r != 0) atomicAdd(&bins[r >> shift & of], 1);
                };
                if (digit == 0 || chunks > 1) {
                    load(chunk, count);
                } else {
#pragma unroll 8
                    for (int e = 0; e < held; ++e) count(mine[e * kChooseThreads]);
                }
            }
            __syncthreads();
            // the bin in which `left` is reached, from above: a thread has two bins or four, thread 0 the highest
            int own[kOwn], sum = 0;
#pragma unroll
            for (int j = 0; j < kOwn; ++j) own[j] = bins[kChooseBins - 1 - (kOwn * tid + j)], sum += own[j];
            int upto = sum;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += up;
            }
            if (lane == 31) s_sum[wid] = upto;
            __syncthreads();
            const int others = lane < wid ? s_sum[lane] : 0;
            upto += __reduce_add_sync(0xffffffffu, others);
            int before = upto - sum;
            if (before < left && upto >= left) {
#pragma unroll
                for (int j = 0; j < kOwn; ++j) {
                    if (before < left && before + own[j] >= left) {
                        s_bin = kChooseBins - 1 - (kOwn * tid + j), s_left = left - before, s_all = own[j] == left - before;
                    }
                    before += own[j];
                }
            }
            __syncthreads();
            prefix |= (unsigned)s_bin << shift, mask |= of << shift;
            left = s_left, all = s_all;
        }
        // kept: ranks above the prefix's, and of those that have it the first `left` (all of them, if their number is that)
        int at_all = p.first, met_all = 0;  // places filled and ranks of the prefix met in the chunks before
        for (int chunk = 0; chunk < chunks; ++chunk) {
            if (chunks > 1) load(chunk, [](unsigned) {});
            // lane e learns which of the warp's 32 ranks of step e are above, and which have the prefix
            unsigned above = 0, equal = 0;
#pragma unroll 8
            for (int e = 0; e < held; ++e) {
                const unsigned r = mine[e * kChooseThreads];
                const unsigned more = __ballot_sync(0xffffffffu, (r & mask) > prefix), same = __ballot_sync(0xffffffffu, (r & mask) == prefix && r != 0);
                if (lane == e) above = more, equal = same;
            }
            int above_to = __popc(above), equal_to = __popc(equal);
            const int own_above = above_to, own_equal = equal_to;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int a = __shfl_up_sync(0xffffffffu, above_to, d), b = __shfl_up_sync(0xffffffffu, equal_to, d);
                if (lane >= d) above_to += a, equal_to += b;
            }
            if (lane == 31) s_above[wid] = above_to, s_equal[wid] = equal_to;
            __syncthreads();
            const int theirs_above = lane < kChooseWarps ? s_above[lane] : 0, theirs_equal = lane < kChooseWarps ? s_equal[lane] : 0;
            const int before_above = __reduce_add_sync(0xffffffffu, lane < wid ? theirs_above : 0);
            int met = met_all + __reduce_add_sync(0xffffffffu, lane < wid ? theirs_equal : 0) + equal_to - own_equal;
            int at = at_all - min(met_all, left) + before_above + above_to - own_above + min(met, left);
            const int met_next = met_all + __reduce_add_sync(0xffffffffu, theirs_equal);
            at_all += __reduce_add_sync(0xffffffffu, theirs_above) + min(met_next, left) - min(met_all, left);
            met_all = met_next;
            // of those that have the prefix, the first ones up to `left`
            unsigned takes = equal;
            for (int drop = own_equal - max(0, left - met); drop > 0; --drop) takes &= ~(0x80000000u >> __clz(takes));
            takes |= above;
            const unsigned from = p.first + (unsigned)chunk * a_warp * kChooseWarps + (begin - lane) + 32 * lane;
            for (; takes; takes &= takes - 1) out[at++] = (int)(from + __ffs(takes) - 1);
            __syncthreads();  // the sums are rewritten
        }
    }
    if (tid == 0) trace_end(blp, iter);
}

// ---- moving ---------------------------------------------------------------------------------------

struct MoveParams {
    LmBatch batch;
    LmAccount account, to_account;  // (weights NULL: none)
    const unsigned char *k_codes, *v_codes;
    const float *k_scale, *v_scale;
    int pages, page_shift;
    unsigned char *to_k, *to_v;
    float *to_k_scale, *to_v_scale;
    int to_pages, to_shift, kv_heads;
    const int *to_table, *kept, *counts;
    long long kept_ld;
    int to_ld;
    int *error;
};

constexpr int kMoveThreads = 256;

__device__ __forceinline__ unsigned f16x2_to_e4m3x2(unsigned halves) {
    unsigned short d;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(d) : "r"(halves));
    return d;
}
// The largest magnitude of sixteen codes, NaN aside (a maximum takes the other of two).
__device__ __forceinline__ float most16(const uint4 &w) {
    auto of = [](unsigned c) {
        const unsigned lo = e4m3x2_to_f16x2((unsigned short)c), hi = e4m3x2_to_f16x2((unsigned short)(c >> 16));
        return __hmax2(__habs2(*reinterpret_cast<const __half2 *>(&lo)), __habs2(*reinterpret_cast<const __half2 *>(&hi)));
    };
    const __half2 m = __hmax2(__hmax2(of(w.x), of(w.y)), __hmax2(of(w.z), of(w.w)));
    const float a = __low2float(m), b = __high2float(m);
    return fmaxf(fmaxf(a, b), 0.f);
}
// Codes of one scale as codes of another, a power of two.  Where the first is one too and they are not very far apart, in halves: a
// code times 2^-20 and more is exact there, or far below half of the smallest code.
__device__ __forceinline__ uint4 again16(const uint4 &w, float scale, float target) {
    if (scale == target) return w;
    uint4 to;
    const float inv = __uint_as_float(0x7f000000u - __float_as_uint(target));  // its reciprocal (a power of two, 2^-126 to 2^121)
    const float ratio = scale * inv;
    auto each = [&](auto &&f) { to = make_uint4(f(w.x), f(w.y), f(w.z), f(w.w)); };
    if ((__float_as_uint(scale) & 0x7fffffu) == 0 && ratio >= 9.5367431640625e-7f && ratio <= 32768.f) {
        const __half2 r = __float2half2_rn(ratio);
        each([&](unsigned c) {
            const unsigned lo = e4m3x2_to_f16x2((unsigned short)c), hi = e4m3x2_to_f16x2((unsigned short)(c >> 16));
            const __half2 a = __hmul2(*reinterpret_cast<const __half2 *>(&lo), r), b = __hmul2(*reinterpret_cast<const __half2 *>(&hi), r);
            return f16x2_to_e4m3x2(*reinterpret_cast<const unsigned *>(&a)) | f16x2_to_e4m3x2(*reinterpret_cast<const unsigned *>(&b)) << 16;
        });
    } else {
        each([&](unsigned c) {
            const unsigned lo = e4m3x2_to_f16x2((unsigned short)c), hi = e4m3x2_to_f16x2((unsigned short)(c >> 16));
            const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&lo)), b = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
            return e4m3x2(a.x * scale * inv, a.y * scale * inv) | e4m3x2(b.x * scale * inv, b.y * scale * inv) << 16;
        });
    }
    return to;
}

__device__ __forceinline__ int move_count(const MoveParams &p, int s) {
    const int count = p.counts[s], context = p.batch.context[s];
    const bool fine = count >= 0 && count <= p.kept_ld && count <= (long long)p.to_ld << p.to_shift && context >= 0 && context <= kMostContext &&
                      context <= (long long)p.batch.table_ld << p.page_shift &&
                      (!p.account.weights || (context <= p.account.ld && count <= p.to_account.ld));
    if (!fine) {
        lm_fail(p.error, LM_BAD_SPAN, s);
        return 0;
    }
    if (p.account.weights && (lm_slot(p.account, s, p.error) < 0 || lm_slot(p.to_account, s, p.error) < 0)) return 0;
    return count;
}

__device__ __forceinline__ void copy_async16(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
template <int N>
__device__ __forceinline__ void copy_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A tile is one page of a head that is written: its tokens are gathered, the largest of them gives the page's scale, and the codes
// wait for it in shared memory, each thread's for itself.  Bound by memory: 2 D bytes read and as many written a token and head.  A token is
// three reads one behind the other (its number, its page, its codes), each some two microseconds on a loaded GPU: the codes of the tile to
// come are on their way while those of this one are rounded.
//
// 64 sequences, 2 048 tokens of each at most, 8 heads of 128, to pages of 32: 144 us (541 MB, 3.8 TB/s), 122 where what is kept lies
// together: rows of 128 bytes from anywhere are what memory has to do.  Pages of 16 take 134, of 128 173.  A thread for every piece took
// 158, look-ups two tiles ahead 165 (registers), magnitudes byte by byte 217.
template <int D, int PASSES>
__global__ void __launch_bounds__(kMoveThreads, 4)
kv_move_kernel(const __grid_constant__ MoveParams p, BlpArgs blp) {
    constexpr int kLanes = D / 16;
    extern __shared__ uint4 held[];  // [2][PASSES][2][threads]: codes of keys and of values; sums over the sequences [seqs + 1]
    __shared__ unsigned s_most[2][2];
    __shared__ int s_tile[kClaimSlots];
    const int tid = threadIdx.x, i = tid % kLanes, r0 = tid / kLanes, rows = blockDim.x / kLanes;
    int *const prefix = reinterpret_cast<int *>(held + 4 * PASSES * blockDim.x);
    pdl_enter();
    const bool dynamic = blp.preempted != nullptr;
    if (tid == 0) trace_begin(blp);
    if (tid < 4) s_most[tid >> 1][tid & 1] = 0;
    const int page_tokens = 1 << p.page_shift, to_tokens = 1 << p.to_shift;
    blp.total_tiles = lm_prefix(prefix, p.batch.seqs, p.error, [&](int s) {
        const long long all = (((long long)move_count(p, s) + to_tokens - 1) >> p.to_shift) * p.kv_heads;
        return all > 0x7fffffff ? 0x7fffffff : (int)all;
    });
    const float a_head = 1.0f / (float)p.kv_heads;
    struct Place {
        int s, index, head, some;  // page `index` of a head of sequence s gets so many tokens
        int token[PASSES];         // this thread's rows: tokens of the source (-1: none)
        float ks[PASSES], vs[PASSES];
        bool fine;
    };
    int at_seq = 0;  // (tiles come in ascending order: often the sequence of the one before, or the next)
    // where a tile's tokens come from; their codes are asked for
    auto find = [&](int tile, int buffer) {
        Place a;
        a.some = 0, a.fine = tile >= 0;
#pragma unroll
        for (int x = 0; x < PASSES; ++x) a.token[x] = -1;
        if (tile < 0) return a;
        if (prefix[at_seq + 1] <= tile && prefix[++at_seq + 1] <= tile) at_seq = lm_find(prefix, p.batch.seqs, tile);
        a.s = at_seq;
        const int within = tile - prefix[a.s];
        a.index = within < 1 << 24 ? sm100::fast_div(within, p.kv_heads, a_head) : within / p.kv_heads;
        a.head = within - a.index * p.kv_heads;
        const int begin = a.index << p.to_shift, context = p.batch.context[a.s];
        a.some = min(p.counts[a.s] - begin, to_tokens);
        const int *const kept = p.kept + ((long long)a.s * p.kv_heads + a.head) * p.kept_ld + begin;
#pragma unroll
        for (int x = 0; x < PASSES; ++x)
            if (r0 + x * rows < a.some) {
                a.token[x] = kept[r0 + x * rows];
                if ((unsigned)a.token[x] >= (unsigned)context) {
                    lm_fail(p.error, LM_BAD_PLACE, a.s);
                    a.fine = false, a.token[x] = -1;
                }
            }
        int page[PASSES];
#pragma unroll
        for (int x = 0; x < PASSES; ++x)
            if (a.token[x] >= 0) page[x] = p.batch.table[(size_t)a.s * p.batch.table_ld + (a.token[x] >> p.page_shift)];
#pragma unroll
        for (int x = 0; x < PASSES; ++x) {
            if (a.token[x] < 0) continue;
            if ((unsigned)page[x] >= (unsigned)p.pages) {
                lm_fail(p.error, LM_BAD_PAGE, a.s);
                a.fine = false, a.token[x] = -1;
                continue;
            }
            const size_t block = (size_t)page[x] * p.kv_heads + a.head;
            const size_t at = ((block << p.page_shift) + (a.token[x] & (page_tokens - 1))) * D + 16 * i;
            uint4 *const to = held + ((buffer * PASSES + x) * 2) * blockDim.x + tid;
            copy_async16(sm100::smem_u32(to), p.k_codes + at), copy_async16(sm100::smem_u32(to + blockDim.x), p.v_codes + at);
            a.ks[x] = __ldg(p.k_scale + block), a.vs[x] = __ldg(p.v_scale + block);
        }
        return a;
    };
    int iter = 0, tile;
    auto claim = [&](int at) {
        if (!dynamic) return blp_claim(blp, at);
        if (tid == 0) s_tile[claim_slot(at)] = blp_claim(blp, at);
        __syncthreads();
        return s_tile[claim_slot(at)];
    };
    tile = claim(0);
    Place now = find(tile, 0);
    asm volatile("cp.async.commit_group;" ::: "memory");
    __syncthreads();  // the magnitudes are set
    for (; tile >= 0; ++iter) {
        const int to = p.to_table[(size_t)now.s * p.to_ld + now.index];
        const uint4 *const codes = held + (iter & 1) * 2 * PASSES * blockDim.x + tid;
        const int next_tile = claim(iter + 1);
        const Place next = find(next_tile, (iter + 1) & 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        copy_async_wait<1>();  // (a thread reads what it has copied itself)
        bool fine = now.fine;
        if ((unsigned)to >= (unsigned)p.to_pages) {
            lm_fail(p.error, LM_BAD_PAGE, now.s);
            fine = false;
        }
        float most_k = 0.f, most_v = 0.f;
#pragma unroll
        for (int x = 0; x < PASSES; ++x)
            if (now.token[x] >= 0) {
                most_k = fmaxf(most_k, most16(codes[2 * x * blockDim.x]) * now.ks[x]);
                most_v = fmaxf(most_v, most16(codes[(2 * x + 1) * blockDim.x]) * now.vs[x]);
            }
        const unsigned mk = __reduce_max_sync(0xffffffffu, __float_as_uint(most_k)), mv = __reduce_max_sync(0xffffffffu, __float_as_uint(most_v));
        unsigned *const most = s_most[iter & 1];
        if ((tid & 31) == 0) atomicMax(&most[0], mk), atomicMax(&most[1], mv);
        fine = __syncthreads_and(fine);
        const float scale_k = lm_scale_for(most[0]), scale_v = lm_scale_for(most[1]);
        if (fine) {
            const size_t block = (size_t)to * p.kv_heads + now.head;
            unsigned char *const to_k = p.to_k + (block << p.to_shift) * D, *const to_v = p.to_v + (block << p.to_shift) * D;
#pragma unroll
            for (int x = 0; x < PASSES; ++x) {
                if (now.token[x] < 0) continue;
                const int at = (r0 + x * rows) * D + 16 * i;
                *reinterpret_cast<uint4 *>(to_k + at) = again16(codes[2 * x * blockDim.x], now.ks[x], scale_k);
                *reinterpret_cast<uint4 *>(to_v + at) = again16(codes[(2 * x + 1) * blockDim.x], now.vs[x], scale_v);
            }
            if (tid == 0) p.to_k_scale[block] = scale_k, p.to_v_scale[block] = scale_v;
            if (p.account.weights) {
                const int s = now.s, slot = p.account.slots ? p.account.slots[s] : s, to_slot = p.to_account.slots ? p.to_account.slots[s] : s;
                const float *const from = p.account.weights + ((long long)slot * p.kv_heads + now.head) * p.account.ld;
                float *const into = p.to_account.weights + ((long long)to_slot * p.kv_heads + now.head) * p.to_account.ld + (now.index << p.to_shift);
#pragma unroll
                for (int x = 0; x < PASSES; ++x)
                    if (i == 0 && now.token[x] >= 0) into[r0 + x * rows] = __ldg(from + now.token[x]);
                if (now.index == 0 && now.head == 0) lm_slot_twice(p.to_account, s, tid, blockDim.x, p.error);
            }
        }
        // (the other pair of magnitudes was read before the barrier of this tile, this one is after that of the next)
        if (tid < 2) s_most[(iter + 1) & 1][tid] = 0;
        __syncthreads();
        tile = next_tile, now = next;
    }
    if (tid == 0) trace_end(blp, iter);
}

}  // namespace gpx

using namespace gpx;

extern "C" {

int gpx_kv_choose(const gpx_kv_batch *batch, const gpx_kv_weights *account, const gpx_kv_choose_args *args, void *ctx, const gpx_blp *blp,
                  gpx_stream stream) {
    GPX_REQUIRE(args && ctx, GPX_FAIL, "args or ctx is NULL");
    GPX_REQUIRE((uintptr_t)ctx % 256 == 0, GPX_FAIL, "ctx must be 256-byte aligned");
    const gpx_kv_choose_args &a = *args;
    LmBatch b;
    ChooseParams p{};
    BlpArgs blp_args;
    GPX_TRY(lm_check_batch(batch, &b));
    GPX_TRY(lm_check_account(account, b, &p.account));
    GPX_TRY(lm_check_blp(blp, &blp_args));
    GPX_REQUIRE(a.kept && a.counts && (uintptr_t)a.kept % 4 == 0 && (uintptr_t)a.counts % 4 == 0, GPX_FAIL,
                "kept or counts is NULL or not 4-byte aligned");
    GPX_REQUIRE(a.keep > 0 && a.first >= 0 && a.last >= 0 && (long long)a.first + a.last <= a.keep, GPX_OUT_OF_RANGE,
                "keep is %d, of which the first %d and the last %d", a.keep, a.first, a.last);
    p.kept_ld = a.kept_ld ? a.kept_ld : a.keep;
    GPX_REQUIRE(p.kept_ld >= a.keep && p.kept_ld <= kMostKept, GPX_OUT_OF_RANGE, "a head keeps %d tokens, the next one's are %lld on", a.keep, p.kept_ld);
    GPX_REQUIRE((long long)b.seqs * p.account.kv_heads <= 0x7fffffff, GPX_OUT_OF_RANGE, "too many heads");
    const DeviceInfo &d = device_info();
    GPX_REQUIRE(d.device >= 0, GPX_FAIL, "gpx_init was not called");
    p.context = b.context, p.kept = (int *)a.kept, p.counts = (int *)a.counts;
    p.keep = a.keep, p.first = a.first, p.last = a.last, p.error = lm_ctx(ctx).error;
    blp_args.total_tiles = b.seqs * p.account.kv_heads;
    auto launch = [&](auto kernel, int threads) {
        p.chunk = (int)std::min<long long>((p.account.ld + threads - 1) / threads, kChooseHeld) * threads;
        const size_t smem = p.chunk * sizeof(unsigned);
        int per_sm;
        const cudaError_t e = lm_resident((const void *)kernel, threads, smem, kChooseHeld * threads * sizeof(unsigned), d.device, &per_sm);
        if (e != cudaSuccess) return e;
        // (accounts are of any length: without a word a CTA for each lets the next one begin where one has ended, 25 us against 33)
        const int grid = blp_args.preempted ? (int)std::min<long long>(blp_args.total_tiles, (long long)d.sm_count * per_sm) : blp_args.total_tiles;
        return launch_layer(kernel, grid, threads, smem, as_stream(stream), p, blp_args);
    };
    // Accounts that may be long and do not fill the SMs anyway have twice as many threads each.  With 1 024 and with 512, 8 heads: 16
    // sequences of up to 32 000 tokens 19.1 and 38.7 us, 4 of up to 40 000 38.8 and 48.8, one of 131 072 100 and 136.  (The host knows what
    // accounts have room for, not how long they are: short ones in long accounts take 0.7 us more, 5.9 and 5.2 for one of 517 tokens, 8.3 and 7.6
    // for 16 of 4 000; 16 of 12 000 take 11.5 and 12.3.)
    const bool wide = p.account.ld > 512 * kChooseHeld && blp_args.total_tiles <= d.sm_count;
    GPX_CUDA(wide ? launch(kv_choose_kernel<1024>, 1024) : launch(kv_choose_kernel<512>, 512));
    return GPX_SUCC;
}

int gpx_kv_move(const gpx_kv_cache *from, const gpx_kv_batch *batch, const gpx_kv_cache *to, const gpx_kv_move_args *args,
                const gpx_kv_weights *account, const gpx_kv_weights *to_account, void *ctx, const gpx_blp *blp, gpx_stream stream) {
    GPX_REQUIRE(from && to && args && ctx, GPX_FAIL, "a cache, args or ctx is NULL");
    GPX_REQUIRE((uintptr_t)ctx % 256 == 0, GPX_FAIL, "ctx must be 256-byte aligned");
    const gpx_kv_move_args &a = *args;
    MoveParams p{};
    BlpArgs b;
    GPX_TRY(lm_check_batch(batch, &p.batch));
    GPX_TRY(lm_check_blp(blp, &b));
    GPX_REQUIRE(from->kv_heads == to->kv_heads && from->dim == to->dim, GPX_OUT_OF_RANGE, "caches of %d heads of %d and %d of %d", from->kv_heads,
                from->dim, to->kv_heads, to->dim);
    GPX_REQUIRE(a.to_table && a.kept && a.counts && ((uintptr_t)a.to_table | (uintptr_t)a.kept | (uintptr_t)a.counts) % 4 == 0, GPX_FAIL,
                "to_table, kept or counts is NULL or not 4-byte aligned");
    GPX_REQUIRE(a.to_ld > 0 && a.kept_ld > 0 && a.kept_ld <= kMostKept, GPX_OUT_OF_RANGE, "to_ld is %d, kept_ld %lld", a.to_ld, a.kept_ld);
    GPX_REQUIRE(!account == !to_account, GPX_FAIL, "one of the accounts is NULL");
    if (account) {
        GPX_TRY(lm_check_account(account, p.batch, &p.account));
        GPX_TRY(lm_check_account(to_account, p.batch, &p.to_account));
        GPX_REQUIRE(p.account.kv_heads == from->kv_heads && p.to_account.kv_heads == from->kv_heads, GPX_OUT_OF_RANGE,
                    "accounts of %d and %d heads for a cache of %d", p.account.kv_heads, p.to_account.kv_heads, from->kv_heads);
        GPX_REQUIRE(p.account.weights != p.to_account.weights, GPX_FAIL, "weights cannot be moved in place");
    }
    const DeviceInfo &d = device_info();
    GPX_REQUIRE(d.device >= 0, GPX_FAIL, "gpx_init was not called");
    p.k_codes = from->k, p.v_codes = from->v, p.k_scale = from->k_scale, p.v_scale = from->v_scale;
    p.pages = from->pages, p.page_shift = __builtin_ctz((unsigned)from->page_tokens), p.kv_heads = from->kv_heads;
    p.to_k = to->k, p.to_v = to->v, p.to_k_scale = to->k_scale, p.to_v_scale = to->v_scale;
    p.to_pages = to->pages, p.to_shift = __builtin_ctz((unsigned)to->page_tokens);
    p.to_table = (const int *)a.to_table, p.kept = (const int *)a.kept, p.counts = (const int *)a.counts;
    p.kept_ld = a.kept_ld, p.to_ld = a.to_ld, p.error = lm_ctx(ctx).error;
    // a page of a head is so many pieces of sixteen codes, four to a thread where that leaves two warps
    const int pieces = to->page_tokens * (to->dim / 16), threads = std::max(64, pieces / 4);
    const size_t codes = (size_t)pieces * 4 * 16, smem = codes + lm_prefix_bytes(p.batch.seqs);
    const size_t most = kMostPageTokens * 128 / 16 * 4 * 16 + lm_prefix_bytes(kLmMaxSeqs);
    const long long tiles = (long long)p.batch.seqs * std::min<long long>(a.to_ld, (a.kept_ld + to->page_tokens - 1) / to->page_tokens) * to->kv_heads;
    auto launch = [&](auto kernel) {
        int per_sm;
        const cudaError_t e = lm_resident((const void *)kernel, threads, smem, most, d.device, &per_sm);
        if (e != cudaSuccess) return e;
        return launch_layer(kernel, (int)std::min<long long>(tiles, (long long)d.sm_count * per_sm), threads, smem, as_stream(stream), p, b);
    };
    auto by_pieces = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        return pieces == threads ? launch(kv_move_kernel<D, 1>) : pieces == 2 * threads ? launch(kv_move_kernel<D, 2>) : launch(kv_move_kernel<D, 4>);
    };
    GPX_CUDA(to->dim == 64 ? by_pieces(std::integral_constant<int, 64>()) : by_pieces(std::integral_constant<int, 128>()));
    return GPX_SUCC;
}

}  // extern "C"
