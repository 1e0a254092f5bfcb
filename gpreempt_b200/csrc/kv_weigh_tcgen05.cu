// What each key has weighed, for many rows a head of keys (prompts and their chunks), on the tcgen05 tensor cores.  The formula is that
// of kv_weigh.cu.
//
// A tile is 128 keys of a head; they stay in shared memory as 16-bit numbers of the queries' type (every e4m3 number is one), the M side
// of the products S^T = K Q^T, and the rows that see some of them go past in chunks of 64, as they are.  Four warps copy the queries of
// chunks ahead and one of them issues the products; four others fetch the keys and then take the scores out of tensor memory, a thread a
// key, so that the sum over a key's rows stays in its thread, and the normalisers of the rows are the same for a warp.  Queries and scores
// have four buffers, and two CTAs share an SM.
//
// What should bound it is the special-function unit, sixteen exponentials a cycle and SM: 512 cycles a chunk, against 128 of the products.
// A chunk takes 1 100 cycles an SM, with two warps of keys and two of rows on a scheduler, and the start and end of a tile 5 us, of which
// the other CTA hides a part.  Four prompts' last 256 of 1 024 tokens over 8 192 keys at most, 32 heads of 128 on 8: 119 us (345 TFLOP/s, 1.3
// T exponentials/s), 324 with the kernel for few rows.  Taken back: queries turned into halves by every tile, 495 us; one CTA an SM, 184;
// chunks of 128 rows in two buffers, 132, and 74 us instead of 54 for tiles of one chunk.
//
// Where a preemptible launch stops between two chunks, the sums of the tile under way go to the context, and the next launch goes on with
// them.
#include "act_layout.h"
#include "kv_weigh.h"
#include "planes.cuh"
#include "sm100.cuh"

#include <algorithm>

namespace gpx {

using namespace sm100;

constexpr int kManyThreads = 256;  // four warps of keys, four of rows
constexpr int kManyKeys = 128, kChunkRows = 64;
constexpr int kSlots = 4, kLag = 2;  // buffers of queries and scores; chunks whose copies are under way when one is multiplied
constexpr int kManyNotes = 1024;   // the last counters of the context: {tile + 1, next chunk} of a CTA's unfinished tile
constexpr unsigned long long kManyWaitNs = 2000000000ull;

template <int D>
struct WeighCfg {
    static constexpr uint32_t kKeys = kManyKeys * D * 2, kQueries = kChunkRows * D * 2;  // bytes
    static constexpr uint32_t kCtlAt = kKeys + kSlots * kQueries;
};
struct WeighCtl {
    unsigned long long q_full[kSlots], s_full[kSlots], s_empty[kSlots], k_full;
    alignas(16) float lse[kSlots][kChunkRows];                     // a row's normaliser
    alignas(16) int lo[kSlots][kChunkRows], hi[kSlots][kChunkRows];  // the keys it sees
    float scale[kManyKeys];
    int no_page[kManyKeys];
    uint32_t tmem;
    int tile, resume, more[kSlots], abort_flag;
};

__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 of_pair(uint64_t p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

template <int D, bool HALF>
__global__ void __launch_bounds__(kManyThreads, 2)
kv_weigh_many_kernel(const __grid_constant__ WeighParams p, BlpArgs blp) {
    using Cfg = WeighCfg<D>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    WeighCtl *ctl = reinterpret_cast<WeighCtl *>(smem + Cfg::kCtlAt);
    int *const prefix = reinterpret_cast<int *>(ctl + 1);  // [seqs + 1]
    volatile int *abort_flag = &ctl->abort_flag;
    const uint32_t keys_at = smem_u32(smem), queries_at = keys_at + Cfg::kKeys;
    const int tid = threadIdx.x, lane = tid & 31, wid = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const bool elected = elect_one();
    if (tid == 0) {
        for (int i = 0; i < kSlots; ++i) mbar_init(smem_u32(&ctl->q_full[i]), 4), mbar_init(smem_u32(&ctl->s_full[i]), 1), mbar_init(smem_u32(&ctl->s_empty[i]), 4);
        mbar_init(smem_u32(&ctl->k_full), 4);
        ctl->abort_flag = 0;
        fence_barrier_init();
        fence_proxy_async();
    }
    if (wid == 4) tmem_alloc(smem_u32(&ctl->tmem), 256);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    pdl_enter();
    const bool dynamic = blp.preempted != nullptr;
    if (tid == 0) trace_begin(blp);
    const uint32_t tmem = ctl->tmem;
    const int group = p.heads / p.kv_heads, page_tokens = 1 << p.page_shift;
    auto wait = [&](unsigned long long *bar, uint32_t phase) {
        if (!mbar_wait(smem_u32(bar), phase, abort_flag, kManyWaitNs)) {
            *abort_flag = 1;
            lm_fail(p.error, LM_GAVE_UP, (int)blockIdx.x);
        }
    };
    blp.total_tiles = lm_prefix(prefix, p.batch.seqs, p.error, [&](int s) {
        const LmSpan span = weigh_span(p, s);
        const long long all = span.n ? (long long)p.kv_heads * ((span.context + kManyKeys - 1) / kManyKeys) : 0;
        return all > 0x7fffffff ? 0x7fffffff : (int)all;
    });
    int *const note = p.counters + kLmCounters - kManyNotes + 2 * blockIdx.x;
    float4 *const left = reinterpret_cast<float4 *>(p.parts) + (size_t)blockIdx.x * kManyKeys;
    int pending = dynamic && tid == 0 ? note[0] - 1 : -1;
    int n = 0, n_keys = 0;  // chunks so far, and tiles of keys
    int rounds = 0;
    for (int iter = 0;; ++rounds) {
        if (tid == 0) {
            int tile = -1, resume = -1;
            if (*abort_flag) {
            } else if (pending >= 0) {
                if (load_word(blp.preempted) != 0) {  // (the note stays)
                    if (blp.trace) atomicMin(blp.trace + 2, globaltimer_ns());
                    atomicCAS(blp.stop_index, -1, blp.kernel_id);
                } else {
                    tile = pending, resume = note[1];
                    note[0] = note[1] = 0;  // (other kernels' counters and notes are the same words: a note that is taken leaves none behind)
                }
                pending = -1;
            } else {
                tile = blp_claim(blp, iter++);
            }
            ctl->tile = tile, ctl->resume = resume;
        }
        __syncthreads();
        const int tile = ctl->tile, resume = ctl->resume;
        if (tile < 0) break;
        const int s = lm_find(prefix, p.batch.seqs, tile);
        const int first = p.batch.first[s], new_tokens = p.batch.first[s + 1] - first, context = p.batch.context[s];
        const int unit_blocks = (context + kManyKeys - 1) / kManyKeys, within = tile - prefix[s];
        const int head = within / unit_blocks, key0 = (within - head * unit_blocks) * kManyKeys;
        const int votes = p.observed ? min(new_tokens, p.observed) : new_tokens, rows = votes * group, pos0 = context - votes;
        const int slot_row = p.account.slots ? p.account.slots[s] : s;
        float *const account = p.account.weights + ((long long)slot_row * p.kv_heads + head) * p.account.ld;
        const int fresh = p.causal ? max(0, context - new_tokens) : context;  // keys from here on begin their account
        auto upto = [&](int pos) { return p.causal ? min(context, max(pos + 1, 0)) : context; };
        auto from = [&](int pos) { return p.window && pos >= p.window ? pos - p.window + 1 : 0; };
        // the chunks of rows that see some of these keys
        int row_lo = 0, row_hi = rows;
        if (p.causal) {
            row_lo = (int)min((long long)max(key0 - pos0, 0) * group, (long long)rows);
            if (p.window) row_hi = (int)max(0ll, min(((long long)key0 + kManyKeys - 1 + p.window - pos0) * group, (long long)rows));
        }
        const int chunk_lo = row_lo / kChunkRows, chunk_hi = row_lo < row_hi ? (row_hi + kChunkRows - 1) / kChunkRows : chunk_lo;
        const int begin = resume >= 0 ? resume : chunk_lo;
        const int my_key = key0 + tid;  // (of the threads of keys)
        float old = 0.f;
        if (wid < 4 && my_key < fresh) old = account[my_key];
        int next = begin;  // the chunk to go on with
        if (wid >= 4) {
            // ---- rows: queries, products
            using Rows = WarpRows<D>;
            constexpr uint32_t idesc = HALF ? make_idesc_f16_f32(kManyKeys, kChunkRows) : make_idesc_bf16_f32(kManyKeys, kChunkRows);
            constexpr int kWarpRows = kChunkRows / 4, kRowsAtOnce = 32 / Rows::kLanes;
            int asked = next, n_asked = n;
            bool more = next < chunk_hi;
            // (a warp has sixteen rows of a chunk, of which its lanes take two or four at a time; a row of lanes walks on from chunk to chunk)
            constexpr int kRows = kWarpRows / kRowsAtOnce;
            const int piece = lane % Rows::kLanes, r0 = (wid & 3) * kWarpRows + lane / Rows::kLanes * kRows;
            const uint32_t to0 = queries_at + (piece >> 3) * (kChunkRows * 128) + r0 * 128;
            uint32_t swizzle[kRows];
#pragma unroll
            for (int i = 0; i < kRows; ++i) swizzle[i] = i * 128 + (((piece ^ (r0 + i)) & 7) << 4);
            struct Row {
                int token, of_group;
            };
            auto row_of = [&](int row) { return Row{row / group, row % group}; };
            const int step_tokens = kChunkRows / group, step_heads = kChunkRows % group;
            auto step = [&](Row &r) {
                r.token += step_tokens, r.of_group += step_heads;
                if (r.of_group >= group) r.of_group -= group, ++r.token;
            };
            const int r_lse = (wid & 3) * kWarpRows + lane;  // (of lanes that have one)
            Row own = row_of(asked * kChunkRows + r0), own_lse = row_of(asked * kChunkRows + r_lse);
            const long long token0 = first + new_tokens - votes;
            while (more) {
                if (asked < chunk_hi) {
                    const int slot = n_asked % kSlots;
                    wait(&ctl->s_empty[slot], (n_asked / kSlots & 1) ^ 1);
                    const uint32_t to = to0 + slot * Cfg::kQueries;
                    const unsigned short *q = p.q + (token0 + own.token) * p.q_ld + (head * group + own.of_group) * D + 8 * piece;
                    int of_group = own.of_group;
                    const int live = rows - asked * kChunkRows;  // (zeros behind the last row)
#pragma unroll
                    for (int i = 0; i < kRows; ++i) {
                        const bool there = r0 + i < live;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + swizzle[i]), "l"(there ? q : p.q), "r"(there ? 16 : 0) : "memory");
                        q += D;
                        if (++of_group == group) of_group = 0, q += p.q_ld - group * D;
                    }
                    step(own);
                    if (lane < kWarpRows) {
                        if (r_lse < live) {
                            const float *const lse = p.lse + (token0 + own_lse.token) * p.heads + head * group + own_lse.of_group;
                            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&ctl->lse[slot][r_lse])), "l"(lse) : "memory");
                        } else {
                            ctl->lse[slot][r_lse] = INFINITY;
                        }
                        const int pos = pos0 + own_lse.token;
                        ctl->lo[slot][r_lse] = from(pos), ctl->hi[slot][r_lse] = r_lse < live ? upto(pos) : 0;
                        step(own_lse);
                    }
                    ++n_asked;
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (++asked - next <= kLag) continue;
                // ---- the chunk whose copies have arrived
                const int slot = n % kSlots;
                if (wid == 4 && lane == 0) {
                    const int word = dynamic && (next & 3) == 3 ? load_word(blp.preempted) : 0;  // (a read of the word takes as long as a chunk)
                    if (word != 0 && blp.trace) atomicMin(blp.trace + 2, globaltimer_ns());
                    ctl->more[slot] = next + 1 < chunk_hi && word == 0 && !*abort_flag;
                }
                asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->q_full[slot]));
                __syncwarp();
                wait(&ctl->q_full[slot], n / kSlots & 1);
                if (wid == 4) {
                    if (next == begin) wait(&ctl->k_full, n_keys & 1);
                    tc_fence_after_sync();
                    if (elected) {
                        if (!*abort_flag) {
                            const uint64_t dk = make_smem_desc_sw128(keys_at), dq = make_smem_desc_sw128(queries_at + slot * Cfg::kQueries);
#pragma unroll
                            for (int k = 0; k < D / 16; ++k)
                                mma_f16_ss(tmem + slot * kChunkRows, dk + (k & 3) * 2 + (k >> 2) * (kManyKeys * 128 >> 4),
                                           dq + (k & 3) * 2 + (k >> 2) * (kChunkRows * 128 >> 4), idesc, k > 0 ? 1u : 0u);
                        }
                        mma_commit(smem_u32(&ctl->s_full[slot]));
                    }
                    __syncwarp();
                }
                more = ctl->more[slot];
                ++n, ++next;
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else {
            // ---- keys: exponentials, a thread a key
            const uint64_t log2e = pair(-1.4426950408889634f, -1.4426950408889634f);
            uint64_t sum[2] = {0, 0};
            if (resume >= 0) {
                const float4 v = left[tid];
                sum[0] = pair(v.x, v.y), sum[1] = pair(v.z, v.w);
            }
            bool no_page = false;
            float own_scale = 0.f;
            if (next < chunk_hi) {
                // ---- the keys as operand, sixteen codes at a time: neighbouring lanes have a row, a thread a piece of eight rows or four
                constexpr int kPieces = D / 16, kItems = kManyKeys * kPieces / 128;
                const int seen = from(pos0);  // the first key that a row sees
                int page[kItems];
                uint4 codes[kItems];
                float scales[kItems];
#pragma unroll
                for (int i = 0; i < kItems; ++i) {
                    const int key = key0 + (tid + 128 * i) / kPieces;
                    // (what ends below the keys that are seen may be anybody's by now: its page is not looked up)
                    page[i] = key < context && key >= seen ? p.batch.table[(size_t)s * p.batch.table_ld + (key >> p.page_shift)] : -1;
                }
#pragma unroll
                for (int i = 0; i < kItems; ++i) {
                    const int piece = tid % kPieces, key = key0 + (tid + 128 * i) / kPieces;
                    codes[i] = make_uint4(0, 0, 0, 0), scales[i] = 1.f;
                    if ((unsigned)page[i] < (unsigned)p.pages) {
                        const size_t block = (size_t)page[i] * p.kv_heads + head;
                        codes[i] = __ldg(reinterpret_cast<const uint4 *>(p.k_codes + ((block << p.page_shift) + (key & (page_tokens - 1))) * D) + piece);
                        if (piece == 0) scales[i] = __ldg(p.k_scale + block);
                    }
                }
#pragma unroll
                for (int i = 0; i < kItems; ++i) {
                    const int r = (tid + 128 * i) / kPieces, piece = tid % kPieces;
                    if (piece == 0) ctl->scale[r] = scales[i], ctl->no_page[r] = key0 + r < context && key0 + r >= seen && (unsigned)page[i] >= (unsigned)p.pages;
                    const uint32_t words[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
                    uint32_t h[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        h[j] = e4m3x2_to_f16x2((unsigned short)(words[j >> 1] >> 16 * (j & 1)));
                        if (!HALF) {
                            const float2 f = unpack_halves(h[j]);
                            h[j] = pack_out<false>(f.x, f.y);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int at = 2 * piece + j;  // piece of eight numbers of the row
                        st_shared_v4(keys_at + (at >> 3) * (kManyKeys * 128) + r * 128 + (((at ^ r) & 7) << 4),
                                     make_uint4(h[4 * j], h[4 * j + 1], h[4 * j + 2], h[4 * j + 3]));
                    }
                }
                fence_proxy_async();
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (lane == 0) mbar_arrive(smem_u32(&ctl->k_full));
                own_scale = -ctl->scale[tid] * p.scale, no_page = ctl->no_page[tid];
                if (no_page) lm_fail(p.error, LM_BAD_PAGE, s);
            }
            const uint64_t scale = pair(own_scale, own_scale);
            while (next < chunk_hi) {
                const int slot = n % kSlots;
                const int r0 = next * kChunkRows, r1 = min(rows, r0 + kChunkRows) - 1;
                const bool border = rows - r0 < kChunkRows || key0 + kManyKeys > upto(pos0 + r0 / group) || key0 < from(pos0 + r1 / group);
                wait(&ctl->q_full[slot], n / kSlots & 1);
                wait(&ctl->s_full[slot], n / kSlots & 1);
                tc_fence_after_sync();
                const bool more = ctl->more[slot];
                const uint32_t scores = tmem + ((uint32_t)wid << 21) + slot * kChunkRows;
                uint32_t v[2][32];
                tmem_ld_32x32(scores, v[0]);
                auto columns = [&](auto masked) {
#pragma unroll
                    for (int c = 0; c < kChunkRows / 32; ++c) {
                        tmem_ld_wait();
                        if (c + 1 < kChunkRows / 32) tmem_ld_32x32(scores + 32 * (c + 1), v[(c + 1) & 1]);
                        const uint32_t(&x)[32] = v[c & 1];
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const ulonglong2 l = *reinterpret_cast<const ulonglong2 *>(&ctl->lse[slot][32 * c + j]);
                            // (in the units of the normaliser: the difference is rounded once, however large the two are)
                            const uint64_t a = mul2(fma2(pair(__uint_as_float(x[j]), __uint_as_float(x[j + 1])), scale, l.x), log2e);
                            const uint64_t b = mul2(fma2(pair(__uint_as_float(x[j + 2]), __uint_as_float(x[j + 3])), scale, l.y), log2e);
                            const float2 ea = of_pair(a), eb = of_pair(b);
                            float e[4] = {lm_ex2(ea.x), lm_ex2(ea.y), lm_ex2(eb.x), lm_ex2(eb.y)};
                            if (decltype(masked)::value) {
                                const int4 lo = *reinterpret_cast<const int4 *>(&ctl->lo[slot][32 * c + j]), hi = *reinterpret_cast<const int4 *>(&ctl->hi[slot][32 * c + j]);
                                if (my_key < lo.x || my_key >= hi.x) e[0] = 0.f;
                                if (my_key < lo.y || my_key >= hi.y) e[1] = 0.f;
                                if (my_key < lo.z || my_key >= hi.z) e[2] = 0.f;
                                if (my_key < lo.w || my_key >= hi.w) e[3] = 0.f;
                            }
                            sum[0] = add2(sum[0], pair(e[0], e[1])), sum[1] = add2(sum[1], pair(e[2], e[3]));
                        }
                    }
                };
                if (border) columns(std::true_type());
                else columns(std::false_type());
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->s_empty[slot]));
                ++n, ++next;
                if (!more) break;
            }
            const float2 a = of_pair(sum[0]), b = of_pair(sum[1]);
            if (next < chunk_hi) {
                left[tid] = make_float4(a.x, a.y, b.x, b.y);
            } else if (my_key < context && !no_page && (chunk_lo < chunk_hi || my_key >= fresh || p.decay != 1.f)) {
                const float all = (a.x + a.y) + (b.x + b.y);
                account[my_key] = my_key < fresh ? fmaf(p.decay, old, all) : all;
            }
        }
        __syncthreads();
        if (next < chunk_hi) {
            if (tid == 0 && !*abort_flag) {
                note[0] = tile + 1, note[1] = next;
                atomicCAS(blp.stop_index, -1, blp.kernel_id);
            }
            break;
        }
        if (begin < chunk_hi) ++n_keys;
        if (head == 0 && key0 == 0) lm_slot_twice(p.account, s, tid, kManyThreads, p.error);
    }
    if (*abort_flag)
        for (int spin = 0; spin < 64; ++spin) __nanosleep(1000);  // products in flight end before the CTA does
    tc_fence_before_sync();
    __syncthreads();
    if (wid == 4) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 256);
    }
    if (tid == 0) trace_end(blp, rounds);
}

cudaError_t kv_weigh_many_launch(WeighParams &p, int dim, bool half, const DeviceInfo &d, const BlpArgs &blp, cudaStream_t s) {
    auto go = [&](auto kernel, uint32_t fixed) {
        const size_t most = 1024 + fixed + sizeof(WeighCtl) + lm_prefix_bytes(kLmMaxSeqs), smem = 1024 + fixed + sizeof(WeighCtl) + lm_prefix_bytes(p.batch.seqs);
        int per_sm;
        const cudaError_t e = lm_resident((const void *)kernel, kManyThreads, smem, most, d.device, &per_sm);
        if (e != cudaSuccess) return e;
        // (The runtime says one CTA an SM of kernels with tensor memory.  This one takes half of it, 128 registers a thread and, for up to
        // some 2 000 sequences, less than half of shared memory.)
        per_sm = 2 * (smem + 1024) <= 228 * 1024 ? 2 : 1;
        const int grid = std::min(d.sm_count * per_sm, kManyNotes / 2);
        return launch_layer(kernel, grid, kManyThreads, smem, s, p, blp);
    };
    if (dim == 64)
        return half ? go(kv_weigh_many_kernel<64, true>, WeighCfg<64>::kCtlAt) : go(kv_weigh_many_kernel<64, false>, WeighCfg<64>::kCtlAt);
    return half ? go(kv_weigh_many_kernel<128, true>, WeighCfg<128>::kCtlAt) : go(kv_weigh_many_kernel<128, false>, WeighCfg<128>::kCtlAt);
}

}  // namespace gpx
