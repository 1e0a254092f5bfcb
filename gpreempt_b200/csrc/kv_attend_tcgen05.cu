// Attention of new tokens over a paged 8-bit cache, for many rows a head of keys (prompts and their chunks), on the
// tcgen05 tensor cores.  The formula is that of kv_attend.cu.
//
// A tile is a block of 256 rows (a group's heads times the tokens) of one head of keys, against all keys they see
// or, where there are too few such blocks for all SMs, an equal part of those; the CTA that brings the last part
// joins them.  Per block of 128 keys:
//   - one warp fetches keys and values as they are in the cache (TMA), with the pages' scales,
//   - four warps turn the codes into halves (exact: every e4m3 number is a half) in the swizzled layout of the operands,
//   - the scales are left to the softmax, the values' as in kv_attend.cu: relative to the largest of the tile they join the exponents,
//   - one warp issues S = Q K^T and O += P V of the two halves of the rows in turn,
//   - two warpgroups, a thread a row, take the scores out of tensor memory, and put the probabilities back as a 16-bit A
//     operand, where the scores were.  The values lie with keys as rows; their descriptor names that MN-major.
// Queries become halves after a power of two that brings their row's largest to 1, as in kv_attend.cu.
//
// What bounds it: 256 x 128 exponentials a block are 2 048 cycles of the special-function unit, the products 2 048
// of the tensor cores, and shared memory carries 320 KB for them (2 500 cycles).  The halves of the rows are
// half a block apart, so that one's products run under the other's softmax.  Chunks of 2 048 and 1 161 tokens over contexts of
// 8 192 and 3 514, 32 heads of 128 on 8: 512 us (557 TFLOP/s), 2 300 with the kernel for few rows.
//
// A tile can last 100 us.  The fetching warp reads the preempt word before every block; once it is raised the tile
// ends behind the blocks under way, sums and statistics go to the context, and the next launch goes on from there.
#include "act_layout.h"
#include "kv_attend.h"
#include "planes.cuh"
#include "sm100.cuh"

#include <algorithm>
#include <type_traits>

namespace gpx {

using namespace sm100;

constexpr int kManyThreads = 448;  // two warpgroups of rows, one that converts, one warp that issues, one that fetches
constexpr int kTileRows = 256, kTileKeys = 128;
constexpr int kRawStages = 3, kKeyBuffers = 2;  // (a stage of the ring holds a block's keys or its values)
constexpr unsigned long long kManyWaitNs = 2000000000ull;
constexpr int kNotes = 512;  // the last counters of the context: {tile + 1, blocks done} of a CTA's unfinished tile

template <int D>
struct ManyCfg {
    static constexpr uint32_t kQ = 128 * D * 2;            // of a warpgroup
    static constexpr uint32_t kHalves = kTileKeys * D * 2;  // keys or values of a block, as halves
    static constexpr uint32_t kCodes = kTileKeys * D;
    static constexpr uint32_t kKeysAt = 2 * kQ, kValuesAt = kKeysAt + kKeyBuffers * kHalves, kRawAt = kValuesAt + kHalves;
    static constexpr uint32_t kCtlAt = kRawAt + kRawStages * kCodes;
    static constexpr int kSlot = 2 * kTileRows + kTileRows * D;  // floats: maxima, sums, outputs [D / 4][row][4]
};

struct ManyCtl {
    unsigned long long raw_full[kRawStages], raw_empty[kRawStages];
    unsigned long long keys_full[kKeyBuffers], keys_empty[kKeyBuffers];
    unsigned long long values_full, values_empty;
    unsigned long long s_full[2], p_full[2];
    alignas(16) float scales[4][8][4];  // of a block's sixteen keys each: keys' and values' scale, b = log2 of the values' over the largest, 2^-b
    float largest[4];       // value scale, of each converting warp's pages
    uint32_t tmem;
    int tile, done;         // the tile, and the blocks of it that an earlier launch has done
    int end;                // the block at which the tile ends
    int stopped;            // because of the word
    int saw_nan, last, abort_flag;
};

// The largest of three (one instruction on this architecture).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

template <int D, bool HALF>
__global__ void __launch_bounds__(kManyThreads, 1)
kv_attend_many_kernel(const __grid_constant__ AttendParams p, BlpArgs blp) {
    using Cfg = ManyCfg<D>;
    constexpr uint32_t kHalfTile = 128 * 128;  // bytes of 128 rows of 64 halves
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    ManyCtl *ctl = reinterpret_cast<ManyCtl *>(smem + Cfg::kCtlAt);
    int *prefix = reinterpret_cast<int *>(ctl + 1);  // [seqs + 1]
    volatile int *abort_flag = &ctl->abort_flag;
    const uint32_t base = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, wid = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const bool elected = elect_one();
    if (tid == 0) {
        for (int i = 0; i < kRawStages; ++i) mbar_init(smem_u32(&ctl->raw_full[i]), 1), mbar_init(smem_u32(&ctl->raw_empty[i]), 4);
        for (int i = 0; i < kKeyBuffers; ++i) mbar_init(smem_u32(&ctl->keys_full[i]), 4), mbar_init(smem_u32(&ctl->keys_empty[i]), 1);
        mbar_init(smem_u32(&ctl->values_full), 4), mbar_init(smem_u32(&ctl->values_empty), 1);
        for (int w = 0; w < 2; ++w) {
            mbar_init(smem_u32(&ctl->s_full[w]), 1), mbar_init(smem_u32(&ctl->p_full[w]), 4);
        }
        ctl->abort_flag = 0;
        fence_barrier_init();
        fence_proxy_async();
        prefetch_tensormap(&p.map_k), prefetch_tensormap(&p.map_v);
    }
    if (wid == 12) tmem_alloc(smem_u32(&ctl->tmem), 512);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    pdl_enter();
    const bool dynamic = blp.preempted != nullptr;
    if (tid == 0) trace_begin(blp);
    const uint32_t tmem = ctl->tmem;
    const Layout<kTileRows, kTileKeys> lay(p);
    const int group = lay.group, page_tokens = 1 << p.page_shift;
    auto wait = [&](unsigned long long *bar, uint32_t phase) {
        if (!mbar_wait(smem_u32(bar), phase, abort_flag, kManyWaitNs)) {
            *abort_flag = 1;
            lm_fail(p.error, LM_GAVE_UP, (int)blockIdx.x);
        }
    };

    // Tiles: parts of units.  A part for every unit, or as many as give each SM two tiles, if the context holds them.
    const int units = lm_prefix(prefix, p.batch.seqs, p.error, [&](int s) {
        const LmSpan span = lm_span(p.batch, s, page_tokens, false, p.error);
        const long long all = (long long)lay.row_blocks(span.n) * p.kv_heads;
        return all > 0x7fffffff ? 0x7fffffff : (int)all;
    });
    int parts = 1;
    if (units > 0 && units < 2 * (int)gridDim.x) {
        const int most = max(1, (int)min((long long)p.batch.table_ld * page_tokens / 512, 1ll << 20));
        parts = max(1, min(min((2 * (int)gridDim.x + units - 1) / units, (p.max_tiles - (int)gridDim.x) / units), most));
    }
    blp.total_tiles = units > 0x7fffffff / parts ? 0 : units * parts;
    int *const note = p.counters + kLmCounters - kNotes + 2 * blockIdx.x;
    const float *const spill_at = p.parts + (size_t)(p.max_tiles - (int)gridDim.x + (int)blockIdx.x) * Cfg::kSlot;
    int pending = dynamic && tid == 0 ? note[0] - 1 : -1;

    uint32_t n_raw = 0, n_keys = 0, n_values = 0, n_s = 0, n_p0 = 0, n_p1 = 0;  // rounds of the barriers so far
    int iter = 0, rounds = 0;
    for (;; ++rounds) {
        if (tid == 0) {
            int t = -1, done = 0;
            if (*abort_flag) {
            } else if (pending >= 0) {
                if (load_word(blp.preempted) != 0) {  // (the note stays)
                    if (blp.trace) atomicMin(blp.trace + 2, globaltimer_ns());
                    atomicCAS(blp.stop_index, -1, blp.kernel_id);
                } else {
                    t = pending, done = note[1];
                    note[0] = note[1] = 0;
                }
                pending = -1;
            } else {
                t = blp_claim(blp, iter++);
            }
            ctl->tile = t, ctl->done = done;
            ctl->end = 0x7fffffff, ctl->stopped = 0, ctl->saw_nan = 0;
        }
        __syncthreads();
        const int tile = ctl->tile, done = ctl->done;
        if (tile < 0) break;
        const int unit_index = tile / parts, part = tile - unit_index * parts;
        const int s = lm_find(prefix, p.batch.seqs, unit_index);
        // (blocks of rows from the last on: with a causal mask they have the most keys, and the longest tiles go first)
        const int rb_count = lay.row_blocks(p.batch.first[s + 1] - p.batch.first[s]);
        const int in_seq = unit_index - prefix[s];
        const Unit u = lay.unit(s, in_seq % p.kv_heads * rb_count + rb_count - 1 - in_seq / p.kv_heads);
        const int all_blocks = max(0, (u.high - u.key0 + kTileKeys - 1) / kTileKeys);
        const int block0 = (int)((long long)part * all_blocks / parts), blocks = (int)((long long)(part + 1) * all_blocks / parts) - block0;
        const int key_first = u.key0 + block0 * kTileKeys;
        const bool two = u.rows > 128;  // both warpgroups have rows
        // keys that every row sees: [all_lo, all_hi)
        const int pos0 = u.context - u.n + u.row0 / group, pos1 = u.context - u.n + (u.row0 + u.rows - 1) / group;
        const int all_hi = p.causal ? min(u.context, pos0 + 1) : u.context;
        const int all_lo = p.window ? pos1 + 1 - p.window : 0;
        auto border = [&](int key0) { return key0 + kTileKeys > all_hi || key0 < all_lo; };

        if (wid == 13) {
            // ---- fetches
            const int per_page = min(page_tokens, 64), pieces = kTileKeys / per_page, batch = 32 / pieces;
            bool stop = false;
            int j = done;
            for (; j < blocks && !stop; j += batch) {
                const int mine = lane / pieces, sub = lane - mine * pieces;
                const int key = key_first + (j + mine) * kTileKeys + sub * per_page;
                int row = -1;
                float ks = 1.f, vs = 1.f;
                if (j + mine < blocks && key < u.high) {
                    const int page = p.batch.table[(size_t)u.s * p.batch.table_ld + (key >> p.page_shift)];
                    if ((unsigned)page < (unsigned)p.pages) {
                        const long long block = (long long)page * p.kv_heads + u.head;
                        row = (int)((block << p.page_shift) + (key & (page_tokens - 1)));
                        ks = p.k_scale[block], vs = p.v_scale[block];
                    } else {
                        lm_fail(p.error, LM_BAD_PAGE, u.s);
                    }
                }
                const int some = min(batch, blocks - j);
                for (int b = 0; b < some; ++b) {
                    // (a tile runs one block at least, so that whoever is interrupted without end comes to an end)
                    if (dynamic && j + b > done) {
                        int word = 0;
                        if (lane == 0) word = load_word(blp.preempted);
                        if (__shfl_sync(0xffffffffu, word, 0) != 0) {
                            if (blp.trace && lane == 0) atomicMin(blp.trace + 2, globaltimer_ns());
                            if (lane == 0) ctl->stopped = 1;
                            stop = true;
                            j += b - batch;
                            break;
                        }
                    }
                    const bool loads = mine == b && row >= 0;
                    const uint32_t bytes = (uint32_t)(__popc(__ballot_sync(0xffffffffu, loads)) * per_page * D);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int st = n_raw % kRawStages;
                        wait(&ctl->raw_empty[st], (n_raw / kRawStages & 1) ^ 1);
                        if (i == 0 && mine == b)
                            for (int w = sub * per_page / 16; w < (sub + 1) * per_page / 16; ++w)
                                ctl->scales[(j + b) & 3][w][0] = ks, ctl->scales[(j + b) & 3][w][1] = vs;
                        __syncwarp();
                        const uint32_t full = smem_u32(&ctl->raw_full[st]);
                        if (lane == 0) mbar_arrive_expect_tx(full, bytes);
                        __syncwarp();
                        if (loads) tma_load_2d(base + Cfg::kRawAt + st * Cfg::kCodes + sub * per_page * D, i ? &p.map_v : &p.map_k, full, 0, row);
                        __syncwarp();
                        ++n_raw;
                    }
                }
            }
            // the end of the tile goes through the ring like a block's keys
            j = min(j, blocks);
            const int st = n_raw % kRawStages;
            wait(&ctl->raw_empty[st], (n_raw / kRawStages & 1) ^ 1);
            if (lane == 0) {
                ctl->end = j;
                mbar_arrive(smem_u32(&ctl->raw_full[st]));
            }
            __syncwarp();
            ++n_raw;
        } else if (wid == 12) {
            // ---- issues the products
            constexpr uint32_t idesc_s = make_idesc_f16_f32(128, kTileKeys);
            constexpr uint32_t idesc_o = make_idesc_f16_f32(128, D) | (1u << 16);  // B is MN-major: value rows are keys
            auto scores = [&](int w, uint32_t keys) {
                if (elected && !*abort_flag) {
                    const uint64_t dq = make_smem_desc_sw128(base + w * Cfg::kQ), dk = make_smem_desc_sw128(keys);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint32_t step = (k & 3) * 2 + (k >> 2) * (kHalfTile >> 4);
                        mma_f16_ss(tmem + w * 256, dq + step, dk + step, idesc_s, k > 0 ? 1u : 0u);
                    }
                }
                __syncwarp();
            };
            auto commit = [&](unsigned long long *bar) {
                if (elected) mma_commit(smem_u32(bar));
                __syncwarp();
            };
            auto keys_at = [&]() { return base + Cfg::kKeysAt + (n_keys % kKeyBuffers) * Cfg::kHalves; };
            // the queries are there once their warpgroups have arrived for the first time
            wait(&ctl->p_full[0], n_p0++ & 1);
            if (two) wait(&ctl->p_full[1], n_p1++ & 1);
            for (int j = done;; ++j) {
                // scores of block j, the products with the values of block j - 1 before them
                wait(&ctl->keys_full[n_keys % kKeyBuffers], n_keys / kKeyBuffers & 1);
                tc_fence_after_sync();
                const bool ends = j >= *(volatile int *)&ctl->end || *abort_flag;
                const bool has_values = j > done;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    if (w == 1 && !two) break;
                    if (has_values) {
                        if (w == 0) wait(&ctl->values_full, n_values & 1);
                        wait(&ctl->p_full[w], (w ? n_p1++ : n_p0++) & 1);
                        tc_fence_after_sync();
                        if (elected && !*abort_flag) {
                            const uint64_t dv = (make_smem_desc_sw128(base + Cfg::kValuesAt) & ~(0x3fffull << 16)) |
                                                ((uint64_t)(kHalfTile >> 4) << 16);
                            const uint32_t t_o = tmem + w * 256 + 128;
                            const bool fresh = j - 1 == 0;  // (a tile that goes on has its sums in place)
#pragma unroll
                            for (int k = 0; k < kTileKeys / 16; ++k)
                                mma_f16_ts(t_o, tmem + w * 256 + 8 * k, dv + 128 * k, idesc_o, fresh && k == 0 ? 0u : 1u);
                        }
                        __syncwarp();
                    }
                    if (!ends) scores(w, keys_at());
                    commit(&ctl->s_full[w]);
                }
                if (has_values) {
                    commit(&ctl->values_empty);
                    ++n_values;
                }
                commit(&ctl->keys_empty[n_keys % kKeyBuffers]);
                ++n_keys;
                if (ends) break;
            }
        } else if (wid >= 8) {
            // ---- turns codes into halves: a thread a key
            const int r = tid - 256;
            // the largest scale of the tile's values
            float most = 0.f;
            for (int i = (key_first >> p.page_shift) + r; (i << p.page_shift) < min(u.high, key_first + blocks * kTileKeys); i += 128) {
                const int page = p.batch.table[(size_t)u.s * p.batch.table_ld + i];
                if ((unsigned)page < (unsigned)p.pages) most = fmaxf(most, p.v_scale[(long long)page * p.kv_heads + u.head]);
            }
            most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
            if (lane == 0) ctl->largest[wid - 8] = most;
            asm volatile("bar.sync 3, 128;" ::: "memory");
            most = fmaxf(fmaxf(ctl->largest[0], ctl->largest[1]), fmaxf(ctl->largest[2], ctl->largest[3]));
            most = fmaxf(most, 1.17549435e-38f);
            // sixteen codes from a piece of a row to two pieces of a row of halves
            auto convert = [&](const unsigned char *from, unsigned char *to, int c, __half2 factor, bool scaled, bool sanitise, bool drop) {
                const uint4 w = *reinterpret_cast<const uint4 *>(from + (D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4)));
                const uint32_t in[4] = {w.x, w.y, w.z, w.w};
                uint32_t out[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t x = in[i];
                    if (sanitise) {
                        const uint32_t nan = nan_bytes(x);
                        if (nan && !drop) ctl->saw_nan = 1;
                        x = drop ? 0u : x & ~nan;
                    }
                    out[2 * i] = e4m3x2_to_f16x2((unsigned short)x), out[2 * i + 1] = e4m3x2_to_f16x2((unsigned short)(x >> 16));
                    if (scaled) {
#pragma unroll
                        for (int e = 2 * i; e < 2 * i + 2; ++e) {
                            const __half2 y = __hmul2(*reinterpret_cast<__half2 *>(&out[e]), factor);
                            out[e] = *reinterpret_cast<const uint32_t *>(&y);
                        }
                    }
                }
                unsigned char *row = to + (c >> 2) * kHalfTile + r * 128;
                *reinterpret_cast<uint4 *>(row + ((((c & 3) * 2) ^ (r & 7)) << 4)) = make_uint4(out[0], out[1], out[2], out[3]);
                *reinterpret_cast<uint4 *>(row + ((((c & 3) * 2 + 1) ^ (r & 7)) << 4)) = make_uint4(out[4], out[5], out[6], out[7]);
            };
            for (int j = done;; ++j) {
                int st = n_raw % kRawStages;
                wait(&ctl->raw_full[st], n_raw / kRawStages & 1);
                const bool ends = j >= *(volatile int *)&ctl->end || *abort_flag;
                const int buffer = n_keys % kKeyBuffers;
                // (a scale 2^40 below the largest counts as that, or its keys would vanish from the normaliser; the rest
                // goes into the values)
                const float ratio = fmaxf(ctl->scales[j & 3][r >> 4][1], 1.17549435e-38f) / most, used = fmaxf(ratio, 9.094947e-13f);
                if (!ends && (r & 15) == 0) ctl->scales[j & 3][r >> 4][2] = log2f(used), ctl->scales[j & 3][r >> 4][3] = 1.f / used;
                wait(&ctl->keys_empty[buffer], (n_keys / kKeyBuffers & 1) ^ 1);
                if (!ends) {
                    const unsigned char *from = smem + Cfg::kRawAt + st * Cfg::kCodes;
                    unsigned char *to = smem + Cfg::kKeysAt + buffer * Cfg::kHalves;
#pragma unroll 4
                    for (int c = 0; c < D / 16; ++c) convert(from, to, c, __half2(), false, false, false);
                    fence_proxy_async();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->raw_empty[st])), mbar_arrive(smem_u32(&ctl->keys_full[buffer]));
                ++n_raw, ++n_keys;
                if (ends) break;
                st = n_raw % kRawStages;
                wait(&ctl->raw_full[st], n_raw / kRawStages & 1);
                wait(&ctl->values_empty, (n_values & 1) ^ 1);
                const int key0 = key_first + j * kTileKeys;
                const __half2 factor = __float2half2_rn(ratio / used);
                const unsigned char *from = smem + Cfg::kRawAt + st * Cfg::kCodes;
                unsigned char *to = smem + Cfg::kValuesAt;
                if (border(key0)) {
                    // (values of keys that not every row sees: no NaN among them may reach a row that does not)
                    const bool drop = key0 + r >= u.high || key0 + r < u.low;
#pragma unroll 2
                    for (int c = 0; c < D / 16; ++c) convert(from, to, c, factor, true, true, drop);
                } else if (__any_sync(0xffffffffu, ratio != used)) {
#pragma unroll 4
                    for (int c = 0; c < D / 16; ++c) convert(from, to, c, factor, true, false, false);
                } else {
#pragma unroll 4
                    for (int c = 0; c < D / 16; ++c) convert(from, to, c, factor, false, false, false);
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->raw_empty[st])), mbar_arrive(smem_u32(&ctl->values_full));
                ++n_raw, ++n_values;
            }
        } else if (wid < 4 || two) {
            // ---- softmax: a thread a row
            const int w = wid >> 2, row = tid & 127, r = w * 128 + row;
            const bool live = r < u.rows;
            const uint32_t lanes = (uint32_t)((wid & 3) * 32) << 16;
            const uint32_t t_s = tmem + w * 256 + lanes, t_o = t_s + 128;
            const int at = u.row0 + min(r, u.rows - 1);
            const long long token = u.first + at / group;
            const int head = u.head * group + at % group;
            float factor = 1.f;
            {
                // the row's queries, as halves, into the swizzled operand
                const uint4 *q = reinterpret_cast<const uint4 *>(p.q + token * p.q_ld + (long long)head * D);
                unsigned char *to = smem + w * Cfg::kQ + row * 128;
                float inv = 1.f;
                if (!HALF) {
                    uint32_t most = 0;
#pragma unroll 4
                    for (int c = 0; c < D / 8; ++c) {
                        const uint4 x = q[c];
                        const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) most = max(most, max(v[i] << 16 & 0x7fffffffu, v[i] & 0x7fff0000u));
                    }
                    const uint32_t e = most >> 23;
                    if (e > 0 && e < 253) factor = __uint_as_float(e << 23);
                    inv = 1.0f / factor;
                }
#pragma unroll 4
                for (int c = 0; c < D / 8; ++c) {
                    uint4 x = live ? q[c] : make_uint4(0, 0, 0, 0);
                    if (!HALF) {
                        uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = pack_halves(__uint_as_float(v[i] << 16) * inv, __uint_as_float(v[i] & 0xffff0000u) * inv);
                        x = make_uint4(v[0], v[1], v[2], v[3]);
                    }
                    *reinterpret_cast<uint4 *>(to + (c >> 3) * kHalfTile + (((c & 7) ^ (row & 7)) << 4)) = x;
                }
            }
            const float mult = factor * p.scale * 1.4426950408889634f;
            const int pos = u.context - u.n + at / group;
            const int hi = p.causal ? min(u.context, pos + 1) : u.context, lo = p.window ? pos + 1 - p.window : 0;
            float m = -INFINITY, l = 0.f;
            if (done > 0) {
                // an interrupted tile goes on
                m = spill_at[r], l = spill_at[kTileRows + r];
                const float4 *from = reinterpret_cast<const float4 *>(spill_at + 2 * kTileRows) + r;
#pragma unroll
                for (int c = 0; c < D; c += 16) {
                    uint32_t o[16];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 x = __ldcg(from + (c / 4 + i) * kTileRows);
                        o[4 * i] = __float_as_uint(x.x), o[4 * i + 1] = __float_as_uint(x.y), o[4 * i + 2] = __float_as_uint(x.z), o[4 * i + 3] = __float_as_uint(x.w);
                    }
                    tmem_st_32x16(t_o + c, o);
                }
                tmem_st_wait();
            }
            auto arrive = [&]() {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->p_full[w]));
            };
            fence_proxy_async();
            arrive();
            int j = done;
            for (;; ++j) {
                wait(&ctl->s_full[w], n_s++ & 1);
                __syncwarp();
                tc_fence_after_sync();
                if (j >= *(volatile int *)&ctl->end || *abort_flag) break;  // (no scores, but the last products are complete)
                const int key0 = key_first + j * kTileKeys;
                const bool masks = border(key0);
                const float4 *of = reinterpret_cast<const float4 *>(ctl->scales[j & 3]);  // (by groups of sixteen keys)
                // the row's maximum
                float most = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t v[32];
                    tmem_ld_32x32(t_s + 32 * c, v);
                    tmem_ld_wait();
                    if (masks) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const int key = key0 + 32 * c + i;
                            if (key >= hi || key < lo) v[i] = 0xff800000u;
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float x = max3(__uint_as_float(v[16 * h]), __uint_as_float(v[16 * h + 1]), __uint_as_float(v[16 * h + 2]));
                        float y = max3(__uint_as_float(v[16 * h + 3]), __uint_as_float(v[16 * h + 4]), __uint_as_float(v[16 * h + 5]));
#pragma unroll
                        for (int i = 6; i < 14; i += 4) {
                            x = max3(x, __uint_as_float(v[16 * h + i]), __uint_as_float(v[16 * h + i + 1]));
                            y = max3(y, __uint_as_float(v[16 * h + i + 2]), __uint_as_float(v[16 * h + i + 3]));
                        }
                        x = max3(fmaxf(x, y), __uint_as_float(v[16 * h + 14]), __uint_as_float(v[16 * h + 15]));
                        const float4 g = of[2 * c + h];
                        most = fmaxf(most, fmaf(x, g.x * mult, g.z));
                    }
                }
                const float now = fmaxf(m, most);
                if (j == 0) {
                    m = now;
                } else if (__any_sync(0xffffffffu, now > m)) {
                    // (the scores' arrival means that the products before them are complete)
                    const float f = now == -INFINITY ? 1.f : lm_ex2(m - now);
#pragma unroll
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tmem_ld_32x32(t_o + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st_32x32(t_o + c, o);
                    }
                    l *= f;
                    m = now;
                }
                const float ref = m == -INFINITY ? 0.f : m;
                float sum = 0.f;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t v[32], h[16];
                    tmem_ld_32x32(t_s + 32 * c, v);
                    tmem_ld_wait();
                    if (masks) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const int key = key0 + 32 * c + i;
                            if (key >= hi || key < lo) v[i] = 0xff800000u;
                        }
                    }
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const float4 g = of[2 * c + q];
                        const float2 by = make_float2(g.x * mult, g.x * mult), plus = make_float2(g.z - ref, g.z - ref);
                        float2 part = make_float2(0.f, 0.f);
#pragma unroll
                        for (int i = 8 * q; i < 8 * q + 8; ++i) {
                            const float2 x = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), by, plus);
                            const float2 e = make_float2(lm_ex2(x.x), lm_ex2(x.y));
                            part = add2(part, e);
                            h[i] = pack_halves(e.x, e.y);
                        }
                        sum = fmaf(part.x + part.y, g.w, sum);
                    }
                    tmem_st_32x16(t_s + 16 * c, h);
                }
                l += sum;
                tmem_st_wait();
                arrive();
            }
            __syncwarp();
            // ---- the end: a whole tile's rows are finished, a part or an unfinished tile goes to the context
            const bool any = j > 0;  // products have been made
            const float unit = fmaxf(fmaxf(fmaxf(ctl->largest[0], ctl->largest[1]), fmaxf(ctl->largest[2], ctl->largest[3])), 1.17549435e-38f);
            const bool stopped = ctl->stopped != 0;
            const int upto = min(u.high, key_first + j * kTileKeys);
            // elements whose values were NaN for a key that this row sees, in blocks that they were taken out of
            uint32_t nan[D / 32];
#pragma unroll
            for (int i = 0; i < D / 32; ++i) nan[i] = 0;
            if (ctl->saw_nan && live) {
                for (int key = max(lo, key_first + done * kTileKeys); key < min(hi, upto); ++key) {
                    if (!border(key_first + (key - key_first) / kTileKeys * kTileKeys)) continue;
                    const int page = p.batch.table[(size_t)u.s * p.batch.table_ld + (key >> p.page_shift)];
                    if ((unsigned)page >= (unsigned)p.pages) continue;
                    const uint4 *code = reinterpret_cast<const uint4 *>(p.v_codes + ((((long long)page * p.kv_heads + u.head) << p.page_shift) + (key & (page_tokens - 1))) * D);
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        const uint4 x = code[2 * i], y = code[2 * i + 1];
                        const uint32_t v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint32_t b = nan_bytes(v[e]);
                            nan[i] |= ((b & 1u) | (b >> 7 & 2u) | (b >> 14 & 4u) | (b >> 21 & 8u)) << (4 * e);
                        }
                    }
                }
            }
            const bool to_context = stopped || parts > 1;
            float *slot = const_cast<float *>(stopped ? spill_at : p.parts + (size_t)tile * Cfg::kSlot);
            // (a row without keys is zero; one whose keys all score -infinity is not a number, as the formula says)
            const bool empty = hi <= 0;
            float inv = empty ? 0.f : unit / l;
            uint32_t *out = reinterpret_cast<uint32_t *>(p.out + token * p.out_ld + (long long)head * D);
#pragma unroll
            for (int c = 0; c < D; c += 16) {
                uint32_t o[16];
                __syncwarp();
                tmem_ld_32x16(t_o + c, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (!any) o[i] = 0u;
                    if (nan[c / 32] >> ((c & 16) + i) & 1u) o[i] = 0x7fffffffu;
                }
                if (to_context) {
                    // (an unfinished tile's sums stay in its unit, a part's are in none)
                    const float f = stopped ? 1.f : unit;
                    float4 *to = reinterpret_cast<float4 *>(slot + 2 * kTileRows) + r;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        to[(c / 4 + i) * kTileRows] = make_float4(__uint_as_float(o[4 * i]) * f, __uint_as_float(o[4 * i + 1]) * f,
                                                                  __uint_as_float(o[4 * i + 2]) * f, __uint_as_float(o[4 * i + 3]) * f);
                } else if (live) {
                    uint32_t h[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        h[i] = empty ? 0u : pack_out<HALF>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
                    reinterpret_cast<uint4 *>(out + c / 2)[0] = make_uint4(h[0], h[1], h[2], h[3]);
                    reinterpret_cast<uint4 *>(out + c / 2)[1] = make_uint4(h[4], h[5], h[6], h[7]);
                }
            }
            if (to_context) {
                slot[r] = m, slot[kTileRows + r] = l;
            } else if (live && p.lse) {
                p.lse[token * p.heads + head] = empty ? -INFINITY : (m == -INFINITY ? m : m * 0.69314718055994531f) + logf(l);
            }
            if (to_context) __threadfence();
        }
        tc_fence_before_sync();
        // (warpgroups without rows keep step with the barriers' rounds: they took part in none)
        __syncthreads();
        tc_fence_after_sync();
        if (ctl->stopped) {
            if (tid == 0) {
                note[0] = tile + 1, note[1] = ctl->end;
                atomicCAS(blp.stop_index, -1, blp.kernel_id);
            }
            break;
        }
        if (parts > 1) {
            if (tid == 0) {
                __threadfence();
                ctl->last = atomicAdd(&p.counters[unit_index], 1) == parts - 1;
            }
            __syncthreads();
            if (ctl->last && tid < kTileRows && tid < u.rows) {
                __threadfence();
                const int r = tid, at = u.row0 + r;
                const long long token = u.first + at / group;
                const int head = u.head * group + at % group;
                const float *first = p.parts + (size_t)unit_index * parts * Cfg::kSlot;
                float m = -INFINITY, l = 0.f;
                for (int q = 0; q < parts; ++q) m = fmaxf(m, __ldcg(first + (size_t)q * Cfg::kSlot + r));
                const float ref = m == -INFINITY ? 0.f : m;
                for (int q = 0; q < parts; ++q) {
                    const float *slot = first + (size_t)q * Cfg::kSlot;
                    l = fmaf(__ldcg(slot + kTileRows + r), lm_ex2(__ldcg(slot + r) - ref), l);
                }
                const int pos = u.context - u.n + at / group;
                const bool empty = (p.causal ? min(u.context, pos + 1) : u.context) <= 0;
                const float inv = empty ? 0.f : 1.0f / l;
                uint32_t *out = reinterpret_cast<uint32_t *>(p.out + token * p.out_ld + (long long)head * D);
                for (int c = 0; c < D / 4; c += 4) {
                    float4 x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int q = 0; q < parts; ++q) {
                        const float *slot = first + (size_t)q * Cfg::kSlot;
                        const float f = lm_ex2(__ldcg(slot + r) - ref);
                        const float4 *from = reinterpret_cast<const float4 *>(slot + 2 * kTileRows) + r;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float4 y = __ldcg(from + (c + i) * kTileRows);
                            x[i].x = fmaf(y.x, f, x[i].x), x[i].y = fmaf(y.y, f, x[i].y), x[i].z = fmaf(y.z, f, x[i].z), x[i].w = fmaf(y.w, f, x[i].w);
                        }
                    }
                    uint32_t h[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        h[2 * i] = empty ? 0u : pack_out<HALF>(x[i].x * inv, x[i].y * inv);
                        h[2 * i + 1] = empty ? 0u : pack_out<HALF>(x[i].z * inv, x[i].w * inv);
                    }
                    reinterpret_cast<uint4 *>(out + 2 * c)[0] = make_uint4(h[0], h[1], h[2], h[3]);
                    reinterpret_cast<uint4 *>(out + 2 * c)[1] = make_uint4(h[4], h[5], h[6], h[7]);
                }
                if (p.lse) p.lse[token * p.heads + head] = empty ? -INFINITY : (m == -INFINITY ? m : m * 0.69314718055994531f) + logf(l);
            }
            __syncthreads();
            if (ctl->last && tid == 0) p.counters[unit_index] = 0;
        }
        if (*abort_flag) break;
    }
    if (*abort_flag)
        for (int spin = 0; spin < 64; ++spin) __nanosleep(1000);  // copies and products in flight end before the CTA does
    __syncthreads();
    if (wid == 12) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
    if (tid == 0) trace_end(blp, rounds);
}

cudaError_t kv_attend_many_launch(AttendParams &p, int dim, bool half, const DeviceInfo &d, const BlpArgs &blp, cudaStream_t s) {
    auto go = [&](auto kernel, uint32_t fixed, int slot) {
        const size_t smem = 1024 + fixed + sizeof(ManyCtl) + (p.batch.seqs + 1) * sizeof(int);
        int per_sm;
        const cudaError_t e = lm_resident((const void *)kernel, kManyThreads, smem, d.device, &per_sm);
        if (e != cudaSuccess) return e;
        const int grid = std::min(d.sm_count, kNotes / 2);
        p.max_tiles = (int)std::min<size_t>(kLmCounters - kNotes, kLmPartsBytes / ((size_t)slot * sizeof(float)));
        return launch_layer(kernel, grid, kManyThreads, smem, s, p, blp);
    };
    if (dim == 64)
        return half ? go(kv_attend_many_kernel<64, true>, ManyCfg<64>::kCtlAt, ManyCfg<64>::kSlot)
                    : go(kv_attend_many_kernel<64, false>, ManyCfg<64>::kCtlAt, ManyCfg<64>::kSlot);
    return half ? go(kv_attend_many_kernel<128, true>, ManyCfg<128>::kCtlAt, ManyCfg<128>::kSlot)
                : go(kv_attend_many_kernel<128, false>, ManyCfg<128>::kCtlAt, ManyCfg<128>::kSlot);
}

}  // namespace gpx
