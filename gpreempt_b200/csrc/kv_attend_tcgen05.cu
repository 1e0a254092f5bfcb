// Attention of new tokens over a paged 8-bit cache, for many rows a head of keys (prompts and their chunks), on the
// tcgen05 tensor cores.  The formula is that of kv_attend.cu.
//
// A unit is a block of 256 rows (a group's heads times the tokens) of one head of keys against all keys they see.  The
// blocks of 128 keys of all units lie on one line, as many of each as its rows see, and a tile is an equal piece of it, one for
// each SM.  A unit that spans tiles leaves their parts in the context, and the CTA that brings the last one joins them.
// Per block of 128 keys:
//   - one warp fetches keys and values as they are in the cache (TMA), with the pages' scales,
//   - four warps turn the codes into halves (exact: every e4m3 number is a half) in the swizzled layout of the operands,
//   - the scales are left to the softmax, the values' as in kv_attend.cu: relative to the largest of the tile they join the exponents,
//   - one warp issues S = Q K^T and O += P V of the two halves of the rows in turn,
//   - two warpgroups, a thread a row, take the scores out of tensor memory, and put the probabilities back as a 16-bit A
//     operand, where the scores were.  The values lie with keys as rows; their descriptor names that MN-major.
// Queries become halves after a power of two that brings their row's largest to 1, as in kv_attend.cu.  Factors are one half, of fp16
// results too (kv_attend.cu takes two for those): eleven bits, the result's own; a second product of 128 keys would add half to the tensor cores' time.
//
// What bounds it: 256 x 128 exponentials a block are 2 048 cycles of the special-function unit, the products 2 048
// of the tensor cores, and shared memory carries 320 KB for them (2 500 cycles).  The halves of the rows are
// half a block apart, so that one's products run under the other's softmax, and a block takes 3 600 cycles: 2 050 from a
// half's scores to its factors, 1 450 from those to its next scores.  (Four warpgroups for the scores, two threads a row,
// took as long for the factors and 300 more to agree on them: 391 us against 362.)  The start and end of a unit take another
// 25 000.  Chunks of 2 048 and 889 tokens over contexts of 8 192 and 3 474, 32 heads of 128 on 8: 321 us (886 TFLOP/s), 2 300
// with the kernel for few rows.  At 128 registers for the compiler it spills 244 to 320 bytes for heads of 128, 184 to 240 for 64.
//
// A tile can last hundreds of microseconds.  The fetching warp reads the preempt word before every block; once it is
// raised the tile ends behind the blocks under way, sums and statistics go to the context, and the next launch goes on from there: drained
// in 21 us at the median, 23 at most, in the case above, which takes no longer with a word than without.
#include "act_layout.h"
#include "kv_attend.h"
#include "planes.cuh"
#include "sm100.cuh"

#include <algorithm>
#include <type_traits>

namespace gpx {

using namespace sm100;

constexpr int kManyThreads = 512;  // two warpgroups of rows, one that converts, and one with a warp that issues and one that fetches
// registers of a thread of the first two and of the others: together what the CTA was launched with, 128 a thread
constexpr int kManyRegs = 168, kFewRegs = 88;
constexpr int kTileRows = 256, kTileKeys = 128;
constexpr int kRawStages = 2, kKeyBuffers = 2, kValueBuffers = 2;  // (a stage of the ring holds a block's keys or its values)
constexpr unsigned long long kManyWaitNs = 2000000000ull;
// A row's exponents refer to kLift below its maximum in the first block it sees (so that thousands of keys that weigh 2^-26 each beside one
// of that block count: a half ends at 2^-25) until their factors sum to more than this in a block, which a half holds; then the maximum
// is taken anew and the sums are rescaled.  (Asking for the maximum of every block goes through its scores twice, and a new one among
// 32 rows, which are rescaled together, comes in most blocks.  2^7 below and sums up to 2^15 took 327 to 350 us where this takes 317 to 328.)
constexpr float kMostFactors = 60000.f, kLift = 6.f;
// What the start of a unit takes (queries, the first blocks until their products run, outputs), in blocks: that many places of the
// line come before its own, so that a tile of many short units has as long as one of a single long unit.
// (Chunks of 2 048 and 889 tokens: 350 us without, 325 with 6, 323 with 8 and 10, 325 with 14.)
constexpr int kUnitCost = 8;
// Blocks of the longest unit up to which units are not cut.  Uncut and cut, 32 heads of 128 on 8: 8 sequences of 37 tokens over 512
// keys 21.5 and 24.0 us, 2 of 64 over 764 (6 blocks) 29.6 and 35.9.  With units of 9 to 13 blocks it depends on how they fill
// the SMs: 8 of 64 over 1 064 37.7 and 41.9, 2 of 64 over 1 564 44.6 and 41.9.
constexpr int kShortUnit = 8;
constexpr int kNotes = 1024;  // the last counters of the context: {tile + 1, blocks done, whether sums were left} of a CTA's unfinished tile

template <int D>
struct ManyCfg {
    static constexpr uint32_t kQ = 128 * D * 2;            // of a warpgroup
    static constexpr uint32_t kHalves = kTileKeys * D * 2;  // keys or values of a block, as halves
    static constexpr uint32_t kCodes = kTileKeys * D;
    static constexpr uint32_t kKeysAt = 2 * kQ, kValuesAt = kKeysAt + kKeyBuffers * kHalves, kRawAt = kValuesAt + kValueBuffers * kHalves;
    static constexpr uint32_t kCtlAt = kRawAt + kRawStages * kCodes;
    static constexpr int kSlot = 2 * kTileRows + kTileRows * D;  // floats: maxima, sums, outputs [D / 4][row][4]
};

// Sequences whose sums have room in what the operands leave of shared memory; sums of more are read from the context.
constexpr int kFewSeqs = 128;

struct ManyCtl {
    unsigned long long raw_full[kRawStages], raw_empty[kRawStages];
    unsigned long long keys_full[kKeyBuffers], keys_empty[kKeyBuffers];
    unsigned long long values_full[kValueBuffers], values_empty[kValueBuffers];
    unsigned long long s_full[2], p_full[2];
    alignas(16) float scales[4][8][4];  // of a block's sixteen keys each: keys' and values' scale, b = log2 of the values' over the largest, 2^-b
    float largest[4];       // value scale, of each converting warp's pages
    uint32_t tmem;
    int tile, done, spilled;  // the tile, the blocks of it that an earlier launch has done, and whether the last unit's sums were left
    int end;                  // the block of the unit at which the piece ends
    int stopped;              // because of the word
    int saw_nan, last, longest, abort_flag;
    int prefix[kFewSeqs];
};

// Of exponents of 2^20 and more the largest itself: it has no bits for the difference.
__device__ __forceinline__ float reference_of(float largest) { return fabsf(largest) < 1048576.f ? largest - kLift : largest; }

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t from) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
    return v;
}

// A piece of a unit that a tile has.
struct Piece {
    Unit u;
    int tile, line0, unit0, unit_blocks;  // the tile and its first block on the line; the unit's first there, and its blocks
    int b0, b1, done, blocks;             // blocks [b0, b1) of the unit, from `done` on, of which those before `blocks` have keys
    bool whole, goes_on, ran;             // it is all of the unit; its sums are in the context; this launch has run a block already
    bool two;                             // both warpgroups have rows
    int all_lo, all_hi;                   // keys that every row sees
    __device__ int key(int j) const { return u.key0 + j * kTileKeys; }
    __device__ bool border(int j) const { return key(j) + kTileKeys > all_hi || key(j) < all_lo; }
};

template <int D, bool HALF>
__global__ void __launch_bounds__(kManyThreads, 1)
kv_attend_many_kernel(const __grid_constant__ AttendParams p, BlpArgs blp) {
    using Cfg = ManyCfg<D>;
    using Rows = WarpRows<D>;
    constexpr uint32_t kHalfTile = 128 * 128;  // bytes of 128 rows of 64 halves
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    ManyCtl *ctl = reinterpret_cast<ManyCtl *>(smem + Cfg::kCtlAt);
    // [seqs + 1]; of many sequences in the context, the same from every CTA (shared memory is full)
    int *const prefix = p.batch.seqs < kFewSeqs ? ctl->prefix : p.prefix;
    volatile int *abort_flag = &ctl->abort_flag;
    const uint32_t base = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, wid = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const bool elected = elect_one();
    if (tid == 0) {
        for (int i = 0; i < kRawStages; ++i) mbar_init(smem_u32(&ctl->raw_full[i]), 1), mbar_init(smem_u32(&ctl->raw_empty[i]), 4);
        for (int i = 0; i < kKeyBuffers; ++i) mbar_init(smem_u32(&ctl->keys_full[i]), 4), mbar_init(smem_u32(&ctl->keys_empty[i]), 1);
        for (int i = 0; i < kValueBuffers; ++i) mbar_init(smem_u32(&ctl->values_full[i]), 4), mbar_init(smem_u32(&ctl->values_empty[i]), 1);
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

    // ---- the line of blocks
    auto blocks_of = [&](const Unit &u) { return max(1, (u.high - u.key0 + kTileKeys - 1) / kTileKeys); };
    // (Sequences of many blocks of rows are counted by a warp, the others by a thread.  Counts and sums are made where
    // the queries will lie; the sums then go to the context, and no CTA ever writes anything else there.)
    int *const count = reinterpret_cast<int *>(smem);
    if (tid == 0) ctl->longest = 0;
    __syncthreads();
    for (int s = tid; s < p.batch.seqs; s += kManyThreads) {
        const LmSpan span = lm_span(p.batch, s, page_tokens, false, p.error);
        const int rows = lay.row_blocks(span.n);
        long long all = rows > 8 ? -1 : 0;
        for (int i = 0; all >= 0 && i < rows; ++i) {
            const int blocks = blocks_of(lay.unit(s, i));
            if (blocks > kShortUnit) ctl->longest = blocks;
            all += blocks + kUnitCost;
        }
        count[s] = (int)min(all < 0 ? all : all * p.kv_heads, 0x7fffffffll);
    }
    __syncthreads();
    for (int s = wid; s < p.batch.seqs; s += kManyThreads / 32) {
        if (count[s] >= 0) continue;
        const int rows = lay.row_blocks(p.batch.first[s + 1] - p.batch.first[s]);
        long long all = 0;
        for (int i = lane; i < rows; i += 32) {
            const int blocks = blocks_of(lay.unit(s, i));
            if (blocks > kShortUnit) ctl->longest = blocks;
            all += blocks + kUnitCost;
        }
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
        if (lane == 0) count[s] = (int)min(all * p.kv_heads, 0x7fffffffll);
    }
    __syncthreads();
    // Units of a few blocks each are tiles as they are: joining their parts would take longer than their blocks.
    const bool by_unit = ctl->longest == 0;
    const int n_line = lm_prefix(count, p.batch.seqs, p.error, [&](int s) {
        return by_unit && count[s] ? lay.row_blocks(p.batch.first[s + 1] - p.batch.first[s]) * p.kv_heads : count[s];
    });
    for (int s = tid; s <= p.batch.seqs; s += kManyThreads) prefix[s] = n_line ? count[s] : 0;
    __syncthreads();
    const int tiles = by_unit ? n_line : min(n_line, (int)gridDim.x);
    blp.total_tiles = tiles;
    auto on_line = [&](const Unit &u) { return by_unit ? 1 : kUnitCost + blocks_of(u); };  // what a unit takes of the line
    const LmCut cut(n_line, tiles);
    int *const note = p.counters + kLmCounters - kNotes + 4 * blockIdx.x;
    float *const spill = p.parts + (size_t)(p.max_tiles - (int)gridDim.x + (int)blockIdx.x) * Cfg::kSlot;
    auto largest_scale = [&]() { return fmaxf(fmaxf(fmaxf(ctl->largest[0], ctl->largest[1]), fmaxf(ctl->largest[2], ctl->largest[3])), 1.17549435e-38f); };

    // Every warp walks the tiles and their pieces of units alike: role(piece) is its share of one, join(piece, t0, t1) what it does
    // where this CTA is the last to bring a part of the unit, of which tiles t0 .. t1 have one each.
    int rounds = 0;
    auto walk = [&](auto &&role, auto &&join) {
        int iter = 0;
        bool ran = false;  // a block in this launch
        int pending = dynamic && tid == 0 ? note[0] - 1 : -1;
        for (;; ++rounds) {
            if (tid == 0) {
                int t = -1, done = 0, spilled = 0;
                if (*abort_flag) {
                } else if (pending >= 0) {
                    if (load_word(blp.preempted) != 0) {  // (the note stays)
                        if (blp.trace) atomicMin(blp.trace + 2, globaltimer_ns());
                        atomicCAS(blp.stop_index, -1, blp.kernel_id);
                    } else {
                        t = pending, done = note[1], spilled = note[2];
                        note[0] = note[1] = note[2] = 0;  // (other kernels' counters and notes are the same words: a note that is taken leaves none behind)
                    }
                    pending = -1;
                } else {
                    t = blp_claim(blp, iter++);
                }
                ctl->tile = t, ctl->done = done, ctl->spilled = spilled;
                ctl->end = 0x7fffffff, ctl->stopped = 0, ctl->saw_nan = 0;
            }
            __syncthreads();
            Piece x;
            x.tile = ctl->tile;
            if (x.tile < 0) return;
            x.line0 = cut.begin(x.tile);
            const int line1 = cut.begin(x.tile + 1);
            // the first unit: its sequence, head and block of rows
            // (where a unit is a tile, its place on the line is not that of its blocks: what is done of it is added below)
            int at = x.line0 + (by_unit ? 0 : ctl->done);
            int s = lm_find(prefix, p.batch.seqs, at);
            int rb_count = lay.row_blocks(p.batch.first[s + 1] - p.batch.first[s]), rb = 0;
            const int a_head = (prefix[s + 1] - prefix[s]) / p.kv_heads;
            int head = (at - prefix[s]) / a_head;
            x.unit0 = prefix[s] + head * a_head;
            for (;; rb += 32) {
                int upto = rb + lane < rb_count ? on_line(lay.unit(s, rb + lane)) : 0;
                const int own = upto;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, upto, d);
                    if (lane >= d) upto += up;
                }
                const unsigned beyond = __ballot_sync(0xffffffffu, own > 0 && x.unit0 + upto > at);
                if (beyond) {
                    const int first = __ffs(beyond) - 1;
                    x.unit0 += __shfl_sync(0xffffffffu, upto - own, first);
                    rb += first;
                    break;
                }
                x.unit0 += __shfl_sync(0xffffffffu, upto, 31);
            }
            x.goes_on = ctl->spilled != 0;
            for (;;) {
                x.u = lay.unit(s, head * rb_count + rb);
                x.unit_blocks = blocks_of(x.u);
                if (by_unit) x.b0 = 0, x.b1 = x.unit_blocks, x.done = ctl->done;
                else {
                    const int first = x.unit0 + kUnitCost;  // the place of its first block
                    x.b0 = max(x.line0 - first, 0), x.b1 = min(line1 - first, x.unit_blocks), x.done = max(at - first, 0);
                    if (x.b1 <= 0) break;  // (the tile ends before its first block)
                }
                x.blocks = min(x.b1, max(0, (x.u.high - x.u.key0 + kTileKeys - 1) / kTileKeys));
                x.whole = x.b0 == 0 && x.b1 == x.unit_blocks, x.ran = ran;
                x.two = x.u.rows > 128;
                const int pos0 = x.u.context - x.u.n + x.u.row0 / group, pos1 = x.u.context - x.u.n + (x.u.row0 + x.u.rows - 1) / group;
                x.all_hi = p.causal ? min(x.u.context, pos0 + 1) : x.u.context;
                x.all_lo = first_seen(p, pos1);
                role(x);
                tc_fence_before_sync();
                __syncthreads();
                tc_fence_after_sync();
                if (ctl->stopped) {
                    if (tid == 0) {
                        note[0] = x.tile + 1, note[1] = by_unit ? ctl->end : max(x.unit0 + kUnitCost + ctl->end - x.line0, 0), note[2] = ctl->end > x.b0;
                        atomicCAS(blp.stop_index, -1, blp.kernel_id);
                    }
                    return;
                }
                if (!x.whole) {
                    const int first = x.unit0 + kUnitCost, t0 = cut.tile_of(first), t1 = cut.tile_of(first + x.unit_blocks - 1);
                    if (tid == 0) {
                        __threadfence();
                        ctl->last = atomicAdd(&p.counters[t0], 1) == t1 - t0;
                    }
                    __syncthreads();
                    if (ctl->last) {
                        join(x, t0, t1);
                        if (tid == 0) p.counters[t0] = 0;
                    }
                }
                if (*abort_flag) return;
                // ---- the next unit of the tile
                x.unit0 += on_line(x.u);
                ran = true;
                if (x.unit0 >= line1) break;
                at = x.unit0, x.goes_on = false;
                if (++rb == rb_count) {
                    rb = 0;
                    if (++head == p.kv_heads) {
                        head = 0;
                        do ++s;
                        while (prefix[s + 1] == prefix[s]);
                        rb_count = lay.row_blocks(p.batch.first[s + 1] - p.batch.first[s]);
                    }
                }
                if (tid == 0) ctl->end = 0x7fffffff, ctl->saw_nan = 0;
                __syncthreads();
            }
            __syncthreads();
        }
    };
    auto nothing = [](const Piece &, int, int) {};
    uint32_t n_raw = 0, n_keys = 0, n_values = 0, n_s = 0, n_p[2] = {0, 0};  // rounds of the barriers so far
    auto ended = [&](int j) { return j >= *(volatile int *)&ctl->end || *abort_flag; };

    // ---- fetches
    auto fetch = [&](const Piece &x) {
        const Unit &u = x.u;
        const int per_page = min(page_tokens, 64), pieces = kTileKeys / per_page, batch = 32 / pieces;
        bool stop = false;
        int j = x.done;
        for (; j < x.blocks && !stop; j += batch) {
            const int mine = lane / pieces, sub = lane - mine * pieces;
            const int key = x.key(j + mine) + sub * per_page;
            int row = -1;
            float ks = 1.f, vs = 1.f;
            // (what ends below the keys that are seen may be anybody's by now)
            if (j + mine < x.blocks && key < u.high && key + per_page > u.low) {
                const int page = p.batch.table[(size_t)u.s * p.batch.table_ld + (key >> p.page_shift)];
                if ((unsigned)page < (unsigned)p.pages) {
                    const long long block = (long long)page * p.kv_heads + u.head;
                    row = (int)((block << p.page_shift) + (key & (page_tokens - 1)));
                    ks = p.k_scale[block], vs = p.v_scale[block];
                } else {
                    lm_fail(p.error, LM_BAD_PAGE, u.s);
                }
            }
            const int some = min(batch, x.blocks - j);
            for (int b = 0; b < some; ++b) {
                // (a launch runs one block at least, so that whoever is interrupted without end comes to an end)
                if (dynamic && (x.ran || j + b > x.done)) {
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
                    const uint32_t full = smem_u32(&ctl->raw_full[st]);
                    // (ahead of the stage's arrival, which waits for the scales: it cannot complete before)
                    if (loads) tma_load_2d(base + Cfg::kRawAt + st * Cfg::kCodes + sub * per_page * D, i ? &p.map_v : &p.map_k, full, 0, row);
                    if (i == 0 && mine == b)
                        for (int w = sub * per_page / 16; w < (sub + 1) * per_page / 16; ++w)
                            ctl->scales[(j + b) & 3][w][0] = ks, ctl->scales[(j + b) & 3][w][1] = vs;
                    __syncwarp();
                    if (lane == 0) mbar_arrive_expect_tx(full, bytes);
                    __syncwarp();
                    ++n_raw;
                }
            }
        }
        // the end of the piece goes through the ring like a block's keys
        j = stop ? j : max(x.done, x.blocks);
        const int st = n_raw % kRawStages;
        wait(&ctl->raw_empty[st], (n_raw / kRawStages & 1) ^ 1);
        if (lane == 0) {
            ctl->end = j;
            mbar_arrive(smem_u32(&ctl->raw_full[st]));
        }
        __syncwarp();
        ++n_raw;
    };

    // ---- issues the products
    auto multiply = [&](const Piece &x) {
        constexpr uint32_t idesc_s = make_idesc_f16_f32(128, kTileKeys);
        constexpr uint32_t idesc_o = make_idesc_f16_f32(128, D) | (1u << 16);  // B is MN-major: value rows are keys
        auto commit = [&](unsigned long long *bar) {
            if (elected) mma_commit(smem_u32(bar));
            __syncwarp();
        };
        // the queries are there once their warpgroups have arrived for the first time
#pragma unroll
        for (int w = 0; w < 2; ++w)
            if (w == 0 || x.two) wait(&ctl->p_full[w], n_p[w]++ & 1);
        for (int j = x.done;; ++j) {
            // scores of block j, the products with the values of block j - 1 before them
            const int keys = n_keys % kKeyBuffers;
            wait(&ctl->keys_full[keys], n_keys / kKeyBuffers & 1);
            ++n_keys;
            tc_fence_after_sync();
            const bool ends = ended(j), has_values = j > x.done;
            const int buffer = n_values % kValueBuffers;
            if (has_values) wait(&ctl->values_full[buffer], n_values / kValueBuffers & 1);
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                if (w == 1 && !x.two) break;
                if (has_values) {
                    wait(&ctl->p_full[w], n_p[w]++ & 1);
                    tc_fence_after_sync();
                    if (elected && !*abort_flag) {
                        const uint64_t dv = (make_smem_desc_sw128(base + Cfg::kValuesAt + buffer * Cfg::kHalves) & ~(0x3fffull << 16)) |
                                            ((uint64_t)(kHalfTile >> 4) << 16);
                        const uint32_t t_o = tmem + w * 256 + 128;
                        const bool fresh = j - 1 == x.b0;  // (a piece that goes on has its sums in place)
#pragma unroll
                        for (int k = 0; k < kTileKeys / 16; ++k)
                            mma_f16_ts(t_o, tmem + w * 256 + 8 * k, dv + 128 * k, idesc_o, fresh && k == 0 ? 0u : 1u);
                    }
                    __syncwarp();
                }
                if (!ends) {
                    if (elected && !*abort_flag) {
                        const uint64_t dq = make_smem_desc_sw128(base + w * Cfg::kQ), dk = make_smem_desc_sw128(base + Cfg::kKeysAt + keys * Cfg::kHalves);
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            const uint32_t step = (k & 3) * 2 + (k >> 2) * (kHalfTile >> 4);
                            mma_f16_ss(tmem + w * 256, dq + step, dk + step, idesc_s, k > 0 ? 1u : 0u);
                        }
                    }
                    __syncwarp();
                }
                commit(&ctl->s_full[w]);
            }
            if (has_values) {
                commit(&ctl->values_empty[buffer]);
                ++n_values;
            }
            commit(&ctl->keys_empty[keys]);
            if (ends) break;
        }
    };

    // ---- turns codes into halves: a thread a key
    auto convert = [&](const Piece &x) {
        const Unit &u = x.u;
        const int r = tid - 256;
        // the largest scale of the values of the piece
        float most = 0.f;
        for (int i = (max(x.key(x.b0), u.low) >> p.page_shift) + r; (i << p.page_shift) < min(u.high, x.key(x.b1)); i += 128) {
            const int page = p.batch.table[(size_t)u.s * p.batch.table_ld + i];
            if ((unsigned)page < (unsigned)p.pages) most = fmaxf(most, p.v_scale[(long long)page * p.kv_heads + u.head]);
        }
        most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
        if (lane == 0) ctl->largest[wid - 8] = most;
        asm volatile("bar.sync 3, 128;" ::: "memory");
        most = largest_scale();
        // sixteen codes of a piece of a row to two pieces of a row of halves
        auto from_at = [&](const unsigned char *from, int c) {
            return *reinterpret_cast<const uint4 *>(from + (D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4)));
        };
        auto put = [&](unsigned char *to, int c, const uint4 &w, bool scaled, __half2 factor) {
            const uint32_t in[4] = {w.x, w.y, w.z, w.w};
            uint32_t out[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                out[2 * i] = e4m3x2_to_f16x2((unsigned short)in[i]), out[2 * i + 1] = e4m3x2_to_f16x2((unsigned short)(in[i] >> 16));
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
        constexpr int kPieces = D / 16, kBatch = 4;
        auto rows = [&](const unsigned char *from, unsigned char *to) {
#pragma unroll
            for (int c0 = 0; c0 < kPieces; c0 += kBatch) {
                uint4 w[kBatch];
#pragma unroll
                for (int c = 0; c < kBatch; ++c) w[c] = from_at(from, c0 + c);
#pragma unroll
                for (int c = 0; c < kBatch; ++c) put(to, c0 + c, w[c], false, __half2());
            }
        };
        for (int j = x.done;; ++j) {
            int st = n_raw % kRawStages;
            wait(&ctl->raw_full[st], n_raw / kRawStages & 1);
            const bool ends = ended(j);
            // by groups of sixteen keys; a scale 2^40 below the largest counts as that, or its keys would vanish from the
            // normaliser, and the rest goes into the values
            if (!ends && r < 8) {
                const float used = fmaxf(fmaxf(ctl->scales[j & 3][r][1], 1.17549435e-38f) / most, 9.094947e-13f);
                ctl->scales[j & 3][r][2] = log2f(used), ctl->scales[j & 3][r][3] = 1.f / used;
            }
            const int keys = n_keys % kKeyBuffers;
            wait(&ctl->keys_empty[keys], (n_keys / kKeyBuffers & 1) ^ 1);
            ++n_keys;
            if (!ends) {
                rows(smem + Cfg::kRawAt + st * Cfg::kCodes, smem + Cfg::kKeysAt + keys * Cfg::kHalves);
                fence_proxy_async();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ctl->raw_empty[st])), mbar_arrive(smem_u32(&ctl->keys_full[keys]));
            ++n_raw;
            if (ends) break;
            st = n_raw % kRawStages;
            const int buffer = n_values % kValueBuffers;
            wait(&ctl->raw_full[st], n_raw / kRawStages & 1);
            wait(&ctl->values_empty[buffer], (n_values / kValueBuffers & 1) ^ 1);
            const unsigned char *from = smem + Cfg::kRawAt + st * Cfg::kCodes;
            unsigned char *to = smem + Cfg::kValuesAt + buffer * Cfg::kHalves;
            const float scale = ctl->scales[j & 3][r >> 4][1];
            const bool tiny = scale < most * 9.094947e-13f;
            if (x.border(j) || __any_sync(0xffffffffu, tiny)) {
                // (values of keys that not every row sees: no NaN among them may reach a row that does not)
                const bool sanitise = x.border(j);
                const int key = x.key(j) + r;
                const bool drop = key >= u.high || key < u.low;
                const __half2 factor = __float2half2_rn(tiny ? fmaxf(scale, 1.17549435e-38f) / most * 1.099511628e12f : 1.f);
#pragma unroll 1
                for (int c = 0; c < kPieces; ++c) {
                    uint4 w = from_at(from, c);
                    if (drop) w = make_uint4(0, 0, 0, 0);
                    if (sanitise) {
                        const uint4 nan = make_uint4(nan_bytes(w.x), nan_bytes(w.y), nan_bytes(w.z), nan_bytes(w.w));
                        if (nan.x | nan.y | nan.z | nan.w) ctl->saw_nan = 1;
                        w = make_uint4(w.x & ~nan.x, w.y & ~nan.y, w.z & ~nan.z, w.w & ~nan.w);
                    }
                    put(to, c, w, true, factor);
                }
            } else {
                rows(from, to);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ctl->raw_empty[st])), mbar_arrive(smem_u32(&ctl->values_full[buffer]));
            ++n_raw, ++n_values;
        }
    };

    // ---- softmax: a thread a row
    auto softmax = [&](const Piece &x) {
        const Unit &u = x.u;
        const int w = wid >> 2, row = tid & 127, r = w * 128 + row;
        if (w == 1 && !x.two) return;
        const bool live = r < u.rows;
        const uint32_t t_s = tmem + w * 256 + ((uint32_t)((wid & 3) * 32) << 16), t_o = t_s + 128;
        const int row_at = u.row0 + min(r, u.rows - 1);
        const long long token = u.first + row_at / group;
        const int q_head = u.head * group + row_at % group;
        float factor = 1.f;
        {
            // the row's queries, as halves, into the swizzled operand
            unsigned char *to = smem + w * Cfg::kQ + row * 128;
            uint4 v[D / 8];
            {
                const Rows at(base + w * Cfg::kQ, wid, lane);
                const long long own = token * p.q_ld + (long long)q_head * D;
                // (rows past the last have its queries: with a condition, each load waited for the one before)
#pragma unroll
                for (int i = 0; i < Rows::kLanes; ++i) {
                    const long long from = __shfl_sync(0xffffffffu, own, at.first + i);
                    v[i] = reinterpret_cast<const uint4 *>(p.q + from)[at.piece];
                }
#pragma unroll
                for (int i = 0; i < Rows::kLanes; ++i) st_shared_v4(at.in_operand(i), v[i]);
                __syncwarp();
            }
            if (!HALF) {
#pragma unroll
                for (int c = 0; c < D / 8; ++c) v[c] = *reinterpret_cast<const uint4 *>(to + (c >> 3) * kHalfTile + (((c & 7) ^ (row & 7)) << 4));
            }
            float inv = 1.f;
            if (!HALF) {
                uint32_t most = 0;
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    const uint32_t e[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) most = max(most, max(e[i] << 16 & 0x7fffffffu, e[i] & 0x7fff0000u));
                }
                factor = query_factor(most);
                inv = 1.0f / factor;
            }
#pragma unroll
            for (int c = 0; !HALF && c < D / 8; ++c) {
                uint32_t e[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) e[i] = pack_halves(__uint_as_float(e[i] << 16) * inv, __uint_as_float(e[i] & 0xffff0000u) * inv);
                *reinterpret_cast<uint4 *>(to + (c >> 3) * kHalfTile + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(e[0], e[1], e[2], e[3]);
            }
        }
        const float mult = factor * p.scale * 1.4426950408889634f;
        const int pos = u.context - u.n + row_at / group;
        const int hi = p.causal ? min(u.context, pos + 1) : u.context, lo = first_seen(p, pos);
        float m = -INFINITY, l = 0.f;
        if (x.goes_on) {
            // an interrupted piece goes on
            m = __ldcg(spill + r), l = __ldcg(spill + kTileRows + r);
            const float4 *from = reinterpret_cast<const float4 *>(spill + 2 * kTileRows) + r;
#pragma unroll
            for (int c = 0; c < D; c += 16) {
                uint32_t o[16];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 y = __ldcg(from + (c / 4 + i) * kTileRows);
                    o[4 * i] = __float_as_uint(y.x), o[4 * i + 1] = __float_as_uint(y.y), o[4 * i + 2] = __float_as_uint(y.z), o[4 * i + 3] = __float_as_uint(y.w);
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
        int j = x.done;
        for (;; ++j) {
            wait(&ctl->s_full[w], n_s++ & 1);
            __syncwarp();
            tc_fence_after_sync();
            if (ended(j)) break;  // (no scores, but the last products are complete)
            const float4 *of = reinterpret_cast<const float4 *>(ctl->scales[j & 3]);  // (by groups of sixteen keys)
            const bool masks = x.border(j);
            const int high = hi - x.key(j), low = lo - x.key(j);
            auto hides = [&](int i) { return i >= high || i < low; };
            // the largest exponent of the row in this block
            auto largest = [&]() {
                float most = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t v[32];
                    tmem_ld_32x32(t_s + 32 * c, v);
                    tmem_ld_wait();
                    if (masks) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (hides(32 * c + i)) v[i] = 0xff800000u;
                    }
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const float4 g = of[2 * c + q];
                        // (of keys that are all hidden -infinity, or not a number, which is no maximum either)
                        float e = __uint_as_float(v[16 * q]);
#pragma unroll
                        for (int i = 1; i < 16; ++i) e = fmaxf(e, __uint_as_float(v[16 * q + i]));
                        most = fmaxf(most, fmaf(e, g.x * mult, g.z));
                    }
                }
                return most;
            };
            uint32_t h[64];
            float sum, plain;  // of the factors as the normaliser and as the operand has them
            // careful: keys may be masked, and the exponents are rounded as largest() rounds them before the reference is taken off
            auto exponentials = [&](auto careful) {
                const float ref = m == -INFINITY ? 0.f : m;
                sum = plain = 0.f;
                uint32_t both[2][32];
                tmem_ld_32x32(t_s, both[0]);
                float4 next[2] = {of[0], of[1]};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t(&v)[32] = both[c & 1];
                    const float4 g[2] = {next[0], next[1]};
                    tmem_ld_wait();
                    if (c < 3) {
                        // (on its way under this one's exponentials)
                        tmem_ld_32x32(t_s + 32 * (c + 1), both[(c + 1) & 1]);
                        next[0] = of[2 * c + 2], next[1] = of[2 * c + 3];
                    }
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const float less = decltype(careful)::value ? g[q].z : g[q].z - ref;
                        const float2 by = make_float2(g[q].x * mult, g[q].x * mult), plus = make_float2(less, less);
                        float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                        for (int i = 8 * q; i < 8 * q + 8; ++i) {
                            float2 y = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), by, plus);
                            // (hidden behind the factor, which may be as small as zero: that times -infinity is not a number)
                            if (decltype(careful)::value) y.x = hides(32 * c + 2 * i) ? -INFINITY : y.x - ref, y.y = hides(32 * c + 2 * i + 1) ? -INFINITY : y.y - ref;
                            const float2 e = make_float2(lm_ex2(y.x), lm_ex2(y.y));
                            part[i & 1] = add2(part[i & 1], e);
                            h[16 * c + i] = pack_halves(e.x, e.y);
                        }
                        const float all = (part[0].x + part[0].y) + (part[1].x + part[1].y);
                        plain += all, sum = fmaf(all, g[q].w, sum);
                    }
                }
            };
            // The maximum of the first block that a row sees gives its first reference.  Later ones are not asked for theirs: where
            // the factors of a row sum to kMostFactors at most none has left the range of a half.
            if (__any_sync(0xffffffffu, m == -INFINITY)) {
                const float most = largest();
                if (m == -INFINITY) m = reference_of(most);
            }
            // (Exponents of 2^20 and more are rounded first throughout: one sum with the reference would leave the largest off 0 by
            // up to 2^-24 of itself, which can be more than the range of a half.  So it is where the pass is repeated.)
            const bool large = __any_sync(0xffffffffu, fabsf(m) > 1048576.f && m != -INFINITY);
            for (int pass = 0;; ++pass) {
                if (pass || masks || large) exponentials(std::true_type());
                else exponentials(std::false_type());
                // (once is enough, unless a page's scale is not positive, which is no reason to go on without end)
                if (pass || !__any_sync(0xffffffffu, plain > kMostFactors)) break;
                // (the scores' arrival means that the products before them are complete)
                const float now = fmaxf(m, reference_of(largest())), f = now == -INFINITY ? 1.f : lm_ex2(m - now);
#pragma unroll 1
                for (int c = 0; j > x.b0 && c < D; c += 32) {
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
#pragma unroll
            for (int c = 0; c < 2; ++c) tmem_st_32x32(t_s + 32 * c, reinterpret_cast<uint32_t(&)[32]>(h[32 * c]));
            l += sum;
            tmem_st_wait();
            arrive();
        }
        __syncwarp();
        // ---- the end: a whole unit's rows are finished, a part or an unfinished piece goes to the context
        const bool any = j > x.b0;  // products have been made
        const float unit = largest_scale();
        const bool unfinished = ctl->stopped != 0;
        // elements whose values were NaN for a key that this row sees, in blocks that they were taken out of
        uint32_t nan[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) nan[i] = 0;
        if (ctl->saw_nan && live) {
            for (int key = max(lo, x.key(x.done)); key < min(hi, x.key(j)); ++key) {
                if (!x.border((key - u.key0) / kTileKeys)) continue;
                const int page = p.batch.table[(size_t)u.s * p.batch.table_ld + (key >> p.page_shift)];
                if ((unsigned)page >= (unsigned)p.pages) continue;
                const uint4 *code = reinterpret_cast<const uint4 *>(p.v_codes + ((((long long)page * p.kv_heads + u.head) << p.page_shift) + (key & (page_tokens - 1))) * D);
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const uint4 a = code[2 * i], b = code[2 * i + 1];
                    const uint32_t e[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t y = nan_bytes(e[k]);
                        nan[i] |= ((y & 1u) | (y >> 7 & 2u) | (y >> 14 & 4u) | (y >> 21 & 8u)) << (4 * k);
                    }
                }
            }
        }
        const bool to_context = unfinished || !x.whole;
        float *slot = unfinished ? spill : p.parts + (size_t)(2 * x.tile + (x.unit0 + kUnitCost + x.b0 > x.line0 ? 1 : 0)) * Cfg::kSlot;
        // (a row without keys is zero; one whose keys all score -infinity is not a number, as the formula says)
        const bool empty = hi <= 0;
        const float inv = empty ? 0.f : unit / l;
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
                // (unfinished sums stay in their unit, a part's are in none)
                const float f = unfinished ? 1.f : unit;
                float4 *to = reinterpret_cast<float4 *>(slot + 2 * kTileRows) + r;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    to[(c / 4 + i) * kTileRows] = make_float4(__uint_as_float(o[4 * i]) * f, __uint_as_float(o[4 * i + 1]) * f,
                                                              __uint_as_float(o[4 * i + 2]) * f, __uint_as_float(o[4 * i + 3]) * f);
            } else {
                // (to where the queries were, which no product reads any more)
                uint32_t h[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    h[i] = empty ? 0u : pack_out<HALF>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
                unsigned char *to = smem + w * Cfg::kQ + (c >> 6) * kHalfTile + row * 128;
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    *reinterpret_cast<uint4 *>(to + (((c / 8 + i) & 7) ^ (row & 7)) * 16) = make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
            }
        }
        if (!to_context) {
            __syncwarp();
            const Rows at(base + w * Cfg::kQ, wid, lane);
            const long long own = live ? token * p.out_ld + (long long)q_head * D : -1;
#pragma unroll
            for (int i = 0; i < Rows::kLanes; ++i) {
                const long long to = __shfl_sync(0xffffffffu, own, at.first + i);
                const uint4 v = ld_shared_v4(at.in_operand(i));
                if (to >= 0) reinterpret_cast<uint4 *>(p.out + to)[at.piece] = v;
            }
        }
        if (to_context) {
            slot[r] = m, slot[kTileRows + r] = l;
            __threadfence();
        } else if (live && p.lse) {
            p.lse[token * p.heads + q_head] = empty ? -INFINITY : (m == -INFINITY ? m : m * 0.69314718055994531f) + logf(l);
        }
    };

    // ---- the parts of a unit as one, in the order of the line: a thread a row
    auto join = [&](const Piece &x, int t0, int t1) {
        const Unit &u = x.u;
        const int r = tid;
        if (r >= u.rows) return;
        __threadfence();
        const int row_at = u.row0 + r;
        const long long token = u.first + row_at / group;
        const int q_head = u.head * group + row_at % group;
        const int slot0 = 2 * t0 + (x.unit0 + kUnitCost > cut.begin(t0) ? 1 : 0), parts = t1 - t0 + 1;
        auto slot_of = [&](int q) { return p.parts + (size_t)(q == 0 ? slot0 : 2 * (t0 + q)) * Cfg::kSlot; };
        float m = -INFINITY, l = 0.f;
        for (int q = 0; q < parts; ++q) m = fmaxf(m, __ldcg(slot_of(q) + r));
        const float ref = m == -INFINITY ? 0.f : m;
        for (int q = 0; q < parts; ++q) l = fmaf(__ldcg(slot_of(q) + kTileRows + r), lm_ex2(__ldcg(slot_of(q) + r) - ref), l);
        const int pos = u.context - u.n + row_at / group;
        const bool empty = (p.causal ? min(u.context, pos + 1) : u.context) <= 0;
        const float inv = empty ? 0.f : 1.0f / l;
        uint32_t *out = reinterpret_cast<uint32_t *>(p.out + token * p.out_ld + (long long)q_head * D);
        for (int c = 0; c < D / 4; c += 8) {
            float4 y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int q = 0; q < parts; ++q) {
                const float f = lm_ex2(__ldcg(slot_of(q) + r) - ref);
                const float4 *from = reinterpret_cast<const float4 *>(slot_of(q) + 2 * kTileRows) + r;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 z = __ldcg(from + (c + i) * kTileRows);
                    y[i].x = fmaf(z.x, f, y[i].x), y[i].y = fmaf(z.y, f, y[i].y), y[i].z = fmaf(z.z, f, y[i].z), y[i].w = fmaf(z.w, f, y[i].w);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                uint32_t h[4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    h[2 * e] = empty ? 0u : pack_out<HALF>(y[i + e].x * inv, y[i + e].y * inv);
                    h[2 * e + 1] = empty ? 0u : pack_out<HALF>(y[i + e].z * inv, y[i + e].w * inv);
                }
                *reinterpret_cast<uint4 *>(out + 2 * (c + i)) = make_uint4(h[0], h[1], h[2], h[3]);
            }
        }
        if (p.lse) p.lse[token * p.heads + q_head] = empty ? -INFINITY : (m == -INFINITY ? m : m * 0.69314718055994531f) + logf(l);
    };

    if (wid < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegs));
        walk(softmax, join);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
        if (wid < 12) walk(convert, nothing);
        else if (wid == 12) walk(multiply, nothing);
        else if (wid == 13) walk(fetch, nothing);
        else walk([](const Piece &) {}, nothing);
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
        const size_t smem = 1024 + fixed + sizeof(ManyCtl);
        int per_sm;
        const cudaError_t e = lm_resident((const void *)kernel, kManyThreads, smem, smem, d.device, &per_sm);
        if (e != cudaSuccess) return e;
        p.max_tiles = (int)std::min<size_t>(kLmCounters - kNotes, kLmPartsBytes / ((size_t)slot * sizeof(float)));
        // (two parts a tile at most, and an unfinished one)
        const int grid = std::min({d.sm_count, kNotes / 4, p.max_tiles / 3});
        return launch_layer(kernel, grid, kManyThreads, smem, s, p, blp);
    };
    if (dim == 64)
        return half ? go(kv_attend_many_kernel<64, true>, ManyCfg<64>::kCtlAt, ManyCfg<64>::kSlot)
                    : go(kv_attend_many_kernel<64, false>, ManyCfg<64>::kCtlAt, ManyCfg<64>::kSlot);
    return half ? go(kv_attend_many_kernel<128, true>, ManyCfg<128>::kCtlAt, ManyCfg<128>::kSlot)
                : go(kv_attend_many_kernel<128, false>, ManyCfg<128>::kCtlAt, ManyCfg<128>::kSlot);
}

}  // namespace gpx
