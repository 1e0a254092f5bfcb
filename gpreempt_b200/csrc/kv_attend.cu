// Attention of new tokens over a paged 8-bit cache, for few rows a head of keys (single tokens, a few proposed ones).
//
//   s_rj = scale q_r . k_j k_scale(page of j),   o_r = sum_j e^(s_rj - lse_r) v_j v_scale(page of j)
//
// Bound by memory: a key and its value are 2 D bytes, read once, against 4 D operations a row.  The rows of one head of
// keys (its group's heads, times the tokens) are the N side of the tensor instructions and the keys the M side, so that
// eight rows waste nothing:  S^T[16 keys][8 rows] = K Q^T,  O^T[D][8 rows] += V^T[D][16 keys] P^T[16 keys][8 rows].
// Codes go from shared memory to registers as they are and become halves there (every e4m3 number is one): a lane's
// operand elements are contiguous bytes, because the order of a contraction's index is free as long as both sides
// agree on it, and a transposed operand only has to pair the bytes of two keys.  Queries become halves after a power
// of two that brings their row's largest to 1; the scores' factors (that power, the page's scale, scale, log2 e) are
// applied to the sums.
//
// The values' scales join the exponents: what multiplies a code is 2^14 2^(s_rj + b_j - M_r), b_j = log2 v_scale, with M the running
// maximum of s + b, so that none that counts leaves the range of a half, however far apart the scales of pages are, nor does the sum of
// thousands of keys that weigh 2^-26 each beside one that weighs 1 (a half ends at 2^-25 below and 2^16 above); the normaliser adds it times 2^(B - b_j), with B the largest b so far, and is brought to the new B
// when that grows (a page of zeros has the smallest scale there is: sums that count in a first page's scale vanish behind it).  Factors of fp16 results go through the tensor cores in
// two halves (22 bits), those of bf16 results in one (11 bits against the result's 8).  Statistics and sums are float.
//
// Four warps take sixteen keys each of a block of 64, with a running maximum and output of their own, and are merged
// at the end of a unit (a sequence, a head of keys, a block of rows); a fifth keeps the ring of blocks full by TMA,
// with the table's entries and the scales a batch of blocks ahead.
//
// Measured, 32 heads of 128 on 8, bf16: single tokens of 64 sequences over 16 384 keys at most 195 us (5.9 TB/s of 6.5 that a
// copy reaches), of one over 131 071 keys 54.5 (4.9 TB/s: 148 SMs begin and end together, and the parts' join is 5 600 cycles),
// five of 16 over 2 000 21.9, of one over 517 9.1, a chain of 16 000 cycles from the sums over the sequences to the join.
//
// Work is cut evenly, whatever the sequences' lengths: the blocks of all units lie on one line, and a tile is
// an equal piece of it.  A unit that spans several tiles leaves their parts in the context, and the
// CTA that brings the last one joins them in the order of the line.
#include "kv_attend.h"
#include "sm100.cuh"

#include <algorithm>

namespace gpx {

using namespace sm100;

constexpr int kAttWarps = 4, kAttConsumers = 32 * kAttWarps, kAttThreads = kAttConsumers + 32;
constexpr int kAttKeys = 64;
constexpr float kLift = 16384.f;  // of the factors as operands
constexpr int kSumBlocks = 16;
constexpr unsigned long long kAttWaitNs = 2000000000ull;

template <int D, int NT>
struct AttCfg {
    static constexpr int kStages = D == 128 ? 4 : 8;
    static constexpr uint32_t kTile = kAttKeys * D;          // bytes of a block's keys, or values
    static constexpr uint32_t kRing = kStages * 2 * kTile;   // 64 KiB
    static constexpr int kSteps = D / 16;
    static constexpr uint32_t kQ = NT * kSteps * 32 * 8;
    static constexpr uint32_t kMerge = 2 * 8 * NT * D * 4;
    static constexpr uint32_t kFixed = 1024 + kRing + kQ + kMerge;
    static constexpr int kRows = 8 * NT;
};

template <int NT>
struct AttCtl {
    unsigned long long full[8], empty[8];
    float scales[8][4][2];  // of a stage's sixteen keys of each warp: keys' scale, log2 of the values'
    float row_factor[8 * NT];
    float ml[kAttWarps][8 * NT][2];
    int tile, last, abort_flag;
};

// The order in which the eight key rows of an operand tile are taken: with it neither the reads of keys (two
// rows, four pieces a phase) nor of values (four rows, two pieces) meet in a bank.
__device__ __forceinline__ int key_row(int r) { return (r & 1) ? ((r & 6) ^ 4) | 1 : r; }

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ uint4 lds_u4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds_u2(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
template <int D, int NT, bool HALF>
__global__ void __launch_bounds__(kAttThreads)
kv_attend_kernel(const __grid_constant__ AttendParams p, BlpArgs blp) {
    using Cfg = AttCfg<D, NT>;
    constexpr int S = Cfg::kStages, KS = Cfg::kSteps, MT = D / 16, ROWS = Cfg::kRows;
    constexpr bool kTwo = HALF;  // probabilities in two halves
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint2 *q_frag = reinterpret_cast<uint2 *>(smem + Cfg::kRing);
    float4 *merge = reinterpret_cast<float4 *>(smem + Cfg::kRing + Cfg::kQ);
    AttCtl<NT> *ctl = reinterpret_cast<AttCtl<NT> *>(smem + Cfg::kRing + Cfg::kQ + Cfg::kMerge);
    int *prefix = reinterpret_cast<int *>(ctl + 1);  // [seqs + 1]
    volatile int *abort_flag = &ctl->abort_flag;
    const uint32_t ring = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, wid = __shfl_sync(0xffffffffu, tid >> 5, 0);
    if (tid == 0) {
        for (int i = 0; i < S; ++i) mbar_init(smem_u32(&ctl->full[i]), 1), mbar_init(smem_u32(&ctl->empty[i]), kAttWarps);
        ctl->abort_flag = 0;
        fence_barrier_init();
        fence_proxy_async();
        prefetch_tensormap(&p.map_k), prefetch_tensormap(&p.map_v);
    }
    __syncthreads();
    pdl_enter();
    const bool dynamic = blp.preempted != nullptr;
    if (tid == 0) trace_begin(blp);
    const Layout<ROWS, kAttKeys> lay(p);
    const int group = lay.group, page_tokens = 1 << p.page_shift;
    const int n_line = lm_prefix(prefix, p.batch.seqs, p.error, [&](int s) {
        return lay.line(lm_span(p.batch, s, page_tokens, false, p.error));
    });
    int tiles = dynamic ? max((n_line + p.blocks_a_tile - 1) / p.blocks_a_tile, (int)gridDim.x) : (int)gridDim.x;
    tiles = min(min(tiles, n_line), p.max_tiles);
    blp.total_tiles = tiles;
    const LmCut cut(n_line, tiles);
    auto wait = [&](unsigned long long *bar, uint32_t phase) {
        if (!mbar_wait(smem_u32(bar), phase, abort_flag, kAttWaitNs)) {
            *abort_flag = 1;
            lm_fail(p.error, LM_GAVE_UP, (int)blockIdx.x);
        }
    };
    // The pieces of [begin, end) of the line that belong to one unit each: f(unit, first block, blocks, the unit's
    // first block on the line, its blocks there).
    auto each_piece = [&](int begin, int end, auto &&f) {
        while (begin < end) {
            const int s = lm_find(prefix, p.batch.seqs, begin);
            const LmSpan span = {0, p.batch.first[s + 1] - p.batch.first[s], p.batch.context[s]};
            const int blocks = lay.key_blocks(span);
            const int index = (begin - prefix[s]) / blocks;
            const int unit0 = prefix[s] + index * blocks;
            const int stop = min(end, unit0 + blocks);
            f(lay.unit(s, index), begin - unit0, stop - begin, unit0, blocks);
            begin = stop;
        }
    };
    uint32_t stage = 0, phase = 0;
    auto advance = [&]() {
        if (++stage == S) stage = 0, phase ^= 1;
    };

    int iter = 0;
    for (;; ++iter) {
        int tile;
        if (dynamic) {
            if (tid == 0) ctl->tile = blp_claim(blp, iter);
            __syncthreads();
            tile = ctl->tile;
            __syncthreads();
        } else {
            tile = blp_claim(blp, iter);
        }
        if (tile < 0) break;
        const int line0 = cut.begin(tile), line1 = cut.begin(tile + 1);

        if (wid == kAttWarps) {
            // ---- the ring's filler
            const int per_page = min(page_tokens, kAttKeys);
            const int pieces = kAttKeys / per_page;  // of a block: one page each, or a part of one
            const int batch = 32 / pieces;           // blocks whose table entries and scales are fetched together
            each_piece(line0, line1, [&](const Unit &u, int block0, int blocks, int, int) {
                const int blocks_live = min(blocks, max(0, (u.high - u.key0 + kAttKeys - 1) / kAttKeys - block0));
                for (int b0 = 0; b0 < blocks_live; b0 += batch) {
                    const int mine = lane / pieces, sub = lane - mine * pieces;
                    const int key = u.key0 + (block0 + b0 + mine) * kAttKeys + sub * per_page;
                    int row = -1;
                    float ks = 1.f, vs = 0.f;
                    // (what ends below the keys that are seen may be anybody's by now: neither fetched nor asked for its scale)
                    if (b0 + mine < blocks_live && key < u.high && key + per_page > u.low) {
                        const int page = p.batch.table[(size_t)u.s * p.batch.table_ld + (key >> p.page_shift)];
                        if ((unsigned)page < (unsigned)p.pages) {
                            const long long block = (long long)page * p.kv_heads + u.head;
                            row = (int)((block << p.page_shift) + (key & (page_tokens - 1)));
                            ks = p.k_scale[block], vs = p.v_scale[block];
                        } else {
                            lm_fail(p.error, LM_BAD_PAGE, u.s);
                        }
                    }
                    const int some = min(batch, blocks_live - b0);
                    for (int b = 0; b < some; ++b) {
                        wait(&ctl->empty[stage], phase ^ 1);
                        const bool loads = mine == b && row >= 0;
                        const uint32_t full = smem_u32(&ctl->full[stage]);
                        if (loads) {
                            // (ahead of the stage's arrival, which waits for the scales: it cannot complete before)
                            const uint32_t at = ring + stage * 2 * Cfg::kTile + sub * per_page * D;
                            tma_load_2d(at, &p.map_k, full, 0, row);
                            tma_load_2d(at + Cfg::kTile, &p.map_v, full, 0, row);
                        }
                        if (mine == b) {
                            for (int w = sub * per_page / 16; w < (sub + 1) * per_page / 16; ++w)
                                ctl->scales[stage][w][0] = ks, ctl->scales[stage][w][1] = log2f(fmaxf(vs, 1.17549435e-38f));
                        }
                        const int loading = __popc(__ballot_sync(0xffffffffu, loads));
                        __syncwarp();  // the scales are written before the stage is announced
                        if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)(loading * 2 * per_page * D));
                        __syncwarp();
                        advance();
                    }
                }
            });
        } else {
            // ---- four warps, sixteen keys of a block each
            const int g = lane >> 2, t = lane & 3;
            auto sync = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(kAttConsumers) : "memory"); };
            each_piece(line0, line1, [&](const Unit &u, int block0, int blocks, int unit0, int unit_blocks) {
                const int blocks_live = min(blocks, max(0, (u.high - u.key0 + kAttKeys - 1) / kAttKeys - block0));
                const bool whole = blocks == unit_blocks;
                const int t0 = whole ? tile : cut.tile_of(unit0), t1 = whole ? tile : cut.tile_of(unit0 + unit_blocks - 1);
                // ---- the unit's queries as operands: warp w prepares tiles of eight rows w, w + 4, ...
                for (int nt = wid; nt < NT; nt += kAttWarps) {
                    const int r = nt * 8 + g;
                    uint4 raw[KS];  // two of them sixteen elements of a row
                    const bool live = r < u.rows;
                    const int at = u.row0 + r;
                    const unsigned short *row = p.q + (live ? (u.first + at / group) * p.q_ld + (u.head * group + at % group) * D : 0);
#pragma unroll
                    for (int c = 0; c < KS / 4; ++c)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            raw[2 * c + i] = live ? *reinterpret_cast<const uint4 *>(row + 16 * (t + 4 * c) + 8 * i) : make_uint4(0, 0, 0, 0);
                    float factor = 1.f;
                    uint32_t h[KS][2];
                    if (HALF) {
#pragma unroll
                        for (int k = 0; k < KS; ++k) {
                            const uint4 &w = raw[k >> 1];
                            h[k][0] = k & 1 ? w.z : w.x, h[k][1] = k & 1 ? w.w : w.y;
                        }
                    } else {
                        uint32_t most = 0;
#pragma unroll
                        for (int i = 0; i < KS / 2; ++i) {
                            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) most = max(most, max(w[j] << 16 & 0x7fffffffu, w[j] & 0x7fff0000u));
                        }
                        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
                        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
                        factor = query_factor(most);
                        const float inv = 1.0f / factor;
#pragma unroll
                        for (int k = 0; k < KS; ++k) {
                            const uint4 &w = raw[k >> 1];
                            const uint32_t a = k & 1 ? w.z : w.x, b = k & 1 ? w.w : w.y;
                            h[k][0] = pack_halves(__uint_as_float(a << 16) * inv, __uint_as_float(a & 0xffff0000u) * inv);
                            h[k][1] = pack_halves(__uint_as_float(b << 16) * inv, __uint_as_float(b & 0xffff0000u) * inv);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < KS; ++k) q_frag[(nt * KS + k) * 32 + lane] = make_uint2(h[k][0], h[k][1]);
                    if (t == 0) ctl->row_factor[r] = factor;
                }
                sync();
                uint2 qr[NT == 1 ? KS : 1];
                if (NT == 1) {
#pragma unroll
                    for (int k = 0; k < KS; ++k) qr[k] = q_frag[k * 32 + lane];
                }
                // this lane's columns: rows 8 nt + 2 t and the next
                float mult[NT][2], m[NT][2], l[NT][2], before[NT][2];  // (l: of the last kSumBlocks blocks, before: of those ahead)
                int lo[NT][2], hi[NT][2];
                float o[NT][MT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int r = min(8 * nt + 2 * t + c, u.rows - 1);
                        mult[nt][c] = ctl->row_factor[8 * nt + 2 * t + c] * p.scale * 1.4426950408889634f;
                        m[nt][c] = -INFINITY, l[nt][c] = before[nt][c] = 0.f;
                        const int pos = u.context - u.n + (u.row0 + r) / group;
                        hi[nt][c] = p.causal ? min(u.context, pos + 1) : u.context;
                        lo[nt][c] = first_seen(p, pos);
                    }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int c = 0; c < 4; ++c) o[nt][i][c] = 0.f;
                // keys that every row sees: [all_lo, all_hi)
                const int pos0 = u.context - u.n + u.row0 / group, pos1 = u.context - u.n + (u.row0 + u.rows - 1) / group;
                const int all_hi = p.causal ? min(u.context, pos0 + 1) : u.context;
                const int all_lo = first_seen(p, pos1);
                // log2 of the largest value scale so far, in which the normaliser counts: l is in units of 2^(m - most_b).
                // times = 2^below, with `below` what a block's scale lies below the largest
                float most_b = -INFINITY, below = 0.f, times = 1.f;

                for (int b = 0; b < blocks_live; ++b) {
                    wait(&ctl->full[stage], phase);
                    const uint32_t sk = ring + stage * 2 * Cfg::kTile, sv = sk + Cfg::kTile;
                    const float ks = ctl->scales[stage][wid][0], b_true = ctl->scales[stage][wid][1];
                    const int row16 = wid * 16;
                    const int key0 = u.key0 + (block0 + b) * kAttKeys + row16;
                    // ---- S^T
                    float sc[NT][4];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 4; ++c) sc[nt][c] = 0.f;
                    {
                        const int kr = key_row(g);
                        uint4 ka[KS / 4], kb[KS / 4];
#pragma unroll
                        for (int c = 0; c < KS / 4; ++c) {
                            const int piece = t + 4 * c;
                            const uint32_t at = D == 128 ? (row16 + kr) * 128 + ((piece ^ (kr & 7)) << 4)
                                                         : (row16 + kr) * 64 + ((piece ^ ((kr >> 1) & 3)) << 4);
                            ka[c] = lds_u4(sk + at), kb[c] = lds_u4(sk + at + 8 * D);
                        }
                        float odd[4] = {0.f, 0.f, 0.f, 0.f};  // (two chains of sums where there is one tile of rows)
#pragma unroll
                        for (int k = 0; k < KS; ++k) {
                            const uint4 &A = ka[k >> 2], &B = kb[k >> 2];
                            const uint32_t wa = (k & 3) == 0 ? A.x : (k & 3) == 1 ? A.y : (k & 3) == 2 ? A.z : A.w;
                            const uint32_t wb = (k & 3) == 0 ? B.x : (k & 3) == 1 ? B.y : (k & 3) == 2 ? B.z : B.w;
                            const uint32_t a0 = e4m3x2_to_f16x2((unsigned short)wa), a2 = e4m3x2_to_f16x2((unsigned short)(wa >> 16));
                            const uint32_t a1 = e4m3x2_to_f16x2((unsigned short)wb), a3 = e4m3x2_to_f16x2((unsigned short)(wb >> 16));
                            if (NT == 1) {
                                mma_16816(k & 1 ? odd : sc[0], a0, a1, a2, a3, qr[NT == 1 ? k : 0].x, qr[NT == 1 ? k : 0].y);
                            } else {
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    const uint2 q = q_frag[(nt * KS + k) * 32 + lane];
                                    mma_16816(sc[nt], a0, a1, a2, a3, q.x, q.y);
                                }
                            }
                        }
                        if (NT == 1)
#pragma unroll
                            for (int c = 0; c < 4; ++c) sc[0][c] += odd[c];
                    }
                    // ---- scores: factors, masks where a row's border lies in the block.  A scale 2^40 below the largest counts
                    // as that (or its keys would vanish from the normaliser) and the rest goes into the operand.
                    if (b_true > most_b) {
                        // (rare, the same for the warp) The sums go to the new unit.  Where that takes a normaliser beyond 2^64, its row's
                        // reference is raised instead: what then leaves the range of the factors is 2^-100 of the row's weight.
                        if (most_b != -INFINITY) {
                            const float d = b_true - most_b;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    float most = l[nt][c] + before[nt][c];
                                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
                                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
                                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
                                    const float raise = fmaxf(log2f(most) + d - 64.f, 0.f), f = lm_ex2(-raise);
                                    m[nt][c] += raise;
                                    const float up = lm_ex2(fminf(d - raise, 126.f));  // (a row without keys so far has no sum, and its d no bound)
                                    l[nt][c] *= up, before[nt][c] *= up;
#pragma unroll
                                    for (int i = 0; i < MT; ++i) o[nt][i][c] *= f, o[nt][i][c + 2] *= f;
                                }
                        }
                        most_b = b_true;
                    }
                    const float b_used = fmaxf(b_true, most_b - 40.f);
                    if (most_b - b_used != below) below = most_b - b_used, times = lm_ex2(below);
                    const int block_key = u.key0 + (block0 + b) * kAttKeys;
                    const bool border = block_key + kAttKeys > all_hi || block_key < all_lo;
                    uint32_t seen = ~0u;  // bit 4 nt + c
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 4; ++c) sc[nt][c] = fmaf(sc[nt][c], mult[nt][c & 1] * ks, b_used);
                    if (border) {
                        const int ka = key0 + key_row(g), kb = ka + 8;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const int key = c < 2 ? ka : kb;
                                if (key >= hi[nt][c & 1] || key < lo[nt][c & 1]) sc[nt][c] = -INFINITY, seen &= ~(1u << (4 * nt + c));
                            }
                    }
                    bool grown = false;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) grown |= fmaxf(sc[nt][c], sc[nt][c + 2]) > m[nt][c];
                    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                float x = fmaxf(sc[nt][c], sc[nt][c + 2]);
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                                const float now = fmaxf(m[nt][c], x);
                                const float f = now == -INFINITY ? 1.f : lm_ex2(m[nt][c] - now);
                                m[nt][c] = now;
                                l[nt][c] *= f, before[nt][c] *= f;
#pragma unroll
                                for (int i = 0; i < MT; ++i) o[nt][i][c] *= f, o[nt][i][c + 2] *= f;
                            }
                    }
                    if (b % kSumBlocks == 0) {
                        // (thousands of blocks that are small beside one of the first would vanish in one sum)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 2; ++c) before[nt][c] += l[nt][c], l[nt][c] = 0.f;
                    }
                    const float p_factor = b_used != b_true ? kLift * lm_ex2(b_true - b_used) : kLift;
                    uint32_t pb[NT][2], pl[kTwo ? NT : 1][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float e[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float ref = m[nt][c & 1] == -INFINITY ? 0.f : m[nt][c & 1];
                            e[c] = lm_ex2(sc[nt][c] - ref);
                        }
                        l[nt][0] = fmaf(e[0] + e[2], times, l[nt][0]), l[nt][1] = fmaf(e[1] + e[3], times, l[nt][1]);
#pragma unroll
                        for (int c = 0; c < 4; ++c) e[c] *= p_factor;
                        const uint32_t a = pack_halves(e[0], e[1]), c = pack_halves(e[2], e[3]);
                        pb[nt][0] = transpose8x8(a), pb[nt][1] = transpose8x8(c);
                        if (kTwo) {
                            const float2 fa = unpack_halves(a), fc = unpack_halves(c);
                            pl[nt][0] = transpose8x8(pack_halves(e[0] - fa.x, e[1] - fa.y));
                            pl[nt][1] = transpose8x8(pack_halves(e[2] - fc.x, e[3] - fc.y));
                        }
                    }
                    // ---- O^T += V^T P^T: a lane has the elements g D / 8 .. of keys key_row(2 t), key_row(2 t + 1), and those + 8
                    uint32_t v[4][D / 32];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int kr = key_row(2 * t + (x & 1)), row = row16 + kr + (x >> 1) * 8;
                        if (D == 128) {
                            const uint4 w = lds_u4(sv + row * 128 + ((g ^ (kr & 7)) << 4));
                            v[x][0] = w.x, v[x][1] = w.y, v[x][D / 32 - 2] = w.z, v[x][D / 32 - 1] = w.w;
                        } else {
                            const uint2 w = lds_u2(sv + row * 64 + (((g >> 1) ^ ((kr >> 1) & 3)) << 4) + (g & 1) * 8);
                            v[x][0] = w.x, v[x][1] = w.y;
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&ctl->empty[stage]));
                    advance();
                    if (border) {
                        // A NaN of a key that a row does not see must not reach it (nothing times NaN is NaN), those that see
                        // it must get it: NaN codes are taken out, counted by a product of their own where any row sees them.
                        uint32_t any = 0;
#pragma unroll
                        for (int x = 0; x < 4; ++x)
#pragma unroll
                            for (int i = 0; i < D / 32; ++i) any |= nan_bytes(v[x][i]);
                        if (__any_sync(0xffffffffu, any != 0)) {
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                auto one = [&](int c) { return seen >> (4 * nt + c) & 1 ? 1.f : 0.f; };
                                const uint32_t s0 = transpose8x8(pack_halves(one(0), one(1))), s1 = transpose8x8(pack_halves(one(2), one(3)));
#pragma unroll
                                for (int i = 0; i < MT; ++i) {
                                    uint32_t a[4];
#pragma unroll
                                    for (int h = 0; h < 2; ++h) {
                                        const uint32_t sel = i & 1 ? 0x7362 : 0x5140;
                                        const uint32_t w = __byte_perm(nan_bytes(v[2 * h][i >> 1]), nan_bytes(v[2 * h + 1][i >> 1]), sel);
                                        // bytes 0, 1: element 2 i of the two keys; 2, 3: element 2 i + 1.  0x3c00 is a half's one.
                                        a[2 * h] = (w & 0xffu ? 0x3c00u : 0u) | (w & 0xff00u ? 0x3c000000u : 0u);
                                        a[2 * h + 1] = (w & 0xff0000u ? 0x3c00u : 0u) | (w & 0xff000000u ? 0x3c000000u : 0u);
                                    }
                                    float count[4] = {0.f, 0.f, 0.f, 0.f};
                                    mma_16816(count, a[0], a[1], a[2], a[3], s0, s1);
#pragma unroll
                                    for (int c = 0; c < 4; ++c)
                                        if (count[c] > 0.f) o[nt][i][c] = __uint_as_float(0x7fffffffu);
                                }
                            }
#pragma unroll
                            for (int x = 0; x < 4; ++x)
#pragma unroll
                                for (int i = 0; i < D / 32; ++i) v[x][i] &= ~nan_bytes(v[x][i]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const uint32_t sel = i & 1 ? 0x7362 : 0x5140;
                        const uint32_t ab = __byte_perm(v[0][i >> 1], v[1][i >> 1], sel), cd = __byte_perm(v[2][i >> 1], v[3][i >> 1], sel);
                        const uint32_t a0 = e4m3x2_to_f16x2((unsigned short)ab), a1 = e4m3x2_to_f16x2((unsigned short)(ab >> 16));
                        const uint32_t a2 = e4m3x2_to_f16x2((unsigned short)cd), a3 = e4m3x2_to_f16x2((unsigned short)(cd >> 16));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma_16816(o[nt][i], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                            if (kTwo) mma_16816(o[nt][i], a0, a1, a2, a3, pl[kTwo ? nt : 0][0], pl[kTwo ? nt : 0][1]);
                        }
                    }
                }

                // ---- the four warps' results as one: warps 2 and 3 into 0 and 1, 1 into 0.  l counts in 2^(m - most_b).
                const float unit = blocks_live ? most_b : 0.f, unit_scale = lm_ex2(unit);  // (and o 2^14 times as much)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) m[nt][c] -= unit;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        l[nt][c] += before[nt][c];
#pragma unroll
                        for (int d = 4; d <= 16; d <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], d);
                        if (g == 0) {
                            ctl->ml[wid][8 * nt + 2 * t + c][0] = m[nt][c];
                            ctl->ml[wid][8 * nt + 2 * t + c][1] = l[nt][c];
                        }
                    }
                sync();
                float most[NT][2], sum[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int r = 8 * nt + 2 * t + c;
                        float mm = ctl->ml[0][r][0];
#pragma unroll
                        for (int w = 1; w < kAttWarps; ++w) mm = fmaxf(mm, ctl->ml[w][r][0]);
                        const float ref = mm == -INFINITY ? 0.f : mm;
                        float all = 0.f;
#pragma unroll
                        for (int w = 0; w < kAttWarps; ++w) all += ctl->ml[w][r][1] * lm_ex2(ctl->ml[w][r][0] - ref);
                        most[nt][c] = mm, sum[nt][c] = all;
                        const float f = lm_ex2(m[nt][c] - ref) * (1.f / kLift);
#pragma unroll
                        for (int i = 0; i < MT; ++i) o[nt][i][c] = o[nt][i][c] * f * unit_scale, o[nt][i][c + 2] = o[nt][i][c + 2] * f * unit_scale;
                    }
#pragma unroll
                for (int round = 2; round >= 1; round >>= 1) {
                    if (wid >= round && wid < 2 * round) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < MT; ++i)
                                merge[(((wid - round) * NT + nt) * MT + i) * 32 + lane] = make_float4(o[nt][i][0], o[nt][i][1], o[nt][i][2], o[nt][i][3]);
                    }
                    sync();
                    if (wid < round) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < MT; ++i) {
                                const float4 x = merge[((wid * NT + nt) * MT + i) * 32 + lane];
                                o[nt][i][0] += x.x, o[nt][i][1] += x.y, o[nt][i][2] += x.z, o[nt][i][3] += x.w;
                            }
                    }
                    sync();
                }
                // ---- a whole unit is finished here, a part goes to the context
                auto finish_row = [&](int r, float mm, float all, float &inv, float &log_sum) {
                    // (a row without keys is zero; one whose keys all score -infinity is not a number, as the formula says)
                    const int pos = u.context - u.n + (u.row0 + r) / group;
                    const int upto = p.causal ? min(u.context, pos + 1) : u.context;
                    const bool empty = upto <= 0;
                    inv = empty ? 0.f : 1.0f / all;
                    log_sum = empty ? -INFINITY : (mm == -INFINITY ? mm : mm * 0.69314718055994531f) + logf(all);
                };
                auto out_row = [&](int r) {
                    const int at = u.row0 + r;
                    return p.out + (u.first + at / group) * p.out_ld + (u.head * group + at % group) * D;
                };
                auto lse_at = [&](int r) {
                    const int at = u.row0 + r;
                    return p.lse + (long long)(u.first + at / group) * p.heads + u.head * group + at % group;
                };
                constexpr int kSlot = ROWS * (D + 2);  // floats: maxima, sums, outputs
                if (wid == 0) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int r = 8 * nt + 2 * t + c;
                            if (r >= u.rows) continue;
                            // elements g D / 8 + 2 i and the next
                            if (whole) {
                                float inv, log_sum;
                                finish_row(r, most[nt][c], sum[nt][c], inv, log_sum);
                                uint32_t w[MT];
#pragma unroll
                                for (int i = 0; i < MT; ++i) {
                                    const float a = o[nt][i][c], b = o[nt][i][c + 2];
                                    w[i] = inv == 0.f ? 0u : pack_out<HALF>(a * inv, b * inv);
                                }
                                uint4 *to = reinterpret_cast<uint4 *>(out_row(r) + g * (D / 8));
#pragma unroll
                                for (int i = 0; i < MT / 4; ++i) to[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                                if (p.lse && g == 0) *lse_at(r) = log_sum;
                            } else {
                                const int slot = 2 * tile + (unit0 + block0 > line0 ? 1 : 0);
                                float *to = p.parts + (size_t)slot * kSlot;
                                if (g == 0) to[r] = most[nt][c], to[ROWS + r] = sum[nt][c];
                                float4 *at = reinterpret_cast<float4 *>(to + 2 * ROWS + r * D + g * (D / 8));
#pragma unroll
                                for (int i = 0; i < MT / 2; ++i)
                                    at[i] = make_float4(o[nt][2 * i][c], o[nt][2 * i][c + 2], o[nt][2 * i + 1][c], o[nt][2 * i + 1][c + 2]);
                            }
                        }
                    if (!whole) {
                        __threadfence();
                        __syncwarp();
                        if (lane == 0) ctl->last = atomicAdd(&p.counters[t0], 1) == t1 - t0;
                    }
                }
                if (whole) {
                    sync();
                    return;
                }
                sync();
                if (ctl->last) {
                    // ---- join the parts in the order of the line: a warp a row, a lane D / 32 elements
                    __threadfence();
                    const int slot0 = 2 * t0 + (unit0 > cut.begin(t0) ? 1 : 0);
                    auto slot_of = [&](int x) { return p.parts + (size_t)(x == t0 ? slot0 : 2 * x) * kSlot; };
                    for (int r = wid; r < u.rows; r += kAttWarps) {
                        float mm = -INFINITY;
                        for (int x = t0 + lane; x <= t1; x += 32) mm = fmaxf(mm, __ldcg(slot_of(x) + r));
#pragma unroll
                        for (int d = 16; d >= 1; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
                        const float ref = mm == -INFINITY ? 0.f : mm;
                        float all = 0.f, acc[D / 32];
#pragma unroll
                        for (int j = 0; j < D / 32; ++j) acc[j] = 0.f;
#pragma unroll 8
                        for (int x = t0; x <= t1; ++x) {
                            const float *from = slot_of(x);
                            const float f = lm_ex2(__ldcg(from + r) - ref);
                            all = fmaf(__ldcg(from + ROWS + r), f, all);
                            const float *at = from + 2 * ROWS + r * D + lane * (D / 32);
                            if (D == 128) {
                                const float4 y = __ldcg(reinterpret_cast<const float4 *>(at));
                                acc[0] = fmaf(y.x, f, acc[0]), acc[1] = fmaf(y.y, f, acc[1]);
                                acc[D / 32 - 2] = fmaf(y.z, f, acc[D / 32 - 2]), acc[D / 32 - 1] = fmaf(y.w, f, acc[D / 32 - 1]);
                            } else {
                                const float2 y = __ldcg(reinterpret_cast<const float2 *>(at));
                                acc[0] = fmaf(y.x, f, acc[0]), acc[1] = fmaf(y.y, f, acc[1]);
                            }
                        }
                        float inv, log_sum;
                        finish_row(r, mm, all, inv, log_sum);
                        uint32_t w[D / 64];
#pragma unroll
                        for (int j = 0; j < D / 64; ++j) w[j] = inv == 0.f ? 0u : pack_out<HALF>(acc[2 * j] * inv, acc[2 * j + 1] * inv);
                        uint32_t *to = reinterpret_cast<uint32_t *>(out_row(r)) + lane * (D / 64);
                        if (D == 128) *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[D / 64 - 1]);
                        else to[0] = w[0];
                        if (p.lse && lane == 0) *lse_at(r) = log_sum;
                    }
                    if (tid == 0) p.counters[t0] = 0;
                }
                sync();
            });
        }
        if (dynamic) __syncthreads();
    }
    if (tid == 0) trace_end(blp, iter);
    if (*abort_flag)
        for (int spin = 0; spin < 64; ++spin) __nanosleep(1000);  // copies in flight land before the CTA ends
}

template <typename F>
static auto attend_instance(int dim, int rows, bool half, F &&f) {
    auto by_rows = [&](auto d, auto hf) {
        constexpr int D = decltype(d)::value;
        constexpr bool H = decltype(hf)::value;
        if (rows <= 8) return f(kv_attend_kernel<D, 1, H>, AttCfg<D, 1>::kFixed + sizeof(AttCtl<1>), AttCfg<D, 1>::kRows);
        if (rows <= 16) return f(kv_attend_kernel<D, 2, H>, AttCfg<D, 2>::kFixed + sizeof(AttCtl<2>), AttCfg<D, 2>::kRows);
        return f(kv_attend_kernel<D, 4, H>, AttCfg<D, 4>::kFixed + sizeof(AttCtl<4>), AttCfg<D, 4>::kRows);
    };
    using D64 = std::integral_constant<int, 64>;
    using D128 = std::integral_constant<int, 128>;
    if (dim == 64) return half ? by_rows(D64(), std::true_type()) : by_rows(D64(), std::false_type());
    return half ? by_rows(D128(), std::true_type()) : by_rows(D128(), std::false_type());
}

// Rows of a head of keys (its group's heads times the tokens) from which on the other kernel takes over.  This kernel's time grows
// with the blocks of 32 rows, the other's is that of 256 rows.  This and the other, us, 32 heads of 128 on 8:
//   rows                           16           24           32           48           64          128
//    4 sequences over  2 000   22.5 34.4    31.8 34.6    34.5 34.4    42.9 34.7    45.4 34.6    47.0 35.4
//   16 sequences over  2 000   38.9 58.7    57.4 58.5    61.9 58.6    88.0 58.8   106.3 58.6   148.6 59.0
//    2 sequences over 20 000   39.9 62.1    60.3 62.8    66.6 62.6    74.1 62.9    75.5 63.1   121.5 64.1
// At 32 rows the other is ahead by up to 6 %; the line stays at the end of this kernel's largest instance, up to which factors of fp16
// results have 22 bits.  For heads of 128 that instance and the one of two tiles use all 255 registers, and the larger spills 188
// (bf16) and 236 (fp16) bytes.
constexpr int kManyRows = 32;

// Of a preemptible launch: 1024 keys, 256 KiB of a head of 128.  64 sequences over 16 384 keys drain in 21 us at the median, 24 at
// most, and take 257 us on the device; without a word, where a tile is a CTA's whole share, 201.
constexpr int kBlocksATile = 16;

cudaError_t kv_attend_few_launch(AttendParams &p, int dim, bool half, const DeviceInfo &d, const BlpArgs &blp, cudaStream_t s) {
    const int rows = (int)std::min<long long>((long long)p.batch.most_new * (p.heads / p.kv_heads), 1 << 20);
    return attend_instance(dim, rows, half, [&](auto kernel, size_t smem, int tile_rows) {
        const size_t most = smem + lm_prefix_bytes(kLmMaxSeqs);
        smem += lm_prefix_bytes(p.batch.seqs);
        int per_sm;
        const cudaError_t e = lm_resident((const void *)kernel, kAttThreads, smem, most, d.device, &per_sm);
        if (e != cudaSuccess) return e;
        const size_t slot = (size_t)tile_rows * (dim + 2) * sizeof(float);
        p.max_tiles = (int)std::min<size_t>(kLmCounters, kLmPartsBytes / (2 * slot));
        p.blocks_a_tile = kBlocksATile;
        const int grid = std::min(d.sm_count * per_sm, p.max_tiles);
        return launch_layer(kernel, grid, kAttThreads, smem, s, p, blp);
    });
}

}  // namespace gpx

using namespace gpx;

extern "C" int gpx_kv_attend(const gpx_kv_cache *cache, const gpx_kv_batch *batch, const gpx_kv_attend_args *args, void *ctx,
                             const gpx_blp *blp, gpx_stream stream) {
    GPX_REQUIRE(cache && args && ctx, GPX_FAIL, "cache, args or ctx is NULL");
    GPX_REQUIRE((uintptr_t)ctx % 256 == 0, GPX_FAIL, "ctx must be 256-byte aligned");
    const gpx_kv_attend_args &a = *args;
    AttendParams p{};
    BlpArgs b;
    int elem;
    GPX_TRY(lm_check_batch(batch, &p.batch));
    GPX_TRY(lm_check_blp(blp, &b));
    GPX_TRY(lm_elem(a.dtype, false, &elem));
    GPX_REQUIRE(a.q && a.out, GPX_FAIL, "q or out is NULL");
    GPX_REQUIRE(a.heads > 0 && a.heads % cache->kv_heads == 0, GPX_OUT_OF_RANGE, "%d heads are not a multiple of the cache's %d",
                a.heads, cache->kv_heads);
    GPX_REQUIRE(a.window >= 0 && (!a.window || a.causal), GPX_OUT_OF_RANGE, "a window of %d, causal %d", a.window, a.causal);
    GPX_REQUIRE(a.scale == a.scale && a.scale >= 0.f && a.scale <= 3.4e38f, GPX_OUT_OF_RANGE, "scale must be positive and finite, or 0");
    const long long row = (long long)a.heads * cache->dim;
    p.q_ld = a.q_ld ? a.q_ld : row, p.out_ld = a.out_ld ? a.out_ld : row;
    GPX_REQUIRE(p.q_ld >= row && p.out_ld >= row, GPX_OUT_OF_RANGE, "a token's row is longer than the distance to the next");
    GPX_REQUIRE((p.q_ld | p.out_ld) % 8 == 0 && ((uintptr_t)a.q | (uintptr_t)a.out) % 16 == 0 && (uintptr_t)a.lse % 4 == 0, GPX_FAIL,
                "q and out must be 16-byte aligned, their distances multiples of 8 elements, lse 4-byte aligned");
    GPX_REQUIRE((long long)p.batch.most_new * a.heads <= 0x7fffffff - 256, GPX_OUT_OF_RANGE, "too many rows");
    const DeviceInfo &d = device_info();
    GPX_REQUIRE(d.device >= 0, GPX_FAIL, "gpx_init was not called");
    if (p.batch.most_new == 0) return GPX_SUCC;
    p.map_k = cache->map_k, p.map_v = cache->map_v;
    p.v_codes = cache->v, p.k_scale = cache->k_scale, p.v_scale = cache->v_scale;
    p.pages = cache->pages, p.page_shift = __builtin_ctz((unsigned)cache->page_tokens), p.kv_heads = cache->kv_heads, p.heads = a.heads;
    p.q = (const unsigned short *)a.q, p.out = (unsigned short *)a.out, p.lse = (float *)a.lse;
    p.scale = a.scale != 0.f ? a.scale : 1.0f / sqrtf((float)cache->dim);
    p.causal = a.causal != 0, p.window = a.window;
    const LmCtx c = lm_ctx(ctx);
    p.error = c.error, p.counters = c.counters, p.prefix = c.prefix, p.parts = c.parts;
    const bool many = (long long)p.batch.most_new * (a.heads / cache->kv_heads) > kManyRows;
    GPX_CUDA((many ? kv_attend_many_launch : kv_attend_few_launch)(p, cache->dim, elem == LM_F16, d, b, as_stream(stream)));
    return GPX_SUCC;
}
