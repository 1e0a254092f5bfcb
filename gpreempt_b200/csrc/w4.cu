// Products of a few rows with weights of 4 bits that have a scale (and a zero) for each group of a row's elements.
//
//   y[r][i] = sum over groups of scale[i][group] * (sum over j in it of (code[i][j] - zero[i][group]) x[r][j])
//
// The floor is memory: half a byte a weight, read once, against 2 operations a row; what bounds the kernels is their instructions (below).
// Weights are the M side of the tensor instructions (sixteen of their rows), the rows of x the N side; 33 to 64 rows are two groups, for
// which weights are read and converted twice.  A code becomes a 16-bit number without a conversion: or-ed into the mantissa
// of 1024 (fp16) or 128 (bf16) it is that much more, and taking off that and the zero is exact (the method of Kim, Henry, Fahim and
// Hassan Awadalla, 2022).  Products of a group (64 elements at
// most) are summed in float and then multiplied by the scale in float, so that nothing is rounded but the sums.  (Leaving the zeros to
// the sums of x instead saves sixteen subtractions for 512 bytes of weights, and costs as many instructions behind the products.)
//
// Weights are packed once into records of 16 rows by 128 elements with their scales and zeros, in the order in which lanes need them: of
// a block of 16 rows by 64 elements a lane has the sixteen bytes that are its operands of four steps.  The order of elements in a step is free
// as long as both sides agree, so that a lane's elements of x are contiguous too.
#include "lm.h"
#include "kv_attend.h"
#include "sm100.cuh"

#include <algorithm>

namespace gpx {

constexpr int kW4Elements = 128, kW4Blocks = 2;  // of a record; blocks have 64 elements
constexpr int kW4Codes = 1024;                   // bytes of a record: [block][lane][16]
template <int G>
constexpr int kW4Sets = kW4Elements / G;         // scales of a row in a record: [set][8], those of rows g and g + 8; zeros likewise

struct W4Params {
    const unsigned char *packed;
    int n, k, tiles16, records;          // tiles of sixteen rows; records of a row
    int record_bytes, zeros;
    const unsigned short *x;
    unsigned short *y;
    long long x_ld, y_ld;
    int rows;
    int row_groups, group_rows;          // rows of x that are multiplied at a time
    int row_tiles, steps, line;          // tiles of 256 rows of weights, steps of 128 elements of a row, steps of everything
    int steps_a_tile, most_tiles;
    int *counters;
    float *slots;
};

// Bytes of weights from which the kernel of large products takes over.  Both, us, in bf16 groups of 128:
//   rows            4096 x 4096   8192 x 4096   14336 x 4096   8192 x 8192   28672 x 8192   1024 x 16384
//      1   small          7.0          11.4           15.7          18.7           42             16.0
//          large         10.9          12.2           15.0          16.7           37             20.5
//     24   small         12.5          21.6           35.0          36.6          114             16.6
//          large         16.6          18.3           22.7          25.1           58             31.7
//     64   small         27            50             85            86            287             30.9
//          large         20            27             39            42            118             30.9
// (4096 x 4096, 8.9 MB, stays with the small one, which is the slower from 40 rows on)
constexpr long long kW4Large = 12 << 20;
constexpr uint32_t kW4HalfBase = 0x6400, kW4BfBase = 0x4300;  // 1024 in fp16, 128 in bf16: a code is or-ed into the mantissa

struct W4Layout {
    int tiles16, records, record_bytes;
    size_t bytes;
};
static W4Layout w4_layout(const gpx_w4 &w) {
    W4Layout l;
    l.tiles16 = (w.n + 15) / 16, l.records = (w.k + kW4Elements - 1) / kW4Elements;
    l.record_bytes = kW4Codes + kW4Elements / w.group * 32 * (w.zeros ? 2 : 1);
    l.bytes = ((size_t)l.tiles16 * l.records * l.record_bytes + 255) / 256 * 256;
    return l;
}

// Eight codes of a row in the order in which pairs come out of a word: 0 and 1 of its lowest four bits and of those 16 up, and so on.
__device__ __forceinline__ uint32_t w4_order(uint32_t w) {
    uint32_t to = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) to |= (w >> 4 * e & 15u) << (4 * (e >> 1) + 16 * (e & 1));
    return to;
}

// Once a matrix; of 28 672 x 8 192 elements with zeros, groups of 64, 93 us, of 4 096 x 4 096 10.
__global__ void w4_pack_kernel(const unsigned char *codes, const unsigned short *scales, const unsigned char *zeros, int n, int k, int group, int tiles16,
                               int records, bool half, unsigned char *packed) {
    pdl_enter();
    const int groups = k / group, scale_words = kW4Elements / group * 8, bytes = kW4Codes + scale_words * 4 * (zeros ? 2 : 1);
    const int pieces = kW4Codes / 16, all_pieces = pieces + scale_words * (zeros ? 2 : 1);
    const long long all = (long long)tiles16 * records * all_pieces;
    for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < all; e += (long long)gridDim.x * blockDim.x) {
        const long long record = e / all_pieces;
        const int piece = (int)(e - record * all_pieces), row0 = 16 * (int)(record / records), element0 = kW4Elements * (int)(record % records);
        unsigned char *const to = packed + record * bytes;
        if (piece < pieces) {
            const int lane = piece & 31, g = lane >> 2, t = lane & 3, block = piece >> 5;
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = row0 + g + 8 * (j & 1), from = element0 + 64 * block + 32 * (j >> 1) + 8 * t;
                w[j] = row < n && from < k ? w4_order(*reinterpret_cast<const uint32_t *>(codes + (size_t)row * (k / 2) + from / 2)) : 0;
            }
            reinterpret_cast<uint4 *>(to)[piece] = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            const int word = piece - pieces, kind = word / scale_words, at = word - kind * scale_words;
            const int row = row0 + (at & 7), of = element0 / group + (at >> 3);
            auto value = [&](int i) -> uint32_t {
                const bool there = i < n && of < groups;
                if (kind == 0) return there ? scales[(size_t)i * groups + of] : 0u;
                const unsigned zero = there ? zeros[(size_t)i * groups + of] & 15u : 0u;
                return (half ? kW4HalfBase : kW4BfBase) + zero;
            };
            reinterpret_cast<uint32_t *>(to + kW4Codes)[word] = value(row) | value(row + 8) << 16;
        }
    }
}

// d = a b, or + d
template <bool HALF, bool FIRST>
__device__ __forceinline__ void w4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    const float c0 = FIRST ? 0.f : d[0], c1 = FIRST ? 0.f : d[1], c2 = FIRST ? 0.f : d[2], c3 = FIRST ? 0.f : d[3];
    if (HALF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// (a & mask) | or_
template <uint32_t MASK>
__device__ __forceinline__ uint32_t w4_pick(uint32_t a, uint32_t or_) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "n"(MASK), "r"(or_));
    return d;
}
template <bool HALF>
__device__ __forceinline__ float2 w4_scales(uint32_t w) {
    if (HALF) return unpack_halves(w);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}


// The pairs 0, 1 | 2, 3 | 4, 5 | 6, 7 of a word's codes less their zero, as 16-bit numbers: 1024 (128) and the code, less `z`, which is
// 1024 (128) and the zero; in fp16, where a mantissa has room for a code four bits up, without a shift for every other pair.
template <bool HALF>
__device__ __forceinline__ void w4_pairs(uint32_t w, uint32_t z, uint32_t (&a)[4]) {
    if (HALF) {
        const __half2 zero = *reinterpret_cast<const __half2 *>(&z);
        const __half2 less = __hsub2(__floats2half2_rn(960.f, 960.f), zero);  // - 64 - the zero
        const __half2 sixteenth = __floats2half2_rn(0.0625f, 0.0625f);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t lo = w4_pick<0x000f000fu>(w >> 8 * j, kW4HalfBase * 0x10001u);  // 1024 + code
            const uint32_t hi = w4_pick<0x00f000f0u>(w >> 8 * j, kW4HalfBase * 0x10001u);  // 1024 + 16 code
            const __half2 p = __hsub2(*reinterpret_cast<const __half2 *>(&lo), zero);
            const __half2 q = __hfma2(*reinterpret_cast<const __half2 *>(&hi), sixteenth, less);
            a[2 * j] = *reinterpret_cast<const uint32_t *>(&p), a[2 * j + 1] = *reinterpret_cast<const uint32_t *>(&q);
        }
    } else {
        const __nv_bfloat162 zero = *reinterpret_cast<const __nv_bfloat162 *>(&z);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t v = w4_pick<0x000f000fu>(w >> 4 * j, kW4BfBase * 0x10001u);
            const __nv_bfloat162 p = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), zero);
            a[j] = *reinterpret_cast<const uint32_t *>(&p);
        }
    }
}

// One block of sixteen rows: acc += its products with NT times eight rows of x.  `x` are a lane's elements of either half, `scales` and
// `zeros` those of the block's rows, of the set of either half.
template <int NT, bool HALF, int G>
__device__ __forceinline__ void w4_block(float (&acc)[NT][4], const uint4 &w, const uint4 (&x)[NT][2], const uint32_t (&scales)[2], const uint32_t (&zeros)[2]) {
    uint32_t u[2][4], v[2][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const uint32_t zero = zeros[G == 32 ? half : 0];
        w4_pairs<HALF>(half ? w.z : w.x, __byte_perm(zero, 0, 0x1010), u[half]);
        w4_pairs<HALF>(half ? w.w : w.y, __byte_perm(zero, 0, 0x3232), v[half]);
    }
    float2 scale[2];
    scale[0] = w4_scales<HALF>(scales[0]);
    if (G == 32) scale[1] = w4_scales<HALF>(scales[1]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float part[4] = {0.f, 0.f, 0.f, 0.f};
        auto add = [&](const float2 &f) {
            acc[nt][0] = fmaf(part[0], f.x, acc[nt][0]), acc[nt][1] = fmaf(part[1], f.x, acc[nt][1]);
            acc[nt][2] = fmaf(part[2], f.y, acc[nt][2]), acc[nt][3] = fmaf(part[3], f.y, acc[nt][3]);
        };
        w4_mma<HALF, true>(part, u[0][0], v[0][0], u[0][1], v[0][1], x[nt][0].x, x[nt][0].y);
        w4_mma<HALF, false>(part, u[0][2], v[0][2], u[0][3], v[0][3], x[nt][0].z, x[nt][0].w);
        if (G == 32) add(scale[0]);
        w4_mma<HALF, G == 32>(part, u[1][0], v[1][0], u[1][1], v[1][1], x[nt][1].x, x[nt][1].y);
        w4_mma<HALF, false>(part, u[1][2], v[1][2], u[1][3], v[1][3], x[nt][1].z, x[nt][1].w);
        add(scale[G == 32 ? 1 : 0]);
    }
}
template <bool HALF>
constexpr uint32_t kW4Eight = ((HALF ? kW4HalfBase : kW4BfBase) + 8) * 0x10001u;  // zeros of weights that have none

// ---- small products ---------------------------------------------------------------------------------

// A CTA takes sixteen rows of weights and eight of x, its warps a part of the elements each, and adds the parts up in their order: nothing is
// shared with other CTAs.  One row by 1 024 x 4 096 weights takes a launch, by 4 096 x 4 096 (8.7 MB) 7.2 us.
constexpr int kW4Warps = 8, kW4Threads = 32 * kW4Warps;

template <bool HALF, int G>
__global__ void __launch_bounds__(kW4Threads)
w4_small_kernel(const __grid_constant__ W4Params p, BlpArgs blp) {
    constexpr int kWords = (kW4Sets<G> * 8 + 31) / 32;  // of a record's scales in a lane
    __shared__ float sums[kW4Warps][4][32];
    __shared__ int s_tile;
    const int tid = threadIdx.x, lane = tid & 31, wid = __shfl_sync(0xffffffffu, tid >> 5, 0), g = lane >> 2, t = lane & 3;
    pdl_enter();
    const bool dynamic = blp.preempted != nullptr;
    if (tid == 0) trace_begin(blp);
    const int record0 = (int)((long long)p.records * wid / kW4Warps), record1 = (int)((long long)p.records * (wid + 1) / kW4Warps);
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
        const int row_group = tile % p.row_groups, of = tile / p.row_groups;
        const unsigned char *const records = p.packed + (size_t)of * p.records * p.record_bytes;
        // (columns beyond the rows there are go nowhere: they may be any)
        const unsigned short *const row = p.x + min(8 * row_group + g, p.rows - 1) * p.x_ld + 8 * t;
        struct Fetched {
            uint4 codes[kW4Blocks];
            uint32_t scales[kWords], zeros[kWords];
        };
        auto fetch = [&](int r) {
            Fetched f;
            const unsigned char *const at = records + (size_t)min(r, p.records - 1) * p.record_bytes;
#pragma unroll
            for (int b = 0; b < kW4Blocks; ++b) f.codes[b] = __ldg(reinterpret_cast<const uint4 *>(at) + b * 32 + lane);
            const uint32_t *const words = reinterpret_cast<const uint32_t *>(at + kW4Codes);
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                const int word = min(32 * j + lane, kW4Sets<G> * 8 - 1);
                f.scales[j] = __ldg(words + word);
                f.zeros[j] = p.zeros ? __ldg(words + kW4Sets<G> * 8 + word) : kW4Eight<HALF>;
            }
            return f;
        };
        float acc[1][4] = {{0.f, 0.f, 0.f, 0.f}};
        auto multiply = [&](int r, const Fetched &f) {
#pragma unroll
            for (int b = 0; b < kW4Blocks; ++b) {
                const int from = kW4Elements * r + 64 * b;
                if (from >= p.k) break;
                const bool both = G != 32 || from + 32 < p.k;
                uint4 x[1][2];
                x[0][0] = __ldg(reinterpret_cast<const uint4 *>(row + from));
                x[0][1] = both ? __ldg(reinterpret_cast<const uint4 *>(row + from + 32)) : make_uint4(0, 0, 0, 0);
                uint32_t scales[2], zeros[2];
#pragma unroll
                for (int half = 0; half < (G == 32 ? 2 : 1); ++half) {
                    const int word = (64 * b + 32 * half) / G * 8;
                    scales[half] = __shfl_sync(0xffffffffu, f.scales[word / 32], word % 32 + g);
                    zeros[half] = __shfl_sync(0xffffffffu, f.zeros[word / 32], word % 32 + g);
                }
                w4_block<1, HALF, G>(acc, f.codes[b], x, scales, zeros);
            }
        };
        Fetched now = fetch(record0), next = fetch(record0 + 1), after = fetch(record0 + 2);
        for (int r = record0; r < record1; ++r) {
            const Fetched last = fetch(r + 3);
            multiply(r, now);
            now = next, next = after, after = last;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) sums[wid][c][lane] = acc[0][c];
        __syncthreads();
        if (tid < 128) {
            // row r of x and row i of the sixteen: consecutive threads have consecutive rows of the weights
            const int i = tid & 15, r = tid >> 4, at = 16 * of + i;
            if (8 * row_group + r < p.rows && at < p.n) {
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < kW4Warps; ++w) sum += sums[w][(i >> 3) * 2 + (r & 1)][(i & 7) * 4 + (r >> 1)];
                p.y[(8 * row_group + r) * p.y_ld + at] = (unsigned short)pack_out<HALF>(sum, 0.f);
            }
        }
        __syncthreads();
    }
    if (tid == 0) trace_end(blp, iter);
}

// ---- large products ---------------------------------------------------------------------------------

// Eight warps take 32 rows of weights each, over the same elements of x.  The work of all tiles of 256 rows lies on one line, in steps of
// 128 elements, and a tile of the launch is an equal piece of it, so that every SM has as much to read.  Weights and elements of a step are
// copied two or three steps ahead, into rings that go on where 256 rows end.  Rows that a tile has not whole leave their sums in the
// context, and the CTA that brings the last one adds them up in the order of the line; meanwhile the other CTA of the SM reads on.
//
// One row by 28 672 x 8 192 weights with zeros, fp16, groups of 64: 35 us (129 MB, 3.7 TB/s); 24 rows by 13 001 x 5 120, bf16, groups of 32: 24.7.
// 85 instructions for 512 bytes of weights, of which the codes take 36 to 44, fill 58 % of the slots, and the steps' barriers and the
// join take a part of the rest.  Without rings (loads to registers, two steps ahead) 53 and 36 us; sixteen warps a CTA and one CTA an SM 45 and
// 36; x for all elements in shared memory and parts of them where it has no room 36 and 40, with a sum over warps at the end of
// every part 104; 64 rows a warp and rings of three 37.5 and 25.
constexpr int kW4StreamWarps = 8, kW4StreamThreads = 32 * kW4StreamWarps, kW4TileRows = 32 * kW4StreamWarps;
constexpr int kW4Step = kW4Elements;
constexpr int kW4XRow = 2 * kW4Step + 64;  // bytes from a row of x to the next: no two lanes of a phase in a bank

__device__ __forceinline__ void w4_copy16(uint32_t to, const void *from, int bytes = 16) {  // (fewer than 16: zeros behind them)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

template <int NT, bool HALF, int G>
struct W4Stage {
    static constexpr int kSets = kW4Step / G;                        // scales of a row in a step
    static constexpr int kTile = 1024 + 2 * kSets * 32;              // bytes: codes of sixteen rows, scales, zeros
    static constexpr int kWeights = kW4StreamWarps * 2 * kTile, kX = 8 * NT * kW4XRow;
    static constexpr int kBytes = kWeights + kX;
    static constexpr int kRing = 4 * kBytes <= 112 * 1024 ? 4 : 3;
    static constexpr size_t kSmem = kRing * kBytes;
};

template <int NT, bool HALF, int G>
__global__ void __launch_bounds__(kW4StreamThreads, 2)
w4_stream_kernel(const __grid_constant__ W4Params p, BlpArgs blp) {
    using S = W4Stage<NT, HALF, G>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int s_tile, s_last;
    const int tid = threadIdx.x, lane = tid & 31, wid = __shfl_sync(0xffffffffu, tid >> 5, 0), g = lane >> 2, t = lane & 3;
    const uint32_t smem_at = sm100::smem_u32(smem);
    pdl_enter();
    const bool dynamic = blp.preempted != nullptr;
    if (tid == 0) trace_begin(blp);
    int tiles = dynamic ? max((p.line + p.steps_a_tile - 1) / p.steps_a_tile, (int)gridDim.x) : (int)gridDim.x;
    tiles = min(min(tiles, p.line), p.most_tiles);
    blp.total_tiles = tiles;
    const LmCut cut(p.line, tiles);
    // a place on the line
    struct Place {
        int row_group, row_tile, step;
    };
    auto walk = [&](Place &a) {
        if (++a.step < p.steps) return;
        a.step = 0;
        if (++a.row_tile < p.row_tiles) return;
        a.row_tile = 0, ++a.row_group;
    };

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
            __syncthreads();  // the rings are filled anew
        }
        if (tile < 0) break;
        const int line0 = cut.begin(tile), line1 = cut.begin(tile + 1);
        Place now;
        now.row_group = line0 / (p.row_tiles * p.steps);
        now.row_tile = line0 / p.steps - now.row_group * p.row_tiles, now.step = line0 % p.steps;
        Place ahead = now;
        int at_ahead = line0, slot_ahead = 0;
        const unsigned char *from[2];  // records of this warp's tiles of sixteen rows, of x this thread's piece
        const unsigned short *x_from;
        bool there[2], x_there;
        auto begin_rows = [&]() {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const int tile16 = (ahead.row_tile * kW4StreamWarps + wid) * 2 + m;
                there[m] = tile16 < p.tiles16;
                from[m] = p.packed + ((size_t)min(tile16, p.tiles16 - 1) * p.records + ahead.step) * p.record_bytes + 16 * lane;
            }
            // (32 rows have two pieces a thread, sixteen rows apart)
            const int row = ahead.row_group * p.group_rows + (tid >> 4);
            x_there = tid >> 4 < min(p.group_rows, p.rows - ahead.row_group * p.group_rows);
            x_from = p.x + (x_there ? row : 0) * p.x_ld + kW4Step * ahead.step + 8 * (tid & 15);
        };
        begin_rows();
        const uint32_t x_to = smem_at + S::kWeights + (tid >> 4) * kW4XRow + 16 * (tid & 15), w_to = smem_at + wid * 2 * S::kTile + 16 * lane;
        auto copy = [&]() {
            if (at_ahead < line1) {
                const uint32_t stage = slot_ahead * S::kBytes;
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    if (!there[m]) break;
                    const uint32_t to = w_to + stage + m * S::kTile;
                    w4_copy16(to, from[m]), w4_copy16(to + 512, from[m] + 512);
                    if (kW4Codes + 16 * lane < p.record_bytes) w4_copy16(to + 1024, from[m] + 1024);
                    from[m] += p.record_bytes;
                }
                const bool inside = kW4Step * ahead.step + 8 * (tid & 15) < p.k;  // (zeros behind the end of a row)
                if (x_there) w4_copy16(x_to + stage, inside ? x_from : p.x, inside ? 16 : 0);
                if (NT > 2 && (tid >> 4) + 16 < min(p.group_rows, p.rows - ahead.row_group * p.group_rows))
                    w4_copy16(x_to + stage + 16 * kW4XRow, inside ? x_from + 16 * p.x_ld : p.x, inside ? 16 : 0);
                x_from += kW4Step;
                walk(ahead);
                if (++at_ahead < line1 && ahead.step == 0) begin_rows();
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            slot_ahead = slot_ahead + 1 == S::kRing ? 0 : slot_ahead + 1;
        };
        for (int j = 0; j < S::kRing - 1; ++j) copy();
        int slot = 0;

        for (int begin = line0; begin < line1;) {
            // ---- steps [begin, end) of one tile of 256 rows of weights and a group of rows of x
            const int unit0 = begin - now.step, end = min(line1, unit0 + p.steps);
            const int first_row = now.row_group * p.group_rows, rows = min(p.group_rows, p.rows - first_row);
            const int tile16 = (now.row_tile * kW4StreamWarps + wid) * 2;
            float acc[2][NT][4];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[m][nt][c] = 0.f;
            for (int at = begin; at < end; ++at) {
                asm volatile("cp.async.wait_group %0;" ::"n"(S::kRing - 2) : "memory");
                __syncthreads();  // this step has arrived, the one before is done with: its slot can be filled
                copy();
                const unsigned char *const stage = smem + slot * S::kBytes;
                const unsigned char *const x_at = stage + S::kWeights + min(g, rows - 1) * kW4XRow + 16 * t;
                const unsigned char *const weights = stage + wid * 2 * S::kTile;
                if (tile16 < p.tiles16) {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        uint4 x[NT][2];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            // (columns beyond the rows there are go nowhere: they may be any)
                            const unsigned char *const row = NT == 1 ? x_at : stage + S::kWeights + (8 * nt + g) * kW4XRow + 16 * t;
#pragma unroll
                            for (int half = 0; half < 2; ++half) x[nt][half] = *reinterpret_cast<const uint4 *>(row + 128 * b + 64 * half);
                        }
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            const uint4 w = reinterpret_cast<const uint4 *>(weights + m * S::kTile)[b * 32 + lane];
                            const uint32_t *const words = reinterpret_cast<const uint32_t *>(weights + m * S::kTile + 1024) + g;
                            uint32_t scales[2], zeros[2];
#pragma unroll
                            for (int half = 0; half < (G == 32 ? 2 : 1); ++half) {
                                const int word = (64 * b + 32 * half) / G * 8;
                                scales[half] = words[word];
                                zeros[half] = p.zeros ? words[S::kSets * 8 + word] : kW4Eight<HALF>;
                            }
                            w4_block<NT, HALF, G>(acc[m], w, x, scales, zeros);
                        }
                    }
                }
                slot = slot + 1 == S::kRing ? 0 : slot + 1;
                walk(now);
            }
            // ---- complete sums are the result, others wait in the context
            auto put = [&]() {
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int r = 8 * nt + 2 * t + (c & 1), i = 16 * (tile16 + m) + g + 8 * (c >> 1);
                            if (r < rows && i < p.n) p.y[(first_row + r) * p.y_ld + i] = (unsigned short)pack_out<HALF>(acc[m][nt][c], 0.f);
                        }
            };
            if (begin == unit0 && end == unit0 + p.steps) {
                put();
            } else {
                const int t0 = cut.tile_of(unit0), t1 = cut.tile_of(unit0 + p.steps - 1);
                // (a tile has two slots: for rows that it begins in the middle of, and for those that it begins)
                auto slot_of = [&](int x) {
                    return reinterpret_cast<float4 *>(p.slots) + ((size_t)(2 * x + (x == t0)) * kW4StreamWarps + wid) * (2 * NT * 32) + lane;
                };
                float4 *const mine = slot_of(tile);
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mine[(m * NT + nt) * 32] = make_float4(acc[m][nt][0], acc[m][nt][1], acc[m][nt][2], acc[m][nt][3]);
                __threadfence();
                __syncthreads();
                if (tid == 0) s_last = atomicAdd(&p.counters[t0], 1) == t1 - t0;
                __syncthreads();
                if (s_last) {
                    __threadfence();
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 4; ++c) acc[m][nt][c] = 0.f;
#pragma unroll 2
                    for (int x = t0; x <= t1; ++x) {
                        const float4 *const theirs = slot_of(x);
                        float4 v[2][NT];
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) v[m][nt] = __ldcg(theirs + (m * NT + nt) * 32);
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                acc[m][nt][0] += v[m][nt].x, acc[m][nt][1] += v[m][nt].y;
                                acc[m][nt][2] += v[m][nt].z, acc[m][nt][3] += v[m][nt].w;
                            }
                    }
                    put();
                    if (tid == 0) p.counters[t0] = 0;
                }
            }
            begin = end;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    if (tid == 0) trace_end(blp, iter);
}

static int w4_check(const gpx_w4 *w, int *elem) {
    GPX_REQUIRE(w, GPX_FAIL, "the weights are NULL");
    GPX_REQUIRE(w->group == 32 || w->group == 64 || w->group == 128, GPX_OUT_OF_RANGE, "group is 32, 64 or 128, not %d", w->group);
    GPX_REQUIRE(w->n > 0 && w->k > 0 && w->k % w->group == 0, GPX_OUT_OF_RANGE, "weights of %d x %d in groups of %d", w->n, w->k, w->group);
    GPX_REQUIRE(w->n <= 0x7fffffff - 16 && w->k <= 0x7fffffff - 512, GPX_OUT_OF_RANGE, "weights of %d x %d", w->n, w->k);
    GPX_TRY(lm_elem(w->dtype, false, elem));
    return GPX_SUCC;
}
// How a large product is cut; false where it is a small one.
static bool w4_plan(W4Params &p) {
    if ((long long)p.tiles16 * p.records * p.record_bytes < kW4Large) return false;
    p.row_groups = (p.rows + 31) / 32;
    p.group_rows = (p.rows + p.row_groups - 1) / p.row_groups;
    p.row_tiles = (p.n + kW4TileRows - 1) / kW4TileRows, p.steps = (p.k + kW4Step - 1) / kW4Step;
    const long long line = (long long)p.row_groups * p.row_tiles * p.steps;
    if (line > 0x3fffffff) return false;
    const int nt = (p.group_rows + 7) / 8;
    p.line = (int)line, p.steps_a_tile = 8;
    p.most_tiles = (int)std::min<size_t>(kLmCounters, kLmPartsBytes / ((size_t)2 * kW4StreamWarps * 2 * nt * 512));
    return true;
}

static int w4_check_packed(const gpx_w4 *w) {
    GPX_REQUIRE(w->packed && (uintptr_t)w->packed % 256 == 0, GPX_FAIL, "packed is NULL or not 256-byte aligned");
    return GPX_SUCC;
}

}  // namespace gpx

using namespace gpx;

extern "C" {

int gpx_w4_bytes(const gpx_w4 *w, size_t *bytes) {
    int elem;
    GPX_REQUIRE(bytes, GPX_FAIL, "bytes is NULL");
    GPX_TRY(w4_check(w, &elem));
    *bytes = w4_layout(*w).bytes;
    return GPX_SUCC;
}

int gpx_w4_pack(const gpx_w4 *w, const void *codes, const void *scales, const void *zeros, gpx_stream stream) {
    int elem;
    GPX_TRY(w4_check(w, &elem));
    GPX_TRY(w4_check_packed(w));
    GPX_REQUIRE(codes && scales && (uintptr_t)codes % 4 == 0 && (uintptr_t)scales % 2 == 0, GPX_FAIL,
                "codes or scales is NULL, or not aligned to 4 and 2 bytes");
    GPX_REQUIRE(!zeros == !w->zeros, GPX_FAIL, "zeros are given where the weights have none, or the other way round");
    const DeviceInfo &d = device_info();
    GPX_REQUIRE(d.device >= 0, GPX_FAIL, "gpx_init was not called");
    const W4Layout l = w4_layout(*w);
    const long long threads = (long long)l.tiles16 * l.records * (l.record_bytes / 16);
    const int grid = (int)std::min<long long>((threads + 255) / 256, 16 * d.sm_count);
    GPX_CUDA(launch_layer(w4_pack_kernel, grid, 256, 0, as_stream(stream), (const unsigned char *)codes, (const unsigned short *)scales,
                          (const unsigned char *)zeros, w->n, w->k, w->group, l.tiles16, l.records, elem == LM_F16,
                          (unsigned char *)w->packed));
    return GPX_SUCC;
}

int gpx_w4_matvec(const gpx_w4 *w, const gpx_w4_matvec_args *args, void *ctx, const gpx_blp *blp, gpx_stream stream) {
    GPX_REQUIRE(args && ctx, GPX_FAIL, "args or ctx is NULL");
    GPX_REQUIRE((uintptr_t)ctx % 256 == 0, GPX_FAIL, "ctx must be 256-byte aligned");
    int elem;
    BlpArgs b;
    W4Params p{};
    GPX_TRY(w4_check(w, &elem));
    GPX_TRY(w4_check_packed(w));
    GPX_TRY(lm_check_blp(blp, &b));
    const gpx_w4_matvec_args &a = *args;
    GPX_REQUIRE(a.x && a.y, GPX_FAIL, "x or y is NULL");
    GPX_REQUIRE(a.rows >= 1 && a.rows <= 64, GPX_OUT_OF_RANGE, "1 to 64 rows, not %d", a.rows);
    p.x_ld = a.x_ld ? a.x_ld : w->k, p.y_ld = a.y_ld ? a.y_ld : w->n;
    GPX_REQUIRE(p.x_ld >= w->k && p.y_ld >= w->n, GPX_OUT_OF_RANGE, "a row is longer than the distance to the next");
    GPX_REQUIRE(p.x_ld % 8 == 0 && (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.y % 2 == 0, GPX_FAIL,
                "x must be 16-byte aligned, its distance a multiple of 8 elements, y 2-byte aligned");
    const DeviceInfo &d = device_info();
    GPX_REQUIRE(d.device >= 0, GPX_FAIL, "gpx_init was not called");
    const W4Layout l = w4_layout(*w);
    p.packed = (const unsigned char *)w->packed, p.record_bytes = l.record_bytes, p.zeros = w->zeros != 0;
    p.n = w->n, p.k = w->k, p.tiles16 = l.tiles16, p.records = l.records;
    p.x = (const unsigned short *)a.x, p.y = (unsigned short *)a.y, p.rows = a.rows;
    const LmCtx c = lm_ctx(ctx);
    p.counters = c.counters, p.slots = c.parts;
    auto small = [&](auto kernel) {
        int per_sm;
        const cudaError_t e = lm_resident((const void *)kernel, kW4Threads, 0, 0, d.device, &per_sm);
        if (e != cudaSuccess) return e;
        p.row_groups = (a.rows + 7) / 8;
        b.total_tiles = (w->n + 15) / 16 * p.row_groups;
        const int grid = b.preempted ? std::min(b.total_tiles, d.sm_count * per_sm) : b.total_tiles;
        return launch_layer(kernel, grid, kW4Threads, 0, as_stream(stream), p, b);
    };
    auto large = [&](auto kernel, size_t smem) {
        int per_sm;
        const cudaError_t e = lm_resident((const void *)kernel, kW4StreamThreads, smem, smem, d.device, &per_sm);
        if (e != cudaSuccess) return e;
        return launch_layer(kernel, std::min(std::min(p.line, p.most_tiles), d.sm_count * per_sm), kW4StreamThreads, smem, as_stream(stream), p, b);
    };
    auto run = [&](auto half, auto group) {
        constexpr bool H = decltype(half)::value;
        constexpr int G = decltype(group)::value;
        if (!w4_plan(p)) return small(w4_small_kernel<H, G>);
        const int nt = (p.group_rows + 7) / 8;
        if (nt == 1) return large(w4_stream_kernel<1, H, G>, W4Stage<1, H, G>::kSmem);
        if (nt == 2) return large(w4_stream_kernel<2, H, G>, W4Stage<2, H, G>::kSmem);
        if (nt == 3) return large(w4_stream_kernel<3, H, G>, W4Stage<3, H, G>::kSmem);
        return large(w4_stream_kernel<4, H, G>, W4Stage<4, H, G>::kSmem);
    };
    auto by_group = [&](auto half) {
        if (w->group == 32) return run(half, std::integral_constant<int, 32>());
        if (w->group == 64) return run(half, std::integral_constant<int, 64>());
        return run(half, std::integral_constant<int, 128>());
    };
    GPX_CUDA(elem == LM_F16 ? by_group(std::true_type()) : by_group(std::false_type()));
    return GPX_SUCC;
}

}  // extern "C"
