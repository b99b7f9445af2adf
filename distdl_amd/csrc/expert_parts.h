// The experts' products: what their kernels share.  Rows lie expert by expert, expert e's from offsets[e] to offsets[e + 1] (device
// memory: the host knows their number in all, and launches as many workgroups as any distribution of them can need).
#ifndef DDL_EXPERT_PARTS_H
#define DDL_EXPERT_PARTS_H
#include "gemm_tiles.h"

namespace ddl {

// y[rows, n] = a[rows, k] . w[expert]^T by tiles of rows of one expert (w: n rows of k elements; read along n if `transposed`, when
// it is k rows of n), or w's gradient by tiles of every expert's matrix.
struct ExpertArgs {
    const void *a, *w;
    void* y;
    const int32_t* offsets;
    const float *a_scales, *w_scales;     // e4m3
    int experts, rows, out_dtype, cus;
    int64_t n, k, lda, ldw, w_stride, ldy;
    int tiles_m, tiles_n;                 // tiles_m: of an expert's matrix (gradients of the weights)
    int few, places;                      // gradients of the weights: of experts with more rows than this (-1: all), which are as many or less
};

// Kernels of expert_linear16.hip: tiles of 64 or 128 rows and columns at any address (edge 64, 128), or large ones, of 128 x 256 (low) or 256 x 256.
enum class ExpertTile { kAny64, kAny128, kLow, kLarge };
int run_expert_rows16(const char* who, ExpertTile tile, bool f16, bool transposed, ExpertArgs g, int dev, hipStream_t s);
int run_expert_weights16(const char* who, ExpertTile tile, bool f16, ExpertArgs g, int dev, hipStream_t s);
// Of expert_linear32.hip: tiles of 32 x 32 (small) or 64 x 64.
int run_expert_rows32(const char* who, bool small, bool transposed, const ExpertArgs& g, hipStream_t s);
int run_expert_weights32(const char* who, bool small, const ExpertArgs& g, hipStream_t s);
// Of expert_linear32_split.hip: tiles of 128 x 128.
int run_expert_rows32_split(const char* who, bool transposed, ExpertArgs g, hipStream_t s);
int run_expert_weights32_split(const char* who, ExpertArgs g, hipStream_t s);
// Of expert_outer.hip: gradients of the weights of all experts with at most g.few rows (matrices of at least 4 rows, and columns for 16 bytes).
int run_expert_outer(const char* who, const ExpertArgs& g, hipStream_t s);
// Of expert_across.hip: gradients of few rows (matrices with columns for 16 bytes).
int run_expert_across(const char* who, const ExpertArgs& g, hipStream_t s);
// Of expert_linear8.hip: kAny64, kLow and kLarge (aligned operands, all of them).
int run_expert_rows8(const char* who, ExpertTile tile, ExpertArgs g, int dev, hipStream_t s);

#ifdef __HIPCC__
namespace {

// First and last row of expert e, whatever the offsets hold; of e = experts: the rows behind the last expert's.
__device__ inline void rows_of_expert(const ExpertArgs& g, int e, int& lo, int& hi) {
    lo = min(max(g.offsets[e], 0), g.rows);
    hi = e == g.experts ? g.rows : min(max(g.offsets[e + 1], lo), g.rows);
}

// Zeros in `bytes` from `to` on (any address), by the threads `first`, first + step, ...
__device__ inline void zero_run(char* to, int64_t bytes, int64_t first, int64_t step) {
    typedef u32x4 any __attribute__((aligned(1)));
    if (bytes < 16) {
        for (int64_t i = first; i < bytes; i += step) to[i] = 0;
        return;
    }
    for (int64_t i = first * 16; i < bytes; i += step * 16) *reinterpret_cast<any*>(to + (i + 16 <= bytes ? i : bytes - 16)) = u32x4{0, 0, 0, 0};
}

// Zeros in rows from `row` on (they lie side by side), by `blocks` workgroups of which this one is number `block`.
__device__ inline void zero_rows(const ExpertArgs& g, int row, int rows, int64_t block, int64_t blocks) {
    const int64_t size = g.out_dtype == DDL_DT_F32 ? 4 : 2;
    zero_run(static_cast<char*>(g.y) + row * g.ldy * size, rows * g.ldy * size, block * blockDim.x + threadIdx.x, blocks * blockDim.x);
}

struct ExpertTask {
    int expert;        // g.experts: rows that belong to none, which get zeros; -1: nothing to do
    int row, rows;     // first row of the tile, and rows from it to the expert's last
    int tn;
    bool half;         // the tile has edge / 2 rows
};

// Tile number `id` of those of `edge` rows: every XCD has a contiguous part of their sequence, which goes expert by expert and inside
// one in bands of eight tiles of rows, so that the workgroups resident on an XCD share their operands in its L2.  The same in all
// lanes of a wavefront, each of which looks at one expert of 64.  Rows in front of the first expert's get their zeros here, from all workgroups.
// HALVES: where the last round of one workgroup a CU would leave half of them idle or more, its tiles go in halves.  ([8192, 4096] by 4096 to 8 experts, bf16:
// 262 -> 243 us, rows' gradients 260 -> 241; e4m3 tiles of half the rows take too much of a whole one's time to gain.)
template <bool HALVES>
__device__ inline ExpertTask find_tile(const ExpertArgs& g, int edge, int id) {
    const int lane = threadIdx.x & 63;
    ExpertTask task{-1, 0, 0, 0, false};
    auto tiles_of = [&](int e, int& lo, int& n) {
        int hi = 0;
        lo = 0, n = 0;
        if (e <= g.experts) rows_of_expert(g, e, lo, hi), n = hi - lo;
        return (n + edge - 1) / edge;
    };
    int total = 0, lo, n;
    for (int e0 = 0; e0 <= g.experts; e0 += 64) {
        int t = tiles_of(e0 + lane, lo, n);
        const int front = e0 == 0 ? __builtin_amdgcn_readfirstlane(lo) : 0;
        if (front > 0) {
            zero_rows(g, 0, front, blockIdx.x, gridDim.x);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // a tile counts its own requests, and finds none of these
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) t += __shfl_xor(t, d);
        total += __builtin_amdgcn_readfirstlane(t);
    }
    const int all = total * g.tiles_n, per = all / kXcds, main = per * kXcds;
    int lower = 0;
    if (HALVES) {
        const int last = all % g.cus, whole = all - last;   // whole rounds: a multiple of the XCDs, as the CUs are
        if (id >= whole && 2 * last <= g.cus && g.cus % kXcds == 0) {
            const int nth = (id - whole) / kXcds;           // of this XCD
            id = whole + nth / 2 * kXcds + id % kXcds;
            task.half = true, lower = nth & 1;
        }
    }
    if (id >= all) return task;
    if (id < main) id = (id % kXcds) * per + id / kXcds;
    int before = 0;   // tiles of rows of the experts in front
    for (int e0 = 0; e0 <= g.experts; e0 += 64) {
        const int t = tiles_of(e0 + lane, lo, n);
        int run = t;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(run, d);
            if (lane >= d) run += v;
        }
        const int first = (before + run - t) * g.tiles_n, count = t * g.tiles_n;
        const uint64_t here = __ballot(id >= first && id < first + count);
        if (here) {
            const int l = __builtin_ctzll(here);
            const int rest = id - __builtin_amdgcn_readlane(first, l), tiles_m = __builtin_amdgcn_readlane(t, l);
            constexpr int kBand = 8;
            const int band = rest / (kBand * g.tiles_n), band_h = min(kBand, tiles_m - band * kBand), in_band = rest - band * kBand * g.tiles_n;
            const int skip = (band * kBand + in_band % band_h) * edge + lower * (edge / 2);
            task.row = __builtin_amdgcn_readlane(lo, l) + skip, task.rows = __builtin_amdgcn_readlane(n, l) - skip, task.tn = in_band / band_h;
            if (task.rows > 0) task.expert = e0 + l;
            break;
        }
        before += __builtin_amdgcn_readlane(run, 63);
    }
    return task;
}

struct MatrixTask {
    int expert, lo, hi;   // its rows
    int number, tm, tn;   // of the tile, in the order of the workgroups
};
// Tile `id` of those of the experts' matrices; false: there is none of that number.  Experts with many rows come first, so that the last
// tiles are short ones, and every XCD has an eighth of each expert's tiles side by side (of few tiles it takes them in turn): with an
// expert for each XCD, the one with most rows kept its XCD busy for 600 us of [16384, 4096 -> 3584] to 8 experts of 0 to 3200 rows, here 428.
__device__ inline bool find_matrix_tile(const ExpertArgs& g, int id, MatrixTask& task) {
    const int each = g.tiles_m * g.tiles_n;
    int place, rest, expert, lo, hi;
    if (each < 8 * kXcds) {
        place = id / each, rest = id - place * each;
    } else {
        const int xcd = id % kXcds, nth = id / kXcds, first = xcd * each / kXcds, share = (xcd + 1) * each / kXcds - first;
        place = nth / share, rest = first + nth % share;
    }
    if (place >= g.places) return false;
    expert = place;
    const int lane = threadIdx.x & 63;
    if (g.few >= 0) {   // in their order
        int before = 0;   // of them in front
        for (int e0 = 0;; e0 += 64) {
            if (e0 >= g.experts) return false;
            int from = 0, to = 0;
            if (e0 + lane < g.experts) rows_of_expert(g, e0 + lane, from, to);
            const uint64_t long_ones = __ballot(to - from > g.few);
            const uint64_t here = long_ones & __ballot(before + __popcll(long_ones & ((1ull << lane) - 1)) == place);
            if (here) {
                const int l = __builtin_ctzll(here);
                expert = e0 + l, lo = __builtin_amdgcn_readlane(from, l), hi = __builtin_amdgcn_readlane(to, l);
                break;
            }
            before += __popcll(long_ones);
        }
    } else if (g.experts <= 64) {   // a lane for each: how many have more rows, or as many and come before it; of those without rows, how many come before it
        int from = 0, to = 0;
        if (lane < g.experts) rows_of_expert(g, lane, from, to);
        const int rows = to - from;
        const uint64_t some = __ballot(rows > 0), none = __ballot(lane < g.experts && rows == 0);
        int ahead = __popcll(some);
        if (place >= ahead) {
            ahead += __popcll(none & ((1ull << lane) - 1));
            expert = __builtin_ctzll(none & __ballot(ahead == place));
        } else {
            ahead = 0;
            for (uint64_t left = some; left; left &= left - 1) {
                const int e = __builtin_ctzll(left), other = __builtin_amdgcn_readlane(rows, e);
                ahead += other > rows || (other == rows && e < lane);
            }
            expert = __builtin_ctzll(some & __ballot(ahead == place));
        }
        lo = __builtin_amdgcn_readlane(from, expert), hi = __builtin_amdgcn_readlane(to, expert);
    } else {
        rows_of_expert(g, expert, lo, hi);
    }
    constexpr int kBand = 8;
    const int band = rest / (kBand * g.tiles_n), band_h = min(kBand, g.tiles_m - band * kBand), in_band = rest - band * kBand * g.tiles_n;
    const auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };   // so that the compiler knows it
    task = {same(expert), same(lo), same(hi), same(rest), same(band * kBand + in_band % band_h), same(in_band / band_h)};
    return true;
}
// Workgroups that find_matrix_tile needs.
inline int64_t matrix_blocks(const ExpertArgs& g) {
    const int64_t each = static_cast<int64_t>(g.tiles_m) * g.tiles_n;
    return each < 8 * kXcds ? each * g.places : (each + kXcds - 1) / kXcds * kXcds * g.places;
}

// Zeros in `rows` rows of `cols` elements from y on, by all threads of the workgroup: 32 of them for a row.
template <typename E>
__device__ inline void zero_block(E* y, int64_t ldy, int rows, int cols) {
    for (int r = threadIdx.x / 32; r < rows; r += blockDim.x / 32) zero_run(reinterpret_cast<char*>(y + r * ldy), cols * static_cast<int64_t>(sizeof(E)), threadIdx.x % 32, 32);
}

// Zeros in this workgroup's part of an expert's matrix, where all of its tiles' are: parts that lie side by side in the order of the workgroups, in whole lines
// (25 of [26 x 4384, 2296] fp32: 320 us tile by tile, 194 in the tiles' order, here 176: 6.0 TB/s).
template <typename E>
__device__ inline void zero_part(const ExpertArgs& g, const MatrixTask& t) {
    const int64_t bytes = g.n * g.k * static_cast<int64_t>(sizeof(E)), each = static_cast<int64_t>(g.tiles_m) * g.tiles_n;
    const int64_t part = (bytes / each + 128) / 128 * 128, from = part * t.number;
    if (from < bytes) zero_run(static_cast<char*>(g.y) + t.expert * bytes + from, min(part, bytes - from), threadIdx.x, blockDim.x);
}

}  // namespace
#endif

}  // namespace ddl
#endif  // DDL_EXPERT_PARTS_H
