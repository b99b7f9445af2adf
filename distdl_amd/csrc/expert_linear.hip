// The products of rows with the weights of the expert that each was sent to, and their adjoint: the entry points and the
// kernel for few rows.  (expert_linear8.hip, expert_linear16.hip, expert_linear32.hip, expert_linear32_split.hip: tiles; expert_across.hip, expert_outer.hip: gradients of few rows.)
//
// expert_stream (few rows for each expert): bound by reading the weights once.  A workgroup has 16 rows of one
// expert's weights; each of its wavefronts takes a part of the reduction, line after line of 128 bytes, straight from memory into
// registers as a matrix instruction wants them (lane l has bytes 16 (l / 16) and 64 + 16 (l / 16) on of row l % 16: which element of a reduction a
// lane holds is free if both operands agree), next to the same lines of up to 16 MB rows of the expert's.  The wavefronts' sums meet in
// LDS.  More rows than that take the weights' lines again, from the L2.  32 rows of 8192 to eight experts of 3584 (352 MB of
// weights) bf16: eight wavefronts 70 us (5.0 TB/s), four 79, the lines to the wavefronts in turn 76, 32 rows of weights 77 to 95; e4m3 with four
// wavefronts 39, with eight 42.
//
// e4m3 products: the matrix cores' own, which add eight of them at a time and cut each off at 2^-13 of the largest one's power of two, and
// those sums in 32 bits.  Of rows of normally distributed elements that is 2^-12 of a result, next to 2^-9 for its rounding to bf16
// and 2^-5 for the rows' own; bf16 products of the same codes would be exact at half the rate.
#include "expert_parts.h"
#include "gemm16_parts.h"
#include <math.h>

namespace ddl {
namespace {

// ------------------------------------------------------------ few rows --

enum Kind { kBf16, kF16, kE4m3, kF32 };

constexpr int kStreamCols = 16;
template <int KIND>
constexpr int kStreamWaves = KIND == kE4m3 ? 4 : 8;

struct Line {
    uint4 half[2];   // 16 bytes of either half
};
typedef int intx8 __attribute__((ext_vector_type(8)));

template <int KIND>
__device__ inline floatx4 multiply_line(const Line& w, const Line& x, floatx4 acc) {
    if constexpr (KIND == kE4m3) {
        intx8 a, b;
        __builtin_memcpy(&a, &w, 32);
        __builtin_memcpy(&b, &x, 32);
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, 0, 0x7F7F7F7F, 0, 0x7F7F7F7F);   // scales of one
    } else if constexpr (KIND == kF32) {
        float a[8], b[8];
        __builtin_memcpy(a, &w, 32);
        __builtin_memcpy(b, &x, 32);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
        return acc;
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            bf16x8 a, b;
            __builtin_memcpy(&a, &w.half[h], 16);
            __builtin_memcpy(&b, &x.half[h], 16);
            acc = mfma<KIND == kF16>(a, b, acc);
        }
        return acc;
    }
}

__device__ inline Line load_line(const char* p) {
    Line l;
    l.half[0] = *reinterpret_cast<const uint4*>(p), l.half[1] = *reinterpret_cast<const uint4*>(p + 64);
    return l;
}
// Those of its first `left` bytes from here on (a multiple of 16), zeros behind them.
__device__ inline Line load_line_end(const char* p, int left) {
    Line l;
    l.half[0] = left > 0 ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
    l.half[1] = left > 64 ? *reinterpret_cast<const uint4*>(p + 64) : make_uint4(0, 0, 0, 0);
    return l;
}

__device__ inline void store_out(const ExpertArgs& g, int64_t row, int64_t n, float v) {
    const int64_t at = row * g.ldy + n;
    if (g.out_dtype == DDL_DT_F32) static_cast<float*>(g.y)[at] = v;
    else static_cast<uint16_t*>(g.y)[at] = g.out_dtype == DDL_DT_F16 ? f32_to_elem<true>(v) : f32_to_elem<false>(v);
}

template <int KIND, int MB>
__global__ __launch_bounds__(64 * kStreamWaves<KIND>) void expert_stream(const ExpertArgs g) {
    constexpr int kWaves = kStreamWaves<KIND>, kAhead = 4;   // lines in flight together
    constexpr int kBytes = KIND == kE4m3 ? 1 : KIND == kF32 ? 4 : 2;
    __shared__ floatx4 sums[kWaves][MB][64];
    const int e = blockIdx.y;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kStreamCols;
    int lo, hi;
    rows_of_expert(g, e, lo, hi);
    if (e == g.experts) {   // rows of none: those behind the last expert's, and those in front of the first one's
        zero_rows(g, lo, hi - lo, blockIdx.x, gridDim.x);
        zero_rows(g, 0, min(max(g.offsets[0], 0), lo), blockIdx.x, gridDim.x);
        return;
    }
    if (lo == hi) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, part = lane >> 4;
    const int64_t bytes = g.k * kBytes;
    const int lines = static_cast<int>(bytes / 128), end = static_cast<int>(bytes % 128) - part * 16;
    // This wavefront's lines; the one that the rows end in may have some bytes, or none.
    const int share = (lines + kWaves) / kWaves, first = min(wave * share, lines + 1), last = min(first + share, lines + 1);
    const int64_t n = n0 + l16;
    const char* const w = static_cast<const char*>(g.w) + (e * g.w_stride + (n < g.n ? n : g.n - 1) * g.ldw) * kBytes + part * 16;
    const char* x[MB];
    for (int m0 = lo; m0 < hi; m0 += 16 * MB) {
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            const int64_t m = m0 + b * 16 + l16;
            x[b] = static_cast<const char*>(g.a) + (m < hi ? m : hi - 1) * g.lda * kBytes + part * 16;
        }
        floatx4 acc[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[b] = floatx4{0.f, 0.f, 0.f, 0.f};
        int i = first;
        for (; i + kAhead <= min(last, lines); i += kAhead) {
            Line lw[kAhead], lx[kAhead][MB];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int64_t at = static_cast<int64_t>(i + u) * 128;
                lw[u] = load_line(w + at);
#pragma unroll
                for (int b = 0; b < MB; ++b) lx[u][b] = load_line(x[b] + at);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
#pragma unroll
                for (int b = 0; b < MB; ++b) acc[b] = multiply_line<KIND>(lw[u], lx[u][b], acc[b]);
        }
        for (; i < last; ++i) {
            const int64_t at = static_cast<int64_t>(i) * 128;
            const int left = i < lines ? 128 : end;
            const Line lw = load_line_end(w + at, left);
#pragma unroll
            for (int b = 0; b < MB; ++b) acc[b] = multiply_line<KIND>(lw, load_line_end(x[b] + at, left), acc[b]);
        }
        if (m0 != lo) __syncthreads();   // the sums before these have been read
#pragma unroll
        for (int b = 0; b < MB; ++b) sums[wave][b][lane] = acc[b];
        __syncthreads();
        // Lane: row l16, columns 4 part to 4 part + 3 of a block of 16 x 16.
        for (int b = wave; b < MB; b += kWaves) {
            floatx4 v = sums[0][b][lane];
#pragma unroll
            for (int s = 1; s < kWaves; ++s) v += sums[s][b][lane];
            const int64_t m = m0 + b * 16 + l16, c = n0 + 4 * part;
            if (m >= hi) continue;
            const float scale = KIND == kE4m3 ? g.a_scales[m] : 1.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (c + j < g.n) store_out(g, m, c + j, KIND == kE4m3 ? v[j] * scale * g.w_scales[e * g.n + c + j] : v[j]);
            }
        }
    }
}

template <int KIND>
int launch_stream(const char* who, const ExpertArgs& g, hipStream_t s) {
    const int64_t strips = (g.n + kStreamCols - 1) / kStreamCols;
    if (strips > 0x7FFFFF || g.experts + 1 > 65535) return fail(DDL_E_UNSUPP, "%s: %lld columns of %d experts", who, static_cast<long long>(g.n), g.experts);
    const dim3 grid(static_cast<uint32_t>(strips), static_cast<uint32_t>(g.experts + 1)), block(64 * kStreamWaves<KIND>);
    const int64_t each = g.rows / (g.experts > 0 ? g.experts : 1);   // rows that a workgroup has at once: most experts' all
    if (each <= 8) hipLaunchKernelGGL((expert_stream<KIND, 1>), grid, block, 0, s, g);
    else if (each <= 24) hipLaunchKernelGGL((expert_stream<KIND, 2>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((expert_stream<KIND, 4>), grid, block, 0, s, g);
    return check_launch(who);
}

// ------------------------------------------------------------ dispatch --

constexpr int64_t kMostSpan = 0x3FFFFFFF;   // elements that a tile's 32-bit byte offsets reach over

// Estimates in microseconds, fits of sweeps over 1 to 64 experts, 512 to 8192 features and 2 to 2048 rows for each, which are taken to be spread evenly (choices that all go to
// one expert were no slower: 4096 rows to 128 of [512, 1024] 25 and 13 us).  A round is what the chip holds at once: four workgroups of 64 x 64 tiles for a CU, two of 128 x 128, one of the large
// ones, which come in whole rounds.  A round costs its start and its stores, and for each k-tile (128 bytes) some time of its own and some that grows with
// the CUs' load.  ([8 x 512, 8192] by 3584: 64 x 64 414 us, 128 x 128 282, 128 x 256 225, 256 x 256 184; of 64 rows each 99, 104, 126, 154.)
struct TileCost {
    ExpertTile tile;
    int bm, bn, side;             // side: workgroups on a CU
    double start, step, load;     // of a round, of a k-tile, of a k-tile on a full chip in addition
};
const TileCost kCosts16[4] = {{ExpertTile::kAny64, 64, 64, 4, 1.3, 0.20, 0.72},
                              {ExpertTile::kAny128, 128, 128, 2, 3, 0.55, 0.65},
                              {ExpertTile::kLow, 128, 256, 1, 4, 0.47, 0.41},
                              {ExpertTile::kLarge, 256, 256, 1, 7, 0.95, 0.45}};
const TileCost kCosts8[3] = {{ExpertTile::kAny64, 64, 64, 2, 3, 0.30, 0.22}, {ExpertTile::kLow, 128, 256, 1, 6, 0.58, 0.25}, {ExpertTile::kLarge, 256, 256, 1, 9, 0.98, 0.50}};

double tiles_us(const TileCost& c, double tiles, double ktiles, int cus) {
    const double rounds = tiles / (static_cast<double>(c.side) * cus);
    const double whole = rounds <= 1 ? 1 : c.side > 1 ? rounds : ceil(rounds);
    return 4 + whole * (c.start + ktiles * (c.step + c.load * (rounds < 1 ? rounds : 1)));
}

// Tiles of rows: on average every expert has one that is half empty.
double row_tiles(int64_t rows, int64_t experts, int bm) {
    const double half = 0.5 * static_cast<double>(experts < rows ? experts : rows);
    return static_cast<double>(rows) / bm + half;
}

// The quickest kind for `rows` sorted rows by matrices of `cols` columns, a reduction being `depth` bytes of either.
template <int N>
ExpertTile best_for_rows(const TileCost (&costs)[N], bool aligned, int64_t rows, int64_t experts, int64_t cols, int64_t depth, int cus, double* us) {
    ExpertTile best = costs[0].tile;
    *us = 1e30;
    for (const TileCost& c : costs) {
        if (!aligned && (c.tile == ExpertTile::kLow || c.tile == ExpertTile::kLarge)) continue;
        const double t = tiles_us(c, row_tiles(rows, experts, c.bm) * static_cast<double>((cols + c.bn - 1) / c.bn), (depth + kRowBytes - 1.0) / kRowBytes, cus);
        if (t < *us) *us = t, best = c.tile;
    }
    // whatever the tiles, the weights are read: 5.1 TB/s
    const double read = static_cast<double>(rows < experts ? rows : experts) * cols * depth / 5.1e6;
    if (read > *us) *us = read;
    return best;
}

ExpertTile best_for_weights(bool aligned, int64_t rows, int64_t experts, int64_t n, int64_t k, int cus) {
    ExpertTile best = ExpertTile::kAny64;
    double us = 1e30;
    for (const TileCost& c : kCosts16) {
        if (!aligned && (c.tile == ExpertTile::kLow || c.tile == ExpertTile::kLarge)) continue;
        const double tiles = static_cast<double>(experts) * ((n + c.bm - 1) / c.bm) * ((k + c.bn - 1) / c.bn);
        const double t = tiles_us(c, tiles, ceil(static_cast<double>(rows) / experts / 64), cus);
        if (t < us) us = t, best = c.tile;
    }
    return best;
}

// fp32: the edge of the quickest tiles, 128 (bf16 matrix cores, linear_f32_split.hip's own fit), 64 or 32 (fp32 cores).  Each CU's tiles one after the other, a start and some
// time for each 32 of the reduction, which four groups share in the smallest.  `tiles` gives their number for an edge.  ([1024, 8192] by 3584: 64 545 us, 128 468; [64, 4096] by 1024 to
// three experts: 64 71 us, 32 23.)
template <typename Tiles>
int best_edge32(Tiles&& tiles, int64_t depth, int cus, double* us) {
    const double steps = ceil(depth / 32.0), large = tiles(128), fill = large < cus ? large / cus : 1;
    auto turns = [&](double n) { return n < cus ? 1.0 : n / cus; };
    const double us128 = 6 + ceil(large / cus) * (4.5 + steps * (1.57 + 0.15 * fill)), us64 = 5 + turns(tiles(64)) * (1 + steps * 0.57),
                 us32 = 5 + turns(tiles(32)) * (1.5 + ceil(steps / 4) * 0.52);
    *us = fmin(us128, fmin(us64, us32));
    return us128 < us64 ? (us32 < us128 ? 32 : 128) : us32 < us64 ? 32 : 64;
}
// Experts that may have rows, at the most.
double used_experts(int64_t rows, int64_t experts) { return static_cast<double>(rows < experts ? rows : experts); }

// expert_stream for fp32: the weights at 5.5 TB/s, and for each row the 16 lines of rows that every strip of them reads again.  ([1, 8192] by 3584: tiles 39 us, here 21 (5.5 TB/s);
// eight rows to each of eight experts of [1000, 260] 8.1 and 4.7, sixteen of [2048, 2048] 24 and 37.)
bool streams32(const ExpertArgs& g, double tiles_us) {
    if (!aligned_to(g.a, 16) || !aligned_to(g.w, 16) || g.lda % 4 || g.k % 4 || g.rows > 64ll * g.experts) return false;
    const double bytes = used_experts(g.rows, g.experts) * g.n * g.k * 4, each = static_cast<double>(g.rows) / g.experts;
    return 2.5 + bytes / 5.5e6 * (1 + 0.06 * each) < fmax(tiles_us, bytes / 5.1e6);
}
int rows32(const char* who, bool transposed, const ExpertArgs& g, hipStream_t s) {
    const double used = used_experts(g.rows, g.experts);
    double us;
    const int edge = best_edge32([&](int e) { return fmax(row_tiles(g.rows, g.experts, e), used) * static_cast<double>((g.n + e - 1) / e); }, g.k, g.cus, &us);
    if (!transposed && streams32(g, us)) return launch_stream<kF32>(who, g, s);
    return edge == 128 ? run_expert_rows32_split(who, transposed, g, s) : run_expert_rows32(who, edge == 32, transposed, g, s);
}
// Matrices that tiles are chosen for: of the experts that can have too many rows for expert_outer a few do, and then have many.  (All 3000 rows of [128 x 512, 1024] fp32 to one expert: 108 us,
// with tiles for 46 experts of 65 rows 220.)
int64_t likely_places(const ExpertArgs& g) { return g.few < 0 ? g.experts : (g.places + 3) / 4; }
int weights32(const char* who, const ExpertArgs& g, bool within, hipStream_t s) {
    if (!within) return run_expert_weights32_split(who, g, s);   // whose offsets have 64 bits
    const int64_t places = likely_places(g);
    double us;
    const int edge = best_edge32([&](int e) { return static_cast<double>(places) * ((g.n + e - 1) / e) * ((g.k + e - 1) / e); }, g.rows / places, g.cus, &us);
    return edge == 128 ? run_expert_weights32_split(who, g, s) : run_expert_weights32(who, edge == 32, g, s);
}

// Gradients of the weights: experts with few rows go by expert_outer and the others, if there can be any, by tiles in a launch of their own.  Up to how many: where tiles take over if all
// experts have as many (expert_outer's matrix instructions wait for two loads each).  So where most are expected to be of the first kind, and where the second launch costs less than what the first one
// saves, a quarter of a microsecond a megabyte.  ([64 x 1024, 1024] of twelve rows each: fp32 158 -> 56 us, bf16 72 -> 23, of 48 145 -> 107 and 71 -> 30, of 256 317 -> 499 and 83 -> 62;
// [8 x 2048, 2048] of 512 bf16 48 -> 52.)
int few_rows(const ExpertArgs& g) { return g.out_dtype == DDL_DT_F32 ? 64 : 256; }
bool mostly_few(const ExpertArgs& g) {
    const int64_t size = g.out_dtype == DDL_DT_F32 ? 4 : 2;
    return g.rows <= (size == 4 ? 40 : 160) * static_cast<int64_t>(g.experts) && (g.rows <= few_rows(g) || g.experts * g.n * g.k * size >= 12 << 20) && g.n >= 4 && g.k * size >= 16;
}

// expert_stream: the weights at 5.5 TB/s, and the rows that every strip of them reads again; not for more rows than it has in registers.
double stream_us(int64_t rows, int64_t experts, int64_t cols, int64_t depth) {
    if (rows > 64 * experts) return 1e30;
    const double each = static_cast<double>(rows) / experts, used = static_cast<double>(rows < experts ? rows : experts);
    return 2.5 + used * cols * depth / 5.5e6 * (1 + 0.05 * (each > 4 ? each - 4 : 0));
}

// Gradients of rows: expert_across, which reads the weights again for every 16 rows, where no expert is expected to have more, and little is lost if one has them all.
bool few_for_all(const ExpertArgs& g) {
    return (g.rows <= 16 || (g.rows <= 8 * static_cast<int64_t>(g.experts) && g.rows <= 256)) && g.n * (g.out_dtype == DDL_DT_F32 ? 4 : 2) >= 16;
}

int check_product(const char* who, int64_t experts, int64_t rows, int64_t n, int64_t k, int64_t least) {
    if (experts < 0 || rows < 0 || n < 1 || k < 1)
        return fail(DDL_E_ARG, "%s: %lld experts, %lld rows, %lld x %lld features", who, static_cast<long long>(experts), static_cast<long long>(rows), static_cast<long long>(n),
                    static_cast<long long>(k));
    if (n < least || k < least) return fail(DDL_E_UNSUPP, "%s: %lld x %lld features (at least %lld)", who, static_cast<long long>(n), static_cast<long long>(k), static_cast<long long>(least));
    if (rows > 0x3FFFFFFF || experts > 65534 || n > 0x3FFFFF || k > 0x3FFFFF || (n + 64) * (k + 64) > kMostSpan / 2)
        return fail(DDL_E_UNSUPP, "%s: %lld experts of %lld x %lld features and %lld rows", who, static_cast<long long>(experts), static_cast<long long>(n), static_cast<long long>(k),
                    static_cast<long long>(rows));
    return 0;
}

// limited: fp32 weights' gradients of rows beyond 32-bit byte offsets are refused.
int product_backward(const char* who, bool limited, const void* dy, const void* x, const void* w, int dtype, const int32_t* offsets, int64_t experts, int64_t rows, int64_t n,
                     int64_t k, int64_t ld_dy, int64_t ld_x, void* dx, void* dw, void* stream) {
    if (dtype != DDL_DT_F32 && dtype != DDL_DT_BF16 && dtype != DDL_DT_F16) return fail(DDL_E_ARG, "%s: dtype %d", who, dtype);
    if (int rc = check_product(who, experts, rows, n, k, dtype == DDL_DT_F32 ? 1 : 8)) return rc;
    if ((dx && rows) || (dw && experts)) {
        if (!offsets || (rows && !dy) || (dx && experts && !w) || (dw && rows && !x)) return fail(DDL_E_ARG, "%s: null pointer", who);
    }
    if (rows > 1 && (ld_dy < n || (dw && ld_x < k))) return fail(DDL_E_ARG, "%s: pitch below %lld or %lld features", who, static_cast<long long>(n), static_cast<long long>(k));
    if (ld_dy > 0x3FFFFF || (dw && ld_x > 0x3FFFFF)) return fail(DDL_E_UNSUPP, "%s: pitch above 2^22 elements", who);
    const int64_t pitch_dy = rows > 1 ? ld_dy : n, pitch_x = rows > 1 ? ld_x : k;
    const int64_t span = (rows + 64) * (dw && pitch_x > pitch_dy ? pitch_x : pitch_dy);
    const bool within = span <= (dtype == DDL_DT_F32 ? kMostSpan / 2 : kMostSpan);
    if (limited && dw && experts && dtype == DDL_DT_F32 && !within)
        return fail(DDL_E_UNSUPP, "%s: %lld rows, %lld elements apart, are more than 2^31 bytes", who, static_cast<long long>(rows), static_cast<long long>(pitch_x > pitch_dy ? pitch_x : pitch_dy));
    int dev = 0;
    const int cus = compute_units(dev);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool f16 = dtype == DDL_DT_F16;
    ExpertArgs g{};
    g.offsets = offsets, g.experts = static_cast<int>(experts), g.rows = static_cast<int>(rows), g.out_dtype = dtype, g.cus = cus;
    if (dx && rows) {   // rows of n features by w read along its k columns
        ExpertArgs d = g;
        d.a = dy, d.w = w, d.y = dx, d.n = k, d.k = n, d.lda = pitch_dy, d.ldw = k, d.w_stride = n * k, d.ldy = k;
        int rc;
        if (few_for_all(d)) {
            rc = run_expert_across(who, d, s);
        } else if (dtype == DDL_DT_F32) {
            rc = rows32(who, true, d, s);
        } else {
            const bool aligned = aligned_to(dy, 16) && aligned_to(w, 16) && pitch_dy % 8 == 0 && n % 8 == 0 && k % 8 == 0;
            double us;
            rc = run_expert_rows16(who, best_for_rows(kCosts16, aligned, rows, experts, k, 2 * n, cus, &us), f16, true, d, dev, s);
        }
        if (rc) return rc;
    }
    if (dw && experts) {
        ExpertArgs d = g;
        d.a = dy, d.w = x, d.y = dw, d.n = n, d.k = k, d.lda = pitch_dy, d.ldw = pitch_x;
        d.places = d.experts, d.few = -1;
        if (mostly_few(d)) {
            d.few = few_rows(d), d.places = d.rows / (d.few + 1);   // so many can have more
            if (int rc = run_expert_outer(who, d, s)) return rc;
            if (d.places == 0) return 0;
        }
        if (dtype == DDL_DT_F32) return weights32(who, d, within, s);
        const bool aligned = aligned_to(dy, 16) && aligned_to(x, 16) && pitch_dy % 8 == 0 && pitch_x % 8 == 0 && n % 8 == 0 && k % 8 == 0 && within;
        return run_expert_weights16(who, best_for_weights(aligned, rows, likely_places(d), n, k, cus), f16, d, dev, s);
    }
    return 0;
}

}  // namespace
}  // namespace ddl

extern "C" {

int ddl_expert_linear(const void* x, const void* w, int dtype, const int32_t* offsets, int64_t experts, int64_t rows, int64_t n, int64_t k, int64_t ld_x, void* y,
                      void* stream) {
    using namespace ddl;
    const char* who = "ddl_expert_linear";
    if (dtype != DDL_DT_F32 && dtype != DDL_DT_BF16 && dtype != DDL_DT_F16) return fail(DDL_E_ARG, "%s: dtype %d", who, dtype);
    if (int rc = check_product(who, experts, rows, n, k, dtype == DDL_DT_F32 ? 1 : 8)) return rc;
    if (rows == 0) return 0;
    if (!x || !y || !offsets || (experts && !w)) return fail(DDL_E_ARG, "%s: null pointer", who);
    if (rows > 1 && ld_x < k) return fail(DDL_E_ARG, "%s: pitch below %lld features", who, static_cast<long long>(k));
    if (ld_x > 0x3FFFFF) return fail(DDL_E_UNSUPP, "%s: pitch above 2^22 elements", who);
    int dev = 0;
    const int cus = compute_units(dev);
    ExpertArgs g{};
    g.a = x, g.w = w, g.y = y, g.offsets = offsets, g.experts = static_cast<int>(experts), g.rows = static_cast<int>(rows), g.out_dtype = dtype, g.cus = cus;
    g.n = n, g.k = k, g.lda = rows > 1 ? ld_x : k, g.ldw = k, g.w_stride = n * k, g.ldy = n;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == DDL_DT_F32) return rows32(who, false, g, s);
    const bool aligned = aligned_to(x, 16) && aligned_to(w, 16) && g.lda % 8 == 0 && k % 8 == 0;
    double us;
    const ExpertTile tile = best_for_rows(kCosts16, aligned, rows, experts, n, 2 * k, cus, &us);
    if (aligned && (!experts || stream_us(rows, experts, n, 2 * k) < us)) return dtype == DDL_DT_F16 ? launch_stream<kF16>(who, g, s) : launch_stream<kBf16>(who, g, s);
    return run_expert_rows16(who, tile, dtype == DDL_DT_F16, false, g, dev, s);
}

int ddl_expert_linear_8bit(const void* x, const float* x_scales, const void* w, const float* w_scales, const int32_t* offsets, int64_t experts, int64_t rows,
                           int64_t n, int64_t k, int64_t ld_x, void* y, int out_dtype, void* stream) {
    using namespace ddl;
    const char* who = "ddl_expert_linear_8bit";
    if (out_dtype != DDL_DT_F32 && out_dtype != DDL_DT_BF16 && out_dtype != DDL_DT_F16) return fail(DDL_E_ARG, "%s: dtype %d of the result", who, out_dtype);
    if (int rc = check_product(who, experts, rows, n, k, 1)) return rc;
    if (rows == 0) return 0;
    if (!x || !x_scales || !y || !offsets || (experts && (!w || !w_scales))) return fail(DDL_E_ARG, "%s: null pointer", who);
    if (rows > 1 && ld_x < k) return fail(DDL_E_ARG, "%s: pitch below %lld features", who, static_cast<long long>(k));
    const int64_t pitch = rows > 1 ? ld_x : k;
    if (k % 16 || pitch % 16 || !aligned_to(x, 16) || !aligned_to(w, 16))
        return fail(DDL_E_ALIGN, "%s: rows of %lld elements, %lld apart: 16-byte aligned rows of a multiple of 16 elements are taken", who, static_cast<long long>(k),
                    static_cast<long long>(pitch));
    if (pitch > 0x3FFFFF) return fail(DDL_E_UNSUPP, "%s: pitch above 2^22 elements", who);
    ExpertArgs g{};
    g.a = x, g.w = w, g.y = y, g.offsets = offsets, g.a_scales = x_scales, g.w_scales = w_scales, g.experts = static_cast<int>(experts), g.rows = static_cast<int>(rows);
    g.out_dtype = out_dtype, g.n = n, g.k = k, g.lda = pitch, g.ldw = k, g.w_stride = n * k, g.ldy = n;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    int dev = 0;
    double us;
    g.cus = compute_units(dev);
    const ExpertTile tile = best_for_rows(kCosts8, true, rows, experts, n, k, g.cus, &us);
    if (!experts || stream_us(rows, experts, n, k) < us) return launch_stream<kE4m3>(who, g, s);
    return run_expert_rows8(who, tile, g, dev, s);
}

int ddl_expert_linear_backward(const void* dy, const void* x, const void* w, int dtype, const int32_t* offsets, int64_t experts, int64_t rows, int64_t n, int64_t k,
                               int64_t ld_dy, int64_t ld_x, void* dx, void* dw, void* stream) {
    return ddl::product_backward("ddl_expert_linear_backward", true, dy, x, w, dtype, offsets, experts, rows, n, k, ld_dy, ld_x, dx, dw, stream);
}

int ddl_expert_linear_backward_long(const void* dy, const void* x, const void* w, int dtype, const int32_t* offsets, int64_t experts, int64_t rows, int64_t n, int64_t k,
                                    int64_t ld_dy, int64_t ld_x, void* dx, void* dw, void* stream) {
    return ddl::product_backward("ddl_expert_linear_backward_long", false, dy, x, w, dtype, offsets, experts, rows, n, k, ld_dy, ld_x, dx, dw, stream);
}

}  // extern "C"
