// 16-bit products of operands at any address and pitch, for sizes that the large
// tiles and the copies they need in front of them are too much for:
// y[M,N] = a[M,K] . b[N,K]^T + bias[N], operand layouts and arithmetic as in
// linear_gemm.hip (fp32 accumulation, one rounding to the result's type).
//
// gemm16_any (tiles of 64 x 64 or 128 x 128, k-tiles of 64, four wavefronts).
//   Requests into LDS want 4-byte alignment, so a tile comes through registers, 16
//   bytes a lane at any address, and goes into LDS in the layouts of linear_gemm.hip.
//   Bound by a k-tile's latencies while a CU has one workgroup and by LDS and the L1
//   when it has more: what matters is that loads stay in flight.  So the loop has no
//   branch and no masked load: tile i + 2 is requested while tile i is multiplied, one
//   barrier per k-tile, the LDS writes of tile i + 1 between the MFMAs of the second
//   half.  A tile that needs care (K ends in it, or its last chunk would run past the
//   operand) is taken first: its pieces are read from where they still lie inside and
//   shifted (drop), once, ahead of the loop.  With that care inside the loop the
//   compiler waits for every load in flight.  M 2276, N 456, K 3299 (training step of
//   the all-gather linear layer): y 46.3 -> 24.8 us, dx 36.6 -> 20.5, dw 28.4 -> 24.1;
//   M 564, N 1060, K 6838: 30.8 -> 25.9, 29.5 -> 23.5, 39.1 -> 18.2.
//   Tiles of 128 x 128 move half the bytes per flop (0.6 us per k-tile and CU against
//   1.0 for four of 64 x 64), smaller ones fill the chip: see plan_any16.
//
// linear16_adjoint (dx, dw and db of a linear shard).
//   Bound by launches and by CUs that have nothing to do: each of the three leaves most of the
//   chip idle when it is small, and waits for the one before.  Workgroups of all of them in one
//   launch, the product with the longer workgroups first: M 336, N 77, K 603 bf16 14.6 -> 5.7 us,
//   M 120, N 2258, K 3584 41.7 -> 15.4, M 718, N 821, K 5156 60.2 -> 32.8, M 1024, N 4096, K 1024
//   (aligned, before: requests into LDS, tiles of 128 x 256) 38.3 -> 30.0.  See plan_adjoint16.
//
// gemm16_thin (K below 8, at least one operand read along k).
//   A reduction shorter than a 16-byte load.  Bound by the result's stores; an output
//   element per lane.
#include "gemm16_any.h"
#include <type_traits>

namespace ddl {
namespace {

// Two workgroups of 128 x 128 tiles share a CU (64 KiB of LDS and 256 registers each), four of 64 x 64.
template <bool F16, bool XT, bool WT, int T>
__global__ __launch_bounds__(kAnyThreads, T == 2 ? 2 : 4) void gemm16_any(const Part16 p, int splits, float* __restrict__ partial) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    any_product<F16, XT, WT, T>(p, blockIdx.x, splits, partial, lds);
}

// The adjoint of a linear shard in one launch: dx = dy . w and dw = dy^T . x by tiles of 64 TX and 64 TW, db = column sums of dy.
struct Adjoint16 {
    Part16 dx, dw;
    int splits_x, splits_w, blocks_x, blocks_w;   // workgroups of the products; of the sums of their splits
    int first_w;                                  // dw's workgroups come first
    float *partial_x, *partial_w;
    const uint16_t* dy;
    int64_t rows, cols, lddy;
    void* db;
    int strips;
};

template <bool F16, int TX, int TW>
__global__ __launch_bounds__(kAnyThreads, TX == 2 || TW == 2 ? 2 : 4) void linear16_adjoint(const Adjoint16 p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    // Few strips of column sums come first, each a long chain of loads; many would keep the products waiting.
    const int products = p.blocks_x + p.blocks_w, first = p.strips <= kFirstStrips ? p.strips : 0;
    const int b = static_cast<int>(blockIdx.x) - first, x = p.first_w ? b - p.blocks_w : b, w = p.first_w ? b : b - p.blocks_x;
    if (b < 0 || b >= products) {
        typedef typename Elem<F16 ? 1 : 0>::type T;
        colsum_strip<F16 ? 1 : 0, kAnyThreads, 4>(reinterpret_cast<const T*>(p.dy), p.rows, p.cols, p.lddy, static_cast<T*>(p.db), b < 0 ? blockIdx.x : b - products,
                                                   p.strips, lds);
    } else if (x >= 0 && x < p.blocks_x) {
        any_product<F16, false, true, TX>(p.dx, x, p.splits_x, p.partial_x, lds);
    } else {
        any_product<F16, true, true, TW>(p.dw, w, p.splits_w, p.partial_w, lds);
    }
}

// The sums of the splits of both products; a product in one piece has no workgroups.
template <bool F16, int TX, int TW>
__global__ __launch_bounds__(256) void linear16_adjoint_sum(const Adjoint16 p, int blocks_x) {
    const int b = blockIdx.x;
    if (b < blocks_x) sum_splits<F16, 2, 2, 2 * TX, 2 * TX>(p.dx, p.splits_x, p.partial_x, b);
    else sum_splits<F16, 2, 2, 2 * TW, 2 * TW>(p.dw, p.splits_w, p.partial_w, b - blocks_x);
}

template <bool F16, int TX, int TW>
int launch_adjoint(const Adjoint16& p, hipStream_t s) {
    constexpr int lds_bytes = 4 * 64 * (TX > TW ? TX : TW) * kRowBytes;
    static_assert(colsum_lds_bytes(0, kAnyThreads) <= lds_bytes, "the column sums do not fit");
    hipLaunchKernelGGL((linear16_adjoint<F16, TX, TW>), dim3(static_cast<uint32_t>(p.blocks_x + p.blocks_w + p.strips)), dim3(kAnyThreads), lds_bytes, s, p);
    if (int rc = check_launch("linear16_adjoint")) return rc;
    const int sum_x = p.splits_x > 1 ? p.blocks_x / p.splits_x * 4 * TX * TX : 0, sum_w = p.splits_w > 1 ? p.blocks_w / p.splits_w * 4 * TW * TW : 0;
    if (sum_x + sum_w == 0) return 0;
    hipLaunchKernelGGL((linear16_adjoint_sum<F16, TX, TW>), dim3(static_cast<uint32_t>(sum_x + sum_w)), dim3(256), 0, s, p, sum_x);
    return check_launch("linear16_adjoint_sum");
}

template <bool F16>
__global__ __launch_bounds__(kAnyThreads) void gemm16_thin(const Part16 p, int64_t x_row, int64_t x_k, int64_t w_row, int64_t w_k, int64_t strips) {
    const int64_t m = blockIdx.x / strips, n = (blockIdx.x - m * strips) * kAnyThreads + threadIdx.x;
    if (n >= p.N) return;
    float v = 0.f;
    for (int64_t k = 0; k < p.K; ++k) v = fmaf(elem_to_f32<F16>(p.x[m * x_row + k * x_k]), elem_to_f32<F16>(p.w[n * w_row + k * w_k]), v);
    if (p.bias) v += elem_to_f32<F16>(p.bias[n]);
    p.y[m * p.ldy + n] = f32_to_elem<F16>(v);
}

template <bool F16, bool XT, bool WT, int T>
int launch_tiles(Part16 part, int splits, float* partial, hipStream_t s) {
    part.tiles_m = static_cast<int>((part.M + 64 * T - 1) / (64 * T)), part.tiles_n = static_cast<int>((part.N + 64 * T - 1) / (64 * T));
    const int ntiles = part.tiles_m * part.tiles_n;
    hipLaunchKernelGGL((gemm16_any<F16, XT, WT, T>), dim3(static_cast<uint32_t>(ntiles * splits)), dim3(kAnyThreads), 4 * 64 * T * kRowBytes, s, part,
                       splits, partial);
    if (int rc = check_launch("gemm16_any")) return rc;
    if (splits == 1) return 0;
    hipLaunchKernelGGL((gemm16_small_sum<F16, 2, 2, 2 * T, 2 * T>), dim3(static_cast<uint32_t>(ntiles * 4 * T * T)), dim3(256), 0, s, part, splits,
                       static_cast<const float*>(partial));
    return check_launch("gemm16_small_sum");
}

template <bool F16, bool XT, bool WT>
int launch_edge(const Small16& plan, const Part16& part, float* partial, hipStream_t s) {
    return plan.edge == 2 ? launch_tiles<F16, XT, WT, 2>(part, plan.splits, partial, s) : launch_tiles<F16, XT, WT, 1>(part, plan.splits, partial, s);
}

template <bool F16>
int launch(const Small16& plan, bool xt, bool wt, const Part16& part, float* partial, hipStream_t s) {
    if (plan.kind == Small16::kThin) {
        const int64_t strips = (part.N + kAnyThreads - 1) / kAnyThreads;
        hipLaunchKernelGGL((gemm16_thin<F16>), dim3(static_cast<uint32_t>(part.M * strips)), dim3(kAnyThreads), 0, s, part, xt ? 1 : part.ldx,
                           xt ? part.ldx : 1, wt ? 1 : part.ldw, wt ? part.ldw : 1, strips);
        return check_launch("gemm16_thin");
    }
    if (xt && wt) return launch_edge<F16, true, true>(plan, part, partial, s);
    if (xt) return launch_edge<F16, true, false>(plan, part, partial, s);
    if (wt) return launch_edge<F16, false, true>(plan, part, partial, s);
    return launch_edge<F16, false, false>(plan, part, partial, s);
}

}  // namespace

// Fits of a sweep over M 16 .. 8192, N 16 .. 12000, K 32 .. 8192 in the three layouts of a training step (28 000 products,
// 11 % off in the mean, picks 2.5 % behind the best of all ways measured), microseconds:
//   64 x 64    4.1 + 0.25 per k-tile and workgroup of a CU + 0.85 for every workgroup of a CU beyond the first; 8 % more where
//              not all are resident
//   128 x 128  6.1 + 0.62 and 2.5; 17 % more
//   splits     2.5 for the second launch and 3 for what it costs the host + the partial tiles, written and read, at 8 TB/s
//   at least   3 + operands and result once at 6 TB/s
// A CU works through whole workgroups while all are resident (four of 64 x 64, two of 128 x 128), else they even out.
// The other way -- operands copied into padded or transposed temporaries -- is 12 us of launches in front of the product plus
// the copies at 4.5 TB/s.  Measured among other steps, copies and product -> here: y of M 7001, N 1027, K 1001 42.4 -> 32.5 us,
// M 8191, N 1001, K 2051 59.0 -> 54.0; M 6001, N 1501, K 3001 71.7, here 105; M 4097, N 2049, K 2049 61, here 80.
Small16 plan_any16(bool xt, bool wt, int64_t M, int64_t N, int64_t K, int cus, int64_t workspace, double large_us) {
    Small16 best;
    double best_us = 12 + large_us + (static_cast<double>(M) + N) * K * 4 / 4.5e6;
    if (K < 8 && !(xt && wt)) {
        const int64_t strips = (N + kAnyThreads - 1) / kAnyThreads;
        if (strips <= 0xFFFFFF / M && 3 + static_cast<double>(M) * N / 2e6 < best_us) best.kind = Small16::kThin;
        return best;
    }
    const int64_t ktiles = (K + kAnyDepth - 1) / kAnyDepth;
    const double once_us = 3 + ((static_cast<double>(M) + N) * K + static_cast<double>(M) * N) * 2 / 6e6;
    for (const int edge : {1, 2}) {
        const int64_t tiles = ((M + 64 * edge - 1) / (64 * edge)) * ((N + 64 * edge - 1) / (64 * edge));
        const int64_t resident = edge == 1 ? 4 : 2, floats = edge * edge * 4096;
        if (tiles > 16 * static_cast<int64_t>(cus)) continue;
        for (const int splits : {1, 2, 3, 4, 6, 8, 12, 16}) {
            const int64_t workgroups = tiles * splits;
            if (splits > 1 && (workgroups > resident * cus || ktiles < 2 * splits || workgroups * floats > workspace)) break;
            const int64_t per_cu = (workgroups + cus - 1) / cus, steps = (ktiles + splits - 1) / splits;
            const double even = static_cast<double>(workgroups) / cus + 0.5;
            const double load = per_cu <= resident ? per_cu : even > resident ? even : resident;
            double us = edge == 1 ? 4.1 + steps * 0.25 * load + 0.85 * (load - 1) : 6.1 + steps * 0.62 * load + 2.5 * (load - 1);
            if (load > resident) us *= edge == 1 ? 1.08 : 1.17;
            if (us < once_us) us = once_us;
            if (splits > 1) us += 5.5 + static_cast<double>(workgroups) * floats * 8 / 8e6;
            if (us >= best_us) continue;
            best_us = best.us = us;
            best.kind = Small16::kAny, best.edge = edge, best.splits = splits, best.workspace = splits > 1 ? workgroups * floats : 0;
        }
    }
    return best;
}

// Both products on one chip at the same time: a workgroup's k-tile takes what it does above, the rounds of all of them are
// shared by the CUs, and the longest one is the least it can take; 4.1 or 6.1 as above, 5.5 for the launch that adds splits.
// The other way is `apart_us` for the products and 4.5 for the column sum, and 3 for each of the two further launches, of
// which 2 are the host's, where that may be what a step waits for.
// The best of these is taken if it also holds against what they leave out (careful_us): a long reduction in one piece takes 1.55
// times as long where rows are not aligned, and where it is by far the longest it waits for the other product's workgroups while
// not all are resident; the column sums take up to 2 ns a row; large products one after the other take 1.15 times `apart_us`.
// Three launches and one, of calls that therefore stay with three: M 5848, N 24, K 1408 aligned 22.9 and 29.6 us, M 8983, N 47,
// K 1624 39.6 and 62.1, M 8572, N 137, K 827 39.9 and 69.6, M 9975, N 17, K 37 19.6 and 28.2.  GPU time of 2204 calls for which
// the first estimate is for one launch (M 16 .. 16384, N 8 .. 8192, K 32 .. 8192, half of them aligned), in a replayed graph, which
// leaves out the host's share: 2069 take it, 1.5 times as fast as the three, 42 of them less than 0.95 times and at worst
// 0.79 (the former rule: 140 and 0.57); 12 of the 135 others would be faster by more than 5 % in one launch, at most 1.14 times.
// Of 1504 more calls with M above 2000, N up to 1024, drawn after the rule was made: 1312 take it, 1.3 times as fast, 75 less than 0.95
// times and at worst 0.62 (M 2146, N 19, K 931: 12.8 and 20.5 us; the former rule: 206 and 0.57), 24 of 192 lose, at most 1.24 times.
AdjointPlan16 plan_adjoint16(int64_t M, int64_t N, int64_t K, bool aligned, bool want_db, int cus, int64_t workspace, double apart_us) {
    AdjointPlan16 best;
    // operands along their rows have at least eight, dy read along n as well
    if (M < 8 || N < 8 || K < 8 || (want_db && M > kAdjointRows)) return best;
    const double launch_us = apart_us < 35 ? 3 : 1;
    const double other_us = apart_us + (want_db ? 4.5 + launch_us : 0) + launch_us;
    const int64_t strips = want_db ? (N + kNarrow - 1) / kNarrow : 0;
    double best_us = other_us, careful_us = 0;
    double least_us = 3 + 2 * (static_cast<double>(M) * N + (static_cast<double>(M) + N) * K * 2) / 6e6;   // operands and results once
    if (want_db && 4 + M * 0.0016 > least_us) least_us = 4 + M * 0.0016;                                       // one strip of the column sums
    for (int edges = 0; edges < 4; ++edges) {
        const int64_t ex = 1 + (edges & 1), ew = 1 + (edges >> 1);
        auto tiles = [](int64_t rows, int64_t cols, int64_t e) { return ((rows + 64 * e - 1) / (64 * e)) * ((cols + 64 * e - 1) / (64 * e)); };
        const int64_t tiles_x = tiles(M, K, ex), tiles_w = tiles(N, K, ew), kx = (N + kAnyDepth - 1) / kAnyDepth, kw = (M + kAnyDepth - 1) / kAnyDepth;
        const int64_t resident = (ex == 1 && ew == 1 ? 4 : 2) * static_cast<int64_t>(cus);
        if (tiles_x + tiles_w > 16 * static_cast<int64_t>(cus)) continue;
        const double cx = ex == 1 ? 0.25 : 0.62, cw = ew == 1 ? 0.25 : 0.62;
        for (const int sx : {1, 2, 3, 4, 6, 8}) {
            if (sx > 1 && (tiles_x * sx > resident || kx < 2 * sx)) break;
            for (const int sw : {1, 2, 3, 4, 6, 8}) {
                const int64_t bx = tiles_x * sx, bw = tiles_w * sw;
                const int64_t floats = (sx > 1 ? bx * ex * ex : 0) * 4096 + (sw > 1 ? bw * ew * ew : 0) * 4096;
                if ((sw > 1 && (bx + bw > resident || kw < 2 * sw)) || floats > workspace) break;
                const double nx = static_cast<double>((kx + sx - 1) / sx), nw = static_cast<double>((kw + sw - 1) / sw);
                const double all_x = bx * (nx * cx + (ex == 1 ? 0.85 : 2.5)) / cus, all_w = bw * (nw * cw + (ew == 1 ? 0.85 : 2.5)) / cus;
                const double all = (all_x + all_w) * 1.15, longest = nx * cx > nw * cw ? nx * cx : nw * cw;
                const double start_us = (ex == 1 && ew == 1 ? 4.1 : 6.1) + static_cast<double>(strips) / cus;
                const double sums_us = floats ? 5.5 + static_cast<double>(floats) * 8 / 8e6 : 0;
                double us = start_us + (all > longest ? all : longest);
                us = (us > least_us ? us : least_us) + sums_us;
                if (us >= best_us) continue;
                best_us = careful_us = us;
                best.edge_x = static_cast<int>(ex), best.edge_w = static_cast<int>(ew), best.splits_x = sx, best.splits_w = sw, best.workspace = floats;
                best.first_w = nw * cw > nx * cx;
                double chain = longest * (aligned ? 1 : 1.55);
                if (bx + bw > resident && chain > 1.5 * (all_x + all_w)) chain += 0.75 * (best.first_w ? all_x : all_w);
                for (const double t : {start_us + chain, want_db ? 4 + M * 0.002 : 0}) careful_us = t + sums_us > careful_us ? t + sums_us : careful_us;
            }
        }
    }
    return careful_us < (apart_us < 35 ? 1 : 1.15) * other_us ? best : AdjointPlan16{};
}

int run_adjoint16(const AdjointPlan16& plan, bool f16, const Part16& dx, const Part16& dw, void* db, float* workspace, hipStream_t s) {
    Adjoint16 p{};
    p.dx = dx, p.dw = dw, p.splits_x = plan.splits_x, p.splits_w = plan.splits_w, p.first_w = plan.first_w;
    auto tile = [](Part16& part, int edge) {
        part.tiles_m = static_cast<int>((part.M + 64 * edge - 1) / (64 * edge)), part.tiles_n = static_cast<int>((part.N + 64 * edge - 1) / (64 * edge));
        return part.tiles_m * part.tiles_n;
    };
    p.blocks_x = tile(p.dx, plan.edge_x) * plan.splits_x, p.blocks_w = tile(p.dw, plan.edge_w) * plan.splits_w;
    p.partial_x = workspace, p.partial_w = workspace + (plan.splits_x > 1 ? static_cast<int64_t>(p.blocks_x) * plan.edge_x * plan.edge_x * 4096 : 0);
    p.dy = dx.x, p.rows = dx.M, p.cols = dx.K, p.lddy = dx.ldx, p.db = db;
    p.strips = db ? static_cast<int>((p.cols + kNarrow - 1) / kNarrow) : 0;
    const int kind = (f16 ? 4 : 0) + (plan.edge_x == 2 ? 2 : 0) + (plan.edge_w == 2 ? 1 : 0);
    switch (kind) {
        case 0: return launch_adjoint<false, 1, 1>(p, s);
        case 1: return launch_adjoint<false, 1, 2>(p, s);
        case 2: return launch_adjoint<false, 2, 1>(p, s);
        case 3: return launch_adjoint<false, 2, 2>(p, s);
        case 4: return launch_adjoint<true, 1, 1>(p, s);
        case 5: return launch_adjoint<true, 1, 2>(p, s);
        case 6: return launch_adjoint<true, 2, 1>(p, s);
        default: return launch_adjoint<true, 2, 2>(p, s);
    }
}

int run_any16(const Small16& plan, bool f16, bool xt, bool wt, const Part16& part, float* partial, hipStream_t s) {
    return f16 ? launch<true>(plan, xt, wt, part, partial, s) : launch<false>(plan, xt, wt, part, partial, s);
}

}  // namespace ddl
