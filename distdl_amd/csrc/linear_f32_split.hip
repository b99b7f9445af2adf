// fp32 linear products on the bf16 matrix cores, without loss:
// y[M,N] = a[M,K] . b[N,K]^T + bias[N], fp32 in and out.
//
// An fp32 value is the sum of three bf16 values, exactly: its rounding to bf16, the
// rounding of what is left, and what is left then (8 + 8 + 8 significant bits), as
// published by Henry, Tang and Heinecke ("Leveraging the bfloat16 Artificial
// Intelligence Datatype For Higher-Precision Computations", 2019).  Elements are
// multiplied by 2^24 first: then no part of any of them, denormal ones included, is
// below bf16's normal range.  Of the nine products of two such sums the smallest is
// below 2^-33 of the product and left out; the other eight go through
// v_mfma_f32_32x32x16_bf16, which accumulates in fp32: 256 cycles for 32 x 32 x 16 where
// v_mfma_f32_32x32x2_f32 takes 512.
//
// The products of the first parts have an accumulator of their own; they are rounded
// once per 16 terms, and a term that is zero rounds nothing.  The seven others, together
// below 2^-7 of them, have a second one, added once at the end.  (All in one accumulator
// round once per part-product at its full size: 0.5 to 1.5 times the fp32 instruction's
// error, the more the fewer terms are not zero.  With the six largest products alone a
// sum of one term is 1.025 times as far off.)  Error against float64 in the 2-norm,
// fp32 instruction -> here, M = N = 1408, K 8192, share of x that is not zero: all 1.62e-6 -> 0.40e-6, a quarter
// 0.81e-6 -> 0.23e-6, a hundredth 0.164e-6 -> 0.055e-6, one element a row 0.0253e-6 both.
//
// Bound by the matrix instructions' power and, in small products, by issue: while a CU's
// wavefronts multiply, they split (seven instructions an element).  149 to 160 TFLOP/s
// in large products, where the fp32 instruction ends at 148 (M 8192, N 3584, K 8192 3.06 to
// 3.10 ms, its adjoint 3.10 and 3.22).  Measured, fp32 instruction (64 x 64 or
// 256 x 256 tiles) -> here, operands along k or along their rows: M 256, N 3551, K 6575
// 116 -> 101 to 106 us, M 3551, N 6575, K 256 147 to 169 -> 99 to 105, M = N = K = 2048 140 -> 122
// to 128, 4096 968 -> 858 to 897, M 1024, N 8192, K 8192 1050 to 1075 -> 861 to 903; below about 20 us
// the smaller tiles are faster.
//
//   workgroup  256 threads = 4 wavefronts (2 x 2), tile 128 x 128 x 16(k); a wavefront
//              has 2 x 2 blocks of 32 x 32
//   global     a thread fetches eight k of a row of each operand into registers, three
//              k-tiles ahead: 32 bytes of the row, or eight rows' worth of dwords for
//              an operand contiguous along its rows.  Any pitch, length and
//              4-byte-aligned address
//   LDS        every element is split once per workgroup, on its way into LDS: three
//              planes of rows of 32 bytes, halves swapped in eight rows of sixteen, so
//              that 16 lanes reading one half of 16 rows, or writing it, meet no bank
//              twice.  Two stages
//   splits     workgroups share the reduction of a tile through a workspace, whose
//              sums gemm32_small_sum adds
//
// What the parts cannot carry is found on the way: every thread keeps the largest
// magnitude that it fetches.  Tiles with infinities, elements from 2^100 on, or
// elements whose product times the length of the reduction reaches 2^78 (which scaled
// might pass the largest float) are computed again from memory on
// v_mfma_f32_32x32x2_f32.
#include "gemm32_split.h"

namespace ddl {
namespace {

template <bool XT, bool WT>
__global__ __launch_bounds__(kBlock, 2) void gemm32_split(const Part32 p, int splits, float* __restrict__ partial) {
    __shared__ __attribute__((aligned(16))) char lds[2 * kStage];
    split_product<XT, WT>(p, static_cast<int>(blockIdx.x), splits, partial, lds);
}

template <bool XT, bool WT>
int launch(Part32 part, int splits, float* partial, hipStream_t s) {
    part.tiles_m = static_cast<int>((part.M + kTile - 1) / kTile), part.tiles_n = static_cast<int>((part.N + kTile - 1) / kTile);
    hipLaunchKernelGGL((gemm32_split<XT, WT>), dim3(static_cast<uint32_t>(part.tiles_m * part.tiles_n * splits)), dim3(kBlock), 0, s, part, splits, partial);
    if (int rc = check_launch("gemm32_split")) return rc;
    return splits == 1 ? 0 : sum_small32(part, 4, splits, partial, s);
}

}  // namespace

// The estimates are fits to a sweep over M, N, K of 64 .. 8192 on all operand layouts, in microseconds: 6 + for each tile that a
// CU has to work through 4.5 and, per 32 of its reduction, 1.57 (few CUs at work) to 1.72 (all) + for splits a second launch (2.3,
// and 5 for what it and the workspace cost the host) and the partial tiles at 5 TB/s.  Over 66 sizes in three layouts the way they
// choose is on average 1.1 % slower than the faster of both kernels and all splits.
Small32 plan_split32(int64_t M, int64_t N, int64_t K, int cus, int64_t workspace, const Small32& other) {
    Small32 best;
    const int64_t ktiles = (K + kSplitDepth - 1) / kSplitDepth, tiles = ((M + kTile - 1) / kTile) * ((N + kTile - 1) / kTile);
    if (tiles > 0xFFFFFF) return best;   // a launch has fewer than 2^32 threads, 256 per tile
    double best_us = other.groups ? other.us : 1e30;
    for (const int splits : {1, 2, 3, 4, 6, 8, 12, 16}) {
        if (splits > 1 && (tiles * splits > 4 * static_cast<int64_t>(cus) || ktiles < 8 * splits || tiles * splits * kTile * kTile > workspace)) break;
        // Fewer, longer sums than the other way are only taken where this kernel's smaller rounding error makes up for it (0.24 to
        // 0.34 of the other's for dense sums of the same length; it grows by their square root).
        if (4 * splits < other.groups * other.splits) continue;
        const int64_t all = tiles * splits, per_cu = (all + cus - 1) / cus, kt = (ktiles + splits - 1) / splits;
        const double fill = all < cus ? static_cast<double>(all) / cus : 1.0;
        double us = 6 + per_cu * (4.5 + 0.5 * static_cast<double>(kt) * (1.57 + 0.15 * fill));
        if (splits > 1) us += 7.3 + static_cast<double>(all) * kTile * kTile * 8 / 5e6;
        if (us >= best_us) continue;
        best_us = best.us = us;
        best.edge = kTile, best.splits = splits, best.workspace = splits > 1 ? all * kTile * kTile : 0;
    }
    return best;
}

int run_split32(const Small32& plan, bool xt, bool wt, const PartOf<float>& part, float* partial, hipStream_t s) {
    if (xt && wt) return launch<true, true>(part, plan.splits, partial, s);
    if (xt) return launch<true, false>(part, plan.splits, partial, s);
    if (wt) return launch<false, true>(part, plan.splits, partial, s);
    return launch<false, false>(part, plan.splits, partial, s);
}

}  // namespace ddl
