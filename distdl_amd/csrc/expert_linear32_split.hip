// The experts' products of 32-bit elements in large: the 128 x 128 tiles of linear_f32_split.hip, handed out expert by expert as
// expert_linear16.hip does with the 16-bit ones.
#include "expert_parts.h"
#include "gemm32_split.h"

namespace ddl {
namespace {

template <bool WT>
__global__ __launch_bounds__(kBlock, 2) void expert_rows32_split(const ExpertArgs g) {
    __shared__ __attribute__((aligned(16))) char lds[2 * kStage];
    const ExpertTask t = find_tile<false>(g, kTile, blockIdx.x);
    if (t.expert < 0) return;
    const int64_t n0 = static_cast<int64_t>(t.tn) * kTile;
    float* const y = static_cast<float*>(g.y) + t.row * g.ldy + n0;
    if (t.expert == g.experts) {
        zero_block(y, g.ldy, min(t.rows, kTile), static_cast<int>(min(g.n - n0, static_cast<int64_t>(kTile))));
        return;
    }
    Part32 p{};
    p.x = static_cast<const float*>(g.a) + t.row * g.lda;
    p.w = static_cast<const float*>(g.w) + t.expert * g.w_stride + (WT ? n0 : n0 * g.ldw);
    p.y = y, p.M = t.rows, p.N = g.n - n0, p.K = g.k, p.ldx = g.lda, p.ldw = g.ldw, p.ldy = g.ldy, p.tiles_m = p.tiles_n = 1;
    split_product<false, WT>(p, 0, 1, nullptr, lds);
}

__global__ __launch_bounds__(kBlock, 2) void expert_weights32_split(const ExpertArgs g) {
    __shared__ __attribute__((aligned(16))) char lds[2 * kStage];
    MatrixTask t;
    if (!find_matrix_tile(g, blockIdx.x, t)) return;
    if (t.lo == t.hi) {
        zero_part<float>(g, t);
        return;
    }
    const int64_t m0 = static_cast<int64_t>(t.tm) * kTile, n0 = static_cast<int64_t>(t.tn) * kTile;
    Part32 p{};
    p.x = static_cast<const float*>(g.a) + t.lo * g.lda + m0;
    p.w = static_cast<const float*>(g.w) + t.lo * g.ldw + n0;
    p.y = static_cast<float*>(g.y) + t.expert * g.n * g.k + m0 * g.k + n0;
    p.M = g.n - m0, p.N = g.k - n0, p.K = t.hi - t.lo, p.ldx = g.lda, p.ldw = g.ldw, p.ldy = g.k, p.tiles_m = p.tiles_n = 1;
    split_product<true, true>(p, 0, 1, nullptr, lds);
}

}  // namespace

int run_expert_rows32_split(const char* who, bool transposed, ExpertArgs g, hipStream_t s) {
    g.tiles_n = static_cast<int>((g.n + kTile - 1) / kTile);
    const int64_t blocks = ((g.rows + kTile - 1) / kTile + g.experts) * static_cast<int64_t>(g.tiles_n);
    if (blocks * kBlock > 0xFFFFFFFFll) return fail(DDL_E_UNSUPP, "%s: %lld tiles", who, static_cast<long long>(blocks));
    if (transposed) hipLaunchKernelGGL(expert_rows32_split<true>, dim3(static_cast<uint32_t>(blocks)), dim3(kBlock), 0, s, g);
    else hipLaunchKernelGGL(expert_rows32_split<false>, dim3(static_cast<uint32_t>(blocks)), dim3(kBlock), 0, s, g);
    return check_launch(who);
}

int run_expert_weights32_split(const char* who, ExpertArgs g, hipStream_t s) {
    g.tiles_m = static_cast<int>((g.n + kTile - 1) / kTile), g.tiles_n = static_cast<int>((g.k + kTile - 1) / kTile);
    const int64_t blocks = matrix_blocks(g);
    if (blocks * kBlock > 0xFFFFFFFFll) return fail(DDL_E_UNSUPP, "%s: %lld tiles", who, static_cast<long long>(blocks));
    hipLaunchKernelGGL(expert_weights32_split, dim3(static_cast<uint32_t>(blocks)), dim3(kBlock), 0, s, g);
    return check_launch(who);
}

}  // namespace ddl
