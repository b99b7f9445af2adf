// The experts' products of 32-bit elements: the 64 x 64 tiles of linear_f32_small.hip at any address and pitch, handed out expert by
// expert as expert_linear16.hip does with the 16-bit ones.
#include "expert_parts.h"
#include "gemm32_tiles.h"

namespace ddl {
namespace {

constexpr int kEdge32 = 64, kStages32 = 4, kLds32 = kStages32 * 2 * kEdge32 * kRowBytes;

template <bool WT>
__global__ __launch_bounds__(256) void expert_rows32(const ExpertArgs g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const ExpertTask t = find_tile<false>(g, kEdge32, blockIdx.x);
    if (t.expert < 0) return;
    const int64_t n0 = static_cast<int64_t>(t.tn) * kEdge32;
    float* const y = static_cast<float*>(g.y) + t.row * g.ldy + n0;
    if (t.expert == g.experts) {
        zero_block(y, g.ldy, 0, min(t.rows, kEdge32), 0, static_cast<int>(min(g.n - n0, static_cast<int64_t>(kEdge32))));
        return;
    }
    Part32 p{};
    p.x = static_cast<const float*>(g.a) + t.row * g.lda;
    p.w = static_cast<const float*>(g.w) + t.expert * g.w_stride + (WT ? n0 : n0 * g.ldw);
    p.y = y, p.M = t.rows, p.N = g.n - n0, p.K = g.k, p.ldx = g.lda, p.ldw = g.ldw, p.ldy = g.ldy, p.tiles_m = p.tiles_n = 1;
    small_product<false, WT, 2, 2, 1, kStages32>(p, 0, 1, nullptr, lds);
}

__global__ __launch_bounds__(256) void expert_weights32(const ExpertArgs g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int e, tm, tn, lo, hi;
    if (!find_matrix_tile(g, blockIdx.x, e, tm, tn)) return;
    rows_of_expert(g, e, lo, hi);
    lo = __builtin_amdgcn_readfirstlane(lo), hi = __builtin_amdgcn_readfirstlane(hi);
    const int64_t m0 = static_cast<int64_t>(tm) * kEdge32, n0 = static_cast<int64_t>(tn) * kEdge32;
    float* const y = static_cast<float*>(g.y) + e * g.n * g.k + m0 * g.k + n0;
    if (lo == hi) {
        zero_block(y, g.k, 0, static_cast<int>(min(g.n - m0, static_cast<int64_t>(kEdge32))), 0, static_cast<int>(min(g.k - n0, static_cast<int64_t>(kEdge32))));
        return;
    }
    Part32 p{};
    p.x = static_cast<const float*>(g.a) + lo * g.lda + m0;
    p.w = static_cast<const float*>(g.w) + lo * g.ldw + n0;
    p.y = y, p.M = g.n - m0, p.N = g.k - n0, p.K = hi - lo, p.ldx = g.lda, p.ldw = g.ldw, p.ldy = g.k, p.tiles_m = p.tiles_n = 1;
    small_product<true, true, 2, 2, 1, kStages32>(p, 0, 1, nullptr, lds);
}

template <typename Kernel>
int launch32(const char* who, Kernel kernel, const ExpertArgs& g, int64_t blocks, hipStream_t s) {
    if (blocks * 256 > 0xFFFFFFFFll) return fail(DDL_E_UNSUPP, "%s: %lld tiles", who, static_cast<long long>(blocks));
    static_assert(kLds32 <= 65536, "more LDS than a launch gets without asking");
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(256), kLds32, s, g);
    return check_launch(who);
}

}  // namespace

int run_expert_rows32(const char* who, bool transposed, ExpertArgs g, hipStream_t s) {
    g.tiles_n = static_cast<int>((g.n + kEdge32 - 1) / kEdge32);
    const int64_t blocks = ((g.rows + kEdge32 - 1) / kEdge32 + g.experts) * static_cast<int64_t>(g.tiles_n);
    return transposed ? launch32(who, expert_rows32<true>, g, blocks, s) : launch32(who, expert_rows32<false>, g, blocks, s);
}

int run_expert_weights32(const char* who, ExpertArgs g, hipStream_t s) {
    g.tiles_m = static_cast<int>((g.n + kEdge32 - 1) / kEdge32), g.tiles_n = static_cast<int>((g.k + kEdge32 - 1) / kEdge32);
    return launch32(who, expert_weights32, g, matrix_blocks(g), s);
}

}  // namespace ddl
