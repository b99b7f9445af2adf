// The experts' products of 32-bit elements: the 64 x 64 tiles of linear_f32_small.hip, and its 32 x 32 ones whose reduction four groups of a wavefront share,
// at any address and pitch, handed out expert by expert as expert_linear16.hip does with the 16-bit ones.  Sums are folded every 32 rounds: [2576, 7055]
// by 220 is off by 5.7e-7 of its 2-norm, in one chain 1.5e-6.
#include "expert_parts.h"
#include "gemm32_tiles.h"

namespace ddl {
namespace {

// Two stages leave room for a second workgroup on a CU, which hides more than two stages more ([2048, 1024] by 1024 to eight experts 56 -> 53 us, weights' gradients of [512, 1024] by 4096
// 105 -> 82; 32 x 32 tiles, sixteen rows to each of eight experts of [2048, 2048], 27 -> 23).
constexpr int kStages32 = 2;
constexpr int groups_of(int edge) { return edge == 64 ? 1 : 4; }
constexpr int lds_of(int edge) { return groups_of(edge) * kStages32 * 2 * edge * kRowBytes; }

template <int EDGE, bool WT>
__global__ __launch_bounds__(256) void expert_rows32(const ExpertArgs g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const ExpertTask t = find_tile<false>(g, EDGE, blockIdx.x);
    if (t.expert < 0) return;
    const int64_t n0 = static_cast<int64_t>(t.tn) * EDGE;
    float* const y = static_cast<float*>(g.y) + t.row * g.ldy + n0;
    if (t.expert == g.experts) {
        zero_block(y, g.ldy, min(t.rows, EDGE), static_cast<int>(min(g.n - n0, static_cast<int64_t>(EDGE))));
        return;
    }
    Part32 p{};
    p.x = static_cast<const float*>(g.a) + t.row * g.lda;
    p.w = static_cast<const float*>(g.w) + t.expert * g.w_stride + (WT ? n0 : n0 * g.ldw);
    p.y = y, p.M = t.rows, p.N = g.n - n0, p.K = g.k, p.ldx = g.lda, p.ldw = g.ldw, p.ldy = g.ldy, p.tiles_m = p.tiles_n = 1;
    small_product<false, WT, EDGE / 32, EDGE / 32, groups_of(EDGE), kStages32, true>(p, 0, 1, nullptr, lds);
}

template <int EDGE>
__global__ __launch_bounds__(256) void expert_weights32(const ExpertArgs g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    MatrixTask t;
    if (!find_matrix_tile(g, blockIdx.x, t)) return;
    if (t.lo == t.hi) {
        zero_part<float>(g, t);
        return;
    }
    const int64_t m0 = static_cast<int64_t>(t.tm) * EDGE, n0 = static_cast<int64_t>(t.tn) * EDGE;
    Part32 p{};
    p.x = static_cast<const float*>(g.a) + t.lo * g.lda + m0;
    p.w = static_cast<const float*>(g.w) + t.lo * g.ldw + n0;
    p.y = static_cast<float*>(g.y) + t.expert * g.n * g.k + m0 * g.k + n0;
    p.M = g.n - m0, p.N = g.k - n0, p.K = t.hi - t.lo, p.ldx = g.lda, p.ldw = g.ldw, p.ldy = g.k, p.tiles_m = p.tiles_n = 1;
    small_product<true, true, EDGE / 32, EDGE / 32, groups_of(EDGE), kStages32, true>(p, 0, 1, nullptr, lds);
}

template <int EDGE, typename Kernel>
int launch32(const char* who, Kernel kernel, const ExpertArgs& g, int64_t blocks, hipStream_t s) {
    if (blocks * 256 > 0xFFFFFFFFll) return fail(DDL_E_UNSUPP, "%s: %lld tiles", who, static_cast<long long>(blocks));
    static_assert(lds_of(EDGE) <= 64 * 1024, "what a launch gets without asking");
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(256), lds_of(EDGE), s, g);
    return check_launch(who);
}

template <int EDGE, bool WT>
int launch_rows32(const char* who, ExpertArgs g, hipStream_t s) {
    g.tiles_n = static_cast<int>((g.n + EDGE - 1) / EDGE);
    return launch32<EDGE>(who, expert_rows32<EDGE, WT>, g, ((g.rows + EDGE - 1) / EDGE + g.experts) * static_cast<int64_t>(g.tiles_n), s);
}

template <int EDGE>
int launch_weights32(const char* who, ExpertArgs g, hipStream_t s) {
    g.tiles_m = static_cast<int>((g.n + EDGE - 1) / EDGE), g.tiles_n = static_cast<int>((g.k + EDGE - 1) / EDGE);
    return launch32<EDGE>(who, expert_weights32<EDGE>, g, matrix_blocks(g), s);
}

}  // namespace

int run_expert_rows32(const char* who, bool small, bool transposed, const ExpertArgs& g, hipStream_t s) {
    if (small) return transposed ? launch_rows32<32, true>(who, g, s) : launch_rows32<32, false>(who, g, s);
    return transposed ? launch_rows32<64, true>(who, g, s) : launch_rows32<64, false>(who, g, s);
}

int run_expert_weights32(const char* who, bool small, const ExpertArgs& g, hipStream_t s) {
    return small ? launch_weights32<32>(who, g, s) : launch_weights32<64>(who, g, s);
}

}  // namespace ddl
