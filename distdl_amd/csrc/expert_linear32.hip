// The experts' products of 32-bit elements: the 64 x 64 tiles of linear_f32_small.hip, and its 32 x 32 ones whose reduction four groups of a wavefront share,
// at any address and pitch, handed out expert by expert as expert_linear16.hip does with the 16-bit ones.  Sums are folded every 32 rounds: [2576, 7055]
// by 220 is off by 5.7e-7 of its 2-norm, in one chain 1.5e-6.
#include "expert_parts.h"
#include "gemm32_tiles.h"

namespace ddl {
namespace {

constexpr int kStages32 = 4;
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
    int e, tm, tn, lo, hi;
    if (!find_matrix_tile(g, blockIdx.x, e, tm, tn)) return;
    rows_of_expert(g, e, lo, hi);
    lo = __builtin_amdgcn_readfirstlane(lo), hi = __builtin_amdgcn_readfirstlane(hi);
    const int64_t m0 = static_cast<int64_t>(tm) * EDGE, n0 = static_cast<int64_t>(tn) * EDGE;
    float* const y = static_cast<float*>(g.y) + e * g.n * g.k + m0 * g.k + n0;
    if (lo == hi) {
        zero_part(g, static_cast<float*>(g.y) + e * g.n * g.k, tm, tn);
        return;
    }
    Part32 p{};
    p.x = static_cast<const float*>(g.a) + lo * g.lda + m0;
    p.w = static_cast<const float*>(g.w) + lo * g.ldw + n0;
    p.y = y, p.M = g.n - m0, p.N = g.k - n0, p.K = hi - lo, p.ldx = g.lda, p.ldw = g.ldw, p.ldy = g.k, p.tiles_m = p.tiles_n = 1;
    small_product<true, true, EDGE / 32, EDGE / 32, groups_of(EDGE), kStages32, true>(p, 0, 1, nullptr, lds);
}

template <int EDGE, typename Kernel>
int launch32(const char* who, Kernel kernel, std::atomic<bool>* reserved, const ExpertArgs& g, int64_t blocks, int dev, hipStream_t s) {
    if (blocks * 256 > 0xFFFFFFFFll) return fail(DDL_E_UNSUPP, "%s: %lld tiles", who, static_cast<long long>(blocks));
    if (lds_of(EDGE) > 65536 && !reserved[dev].load(std::memory_order_acquire)) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds_of(EDGE));
        if (e != hipSuccess) return fail(static_cast<int>(e), "%s: cannot reserve %d bytes of LDS: %s", who, lds_of(EDGE), hipGetErrorString(e));
        reserved[dev].store(true, std::memory_order_release);
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(256), lds_of(EDGE), s, g);
    return check_launch(who);
}

template <int EDGE, bool WT>
int launch_rows32(const char* who, ExpertArgs g, int dev, hipStream_t s) {
    static std::atomic<bool> reserved[kMaxDevices];
    g.tiles_n = static_cast<int>((g.n + EDGE - 1) / EDGE);
    return launch32<EDGE>(who, expert_rows32<EDGE, WT>, reserved, g, ((g.rows + EDGE - 1) / EDGE + g.experts) * static_cast<int64_t>(g.tiles_n), dev, s);
}

template <int EDGE>
int launch_weights32(const char* who, ExpertArgs g, int dev, hipStream_t s) {
    static std::atomic<bool> reserved[kMaxDevices];
    g.tiles_m = static_cast<int>((g.n + EDGE - 1) / EDGE), g.tiles_n = static_cast<int>((g.k + EDGE - 1) / EDGE);
    return launch32<EDGE>(who, expert_weights32<EDGE>, reserved, g, matrix_blocks(g), dev, s);
}

}  // namespace

int run_expert_rows32(const char* who, bool small, bool transposed, const ExpertArgs& g, int dev, hipStream_t s) {
    if (small) return transposed ? launch_rows32<32, true>(who, g, dev, s) : launch_rows32<32, false>(who, g, dev, s);
    return transposed ? launch_rows32<64, true>(who, g, dev, s) : launch_rows32<64, false>(who, g, dev, s);
}

int run_expert_weights32(const char* who, bool small, const ExpertArgs& g, int dev, hipStream_t s) {
    return small ? launch_weights32<32>(who, g, dev, s) : launch_weights32<64>(who, g, dev, s);
}

}  // namespace ddl
