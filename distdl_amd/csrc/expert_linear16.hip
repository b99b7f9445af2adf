// The experts' products of 16-bit elements: the tiles of linear_gemm.hip (operands aligned to 16 bytes) and linear_any.hip (any others),
// handed out expert by expert.
//
//   rows      y[i] = w[e] a[i], and with w read along its columns the adjoint dx[i] = w[e]^T dy[i]: a tile is some rows of one expert
//             by some columns.  Which expert's is found on the device (expert_parts.h); a workgroup past the last tile ends.
//   weights   dw[e] = dy_e^T x_e: a tile of every expert's matrix, the reduction over its rows; zeros for an expert without any.
#include "expert_parts.h"
#include "gemm16_any.h"
#include "gemm16_large.h"

namespace ddl {
namespace {

template <ExpertTile TILE>
struct Shape {
    static constexpr bool large = TILE == ExpertTile::kLow || TILE == ExpertTile::kLarge;
    static constexpr int bm = TILE == ExpertTile::kAny64 ? 64 : TILE == ExpertTile::kLarge ? 256 : 128;
    static constexpr int bn = TILE == ExpertTile::kAny64 ? 64 : TILE == ExpertTile::kAny128 ? 128 : 256;
    static constexpr int threads = large ? 512 : kAnyThreads;
    static constexpr int lds = large ? kLdsBytes : 4 * bm * kRowBytes;
    static constexpr int per_simd = TILE == ExpertTile::kAny64 ? 4 : 2;
};

template <ExpertTile TILE, bool F16, bool XT, bool WT>
__device__ __forceinline__ void product_tile(const PartOf<uint16_t>& p, char* lds) {
    if constexpr (TILE == ExpertTile::kLarge) gemm_tile<F16, XT, WT, 2, 4, 8, 4>(p, 0, lds);
    else if constexpr (TILE == ExpertTile::kLow) gemm_tile<F16, XT, WT, 2, 4, 4, 4>(p, 0, lds);
    else any_product<F16, XT, WT, TILE == ExpertTile::kAny128 ? 2 : 1>(p, 0, 1, nullptr, lds);
}

template <ExpertTile TILE, bool F16, bool WT>
__global__ __launch_bounds__(Shape<TILE>::threads, Shape<TILE>::per_simd) void expert_rows16(const ExpertArgs g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const ExpertTask t = find_tile<TILE == ExpertTile::kLarge>(g, Shape<TILE>::bm, blockIdx.x);
    if (t.expert < 0) return;
    const int64_t n0 = static_cast<int64_t>(t.tn) * Shape<TILE>::bn;
    uint16_t* const y = static_cast<uint16_t*>(g.y) + t.row * g.ldy + n0;
    if (t.expert == g.experts) {
        zero_block(y, g.ldy, min(t.rows, t.half ? Shape<TILE>::bm / 2 : Shape<TILE>::bm), static_cast<int>(min(g.n - n0, static_cast<int64_t>(Shape<TILE>::bn))));
        return;
    }
    PartOf<uint16_t> p{};
    p.x = static_cast<const uint16_t*>(g.a) + t.row * g.lda;
    p.w = static_cast<const uint16_t*>(g.w) + t.expert * g.w_stride + (WT ? n0 : n0 * g.ldw);
    p.y = y, p.M = t.rows, p.N = g.n - n0, p.K = g.k, p.ldx = g.lda, p.ldw = g.ldw, p.ldy = g.ldy, p.tiles_m = p.tiles_n = 1;
    if (TILE == ExpertTile::kLarge && t.half) product_tile<ExpertTile::kLow, F16, false, WT>(p, lds);
    else product_tile<TILE, F16, false, WT>(p, lds);
}

// a: dy [rows, n], w: x [rows, k]; y: dw, n x k for each expert.
template <ExpertTile TILE, bool F16>
__global__ __launch_bounds__(Shape<TILE>::threads, Shape<TILE>::per_simd) void expert_weights16(const ExpertArgs g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    MatrixTask t;
    if (!find_matrix_tile(g, blockIdx.x, t)) return;
    if (t.lo == t.hi) {
        zero_part<uint16_t>(g, t);
        return;
    }
    const int64_t m0 = static_cast<int64_t>(t.tm) * Shape<TILE>::bm, n0 = static_cast<int64_t>(t.tn) * Shape<TILE>::bn;
    PartOf<uint16_t> p{};
    p.x = static_cast<const uint16_t*>(g.a) + t.lo * g.lda + m0;
    p.w = static_cast<const uint16_t*>(g.w) + t.lo * g.ldw + n0;
    p.y = static_cast<uint16_t*>(g.y) + t.expert * g.n * g.k + m0 * g.k + n0;
    p.M = g.n - m0, p.N = g.k - n0, p.K = t.hi - t.lo, p.ldx = g.lda, p.ldw = g.ldw, p.ldy = g.k, p.tiles_m = p.tiles_n = 1;
    product_tile<TILE, F16, true, true>(p, lds);
}

template <ExpertTile TILE, typename Kernel>
int launch(const char* who, Kernel kernel, std::atomic<bool>* reserved, const ExpertArgs& g, int64_t blocks, int dev, hipStream_t s) {
    if (blocks * Shape<TILE>::threads > 0xFFFFFFFFll) return fail(DDL_E_UNSUPP, "%s: %lld tiles", who, static_cast<long long>(blocks));
    if (Shape<TILE>::lds > 65536 && !reserved[dev].load(std::memory_order_acquire)) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, Shape<TILE>::lds);
        if (e != hipSuccess) return fail(static_cast<int>(e), "%s: cannot reserve %d bytes of LDS: %s", who, Shape<TILE>::lds, hipGetErrorString(e));
        reserved[dev].store(true, std::memory_order_release);
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(Shape<TILE>::threads), Shape<TILE>::lds, s, g);
    return check_launch(who);
}

template <ExpertTile TILE, bool F16, bool WT>
int launch_rows(const char* who, ExpertArgs g, int dev, hipStream_t s) {
    static std::atomic<bool> reserved[kMaxDevices];
    g.tiles_n = static_cast<int>((g.n + Shape<TILE>::bn - 1) / Shape<TILE>::bn);
    // every expert, and the rows behind them, can end inside a tile
    const int64_t tiles_m = (g.rows + Shape<TILE>::bm - 1) / Shape<TILE>::bm + g.experts;
    const int64_t halves = TILE == ExpertTile::kLarge ? g.cus : 0;   // workgroups for those of the last round
    return launch<TILE>(who, expert_rows16<TILE, F16, WT>, reserved, g, tiles_m * g.tiles_n + halves, dev, s);
}

template <ExpertTile TILE, bool F16>
int launch_weights(const char* who, ExpertArgs g, int dev, hipStream_t s) {
    static std::atomic<bool> reserved[kMaxDevices];
    g.tiles_m = static_cast<int>((g.n + Shape<TILE>::bm - 1) / Shape<TILE>::bm), g.tiles_n = static_cast<int>((g.k + Shape<TILE>::bn - 1) / Shape<TILE>::bn);
    return launch<TILE>(who, expert_weights16<TILE, F16>, reserved, g, matrix_blocks(g), dev, s);
}

template <typename Fn>
int with_tile(ExpertTile tile, Fn&& fn) {
    switch (tile) {
        case ExpertTile::kAny64: return fn(std::integral_constant<ExpertTile, ExpertTile::kAny64>{});
        case ExpertTile::kAny128: return fn(std::integral_constant<ExpertTile, ExpertTile::kAny128>{});
        case ExpertTile::kLow: return fn(std::integral_constant<ExpertTile, ExpertTile::kLow>{});
        default: return fn(std::integral_constant<ExpertTile, ExpertTile::kLarge>{});
    }
}

}  // namespace

int run_expert_rows16(const char* who, ExpertTile tile, bool f16, bool transposed, ExpertArgs g, int dev, hipStream_t s) {
    return with_tile(tile, [&](auto t) {
        constexpr ExpertTile TILE = decltype(t)::value;
        if (f16) return transposed ? launch_rows<TILE, true, true>(who, g, dev, s) : launch_rows<TILE, true, false>(who, g, dev, s);
        return transposed ? launch_rows<TILE, false, true>(who, g, dev, s) : launch_rows<TILE, false, false>(who, g, dev, s);
    });
}

int run_expert_weights16(const char* who, ExpertTile tile, bool f16, ExpertArgs g, int dev, hipStream_t s) {
    return with_tile(tile, [&](auto t) {
        constexpr ExpertTile TILE = decltype(t)::value;
        return f16 ? launch_weights<TILE, true>(who, g, dev, s) : launch_weights<TILE, false>(who, g, dev, s);
    });
}

}  // namespace ddl
