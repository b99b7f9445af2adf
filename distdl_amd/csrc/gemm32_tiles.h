// The tile of the smaller fp32 products, for the kernels that hand out such tiles: its layout and schedule are described at the
// head of linear_f32_small.hip.
#ifndef DDL_GEMM32_TILES_H
#define DDL_GEMM32_TILES_H
#include "gemm_tiles.h"
#include "gemm32_small.h"
#include <type_traits>

namespace ddl {
namespace {

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float floatx16;

constexpr int kDepth32 = kRowBytes / 4;   // floats of a k-tile
typedef PartOf<float> Part32;

// Workgroup `number` of the tiles_m x tiles_n x splits of a product.  FOLD: the sum of every kFold rounds goes into another one, so that a long reduction is
// not one chain of roundings.
constexpr int kFold = 32;
template <bool XT, bool WT, int NWM, int NWN, int KG, int STAGES, bool FOLD = false>
__device__ __forceinline__ void small_product(const Part32& p, int number, int splits, float* __restrict__ partial, char* lds) {
    constexpr int NW = NWM * NWN, BM = 32 * NWM, BN = 32 * NWN;
    static_assert(NW * KG == 4, "four wavefronts per workgroup");
    constexpr int JW_W = BN / 8 / NW, JW_X = BM / 8 / NW;   // request instructions (1 KiB each) per wavefront and tile
    constexpr int kStage = (BM + BN) * kRowBytes, kX = BN * kRowBytes;   // a stage holds the w tile and then the x tile
    const int ntiles = p.tiles_m * p.tiles_n;
    const int split = number / ntiles, tile = number - split * ntiles;
    int tm, tn;
    tile_of_workgroup(tile, p.tiles_m, p.tiles_n, tm, tn);
    const int64_t M = p.M, N = p.N, K = p.K;
    const int64_t m0 = static_cast<int64_t>(tm) * BM, n0 = static_cast<int64_t>(tn) * BN;
    const int lane = threadIdx.x & 63, group = __builtin_amdgcn_readfirstlane(threadIdx.x / (NW * 64));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) - group * NW;   // inside its group
    const int l32 = lane & 31, kh = lane >> 5;
    const int sub_w = wave / NWM, sub_x = wave % NWM;   // 32-row block of this wavefront in the w and x tiles

    const int ktiles = static_cast<int>((K + kDepth32 - 1) / kDepth32);
    // Tiles from here on go through registers (see the head of the file).
    const bool w_over = WT && N % 4 != 0, x_over = XT && M % 4 != 0;
    const int full_tiles = static_cast<int>((w_over || x_over ? K - 1 : K) / kDepth32);
    const int per = (ktiles + splits - 1) / splits;
    const int t_begin = split * per < ktiles ? split * per : ktiles, t_end = t_begin + per < ktiles ? t_begin + per : ktiles;
    char* const ring = lds + group * (STAGES * kStage);

    // Piece i = NW j + wave of a tile.  Along k: rows 8 i .. + 7, lane l on row l / 8, physical chunk l % 8.  Along rows:
    // panel i / 4, k-lines 8 (i % 4) .. + 7 with neighbours swapped in lines 4 .. 7, rows 4 (l % 8) .. + 3 of the panel.
    // Rows past the end repeat the last one, chunks that start past it the first of the tile; never stored.
    const char* const base_w = reinterpret_cast<const char*>(WT ? p.w + n0 : p.w + n0 * p.ldw);
    const char* const base_x = reinterpret_cast<const char*>(XT ? p.x + m0 : p.x + m0 * p.ldx);
    const u32x4 buf_w = raw_buffer(base_w), buf_x = raw_buffer(base_x);
    const int step_w = WT ? static_cast<int>(p.ldw) * (kDepth32 * 4) : kDepth32 * 4;
    const int step_x = XT ? static_cast<int>(p.ldx) * (kDepth32 * 4) : kDepth32 * 4;
    auto chunk_k = [&](bool transposed, int i) {   // first k of this lane's chunk, or its k-line, inside a k-tile
        const int row = i * 8 + (lane >> 3), q = lane >> 3;
        return transposed ? 8 * (i & 3) + (q ^ ((q >> 2) & 1)) : ((lane & 7) ^ ((row >> 1) & 7)) * 4;
    };
    auto chunk_row = [&](bool transposed, int i, int64_t origin, int64_t rows) -> int {   // (first) row inside the tile
        if (!transposed) {
            const int row = i * 8 + (lane >> 3);
            return origin + row < rows ? row : static_cast<int>(rows - 1 - origin);
        }
        const int col = (i >> 2) * 32 + (lane & 7) * 4;
        return origin + col < rows ? col : 0;
    };
    auto lane_offset = [&](bool transposed, int i, int64_t origin, int64_t rows, int64_t ld) -> int {
        const int64_t k = chunk_k(transposed, i), r = chunk_row(transposed, i, origin, rows);
        return static_cast<int>((transposed ? k * ld + r : r * ld + k) * 4);
    };
    int off_w[JW_W], off_x[JW_X];
#pragma unroll
    for (int j = 0; j < JW_W; ++j) off_w[j] = lane_offset(WT, NW * j + wave, n0, N, p.ldw);
#pragma unroll
    for (int j = 0; j < JW_X; ++j) off_x[j] = lane_offset(XT, NW * j + wave, m0, M, p.ldx);
    // One chunk through registers: elements past K or past the rows are zeros.
    auto careful = [&](bool transposed, const char* base, int off, int64_t step, int t, int i, int64_t origin, int64_t rows, char* dst) {
        const int64_t at = off + t * step;
        const int64_t k = static_cast<int64_t>(t) * kDepth32 + chunk_k(transposed, i), r = origin + chunk_row(transposed, i, origin, rows);
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool inside = transposed ? k < K && r + e < rows : k + e < K;
            const float f = *reinterpret_cast<const float*>(base + (inside ? at + 4 * e : 0));   // the tile's first element otherwise
            v[e] = inside ? f : 0.f;
        }
        *reinterpret_cast<floatx4*>(dst + lane * 16) = floatx4{v[0], v[1], v[2], v[3]};
    };
    constexpr int J = JW_W + JW_X;
    auto request_piece = [&](int j, int t, char* stage) {
        if (j < JW_W) dma16(buf_w, off_w[j], t * step_w, stage + (NW * j + wave) * 1024);
        else dma16(buf_x, off_x[j - JW_W], t * step_x, stage + kX + (NW * (j - JW_W) + wave) * 1024);
    };
    auto request = [&](int t, int slot) {
        char* stage = ring + slot * kStage;
        if (t < full_tiles) {
#pragma unroll
            for (int j = 0; j < J; ++j) request_piece(j, t, stage);
        } else {
#pragma unroll
            for (int j = 0; j < JW_W; ++j) careful(WT, base_w, off_w[j], step_w, t, NW * j + wave, n0, N, stage + (NW * j + wave) * 1024);
#pragma unroll
            for (int j = 0; j < JW_X; ++j) careful(XT, base_x, off_x[j], step_x, t, NW * j + wave, m0, M, stage + kX + (NW * j + wave) * 1024);
        }
    };
    // Floats k = 8 g + 4 kh + {0..3} of row l32 of block `sub`.
    auto fragment = [&](auto transposed, const char* tile_base, int sub, int g) -> floatx4 {
        const char* block = tile_base + sub * 4096;
        if (!decltype(transposed)::value)
            return *reinterpret_cast<const floatx4*>(block + l32 * kRowBytes + (((2 * g + kh) ^ ((l32 >> 1) & 7)) << 4));
        floatx4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int line = 4 * kh + e;   // of the eight of group g
            v[e] = *reinterpret_cast<const float*>(block + (8 * g + (line ^ ((line >> 2) & 1))) * 128 + l32 * 4);
        }
        return v;
    };

    floatx16 acc, folded;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = folded[e] = 0.f;
    auto fold = [&]() {
#pragma unroll
        for (int e = 0; e < 16; ++e) folded[e] += acc[e], acc[e] = 0.f;
    };
    // Group i takes k-tiles t_begin + i, + KG, ...; all groups walk the same number of rounds, for the barriers.
    const int rounds = (t_end - t_begin + KG - 1) / KG;
    auto tile_at = [&](int r) { return t_begin + r * KG + group; };
#pragma unroll 1   // unrolled, the instructions of four requests are what a short product waits for
    for (int i = 0; i < STAGES; ++i)
        if (tile_at(i) < t_end) request(tile_at(i), i);
    // Requests up to tile r - 1 of this group have landed and this wavefront's LDS reads have returned; the `behind` tiles
    // from r on may be in flight if all went out as requests.
    auto landed = [&](int r, auto behind) {
        const int last = tile_at(r + decltype(behind)::value - 1);
        if (last < t_end && last < full_tiles)
            __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(decltype(behind)::value * J));
        else
            __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    floatx4 fw[4], fx[4];
    auto read_half = [&](int slot, auto half) {
        constexpr int g0 = decltype(half)::value * 2;
        const char* wt = ring + slot * kStage;
        const char* xt = wt + kX;
#pragma unroll
        for (int g = g0; g < g0 + 2; ++g) {
            fw[g] = fragment(std::integral_constant<bool, WT>{}, wt, sub_w, g);
            fx[g] = fragment(std::integral_constant<bool, XT>{}, xt, sub_x, g);
        }
        __builtin_amdgcn_sched_barrier(0);   // left alone, the compiler puts each pair in front of its MFMAs
    };
    auto multiply = [&](auto half, auto from, auto upto) {   // instructions [from, upto) of eight
        constexpr int g0 = decltype(half)::value * 2;
#pragma unroll
        for (int i = decltype(from)::value; i < decltype(upto)::value; ++i)
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(fw[g0 + i / 4][i % 4], fx[g0 + i / 4][i % 4], acc, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    typedef std::integral_constant<int, 0> First;
    typedef std::integral_constant<int, 1> Second;
    typedef std::integral_constant<int, 8> End;
    // Seven instructions on one half of a k-tile hide the reads of the other half, or of the first half of the next k-tile.
    // The one in front of the reads has waited for what came before them.
    landed(1, std::integral_constant<int, STAGES - 1>{});
    read_half(0, First{});
    int slot = 0, r = 0;
    // While all that is requested goes out as requests: nothing to decide, and an instruction's shadow has at most two of them.
    const int plain = (t_end < full_tiles ? t_end : full_tiles) - t_begin - group;   // tiles of the range, counted from the group's first
#pragma unroll 1
    for (; (r + STAGES) * KG < plain; ++r) {
        if (FOLD && r % kFold == kFold - 1) fold();
        multiply(First{}, First{}, Second{});
        read_half(slot, Second{});
        multiply(First{}, Second{}, End{});
        __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0((STAGES - 2) * J));   // tile r + 1 is readable, the slot of tile r free
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        char* const stage = ring + slot * kStage;
        slot = slot + 1 == STAGES ? 0 : slot + 1;
        multiply(Second{}, First{}, Second{});
        read_half(slot, First{});
#pragma unroll
        for (int i = 1; i < 8; ++i) {
#pragma unroll
            for (int j = (i - 1) * J / 7; j < i * J / 7; ++j) request_piece(j, tile_at(r + STAGES), stage);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(fw[2 + i / 4][i % 4], fx[2 + i / 4][i % 4], acc, 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll 1
    for (; r < rounds; ++r) {
        if (KG > 1 && tile_at(r) >= t_end) break;   // the last round of a group that has one tile less
        multiply(First{}, First{}, Second{});
        read_half(slot, Second{});
        multiply(First{}, Second{}, End{});
        if (r + 1 < rounds) landed(r + 2, std::integral_constant<int, STAGES - 2>{});
        const int next = slot + 1 == STAGES ? 0 : slot + 1;
        multiply(Second{}, First{}, Second{});
        read_half(next, First{});   // behind the last tile what the slot holds, for nothing
        if (tile_at(r + STAGES) < t_end) request(tile_at(r + STAGES), slot);
        multiply(Second{}, Second{}, End{});
        slot = next;
    }
    wait_states_acc<18>(acc);
    if (FOLD) {
        fold();
        acc = folded;
    }
    // Lane holds row m = l32 and columns n = 8 g + 4 kh + {0..3} in acc[4 g + {0..3}].
    floatx4 quad[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) quad[g] = floatx4{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
    if (KG > 1) {   // the groups' sums meet in group 0, in the order of the groups
        __syncthreads();
        floatx4* fold = reinterpret_cast<floatx4*>(lds);
        if (group > 0) {
#pragma unroll
            for (int g = 0; g < 4; ++g) fold[(((group - 1) * NW + wave) * 4 + g) * 64 + lane] = quad[g];
        }
        __syncthreads();
        if (group > 0) return;
#pragma unroll
        for (int i = 0; i < KG - 1; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) quad[g] += fold[((i * NW + wave) * 4 + g) * 64 + lane];
    }
    if (splits > 1) {   // lane order, so that the partial sums are written and read in whole lines
        floatx4* dst = reinterpret_cast<floatx4*>(partial) + (static_cast<int64_t>(number) * NW + wave) * 256 + lane;
#pragma unroll
        for (int g = 0; g < 4; ++g) dst[g * 64] = quad[g];
        return;
    }
    const int64_t m = m0 + sub_x * 32 + l32;
    if (m >= M) return;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int64_t n = n0 + sub_w * 32 + 8 * g + 4 * kh;
        store_four(p.y + m * p.ldy + n, n, N, quad[g] + bias_of(p.bias, n, N));
    }
}

}  // namespace
}  // namespace ddl
#endif  // DDL_GEMM32_TILES_H
