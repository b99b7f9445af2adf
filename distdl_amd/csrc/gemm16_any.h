// The tile of the 16-bit products of operands at any address and pitch, for the kernels that hand out such tiles: its
// schedule is described at the head of linear_any.hip.
#ifndef DDL_GEMM16_ANY_H
#define DDL_GEMM16_ANY_H
#include "colsum.h"
#include "gemm16_parts.h"
#include <type_traits>

namespace ddl {
namespace {

constexpr int kAnyDepth = kRowBytes / 2;   // 16-bit elements of a k-tile
constexpr int kAnyThreads = 256;

// The eight elements of `v` from number `s` on, zeros behind them.
__device__ inline uint4 drop(uint4 v, int s) {
    uint32_t w[5] = {v.x, v.y, v.z, v.w, 0};
    if (s & 4) w[0] = w[2], w[1] = w[3], w[2] = 0, w[3] = 0;
    if (s & 2) w[0] = w[1], w[1] = w[2], w[2] = w[3], w[3] = 0;
    if (s & 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (w[e] >> 16) | (w[e + 1] << 16);
    }
    if (s >= 8) w[0] = w[1] = w[2] = w[3] = 0;
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Workgroup `block` of the tiles_m x tiles_n x splits of a product: tiles of 64 T x 64 T, a wavefront has 32 T x 32 T.
template <bool F16, bool XT, bool WT, int T>
__device__ __forceinline__ void any_product(const Part16& p, int block, int splits, float* __restrict__ partial, char* lds) {
    constexpr int NWM = 2, TM = 2 * T, TN = 2 * T, NW = 4, J = 2 * T, B = 64 * T;   // J: 1 KiB pieces per wavefront and operand
    constexpr int kStage = 2 * B * kRowBytes, kX = B * kRowBytes;
    const int ntiles = p.tiles_m * p.tiles_n;
    const int split = block / ntiles, tile = block - split * ntiles;
    int tm, tn;
    tile_of_workgroup(tile, p.tiles_m, p.tiles_n, tm, tn);
    const int64_t M = p.M, N = p.N, K = p.K, m0 = static_cast<int64_t>(tm) * B, n0 = static_cast<int64_t>(tn) * B;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, kg = lane >> 4;
    const int sub_w = (wave / NWM) * TN, sub_x = (wave % NWM) * TM;

    // k-tiles [t_begin, t_end) of this split.  The last one of all needs care where K ends in it, or where an operand read
    // along its rows has a chunk there that would run over into a k-line which the last one has not.
    const int ktiles = static_cast<int>((K + kAnyDepth - 1) / kAnyDepth);
    const int full_tiles = static_cast<int>(((WT && N % 8 != 0) || (XT && M % 8 != 0) ? K - 1 : K) / kAnyDepth);
    const int per = (ktiles + splits - 1) / splits;
    const int t_begin = split * per < ktiles ? split * per : ktiles, t_end = t_begin + per < ktiles ? t_begin + per : ktiles;
    const int n = t_end - t_begin, has_tail = n > 0 && t_end > full_tiles ? 1 : 0;

    const uint16_t* const base_w = WT ? p.w + n0 : p.w + n0 * p.ldw;
    const uint16_t* const base_x = XT ? p.x + m0 : p.x + m0 * p.ldx;
    const int64_t step_w = WT ? p.ldw * kAnyDepth : kAnyDepth, step_x = XT ? p.ldx * kAnyDepth : kAnyDepth;   // elements from one k-tile to the next
    // Where this lane's chunk of piece i lies, from the tile's first row and k-tile 0 on: swizzles as in linear_gemm.hip, rows
    // past the end repeat the last one, chunks past it the first of the tile.
    auto row_of = [&](int i) { return i * 8 + (lane >> 3); };
    auto first_k = [&](int i) { return ((lane & 7) ^ ((row_of(i) >> 1) & 7)) * 8; };
    auto line_of = [&](int i) { return 8 * (i & 7) + (lane >> 3); };
    auto first_row = [&](int i, int64_t left) -> int64_t {
        const int k = line_of(i), h = ((k >> 1) & 1) | (((k >> 3) & 1) << 1);
        const int col = (i >> 3) * 64 + ((lane & 7) ^ (h << 1)) * 8;
        return col < left ? col : 0;
    };
    auto place = [&](bool transposed, int i, int64_t left, int64_t ld) -> int64_t {   // left: rows of the operand from the tile's first on
        if (transposed) return line_of(i) * ld + first_row(i, left);
        return (row_of(i) < left ? row_of(i) : left - 1) * ld + first_k(i);
    };
    // The same in the tile that needs care: moved back to where 16 bytes still lie inside the operand, by `s` elements; 8 for
    // a chunk that is all zeros.
    auto place_tail = [&](bool transposed, int i, int64_t left, int64_t ld, int& s) -> int64_t {
        const int64_t k0 = static_cast<int64_t>(ktiles - 1) * kAnyDepth;
        if (transposed) {
            const int64_t k = k0 + line_of(i), at = (k < K ? k : K - 1) * ld + first_row(i, left), last = (K - 1) * ld + left - 8;
            const int back = at > last ? static_cast<int>(at - last) : 0;
            s = k < K ? back : 8;
            return at - back;
        }
        const int64_t k = k0 + first_k(i);
        s = k > K - 8 ? static_cast<int>(k - (K - 8)) : 0;
        return (row_of(i) < left ? row_of(i) : left - 1) * ld + (k - s);
    };

    struct Regs {
        uint4 w[J], x[J];
    };
    Regs regs[2];   // tiles i and i + 1 of this split, the one that needs care being number 0
    int64_t off_w[J], off_x[J];
    int drop_w[J], drop_x[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int i = NW * j + wave;
        off_w[j] = place(WT, i, N - n0, p.ldw), off_x[j] = place(XT, i, M - m0, p.ldx);
        const int64_t tail_w = place_tail(WT, i, N - n0, p.ldw, drop_w[j]), tail_x = place_tail(XT, i, M - m0, p.ldx, drop_x[j]);
        if (full_tiles == 0) off_w[j] = tail_w, off_x[j] = tail_x;   // k-tile 0 is the one to be careful with
        const int64_t first = n > 0 ? t_begin : 0;
        regs[0].w[j] = load16(base_w + (has_tail ? tail_w : off_w[j] + first * step_w));
        regs[0].x[j] = load16(base_x + (has_tail ? tail_x : off_x[j] + first * step_x));
    }
    // Tile i >= 1; past the last one k-tile 0 again, which nobody multiplies.
    auto load = [&](int i, Regs& r) {
        const int t = i < n ? t_begin + i - has_tail : 0;
        const uint16_t *bw = base_w + t * step_w, *bx = base_x + t * step_x;
#pragma unroll
        for (int j = 0; j < J; ++j) r.w[j] = load16(bw + off_w[j]);
#pragma unroll
        for (int j = 0; j < J; ++j) r.x[j] = load16(bx + off_x[j]);
    };
    auto stash = [&](int slot, const Regs& r, int piece) {   // pieces 0 .. J - 1 are w's
        char* const to = lds + slot * kStage + (piece < J ? 0 : kX) + (NW * (piece % J) + wave) * 1024 + lane * 16;
        *reinterpret_cast<uint4*>(to) = piece < J ? r.w[piece % J] : r.x[piece % J];
    };
    load(1, regs[1]);
    if (has_tail) {
#pragma unroll
        for (int j = 0; j < J; ++j) regs[0].w[j] = drop(regs[0].w[j], drop_w[j]), regs[0].x[j] = drop(regs[0].x[j], drop_x[j]);
    }
#pragma unroll
    for (int q = 0; q < 2 * J; ++q) stash(0, regs[0], q);

    // Fragment reads: as in linear_gemm.hip.
    const int tr_lane = (8 * kg + (l16 >> 2)) * 128 + (l16 & 3) * 8;
    const int tr_h = (((l16 >> 3) & 1) | ((kg & 1) << 1)) << 5;
    typedef short short4v __attribute__((ext_vector_type(4)));
    typedef short short8v __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) short4v* lds_short4;
    auto fragment = [&](auto transposed, const char* tile_base, int sub, int ks) -> bf16x8 {
        bf16x8 out;
        if (decltype(transposed)::value) {
            const char* q = tile_base + (sub >> 2) * 8192 + ks * (32 * 128) + (tr_lane + (((sub & 3) << 5) ^ tr_h));
            const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4)(q));
            const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4)(q + 4 * 128));
            const short8v both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            __builtin_memcpy(&out, &both, 16);
        } else {
            out = *reinterpret_cast<const bf16x8*>(tile_base + sub * (16 * kRowBytes) + l16 * kRowBytes + (((4 * ks + kg) ^ ((l16 >> 1) & 7)) << 4));
        }
        return out;
    };
    floatx4 acc[TN][TM];
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b) acc[a][b] = floatx4{0.f, 0.f, 0.f, 0.f};
    // The tile in `slot`: all fragments, the MFMAs of the first half, those of the second with between(q) in front of every
    // second one (q = 0 .. TN TM / 2 - 1).  The barriers to the scheduler keep that order.
    auto multiply = [&](int slot, auto between) {
        const char* const wt = lds + slot * kStage;
        bf16x8 fw[2][TN], fx[2][TM];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
            for (int a = 0; a < TN; ++a) fw[ks][a] = fragment(std::integral_constant<bool, WT>{}, wt, sub_w + a, ks);
#pragma unroll
            for (int b = 0; b < TM; ++b) fx[ks][b] = fragment(std::integral_constant<bool, XT>{}, wt + kX, sub_x + b, ks);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int a = 0; a < TN; ++a)
#pragma unroll
            for (int b = 0; b < TM; ++b) acc[a][b] = mfma<F16>(fw[0][a], fx[0][b], acc[a][b]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int a = 0; a < TN; ++a)
#pragma unroll
            for (int b = 0; b < TM; ++b) {
                if (b % 2 == 0) {
                    between((a * TM + b) / 2);
                    __builtin_amdgcn_sched_barrier(0);
                }
                acc[a][b] = mfma<F16>(fw[1][a], fx[1][b], acc[a][b]);
            }
    };
    constexpr int kPer = 2 * J / (TN * TM / 2);   // pieces written in front of each of them
    int i = 0;
#pragma unroll 1
    for (; i + 2 <= n; i += 2) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            __syncthreads();   // tile i + u is complete; nobody reads the other slot any more
            load(i + u + 2, regs[u]);
            __builtin_amdgcn_sched_barrier(0);
            multiply(u, [&](int q) {
#pragma unroll
                for (int v = 0; v < kPer; ++v) stash(u ^ 1, regs[u ^ 1], q * kPer + v);
            });
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (i < n) {
        __syncthreads();
        multiply(0, [](int) {});
    }
    if (splits > 1) {   // lane order, so that the partial sums are written and read in whole lines
        floatx4* dst = reinterpret_cast<floatx4*>(partial) + (static_cast<int64_t>(block) * NW + wave) * (TN * TM * 64) + lane;
#pragma unroll
        for (int a = 0; a < TN; ++a)
#pragma unroll
            for (int b = 0; b < TM; ++b) dst[(a * TM + b) * 64] = acc[a][b];
        return;
    }
    // Through LDS, so that whole row segments of the tile leave 16 bytes a lane, at any address: with eight bytes a lane, as a
    // wavefront holds them, the adjoint of M 23, N 6400, K 2496 took 32.8 us, here 30.6.
    constexpr int kPitch = 2 * B + 16;   // staggers consecutive rows over the banks
    static_assert(B * kPitch <= 2 * kStage, "the result does not fit where the operands were");
    __syncthreads();   // nobody reads the operands any more
#pragma unroll
    for (int a = 0; a < TN; ++a) {
        const int64_t c = n0 + (sub_w + a) * 16 + 4 * kg;
        float bv[4] = {0.f, 0.f, 0.f, 0.f};
        if (p.bias) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < N) bv[e] = elem_to_f32<F16>(p.bias[c + e]);
        }
#pragma unroll
        for (int b = 0; b < TM; ++b) {
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = f32_to_elem<F16>(acc[a][b][e] + bv[e]);
            *reinterpret_cast<uint2*>(lds + ((sub_x + b) * 16 + l16) * kPitch + ((sub_w + a) * 16 + 4 * kg) * 2) = make_uint2(o[0] | o[1] << 16, o[2] | o[3] << 16);
        }
    }
    __syncthreads();
    constexpr int kChunks = B / 8;   // of a row
#pragma unroll
    for (int q = 0; q < B * kChunks / kAnyThreads; ++q) {
        const int at = q * kAnyThreads + threadIdx.x, row = at / kChunks, chunk = at % kChunks;
        const int64_t m = m0 + row, c = n0 + chunk * 8;
        if (m >= M || c >= N) continue;
        const uint4 v = *reinterpret_cast<const uint4*>(lds + row * kPitch + chunk * 16);
        uint16_t* const dst = p.y + m * p.ldy + c;
        if (c + 8 <= N) {
            typedef u32x4 any __attribute__((aligned(2)));
            *reinterpret_cast<any*>(dst) = u32x4{v.x, v.y, v.z, v.w};
        } else {
            const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < N) dst[e] = static_cast<uint16_t>(words[e >> 1] >> (16 * (e & 1)));
        }
    }
}

}  // namespace
}  // namespace ddl
#endif  // DDL_GEMM16_ANY_H
