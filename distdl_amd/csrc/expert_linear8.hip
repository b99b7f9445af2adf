// The experts' products of e4m3 rows and weights by tiles: y[i, j] = x_scales[i] w_scales[e, j] sum over k of w[e, j, k] x[i, k].
//
// The layout, the ring of operand tiles and the requests are those of the 16-bit tiles (described at the head of linear_gemm.hip): a k-tile is
// 128 bytes deep, here 128 elements, which one v_mfma_f32_16x16x128_f8f6f4 takes whole.  A workgroup of eight wavefronts has 256 (or 128) rows by
// 256 columns, a wavefront 16 TM x 64 of them.  Registers decide the schedule: a piece of an operand (16 rows) is eight registers, so the
// pieces of x come two ahead of their products, four at a time for each of them, and those of w one k-tile ahead, during the last two pieces.
// In front of those two is the k-tile's barrier: every wavefront has read what it needs of this tile, and the next one has landed.
#include "expert_parts.h"
#include "gemm16_parts.h"
#include <type_traits>

namespace ddl {
namespace {

typedef int intx8 __attribute__((ext_vector_type(8)));

// acc += a . b (16 x 16 x 128, e4m3 in); accumulators in their own registers, for the reason given at mfma_16x16x32.
__device__ inline void mfma_e4m3(floatx4& acc, const intx8& a, const intx8& b) {
    asm volatile("v_mfma_f32_16x16x128_f8f6f4 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

constexpr int kTN = 4, kColumns = 256, kThreads8 = 512;

// The tile of p.M x p.N elements (of those at most 32 TM x 256) from the first of x, w and y on.
struct Tile8 {
    const uint8_t *x, *w;
    const float *x_scales, *w_scales;
    void* y;
    int M, N, out_dtype;
    int64_t K, ldx, ldw, ldy;
};

// Four consecutive columns of a row.
__device__ inline void store_floats(float* row, int n, int N, const float* v) {
    if (n + 4 <= N) {
        typedef floatx4 any __attribute__((aligned(4)));
        *reinterpret_cast<any*>(row + n) = floatx4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < N) row[n + e] = v[e];
    }
}

template <int TM>
__device__ __forceinline__ void tile8(const Tile8& p, char* lds) {
    constexpr int NW = 8, BM = 32 * TM, JW = kColumns / 8 / NW, JX = BM / 8 / NW, kLast = TM - 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = (wave % 2) * (TM * 16), wn = (wave / 2) * (kTN * 16);
    const int l16 = lane & 15, kg = lane >> 4;

    floatx4 acc[kTN][TM];
#pragma unroll
    for (int a = 0; a < kTN; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[a][b][e] = 0.f;

    const u32x4 buf_w = raw_buffer(p.w), buf_x = raw_buffer(p.x);
    int off_w[JW], off_x[JX];
    auto lane_offset = [&](int J, int j, int rows, int64_t ld) -> int {
        const int row = (J * wave + j) * 8 + (lane >> 3);
        return static_cast<int>(static_cast<int64_t>(row < rows ? row : rows - 1) * ld) + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
    };
#pragma unroll
    for (int j = 0; j < JW; ++j) off_w[j] = lane_offset(JW, j, p.N, p.ldw);
#pragma unroll
    for (int j = 0; j < JX; ++j) off_x[j] = lane_offset(JX, j, p.M, p.ldx);
    const int ktiles = static_cast<int>((p.K + kRowBytes - 1) / kRowBytes), full_tiles = static_cast<int>(p.K / kRowBytes);

    auto request_w = [&](int t, int unit_off, int j) { dma16(buf_w, off_w[j], t * kRowBytes, lds + unit_off + (JW * wave + j) * 1024); };
    auto request_x = [&](int t, int unit_off, int j) { dma16(buf_x, off_x[j], t * kRowBytes, lds + unit_off + (JX * wave + j) * 1024); };
    // A whole operand tile; one that K ends in goes through registers, zeros behind its end.
    auto through = [&](const uint8_t* base, int off, int J, int j, int t, int unit_off) {
        const int row = (J * wave + j) * 8 + (lane >> 3), chunk = (lane & 7) ^ ((row >> 1) & 7);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (static_cast<int64_t>(t) * kRowBytes + chunk * 16 < p.K) v = *reinterpret_cast<const uint4*>(base + off + static_cast<int64_t>(t) * kRowBytes);
        *reinterpret_cast<uint4*>(lds + unit_off + (J * wave + j) * 1024 + lane * 16) = v;
    };
    auto request_w_tile = [&](int t, int unit_off) {
#pragma unroll
        for (int j = 0; j < JW; ++j) {
            if (t < full_tiles) request_w(t, unit_off, j);
            else through(p.w, off_w[j], JW, j, t, unit_off);
        }
    };
    auto request_x_tile = [&](int t, int unit_off) {
#pragma unroll
        for (int j = 0; j < JX; ++j) {
            if (t < full_tiles) request_x(t, unit_off, j);
            else through(p.x, off_x[j], JX, j, t, unit_off);
        }
    };

    // This lane's 32 bytes of its row of a piece: chunks kg and 4 + kg, as the 16-bit tiles read them one after the other, where the swizzle has them (chunks
    // 2 kg and 2 kg + 1 meet on their banks: half of the LDS cycles).
    const int sw = (l16 >> 1) & 7, at0 = l16 * kRowBytes + ((kg ^ sw) << 4), at1 = l16 * kRowBytes + (((4 + kg) ^ sw) << 4);
    auto read = [&](const char* tile, int row) -> intx8 {
        intx8 v;
        const uint4 a = *reinterpret_cast<const uint4*>(tile + row * kRowBytes + at0), b = *reinterpret_cast<const uint4*>(tile + row * kRowBytes + at1);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        return v;
    };

    auto unit_off = [](int slot) { return (slot >= kUnits ? slot - kUnits : slot) * kUnitBytes; };
    int s0 = 0;                          // ring slot of W(t); X(t), W(t+1), X(t+1), W(t+2) follow
    intx8 fw[2][kTN], fx[3];             // piece o of x is in fx[o % 3] (of the next tile: piece 0 in fx[TM % 3], moved on by `turn`)

    // k-tile t; pieces 0 and 1 of its x and all of its w are in registers or on their way.  PARITY: which half of fw; TURN: where piece 0 of x is.
    auto k_tile = [&](int t, auto steady, auto slot, auto parity, auto turn) {
        constexpr bool STEADY = decltype(steady)::value;
        constexpr int C = decltype(parity)::value, R = decltype(turn)::value;
        const int s = slot;
        const char* xt = lds + unit_off(s + 1) + wm * kRowBytes;
        const char* wn1 = lds + unit_off(s + 2) + wn * kRowBytes;
        const char* xn1 = lds + unit_off(s + 3) + wm * kRowBytes;
        const int w2_off = unit_off(s + 4), x2_off = unit_off(s);
        if (!STEADY && t + 2 < ktiles) request_w_tile(t + 2, w2_off);
#pragma unroll
        for (int o = 0; o < TM; ++o) {
            if (o == kLast) {
                __builtin_amdgcn_s_waitcnt(STEADY ? wait_vm_lgkm0(JW) : wait_vm_lgkm0(0));
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (!STEADY && t + 2 < ktiles) request_x_tile(t + 2, x2_off);
            }
#pragma unroll
            for (int q = 0; q < kTN; ++q) {
                const int i = (o & 1) ? kTN - 1 - q : q;
                mfma_e4m3(acc[i][o], fw[C][i], fx[(R + o) % 3]);
                const int n = o * kTN + q;       // number of the product
                if (o < kLast) {
                    if (q == 1) fx[(R + o + 2) % 3] = read(xt, (o + 2) * 16);
                    constexpr int kGap = kLast * kTN / JW;
                    if (STEADY && n % kGap == kGap - 1 && n / kGap < JW) request_w(t + 2, w2_off, n / kGap);
                } else {
                    const int m = n - kLast * kTN;   // 0 .. 7 behind the barrier; past the last tile they read what nobody uses
                    if (m == 0) fx[(R + TM) % 3] = read(xn1, 0);
                    if (m >= 1 && m <= 4) fw[C ^ 1][m - 1] = read(wn1, (m - 1) * 16);
                    if (m == 5) fx[(R + TM + 1) % 3] = read(xn1, 16);
                    if (STEADY && m < JX) request_x(t + 2, x2_off, m);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    // fx[(R + TM) % 3] must not be read any more when piece 0 of the next tile goes there: it is that of piece TM - 3.
    static_assert(TM >= 4, "pieces of x two ahead");

    request_w_tile(0, 0);
    request_x_tile(0, kUnitBytes);
    if (ktiles > 1) {
        request_w_tile(1, 2 * kUnitBytes);
        request_x_tile(1, 3 * kUnitBytes);
    }
    if (full_tiles > 1) __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(JW + JX));
    else __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    fx[0] = read(lds + kUnitBytes + wm * kRowBytes, 0);
#pragma unroll
    for (int i = 0; i < kTN; ++i) fw[0][i] = read(lds + wn * kRowBytes, i * 16);
    fx[1] = read(lds + kUnitBytes + wm * kRowBytes, 16);

    typedef std::integral_constant<int, 0> I0;
    const int steady_end = full_tiles - 2 > 0 ? full_tiles - 2 : 0;
    int t = 0;
    // The state that has to be known when compiled (slot, parity, turn) repeats after 30 tiles; pairs of tiles with the slot in a register
    // and the turn brought back by moving two pieces cost less code.
    auto back = [&](auto turn) {         // pieces 0 and 1 to fx[0] and fx[1]
        constexpr int R = decltype(turn)::value;
        if constexpr (R == 1) {
            const intx8 a = fx[1], b = fx[2];
            fx[0] = a, fx[1] = b;
        } else if constexpr (R == 2) {
            const intx8 a = fx[2], b = fx[0];
            fx[0] = a, fx[1] = b;
        }
    };
    auto advance = [&]() { s0 = s0 + 2 >= kUnits ? s0 + 2 - kUnits : s0 + 2; };
    constexpr int R1 = TM % 3, R2 = 2 * TM % 3;
    typedef std::integral_constant<int, 1> I1;
    auto pair = [&](int t, auto steady) {
        k_tile(t, steady, s0, I0{}, I0{});
        advance();
        k_tile(t + 1, steady, s0, I1{}, std::integral_constant<int, R1>{});
        advance();
        back(std::integral_constant<int, R2>{});
    };
#pragma unroll 1
    for (; t + 2 <= steady_end; t += 2) pair(t, std::true_type{});
#pragma unroll 1
    for (; t + 2 <= ktiles; t += 2) pair(t, std::false_type{});
    if (t < ktiles) k_tile(t, std::false_type{}, s0, I0{}, I0{});

    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");   // the last products have left the pipeline
    // Lane: of each 16 x 16 block row l16 and columns 4 kg .. + 3.
    float xs[TM];
#pragma unroll
    for (int b = 0; b < TM; ++b) {
        const int m = wm + b * 16 + l16;
        xs[b] = p.x_scales[m < p.M ? m : p.M - 1];
    }
    __syncthreads();   // nobody reads the operands any more, and every request has landed
    if (p.out_dtype == DDL_DT_F32) {
        float* const y = static_cast<float*>(p.y);
#pragma unroll
        for (int a = 0; a < kTN; ++a) {
            const int n = wn + a * 16 + 4 * kg;
            float ws[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) ws[e] = p.w_scales[n + e < p.N ? n + e : p.N - 1];
#pragma unroll
            for (int b = 0; b < TM; ++b) {
                const int m = wm + b * 16 + l16;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[a][b][e] * xs[b] * ws[e];
                if (m < p.M) store_floats(y + m * p.ldy, n, p.N, v);
            }
        }
        return;
    }
    // Through LDS, so that rows leave 16 bytes a lane, as the 16-bit tiles' do.
    constexpr int kPitch = kTN * 32;
    char* const region = lds + wave * (TM * 16 * kPitch);
#pragma unroll
    for (int a = 0; a < kTN; ++a) {
        const int n = wn + a * 16 + 4 * kg;
        float ws[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) ws[e] = p.w_scales[n + e < p.N ? n + e : p.N - 1];
#pragma unroll
        for (int b = 0; b < TM; ++b) {
            const int row = b * 16 + l16;
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = acc[a][b][e] * xs[b] * ws[e];
                o[e] = p.out_dtype == DDL_DT_F16 ? f32_to_elem<true>(v) : f32_to_elem<false>(v);
            }
            *reinterpret_cast<uint2*>(region + row * kPitch + (((a * 2 + (kg >> 1)) ^ ((row >> 1) & 7)) << 4) + (kg & 1) * 8) = make_uint2(o[0] | o[1] << 16, o[2] | o[3] << 16);
        }
    }
    asm volatile("" ::: "memory");   // a wavefront's LDS operations complete in order
    uint16_t* const y = static_cast<uint16_t*>(p.y);
#pragma unroll 4
    for (int q = 0; q < TM * 16 * 8 / 64; ++q) {
        const int at = q * 64 + lane, row = at / 8, chunk = at % 8, m = wm + row, n = wn + chunk * 8;
        const uint4 v = *reinterpret_cast<const uint4*>(region + row * kPitch + ((chunk ^ ((row >> 1) & 7)) << 4));
        if (m >= p.M || n >= p.N) continue;
        uint16_t* const dst = y + m * p.ldy + n;
        if (n + 8 <= p.N) {
            typedef u32x4 any __attribute__((aligned(2)));
            *reinterpret_cast<any*>(dst) = u32x4{v.x, v.y, v.z, v.w};
        } else {
            const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (n + e < p.N) dst[e] = static_cast<uint16_t>(words[e >> 1] >> (16 * (e & 1)));
        }
    }
}

// Tiles of 64 x 64 for products that do not fill the chip with larger ones: four wavefronts with 32 x 32 each, k-tiles through a ring of four, three of them
// in flight, one barrier a k-tile.  Bound by a k-tile's latencies.  ([8 x 16, 8192] by 3584: 38 us, tiles of 128 x 256 47, wavefronts on parts of the
// reduction 58; [16 x 128, 4096] by 512: 20, 28 and 41.)
constexpr int kSmall = 64, kSmallThreads = 256, kSmallRing = 4, kSmallStage = 2 * kSmall * kRowBytes;

__device__ __forceinline__ void small_tile8(const Tile8& p, char* lds) {
    constexpr int J = kSmall / 8 / 4;   // request instructions of a wavefront for either operand
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, kg = lane >> 4;
    const u32x4 buf_w = raw_buffer(p.w), buf_x = raw_buffer(p.x);
    int off_w[J], off_x[J];
    auto lane_offset = [&](int j, int rows, int64_t ld) -> int {
        const int row = (J * wave + j) * 8 + (lane >> 3);
        return static_cast<int>(static_cast<int64_t>(row < rows ? row : rows - 1) * ld) + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
    };
#pragma unroll
    for (int j = 0; j < J; ++j) off_w[j] = lane_offset(j, p.N, p.ldw), off_x[j] = lane_offset(j, p.M, p.ldx);
    const int ktiles = static_cast<int>((p.K + kRowBytes - 1) / kRowBytes), full_tiles = static_cast<int>(p.K / kRowBytes);
    auto through = [&](const uint8_t* base, int off, int j, int t, char* to) {   // of the k-tile that K ends in, zeros behind its end
        const int row = (J * wave + j) * 8 + (lane >> 3), chunk = (lane & 7) ^ ((row >> 1) & 7);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (static_cast<int64_t>(t) * kRowBytes + chunk * 16 < p.K) v = *reinterpret_cast<const uint4*>(base + off + static_cast<int64_t>(t) * kRowBytes);
        *reinterpret_cast<uint4*>(to + (J * wave + j) * 1024 + lane * 16) = v;
    };
    auto request = [&](int t) {
        char* const w = lds + t % kSmallRing * kSmallStage;
        char* const x = w + kSmall * kRowBytes;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (t < full_tiles) {
                dma16(buf_w, off_w[j], t * kRowBytes, w + (J * wave + j) * 1024);
                dma16(buf_x, off_x[j], t * kRowBytes, x + (J * wave + j) * 1024);
            } else {
                through(p.w, off_w[j], j, t, w);
                through(p.x, off_x[j], j, t, x);
            }
        }
    };
    const int sw = (l16 >> 1) & 7, at0 = l16 * kRowBytes + ((kg ^ sw) << 4), at1 = l16 * kRowBytes + (((4 + kg) ^ sw) << 4);
    auto read = [&](const char* tile, int row) -> intx8 {
        intx8 v;
        const uint4 a = *reinterpret_cast<const uint4*>(tile + row * kRowBytes + at0), b = *reinterpret_cast<const uint4*>(tile + row * kRowBytes + at1);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        return v;
    };
    const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
    floatx4 acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < kSmallRing - 1; ++t)
        if (t < ktiles) request(t);
#pragma unroll 1
    for (int t = 0; t < ktiles; ++t) {
        // Tile t has landed (the two behind it may be in flight), and this wavefront has read tile t - 1.
        if (t + kSmallRing - 2 < full_tiles) __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(2 * J * (kSmallRing - 2)));
        else __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (t + kSmallRing - 1 < ktiles) request(t + kSmallRing - 1);
        const char* const w = lds + t % kSmallRing * kSmallStage + wn * kRowBytes;
        const char* const x = lds + t % kSmallRing * kSmallStage + (kSmall + wm) * kRowBytes;
        const intx8 fw[2] = {read(w, 0), read(w, 16)}, fx[2] = {read(x, 0), read(x, 16)};
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int b = 0; b < 2; ++b)
                acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[a], fx[b], acc[a][b], 0, 0, 0, 0x7F7F7F7F, 0, 0x7F7F7F7F);   // scales of one
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int m = wm + b * 16 + l16;
        if (m >= p.M) continue;
        const float xs = p.x_scales[m];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int n = wn + a * 16 + 4 * kg;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[a][b][e] * xs * p.w_scales[n + e < p.N ? n + e : p.N - 1];
            if (p.out_dtype == DDL_DT_F32) store_floats(static_cast<float*>(p.y) + m * p.ldy, n, p.N, v);
            else if (p.out_dtype == DDL_DT_F16) store_four<true>(static_cast<uint16_t*>(p.y), p.ldy, m, n, p.N, v);
            else store_four<false>(static_cast<uint16_t*>(p.y), p.ldy, m, n, p.N, v);
        }
    }
}

// The tile of workgroup `id`, if it has one to compute (rows of no expert get their zeros here).
template <int BM, int BN>
__device__ inline bool tile_of(const ExpertArgs& g, int id, Tile8& p) {
    const ExpertTask t = find_tile<false>(g, BM, id);
    if (t.expert < 0) return false;
    const int64_t n0 = static_cast<int64_t>(t.tn) * BN;
    const int cols = static_cast<int>(min(g.n - n0, static_cast<int64_t>(BN))), rows = min(t.rows, BM);
    const int64_t at = t.row * g.ldy + n0;
    if (t.expert == g.experts) {
        if (g.out_dtype == DDL_DT_F32) zero_block(static_cast<float*>(g.y) + at, g.ldy, rows, cols);
        else zero_block(static_cast<uint16_t*>(g.y) + at, g.ldy, rows, cols);
        return false;
    }
    p.x = static_cast<const uint8_t*>(g.a) + t.row * g.lda, p.w = static_cast<const uint8_t*>(g.w) + t.expert * g.w_stride + n0 * g.ldw;
    p.x_scales = g.a_scales + t.row, p.w_scales = g.w_scales + t.expert * g.n + n0;
    p.y = g.out_dtype == DDL_DT_F32 ? static_cast<void*>(static_cast<float*>(g.y) + at) : static_cast<void*>(static_cast<uint16_t*>(g.y) + at);
    p.M = rows, p.N = cols, p.out_dtype = g.out_dtype, p.K = g.k, p.ldx = g.lda, p.ldw = g.ldw, p.ldy = g.ldy;
    return true;
}

template <int TM>
__global__ __launch_bounds__(kThreads8, 2) void expert_rows8(const ExpertArgs g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    Tile8 p;
    if (tile_of<32 * TM, kColumns>(g, blockIdx.x, p)) tile8<TM>(p, lds);
}

__global__ __launch_bounds__(kSmallThreads, 2) void expert_rows8_small(const ExpertArgs g) {
    __shared__ __attribute__((aligned(16))) char lds[kSmallRing * kSmallStage];
    Tile8 p;
    if (tile_of<kSmall, kSmall>(g, blockIdx.x, p)) small_tile8(p, lds);
}

template <int TM>
int launch8(const char* who, ExpertArgs g, int dev, hipStream_t s) {
    static std::atomic<bool> reserved[kMaxDevices];
    const auto kernel = expert_rows8<TM>;
    if (!reserved[dev].load(std::memory_order_acquire)) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes);
        if (e != hipSuccess) return fail(static_cast<int>(e), "%s: cannot reserve %d bytes of LDS: %s", who, kLdsBytes, hipGetErrorString(e));
        reserved[dev].store(true, std::memory_order_release);
    }
    g.tiles_n = static_cast<int>((g.n + kColumns - 1) / kColumns);
    const int64_t blocks = ((g.rows + 32 * TM - 1) / (32 * TM) + g.experts) * static_cast<int64_t>(g.tiles_n);
    if (blocks * kThreads8 > 0xFFFFFFFFll) return fail(DDL_E_UNSUPP, "%s: %lld tiles", who, static_cast<long long>(blocks));
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads8), kLdsBytes, s, g);
    return check_launch(who);
}

}  // namespace

int run_expert_rows8(const char* who, ExpertTile tile, ExpertArgs g, int dev, hipStream_t s) {
    if (tile == ExpertTile::kLarge) return launch8<8>(who, g, dev, s);
    if (tile == ExpertTile::kLow) return launch8<4>(who, g, dev, s);
    g.tiles_n = static_cast<int>((g.n + kSmall - 1) / kSmall);
    const int64_t blocks = ((g.rows + kSmall - 1) / kSmall + g.experts) * static_cast<int64_t>(g.tiles_n);
    if (blocks * kSmallThreads > 0xFFFFFFFFll) return fail(DDL_E_UNSUPP, "%s: %lld tiles", who, static_cast<long long>(blocks));
    hipLaunchKernelGGL(expert_rows8_small, dim3(static_cast<uint32_t>(blocks)), dim3(kSmallThreads), 0, s, g);
    return check_launch(who);
}

}  // namespace ddl
