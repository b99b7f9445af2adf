// The products of rows with the weights of the expert that each was sent to, and their adjoint: the entry points and the
// kernel for few rows.  (expert_linear8.hip, expert_linear16.hip, expert_linear32.hip: tiles.)
//
// expert_stream (bf16, fp16 and e4m3; few rows for each expert): bound by reading the weights once.  A workgroup has 32 rows of one
// expert's weights; its wavefronts take the 128-byte lines of those in turn, 16 rows at a time straight from memory into registers
// as a matrix instruction wants them (lane l reads 32 bytes of row l % 16: which element of a reduction a lane holds is free if both
// operands agree), next to the same lines of up to 16 MB rows of the expert's.  The wavefronts' sums meet in LDS.  More rows than
// that take the weights' lines again, from the L2.
//
// e4m3 products: the matrix cores' own, which add eight of them at a time and cut each off at 2^-13 of the largest one's power of two, and
// those sums in 32 bits.  Of rows of normally distributed elements that is 2^-12 of a result, next to 2^-9 for its rounding to bf16
// and 2^-5 for the rows' own; bf16 products of the same codes would be exact at half the rate.
#include "expert_parts.h"
#include "gemm16_parts.h"

namespace ddl {
namespace {

// ------------------------------------------------------------ few rows --

enum Kind { kBf16, kF16, kE4m3 };

constexpr int kStreamWaves = 4, kStreamCols = 32;

struct Line {
    uint4 half[2];   // 32 bytes of a row
};
typedef int intx8 __attribute__((ext_vector_type(8)));

template <int KIND>
__device__ inline floatx4 multiply_line(const Line& w, const Line& x, floatx4 acc) {
    if constexpr (KIND == kE4m3) {
        intx8 a, b;
        __builtin_memcpy(&a, &w, 32);
        __builtin_memcpy(&b, &x, 32);
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, 0, 0x7F7F7F7F, 0, 0x7F7F7F7F);   // scales of one
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            bf16x8 a, b;
            __builtin_memcpy(&a, &w.half[h], 16);
            __builtin_memcpy(&b, &x.half[h], 16);
            acc = mfma<KIND == kF16>(a, b, acc);
        }
        return acc;
    }
}

__device__ inline Line load_line(const char* p) {
    Line l;
    l.half[0] = *reinterpret_cast<const uint4*>(p), l.half[1] = *reinterpret_cast<const uint4*>(p + 16);
    return l;
}
// Up to `left` bytes of it (a multiple of 16), zeros behind them.
__device__ inline Line load_line_end(const char* p, int left) {
    Line l;
    l.half[0] = left > 0 ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
    l.half[1] = left > 16 ? *reinterpret_cast<const uint4*>(p + 16) : make_uint4(0, 0, 0, 0);
    return l;
}

__device__ inline void store_out(const ExpertArgs& g, int64_t row, int64_t n, float v) {
    const int64_t at = row * g.ldy + n;
    if (g.out_dtype == DDL_DT_F32) static_cast<float*>(g.y)[at] = v;
    else static_cast<uint16_t*>(g.y)[at] = g.out_dtype == DDL_DT_F16 ? f32_to_elem<true>(v) : f32_to_elem<false>(v);
}

template <int KIND, int MB>
__global__ __launch_bounds__(64 * kStreamWaves) void expert_stream(const ExpertArgs g) {
    constexpr int NB = kStreamCols / 16, kAhead = 4;   // lines in flight together
    constexpr int kBytes = KIND == kE4m3 ? 1 : 2;
    __shared__ floatx4 sums[kStreamWaves][NB * MB][64];
    const int e = blockIdx.y;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kStreamCols;
    int lo, hi;
    rows_of_expert(g, e, lo, hi);
    if (lo == hi) return;
    if (e == g.experts) {
        const int cols = static_cast<int>(min(g.n - n0, static_cast<int64_t>(kStreamCols)));
        for (int64_t i = threadIdx.x; i < static_cast<int64_t>(hi - lo) * cols; i += blockDim.x) store_out(g, lo + i / cols, n0 + i % cols, 0.f);
        return;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, part = lane >> 4;
    const int64_t bytes = g.k * kBytes;
    const int lines = static_cast<int>(bytes / 128), end = static_cast<int>(bytes % 128) - part * 32;
    const char *w[NB], *x[MB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t n = n0 + b * 16 + l16;
        w[b] = static_cast<const char*>(g.w) + (e * g.w_stride + (n < g.n ? n : g.n - 1) * g.ldw) * kBytes + part * 32;
    }
    for (int m0 = lo; m0 < hi; m0 += 16 * MB) {
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            const int64_t m = m0 + b * 16 + l16;
            x[b] = static_cast<const char*>(g.a) + (m < hi ? m : hi - 1) * g.lda * kBytes + part * 32;
        }
        floatx4 acc[NB][MB];
#pragma unroll
        for (int a = 0; a < NB; ++a)
#pragma unroll
            for (int b = 0; b < MB; ++b) acc[a][b] = floatx4{0.f, 0.f, 0.f, 0.f};
        int i = wave;
        for (; i + (kAhead - 1) * kStreamWaves < lines; i += kAhead * kStreamWaves) {
            Line lw[kAhead][NB], lx[kAhead][MB];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int64_t at = static_cast<int64_t>(i + u * kStreamWaves) * 128;
#pragma unroll
                for (int b = 0; b < NB; ++b) lw[u][b] = load_line(w[b] + at);
#pragma unroll
                for (int b = 0; b < MB; ++b) lx[u][b] = load_line(x[b] + at);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
#pragma unroll
                for (int a = 0; a < NB; ++a)
#pragma unroll
                    for (int b = 0; b < MB; ++b) acc[a][b] = multiply_line<KIND>(lw[u][a], lx[u][b], acc[a][b]);
        }
        for (; i <= lines; i += kStreamWaves) {
            const int64_t at = static_cast<int64_t>(i) * 128;
            const int left = i < lines ? 128 : end;   // the last line may have some bytes, or none
            Line lw[NB], lx[MB];
#pragma unroll
            for (int b = 0; b < NB; ++b) lw[b] = load_line_end(w[b] + at, left);
#pragma unroll
            for (int b = 0; b < MB; ++b) lx[b] = load_line_end(x[b] + at, left);
#pragma unroll
            for (int a = 0; a < NB; ++a)
#pragma unroll
                for (int b = 0; b < MB; ++b) acc[a][b] = multiply_line<KIND>(lw[a], lx[b], acc[a][b]);
        }
        if (m0 != lo) __syncthreads();   // the sums before these have been read
#pragma unroll
        for (int a = 0; a < NB; ++a)
#pragma unroll
            for (int b = 0; b < MB; ++b) sums[wave][a * MB + b][lane] = acc[a][b];
        __syncthreads();
        // Lane: row l16, columns 4 part to 4 part + 3 of a block of 16 x 16.
        for (int q = wave; q < NB * MB; q += kStreamWaves) {
            floatx4 v = sums[0][q][lane];
#pragma unroll
            for (int s = 1; s < kStreamWaves; ++s) v += sums[s][q][lane];
            const int64_t m = m0 + (q % MB) * 16 + l16, n = n0 + (q / MB) * 16 + 4 * part;
            if (m >= hi) continue;
            const float scale = KIND == kE4m3 ? g.a_scales[m] : 1.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (n + j < g.n) store_out(g, m, n + j, KIND == kE4m3 ? v[j] * scale * g.w_scales[e * g.n + n + j] : v[j]);
            }
        }
    }
}

template <int KIND>
int launch_stream(const char* who, const ExpertArgs& g, hipStream_t s) {
    const int64_t strips = (g.n + kStreamCols - 1) / kStreamCols;
    if (strips > 0x7FFFFF || g.experts + 1 > 65535) return fail(DDL_E_UNSUPP, "%s: %lld columns of %d experts", who, static_cast<long long>(g.n), g.experts);
    const dim3 grid(static_cast<uint32_t>(strips), static_cast<uint32_t>(g.experts + 1)), block(64 * kStreamWaves);
    const int64_t each = g.rows / (g.experts > 0 ? g.experts : 1);
    if (each <= 8) hipLaunchKernelGGL((expert_stream<KIND, 1>), grid, block, 0, s, g);
    else if (each <= 24) hipLaunchKernelGGL((expert_stream<KIND, 2>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((expert_stream<KIND, 4>), grid, block, 0, s, g);
    return check_launch(who);
}

// ------------------------------------------------------------ dispatch --

constexpr int64_t kMostSpan = 0x3FFFFFFF;   // elements that a tile's 32-bit byte offsets reach over

// Rows for an expert on average, above which tiles are the faster way.
constexpr int64_t kStreamRows = 32;

ExpertTile tile_for(bool aligned, int64_t tiles_large, int64_t rows_each, int cus) {
    if (!aligned) return rows_each >= 128 && tiles_large >= cus / 2 ? ExpertTile::kAny128 : ExpertTile::kAny64;
    if (tiles_large >= 2 * cus && rows_each >= 512) return ExpertTile::kLarge;
    return tiles_large * 2 >= cus ? ExpertTile::kLow : ExpertTile::kAny64;
}

int check_product(const char* who, int64_t experts, int64_t rows, int64_t n, int64_t k, int64_t least) {
    if (experts < 0 || rows < 0 || n < 1 || k < 1)
        return fail(DDL_E_ARG, "%s: %lld experts, %lld rows, %lld x %lld features", who, static_cast<long long>(experts), static_cast<long long>(rows), static_cast<long long>(n),
                    static_cast<long long>(k));
    if (n < least || k < least) return fail(DDL_E_UNSUPP, "%s: %lld x %lld features (at least %lld)", who, static_cast<long long>(n), static_cast<long long>(k), static_cast<long long>(least));
    if (rows > 0x3FFFFFFF || experts > 65534 || n > 0x3FFFFF || k > 0x3FFFFF || (n + 64) * (k + 64) > kMostSpan / 2)
        return fail(DDL_E_UNSUPP, "%s: %lld experts of %lld x %lld features and %lld rows", who, static_cast<long long>(experts), static_cast<long long>(n), static_cast<long long>(k),
                    static_cast<long long>(rows));
    return 0;
}

}  // namespace
}  // namespace ddl

extern "C" {

int ddl_expert_linear(const void* x, const void* w, int dtype, const int32_t* offsets, int64_t experts, int64_t rows, int64_t n, int64_t k, int64_t ld_x, void* y,
                      void* stream) {
    using namespace ddl;
    const char* who = "ddl_expert_linear";
    if (dtype != DDL_DT_F32 && dtype != DDL_DT_BF16 && dtype != DDL_DT_F16) return fail(DDL_E_ARG, "%s: dtype %d", who, dtype);
    if (int rc = check_product(who, experts, rows, n, k, dtype == DDL_DT_F32 ? 1 : 8)) return rc;
    if (rows == 0) return 0;
    if (!x || !y || !offsets || (experts && !w)) return fail(DDL_E_ARG, "%s: null pointer", who);
    if (rows > 1 && ld_x < k) return fail(DDL_E_ARG, "%s: pitch below %lld features", who, static_cast<long long>(k));
    if (ld_x > 0x3FFFFF) return fail(DDL_E_UNSUPP, "%s: pitch above 2^22 elements", who);
    int dev = 0;
    const int cus = compute_units(dev);
    ExpertArgs g{};
    g.a = x, g.w = w, g.y = y, g.offsets = offsets, g.experts = static_cast<int>(experts), g.rows = static_cast<int>(rows), g.out_dtype = dtype;
    g.n = n, g.k = k, g.lda = rows > 1 ? ld_x : k, g.ldw = k, g.w_stride = n * k, g.ldy = n;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == DDL_DT_F32) return run_expert_rows32(who, false, g, s);
    const bool aligned = aligned_to(x, 16) && aligned_to(w, 16) && g.lda % 8 == 0 && k % 8 == 0;
    const int64_t each = rows / (experts ? experts : 1);
    if (aligned && each <= kStreamRows) return dtype == DDL_DT_F16 ? launch_stream<kF16>(who, g, s) : launch_stream<kBf16>(who, g, s);
    return run_expert_rows16(who, tile_for(aligned, (rows + 255) / 256 * ((n + 255) / 256), each, cus), dtype == DDL_DT_F16, false, g, dev, s);
}

int ddl_expert_linear_8bit(const void* x, const float* x_scales, const void* w, const float* w_scales, const int32_t* offsets, int64_t experts, int64_t rows,
                           int64_t n, int64_t k, int64_t ld_x, void* y, int out_dtype, void* stream) {
    using namespace ddl;
    const char* who = "ddl_expert_linear_8bit";
    if (out_dtype != DDL_DT_F32 && out_dtype != DDL_DT_BF16 && out_dtype != DDL_DT_F16) return fail(DDL_E_ARG, "%s: dtype %d of the result", who, out_dtype);
    if (int rc = check_product(who, experts, rows, n, k, 1)) return rc;
    if (rows == 0) return 0;
    if (!x || !x_scales || !y || !offsets || (experts && (!w || !w_scales))) return fail(DDL_E_ARG, "%s: null pointer", who);
    if (rows > 1 && ld_x < k) return fail(DDL_E_ARG, "%s: pitch below %lld features", who, static_cast<long long>(k));
    const int64_t pitch = rows > 1 ? ld_x : k;
    if (k % 16 || pitch % 16 || !aligned_to(x, 16) || !aligned_to(w, 16))
        return fail(DDL_E_ALIGN, "%s: rows of %lld elements, %lld apart: 16-byte aligned rows of a multiple of 16 elements are taken", who, static_cast<long long>(k),
                    static_cast<long long>(pitch));
    if (pitch > 0x3FFFFF) return fail(DDL_E_UNSUPP, "%s: pitch above 2^22 elements", who);
    ExpertArgs g{};
    g.a = x, g.w = w, g.y = y, g.offsets = offsets, g.a_scales = x_scales, g.w_scales = w_scales, g.experts = static_cast<int>(experts), g.rows = static_cast<int>(rows);
    g.out_dtype = out_dtype, g.n = n, g.k = k, g.lda = pitch, g.ldw = k, g.w_stride = n * k, g.ldy = n;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t each = rows / (experts ? experts : 1);
    if (each <= kStreamRows) return launch_stream<kE4m3>(who, g, s);
    int dev = 0;
    const int cus = compute_units(dev);
    return run_expert_rows8(who, tile_for(true, (rows + 255) / 256 * ((n + 255) / 256), each, cus) != ExpertTile::kLarge, g, dev, s);
}

int ddl_expert_linear_backward(const void* dy, const void* x, const void* w, int dtype, const int32_t* offsets, int64_t experts, int64_t rows, int64_t n, int64_t k,
                               int64_t ld_dy, int64_t ld_x, void* dx, void* dw, void* stream) {
    using namespace ddl;
    const char* who = "ddl_expert_linear_backward";
    if (dtype != DDL_DT_F32 && dtype != DDL_DT_BF16 && dtype != DDL_DT_F16) return fail(DDL_E_ARG, "%s: dtype %d", who, dtype);
    if (int rc = check_product(who, experts, rows, n, k, dtype == DDL_DT_F32 ? 1 : 8)) return rc;
    if ((dx && rows) || (dw && experts)) {
        if (!offsets || (rows && !dy) || (dx && experts && !w) || (dw && rows && !x)) return fail(DDL_E_ARG, "%s: null pointer", who);
    }
    if (rows > 1 && (ld_dy < n || (dw && ld_x < k))) return fail(DDL_E_ARG, "%s: pitch below %lld or %lld features", who, static_cast<long long>(n), static_cast<long long>(k));
    if (ld_dy > 0x3FFFFF || (dw && ld_x > 0x3FFFFF)) return fail(DDL_E_UNSUPP, "%s: pitch above 2^22 elements", who);
    const int64_t pitch_dy = rows > 1 ? ld_dy : n, pitch_x = rows > 1 ? ld_x : k;
    const int64_t span = (rows + 64) * (dw && pitch_x > pitch_dy ? pitch_x : pitch_dy);
    const bool within = span <= (dtype == DDL_DT_F32 ? kMostSpan / 2 : kMostSpan);
    if (dw && experts && dtype == DDL_DT_F32 && !within)
        return fail(DDL_E_UNSUPP, "%s: %lld rows, %lld elements apart, are more than 2^31 bytes", who, static_cast<long long>(rows), static_cast<long long>(pitch_x > pitch_dy ? pitch_x : pitch_dy));
    int dev = 0;
    const int cus = compute_units(dev);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool f16 = dtype == DDL_DT_F16;
    const int64_t each = rows / (experts ? experts : 1);
    ExpertArgs g{};
    g.offsets = offsets, g.experts = static_cast<int>(experts), g.rows = static_cast<int>(rows), g.out_dtype = dtype;
    if (dx && rows) {   // rows of n features by w read along its k columns
        ExpertArgs d = g;
        d.a = dy, d.w = w, d.y = dx, d.n = k, d.k = n, d.lda = pitch_dy, d.ldw = k, d.w_stride = n * k, d.ldy = k;
        int rc;
        if (dtype == DDL_DT_F32) {
            rc = run_expert_rows32(who, true, d, s);
        } else {
            const bool aligned = aligned_to(dy, 16) && aligned_to(w, 16) && pitch_dy % 8 == 0 && n % 8 == 0 && k % 8 == 0;
            rc = run_expert_rows16(who, tile_for(aligned, (rows + 255) / 256 * ((k + 255) / 256), each, cus), f16, true, d, dev, s);
        }
        if (rc) return rc;
    }
    if (dw && experts) {
        ExpertArgs d = g;
        d.a = dy, d.w = x, d.y = dw, d.n = n, d.k = k, d.lda = pitch_dy, d.ldw = pitch_x;
        if (dtype == DDL_DT_F32) return run_expert_weights32(who, d, s);
        const bool aligned = aligned_to(dy, 16) && aligned_to(x, 16) && pitch_dy % 8 == 0 && pitch_x % 8 == 0 && n % 8 == 0 && k % 8 == 0 && within;
        return run_expert_weights16(who, tile_for(aligned, experts * ((n + 255) / 256) * ((k + 255) / 256), 1 << 20, cus), f16, d, dev, s);
    }
    return 0;
}

}  // extern "C"
