// Root-mean-square norm of rows, with the addition of a residual in front and an 8-bit output behind it in the same pass:
//   h = x + residual (rounded to its type: the stream that goes on),  y = h / sqrt(mean of h^2 + eps) * weight,
// or, in 8 bits, scale = max(max |y| / 448, 2^-126) and code = e4m3(y / scale) for each row (the quotient rounded once); and the adjoint,
//   g = dy weight,  xhat = h rstd,  dx = rstd (g - xhat mean(g xhat)) + dh,  dweight = sum over rows of dy xhat.
//
// Bound by HBM: every operand is read and every result written once.  A row is held in the registers of a group of 64 to 1024
// threads, eight elements a thread and piece, so the sums, the largest value and the results need no second reading; the adjoint
// forms rstd again from h, which it reads for the gradient anyway, instead of keeping it.  A group walks over some rows, the next one asked for
// while one is summed ([8192, 8192] bf16 on operands that stay: norm with a residual 92 -> 80 us, adjoint 132 -> 107; groups of 256 or
// 512 threads with more pieces were no faster, the adjoint 119 to 180).  Rows at any address and of any
// length: the last piece of a row is moved back until it ends with the row, and what it then holds twice does not count in the
// sums.  Sums, rstd, scales and the weight's partial sums are 32-bit floats; results are rounded once.
//
// Where the columns of a row are spread over workers, a launch leaves this worker's sum for each row (own_squares, own_sums),
// and another takes those of all of them (part_squares, part_sums, one after the other as the workers are numbered).
#include "ln_elements.h"

namespace ddl {
namespace {

constexpr int kPiece = 8;            // elements of a thread's piece of a row
constexpr int kMaxCols = 16384;
constexpr float kE4m3Max = 448.f, kSmallestScale = 1.17549435e-38f;   // 2^-126: its reciprocal is still finite

struct RmsArgs {
    const void *x, *residual, *weight, *dy, *dh;
    void *h, *y;                      // y: dx in the adjoint
    uint8_t* codes;
    float* scales;
    float* own;                       // this worker's sums only
    const float *part_squares, *part_sums;
    float* partial;                   // weight's partial sums, [gridDim.x, cols]
    int64_t rows, ld_x, ld_r, ld_dy, ld_dh;
    int cols, nparts;
    float inv_cols, eps;
};

// Eight elements as they lie, at the alignment of one.
template <typename T>
struct Raw {
    uint32_t word[2 * sizeof(T)];
};
template <typename T>
__device__ inline Raw<T> load_raw(const T* p) {
    struct __attribute__((packed, aligned(sizeof(T)))) Any {
        Raw<T> raw;
    };
    return reinterpret_cast<const Any*>(p)->raw;
}
template <typename T>
__device__ inline void store_raw(T* p, const Raw<T>& r) {
    typedef uint32_t u32x4_v __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
        store_stream(reinterpret_cast<char*>(p) + 16 * i, u32x4_v{r.word[4 * i], r.word[4 * i + 1], r.word[4 * i + 2], r.word[4 * i + 3]});
}
__device__ inline void unpack(const Raw<float>& r, float (&v)[kPiece]) {
#pragma unroll
    for (int e = 0; e < kPiece; ++e) v[e] = __uint_as_float(r.word[e]);
}
__device__ inline void unpack(const Raw<bf16_t>& r, float (&v)[kPiece]) {
#pragma unroll
    for (int e = 0; e < kPiece; ++e) v[e] = __uint_as_float(e % 2 ? r.word[e / 2] & 0xFFFF0000u : r.word[e / 2] << 16);
}
__device__ inline void unpack(const Raw<__half>& r, float (&v)[kPiece]) {
#pragma unroll
    for (int e = 0; e < kPiece; e += 2) {
        const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&r.word[e / 2]));
        v[e] = two.x, v[e + 1] = two.y;
    }
}
__device__ inline Raw<float> pack(const float (&v)[kPiece], float*) {
    Raw<float> r;
#pragma unroll
    for (int e = 0; e < kPiece; ++e) r.word[e] = __float_as_uint(v[e]);
    return r;
}
__device__ inline Raw<bf16_t> pack(const float (&v)[kPiece], bf16_t*) {
    Raw<bf16_t> r;
#pragma unroll
    for (int e = 0; e < kPiece; e += 2) r.word[e / 2] = f32x2_to_bf16(v[e], v[e + 1]);
    return r;
}
__device__ inline Raw<__half> pack(const float (&v)[kPiece], __half*) {
    Raw<__half> r;
#pragma unroll
    for (int e = 0; e < kPiece; e += 2) {
        const __half2 two = __floats2half2_rn(v[e], v[e + 1]);
        __builtin_memcpy(&r.word[e / 2], &two, 4);
    }
    return r;
}

// Where a piece lies in its row.  count: its elements (0: none; below 8 only in rows shorter than that), skip: those at its front
// that belong to the piece before it.
struct Place {
    int at, count, skip;
};
__device__ inline Place place_of(int piece, int cols) {
    const int at = piece * kPiece;
    if (at >= cols) return {0, 0, 0};
    if (at + kPiece <= cols) return {at, kPiece, 0};
    return cols >= kPiece ? Place{cols - kPiece, kPiece, at + kPiece - cols} : Place{0, cols, 0};
}

template <typename T>
__device__ inline Raw<T> load_place(const T* row, const Place& p) {
    Raw<T> r{};
    if (p.count == kPiece) return load_raw(row + p.at);
    T own[kPiece];
    __builtin_memcpy(own, &r, sizeof(r));
#pragma unroll
    for (int e = 0; e < kPiece; ++e)
        if (e < p.count) own[e] = row[e];
    __builtin_memcpy(&r, own, sizeof(r));
    return r;
}
template <typename T>
__device__ inline void store_place(T* row, const Place& p, const Raw<T>& r) {
    if (p.count == kPiece) return store_raw(row + p.at, r);
    T own[kPiece];
    __builtin_memcpy(own, &r, sizeof(r));
#pragma unroll
    for (int e = 0; e < kPiece; ++e)
        if (e < p.count) row[e] = own[e];
}
__device__ inline void store_codes(uint8_t* row, const Place& p, uint32_t lo, uint32_t hi) {
    if (p.count == kPiece) {
        typedef uint32_t u32x2_v __attribute__((ext_vector_type(2)));
        typedef u32x2_v any __attribute__((aligned(1)));
        *reinterpret_cast<any*>(row + p.at) = u32x2_v{lo, hi};
        return;
    }
#pragma unroll
    for (int e = 0; e < kPiece; ++e)
        if (e < p.count) row[e] = static_cast<uint8_t>((e < 4 ? lo : hi) >> (8 * (e & 3)));
}

// Largest of the 64 lanes' values, none of them below zero, in every lane; moves as wave_sum's.
__device__ inline float wave_max(float v) {
    v = fmaxf(v, dpp_moved<0xB1, 0xF>(v));
    v = fmaxf(v, dpp_moved<0x4E, 0xF>(v));
    v = fmaxf(v, dpp_moved<0x141, 0xF>(v));
    v = fmaxf(v, dpp_moved<0x140, 0xF>(v));
    v = fmaxf(v, dpp_moved<0x142, 0xA>(v));
    v = fmaxf(v, dpp_moved<0x143, 0xC>(v));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// N sums (or largest values) over the group's threads, the same in all of them.  One barrier: the next reduction takes the other
// half of `lds`, and nobody is two reductions ahead.
template <int THREADS, int N, bool MAX>
__device__ inline void over_group(float (&v)[N], float* lds, int& turn) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = MAX ? wave_max(v[i]) : wave_sum(v[i]);
    if constexpr (THREADS > 64) {
        constexpr int kWaves = THREADS / 64;
        float* const mine = lds + turn * (2 * kWaves);
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) mine[i * kWaves + threadIdx.x / 64] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float t = mine[i * kWaves];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) t = MAX ? fmaxf(t, mine[i * kWaves + w]) : t + mine[i * kWaves + w];
            v[i] = t;
        }
    }
}

__device__ inline float over_parts(const float* sums, int nparts, int64_t rows, int64_t row) {
    float t = 0.f;
    for (int p = 0; p < nparts; ++p) t += sums[p * rows + row];
    return t;
}

// v / scale as one rounding gives it, from the rounded reciprocal: the first product is off by less than 1.5 steps, the first correction leaves less than one, and the
// second, of an exact remainder, the rounded quotient.  Both factors are lifted where remainders of quotients that are no code of zero would be subnormal numbers.  A remainder of
// zero leaves a zero its sign.  ([8192, 8192] bf16 in 8 bits 40 us, by divisions 48; by the reciprocal alone 35, but next to a border some codes were their neighbours.  With norm and residual 95, 99
// and 91.)
__device__ inline float quotient(float v, float scale, float inverse) {
    float q = v * inverse;
    q = fmaf(-fmaf(q, scale, -v), inverse, q);
    return fmaf(-fmaf(q, scale, -v), inverse, q);
}

template <int THREADS>
constexpr int kBlockOf = THREADS < 256 ? 256 : THREADS;

// NORM false: the rows themselves in 8 bits.
template <typename T, int THREADS, int PIECES, bool EIGHT, bool NORM>
__global__ __launch_bounds__(kBlockOf<THREADS>) void rms_rows(const RmsArgs a) {
    constexpr int kGroups = kBlockOf<THREADS> / THREADS;
    __shared__ float lds[4 * (THREADS / 64)];
    int turn = 0;
    const int t = threadIdx.x % THREADS;
    Place place[PIECES];
    Raw<T> w[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        place[p] = place_of(p * THREADS + t, a.cols);
        if (NORM && a.weight) w[p] = load_place(static_cast<const T*>(a.weight), place[p]);
    }
    const bool odd = a.cols % kPiece != 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
    Raw<T> next_x[PIECES], next_r[PIECES];   // of the row behind the one that is worked on
    auto ask = [&](int64_t row) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            next_x[p] = load_place(static_cast<const T*>(a.x) + row * a.ld_x, place[p]);
            if (NORM && a.residual) next_r[p] = load_place(static_cast<const T*>(a.residual) + row * a.ld_r, place[p]);
        }
    };
    int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / THREADS;
    if (row < a.rows) ask(row);
    for (; row < a.rows; row += step) {
        Raw<T> h[PIECES], r[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) h[p] = next_x[p], r[p] = next_r[p];
        if (row + step < a.rows) ask(row + step);
        if (NORM && a.residual) {
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                float u[kPiece], v[kPiece];
                unpack(h[p], u), unpack(r[p], v);
#pragma unroll
                for (int e = 0; e < kPiece; ++e) u[e] += v[e];
                h[p] = pack(u, static_cast<T*>(nullptr));
                if (place[p].count) store_place(static_cast<T*>(a.h) + row * a.cols, place[p], h[p]);
            }
        }
        float rstd = 1.f;
        if (NORM) {
            float sum[1] = {0.f};
            if (!a.part_squares) {
#pragma unroll
                for (int p = 0; p < PIECES; ++p) {
                    float v[kPiece];
                    unpack(h[p], v);
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) sum[0] += !odd || e >= place[p].skip ? v[e] * v[e] : 0.f;
                }
                over_group<THREADS, 1, false>(sum, lds, turn);
            } else {
                sum[0] = over_parts(a.part_squares, a.nparts, a.rows, row);
            }
            if (a.own) {
                if (t == 0) a.own[row] = sum[0];
                continue;
            }
            rstd = 1.f / sqrtf(sum[0] * a.inv_cols + a.eps);
        }
        auto result = [&](int p, float (&y)[kPiece]) {
            unpack(h[p], y);
            if (NORM) {
                float v[kPiece];
                if (a.weight) unpack(w[p], v);
#pragma unroll
                for (int e = 0; e < kPiece; ++e) y[e] = a.weight ? y[e] * rstd * v[e] : y[e] * rstd;
            }
        };
        if constexpr (!EIGHT) {
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                float y[kPiece];
                result(p, y);
                if (place[p].count) store_place(static_cast<T*>(a.y) + row * a.cols, place[p], pack(y, static_cast<T*>(nullptr)));
            }
        } else {
            float top[1] = {0.f};
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                float y[kPiece];
                result(p, y);
                if (place[p].count) {
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) top[0] = fmaxf(top[0], fabsf(y[e]));
                }
            }
            over_group<THREADS, 1, true>(top, lds, turn);
            const float scale = fmaxf(top[0] * (1.f / kE4m3Max), kSmallestScale);   // the rounded reciprocal's product
            const float lift = scale < 0x1p-60f ? 0x1p64f : 1.f, lifted = scale * lift, inverse = 1.f / lifted;
            if (t == 0) a.scales[row] = scale;
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                float y[kPiece];
                result(p, y);
#pragma unroll
                for (int e = 0; e < kPiece; ++e) {
                    const float v = quotient(y[e] * lift, lifted, inverse);   // up to 448 and a rounding; not a number stays none
                    y[e] = v != v ? v : fminf(fmaxf(v, -kE4m3Max), kE4m3Max);
                }
                int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
                lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true), hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
                if (place[p].count) store_codes(a.codes + row * a.cols, place[p], static_cast<uint32_t>(lo), static_cast<uint32_t>(hi));
            }
        }
    }
}

template <typename T, int THREADS, int PIECES>
__global__ __launch_bounds__(kBlockOf<THREADS>) void rms_rows_backward(const RmsArgs a) {
    constexpr int kGroups = kBlockOf<THREADS> / THREADS;
    __shared__ float lds[4 * (THREADS / 64)];
    int turn = 0;
    const int t = threadIdx.x % THREADS;
    const int64_t group = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / THREADS;
    Place place[PIECES];
    Raw<T> w[PIECES];
    float dw[PIECES][kPiece];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        place[p] = place_of(p * THREADS + t, a.cols);
        if (a.weight) w[p] = load_place(static_cast<const T*>(a.weight), place[p]);
#pragma unroll
        for (int e = 0; e < kPiece; ++e) dw[p][e] = 0.f;
    }
    const bool odd = a.cols % kPiece != 0;
    const bool more = a.dh && a.y;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
    // The next row is asked for ahead where the registers have room for it.
    constexpr bool kAhead = THREADS < 1024 || PIECES * sizeof(T) <= 4;
    Raw<T> next_h[PIECES], next_dy[PIECES], next_dh[PIECES];
    auto ask = [&](int64_t row) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            next_h[p] = load_place(static_cast<const T*>(a.x) + row * a.ld_x, place[p]);
            next_dy[p] = load_place(static_cast<const T*>(a.dy) + row * a.ld_dy, place[p]);
            if (more) next_dh[p] = load_place(static_cast<const T*>(a.dh) + row * a.ld_dh, place[p]);
        }
    };
    if (kAhead && group < a.rows) ask(group);
    for (int64_t row = group; row < a.rows; row += step) {
        Raw<T> h[PIECES], dy[PIECES], dh[PIECES];
        if (!kAhead) ask(row);
#pragma unroll
        for (int p = 0; p < PIECES; ++p) h[p] = next_h[p], dy[p] = next_dy[p], dh[p] = next_dh[p];
        if (kAhead && row + step < a.rows) ask(row + step);
        // g of piece p and its rows
        auto both = [&](int p, float (&g)[kPiece], float (&v)[kPiece]) {
            unpack(dy[p], g), unpack(h[p], v);
            if (a.weight) {
                float u[kPiece];
                unpack(w[p], u);
#pragma unroll
                for (int e = 0; e < kPiece; ++e) g[e] *= u[e];
            }
        };
        float sum[2] = {0.f, 0.f};   // of h^2, of g h
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            float g[kPiece], v[kPiece];
            both(p, g, v);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                const bool counts = !odd || e >= place[p].skip;
                sum[0] += counts ? v[e] * v[e] : 0.f;
                sum[1] += counts ? g[e] * v[e] : 0.f;
            }
        }
        if (!a.part_sums) over_group<THREADS, 2, false>(sum, lds, turn);
        if (a.own) {
            if (t == 0) a.own[row] = sum[1];
            continue;
        }
        if (a.part_squares) sum[0] = over_parts(a.part_squares, a.nparts, a.rows, row);
        if (a.part_sums) sum[1] = over_parts(a.part_sums, a.nparts, a.rows, row);
        const float rstd = 1.f / sqrtf(sum[0] * a.inv_cols + a.eps), mean = sum[1] * rstd * a.inv_cols;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            float g[kPiece], v[kPiece], own[kPiece];
            both(p, g, v);
            unpack(dy[p], own);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                const float xhat = v[e] * rstd;
                dw[p][e] += own[e] * xhat;
                g[e] = rstd * (g[e] - xhat * mean);
            }
            if (a.y) {
                if (more) {
                    unpack(dh[p], v);
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) g[e] += v[e];
                }
                if (place[p].count) store_place(static_cast<T*>(a.y) + row * a.cols, place[p], pack(g, static_cast<T*>(nullptr)));
            }
        }
    }
    if (!a.partial) return;
    float* const to = a.partial + group * a.cols;
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
        for (int e = 0; e < kPiece; ++e)
            if (e >= place[p].skip && e < place[p].count) to[place[p].at + e] = dw[p][e];
}

// dw[c] = sum of the groups' partial sums, in one order: 32 columns by 32 of them at a time.
template <typename T>
__global__ __launch_bounds__(1024) void rms_weight_grad(const float* __restrict__ partial, int64_t groups, int cols, T* dw) {
    __shared__ float sums[32][33];
    const int col = threadIdx.x & 31, lane = threadIdx.x >> 5, c = static_cast<int>(blockIdx.x) * 32 + col;
    float t = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (int64_t g = lane; g < groups; g += 32) t += partial[g * cols + c];
    }
    sums[lane][col] = t;
    __syncthreads();
    if (lane == 0 && c < cols) {
        float all = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) all += sums[k][col];
        store1(dw + c, all);
    }
}

constexpr int kGradBlocks = 512;   // of the adjoint where the weight's gradient is wanted: two for each CU

int groups_of(int64_t cols) { return cols <= 1024 ? 4 : 1; }   // rows that a workgroup has side by side

// Calls fn(threads of a row, pieces of a thread) as constants.
template <typename Fn>
int with_shape(int64_t cols, Fn&& fn) {
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<int, 2> Two;
    if (cols <= 512) return fn(std::integral_constant<int, 64>{}, One{});
    if (cols <= 1024) return fn(std::integral_constant<int, 64>{}, Two{});
    if (cols <= 2048) return fn(std::integral_constant<int, 256>{}, One{});
    if (cols <= 4096) return fn(std::integral_constant<int, 512>{}, One{});
    if (cols <= 8192) return fn(std::integral_constant<int, 1024>{}, One{});
    return fn(std::integral_constant<int, 1024>{}, Two{});
}

template <typename Fn>
int with_element(int dtype, Fn&& fn) {
    int rc = 0;
    with_ln_element(dtype, [&](auto* p) { rc = fn(p); });
    return rc;
}

int check_rows(const char* who, int dtype, int64_t rows, int64_t cols) {
    if (dtype != DDL_DT_F32 && dtype != DDL_DT_BF16 && dtype != DDL_DT_F16) return fail(DDL_E_ARG, "%s: dtype %d", who, dtype);
    if (rows < 0 || cols < 1) return fail(DDL_E_ARG, "%s: %lld rows of %lld columns", who, static_cast<long long>(rows), static_cast<long long>(cols));
    if (cols > kMaxCols) return fail(DDL_E_UNSUPP, "%s: rows of %lld columns (at most %d)", who, static_cast<long long>(cols), kMaxCols);
    return 0;
}

int check_parts(const char* who, int64_t cols, const float* own, const float* parts, int nparts, int64_t total_cols) {
    if (own && parts) return fail(DDL_E_ARG, "%s: this worker's sums are asked for, and all workers' given", who);
    if (parts && nparts < 1) return fail(DDL_E_ARG, "%s: sums of %d workers", who, nparts);
    if (parts && total_cols < cols) return fail(DDL_E_ARG, "%s: %lld of %lld columns", who, static_cast<long long>(cols), static_cast<long long>(total_cols));
    return 0;
}

template <typename T, bool EIGHT, bool NORM>
int launch_rows(const RmsArgs& a, int64_t grid, hipStream_t s) {
    return with_shape(a.cols, [&](auto threads, auto pieces) {
        hipLaunchKernelGGL((rms_rows<T, decltype(threads)::value, decltype(pieces)::value, EIGHT, NORM>), dim3(static_cast<uint32_t>(grid)),
                           dim3(kBlockOf<decltype(threads)::value>), 0, s, a);
        return check_launch(NORM ? "ddl_rms_norm" : "ddl_quantize_rows");
    });
}

// Every workgroup has some rows one after the other (its weights are read once) where there are enough for eight of 256 threads a CU.
int64_t grid_of(int64_t rows, int64_t cols) {
    int dev;
    const int64_t per = groups_of(cols), blocks = (rows + per - 1) / per;
    const int64_t resident = cols <= 2048 ? 8 : cols <= 4096 ? 4 : 2, most = compute_units(dev) * resident;
    return blocks < most ? blocks : most;
}

}  // namespace
}  // namespace ddl

extern "C" {

int ddl_rms_norm(const void* x, const void* residual, const void* weight, int dtype, int64_t rows, int64_t cols, int64_t ld_x, int64_t ld_residual, float eps,
                 void* sum, void* y, void* codes, float* scales, float* own_squares, const float* part_squares, int nparts, int64_t total_cols, void* stream) {
    using namespace ddl;
    if (int rc = check_rows("ddl_rms_norm", dtype, rows, cols)) return rc;
    if (int rc = check_parts("ddl_rms_norm", cols, own_squares, part_squares, nparts, total_cols)) return rc;
    if (!(eps >= 0.f)) return fail(DDL_E_ARG, "ddl_rms_norm: eps %g", static_cast<double>(eps));
    if (codes && (y || !scales || own_squares || part_squares)) return fail(DDL_E_ARG, "ddl_rms_norm: codes come with scales, of whole rows, instead of y");
    if (rows == 0) return 0;
    if (!x || (residual && !sum) || (!codes && !own_squares && !y)) return fail(DDL_E_ARG, "ddl_rms_norm: null pointer");
    if ((rows > 1 && ld_x < cols) || (residual && rows > 1 && ld_residual < cols)) return fail(DDL_E_ARG, "ddl_rms_norm: pitch below %lld columns", static_cast<long long>(cols));
    RmsArgs a{};
    a.x = x, a.residual = residual, a.weight = weight, a.h = sum, a.y = y, a.codes = static_cast<uint8_t*>(codes), a.scales = scales, a.own = own_squares;
    a.part_squares = part_squares, a.nparts = nparts, a.rows = rows, a.cols = static_cast<int>(cols), a.ld_x = ld_x, a.ld_r = ld_residual, a.eps = eps;
    a.inv_cols = 1.f / static_cast<float>(part_squares ? total_cols : cols);
    const int64_t grid = grid_of(rows, cols);
    return with_element(dtype, [&](auto* e) {
        typedef std::remove_pointer_t<decltype(e)> T;
        const hipStream_t s = static_cast<hipStream_t>(stream);
        return codes ? launch_rows<T, true, true>(a, grid, s) : launch_rows<T, false, true>(a, grid, s);
    });
}

int ddl_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld_x, void* codes, float* scales, void* stream) {
    using namespace ddl;
    if (int rc = check_rows("ddl_quantize_rows", dtype, rows, cols)) return rc;
    if (rows == 0) return 0;
    if (!x || !codes || !scales) return fail(DDL_E_ARG, "ddl_quantize_rows: null pointer");
    if (rows > 1 && ld_x < cols) return fail(DDL_E_ARG, "ddl_quantize_rows: pitch below %lld columns", static_cast<long long>(cols));
    RmsArgs a{};
    a.x = x, a.codes = static_cast<uint8_t*>(codes), a.scales = scales, a.rows = rows, a.cols = static_cast<int>(cols), a.ld_x = ld_x;
    const int64_t grid = grid_of(rows, cols);
    return with_element(dtype, [&](auto* e) {
        return launch_rows<std::remove_pointer_t<decltype(e)>, true, false>(a, grid, static_cast<hipStream_t>(stream));
    });
}

int64_t ddl_rms_norm_backward_workspace(int64_t rows, int64_t cols) {
    if (rows < 1 || cols < 1 || cols > ddl::kMaxCols) return 0;
    const int64_t per = ddl::groups_of(cols), blocks = (rows + per - 1) / per;
    return (blocks < ddl::kGradBlocks ? blocks : ddl::kGradBlocks) * per * cols;
}

int ddl_rms_norm_backward(const void* dy, const void* h, const void* dh, const void* weight, int dtype, int64_t rows, int64_t cols, int64_t ld_dy, int64_t ld_h,
                          int64_t ld_dh, float eps, void* dx, void* dweight, float* workspace, int64_t workspace_elems, float* own_sums,
                          const float* part_squares, const float* part_sums, int nparts, int64_t total_cols, void* stream) {
    using namespace ddl;
    if (int rc = check_rows("ddl_rms_norm_backward", dtype, rows, cols)) return rc;
    if (int rc = check_parts("ddl_rms_norm_backward", cols, own_sums, part_sums, nparts, total_cols)) return rc;
    if ((part_sums != nullptr) != (part_squares != nullptr)) return fail(DDL_E_ARG, "ddl_rms_norm_backward: sums of all workers come with their squares");
    if (!(eps >= 0.f)) return fail(DDL_E_ARG, "ddl_rms_norm_backward: eps %g", static_cast<double>(eps));
    if (own_sums && (dx || dweight)) return fail(DDL_E_ARG, "ddl_rms_norm_backward: this worker's sums, or gradients");
    const int64_t need = ddl_rms_norm_backward_workspace(rows, cols);
    if (dweight && need && (!workspace || workspace_elems < need))
        return fail(DDL_E_ARG, "ddl_rms_norm_backward: workspace of %lld floats, %lld are needed", static_cast<long long>(workspace ? workspace_elems : 0),
                    static_cast<long long>(need));
    if (!dx && !dweight && !own_sums) return 0;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t groups = rows ? need / cols : 0;
    if (rows) {
        if (!dy || !h) return fail(DDL_E_ARG, "ddl_rms_norm_backward: null pointer");
        if (rows > 1 && (ld_dy < cols || ld_h < cols || (dh && ld_dh < cols))) return fail(DDL_E_ARG, "ddl_rms_norm_backward: pitch below %lld columns", static_cast<long long>(cols));
        RmsArgs a{};
        a.x = h, a.dy = dy, a.dh = dh, a.weight = weight, a.y = dx, a.own = own_sums, a.part_squares = part_squares, a.part_sums = part_sums, a.nparts = nparts;
        a.partial = dweight ? workspace : nullptr;
        a.rows = rows, a.cols = static_cast<int>(cols), a.ld_x = ld_h, a.ld_dy = ld_dy, a.ld_dh = ld_dh, a.eps = eps;
        a.inv_cols = 1.f / static_cast<float>(part_sums ? total_cols : cols);
        const int rc = with_element(dtype, [&](auto* e) {
            return with_shape(cols, [&](auto threads, auto pieces) {
                hipLaunchKernelGGL((rms_rows_backward<std::remove_pointer_t<decltype(e)>, decltype(threads)::value, decltype(pieces)::value>),
                                   dim3(static_cast<uint32_t>(groups / groups_of(cols))), dim3(kBlockOf<decltype(threads)::value>), 0, s, a);
                return check_launch("ddl_rms_norm_backward");
            });
        });
        if (rc) return rc;
    }
    if (!dweight) return 0;
    return with_element(dtype, [&](auto* e) {
        typedef std::remove_pointer_t<decltype(e)> T;
        hipLaunchKernelGGL((rms_weight_grad<T>), dim3(static_cast<uint32_t>((cols + 31) / 32)), dim3(1024), 0, s, workspace, groups, static_cast<int>(cols),
                           static_cast<T*>(dweight));
        return check_launch("ddl_rms_norm_backward");
    });
}

}  // extern "C"
