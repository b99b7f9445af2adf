// DistributedLinear shard GEMM: y[M,N] = x[M,K] . w[N,K]^T + bias[N], bf16 (or
// fp16) operands, fp32 accumulation on the matrix cores, result in the operands'
// type (reference: nn/linear.py:103, nn/linear_ag.py:486 --
// torch.nn.functional.linear).
//
// Both operands are K-contiguous, so a 16-byte load anywhere gives eight
// consecutive k of one row: exactly one lane's share of an MFMA operand.  The
// product is formed transposed (w rows feed the A port, x rows the B port) so
// that each lane ends up with four consecutive n of one output row and can
// store them as one 8-byte word.
//
//   workgroup  512 threads = 8 wavefronts (2 along m x 4 along n), tile
//              256(m) x 256(n); two wavefronts share a SIMD so that one can
//              issue MFMAs while the other waits
//   wavefront  128(m) x 64(n) = 8 x 4 tiles of v_mfma_f32_16x16x32_bf16, 128 fp32
//              accumulators per lane.  On random operands the chip is limited
//              by power, and this instruction delivers about 14 % more flop/s
//              under that limit than the 32x32x16 one (it moves half as many
//              accumulator bytes per flop)
//   LDS        ring of five operand tiles (W0 X0 W1 X1 W2 | X2 W3 ...), each
//              256 rows x 64 k = 32 KiB, 160 KiB in all.  Rows are 128 B; the
//              16-byte chunk index is XOR-ed with ((row >> 1) & 7): the 16
//              lanes served per LDS cycle read 16 consecutive rows, and
//              (row & 1, (row >> 1) & 7) is distinct for each, so they cover all
//              64 banks (an MFMA operand piece is 16 rows x 32 k: lane l reads
//              row l % 16, chunk l / 16 of the k-step)
//   global     tiles go from global memory straight into LDS
//              (buffer_load_dwordx4 ... lds: each wavefront instruction fills
//              1 KiB = 8 rows, the eight lanes of a row fetching one whole
//              128-byte line; half-line requests run at little more than half
//              the rate).  No staging registers, no LDS stores, one 32-bit
//              offset per lane and the k offset in a scalar
//   schedule   per k-tile of 64: two k-steps of 32 MFMAs, one LDS fragment
//              read issued behind every second MFMA (the fragments of the next
//              k-step, crossing into tile t+1 in the second k-step).  W(t+2) is
//              requested during k-step 0 into the slot X(t-1) left, X(t+2)
//              during k-step 1 into the slot of W(t); between the two k-steps
//              each wavefront waits for its own requests of tile t+1 and all
//              its LDS reads, then one barrier: tile t+1 is readable, tile t's
//              slots are free
//   epilogue   bias add and bf16 rounding in registers, then each wavefront
//              transposes its block through LDS so that rows of y are written
//              in 16-byte pieces, whole 128-byte lines per instruction
//   launch     one workgroup per CU is resident, so the tiles run in rounds of
//              one per CU and a last round that is only partly filled costs as
//              much as a full one; when it pays, the columns are split between
//              256-wide tiles (whole rounds) and 192-wide tiles (4 x 2
//              wavefronts of 64 x 96), whose rounds are shorter.  One launch:
//              workgroup b computes wide tile b and then narrow tile b, so the
//              stores of its first tile drain while it computes the second and
//              the workgroups of an XCD stay in step.  (Both kinds as separate
//              workgroups of one grid, so that a CU starts on a narrow tile the
//              moment its wide one is stored, measured 2 % slower: the
//              workgroups of an XCD then drift apart in k and share fewer
//              operand lines in its L2; two launches measured 1 % slower.)
//              Workgroup ids are regrouped so that the 32 workgroups resident on
//              one XCD cover a compact patch of the tile grid and share their
//              operand panels in that XCD's L2
#include "gemm16_large.h"
#include "gemm16_small.h"
#include "gemm32_small.h"
#include <type_traits>

namespace ddl {
namespace {

constexpr int kThreads = 512;

typedef PartsOf<uint16_t> Parts;

// Workgroup b computes wide tile b and then narrow tile b (where they exist):
// the stores of the first tile drain while the second is computed, and there
// is no kernel boundary between the two rounds.
template <bool F16, bool XT, bool WT>
__global__ __launch_bounds__(kThreads) void gemm16_tiles(const Parts parts) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int b = static_cast<int>(blockIdx.x);
    const bool has_wide = b < parts.wide.tiles_m * parts.wide.tiles_n;
    if (has_wide) gemm_tile<F16, XT, WT, 2, 4, 8, 4>(parts.wide, b, lds);
    if (b < parts.narrow.tiles_m * parts.narrow.tiles_n) {
        if (has_wide) __syncthreads();   // every wavefront has read its part of the first tile out of LDS
        gemm_tile<F16, XT, WT, 4, 2, 4, 6>(parts.narrow, b, lds);
    }
}

// Tiles of 128 x 256 (2 x 4 wavefronts of 64 x 64), for products too small to
// give every CU a 256 x 256 tile: twice as many workgroups, each half the work.
template <bool F16, bool XT, bool WT>
__global__ __launch_bounds__(kThreads) void gemm16_low_tiles(const Part part) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    gemm_tile<F16, XT, WT, 2, 4, 4, 4>(part, blockIdx.x, lds);
}

typedef void (*LowKernel)(const Part);
const LowKernel kLowKernels[8] = {
    gemm16_low_tiles<false, false, false>, gemm16_low_tiles<false, false, true>, gemm16_low_tiles<false, true, false>, gemm16_low_tiles<false, true, true>,
    gemm16_low_tiles<true, false, false>,  gemm16_low_tiles<true, false, true>,  gemm16_low_tiles<true, true, false>,  gemm16_low_tiles<true, true, true>,
};

typedef void (*Kernel)(const Parts);
// index: 4 fp16 + 2 (x transposed) + (w transposed)
const Kernel kKernels[8] = {
    gemm16_tiles<false, false, false>, gemm16_tiles<false, false, true>, gemm16_tiles<false, true, false>, gemm16_tiles<false, true, true>,
    gemm16_tiles<true, false, false>,  gemm16_tiles<true, false, true>,  gemm16_tiles<true, true, false>,  gemm16_tiles<true, true, true>,
};

std::atomic<bool> lds_reserved[kMaxDevices][16];   // the dynamic LDS size of kKernels[i] (8 + i: kLowKernels[i]) has been raised on that device (first use, any thread)

// What the kernel asks of an operand with `rows` rows; 0 or an error code.
int check_operand(const char* who, const char* name, const Operand16& o, int64_t rows, int64_t K) {
    if (o.row_stride != 1 && o.k_stride != 1)
        return fail(DDL_E_UNSUPP, "%s: operand %s has no unit stride (row stride %lld, k stride %lld)", who, name, (long long)o.row_stride,
                    (long long)o.k_stride);
    const int64_t ld = o.ld();
    if (!aligned_to(o.p, 16) || ld % 8 != 0) return fail(DDL_E_ALIGN, "%s: operand %s must be 16-byte aligned with a pitch that is a multiple of 8", who, name);
    if (ld > 0x3FFFFF) return fail(DDL_E_UNSUPP, "%s: pitch of %s above 2^22 elements", who, name);   // 32-bit byte offsets inside a tile
    if (o.transposed()) {
        if (ld < rows) return fail(DDL_E_ARG, "%s: pitch %lld of %s below its %lld rows", who, (long long)ld, name, (long long)rows);
        if (rows % 8 != 0) return fail(DDL_E_ALIGN, "%s: %s is read along its rows, whose number must be a multiple of 8", who, name);
        if ((K + BK) * ld > 0x3FFFFFFF) return fail(DDL_E_UNSUPP, "%s: %s spans more than 2^31 bytes along k", who, name);
    } else {
        if (ld < K) return fail(DDL_E_ARG, "%s: pitch %lld of %s below K=%lld", who, (long long)ld, name, (long long)K);
        if (K % 8 != 0) return fail(DDL_E_ALIGN, "%s: %s is read along k, so K must be a multiple of 8", who, name);
        if (K > 0x3FFFFFFF) return fail(DDL_E_UNSUPP, "%s: K above 2^30", who);
    }
    return 0;
}

// Estimated duration of the large tiles' schedule in microseconds (fits of a sweep, as in linear_small.hip): per k-tile
// 0.47 (tiles of 128 x 256) or 0.95 us while few CUs work, up to 0.74 or 1.43 when all do and the chip runs into its
// power limit.  `cost` is the schedule's length in tile rows or columns (see wide_tile_columns), `tiles` the workgroups.
double large_us(bool low, int64_t cost, int64_t tiles, int64_t K, int cus) {
    const double rounds = cost / (low ? 128.0 : 256.0), fill = tiles < cus ? static_cast<double>(tiles) / cus : 1.0;
    return 6.5 + static_cast<double>((K + BK - 1) / BK) * rounds * (low ? 0.47 + 0.27 * fill * fill : 0.95 + 0.48 * fill * fill);
}

// Are the pitch and the lengths of an operand multiples of 16 bytes, as the aligned kernels ask?
bool pitches_ok(const Operand16& o, int64_t rows, int64_t K) { return o.ld() % 8 == 0 && (o.transposed() ? rows : K) % 8 == 0; }

struct Plan16 {
    Small16 small;            // kind other than kNone: linear_small.hip computes the product
    int64_t low_tiles = 0;    // otherwise this many tiles of 128 x 256, if not 0
    double large = 0;         // estimate for the large tiles, microseconds
    int64_t wide_cols = 0;    // otherwise 256 x 256 tiles for the first columns, 256 x 192 for the rest
};

Plan16 plan16(bool at, bool bt, int64_t M, int64_t N, int64_t K, int cus, int64_t workspace) {
    Plan16 plan;
    const int64_t tiles_m = (M + 255) / 256, cols = (N + 255) / 256;
    int64_t cost = 0;
    plan.wide_cols = wide_tile_columns(tiles_m, N, cus, &cost);
    // Tiles of half the height: twice the workgroups.  Taken when that shortens
    // the schedule by more than the 10 % a smaller tile loses in efficiency.
    const int64_t low_tiles = ((M + 127) / 128) * cols;
    const int64_t low_cost = (low_tiles + cus - 1) / cus * 128;
    const bool low = low_cost * 11 < cost * 10;
    if (low) plan.low_tiles = low_tiles;
    // Products that leave most of the chip idle either way.
    plan.large = large_us(low, low ? low_cost : cost, low ? low_tiles : tiles_m * cols, K, cus);
    plan.small = plan_small16(at, bt, M, N, K, cus, workspace, plan.large);
    return plan;
}

// Can an operand with `rows` rows be read from wherever it lies (linear_any.hip)?
bool readable_anywhere(const Operand16& o, int64_t rows, int64_t K) {
    if (o.row_stride != 1 && o.k_stride != 1) return false;
    return o.transposed() ? rows >= 8 && o.ld() >= rows : rows == 1 || o.ld() >= K;
}

// How linear_any.hip computes the product of such operands, if it does.  Whether it does is a matter of sizes and strides (the
// caller copies the operands otherwise, and has no such way out later); the workspace only decides how.  `leeway`: by how many
// microseconds copying them may be the faster way.
Small16 plan_anywhere(const Operand16& a, const Operand16& b, int64_t M, int64_t N, int64_t K, int cus, int64_t workspace, double leeway) {
    if (!readable_anywhere(a, M, K) || !readable_anywhere(b, N, K)) return Small16{};
    const bool at = a.transposed(), bt = b.transposed();
    const double large = plan16(at, bt, M, N, K, cus, 0).large;
    const Small16 best = plan_any16(at, bt, M, N, K, cus, INT64_MAX, large + leeway);
    return best.kind == Small16::kNone || best.workspace <= workspace ? best : plan_any16(at, bt, M, N, K, cus, workspace, 1e30);
}

// The product itself is computed for callers that do not have the copies, too, up to here.
constexpr double kLeeway = 18;

// Estimate for one product, as it is computed when it is alone; negative where it is not (the caller copies the operands).
double alone_us(const Operand16& a, const Operand16& b, bool aligned, int64_t M, int64_t N, int64_t K, int cus) {
    if (aligned && pitches_ok(a, M, K) && pitches_ok(b, N, K)) {
        const Plan16 plan = plan16(a.transposed(), b.transposed(), M, N, K, cus, INT64_MAX);
        return plan.small.kind != Small16::kNone ? plan.small.us : plan.large;
    }
    const Small16 any = plan_anywhere(a, b, M, N, K, cus, INT64_MAX, kLeeway);
    return any.kind == Small16::kNone ? -1 : any.kind == Small16::kThin ? 8 : any.us;
}

// y[M, N] = a[M, K] . b[N, K]^T + bias in 16-bit elements.  `workspace` (may be null) for the sums of a split reduction;
// `anywhere`: operands that are not aligned to 16 bytes are taken where linear_any.hip reads them.
int gemm16(const char* who, bool f16, Operand16 a, Operand16 b, const uint16_t* bias, uint16_t* y, int64_t ldy, int64_t M, int64_t N, int64_t K,
           float* workspace, int64_t workspace_elems, bool anywhere, void* stream) {
    if (M < 0 || N < 0 || K < 0 || ldy < N)
        return fail(DDL_E_ARG, "%s: M=%lld N=%lld K=%lld ldy=%lld", who, (long long)M, (long long)N, (long long)K, (long long)ldy);
    if (M == 0 || N == 0) return 0;
    if (!a.p || !b.p || !y) return fail(DDL_E_ARG, "%s: null pointer", who);
    if (K == 0) return fail(DDL_E_UNSUPP, "%s: K = 0", who);
    if (anywhere && aligned_to(a.p, 2) && aligned_to(b.p, 2) && aligned_to(y, 2) && aligned_to(bias, 2) &&
        !(aligned_to(a.p, 16) && aligned_to(b.p, 16) && pitches_ok(a, M, K) && pitches_ok(b, N, K))) {
        int dev = 0;
        const int cus = compute_units(dev);
        const Small16 any = plan_anywhere(a, b, M, N, K, cus, workspace ? workspace_elems : 0, kLeeway);
        if (any.kind != Small16::kNone) {
            Part16 p{};
            p.x = a.p, p.w = b.p, p.bias = bias, p.y = y, p.M = M, p.N = N, p.K = K, p.ldx = a.ld(), p.ldw = b.ld(), p.ldy = ldy;
            return run_any16(any, f16, a.transposed(), b.transposed(), p, workspace, static_cast<hipStream_t>(stream));
        }
    }
    if (int rc = check_operand(who, "a", a, M, K)) return rc;
    if (int rc = check_operand(who, "b", b, N, K)) return rc;
    if (!aligned_to(y, 2) || (bias && !aligned_to(bias, 2))) return fail(DDL_E_ALIGN, "%s: y / bias misaligned", who);
    const bool at = a.transposed(), bt = b.transposed();

    int dev = 0;
    const int cus = compute_units(dev);
    const int64_t tiles_m = (M + 255) / 256, cols = (N + 255) / 256;
    if (tiles_m > 0x7FFFFFll || cols > 0x7FFFFFll || tiles_m * (cols + 1) > 0x7FFFFFFFll)
        return fail(DDL_E_UNSUPP, "%s: too many output tiles", who);
    const Plan16 plan = plan16(at, bt, M, N, K, cus, workspace_elems);
    const int64_t wide_cols = plan.wide_cols;
    // Columns [n_begin, n_begin + n_count) of the output with tiles of bm x bn.
    auto part = [&](int bm, int bn, int64_t n_begin, int64_t n_count) {
        Part p{};
        p.x = a.p, p.w = b.p + n_begin * b.row_stride, p.bias = bias ? bias + n_begin : nullptr, p.y = y + n_begin;
        p.M = M, p.N = n_count, p.K = K, p.ldx = a.ld(), p.ldw = b.ld(), p.ldy = ldy;
        p.tiles_m = static_cast<int>((M + bm - 1) / bm), p.tiles_n = static_cast<int>((n_count + bn - 1) / bn);
        return p;
    };
    const int k = (f16 ? 4 : 0) + (at ? 2 : 0) + (bt ? 1 : 0);
    auto reserve_lds = [&](int slot, const void* kernel) -> int {
        if (!lds_reserved[dev][slot].load(std::memory_order_acquire)) {   // the attribute sticks to the function on this device
            const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes);
            if (e != hipSuccess) return fail(static_cast<int>(e), "%s: cannot reserve %d bytes of LDS: %s", who, kLdsBytes, hipGetErrorString(e));
            lds_reserved[dev][slot].store(true, std::memory_order_release);
        }
        return 0;
    };
    if (plan.small.kind != Small16::kNone)
        return run_small16(who, plan.small, f16, at, bt, part(64, 64, 0, N), workspace, dev, static_cast<hipStream_t>(stream));
    if (plan.low_tiles) {
        if (int rc = reserve_lds(8 + k, reinterpret_cast<const void*>(kLowKernels[k]))) return rc;
        hipLaunchKernelGGL(kLowKernels[k], dim3(static_cast<uint32_t>(plan.low_tiles)), dim3(kThreads), kLdsBytes, static_cast<hipStream_t>(stream),
                           part(128, 256, 0, N));
        return check_launch("gemm16_low_tiles");
    }
    Parts parts{};
    if (wide_cols > 0) parts.wide = part(256, 256, 0, wide_cols);
    if (wide_cols < N) parts.narrow = part(256, 192, wide_cols, N - wide_cols);
    const int n_wide = parts.wide.tiles_m * parts.wide.tiles_n, n_narrow = parts.narrow.tiles_m * parts.narrow.tiles_n;
    if (int rc = reserve_lds(k, reinterpret_cast<const void*>(kKernels[k]))) return rc;
    hipLaunchKernelGGL(kKernels[k], dim3(static_cast<uint32_t>(n_wide > n_narrow ? n_wide : n_narrow)), dim3(kThreads), kLdsBytes,
                       static_cast<hipStream_t>(stream), parts);
    return check_launch("gemm16_tiles");
}

}  // namespace
}  // namespace ddl

namespace ddl {

// How the adjoint of a 16-bit linear shard is computed in one launch, if it is (edge_x 0 otherwise): where the two products
// would each be computed with their operands as they lie.
AdjointPlan16 adjoint16(int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t lddy, bool aligned, bool want_db, int64_t workspace) {
    int dev = 0;
    const int cus = compute_units(dev);
    const Operand16 dy{nullptr, lddy, 1}, dy_t{nullptr, 1, lddy}, w{nullptr, 1, ldw}, x{nullptr, 1, ldx};
    if (M < 2 || N < 2 || K < 2 || !readable_anywhere(dy, M, N) || !readable_anywhere(w, K, N) || !readable_anywhere(dy_t, N, M) || !readable_anywhere(x, K, M))
        return AdjointPlan16{};
    const double dx_us = alone_us(dy, w, aligned, M, K, N, cus), dw_us = alone_us(dy_t, x, aligned, N, K, M, cus);
    if (dx_us < 0 || dw_us < 0) return AdjointPlan16{};
    return plan_adjoint16(M, N, K, aligned, want_db, cus, workspace, dx_us + dw_us);
}

}  // namespace ddl

namespace ddl {
int gemm_f32(const float* a, int64_t a_row_stride, int64_t a_k_stride, const float* b, int64_t b_row_stride, int64_t b_k_stride,
             const float* bias, float* y, int64_t ldy, int64_t M, int64_t N, int64_t K, float* workspace, int64_t workspace_elems,
             void* stream);
Small32 plan32(int64_t a_rs, int64_t a_ks, int64_t b_rs, int64_t b_ks, int64_t M, int64_t N, int64_t K, int cus, int64_t workspace);
}  // namespace ddl

extern "C" int ddl_linear_bf16(const void* x, const void* w, const void* bias, void* y, int64_t M, int64_t N, int64_t K,
                               int64_t ldx, int64_t ldw, int64_t ldy, void* stream) {
    return ddl_linear(x, w, bias, y, DDL_DT_BF16, M, N, K, ldx, ldw, ldy, stream);
}

extern "C" int ddl_linear(const void* x, const void* w, const void* bias, void* y, int dtype, int64_t M, int64_t N, int64_t K,
                          int64_t ldx, int64_t ldw, int64_t ldy, void* stream) {
    using namespace ddl;
    if (dtype != DDL_DT_BF16 && dtype != DDL_DT_F16 && dtype != DDL_DT_F32)
        return fail(DDL_E_UNSUPP, "linear: dtype %d (bf16, f16 and f32 only)", dtype);
    if (ldx < K || ldw < K) return fail(DDL_E_ARG, "linear: ldx=%lld ldw=%lld below K=%lld", (long long)ldx, (long long)ldw, (long long)K);
    // A pitch of 1 would read as "contiguous along the rows" below; it can only belong to a K = 1 operand, which the 16-bit kernel refuses anyway.
    return ddl_gemm(x, ldx, 1, w, ldw, 1, bias, y, dtype, ldy, M, N, K, stream);
}

namespace ddl {
namespace {

int gemm(const void* a, int64_t a_row_stride, int64_t a_k_stride, const void* b, int64_t b_row_stride, int64_t b_k_stride, const void* bias,
         void* y, int dtype, int64_t ldy, int64_t M, int64_t N, int64_t K, float* workspace, int64_t workspace_elems, bool anywhere,
         void* stream) {
    if (workspace && !aligned_to(workspace, 16)) return fail(DDL_E_ALIGN, "gemm: workspace must be 16-byte aligned");
    if (dtype == DDL_DT_F32)
        return gemm_f32(static_cast<const float*>(a), a_row_stride, a_k_stride, static_cast<const float*>(b), b_row_stride, b_k_stride,
                        static_cast<const float*>(bias), static_cast<float*>(y), ldy, M, N, K, workspace, workspace_elems, stream);
    if (dtype != DDL_DT_BF16 && dtype != DDL_DT_F16) return fail(DDL_E_UNSUPP, "gemm: dtype %d (bf16, f16 and f32 only)", dtype);
    const Operand16 oa{static_cast<const uint16_t*>(a), a_row_stride, a_k_stride};
    const Operand16 ob{static_cast<const uint16_t*>(b), b_row_stride, b_k_stride};
    return gemm16("gemm", dtype == DDL_DT_F16, oa, ob, static_cast<const uint16_t*>(bias), static_cast<uint16_t*>(y), ldy, M, N, K, workspace,
                  workspace ? workspace_elems : 0, anywhere, stream);
}

}  // namespace
}  // namespace ddl

extern "C" int ddl_gemm(const void* a, int64_t a_row_stride, int64_t a_k_stride, const void* b, int64_t b_row_stride, int64_t b_k_stride,
                        const void* bias, void* y, int dtype, int64_t ldy, int64_t M, int64_t N, int64_t K, void* stream) {
    return ddl::gemm(a, a_row_stride, a_k_stride, b, b_row_stride, b_k_stride, bias, y, dtype, ldy, M, N, K, nullptr, 0, false, stream);
}

extern "C" int ddl_gemm_in_place(int dtype, int aligned, int64_t a_row_stride, int64_t a_k_stride, int64_t b_row_stride, int64_t b_k_stride,
                                 int64_t M, int64_t N, int64_t K) {
    using namespace ddl;
    if (dtype == DDL_DT_F32) return 1;
    if (M <= 0 || N <= 0 || K <= 0 || (dtype != DDL_DT_BF16 && dtype != DDL_DT_F16)) return 0;
    const Operand16 a{nullptr, a_row_stride, a_k_stride}, b{nullptr, b_row_stride, b_k_stride};
    // a null pointer is aligned: what is left to check are the sizes
    if (aligned && pitches_ok(a, M, K) && pitches_ok(b, N, K))
        return check_operand("gemm", "a", a, M, K) == 0 && check_operand("gemm", "b", b, N, K) == 0;
    int dev = 0;
    const int cus = compute_units(dev);
    return plan_anywhere(a, b, M, N, K, cus, INT64_MAX, 0).kind != Small16::kNone;
}

extern "C" int64_t ddl_gemm_workspace_at(int dtype, int aligned, int64_t a_row_stride, int64_t a_k_stride, int64_t b_row_stride,
                                         int64_t b_k_stride, int64_t M, int64_t N, int64_t K) {
    using namespace ddl;
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    int dev = 0;
    const int cus = compute_units(dev);
    if (dtype == DDL_DT_F32) return plan32(a_row_stride, a_k_stride, b_row_stride, b_k_stride, M, N, K, cus, INT64_MAX).workspace;
    if (dtype != DDL_DT_BF16 && dtype != DDL_DT_F16) return 0;
    const Operand16 a{nullptr, a_row_stride, a_k_stride}, b{nullptr, b_row_stride, b_k_stride};
    if (aligned && pitches_ok(a, M, K) && pitches_ok(b, N, K)) return plan16(a.transposed(), b.transposed(), M, N, K, cus, INT64_MAX).small.workspace;
    return plan_anywhere(a, b, M, N, K, cus, INT64_MAX, kLeeway).workspace;
}

extern "C" int64_t ddl_gemm_workspace(int dtype, int64_t a_row_stride, int64_t a_k_stride, int64_t b_row_stride, int64_t b_k_stride,
                                      int64_t M, int64_t N, int64_t K) {
    return ddl_gemm_workspace_at(dtype, 1, a_row_stride, a_k_stride, b_row_stride, b_k_stride, M, N, K);
}

extern "C" int ddl_gemm_ws(const void* a, int64_t a_row_stride, int64_t a_k_stride, const void* b, int64_t b_row_stride, int64_t b_k_stride,
                           const void* bias, void* y, int dtype, int64_t ldy, int64_t M, int64_t N, int64_t K, float* workspace,
                           int64_t workspace_elems, void* stream) {
    return ddl::gemm(a, a_row_stride, a_k_stride, b, b_row_stride, b_k_stride, bias, y, dtype, ldy, M, N, K, workspace, workspace_elems, true,
                     stream);
}
