// The gradients of few rows: dx_r = w[e]^T dy_r, w read along its columns.
//
// Bound by reading the weights once.  A workgroup has 16 C columns of an expert's weights, C of them a lane, and each of its wavefronts a part of the reduction.  A lane reads C
// elements of as many rows of w as a vector of 16 bytes has elements, and such a vector of dy; matrix instruction j takes element j of every lane's C, so which column it computes
// is spread over the lanes, and a lane ends up with C of them side by side.  (16-bit elements: pairs of rows are put into one register first.)  The wavefronts' sums meet in LDS, half of the wavefronts at a
// time.  ([8, 4096] bf16 by 4096 20 us by tiles, here 13; three of five experts' [2816, 1024] with a row each 15 and 9; [32 x 1024, 1024] fp32 of five rows each 29 and 24 (5.6 TB/s).)
// Operands of any address and pitch: the last columns are moved back to end with the row, what is written twice is the same.
#include "expert_parts.h"
#include "expert_vectors.h"

namespace ddl {
namespace {

constexpr int kAcrossWaves = 8;

template <typename T, int C>
__global__ __launch_bounds__(64 * kAcrossWaves) void expert_across(const ExpertArgs g) {
    constexpr bool k16 = sizeof(T) == 2;
    constexpr int N = 16 / static_cast<int>(sizeof(T)), kStep = 4 * N;   // rows of w of a lane, and of all four lanes with the same columns, at a time
    __shared__ floatx4 sums[kAcrossWaves / 2][C][64];
    const int e = blockIdx.y;
    int lo, hi;
    rows_of_expert(g, e, lo, hi);
    T* const y = static_cast<T*>(g.y);
    if (e == g.experts) {   // rows of none: those behind the last expert's, and those in front of the first one's
        zero_rows(g, lo, hi - lo, blockIdx.x, gridDim.x);
        zero_rows(g, 0, min(max(g.offsets[0], 0), lo), blockIdx.x, gridDim.x);
        return;
    }
    if (lo == hi) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, part = lane >> 4;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * (16 * C);
    const T* const w = static_cast<const T*>(g.w) + e * g.w_stride + min(c0 + l16 * C, g.n - C);
    const int steps = static_cast<int>((g.k + kStep - 1) / kStep), share = (steps + kAcrossWaves - 1) / kAcrossWaves;
    const int first = min(wave * share, steps), last = min(first + share, steps);
    for (int m0 = lo; m0 < hi; m0 += 16) {
        const int row = min(m0 + l16, hi - 1);
        const T* const dy = static_cast<const T*>(g.a) + row * g.lda;
        floatx4 sum[C];
#pragma unroll
        for (int j = 0; j < C; ++j) sum[j] = floatx4{0.f, 0.f, 0.f, 0.f};
        for (int s = first; s < last; ++s) {
            const int64_t r0 = static_cast<int64_t>(s) * kStep + part * N;
            Vector<T, C> down[N];
            Vector<T, N> across;
            if ((s + 1) * static_cast<int64_t>(kStep) <= g.k) {
#pragma unroll
                for (int u = 0; u < N; ++u) down[u] = load_vector<T, C>(w + (r0 + u) * g.ldw);
                across = load_vector<T, N>(dy + r0);
            } else {   // zeros for rows behind the last one
                T own[N];
#pragma unroll
                for (int u = 0; u < N; ++u) {
                    const int64_t r = min(r0 + u, g.k - 1);
                    down[u] = load_vector<T, C>(w + r * g.ldw);
                    own[u] = dy[r];
                    if (r0 + u >= g.k) down[u] = {}, own[u] = T{};
                }
                __builtin_memcpy(&across, own, 16);
            }
            if constexpr (k16) {
                const bf16x8 b = __builtin_bit_cast(bf16x8, across);
#pragma unroll
                for (int j = 0; j < C; ++j) sum[j] = mfma<std::is_same_v<T, __half>>(column(down, j), b, sum[j]);
            } else {
#pragma unroll
                for (int u = 0; u < N; ++u)
#pragma unroll
                    for (int j = 0; j < C; ++j)
                        sum[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(down[u].word[j]), __uint_as_float(across.word[u]), sum[j], 0, 0, 0);
            }
        }
#pragma unroll
        for (int half = kAcrossWaves / 2; half; half /= 2) {
            __syncthreads();   // the sums before these have been read
            if (wave >= half && wave < 2 * half) {
#pragma unroll
                for (int j = 0; j < C; ++j) sums[wave - half][j][lane] = sum[j];
            }
            __syncthreads();
            if (wave < half) {
#pragma unroll
                for (int j = 0; j < C; ++j) sum[j] += sums[wave][j][lane];
            }
        }
        if (wave || m0 + l16 >= hi) continue;
        // Element q of sum[j]: this lane's row of dy, and element j of what lane 4 part + q has of a row of w.
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t c = c0 + (4 * part + q) * C;
            if (c >= g.n) continue;
            float v[C];
#pragma unroll
            for (int j = 0; j < C; ++j) v[j] = sum[j][q];
            store_vector<C>(y + row * g.ldy + min(c, g.n - C), v);
        }
    }
}

template <typename T>
void launch_across(const ExpertArgs& g, bool narrow, hipStream_t s) {
    constexpr int N = 16 / static_cast<int>(sizeof(T));
    const int columns = 16 * (narrow ? N / 2 : N);
    const dim3 grid(static_cast<uint32_t>((g.n + columns - 1) / columns), static_cast<uint32_t>(g.experts + 1)), threads(64 * kAcrossWaves);
    if (narrow) hipLaunchKernelGGL((expert_across<T, N / 2>), grid, threads, 0, s, g);
    else hipLaunchKernelGGL((expert_across<T, N>), grid, threads, 0, s, g);
}

}  // namespace

int run_expert_across(const char* who, const ExpertArgs& g, hipStream_t s) {
    // Half a vector a lane where whole ones make too few workgroups: one row of [3584, 8192] bf16 15 -> 12 us, fp32 30 -> 23; with 146 of them, [4480, 4640] fp32 to two experts, 36 and 43.
    const int64_t columns = g.out_dtype == DDL_DT_F32 ? 64 : 128, used = g.rows < g.experts ? g.rows : g.experts;
    const bool narrow = (g.n + columns - 1) / columns * used < 140;
    if (g.out_dtype == DDL_DT_F32) launch_across<float>(g, narrow, s);
    else if (g.out_dtype == DDL_DT_BF16) launch_across<bf16_t>(g, narrow, s);
    else launch_across<__half>(g, narrow, s);
    return check_launch(who);
}

}  // namespace ddl
