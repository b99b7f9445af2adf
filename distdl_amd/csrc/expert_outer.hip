// The gradients of the experts' weights from few rows: dw[e] = sum over the expert's rows of dy_r x_r^T.
//
// Bound by writing dw once.  A wavefront has a tile of 64 rows by 16 vectors of 16 bytes of a matrix, its sums in registers, and takes both operands from memory as they lie: a lane
// reads, of some rows, four elements of dy and one vector of x.  Matrix instruction (i, j) takes element i of every lane's four and element j of its vector, so which row
// and column of the tile it computes is spread over the lanes, and a lane ends up with whole vectors of dw.  (16-bit elements: eight rows' pairs are put into one register first.)
// No LDS, no barrier: what a tile of expert_linear16.hip or expert_linear32.hip waits for at its start and end takes longer than writing it.  ([8 x 2048, 2048] bf16 of 2 to 32 rows each 29 us by
// tiles, here 13 to 14 (5 TB/s), of 128 29 and 20; fp32 of 2 to 16 57 and 28, of 32 49 and 41.  With the products on the vector units, bf16 13 for two rows and 37 for 32; quicker for one row
// and matrices of no whole lines, [16 x 3743, 4476] bf16 90 and here 100, fp32 171 and 264, by tiles 409.)
// An expert without rows gets its zeros the same way.  Operands of any address and pitch: the last vector of a row and the last rows of a matrix are moved
// back to end with it, what is written twice is the same.  Every XCD has an eighth of each expert's wavefronts side by side.
#include "expert_parts.h"
#include "expert_vectors.h"

namespace ddl {
namespace {

constexpr int kOuterThreads = 256, kOuterWaves = kOuterThreads / 64, kDown = 4;   // kDown: elements of dy that a lane has of a row

struct Outer {
    ExpertArgs g;
    int strips, groups, blocks, share;   // of an expert's matrix: wavefronts across and down, workgroups, of those an XCD's
};

// STREAM: past the caches.
template <typename T, bool STREAM>
__global__ __launch_bounds__(kOuterThreads, 2) void expert_outer(const Outer a) {
    constexpr bool k16 = sizeof(T) == 2;
    constexpr int N = 16 / static_cast<int>(sizeof(T));               // elements of x that a lane has of a row
    constexpr int kOwn = k16 ? 8 : 4, kRows = 4 * kOwn;               // rows of a lane, and of all four lanes with the same columns, at a time
    const ExpertArgs& g = a.g;
    const int xcd = blockIdx.x % kXcds, nth = blockIdx.x / kXcds, e = nth / a.share;
    const int block = (xcd + e) % kXcds * a.share + nth % a.share;   // few workgroups of an expert: another XCD's for the next one
    const int lane = threadIdx.x & 63, l16 = lane & 15, part = lane >> 4, wave = block * kOuterWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = wave / a.strips;
    if (block >= a.blocks || group >= a.groups) return;
    int lo, hi;
    rows_of_expert(g, e, lo, hi);
    if (hi - lo > g.few) return;
    const int64_t k0 = static_cast<int64_t>(wave - group * a.strips) * (16 * N) + l16 * N, n0 = static_cast<int64_t>(group) * (16 * kDown);   // k0: of this lane
    const int64_t at_k = min(k0, g.k - N), at_n = min(n0 + l16 * kDown, g.n - kDown);
    floatx4 sum[kDown][N];
#pragma unroll
    for (int i = 0; i < kDown; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) sum[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    for (int r0 = lo; r0 < hi; r0 += kRows) {
        Vector<T, N> x[kOwn];
        Vector<T, kDown> dy[kOwn];
#pragma unroll
        for (int u = 0; u < kOwn; ++u) {
            const int64_t row = min(r0 + (k16 ? part * kOwn + u : u * 4 + part), hi - 1);
            x[u] = load_vector<T, N>(static_cast<const T*>(g.w) + row * g.ldw + at_k);
            dy[u] = load_vector<T, kDown>(static_cast<const T*>(g.a) + row * g.lda + at_n);
        }
        if (r0 + kRows > hi) {   // zeros for rows behind the expert's
#pragma unroll
            for (int u = 0; u < kOwn; ++u) {
                if (r0 + (k16 ? part * kOwn + u : u * 4 + part) >= hi) x[u] = {}, dy[u] = {};
            }
        }
        if constexpr (k16) {
            bf16x8 down[kDown];
#pragma unroll
            for (int i = 0; i < kDown; ++i) down[i] = column(dy, i);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const bf16x8 across = column(x, j);
#pragma unroll
                for (int i = 0; i < kDown; ++i) sum[i][j] = mfma<std::is_same_v<T, __half>>(down[i], across, sum[i][j]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < kOwn; ++u)
#pragma unroll
                for (int i = 0; i < kDown; ++i)
#pragma unroll
                    for (int j = 0; j < N; ++j)
                        sum[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(dy[u].word[i]), __uint_as_float(x[u].word[j]), sum[i][j], 0, 0, 0);
        }
    }
    // Element q of sum[i][j]: what lane 4 part + q has as element i of dy, and this one as element j of x.
    T* const y = static_cast<T*>(g.y) + e * g.n * g.k + at_k;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int64_t n = n0 + (4 * part + q) * kDown, from = min(n, g.n - kDown);
        if (n >= g.n || k0 >= g.k) continue;
#pragma unroll
        for (int i = 0; i < kDown; ++i) {
            float v[N];
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = sum[i][j][q];
            store_vector<N, STREAM>(y + (from + i) * g.k, v);
        }
    }
}

}  // namespace

int run_expert_outer(const char* who, const ExpertArgs& g, hipStream_t s) {
    const int elements = g.out_dtype == DDL_DT_F32 ? 4 : 8;
    Outer a{g};
    a.strips = static_cast<int>((g.k + 16 * elements - 1) / (16 * elements)), a.groups = static_cast<int>((g.n + 16 * kDown - 1) / (16 * kDown));
    a.blocks = (a.strips * a.groups + kOuterWaves - 1) / kOuterWaves, a.share = (a.blocks + kXcds - 1) / kXcds;
    const int64_t blocks = static_cast<int64_t>(a.share) * kXcds * g.experts;
    if (blocks * kOuterThreads > 0xFFFFFFFFll) return fail(DDL_E_UNSUPP, "%s: %lld workgroups", who, static_cast<long long>(blocks));
    // Rows of whole lines need no cache to put them together, and more rows of x and dy stay there: [8 x 3584, 8192] bf16 of 64 rows each 121 -> 81 us; of no whole lines [16 x 3743, 4476]
    // of one row 99 -> 186, of 24 118 -> 194, of 100 as much, of 256 335 -> 251.
    const bool stream = (g.k * (16 / elements) % 128 == 0 && aligned_to(g.y, 128)) || g.rows >= 100ll * g.experts;
    const dim3 grid(static_cast<uint32_t>(blocks)), threads(kOuterThreads);
    auto launch = [&](auto* element) {
        typedef std::remove_pointer_t<decltype(element)> T;
        if (stream) hipLaunchKernelGGL((expert_outer<T, true>), grid, threads, 0, s, a);
        else hipLaunchKernelGGL((expert_outer<T, false>), grid, threads, 0, s, a);
    };
    with_ln_element(g.out_dtype, launch);
    return check_launch(who);
}

}  // namespace ddl
