// The gradients of the experts' weights from few rows: dw[e] = sum over the expert's rows of dy_r x_r^T, an outer product for each.
//
// Bound by writing dw once.  A wavefront has kSide rows of a matrix by 64 vectors of 16 bytes, kept as 32-bit sums in registers; for each row it reads its vectors of x and
// (the same in all lanes) kSide elements of dy, and adds kSide products for each element of x.  No LDS, no barrier: what a tile of expert_linear16.hip or expert_linear32.hip waits
// for at its start and end takes longer than writing it.  ([8 x 2048, 2048] of two rows each: fp32 57 -> 24 us (5.6 TB/s), bf16 29 -> 13; of eight 57 -> 27 and
// 30 -> 19.)  An expert without rows gets its zeros the same way.  Operands of any address and pitch: the last vector of a row and the last rows of a matrix are moved
// back to end with it, what is written twice is the same.  Every XCD has an eighth of each expert's wavefronts side by side.
#include "expert_parts.h"
#include "ln_elements.h"

namespace ddl {
namespace {

constexpr int kSide = 8, kOuterThreads = 256, kOuterWaves = kOuterThreads / 64;

struct Outer {
    ExpertArgs g;
    int strips, groups, blocks, share;   // of an expert's matrix: wavefronts across and down, workgroups, of those an XCD's
};

// N elements as they lie.
template <typename T, int N>
struct Vector {
    uint32_t word[N * sizeof(T) / 4];
};
template <typename T, int N>
__device__ inline Vector<T, N> load_vector(const T* p) {
    struct __attribute__((packed, aligned(sizeof(T)))) Any {
        Vector<T, N> v;
    };
    return reinterpret_cast<const Any*>(p)->v;
}
__device__ inline float element(const uint32_t* w, int i, const float*) { return __uint_as_float(w[i]); }
__device__ inline float element(const uint32_t* w, int i, const bf16_t*) { return __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16); }
__device__ inline float element(const uint32_t* w, int i, const __half*) {
    const __half2 two = __builtin_bit_cast(__half2, w[i / 2]);
    return i % 2 ? __high2float(two) : __low2float(two);
}
__device__ inline u32x4 packed(const float* v, const float*) { return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])}; }
__device__ inline u32x4 packed(const float* v, const bf16_t*) {
    return u32x4{f32x2_to_bf16(v[0], v[1]), f32x2_to_bf16(v[2], v[3]), f32x2_to_bf16(v[4], v[5]), f32x2_to_bf16(v[6], v[7])};
}
__device__ inline u32x4 packed(const float* v, const __half*) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __builtin_bit_cast(uint32_t, __floats2half2_rn(v[2 * i], v[2 * i + 1]));
    return o;
}

// STREAM: past the caches.
template <typename T, bool STREAM>
__global__ __launch_bounds__(kOuterThreads) void expert_outer(const Outer a) {
    constexpr int N = 16 / static_cast<int>(sizeof(T)), kAhead = 4;   // rows in flight together
    const ExpertArgs& g = a.g;
    const int xcd = blockIdx.x % kXcds, nth = blockIdx.x / kXcds, e = nth / a.share;
    const int block = (xcd + e) % kXcds * a.share + nth % a.share;   // few workgroups of an expert: another XCD's for the next one
    const int lane = threadIdx.x & 63, wave = block * kOuterWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = wave / a.strips, vector = (wave - group * a.strips) * 64 + lane;
    if (block >= a.blocks || group >= a.groups || vector * static_cast<int64_t>(N) >= g.k) return;
    int lo, hi;
    rows_of_expert(g, e, lo, hi);
    if (hi - lo > g.few) return;
    const int64_t k0 = min(vector * static_cast<int64_t>(N), g.k - N), n0 = min(group * static_cast<int64_t>(kSide), g.n - kSide);
    const T* dy = static_cast<const T*>(g.a) + lo * g.lda + n0;
    const T* x = static_cast<const T*>(g.w) + lo * g.ldw + k0;
    float sum[kSide][N];
#pragma unroll
    for (int i = 0; i < kSide; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) sum[i][j] = 0.f;
    for (int left = hi - lo; left > 0; left -= kAhead, dy += kAhead * g.lda, x += kAhead * g.ldw) {
        Vector<T, N> vx[kAhead];
        Vector<T, kSide> vd[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int row = u < left ? u : 0;
            vx[u] = load_vector<T, N>(x + row * g.ldw), vd[u] = load_vector<T, kSide>(dy + row * g.lda);
        }
        asm volatile("" ::: "memory");   // else the compiler moves each row's loads behind the sums of the one before it
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (u >= left) break;
            uint32_t same[kSide * sizeof(T) / 4];
#pragma unroll
            for (int i = 0; i < static_cast<int>(kSide * sizeof(T) / 4); ++i) same[i] = __builtin_amdgcn_readfirstlane(vd[u].word[i]);
#pragma unroll
            for (int i = 0; i < kSide; ++i) {
                const float d = element(same, i, static_cast<const T*>(nullptr));
#pragma unroll
                for (int j = 0; j < N; ++j) sum[i][j] += d * element(vx[u].word, j, static_cast<const T*>(nullptr));
            }
        }
    }
    T* const y = static_cast<T*>(g.y) + (e * g.n + n0) * g.k + k0;
#pragma unroll
    for (int i = 0; i < kSide; ++i) {
        typedef u32x4 any __attribute__((aligned(2)));
        any* const to = reinterpret_cast<any*>(y + i * g.k);
        const u32x4 v = packed(sum[i], static_cast<const T*>(nullptr));
        if constexpr (STREAM) __builtin_nontemporal_store(v, to);
        else *to = v;
    }
}

}  // namespace

int run_expert_outer(const char* who, const ExpertArgs& g, hipStream_t s) {
    const int elements = g.out_dtype == DDL_DT_F32 ? 4 : 8;
    Outer a{g};
    a.strips = static_cast<int>((g.k + 64 * elements - 1) / (64 * elements)), a.groups = static_cast<int>((g.n + kSide - 1) / kSide);
    a.blocks = (a.strips * a.groups + kOuterWaves - 1) / kOuterWaves, a.share = (a.blocks + kXcds - 1) / kXcds;
    const int64_t blocks = static_cast<int64_t>(a.share) * kXcds * g.experts;
    if (blocks * kOuterThreads > 0xFFFFFFFFll) return fail(DDL_E_UNSUPP, "%s: %lld workgroups", who, static_cast<long long>(blocks));
    // Rows of whole lines need no cache to put them together, and more rows of x and dy stay in the caches: [8 x 3584, 8192] bf16 of four rows each 85 -> 75 us, [16 x 3743, 4476] of
    // 24 256 -> 220, of one 90 -> 128.
    const bool stream = (g.k * (16 / elements) % 128 == 0 && aligned_to(g.y, 128)) || g.rows >= 8 * g.experts;
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
