// Vectors of elements that lie anywhere, for the experts' kernels that take operands from memory into matrix instructions.
#ifndef DDL_EXPERT_VECTORS_H
#define DDL_EXPERT_VECTORS_H
#include "gemm16_parts.h"
#include "ln_elements.h"

namespace ddl {
namespace {

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
__device__ inline uint32_t word_of(const float* v, int i, const float*) { return __float_as_uint(v[i]); }
__device__ inline uint32_t word_of(const float* v, int i, const bf16_t*) { return f32x2_to_bf16(v[2 * i], v[2 * i + 1]); }
__device__ inline uint32_t word_of(const float* v, int i, const __half*) { return __builtin_bit_cast(uint32_t, __floats2half2_rn(v[2 * i], v[2 * i + 1])); }
// N values, rounded once.  STREAM: past the caches.
template <int N, bool STREAM = false, typename T>
__device__ inline void store_vector(T* p, const float* v) {
    constexpr int kWords = N * static_cast<int>(sizeof(T)) / 4;
    typedef uint32_t words __attribute__((ext_vector_type(kWords)));
    typedef words any __attribute__((aligned(2)));
    words o;
#pragma unroll
    for (int i = 0; i < kWords; ++i) o[i] = word_of(v, i, static_cast<const T*>(nullptr));
    if constexpr (STREAM) __builtin_nontemporal_store(o, reinterpret_cast<any*>(p));
    else *reinterpret_cast<any*>(p) = o;
}
// Element c of eight rows, side by side.
template <typename V>
__device__ inline bf16x8 column(const V (&rows)[8], int c) {
    u32x4 o;
#pragma unroll
    for (int p = 0; p < 4; ++p) o[p] = __builtin_amdgcn_perm(rows[2 * p + 1].word[c / 2], rows[2 * p].word[c / 2], c % 2 ? 0x07060302u : 0x05040100u);
    return __builtin_bit_cast(bf16x8, o);
}

}  // namespace
}  // namespace ddl
#endif  // DDL_EXPERT_VECTORS_H
