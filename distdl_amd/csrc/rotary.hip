// Rotation of queries and keys by their positions, alone or behind a norm of each head, on heads that a worker holds whole.
//
//   rotation   pair p of a head turns by t = position * frequency[p]:
//                y[p] = a (x[p] cos t - x[p'] sin t),   y[p'] = a (x[p'] cos t + x[p] sin t)
//              p' is p + rotated/2 (halves) or the next element (neighbours, p even); elements behind `rotated` pass through
//   adjoint    the same with -t
//   head norm  xhat = x rstd, rstd = 1 / sqrt(mean(x^2) + eps) over the head, y = rotation(xhat * w)
//   adjoint    g = inverse rotation of dy, dw = sum over tokens and heads of g xhat,
//              dx = rstd (w g - xhat mean(w g xhat))
//
// Bound by memory: every element is read and written once, an element of 16 bits pays four bytes for its four or so
// operations.  The angles are what could cost more than that: position * frequency needs 64 bits (a position of 10^6 leaves
// 32-bit products off by 0.06), so a wavefront computes those of a token once, in turns, of which the whole ones are dropped
// before 32 bits take over, and uses them for all heads of the token.
//
// [4,2048,64+8,128] bf16: 66 us (4.6 TB/s), with the norm 66, its adjoint 104 (4.4 TB/s) and 5 for the weights' sums; one token of 16
// sequences, 8+1 heads: 4 and 5 us, most of them the launch.
//
// A head lies in LPH = 1 .. 64 neighbouring lanes of a wavefront, eight elements a lane: the two members of a pair in the same
// lane, so that nothing but the norm's sum crosses lanes.
#include "ddl_common.h"

#include "ln_elements.h"

namespace ddl {
namespace {

constexpr int kWave = 64;
constexpr int kBlock = 256;
constexpr int kWavesPerBlock = kBlock / kWave;
constexpr int kMaxHeadDim = 512;      // 64 lanes of eight elements
constexpr int kGradBlocks = 1024;     // workgroups of the norm's adjoint at most, each with a partial sum of dw ([4,2048,64+8,128] bf16: 106 us with both, 512: 149)

struct Place {   // of a [batch, tokens, heads, head_dim] tensor: strides in elements, head_dim's is 1
    int64_t batch, token, head;
};

struct RotaryArgs {
    const void* x[2];    // queries, keys
    const void* dy[2];
    void* y[2];
    Place x_at[2], dy_at[2], y_at[2];
    const void* weight[2];
    const double* frequency;
    const void* position;
    int64_t position_batch;   // stride of a sequence's positions
    int32_t position_bytes;   // 0: token t is at position t
    int32_t heads[2];
    int32_t rows, tokens;     // batch * tokens, tokens
    int32_t slices;           // wavefronts that share the heads of a token
    int32_t dim, half;        // half: pairs that turn
    int32_t lph_log2;
    float eps, amplitude, inv_dim;
    float sign;               // of the angles
    float* partial;           // [blocks][2][dim] sums for dw
};

// N elements at element alignment as floats, and back.
template <int BYTES, int ALIGN>
struct __attribute__((packed, aligned(ALIGN))) Raw {
    uint8_t byte[BYTES];
};
template <typename T, int N>
__device__ inline void load_n(const T* p, float (&v)[N]) {
    T e[N];
    const Raw<N * sizeof(T), sizeof(T)> r = *reinterpret_cast<const Raw<N * sizeof(T), sizeof(T)>*>(p);
    __builtin_memcpy(e, &r, sizeof(e));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = load1(&e[i]);
}
template <typename T, int N>
__device__ inline void store_n(T* p, const float (&v)[N]) {
    Raw<N * sizeof(T), sizeof(T)> r;
    if constexpr (std::is_same_v<T, bf16_t> && N % 2 == 0) {
        uint32_t w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = f32x2_to_bf16(v[2 * i], v[2 * i + 1]);
        __builtin_memcpy(&r, w, sizeof(r));
    } else {
        T e[N];
#pragma unroll
        for (int i = 0; i < N; ++i) store1(&e[i], v[i]);
        __builtin_memcpy(&r, e, sizeof(r));
    }
    *reinterpret_cast<Raw<N * sizeof(T), sizeof(T)>*>(p) = r;
}

// Sum over the 2^log2 neighbouring lanes that hold a head, the same in each of them.
__device__ inline float head_sum(float v, int log2) {
    if (log2 > 0) v += dpp_moved<0xB1, 0xF>(v);     // quad_perm [1,0,3,2]
    if (log2 > 1) v += dpp_moved<0x4E, 0xF>(v);     // quad_perm [2,3,0,1]
    if (log2 > 2) v += dpp_moved<0x141, 0xF>(v);    // row_half_mirror
    if (log2 > 3) v += dpp_moved<0x140, 0xF>(v);    // row_mirror
    if (log2 > 4) v += __shfl_xor(v, 16);
    if (log2 > 5) v += __shfl_xor(v, 32);
    return v;
}

enum RotaryMode {
    kRotate = 0,
    kNormRotate = 1,
    kNormRotateBackward = 2,
};

// Eight elements of a head: 4 / VP slots of VP pairs, the slots of a head dealt to its lanes in turn.  VP is the largest of
// 4, 2, 1 that divides the pairs that turn and the pairs of the head, so a slot's members a and b are runs of VP elements.
template <typename T, int VP, bool NEIGHBOURS>
struct HeadPiece {
    static constexpr int NS = 4 / VP;
    int a[NS], b[NS];     // offsets in the head; a < 0: nothing; b < 0: no second member (an odd head's last element)

    __device__ void place(int lane_in_head, int lph, int dim, int half) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int first = (lane_in_head + s * lph) * VP;    // first pair of the slot
            const bool halves = !NEIGHBOURS && first < half;
            a[s] = halves ? first : 2 * first;
            b[s] = halves ? half + first : 2 * first + VP;
            if (a[s] >= dim) a[s] = -1, b[s] = -1;
            else if (b[s] >= dim) b[s] = -1;
        }
    }
    // v[2 i], v[2 i + 1]: the members of pair i where pairs turn (in any order of the elements where they pass through)
    __device__ void load(const T* head, bool there, float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
        if (!there) return;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            if (a[s] < 0) continue;
            if constexpr (NEIGHBOURS && VP > 1) {
                float both[2 * VP];
                load_n<T, 2 * VP>(head + a[s], both);
#pragma unroll
                for (int i = 0; i < 2 * VP; ++i) v[2 * VP * s + i] = both[i];
            } else {
                float first[VP], second[VP] = {};
                load_n<T, VP>(head + a[s], first);
                if (VP > 1 || b[s] >= 0) load_n<T, VP>(head + b[s], second);
#pragma unroll
                for (int i = 0; i < VP; ++i) v[2 * (VP * s + i)] = first[i], v[2 * (VP * s + i) + 1] = second[i];
            }
        }
    }
    __device__ void store(T* head, bool there, const float (&v)[8]) const {
        if (!there) return;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            if (a[s] < 0) continue;
            if constexpr (NEIGHBOURS && VP > 1) {
                float both[2 * VP];
#pragma unroll
                for (int i = 0; i < 2 * VP; ++i) both[i] = v[2 * VP * s + i];
                store_n<T, 2 * VP>(head + a[s], both);
            } else {
                float first[VP], second[VP];
#pragma unroll
                for (int i = 0; i < VP; ++i) first[i] = v[2 * (VP * s + i)], second[i] = v[2 * (VP * s + i) + 1];
                store_n<T, VP>(head + a[s], first);
                if (VP > 1 || b[s] >= 0) store_n<T, VP>(head + b[s], second);
            }
        }
    }
};

__device__ inline void turned(float (&v)[8], const float (&c)[4], const float (&s)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = v[2 * i], b = v[2 * i + 1];
        v[2 * i] = a * c[i] - b * s[i];
        v[2 * i + 1] = b * c[i] + a * s[i];
    }
}

// UN: heads of a lane in flight at once.  The adjoint holds two tensors and the weights' sums: with two heads [4,2048,64+8,128] bf16 took 111 us instead
// of 106, [16,4096,8+1,128] 163 instead of 137.
template <typename T, int VP, bool NEIGHBOURS, int MODE, int UN>
__global__ __launch_bounds__(kBlock) void rotary_heads(const RotaryArgs arg) {
    typedef HeadPiece<T, VP, NEIGHBOURS> Piece;
    const int lane = threadIdx.x & (kWave - 1), lph = 1 << arg.lph_log2, step = kWave >> arg.lph_log2;
    const int in_head = lane & (lph - 1), sub = lane >> arg.lph_log2;
    const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * kWavesPerBlock + threadIdx.x / kWave);
    Piece piece;
    piece.place(in_head, lph, arg.dim, arg.half);
    // In turns; pairs that pass through stay at angle 0 with amplitude 1.
    constexpr double kTurn = 0.15915494309189533577;   // 1 / (2 pi)
    double frequency[4];
    bool turns[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int pair = (in_head + (i / VP) * lph) * VP + i % VP;
        turns[i] = pair < arg.half;
        frequency[i] = turns[i] ? arg.frequency[pair] * kTurn : 0.0;
    }
    float w[2][8], dw[2][8];
    if (MODE != kRotate) {
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            if (arg.weight[part]) {
                piece.load(static_cast<const T*>(arg.weight[part]), true, w[part]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) w[part][i] = 1.f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) dw[part][i] = 0.f;
        }
    }
    const int64_t items = static_cast<int64_t>(arg.rows) * arg.slices;
    for (int64_t item = wave; item < items; item += static_cast<int64_t>(gridDim.x) * kWavesPerBlock) {
        const uint32_t row = arg.slices == 1 ? static_cast<uint32_t>(item) : static_cast<uint32_t>(item / arg.slices);
        const int slice = static_cast<int>(item - static_cast<int64_t>(row) * arg.slices);
        const uint32_t batch = row / static_cast<uint32_t>(arg.tokens), token = row - batch * arg.tokens;
        double position = token;
        if (arg.position_bytes) {
            const int64_t at = batch * arg.position_batch + token;
            position = arg.position_bytes == 8 ? static_cast<double>(static_cast<const int64_t*>(arg.position)[at])
                                               : static_cast<double>(static_cast<const int32_t*>(arg.position)[at]);
        }
        float c[4], s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double t = position * frequency[i];
            const float rest = static_cast<float>(t - rint(t));      // of a turn, in [-1/2, 1/2]
            sincospif(2.f * rest, &s[i], &c[i]);
            c[i] = turns[i] ? c[i] * arg.amplitude : 1.f;
            s[i] = turns[i] ? s[i] * (arg.amplitude * arg.sign) : 0.f;
        }
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const int share = (arg.heads[part] + arg.slices - 1) / arg.slices;
            const int lo = slice * share, hi = min(arg.heads[part], lo + share);
            const Place &xa = arg.x_at[part], &da = arg.dy_at[part], &ya = arg.y_at[part];
            const T* x = static_cast<const T*>(arg.x[part]) + (batch * xa.batch + token * xa.token);
            const T* dy = static_cast<const T*>(arg.dy[part]) + (batch * da.batch + token * da.token);
            T* y = static_cast<T*>(arg.y[part]) + (batch * ya.batch + token * ya.token);
            for (int h0 = lo; h0 < hi; h0 += UN * step) {
                float v[UN][8], g[UN][8];
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    if (u > 0 && h0 + u * step >= hi) continue;      // for all lanes
                    const int h = h0 + u * step + sub;
                    piece.load(x + h * xa.head, h < hi, v[u]);
                    if (MODE == kNormRotateBackward) piece.load(dy + h * da.head, h < hi, g[u]);
                }
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    if (u > 0 && h0 + u * step >= hi) continue;
                    const int h = h0 + u * step + sub;
                    if (MODE != kRotate) {
                        float q = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) q += v[u][i] * v[u][i];
                        // (of no head: 0, so that eps = 0 makes no NaN of it)
                        const float rstd = h < hi ? 1.0f / sqrtf(head_sum(q, arg.lph_log2) * arg.inv_dim + arg.eps) : 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[u][i] *= rstd;
                        if (MODE == kNormRotateBackward) {
                            turned(g[u], c, s);
                            float m = 0.f;
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                dw[part][i] += g[u][i] * v[u][i];
                                g[u][i] *= w[part][i];
                                m += g[u][i] * v[u][i];
                            }
                            m = head_sum(m, arg.lph_log2) * arg.inv_dim;
#pragma unroll
                            for (int i = 0; i < 8; ++i) v[u][i] = rstd * (g[u][i] - v[u][i] * m);
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; ++i) v[u][i] *= w[part][i];
                        }
                    }
                    if (MODE != kNormRotateBackward) turned(v[u], c, s);
                    piece.store(y + h * ya.head, h < hi, v[u]);
                }
            }
        }
    }
    if (MODE == kNormRotateBackward && arg.partial) {
        // Over the heads that a wavefront has side by side, then over the workgroup's wavefronts in their order.
        __shared__ float sums[kWavesPerBlock][2][kMaxHeadDim];
        const int w_in_block = threadIdx.x / kWave;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                for (int m = lph; m < kWave; m <<= 1) dw[part][i] += __shfl_xor(dw[part][i], m);
            if (sub == 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int slot = i / (2 * VP), pair = (i / 2) % VP, second = i & 1;
                    int e;
                    if (NEIGHBOURS && VP > 1) e = piece.a[slot] + i % (2 * VP);
                    else e = (second ? piece.b[slot] : piece.a[slot]) + pair;
                    if (piece.a[slot] >= 0 && (VP > 1 || !second || piece.b[slot] >= 0)) sums[w_in_block][part][e] = dw[part][i];
                }
            }
        }
        __syncthreads();
        float* out = arg.partial + static_cast<int64_t>(blockIdx.x) * 2 * arg.dim;
        for (int e = threadIdx.x; e < 2 * arg.dim; e += kBlock) {
            const int part = e >= arg.dim, col = e - part * arg.dim;
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < kWavesPerBlock; ++k) t += sums[k][part][col];
            out[e] = t;
        }
    }
}

// dw[e] = sum over the workgroups' partial sums, in one order: 16 columns x 64 rows at a time.
template <typename T>
__global__ __launch_bounds__(1024) void weight_grads(const float* __restrict__ partial, int blocks, int dim, T* dwq, T* dwk) {
    __shared__ float sums[64][17];
    const int col = threadIdx.x & 15, lane = threadIdx.x >> 4;
    const int e = blockIdx.x * 16 + col;
    float t = 0.f;
    if (e < 2 * dim) {
#pragma unroll 8
        for (int b = lane; b < blocks; b += 64) t += partial[static_cast<int64_t>(b) * 2 * dim + e];
    }
    sums[lane][col] = t;
    __syncthreads();
    if (lane == 0 && e < 2 * dim) {
        float all = 0.f;
#pragma unroll
        for (int k = 0; k < 64; ++k) all += sums[k][col];
        T* out = e < dim ? dwq : dwk;
        if (out) store1(out + (e < dim ? e : e - dim), all);
    }
}

int grid_for(const RotaryArgs& a, int blocks_per_cu) {
    int dev;
    const int64_t waves = static_cast<int64_t>(a.rows) * a.slices, blocks = (waves + kWavesPerBlock - 1) / kWavesPerBlock;
    const int64_t most = static_cast<int64_t>(compute_units(dev)) * blocks_per_cu;
    return static_cast<int>(blocks < most ? blocks : most);
}

template <typename T, int VP, bool NEIGHBOURS>
int launch(const RotaryArgs& a, int mode, int grid, hipStream_t s) {
    switch (mode) {
        case kRotate: hipLaunchKernelGGL((rotary_heads<T, VP, NEIGHBOURS, kRotate, 4>), dim3(grid), dim3(kBlock), 0, s, a); break;
        case kNormRotate: hipLaunchKernelGGL((rotary_heads<T, VP, NEIGHBOURS, kNormRotate, 4>), dim3(grid), dim3(kBlock), 0, s, a); break;
        default: hipLaunchKernelGGL((rotary_heads<T, VP, NEIGHBOURS, kNormRotateBackward, 1>), dim3(grid), dim3(kBlock), 0, s, a); break;
    }
    return check_launch("ddl_rotary");
}

template <typename T>
int launch_pairs(const RotaryArgs& a, bool neighbours, int mode, int grid, hipStream_t s) {
    if (a.dim % 8 == 0 && a.half % 4 == 0) return neighbours ? launch<T, 4, true>(a, mode, grid, s) : launch<T, 4, false>(a, mode, grid, s);
    if (a.dim % 4 == 0 && a.half % 2 == 0) return neighbours ? launch<T, 2, true>(a, mode, grid, s) : launch<T, 2, false>(a, mode, grid, s);
    return neighbours ? launch<T, 1, true>(a, mode, grid, s) : launch<T, 1, false>(a, mode, grid, s);
}

Place place_of(const int64_t* strides) { return strides ? Place{strides[0], strides[1], strides[2]} : Place{0, 0, 0}; }

// The arguments that all entry points share; 0 or a refusal.
int fill(RotaryArgs& a, int dtype, int64_t batch, int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t dim, const double* frequencies,
         int64_t rotated, const void* positions, int position_bytes, int64_t position_batch, float amplitude, int inverse) {
    if (batch < 0 || tokens < 0 || q_heads < 0 || k_heads < 0 || dim < 1) return fail(DDL_E_ARG, "rotary: negative extent or empty heads");
    if (dtype != DDL_DT_F32 && dtype != DDL_DT_BF16 && dtype != DDL_DT_F16) return fail(DDL_E_ARG, "rotary: dtype %d", dtype);
    if (dim > kMaxHeadDim) return fail(DDL_E_UNSUPP, "rotary: heads of %lld elements (at most %d)", static_cast<long long>(dim), kMaxHeadDim);
    if (rotated < 0 || rotated > dim || rotated % 2) return fail(DDL_E_SHAPE, "rotary: %lld of %lld elements cannot turn in pairs", static_cast<long long>(rotated), static_cast<long long>(dim));
    if (rotated && !frequencies) return fail(DDL_E_ARG, "rotary: no frequencies");
    if (position_bytes != 0 && position_bytes != 4 && position_bytes != 8) return fail(DDL_E_ARG, "rotary: positions of %d bytes", position_bytes);
    if (position_bytes && !positions && batch * tokens) return fail(DDL_E_ARG, "rotary: no positions");
    if (q_heads > 0x7FFFFFFF || k_heads > 0x7FFFFFFF || (tokens && batch > 0x7FFFFFFF / tokens)) return fail(DDL_E_UNSUPP, "rotary: 2^31 tokens or heads");
    a.frequency = frequencies, a.position = positions, a.position_bytes = position_bytes, a.position_batch = position_batch;
    a.heads[0] = static_cast<int>(q_heads), a.heads[1] = static_cast<int>(k_heads);
    a.rows = static_cast<int>(batch * tokens), a.tokens = static_cast<int>(tokens);
    a.dim = static_cast<int>(dim), a.half = static_cast<int>(rotated / 2);
    a.amplitude = amplitude, a.sign = inverse ? -1.f : 1.f, a.inv_dim = 1.0f / static_cast<float>(dim);
    a.lph_log2 = 0;
    while ((8 << a.lph_log2) < dim) ++a.lph_log2;
    // Few tokens: their heads are shared by as many wavefronts as have some in every step (2048 are eight for each CU).
    const int64_t at_once = 4 * (kWave >> a.lph_log2), heads = q_heads > k_heads ? q_heads : k_heads;
    int64_t slices = 1;
    while (a.rows * slices < 2048 && slices * at_once < heads) slices *= 2;
    a.slices = static_cast<int>(slices);
    return 0;
}

template <typename Fn>
int with_element(int dtype, Fn&& fn) {
    int rc = 0;
    with_ln_element(dtype, [&](auto* p) { rc = fn(p); });
    return rc;
}

}  // namespace
}  // namespace ddl

extern "C" {

int ddl_head_rotary(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, int dtype, int64_t batch, int64_t tokens,
                    int64_t q_heads, int64_t k_heads, int64_t dim, const void* q_weight, const void* k_weight, int norm, float eps,
                    const double* frequencies, int64_t rotated, const void* positions, int position_bytes, int64_t position_batch,
                    int neighbours, float amplitude, int inverse, void* yq, const int64_t* yq_strides, void* yk, const int64_t* yk_strides,
                    void* stream) {
    using namespace ddl;
    RotaryArgs a{};
    if (const int rc = fill(a, dtype, batch, tokens, q_heads, k_heads, dim, frequencies, rotated, positions, position_bytes, position_batch, amplitude, inverse)) return rc;
    if (a.rows == 0 || (q_heads == 0 && k_heads == 0)) return 0;
    if ((q_heads && (!q || !yq || !q_strides || !yq_strides)) || (k_heads && (!k || !yk || !k_strides || !yk_strides)))
        return fail(DDL_E_ARG, "ddl_head_rotary: null tensor");
    if (!norm && (q_weight || k_weight)) return fail(DDL_E_ARG, "ddl_head_rotary: weights without a norm");
    if (norm && inverse) return fail(DDL_E_ARG, "ddl_head_rotary: the adjoint of a norm is ddl_head_norm_rotary_backward");
    a.x[0] = q, a.x[1] = k, a.y[0] = yq, a.y[1] = yk, a.weight[0] = q_weight, a.weight[1] = k_weight, a.eps = eps;
    a.x_at[0] = place_of(q_strides), a.x_at[1] = place_of(k_strides), a.y_at[0] = place_of(yq_strides), a.y_at[1] = place_of(yk_strides);
    const int grid = grid_for(a, 16);
    return with_element(dtype, [&](auto* e) {
        return launch_pairs<std::remove_pointer_t<decltype(e)>>(a, neighbours != 0, norm ? kNormRotate : kRotate, grid, static_cast<hipStream_t>(stream));
    });
}

int64_t ddl_head_norm_rotary_backward_workspace(int64_t dim) { return dim < 1 ? 0 : static_cast<int64_t>(ddl::kGradBlocks) * 2 * dim; }

int ddl_head_norm_rotary_backward(const void* dyq, const int64_t* dyq_strides, const void* dyk, const int64_t* dyk_strides, const void* q,
                                  const int64_t* q_strides, const void* k, const int64_t* k_strides, int dtype, int64_t batch, int64_t tokens,
                                  int64_t q_heads, int64_t k_heads, int64_t dim, const void* q_weight, const void* k_weight, float eps,
                                  const double* frequencies, int64_t rotated, const void* positions, int position_bytes, int64_t position_batch,
                                  int neighbours, float amplitude, void* dq, const int64_t* dq_strides, void* dk, const int64_t* dk_strides,
                                  void* dq_weight, void* dk_weight, float* workspace, int64_t workspace_elems, void* stream) {
    using namespace ddl;
    RotaryArgs a{};
    if (const int rc = fill(a, dtype, batch, tokens, q_heads, k_heads, dim, frequencies, rotated, positions, position_bytes, position_batch, amplitude, 1)) return rc;
    const bool sums = dq_weight || dk_weight;
    if (sums && (!workspace || workspace_elems < ddl_head_norm_rotary_backward_workspace(dim)))
        return fail(DDL_E_ARG, "ddl_head_norm_rotary_backward: workspace of %lld floats, %lld are needed", static_cast<long long>(workspace ? workspace_elems : 0),
                    static_cast<long long>(ddl_head_norm_rotary_backward_workspace(dim)));
    int grid = 0;
    if (a.rows && (q_heads || k_heads)) {
        if ((q_heads && (!q || !dyq || !dq || !q_strides || !dyq_strides || !dq_strides)) || (k_heads && (!k || !dyk || !dk || !k_strides || !dyk_strides || !dk_strides)))
            return fail(DDL_E_ARG, "ddl_head_norm_rotary_backward: null tensor");
        a.x[0] = q, a.x[1] = k, a.dy[0] = dyq, a.dy[1] = dyk, a.y[0] = dq, a.y[1] = dk, a.weight[0] = q_weight, a.weight[1] = k_weight, a.eps = eps;
        a.x_at[0] = place_of(q_strides), a.x_at[1] = place_of(k_strides), a.dy_at[0] = place_of(dyq_strides), a.dy_at[1] = place_of(dyk_strides);
        a.y_at[0] = place_of(dq_strides), a.y_at[1] = place_of(dk_strides);
        a.partial = sums ? workspace : nullptr;
        grid = grid_for(a, 4);
        if (grid > kGradBlocks) grid = kGradBlocks;
        const int rc = with_element(dtype, [&](auto* e) {
            return launch_pairs<std::remove_pointer_t<decltype(e)>>(a, neighbours != 0, kNormRotateBackward, grid, static_cast<hipStream_t>(stream));
        });
        if (rc) return rc;
    }
    if (!sums) return 0;
    return with_element(dtype, [&](auto* e) {
        typedef std::remove_pointer_t<decltype(e)> T;
        hipLaunchKernelGGL((weight_grads<T>), dim3((2 * static_cast<int>(dim) + 15) / 16), dim3(1024), 0, static_cast<hipStream_t>(stream), workspace, grid,
                           static_cast<int>(dim), static_cast<T*>(dq_weight), static_cast<T*>(dk_weight));
        return check_launch("ddl_head_norm_rotary_backward");
    });
}

}  // extern "C"
