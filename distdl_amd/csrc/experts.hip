// Tokens to their experts and back: the order of the choices (plan), rows copied into it (sort), rows added up from it with the
// router's weights (combine), and the adjoints of both.
//
// The plan is a counting sort by expert that keeps the slots' order within one, so that results do not depend on which wavefront
// came first.  A wavefront walks over its part of the slots 64 at a time; the lanes with the same expert find each other by
// one ballot for each bit of the number.  Up to kAlone slots it is one launch of one workgroup; more are counted by one launch and
// placed by a second, whose workgroups add up the counts of those in front of them: bound by latency, so a workgroup has 512 slots while
// that makes no more than kMostParts of them.
//
// Everything that moves rows goes by tokens, not by sorted rows: a token's row is read once, however many experts it goes to
// (sort; adjoint of combine), and what comes back is added up in registers in the order of the choices (combine; adjoint of the sort).  Bound by
// HBM.  A row is cut into vectors of 16 bytes at any address, the last one moved back to end with the row; rows shorter than a
// vector go element by element.
#include "ln_elements.h"

namespace ddl {
namespace {

constexpr int kWave = 64;
constexpr int kPlanThreads = 512, kPlanWaves = kPlanThreads / kWave;
constexpr int kAlone = 2048;            // slots up to which one workgroup makes the plan
constexpr int kMostParts = 128;         // workgroups otherwise
constexpr int kMaxHeld = 2047;          // experts; one bucket more for what is not held

struct PlanArgs {
    const void* ids;
    int id_bytes;
    int64_t ld_ids, low;
    int slots, part, held, bits;        // part: slots of a workgroup; bits: of bucket numbers 0 .. held
    FastDiv chosen;
    int32_t *place, *offsets, *counts;  // counts: [workgroups, held + 1]
};

__device__ inline int bucket_of(const PlanArgs& a, int slot) {
    const uint32_t token = fd_div(static_cast<uint32_t>(slot), a.chosen);
    const int64_t at = static_cast<int64_t>(token) * a.ld_ids + (static_cast<uint32_t>(slot) - token * a.chosen.div);
    const int64_t id = a.id_bytes == 8 ? static_cast<const int64_t*>(a.ids)[at] : static_cast<const int32_t*>(a.ids)[at];
    return id >= a.low && id - a.low < a.held ? static_cast<int>(id - a.low) : a.held;
}

// Lanes with the same bucket as this one (only lanes that are `on` have any).
__device__ inline uint64_t lanes_alike(int bucket, bool on, int bits) {
    uint64_t same = __ballot(on);
    for (int b = 0; b < bits; ++b) {
        const bool one = (bucket >> b) & 1;
        const uint64_t ones = __ballot(one);
        same &= one ? ones : ~ones;
    }
    return same;
}

// Counters that other lanes of the wavefront change: read and written where it says so.
__device__ inline int get(const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }
__device__ inline void put(int* p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }

// Slots of each bucket that each wavefront of the workgroup has, in lds[wave][bucket].
__device__ inline void count_slots(const PlanArgs& a, int first, int last, int per_wave, int* lds) {
    const int buckets = a.held + 1, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    for (int i = threadIdx.x; i < kPlanWaves * buckets; i += kPlanThreads) lds[i] = 0;
    __syncthreads();
    const int from = min(wave * per_wave, last - first) + first, to = min(last - from, per_wave) + from;
    int* const mine = lds + wave * buckets;   // of this wavefront alone: its own LDS accesses complete in order
    for (int s = from + lane; s - lane < to; s += kWave) {
        const bool on = s < to;
        const int bucket = on ? bucket_of(a, s) : 0;
        const uint64_t same = lanes_alike(bucket, on, a.bits);
        if (on && (same & ((1ull << lane) - 1)) == 0) put(mine + bucket, get(mine + bucket) + __popcll(same));
    }
    __syncthreads();
}

__global__ __launch_bounds__(kPlanThreads) void expert_count(const PlanArgs a) {
    extern __shared__ int lds[];
    const int buckets = a.held + 1, first = static_cast<int>(blockIdx.x) * a.part, last = min(a.slots - first, a.part) + first;
    count_slots(a, first, last, a.part / kPlanWaves, lds);
    for (int b = threadIdx.x; b < buckets; b += kPlanThreads) {
        int n = 0;
#pragma unroll
        for (int w = 0; w < kPlanWaves; ++w) n += lds[w * buckets + b];
        a.counts[static_cast<int64_t>(blockIdx.x) * buckets + b] = n;
    }
}

// lds: kPlanWaves x buckets counts, then the first place of this workgroup's slots of each bucket, then the scan's sums.
__global__ __launch_bounds__(kPlanThreads) void expert_place(const PlanArgs a) {
    extern __shared__ int lds[];
    const int buckets = a.held + 1, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    int* const base = lds + kPlanWaves * buckets;
    int* const sums = base + buckets;
    const int first = static_cast<int>(blockIdx.x) * a.part, last = min(a.slots - first, a.part) + first;
    const int per_wave = a.part / kPlanWaves;
    count_slots(a, first, last, per_wave, lds);
    // Slots of the buckets in front of each one: a running sum over the buckets, kPlanThreads at a time.
    int carry = 0;
    for (int b0 = 0; b0 < buckets; b0 += kPlanThreads) {
        const int b = b0 + threadIdx.x;
        int total = 0, before = 0;   // in all workgroups; in those in front of this one
        if (b < buckets) {
            if (gridDim.x == 1) {
#pragma unroll
                for (int w = 0; w < kPlanWaves; ++w) total += lds[w * buckets + b];
            } else {
#pragma unroll 8
                for (int g = 0; g < static_cast<int>(gridDim.x); ++g) {
                    const int n = a.counts[static_cast<int64_t>(g) * buckets + b];
                    total += n;
                    before += g < static_cast<int>(blockIdx.x) ? n : 0;
                }
            }
        }
        int run = total;   // inclusive, over the wavefront
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const int v = __shfl_up(run, d);
            if (lane >= d) run += v;
        }
        if (lane == kWave - 1) sums[wave] = run;
        __syncthreads();
        int front = carry, all = 0;
#pragma unroll
        for (int w = 0; w < kPlanWaves; ++w) {
            front += w < wave ? sums[w] : 0;
            all += sums[w];
        }
        if (b < buckets) {
            base[b] = front + run - total + before;
            if (blockIdx.x == 0) a.offsets[b] = front + run - total;   // bucket `held` starts where the held slots end
        }
        carry += all;
        __syncthreads();
    }
    // Each wavefront's first place, instead of its count.
    for (int b = threadIdx.x; b < buckets; b += kPlanThreads) {
        int at = base[b];
#pragma unroll
        for (int w = 0; w < kPlanWaves; ++w) {
            const int n = lds[w * buckets + b];
            lds[w * buckets + b] = at;
            at += n;
        }
    }
    __syncthreads();
    const int from = min(wave * per_wave, last - first) + first, to = min(last - from, per_wave) + from;
    int* const next = lds + wave * buckets;
    for (int s = from + lane; s - lane < to; s += kWave) {
        const bool on = s < to;
        const int bucket = on ? bucket_of(a, s) : 0;
        const uint64_t same = lanes_alike(bucket, on, a.bits), lower = same & ((1ull << lane) - 1);
        if (on) {
            const int at = get(next + bucket);
            a.place[s] = at + __popcll(lower);
            if (lower == 0) put(next + bucket, at + __popcll(same));
        }
    }
}

// -------------------------------------------------------------- rows --

// Whatever a plan's tensors hold, only rows 0 .. slots - 1 are touched: places from `held` on have no row in the sums, places outside the slots none at all.
struct RowArgs {
    const void *in, *y;                 // by tokens; by places
    void *out, *dy;
    const float *weights, *scales;
    float *out_scales, *dweights;
    const int32_t *place, *held;
    int64_t ld_in, ld_y, tokens;
    uint32_t slots;
    int chosen, cols;                   // cols in elements of the kernel's type
    int vectors;                        // of a row
    int lanes_log2;                     // lanes of a row's group: 1 to 64
    FastDiv groups;                     // wavefronts (of one token) side by side in the columns
};

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// VEC: vectors of 16 bytes at any address; otherwise elements.
template <typename T, bool VEC>
struct Chunk {
    static constexpr int n = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
    std::conditional_t<VEC, u32x4_t, T> v;
};
template <typename T, bool VEC>
__device__ inline Chunk<T, VEC> load_chunk(const T* p) {
    Chunk<T, VEC> c;
    if constexpr (VEC) {
        typedef u32x4_t any __attribute__((aligned(1)));
        c.v = *reinterpret_cast<const any*>(p);
    } else {
        c.v = *p;
    }
    return c;
}
template <typename T, bool VEC>
__device__ inline void store_chunk(T* p, const Chunk<T, VEC>& c) {
    if constexpr (VEC) {
        typedef u32x4_t any __attribute__((aligned(1)));
        __builtin_nontemporal_store(c.v, reinterpret_cast<any*>(p));
    } else {
        *p = c.v;
    }
}
__device__ inline float as_float(float v) { return v; }
__device__ inline float as_float(bf16_t v) { return bf16_to_f32(v.bits); }
__device__ inline float as_float(__half v) { return __half2float(v); }
template <typename T, bool VEC>
__device__ inline void floats_of(const Chunk<T, VEC>& c, float (&f)[Chunk<T, VEC>::n]) {
    if constexpr (!VEC) {
        f[0] = as_float(c.v);
    } else {
        T e[Chunk<T, VEC>::n];
        __builtin_memcpy(e, &c.v, 16);
#pragma unroll
        for (int i = 0; i < Chunk<T, VEC>::n; ++i) f[i] = as_float(e[i]);
    }
}
template <bool VEC>
__device__ inline Chunk<float, VEC> chunk_of(const float (&f)[Chunk<float, VEC>::n], float*) {
    Chunk<float, VEC> c;
    __builtin_memcpy(&c.v, f, sizeof(c.v));
    return c;
}
template <bool VEC>
__device__ inline Chunk<bf16_t, VEC> chunk_of(const float (&f)[Chunk<bf16_t, VEC>::n], bf16_t*) {
    Chunk<bf16_t, VEC> c;
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c.v[i] = f32x2_to_bf16(f[2 * i], f[2 * i + 1]);
    } else {
        c.v.bits = static_cast<uint16_t>(f32_to_bf16(f[0]));
    }
    return c;
}
template <bool VEC>
__device__ inline Chunk<__half, VEC> chunk_of(const float (&f)[Chunk<__half, VEC>::n], __half*) {
    Chunk<__half, VEC> c;
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 two = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            uint32_t bits;
            __builtin_memcpy(&bits, &two, 4);
            c.v[i] = bits;
        }
    } else {
        c.v = __float2half_rn(f[0]);
    }
    return c;
}
template <typename T, bool VEC>
__device__ inline Chunk<T, VEC> zero_chunk() {
    Chunk<T, VEC> c;
    __builtin_memset(&c, 0, sizeof(c));
    return c;
}

constexpr int kAtOnce = 4;          // chunks of a row that a lane has in flight
constexpr int kRowThreads = 256;

// Which token and which columns this lane has: the group's token, and chunks first, first + lanes, ... of kAtOnce.
struct Task {
    int64_t token;
    int first, lanes;
    bool on;
};
__device__ inline Task task_of(const RowArgs& a) {
    const uint32_t wave = blockIdx.x * (kRowThreads / kWave) + threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const uint32_t step = fd_div(wave, a.groups), group = wave - step * a.groups.div;
    const int lanes = 1 << a.lanes_log2;
    Task t;
    t.token = static_cast<int64_t>(step) * (kWave >> a.lanes_log2) + (lane >> a.lanes_log2);
    t.lanes = lanes, t.first = static_cast<int>(group) * lanes * kAtOnce + (lane & (lanes - 1));
    t.on = t.token < a.tokens;
    return t;
}
// First element of chunk c, which ends with the row at the latest.
template <int N>
__device__ inline int start_of(int c, int cols) {
    const int at = c * N;
    return at + N <= cols ? at : cols - N;
}

template <typename T, bool VEC>
__global__ __launch_bounds__(kRowThreads) void sort_rows(const RowArgs a) {
    constexpr int N = Chunk<T, VEC>::n;
    const Task task = task_of(a);
    if (!task.on) return;
    const int held = *a.held;
    const T* const x = static_cast<const T*>(a.in) + task.token * a.ld_in;
    Chunk<T, VEC> c[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
        const int at = task.first + u * task.lanes;
        if (at < a.vectors) c[u] = load_chunk<T, VEC>(x + start_of<N>(at, a.cols));
    }
    const float scale = a.scales && task.first == 0 ? a.scales[task.token] : 0.f;
    for (int j = 0; j < a.chosen; ++j) {
        const int to = a.place[task.token * a.chosen + j];
        if (static_cast<uint32_t>(to) >= a.slots) continue;
        const bool here = to < held;
        T* const out = static_cast<T*>(a.out) + static_cast<int64_t>(to) * a.cols;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int at = task.first + u * task.lanes;
            if (at < a.vectors) store_chunk<T, VEC>(out + start_of<N>(at, a.cols), here ? c[u] : zero_chunk<T, VEC>());
        }
        if (a.scales && task.first == 0) a.out_scales[to] = here ? scale : 0.f;
    }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(kRowThreads) void combine_rows(const RowArgs a) {
    constexpr int N = Chunk<T, VEC>::n;
    const Task task = task_of(a);
    if (!task.on) return;
    const int held = *a.held;
    float sum[kAtOnce][N];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) sum[u][e] = 0.f;
    for (int j = 0; j < a.chosen; ++j) {
        const int64_t slot = task.token * a.chosen + j;
        const int from = a.place[slot];
        if (from >= held || static_cast<uint32_t>(from) >= a.slots) continue;
        const float weight = a.weights ? a.weights[slot] : 1.f;
        const T* const y = static_cast<const T*>(a.y) + from * a.ld_y;
        Chunk<T, VEC> c[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int at = task.first + u * task.lanes;
            if (at < a.vectors) c[u] = load_chunk<T, VEC>(y + start_of<N>(at, a.cols));
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            float f[N];
            floats_of<T, VEC>(c[u], f);
#pragma unroll
            for (int e = 0; e < N; ++e) sum[u][e] += weight * f[e];
        }
    }
    T* const out = static_cast<T*>(a.out) + task.token * a.cols;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
        const int at = task.first + u * task.lanes;
        if (at < a.vectors) store_chunk<T, VEC>(out + start_of<N>(at, a.cols), chunk_of<VEC>(sum[u], static_cast<T*>(nullptr)));
    }
}

// A group of lanes has a token's whole row, kAtOnce chunks at a time.
template <typename T, bool VEC>
__global__ __launch_bounds__(kRowThreads) void combine_rows_backward(const RowArgs a) {
    constexpr int N = Chunk<T, VEC>::n;
    Task task = task_of(a);
    const int held = *a.held;
    const int64_t token = task.on ? task.token : 0;
    const T* const dout = static_cast<const T*>(a.in) + token * a.ld_in;
    for (int j = 0; j < a.chosen; ++j) {
        const int64_t slot = token * a.chosen + j;
        const int at_row = a.place[slot];
        const bool row = static_cast<uint32_t>(at_row) < a.slots, here = row && at_row < held;
        const float weight = here ? a.weights[slot] : 0.f;
        const T* const y = static_cast<const T*>(a.y) + (a.dweights && here ? at_row * a.ld_y : 0);
        T* const dy = static_cast<T*>(a.dy) + (row ? static_cast<int64_t>(at_row) * a.cols : 0);
        float dot = 0.f;
        for (int c0 = task.first; task.on && c0 < a.vectors; c0 += kAtOnce * task.lanes) {
            Chunk<T, VEC> g[kAtOnce], v[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int at = c0 + u * task.lanes;
                if (at < a.vectors) g[u] = load_chunk<T, VEC>(dout + start_of<N>(at, a.cols));
                if (at < a.vectors && a.dweights && here) v[u] = load_chunk<T, VEC>(y + start_of<N>(at, a.cols));
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int at = c0 + u * task.lanes;
                if (at >= a.vectors) continue;
                float f[N];
                floats_of<T, VEC>(g[u], f);
                if (a.dweights && here) {
                    float e[N];
                    floats_of<T, VEC>(v[u], e);
                    const int twice = at * N + N > a.cols ? at * N + N - a.cols : 0;   // elements of the chunk before it
#pragma unroll
                    for (int i = 0; i < N; ++i) dot += i >= twice ? f[i] * e[i] : 0.f;
                }
                if (a.dy && row) {
#pragma unroll
                    for (int i = 0; i < N; ++i) f[i] = here ? f[i] * weight : 0.f;
                    store_chunk<T, VEC>(dy + start_of<N>(at, a.cols), chunk_of<VEC>(f, static_cast<T*>(nullptr)));
                }
            }
        }
        if (a.dweights) {
            for (int d = 1; d < task.lanes; d <<= 1) dot += __shfl_xor(dot, d);
            if (task.on && task.first == 0) a.dweights[slot] = here ? dot : 0.f;
        }
    }
}

// The grid and the row's division; a wavefront has whole rows if `whole`.  0 or a refusal.
int lay_out(const char* who, RowArgs& a, int per, bool whole, int64_t& blocks) {
    a.vectors = (a.cols + per - 1) / per;
    a.lanes_log2 = 0;
    while (a.lanes_log2 < 6 && (1 << a.lanes_log2) < a.vectors) ++a.lanes_log2;
    const int lanes = 1 << a.lanes_log2;
    const int groups = whole ? 1 : (a.vectors + lanes * kAtOnce - 1) / (lanes * kAtOnce);
    a.groups = make_fastdiv(static_cast<uint32_t>(groups));
    const int64_t side = kWave >> a.lanes_log2, steps = (a.tokens + side - 1) / side;
    if (steps > (0x7FFFFFFFll - 8) / groups) return fail(DDL_E_UNSUPP, "%s: %lld tokens of %d columns are more than 2^31 wavefronts", who, static_cast<long long>(a.tokens), a.cols);
    blocks = (steps * groups + kRowThreads / kWave - 1) / (kRowThreads / kWave);
    if (blocks * kRowThreads > 0xFFFFFFFFll) return fail(DDL_E_UNSUPP, "%s: %lld tokens of %d columns are more than 2^32 threads", who, static_cast<long long>(a.tokens), a.cols);
    return 0;
}

int check_tokens(const char* who, int64_t tokens, int64_t chosen, int64_t cols) {
    if (tokens < 0 || chosen < 0 || cols < 1)
        return fail(DDL_E_ARG, "%s: %lld tokens of %lld choices, rows of %lld columns", who, static_cast<long long>(tokens), static_cast<long long>(chosen), static_cast<long long>(cols));
    if (cols > 0x3FFFFFFF || chosen > 0x7FFFFFFF || (chosen && tokens > 0x40000000 / chosen) || tokens > 0x40000000)
        return fail(DDL_E_UNSUPP, "%s: more than 2^30 slots or columns", who);
    return 0;
}

// fn(element pointer, whether rows are vectors) for elements of `bytes` that are only moved, or of `dtype`.
template <typename Fn>
int with_moved(int bytes, int64_t cols, Fn&& fn) {
    switch (bytes) {
        case 1: return cols >= 16 ? fn(static_cast<uint8_t*>(nullptr), std::true_type{}) : fn(static_cast<uint8_t*>(nullptr), std::false_type{});
        case 2: return cols >= 8 ? fn(static_cast<uint16_t*>(nullptr), std::true_type{}) : fn(static_cast<uint16_t*>(nullptr), std::false_type{});
        default: return cols >= 4 ? fn(static_cast<uint32_t*>(nullptr), std::true_type{}) : fn(static_cast<uint32_t*>(nullptr), std::false_type{});
    }
}
template <typename Fn>
int with_added(int dtype, int64_t cols, Fn&& fn) {
    int rc = 0;
    with_ln_element(dtype, [&](auto* p) {
        rc = cols >= static_cast<int64_t>(16 / sizeof(*p)) ? fn(p, std::true_type{}) : fn(p, std::false_type{});
    });
    return rc;
}

// Slots of a workgroup of the plan: a whole number of wavefronts for each of its own.
int64_t part_of(int64_t slots) {
    const int64_t least = (slots + kPlanThreads - 1) / kPlanThreads, rest = (least + kMostParts - 1) / kMostParts;
    return kPlanThreads * (slots <= kAlone ? (least > 0 ? least : 1) : rest);
}

int check_dtype(const char* who, int dtype) {
    return dtype == DDL_DT_F32 || dtype == DDL_DT_BF16 || dtype == DDL_DT_F16 ? 0 : fail(DDL_E_ARG, "%s: dtype %d", who, dtype);
}

}  // namespace
}  // namespace ddl

extern "C" {

int64_t ddl_expert_plan_workspace(int64_t slots, int64_t held_experts) {
    if (slots <= ddl::kAlone || slots > 0x40000000 || held_experts < 0 || held_experts > ddl::kMaxHeld) return 0;
    const int64_t part = ddl::part_of(slots);
    return (slots + part - 1) / part * (held_experts + 1);
}

int ddl_expert_plan(const void* ids, int id_bytes, int64_t tokens, int64_t chosen, int64_t ld_ids, int64_t low, int64_t high, int32_t* place, int32_t* offsets,
                    int32_t* workspace, int64_t workspace_elems, void* stream) {
    using namespace ddl;
    if (int rc = check_tokens("ddl_expert_plan", tokens, chosen, 1)) return rc;
    if (id_bytes != 4 && id_bytes != 8) return fail(DDL_E_ARG, "ddl_expert_plan: numbers of %d bytes", id_bytes);
    if (high < low || low < 0) return fail(DDL_E_ARG, "ddl_expert_plan: experts %lld to %lld", static_cast<long long>(low), static_cast<long long>(high));
    if (high - low > kMaxHeld) return fail(DDL_E_UNSUPP, "ddl_expert_plan: %lld experts (at most %d)", static_cast<long long>(high - low), kMaxHeld);
    const int64_t slots = tokens * chosen, need = ddl_expert_plan_workspace(slots, high - low);
    if (!offsets || (slots && (!ids || !place))) return fail(DDL_E_ARG, "ddl_expert_plan: null pointer");
    if (need && (!workspace || workspace_elems < need))
        return fail(DDL_E_ARG, "ddl_expert_plan: workspace of %lld int32, %lld are needed", static_cast<long long>(workspace ? workspace_elems : 0), static_cast<long long>(need));
    PlanArgs a{};
    a.ids = ids, a.id_bytes = id_bytes, a.ld_ids = ld_ids, a.low = low, a.slots = static_cast<int>(slots), a.held = static_cast<int>(high - low);
    a.chosen = make_fastdiv(static_cast<uint32_t>(chosen ? chosen : 1)), a.place = place, a.offsets = offsets, a.counts = workspace;
    while ((1 << a.bits) <= a.held) ++a.bits;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    a.part = static_cast<int>(part_of(slots));
    const uint32_t blocks = slots ? static_cast<uint32_t>((slots + a.part - 1) / a.part) : 1;
    const int count_bytes = kPlanWaves * (a.held + 1) * 4, lds_bytes = count_bytes + (a.held + 1 + kPlanWaves) * 4;
    static_assert((kPlanWaves + 1) * (kMaxHeld + 1) * 4 + kPlanWaves * 4 <= 160 * 1024, "the counters do not fit");
    if (lds_bytes > 64 * 1024) {   // what a launch gets without asking
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(expert_place), hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes);
        if (e != hipSuccess) return fail(static_cast<int>(e), "ddl_expert_plan: cannot reserve %d bytes of LDS: %s", lds_bytes, hipGetErrorString(e));
    }
    if (blocks > 1) {
        hipLaunchKernelGGL(expert_count, dim3(blocks), dim3(kPlanThreads), count_bytes, s, a);
        if (int rc = check_launch("ddl_expert_plan")) return rc;
    }
    hipLaunchKernelGGL(expert_place, dim3(blocks), dim3(kPlanThreads), lds_bytes, s, a);
    return check_launch("ddl_expert_plan");
}

int ddl_expert_sort(const void* x, int elem_bytes, int64_t tokens, int64_t chosen, int64_t cols, int64_t ld_x, const int32_t* place, const int32_t* held,
                    void* out, const float* scales, float* out_scales, void* stream) {
    using namespace ddl;
    if (int rc = check_tokens("ddl_expert_sort", tokens, chosen, cols)) return rc;
    if (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4) return fail(DDL_E_ARG, "ddl_expert_sort: elements of %d bytes", elem_bytes);
    if (tokens == 0 || chosen == 0) return 0;
    if (!x || !place || !held || !out || (scales && !out_scales)) return fail(DDL_E_ARG, "ddl_expert_sort: null pointer");
    if (tokens > 1 && ld_x < cols) return fail(DDL_E_ARG, "ddl_expert_sort: pitch below %lld columns", static_cast<long long>(cols));
    RowArgs a{};
    a.in = x, a.out = out, a.scales = scales, a.out_scales = out_scales, a.place = place, a.held = held, a.ld_in = ld_x, a.tokens = tokens;
    a.slots = static_cast<uint32_t>(tokens * chosen), a.chosen = static_cast<int>(chosen), a.cols = static_cast<int>(cols);
    return with_moved(elem_bytes, cols, [&](auto* e, auto vec) {
        typedef std::remove_pointer_t<decltype(e)> T;
        constexpr bool VEC = decltype(vec)::value;
        int64_t blocks;
        if (int rc = lay_out("ddl_expert_sort", a, Chunk<T, VEC>::n, false, blocks)) return rc;
        hipLaunchKernelGGL((sort_rows<T, VEC>), dim3(static_cast<uint32_t>(blocks)), dim3(kRowThreads), 0, static_cast<hipStream_t>(stream), a);
        return check_launch("ddl_expert_sort");
    });
}

int ddl_expert_combine(const void* y, int dtype, int64_t tokens, int64_t chosen, int64_t cols, int64_t ld_y, const int32_t* place, const int32_t* held,
                       const float* weights, void* out, void* stream) {
    using namespace ddl;
    if (int rc = check_dtype("ddl_expert_combine", dtype)) return rc;
    if (int rc = check_tokens("ddl_expert_combine", tokens, chosen, cols)) return rc;
    if (tokens == 0) return 0;
    if (!out || !held || (chosen && (!y || !place))) return fail(DDL_E_ARG, "ddl_expert_combine: null pointer");
    if (tokens * chosen > 1 && ld_y < cols) return fail(DDL_E_ARG, "ddl_expert_combine: pitch below %lld columns", static_cast<long long>(cols));
    RowArgs a{};
    a.y = y, a.out = out, a.weights = weights, a.place = place, a.held = held, a.ld_y = ld_y, a.tokens = tokens;
    a.slots = static_cast<uint32_t>(tokens * chosen), a.chosen = static_cast<int>(chosen), a.cols = static_cast<int>(cols);
    return with_added(dtype, cols, [&](auto* e, auto vec) {
        typedef std::remove_pointer_t<decltype(e)> T;
        constexpr bool VEC = decltype(vec)::value;
        int64_t blocks;
        if (int rc = lay_out("ddl_expert_combine", a, Chunk<T, VEC>::n, false, blocks)) return rc;
        hipLaunchKernelGGL((combine_rows<T, VEC>), dim3(static_cast<uint32_t>(blocks)), dim3(kRowThreads), 0, static_cast<hipStream_t>(stream), a);
        return check_launch("ddl_expert_combine");
    });
}

int ddl_expert_combine_backward(const void* dout, const void* y, int dtype, int64_t tokens, int64_t chosen, int64_t cols, int64_t ld_dout, int64_t ld_y,
                                const int32_t* place, const int32_t* held, const float* weights, void* dy, float* dweights, void* stream) {
    using namespace ddl;
    if (int rc = check_dtype("ddl_expert_combine_backward", dtype)) return rc;
    if (int rc = check_tokens("ddl_expert_combine_backward", tokens, chosen, cols)) return rc;
    if (tokens == 0 || chosen == 0 || (!dy && !dweights)) return 0;
    if (!dout || !place || !held || !weights || (dweights && !y)) return fail(DDL_E_ARG, "ddl_expert_combine_backward: null pointer");
    if ((tokens > 1 && ld_dout < cols) || (dweights && tokens * chosen > 1 && ld_y < cols))
        return fail(DDL_E_ARG, "ddl_expert_combine_backward: pitch below %lld columns", static_cast<long long>(cols));
    RowArgs a{};
    a.in = dout, a.y = y, a.dy = dy, a.weights = weights, a.dweights = dweights, a.place = place, a.held = held, a.ld_in = ld_dout, a.ld_y = ld_y;
    a.tokens = tokens, a.slots = static_cast<uint32_t>(tokens * chosen), a.chosen = static_cast<int>(chosen), a.cols = static_cast<int>(cols);
    return with_added(dtype, cols, [&](auto* e, auto vec) {
        typedef std::remove_pointer_t<decltype(e)> T;
        constexpr bool VEC = decltype(vec)::value;
        int64_t blocks;
        if (int rc = lay_out("ddl_expert_combine_backward", a, Chunk<T, VEC>::n, true, blocks)) return rc;
        hipLaunchKernelGGL((combine_rows_backward<T, VEC>), dim3(static_cast<uint32_t>(blocks)), dim3(kRowThreads), 0, static_cast<hipStream_t>(stream), a);
        return check_launch("ddl_expert_combine_backward");
    });
}

}  // extern "C"
