// Adjoint of attention.hip: with p_ij of the forward (formed anew from the scores and each row's sum), dO the gradient of out and
//   D_i = sum of dO_i out_i,   dS_ij = p_ij (dO_i . v_j - D_i):
//   dq_i = scale sum over j of dS_ij k_j,   dk_j = scale sum over i of dS_ij q_i,   dv_j = sum over i of p_ij dO_i
//
// Two kernels, so that every sum has one owner and one order and nothing is added atomically, at the price of forming the
// scores and dO . v twice (seven products instead of five): attention_backward_rows, a wavefront for 32 queries that walks over
// the keys, and attention_backward_keys, a wavefront for 32 keys that walks over the queries of all heads that share
// them -- the gradient of a shared key head is summed there, in registers (attention_backward_pairs: the same by two wavefronts).
//
// 16-bit types: dS is rounded for the product (gradients are then off by 1.4 times what rounding the exact ones gives).  D comes from out and the rest
// that the forward kept, or, where all keys are in one tile, from p and dP themselves; from the rounded out alone the gradients of a
// query with four keys were off by 2.4 times as much, with 200 keys by 1.6.
#include "ddl_common.h"

#include "attention_parts.h"

namespace ddl {
namespace {

template <typename T>
constexpr int tile_rows() { return sizeof(T) == 2 ? 64 : 32; }

template <int N>
__device__ inline void clear(floatx16 (&acc)[N]) {
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
}

__device__ inline float chunk_dot(const floatx4v& a, const floatx4v& b, const float*) { return (a[0] * b[0] + a[1] * b[1]) + (a[2] * b[2] + a[3] * b[3]); }
template <typename T>
__device__ inline float chunk_dot(const shortx8& a, const shortx8& b, const T*) {
    float s = 0.f;
    T x[8], y[8];
    __builtin_memcpy(x, &a, 16);
    __builtin_memcpy(y, &b, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += load1(&x[i]) * load1(&y[i]);
    return s;
}

// dS in fp16, which has steps down to 2^-24 and values up to 2^16: gradients of 10^-5 would be lost over some thousand keys, and those of 10^5 infinite.  So a
// column's dS are multiplied by a power of two, `up`, with which the largest so far is below 2^15, and its sum is with it; the factor only
// falls, where a larger dS comes, and then to where that one is below 2^10.  The other types have the range of 32 bits and need none.
// ([4,4096,16,64] fp16 forward and adjoint 1500 us instead of 1382 without, head size 128: 2690 and 2490; with the largest found while the matrix cores are
// busy, before the look, 1540 and 2720.)
template <typename T>
struct Fitted {
    static constexpr bool kNeeded = false;
    template <int N>
    __device__ void fit(floatx16&, floatx16 (&)[N]) {}
    template <int N>
    __device__ void undo(floatx16 (&)[N]) {}
};
template <>
struct Fitted<__half> {
    static constexpr bool kNeeded = true;
    float up = 0x1p100f;      // of this lane's column: both halves of the lanes have the same

    static __device__ int exponent(float power) { return __builtin_amdgcn_frexp_expf(power) - 1; }
    template <int N>
    static __device__ void scale(floatx16 (&acc)[N], float factor) {
#pragma unroll
        for (int d = 0; d < N; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] *= factor;
    }
    // Multiplies these dS; moved(factor): so is what they are added to.
    template <typename Fn>
    __device__ void look(floatx16& d, Fn&& moved) {
        float m = fmaxf(fabsf(d[0]), fabsf(d[1]));
#pragma unroll
        for (int r = 2; r < 16; ++r) m = fmaxf(m, fabsf(d[r]));
        m = max_halves(m);
        if (__any(m * up > 32768.f)) {
            const int was = exponent(up), to = m * up > 32768.f ? min(10 - __builtin_amdgcn_frexp_expf(m), was) : was;
            up = ldexpf(1.f, to);
            moved(ldexpf(1.f, to - was));
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) d[r] *= up;
    }
    template <int N>
    __device__ void fit(floatx16& d, floatx16 (&acc)[N]) {
        look(d, [&](float factor) { scale(acc, factor); });
    }
    // The same where another wavefront has multiplied them, by `given`.
    template <int N>
    __device__ void take_over(float given, floatx16 (&acc)[N]) {
        if (__any(given != up)) {
            scale(acc, ldexpf(1.f, exponent(given) - exponent(up)));
            up = given;
        }
    }
    template <int N>
    __device__ void undo(floatx16 (&acc)[N]) { scale(acc, ldexpf(1.f, -exponent(up))); }
};

// A column's row of a tensor as the straight product takes it; zeros where `there` is false.
template <typename T, int DP, typename Frag>
__device__ inline void load_column(Frag* column, const T* row, bool there, int chunks, int side) {
    typedef AttnTile<T, DP> Tile;
#pragma unroll
    for (int s = 0; s < Tile::kSteps; ++s) {
        Frag f = {};
        if (there && 2 * s + side < chunks) f = *reinterpret_cast<const Frag*>(row + (2 * s + side) * Tile::kPerChunk);
        column[s] = f;
    }
}

// dq of 32 queries a wavefront, 128 a workgroup, tiles of keys and values through LDS as in attention_rows; and their D.
// [4,4096,16,128] bf16, all keys: 717 us (1150 TFLOP/s for three products), head size 64: 414, causal [4,2048,8,128] 72; fp16 800 and 477.  Bound by the matrix
// cores (62 % busy) and the vector work that does not fit next to them.
// Where there are few blocks of queries, `splits` workgroups share the keys of one and leave sums in fp32.
// ONE (16-bit types): all keys are in one tile, D from them.
template <typename T, int DP, bool ONE>
__global__ __launch_bounds__(kThreads, DP * sizeof(T) > 256 ? 1 : 2) void attention_backward_rows(const AttnArgs a) {
    typedef AttnTile<T, DP> Tile;
    typedef typename Tile::Frag Frag;
    constexpr int KEYS = tile_rows<T>(), NS = KEYS / 32, kTileBytes = KEYS * Tile::kRowBytes;
    extern __shared__ __align__(16) char lds[];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave), half = lane >> 5;
    const int split = blockIdx.y;
    int u, block, batch, head;
    bool late;
    block_of(blockIdx.x, a.batch * a.heads, a.blocks, a.folded, u, block, late);
    head_of(a, u, a.heads, a.group, late, batch, head);
    const int bh = batch * a.heads + head, kv_head = head / a.group;
    const int length = sequence_keys(a, batch);
    const int first_row = block * kRows * kWaves, wave_row = first_row + wave * kRows, my_row = wave_row + (lane & 31);
    const bool mine = my_row < a.tokens;
    const int seen = keys_seen(a, my_row, length);
    auto scalar = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const int end = scalar(keys_seen(a, min(first_row + kRows * kWaves, a.tokens) - 1, length));
    const int wave_most = scalar(wave_row < a.tokens ? keys_seen(a, min(wave_row + kRows, a.tokens) - 1, length) : 0);
    const int wave_least = scalar(keys_seen(a, wave_row, length));
    const T* k = static_cast<const T*>(a.k) + batch * a.k_at.batch + kv_head * a.k_at.head;
    const T* v = static_cast<const T*>(a.v) + batch * a.v_at.batch + kv_head * a.v_at.head;
    Tile tile(lds, lane);
    const int tiles = (end + KEYS - 1) / KEYS, share = scalar(tiles / a.splits), more = tiles - share * a.splits;
    const int t0 = share * split + min(split, more), t1 = t0 + share + (split < more ? 1 : 0), limit = min(end, t1 * KEYS);
    const AttnCopy<T, DP, KEYS, kWaves, (DP > 96)> k_copy(k, a.k_at.token, a.chunks, wave, lane), v_copy(v, a.v_at.token, a.chunks, wave, lane);
    auto request = [&](int t, int set) {
        const char* to = lds + set;
        k_copy.request(to, t * KEYS, limit), v_copy.request(to + 2 * kTileBytes, t * KEYS, limit);
    };
    if (ONE || a.dq) request(t0, 0);
    Frag q_column[Tile::kSteps], g_column[Tile::kSteps];
    load_column<T, DP>(q_column, static_cast<const T*>(a.q) + batch * a.q_at.batch + my_row * a.q_at.token + head * a.q_at.head, mine, a.chunks, half);
    load_column<T, DP>(g_column, static_cast<const T*>(a.dout) + batch * a.dout_at.batch + my_row * a.dout_at.token + head * a.dout_at.head, mine, a.chunks, half);
    float delta = 0.f, lse = INFINITY;
    const int64_t stat = static_cast<int64_t>(bh) * a.tokens + my_row;
    if (mine) lse = a.lse[stat];
    constexpr uint32_t kK = 0, kV = 2 * kTileBytes, kNext = 32 * Tile::kRowBytes;
    if constexpr (ONE) {
        wait_for_copies();
        lds_barrier();
#pragma unroll 1
        for (int n = 0; 32 * n < wave_most; ++n) {
            floatx16 s[2];
            clear(s);
            tile.straight(s[0], kK, n, q_column);
            tile.straight(s[1], kV, n, g_column);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r], a.scale_log2, -lse));
                if (32 * n + (r & 3) + 8 * (r >> 2) < seen - 4 * half) delta = __builtin_fmaf(p, s[1][r], delta);
            }
        }
    } else {
        const int64_t row = batch * a.out_at.batch + my_row * a.out_at.token + head * a.out_at.head;
        for (const void* of : {static_cast<const void*>(a.out), static_cast<const void*>(a.rest)}) {
            if (!of) continue;
            Frag o_column[Tile::kSteps];
            load_column<T, DP>(o_column, static_cast<const T*>(of) + row, mine, a.chunks, half);
#pragma unroll
            for (int s = 0; s < Tile::kSteps; ++s) delta += chunk_dot(g_column[s], o_column[s], static_cast<const T*>(nullptr));
        }
    }
    delta = add_halves(delta);
    if (mine && half == 0 && split == 0) a.delta[stat] = delta;
    if (!a.dq) return;      // D alone
    floatx16 acc[Tile::kBlocks];
    clear(acc);
    Fitted<T> fitted;
    int set = 0;      // of tiles: the first or the second
    for (int t = t0; t < t1; ++t) {
        wait_for_copies();
        lds_barrier();
        // Behind the first product where there is other work as well: in front of it the kernel spills with DP = 128, and what it reads back waits for
        // these copies (dq of [4,4096,16,128] bf16 785 us instead of 717, of [4,2048,8,128] causal 82 instead of 71).
        auto ask = [&] { request(t + 1, kTileBytes - set); };
        bool done = t * KEYS >= wave_most, asked = false;
        if constexpr (sizeof(T) == 2 && NS == 2 && !ONE) {
            if (!done && (t + 1) * KEYS <= wave_least) {     // 64 keys that all see: the vector units are at 32 of them while the matrix cores are at others
                done = asked = true;
                floatx16 p0, p1, d0, d1;
#pragma unroll
                for (int r = 0; r < 16; ++r) p0[r] = p1[r] = d0[r] = d1[r] = 0.f;
                auto exponential = [&](floatx16& p) {
                    return [&](int r) { p[r] = pinned(__builtin_amdgcn_exp2f(__builtin_fmaf(p[r], a.scale_log2, -lse))); };
                };
                auto difference = [&](floatx16& d, const floatx16& p) {
                    return [&](int r) { d[r] = pinned(p[r] * (d[r] - delta)); };
                };
                auto nothing = [](int) {};
                tile.template straight_woven<0>(p0, kK, q_column, nothing);
                ask();
                tile.template straight_woven<16>(d0, kV, g_column, exponential(p0));
                tile.template straight_woven<16>(p1, kK + kNext, q_column, difference(d0, p0));
                fitted.fit(d0, acc);
                const typename Tile::Packed first = Tile::pack(d0);
                tile.template straight_woven<16>(d1, kV + kNext, g_column, exponential(p1));
                tile.template transposed_woven<16>(acc, kK, first, difference(d1, p1));
                fitted.fit(d1, acc);
                tile.template transposed_woven<0>(acc, kK + kNext, Tile::pack(d1), nothing);
            }
        }
        if (!asked) ask();
        if (!done) {
            const bool masked = (t + 1) * KEYS > wave_least;
            const int rest = seen - t * KEYS - 4 * half;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                floatx16 s[2];
                clear(s);
                tile.straight(s[0], kK, n, q_column);
                tile.straight(s[1], kV, n, g_column);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r], a.scale_log2, -lse));
                    if (masked) p = 32 * n + (r & 3) + 8 * (r >> 2) < rest ? p : 0.f;
                    s[0][r] = p * (s[1][r] - delta);
                }
                fitted.fit(s[0], acc);
                tile.transposed(acc, kK, n, Tile::pack(s[0]));
            }
        }
        tile.shift(kTileBytes - 2 * set), set = kTileBytes - set;
    }
    fitted.undo(acc);
    wait_for_copies();
    lds_barrier();
    if (a.splits > 1) {
        typedef AttnOut<float, DP> Out;
        char* room = lds + wave * Out::kRoom;
        Out::park(room, acc, a.scale, lane);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int dim = a.chunks * Tile::kPerChunk;
        float* to = a.partial + (static_cast<int64_t>(split) * a.batch * a.heads + bh) * a.tokens * dim;
        Out::write(room, dim / 4, lane, [&](int col) -> float* { return wave_row + col < a.tokens ? to + static_cast<int64_t>(wave_row + col) * dim : nullptr; });
        return;
    }
    typedef AttnOut<T, DP> Out;
    char* room = lds + wave * Out::kRoom;
    Out::park(room, acc, a.scale, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    T* dq = static_cast<T*>(a.dq) + batch * a.dq_at.batch + head * a.dq_at.head;
    Out::write(room, a.chunks, lane, [&](int col) -> T* { return wave_row + col < a.tokens ? dq + (wave_row + col) * a.dq_at.token : nullptr; });
}

// dq from the splits' sums, in their order: four elements a thread.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_backward_rows_join(const AttnArgs a) {
    const int quads = a.chunks * AttnElem<T>::kPerChunk / 4;
    const int64_t all = static_cast<int64_t>(a.batch) * a.heads * a.tokens * quads, at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (at >= all) return;
    const float4* p = reinterpret_cast<const float4*>(a.partial) + at;
    float4 sum = p[0];
    for (int s = 1; s < a.splits; ++s) {
        const float4 more = p[all * s];
        sum.x += more.x, sum.y += more.y, sum.z += more.z, sum.w += more.w;
    }
    const int64_t row = at / quads;
    const int d = 4 * static_cast<int>(at - row * quads), bh = static_cast<int>(row / a.tokens), token = static_cast<int>(row - static_cast<int64_t>(bh) * a.tokens);
    const int batch = bh / a.heads, head = bh - batch * a.heads;
    store_piece<true>(static_cast<T*>(a.dq) + batch * a.dq_at.batch + token * a.dq_at.token + head * a.dq_at.head + d, sum);
}

constexpr int kPairRows = 64;
constexpr int kHandedBytes = 2 * kWaves * 4 * 16 * kWave;      // probabilities and dS of 64 queries and 128 keys, 16 bytes a lane and piece
template <typename T, int DP>
constexpr int query_tile() { return sizeof(T) == 2 || AttnTile<T, DP>::kRowBytes <= 128 ? 64 : 32; }

// Probabilities of many keys are small, and fp16 has full steps down to 2^-14 only: they are formed as 2^kUp times as much, from sums that are less by kUp,
// and so are the sums of dv and, next to Fitted's factor, dk.  (A probability is at most one; the rest of the range is for large scores, whose sums are
// off by their rounding.)
template <typename T>
constexpr int kUp = Fitted<T>::kNeeded ? 10 : 0;

// Which queries a wavefront's 32 keys are seen by, and which of them, ROWS of one head at a time, are this workgroup's share.
template <int ROWS>
struct QueriesOfKeys {
    int wave_key, my_key;
    int need;                      // first query that sees this lane's key
    int wave_need, wave_all;       // first one that sees any of the wavefront's, and from where on they see all
    int first_tile, head_tiles;    // of a head, for the workgroup
    int it0, it1;                  // its share of all heads' tiles
    __device__ QueriesOfKeys(const AttnArgs& a, int first_key, int wave, int lane, int length, int split) {
        auto scalar = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
        wave_key = first_key + wave * kRows, my_key = wave_key + (lane & 31);
        const int shift = a.causal ? causal_shift(a, length) : 0x3FFFFFFF;      // query i sees key j from i = j - shift on
        need = my_key < length ? max(my_key - shift, 0) : 0x7FFFFFFF;
        const int block_need = scalar(first_key < length ? max(first_key - shift, 0) : a.tokens);
        wave_need = scalar(wave_key < length ? max(wave_key - shift, 0) : 0x7FFFFFFF);
        wave_all = scalar(wave_key + kRows <= length ? max(wave_key + kRows - 1 - shift, 0) : 0x7FFFFFFF);
        first_tile = min(block_need, a.tokens) / ROWS, head_tiles = block_need < a.tokens ? (a.tokens + ROWS - 1) / ROWS - first_tile : 0;
        const int64_t all = static_cast<int64_t>(head_tiles) * a.group;
        it0 = static_cast<int>(all * split / a.splits), it1 = static_cast<int>(all * (split + 1) / a.splits);
    }
    struct At {                    // an iteration's head of the group and tile
        int head, tile;
    };
    __device__ At start() const {
        At at{0, 0};
        if (it0 < it1) at.head = it0 / head_tiles, at.tile = it0 - at.head * head_tiles;
        return at;
    }
    __device__ At after(At at) const {
        if (++at.tile == head_tiles) at.tile = 0, ++at.head;
        return at;
    }
};

// Row values (sums or D) of the rows that this half of the lanes holds, four at a time, the next four on their way.
struct OfRows {
    const float* at;
    floatx4v now, next;
    __device__ explicit OfRows(const float* rows) : at(rows), next(*reinterpret_cast<const floatx4v*>(rows)) {}
    __device__ float operator()(int r) {
        if (r % 4 == 0) {
            now = next;
            if (r < 12) next = *reinterpret_cast<const floatx4v*>(at + 2 * (r + 4));
        }
        return now[r % 4];
    }
};

// dk and dv of 32 keys a wavefront, 128 a workgroup; 32 or 64 queries of one head at a time through LDS, with their sums and D.  Where
// there are few blocks of keys, `splits` workgroups share the queries of one and leave sums in fp32.
// [4,4096,16,64] bf16: 565 us (before its two kinds of work were woven 703), fp16 655.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads, DP * sizeof(T) > 128 ? 1 : 2) void attention_backward_keys(const AttnArgs a) {
    typedef AttnTile<T, DP> Tile;
    typedef typename Tile::Frag Frag;
    constexpr int ROWS = query_tile<T, DP>(), NS = ROWS / 32;
    constexpr int kTileBytes = ROWS * Tile::kRowBytes, kSetBytes = 2 * kTileBytes + 2 * ROWS * 4;
    extern __shared__ __align__(16) char lds[];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave), half = lane >> 5;
    const int pairs = a.batch * a.kv_heads;
    int u, unit, batch, kv_head;
    bool late;
    block_of(blockIdx.x, pairs, a.blocks * a.splits, false, u, unit, late);
    head_of(a, u, a.kv_heads, 1, false, batch, kv_head);
    const int bk = batch * a.kv_heads + kv_head;
    unit = a.blocks * a.splits - 1 - unit;      // the first keys, which most queries see in the causal form, first
    const int block = unit / a.splits, split = unit - block * a.splits;
    const int length = sequence_keys(a, batch);
    const QueriesOfKeys<ROWS> see(a, block * kRows * kWaves, wave, lane, length, split);
    typedef typename QueriesOfKeys<ROWS>::At At;
    const int it0 = see.it0, it1 = see.it1, wave_key = see.wave_key, my_key = see.my_key;
    const T* q0 = static_cast<const T*>(a.q) + batch * a.q_at.batch + static_cast<int64_t>(kv_head) * a.group * a.q_at.head;
    const T* g0 = static_cast<const T*>(a.dout) + batch * a.dout_at.batch + static_cast<int64_t>(kv_head) * a.group * a.dout_at.head;
    const int64_t row0 = (static_cast<int64_t>(batch) * a.heads + static_cast<int64_t>(kv_head) * a.group) * a.tokens;
    Tile tile(lds, lane);
    AttnCopy<T, DP, ROWS, kWaves> q_copy(q0, a.q_at.token, a.chunks, wave, lane), g_copy(g0, a.dout_at.token, a.chunks, wave, lane);
    auto set_of = [&](int it) { return ((it - it0) & 1) * kSetBytes; };
    auto request = [&](int it, At at) {
        if (it >= it1) return;
        char* to = lds + set_of(it);
        q_copy.base = reinterpret_cast<const char*>(q0 + at.head * a.q_at.head), g_copy.base = reinterpret_cast<const char*>(g0 + at.head * a.dout_at.head);
        const int first = (see.first_tile + at.tile) * ROWS;
        q_copy.request(to, first, a.tokens), g_copy.request(to + kTileBytes, first, a.tokens);
    };
    float row_next = 0.f;       // of the queries on their way: threads 0 .. ROWS - 1 their sums, the next as many their D
    auto load_rows = [&](int it, At at) {
        if (it >= it1 || tid >= 2 * ROWS) return;
        const int row = (see.first_tile + at.tile) * ROWS + (tid & (ROWS - 1));
        const int64_t place = row0 + static_cast<int64_t>(at.head) * a.tokens + row;
        row_next = tid < ROWS ? (row < a.tokens ? a.lse[place] - kUp<T> : INFINITY) : (row < a.tokens ? a.delta[place] : 0.f);
    };
    auto store_rows = [&](int it) {
        if (it < it1 && tid < 2 * ROWS) reinterpret_cast<float*>(lds + set_of(it) + 2 * kTileBytes)[tid] = row_next;
    };
    At next = see.start(), now = next;
    request(it0, next);
    load_rows(it0, next), store_rows(it0);
    next = see.after(next);
    load_rows(it0 + 1, next);
    Frag k_column[Tile::kSteps], v_column[Tile::kSteps];
    const bool mine = my_key < length;
    load_column<T, DP>(k_column, static_cast<const T*>(a.k) + batch * a.k_at.batch + my_key * a.k_at.token + kv_head * a.k_at.head, mine, a.chunks, half);
    load_column<T, DP>(v_column, static_cast<const T*>(a.v) + batch * a.v_at.batch + my_key * a.v_at.token + kv_head * a.v_at.head, mine, a.chunks, half);
    floatx16 dk[Tile::kBlocks], dv[Tile::kBlocks];
    clear(dk), clear(dv);
    Fitted<T> fitted;      // (dk's)
    auto nothing = [](int) {};
    auto exponential = [&](floatx16& p, OfRows& lse) {
        return [&](int r) { p[r] = pinned(__builtin_amdgcn_exp2f(__builtin_fmaf(p[r], a.scale_log2, -lse(r)))); };
    };
    auto difference = [&](floatx16& d, const floatx16& p, OfRows& delta) {
        return [&](int r) { d[r] = pinned(p[r] * (d[r] - delta(r))); };
    };
    constexpr uint32_t kQ = 0, kG = kTileBytes, kNext = 32 * Tile::kRowBytes;
    auto zero = [](floatx16& v) {
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = 0.f;
    };
    // 32 queries, some of which (`masked`) may not see some of the wavefront's keys.
    auto block_step = [&](int n, int first, const float* rows, bool masked) {
        floatx16 p, d;
        zero(p), zero(d);
        tile.straight(p, kQ, n, k_column);
        tile.straight(d, kG, n, v_column);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const floatx4v lse = *reinterpret_cast<const floatx4v*>(rows + 32 * n + 8 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) p[4 * g + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[4 * g + i], a.scale_log2, -lse[i]));
        }
        if (masked) {
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r] = first + 32 * n + 4 * half + (r & 3) + 8 * (r >> 2) >= see.need ? p[r] : 0.f;
        }
        tile.transposed(dv, kG, n, Tile::pack(p));
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const floatx4v delta = *reinterpret_cast<const floatx4v*>(rows + ROWS + 32 * n + 8 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) d[4 * g + i] = p[4 * g + i] * (d[4 * g + i] - delta[i]);
        }
        fitted.fit(d, dk);
        tile.transposed(dk, kQ, n, Tile::pack(d));
    };
    // 64 queries that see all of the wavefront's keys: while the vector units are at the first 32, the matrix cores form the scores of the
    // others, and while they are at those, the sums of the first.
    auto pair_step = [&](const float* rows, auto&& ask) {
        floatx16 p0, p1, d0, d1;
        zero(p0), zero(p1), zero(d0), zero(d1);
        OfRows lse0(rows);
        tile.template straight_woven<0>(p0, kQ, k_column, nothing);
        ask();
        tile.template straight_woven<16>(d0, kG, v_column, exponential(p0, lse0));
        const typename Tile::Packed b0 = Tile::pack(p0);
        OfRows delta0(rows + ROWS);
        tile.template straight_woven<16>(p1, kQ + kNext, k_column, difference(d0, p0, delta0));
        fitted.fit(d0, dk);
        const typename Tile::Packed a0 = Tile::pack(d0);
        OfRows lse1(rows + 32);
        tile.template straight_woven<16>(d1, kG + kNext, v_column, exponential(p1, lse1));
        const typename Tile::Packed b1 = Tile::pack(p1);
        OfRows delta1(rows + ROWS + 32);
        tile.template transposed_woven<0>(dv, kG, b0, nothing);
        tile.template transposed_woven<16>(dk, kQ, a0, difference(d1, p1, delta1));
        tile.template transposed_woven<0>(dv, kG + kNext, b1, nothing);
        fitted.fit(d1, dk);
        tile.template transposed_woven<0>(dk, kQ + kNext, Tile::pack(d1), nothing);
    };
    for (int it = it0; it < it1; ++it) {
        wait_for_copies();
        lds_barrier();
        const int first = (see.first_tile + now.tile) * ROWS, set = set_of(it);
        // `next` is the iteration after this one: its tiles are asked for, its rows' sums stored; those of the one after it loaded
        auto ask = [&] {
            request(it + 1, next), store_rows(it + 1);
            now = next, next = see.after(next);
            load_rows(it + 2, next);
        };
        const float* rows = reinterpret_cast<const float*>(lds + set + 2 * kTileBytes) + 4 * half;
        bool done = false;
        if constexpr (sizeof(T) == 2 && NS == 2) {
            done = first >= see.wave_all;
            if (done) pair_step(rows, ask);
        }
        if (!done) {
            ask();
#pragma unroll
            for (int n = 0; n < NS; ++n)
                if (first + 32 * (n + 1) > see.wave_need) block_step(n, first, rows, first + 32 * n < see.wave_all);
        }
        tile.shift(set ? -kSetBytes : kSetBytes);
    }
    fitted.undo(dk);
    wait_for_copies();
    lds_barrier();
    const int dim = a.chunks * Tile::kPerChunk;
    constexpr float kDown = 1.f / (1 << kUp<T>);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (a.splits == 1) {
            typedef AttnOut<T, DP> Out;
            char* room = lds + wave * Out::kRoom;
            const HeadsAt& at = which ? a.dv_at : a.dk_at;
            T* to = static_cast<T*>(which ? a.dv : a.dk);
            if (!to) continue;
            to += batch * at.batch + kv_head * at.head;
            if (which) Out::park(room, dv, kDown, lane);
            else Out::park(room, dk, a.scale * kDown, lane);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            Out::write(room, a.chunks, lane, [&](int col) -> T* { return wave_key + col < a.keys ? to + (wave_key + col) * at.token : nullptr; });
        } else {
            typedef AttnOut<float, DP> Out;
            char* room = lds + wave * Out::kRoom;
            float* to = a.partial + ((static_cast<int64_t>(split) * 2 + which) * pairs + bk) * a.keys * dim;
            if (which) Out::park(room, dv, kDown, lane);
            else Out::park(room, dk, a.scale * kDown, lane);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            Out::write(room, dim / 4, lane, [&](int col) -> float* { return wave_key + col < a.keys ? to + static_cast<int64_t>(wave_key + col) * dim : nullptr; });
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// The same for 16-bit heads of more than 64 elements.  Keys and values, both sums and both products of a step are more than the 256 registers with which
// two wavefronts fit on a SIMD, and one alone leaves the matrix cores idle while it forms probabilities.  So two sets of four wavefronts share
// the work: the first form the probabilities and dS of 32 queries and leave them in LDS, rounded as the products take them and for the lanes that
// take them, and the second add them to both sums a step later, two products each.  Three sets of tiles: of the queries whose turn it is, those
// before and those on their way.
//
// dk and dv of [4,4096,16,128] bf16: 1154 us (953 TFLOP/s), causal 590 to 630, fp16 1330.  Both sums in one wavefront took 2460; dk in one set and dv in the other, both
// forming the probabilities, 1409; the first set without the scores of the step ahead 1317.  Bound by the first set's steps and their barriers:
// matrix cores (46 %) and LDS (38 %) are each busy for less than half of the time.
template <typename T, int DP>
__global__ __launch_bounds__(2 * kThreads, 2) void attention_backward_pairs(const AttnArgs a) {
    typedef AttnTile<T, DP> Tile;
    typedef typename Tile::Frag Frag;
    constexpr int WAVES = 2 * kWaves, ROWS = kPairRows, kTileBytes = ROWS * Tile::kRowBytes, kSetBytes = 2 * kTileBytes, kSets = 3;
    constexpr int kRowsAt = kSets * kSetBytes, kHandedAt = kRowsAt + kSets * 2 * ROWS * 4, kUpAt = kHandedAt + kHandedBytes;
    constexpr uint32_t kQ = 0, kG = kTileBytes, kBlock = 32 * Tile::kRowBytes;
    extern __shared__ __align__(16) char lds[];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave), half = lane >> 5;
    const int pairs = a.batch * a.kv_heads;
    int u, unit, batch, kv_head;
    bool late;
    block_of(blockIdx.x, pairs, a.blocks * a.splits, false, u, unit, late);
    head_of(a, u, a.kv_heads, 1, false, batch, kv_head);
    const int bk = batch * a.kv_heads + kv_head;
    unit = a.blocks * a.splits - 1 - unit;      // the first keys, which most queries see in the causal form, first
    const int block = unit / a.splits, split = unit - block * a.splits;
    const int length = sequence_keys(a, batch);
    typedef typename QueriesOfKeys<ROWS>::At At;
    const QueriesOfKeys<ROWS> see(a, block * kRows * kWaves, wave % kWaves, lane, length, split);
    const T* q0 = static_cast<const T*>(a.q) + batch * a.q_at.batch + static_cast<int64_t>(kv_head) * a.group * a.q_at.head;
    const T* g0 = static_cast<const T*>(a.dout) + batch * a.dout_at.batch + static_cast<int64_t>(kv_head) * a.group * a.dout_at.head;
    const int64_t row0 = (static_cast<int64_t>(batch) * a.heads + static_cast<int64_t>(kv_head) * a.group) * a.tokens;
    Tile tile(lds, lane);
    AttnCopy<T, DP, ROWS, WAVES> q_copy(q0, a.q_at.token, a.chunks, wave, lane), g_copy(g0, a.dout_at.token, a.chunks, wave, lane);
    auto request = [&](int it, const At& at, int set) {
        if (it >= see.it1) return;
        char* to = lds + set * kSetBytes;
        q_copy.base = reinterpret_cast<const char*>(q0 + at.head * a.q_at.head), g_copy.base = reinterpret_cast<const char*>(g0 + at.head * a.dout_at.head);
        const int first = (see.first_tile + at.tile) * ROWS;
        q_copy.request(to, first, a.tokens), g_copy.request(to + kTileBytes, first, a.tokens);
    };
    float row_next = 0.f;       // of the queries on their way: threads 0 .. ROWS - 1 their sums, the next as many their D
    auto load_rows = [&](int it, const At& at) {
        if (it >= see.it1 || tid >= 2 * ROWS) return;
        const int row = (see.first_tile + at.tile) * ROWS + (tid & (ROWS - 1));
        const int64_t place = row0 + static_cast<int64_t>(at.head) * a.tokens + row;
        row_next = tid < ROWS ? (row < a.tokens ? a.lse[place] - kUp<T> : INFINITY) : (row < a.tokens ? a.delta[place] : 0.f);
    };
    auto store_rows = [&](int it, int set) {
        if (it < see.it1 && tid < 2 * ROWS) reinterpret_cast<float*>(lds + kRowsAt + set * 2 * ROWS * 4)[tid] = row_next;
    };
    At now = see.start(), next = see.after(now);
    request(see.it0, now, 0);
    load_rows(see.it0, now), store_rows(see.it0, 0);
    load_rows(see.it0 + 1, next);
    // What wavefronts w and w + 4 hand on: 32 queries of either half of a tile have a place.
    auto handed = [&](int n, int which) { return lds + kHandedAt + ((n * kWaves + wave % kWaves) * 4 + which) * 16 * kWave + 16 * lane; };
    auto handed_up = [&](int n) { return reinterpret_cast<float*>(lds + kUpAt) + (n * kWaves + wave % kWaves) * kWave + lane; };      // Fitted's
    auto seen = [&](int first) { return first + 32 > see.wave_need; };      // any of these 32 queries, by any of the wavefront's keys?
    auto first_of = [&](const At& at) { return (see.first_tile + at.tile) * ROWS; };
    // All wavefronts, tile by tile: what one set does between the barriers.  A tile is asked for as soon as nobody is at the one before the last, and has
    // come when half of the last is done.
    int set = 0;
    auto walk = [&](auto&& start, auto&& one, auto&& other) {
        wait_for_copies();
        lds_barrier();
        request(see.it0 + 1, next, 1);
        if (see.it0 < see.it1) start();
        for (int it = see.it0; it < see.it1; ++it) {
            const At third = see.after(next);
            const int after = set == kSets - 1 ? 0 : set + 1;
            store_rows(it + 1, after), load_rows(it + 2, third);
            one(first_of(now));
            wait_for_copies();
            lds_barrier();
            request(it + 2, third, after == kSets - 1 ? 0 : after + 1);
            other(first_of(now), it + 1 < see.it1);
            now = next, next = third, set = after;
            lds_barrier();
        }
    };
    auto nothing = [](int) {};
    if (wave < kWaves) {
        Frag k_column[Tile::kSteps], v_column[Tile::kSteps];
        const bool mine = see.my_key < length;
        load_column<T, DP>(k_column, static_cast<const T*>(a.k) + batch * a.k_at.batch + see.my_key * a.k_at.token + kv_head * a.k_at.head, mine, a.chunks, half);
        load_column<T, DP>(v_column, static_cast<const T*>(a.v) + batch * a.v_at.batch + see.my_key * a.v_at.token + kv_head * a.v_at.head, mine, a.chunks, half);
        // The scores run a step ahead, so that every product has vector work next to it: dO . v the exponentials, the next scores dS.
        floatx16 p, ahead;
        Fitted<T> fitted;
        auto zero = [](floatx16& v) {
#pragma unroll
            for (int r = 0; r < 16; ++r) v[r] = 0.f;
        };
        // Queries first .. + 31, half n of this tile; then the scores at `scores` of the next tile or half, unless nobody needs them.
        auto form = [&](int n, int first, bool more, auto&& move, uint32_t scores) {
            const float* rows = reinterpret_cast<const float*>(lds + kRowsAt + set * 2 * ROWS * 4) + 32 * n + 4 * half;
            if (!seen(first)) {
                move();
                zero(ahead);
                if (more) tile.template straight_woven<0>(ahead, scores, k_column, nothing);
                p = ahead;
                return;
            }
            floatx16 d;
            zero(d), zero(ahead);
            OfRows lse(rows), delta(rows + ROWS);
            tile.template straight_woven<16>(d, kG + n * kBlock, v_column, [&](int r) { p[r] = pinned(__builtin_amdgcn_exp2f(__builtin_fmaf(p[r], a.scale_log2, -lse(r)))); });
            if (first < see.wave_all) {
#pragma unroll
                for (int r = 0; r < 16; ++r) p[r] = first + 4 * half + (r & 3) + 8 * (r >> 2) >= see.need ? p[r] : 0.f;
            }
            const typename Tile::Packed b = Tile::pack(p);
            *reinterpret_cast<shortx8*>(handed(n, 0)) = b.lo, *reinterpret_cast<shortx8*>(handed(n, 1)) = b.hi;
            move();
            auto difference = [&](int r) { d[r] = pinned(p[r] * (d[r] - delta(r))); };
            if (more) {
                tile.template straight_woven<16>(ahead, scores, k_column, difference);
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) difference(r);
            }
            if constexpr (Fitted<T>::kNeeded) fitted.look(d, [](float) {}), *handed_up(n) = fitted.up;
            const typename Tile::Packed s = Tile::pack(d);
            *reinterpret_cast<shortx8*>(handed(n, 2)) = s.lo, *reinterpret_cast<shortx8*>(handed(n, 3)) = s.hi;
            p = ahead;
        };
        walk(
            [&] {
                zero(p);
                tile.template straight_woven<0>(p, kQ, k_column, nothing);
            },
            [&](int first) { form(0, first, true, [] {}, kQ + kBlock); },
            [&](int first, bool more) {
                form(1, first + 32, more, [&] { tile.shift(set == kSets - 1 ? -(kSets - 1) * kSetBytes : kSetBytes); }, kQ);
            });
        lds_barrier();      // (the others' last step)
        return;
    }
    floatx16 dk[Tile::kBlocks], dv[Tile::kBlocks];
    clear(dk), clear(dv);
    Fitted<T> fitted;
    auto add = [&](int n, int first) {
        if (!seen(first)) return;
        typename Tile::Packed p, d;
        p.lo = *reinterpret_cast<const shortx8*>(handed(n, 0)), p.hi = *reinterpret_cast<const shortx8*>(handed(n, 1));
        d.lo = *reinterpret_cast<const shortx8*>(handed(n, 2)), d.hi = *reinterpret_cast<const shortx8*>(handed(n, 3));
        tile.template transposed_woven<0>(dv, kG + n * kBlock, p, nothing);
        if constexpr (Fitted<T>::kNeeded) fitted.take_over(*handed_up(n), dk);
        tile.template transposed_woven<0>(dk, kQ + n * kBlock, d, nothing);
    };
    int before = -1;      // first query of the tile before, whose second half is still to be added
    walk([] {},
         [&](int first) {
             if (before >= 0) {
                 add(1, before + 32);
                 tile.shift(set == 0 ? -(kSets - 1) * kSetBytes : kSetBytes);      // from the set before this one
             }
             before = first;
         },
         [&](int first, bool) { add(0, first); });
    if (before >= 0) add(1, before + 32);
    fitted.undo(dk);
    lds_barrier();
    const int dim = a.chunks * Tile::kPerChunk, wave_key = see.wave_key;
    constexpr float kDown = 1.f / (1 << kUp<T>);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (a.splits == 1) {
            typedef AttnOut<T, DP> Out;
            char* room = lds + (wave - kWaves) * Out::kRoom;
            const HeadsAt& at = which ? a.dv_at : a.dk_at;
            T* to = static_cast<T*>(which ? a.dv : a.dk);
            if (!to) continue;
            to += batch * at.batch + kv_head * at.head;
            if (which) Out::park(room, dv, kDown, lane);
            else Out::park(room, dk, a.scale * kDown, lane);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            Out::write(room, a.chunks, lane, [&](int col) -> T* { return wave_key + col < a.keys ? to + (wave_key + col) * at.token : nullptr; });
        } else {
            typedef AttnOut<float, DP> Out;
            char* room = lds + (wave - kWaves) * Out::kRoom;
            float* to = a.partial + ((static_cast<int64_t>(split) * 2 + which) * pairs + bk) * a.keys * dim;
            if (which) Out::park(room, dv, kDown, lane);
            else Out::park(room, dk, a.scale * kDown, lane);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            Out::write(room, dim / 4, lane, [&](int col) -> float* { return wave_key + col < a.keys ? to + static_cast<int64_t>(wave_key + col) * dim : nullptr; });
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// dk and dv from the splits' sums, in their order: four elements a thread.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_backward_join(const AttnArgs a) {
    const int quads = a.chunks * AttnElem<T>::kPerChunk / 4, pairs = a.batch * a.kv_heads;
    const int64_t one = static_cast<int64_t>(pairs) * a.keys * quads, at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (at >= 2 * one) return;
    const int which = at >= one;
    const int64_t in = at - which * one;
    const float4* p = reinterpret_cast<const float4*>(a.partial) + at;
    float4 sum = p[0];
    for (int s = 1; s < a.splits; ++s) {
        const float4 more = p[2 * one * s];
        sum.x += more.x, sum.y += more.y, sum.z += more.z, sum.w += more.w;
    }
    const int64_t row = in / quads;
    const int d = 4 * static_cast<int>(in - row * quads), bk = static_cast<int>(row / a.keys), key = static_cast<int>(row - static_cast<int64_t>(bk) * a.keys);
    const int batch = bk / a.kv_heads, kv_head = bk - batch * a.kv_heads;
    const HeadsAt& to = which ? a.dv_at : a.dk_at;
    T* base = static_cast<T*>(which ? a.dv : a.dk);
    if (base) store_piece<true>(base + batch * to.batch + key * to.token + kv_head * to.head + d, sum);
}

template <typename T, int DP>
constexpr int backward_rows_lds() {
    constexpr int tiles = 4 * tile_rows<T>() * AttnTile<T, DP>::kRowBytes, out = kWaves * AttnOut<float, DP>::kRoom;
    return tiles > out ? tiles : out;
}
template <typename T, int DP>
constexpr int backward_keys_lds() {
    constexpr int tiles = 2 * query_tile<T, DP>() * (2 * AttnTile<T, DP>::kRowBytes + 2 * 4), out = kWaves * AttnOut<float, DP>::kRoom;
    return tiles > out ? tiles : out;
}

template <typename T, int DP>
constexpr int backward_pairs_lds() {
    constexpr int tiles = 3 * kPairRows * (2 * AttnTile<T, DP>::kRowBytes + 2 * 4) + kHandedBytes + (Fitted<T>::kNeeded ? 2 * kWaves * kWave * 4 : 0), out = kWaves * AttnOut<float, DP>::kRoom;
    return tiles > out ? tiles : out;
}

// Workgroups that share the queries of a block of keys: as many as the chip has CUs in all, twice that where the blocks' lengths differ (causal), and
// with at least `least` times 32 queries.  (dk and dv of [2,448,16,64] bf16, 1500 keys, in one part 22 us, in two 43: the sums' way through memory;
// [2,2048,8,128] in one part each 78 us, in two 110; [4,2048,8,128] causal, one key head, eight parts each 102 us, four 129, twelve 120.
// fp32 [3,333,8,40], 77 keys, at least 64 queries each: 16 us, 256: 43.)
int key_splits(int64_t batch, int64_t tokens, int64_t keys, int64_t heads, int64_t kv_heads, bool causal, int least) {
    if (batch < 1 || tokens < 1 || keys < 1 || heads < 1 || kv_heads < 1) return 1;
    int dev;
    const int64_t units = batch * kv_heads * blocks_of(keys), tiles = heads / kv_heads * ((tokens + 31) / 32);
    int64_t splits = (causal ? 2 : 1) * static_cast<int64_t>(compute_units(dev)) / units;
    if (splits > tiles / least) splits = tiles / least;
    return static_cast<int>(splits < 1 ? 1 : splits > 64 ? 64 : splits);
}
template <typename T>
constexpr int least_of_split() { return sizeof(T) == 2 ? 8 : 2; }

// Workgroups that share the keys of a block of queries: as many as the chip has CUs in all, with at least `least` keys.  (dq of fp32 [1,64,8,64],
// 4096 keys: 40 us, most of it the call, instead of 403; fp32 [1,448,16,64], 1500 keys: 56 instead of 153; [1,2048,8,128] bf16 57 instead of 61.)
int row_splits(int64_t batch, int64_t tokens, int64_t keys, int64_t heads, int64_t least) {
    if (batch < 1 || tokens < 1 || keys < 1 || heads < 1) return 1;
    int dev;
    int64_t splits = compute_units(dev) / (batch * heads * blocks_of(tokens));
    if (splits > keys / least) splits = keys / least;
    return static_cast<int>(splits < 1 ? 1 : splits);
}
template <typename T>
constexpr int least_keys() { return sizeof(T) == 2 ? 256 : 64; }

int64_t rounded4(int64_t n) { return (n + 3) / 4 * 4; }

}  // namespace
}  // namespace ddl

extern "C" {

int64_t ddl_attention_backward_workspace(int64_t batch, int64_t tokens, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim) {
    using namespace ddl;
    if (!has_work(batch, tokens, keys, heads, kv_heads, dim)) return 0;
    const int64_t splits = key_splits(batch, tokens, keys, heads, kv_heads, true, least_of_split<float>());      // the most that a call takes
    const int64_t shares = row_splits(batch, tokens, keys, heads, least_keys<float>());
    const int64_t of_keys = splits > 1 ? splits * 2 * batch * kv_heads * keys * dim : 0, of_rows = shares > 1 ? shares * batch * heads * tokens * dim : 0;
    return rounded4(batch * heads * tokens) + (of_keys > of_rows ? of_keys : of_rows);      // (the kernels run one after the other)
}

int ddl_attention_backward(const void* dout, const int64_t* dout_strides, const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                           const void* v, const int64_t* v_strides, const void* out, const int64_t* out_strides, const void* out_rest, const float* lse, int dtype, int64_t batch,
                           int64_t tokens, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim, const int32_t* lengths, int causal, float scale,
                           void* dq, const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv, const int64_t* dv_strides, float* workspace,
                           int64_t workspace_elems, void* stream) {
    using namespace ddl;
    AttnArgs a{};
    bool nothing;
    if (const int rc = fill_attention(a, nothing, "ddl_attention_backward", {{q, q_strides}, {k, k_strides}, {v, v_strides}, {out, out_strides}, {dout, dout_strides}}, dtype,
                                      batch, tokens, keys, heads, kv_heads, dim, lengths, causal, scale))
        return rc;
    if (nothing || (!dq && !dk && !dv)) return 0;
    const struct { void* p; const int64_t* s; } results[3] = {{dq, dq_strides}, {dk, dk_strides}, {dv, dv_strides}};
    for (const auto& r : results) {
        if (!r.p) continue;
        const int per = dtype == DDL_DT_F32 ? 4 : 8;
        if (!r.s) return fail(DDL_E_ARG, "ddl_attention_backward: no strides");
        if (!aligned_to(r.p, 16) || r.s[0] % per || r.s[1] % per || r.s[2] % per) return fail(DDL_E_ALIGN, "ddl_attention_backward: gradients are not 16-byte aligned");
    }
    if (out_rest && dtype == DDL_DT_F32) return fail(DDL_E_ARG, "ddl_attention_backward: only 16-bit results have a rest");
    if (!aligned_to(out_rest, 16)) return fail(DDL_E_ALIGN, "ddl_attention_backward: the rest is not 16-byte aligned");
    if (tokens && !lse) return fail(DDL_E_ARG, "ddl_attention_backward: no row sums");
    const int64_t need = ddl_attention_backward_workspace(batch, tokens, keys, heads, kv_heads, dim);
    if (need && (!workspace || workspace_elems < need))
        return fail(DDL_E_ARG, "ddl_attention_backward: workspace of %lld floats, %lld are needed", static_cast<long long>(workspace ? workspace_elems : 0), static_cast<long long>(need));
    if (need && !aligned_to(workspace, 16)) return fail(DDL_E_ALIGN, "ddl_attention_backward: workspace is not 16-byte aligned");
    if (!adjoint_launches(a, dtype, dim)) return fail(DDL_E_UNSUPP, "ddl_attention_backward: 2^32 threads");
    a.dout = dout, a.dout_at = place_of(dout_strides), a.out = const_cast<void*>(out), a.out_at = place_of(out_strides), a.rest = const_cast<void*>(out_rest), a.lse = const_cast<float*>(lse);
    a.dq = dq, a.dk = dk, a.dv = dv, a.dq_at = place_of(dq_strides), a.dk_at = place_of(dk_strides), a.dv_at = place_of(dv_strides);
    a.delta = workspace, a.partial = workspace + rounded4(batch * heads * tokens);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return with_attention_kernel(dtype, dim, [&](auto* e, auto dp) {
        typedef std::remove_pointer_t<decltype(e)> T;
        constexpr int DP = decltype(dp)::value;
        constexpr int kRowsLds = backward_rows_lds<T, DP>();
        if (a.tokens) {
            a.blocks = static_cast<int>(blocks_of(a.tokens));
            a.splits = a.dq ? row_splits(batch, tokens, keys, heads, least_keys<T>()) : 1;
            const int64_t grid = static_cast<int64_t>(a.blocks) * a.batch * a.heads;
            a.folded = folds(a, grid);
            const auto launch = [&](auto one) {
                constexpr bool ONE = decltype(one)::value;
                if (const int rc = grant_lds<attention_backward_rows<T, DP, ONE>>(kRowsLds, "ddl_attention_backward")) return rc;
                hipLaunchKernelGGL((attention_backward_rows<T, DP, ONE>), dim3(static_cast<uint32_t>(grid), a.splits), dim3(kThreads), kRowsLds, s, a);
                return check_launch("ddl_attention_backward");
            };
            int rc;
            if constexpr (sizeof(T) == 2) rc = a.keys <= tile_rows<T>() ? launch(std::true_type{}) : launch(std::false_type{});
            else rc = launch(std::false_type{});
            if (rc) return rc;
            if (a.splits > 1) {
                const int64_t threads = static_cast<int64_t>(a.batch) * a.heads * a.tokens * (dim / 4);
                hipLaunchKernelGGL((attention_backward_rows_join<T>), dim3(static_cast<uint32_t>((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, a);
                if (const int joined = check_launch("ddl_attention_backward")) return joined;
            }
        }
        if (a.keys == 0 || (!a.dk && !a.dv)) return 0;
        a.splits = key_splits(batch, tokens, keys, heads, kv_heads, a.causal, least_of_split<T>());
        a.blocks = static_cast<int>(blocks_of(a.keys));
        const int64_t pairs = static_cast<int64_t>(a.batch) * a.kv_heads, grid = pairs * a.blocks * a.splits;
        if constexpr (in_pairs(sizeof(T), DP)) {
            constexpr int kLds = backward_pairs_lds<T, DP>();
            if (const int rc = grant_lds<attention_backward_pairs<T, DP>>(kLds, "ddl_attention_backward")) return rc;
            hipLaunchKernelGGL((attention_backward_pairs<T, DP>), dim3(static_cast<uint32_t>(grid)), dim3(2 * kThreads), kLds, s, a);
        } else {
            constexpr int kLds = backward_keys_lds<T, DP>();
            if (const int rc = grant_lds<attention_backward_keys<T, DP>>(kLds, "ddl_attention_backward")) return rc;
            hipLaunchKernelGGL((attention_backward_keys<T, DP>), dim3(static_cast<uint32_t>(grid)), dim3(kThreads), kLds, s, a);
        }
        if (const int rc = check_launch("ddl_attention_backward")) return rc;
        if (a.splits == 1) return 0;
        const int64_t threads = 2 * pairs * a.keys * (dim / 4);
        hipLaunchKernelGGL((attention_backward_join<T>), dim3(static_cast<uint32_t>((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, a);
        return check_launch("ddl_attention_backward");
    });
}

}  // extern "C"
