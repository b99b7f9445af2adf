// Attention of queries to keys and values of another (or the same) length, on heads that a worker holds whole, forward.
//
//   out[i] = sum over the keys j that query i sees of p_ij v_j,   p_ij = exp(scale q_i . k_j) / sum over j of the same
//
// in one pass over the keys with the running maximum and sum of the softmax (fp32); 2^x takes the place of e^x, log2(e) goes
// into the scale.  A query that sees no key gives zeros.  Kept for the adjoint: log2 of each row's sum (+inf for a row
// without keys, so that its probabilities come out as zero there) and, of 16-bit results, what their rounding took: the adjoint's
// D = dO . out is a difference's second member, and off by that rounding where few keys share the weight (see there).
//
// Two forms, attention_rows and attention_split below; what they are made of is in attention_parts.h.
#include "ddl_common.h"

#include "attention_parts.h"

#include <utility>

namespace ddl {
namespace {

constexpr int kStats = 4;               // behind the sums of a row over a split's keys: its maximum, its two totals, nothing
// In powers of two: what a probability may come to before the running maximum is moved, and what the largest one then comes to.
//
// fp16 has full steps only down to 2^-14, and next to a key of large weight many small ones would lose theirs (of 299 keys with 2^-23 of the largest
// one's weight each, whose values are the result, a fifth): what its range has above one is used, up to 2^15.  The room between the two is what keeps
// most blocks from moving anything ([4,4096,16,64], all keys: 310 us with eight of them or six, 316 with four, 319 with three).
template <typename T>
constexpr float kMost = std::is_same_v<T, __half> ? 15.f : 8.f;
template <typename T>
constexpr float kLargest = std::is_same_v<T, __half> ? 9.f : 0.f;
constexpr float kHuge = 1048576.f;      // a maximum from which on its rounding shows (by 2^-4)

// The softmax of a wavefront's columns as far as it has come.
//
// Two totals: of the probabilities as they are rounded for the product, which is what the result is divided by (the weights of a mean add
// up to one then, and a single large one is exact), and, EXACT, of the unrounded ones, from which the adjoint forms them anew:
// divided by the other one they would all be off by its rounding, up to half a step where one key has most of the weight.
template <typename T, int BLOCKS, bool EXACT>
struct Running {
    floatx16 acc[BLOCKS];
    float top = -INFINITY, total = 0.f, exact = 0.f;      // of this lane's column; the totals of this lane's half of the rows
    float mul, base = 0.f;                                // a probability is 2^(mul score - base)
    float lag = kMost<T>;                                 // from where on the maximum follows

    __device__ explicit Running(float scale) : mul(scale) {
#pragma unroll
        for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
    }
    // The maximum follows the scores of 32 keys, which this looks at: only where a probability would get too large, since the sums have room until then
    // and most blocks leave them alone, and to a whole power of two, so that what has been summed (and `before`, what waits to
    // be) moves without a rounding.
    //
    // Once a maximum is huge the rounding of score times scale shows, and the difference to it is formed from the rounded products, whose largest is the
    // maximum itself: here, for every block from then on.
    template <typename Tile>
    __device__ void follow(floatx16& s, float scale, const Tile&, typename Tile::Packed* before) {
        float m = fmaxf(s[0], s[1]);
#pragma unroll
        for (int r = 2; r < 16; ++r) m = fmaxf(m, s[r]);
        m = max_halves(m) * scale;
        if (__any(m > top + lag)) {
            const float moved = fmaxf(top, ceilf(m) - kLargest<T>), factor = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - moved);
            top = moved;
            total *= factor;
            if (EXACT) exact *= factor;
#pragma unroll
            for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= factor;
            if (before) Tile::scale_packed(*before, factor);
            base = top == -INFINITY ? 0.f : top;
            if (__any(fabsf(base) > kHuge)) lag = -INFINITY, mul = 1.f;
            if (lag < 0.f) {
                const float from = base;
                base = 0.f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float d = pinned(s[r] * scale) - from;
                    s[r] = d > kMost<T> ? kMost<T> : d;      // (`moved` is a multiple of 16 and more there)
                }
            }
        }
    }
    // Scores to probabilities relative to the maximum, packed and added to the total.
    template <typename Tile>
    __device__ typename Tile::Packed take(floatx16& s, const Tile&) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], mul, -base));
        const typename Tile::Packed p = Tile::pack(s);
        total = Tile::add_packed(total, p);
        add_exact(s);
        return p;
    }
    __device__ void add_exact(const floatx16& p) {
        if constexpr (EXACT) {
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) sum += p[r];
            exact += sum;
        }
    }
    __device__ float exact_total() const { return EXACT ? exact : total; }
};

// `rest`: keys of these 32 that this lane's column sees, from this lane's half's first one on.
__device__ inline void mask_scores(floatx16& s, int rest) {
#pragma unroll
    for (int r = 0; r < 16; ++r)
        if ((r & 3) + 8 * (r >> 2) >= rest) s[r] = -INFINITY;
}

template <typename T>
constexpr int keys_of_tile() { return sizeof(T) == 2 ? 64 : 32; }

// One wavefront, 32 queries of one head; a workgroup, 128 of them, walks over the keys tile by tile through LDS, each tile on its way from
// memory while those before are worked on.
//
// Steps of 32 keys.  Step s has three parts that do not wait for each other, so that the matrix cores and the vector
// units both have work: the scores of block s + 1, the softmax of block s, and the product of block s - 1 with its values.
// With tiles of NS blocks, keys are read up to one block before and values one block after the softmax: one barrier a tile, in
// front of its last block, is then enough for two buffers of each.  What follows it is copied to where
// everybody has just finished reading: keys two tiles ahead, values NS - 1 blocks ahead.
//
// [4,4096,16,128] bf16, all keys, in runs of 20 calls: 551 us (997 TFLOP/s); the first launches of a process, whose clock has yet to rise, take up to 624,
// where the parts one behind the other and tiles through registers took 729.  Head size 64: 310 us; causal, with sums kept: 292; fp16 551 and 325; fp32 [2,2048,8,64]
// 160 us (108 TFLOP/s).  Bound by issue: the exponentials and the softmax's other vector work next to the matrix instructions, of which each pipe is busy
// about half of the time (matrix 55 %, vector 46 %).
template <typename T, int DP, bool LSE>
__global__ __launch_bounds__(kThreads, DP * sizeof(T) > 384 ? 1 : 2) void attention_rows(const AttnArgs a) {
    typedef AttnTile<T, DP> Tile;
    typedef typename Tile::Frag Frag;
    constexpr int KEYS = keys_of_tile<T>(), NS = KEYS / 32, kTileBytes = KEYS * Tile::kRowBytes;
    extern __shared__ __align__(16) char lds[];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave), half = lane >> 5;
    int u, block, batch, head;
    bool late;
    block_of(blockIdx.x, a.batch * a.heads, a.blocks, a.folded, u, block, late);     // the last rows, which see most keys in the causal form, first
    head_of(a, u, a.heads, a.group, late, batch, head);
    const int bh = batch * a.heads + head, kv_head = head / a.group;
    const int length = sequence_keys(a, batch);
    const int first_row = block * kRows * kWaves, wave_row = first_row + wave * kRows, my_row = wave_row + (lane & 31);
    const int seen = keys_seen(a, my_row, length);
    auto scalar = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const int end = scalar(keys_seen(a, min(first_row + kRows * kWaves, a.tokens) - 1, length));    // most that a row of the workgroup sees
    const int wave_most = scalar(wave_row < a.tokens ? keys_seen(a, min(wave_row + kRows, a.tokens) - 1, length) : 0);   // rows of a wavefront: most,
    const int wave_least = scalar(keys_seen(a, wave_row, length));                                  // and least
    const T* q = static_cast<const T*>(a.q) + batch * a.q_at.batch + head * a.q_at.head;
    const T* k = static_cast<const T*>(a.k) + batch * a.k_at.batch + kv_head * a.k_at.head;
    const T* v = static_cast<const T*>(a.v) + batch * a.v_at.batch + kv_head * a.v_at.head;

    const Tile tile(lds, lane);
    const int tiles = (end + KEYS - 1) / KEYS, steps = (wave_most + 31) / 32;
    constexpr int kPhases = 2 * NS;      // steps after which the tiles' places come again
    auto k_tile = [](int t) { return (t & 1) * kTileBytes; };
    auto v_tile = [](int t) { return (2 + (t & 1)) * kTileBytes; };
    auto k_block = [&](int s) { return k_tile(s / NS) + s % NS * (32 * Tile::kRowBytes); };
    auto v_block = [&](int s) { return v_tile(s / NS) + s % NS * (32 * Tile::kRowBytes); };
    const AttnCopy<T, DP, KEYS, kWaves> k_copy(k, a.k_at.token, a.chunks, wave, lane), v_copy(v, a.v_at.token, a.chunks, wave, lane);
    k_copy.request(lds + k_tile(0), 0, end), k_copy.request(lds + k_tile(1), KEYS, end);
    if (NS > 1) v_copy.request(lds + v_tile(0), 0, end);
    Frag column[Tile::kSteps];
#pragma unroll
    for (int s = 0; s < Tile::kSteps; ++s) {
        Frag f = {};
        if (my_row < a.tokens && 2 * s + half < a.chunks) f = *reinterpret_cast<const Frag*>(q + my_row * a.q_at.token + (2 * s + half) * Tile::kPerChunk);
        column[s] = f;
    }
    wait_for_copies();
    lds_barrier();
    Running<T, Tile::kBlocks, LSE && sizeof(T) == 2> run(a.scale_log2);
    floatx16 scores;
    typename Tile::Packed before;
    auto score = [&](floatx16& to, int s) {
#pragma unroll
        for (int r = 0; r < 16; ++r) to[r] = 0.f;
        tile.straight(to, k_block(s), 0, column);
    };
    auto values = [&](int s) { tile.transposed(run.acc, v_block(s), 0, before); };
    auto step = [&](int s, auto ahead, auto behind) {
        if constexpr (sizeof(T) == 2) wait_states<12>(scores);
        if (32 * (s + 1) > wave_least) mask_scores(scores, seen - 32 * s - 4 * half);
        run.follow(scores, a.scale_log2, tile, behind ? &before : nullptr);
        floatx16 next;
        if constexpr (ahead) score(next, s + 1);
        if constexpr (behind) values(s - 1);
        before = run.take(scores, tile);
        if constexpr (ahead) scores = next;
    };
    // The same in full, 16-bit types: after every matrix instruction (32 cycles) an LDS read for the one after the next two and a share of the
    // sixteen exponentials, in this order -- left to itself the compiler puts one part behind the other.  `phase`: s modulo kPhases.
    auto full_step = [&](int s, auto phase) {
        if (32 * (s + 1) > wave_least) mask_scores(scores, seen - 32 * s - 4 * half);
        run.follow(scores, a.scale_log2, tile, &before);
        if constexpr (sizeof(T) == 2) {
            constexpr int kPhase = decltype(phase)::value, kSlots = 2 * Tile::kSteps;
            const uint32_t kb = k_block((kPhase + 1) % kPhases), vb = v_block((kPhase + kPhases - 1) % kPhases);
            floatx16 next;
#pragma unroll
            for (int r = 0; r < 16; ++r) next[r] = 0.f;
            Frag kf[Tile::kSteps], vf[Tile::kSteps];
            auto read = [&](int i) {
                if (i >= Tile::kSteps) return;
                kf[i] = tile.read_straight(kb, i), vf[i] = tile.read_transposed(vb, i / Tile::kBlocks, i % Tile::kBlocks);
            };
            auto share = [&](int slot) {
#pragma unroll
                for (int r = 16 * slot / kSlots; r < 16 * (slot + 1) / kSlots; ++r) scores[r] = pinned(__builtin_amdgcn_exp2f(__builtin_fmaf(scores[r], run.mul, -run.base)));
            };
            read(0), read(1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < Tile::kSteps; ++i) {
                mfma_chunk(next, kf[i], column[i], static_cast<const T*>(nullptr));
                if (i + 2 < Tile::kSteps) kf[i + 2] = tile.read_straight(kb, i + 2);
                share(2 * i);
                __builtin_amdgcn_sched_barrier(0);
                mfma_chunk(run.acc[i % Tile::kBlocks], vf[i], i / Tile::kBlocks ? before.hi : before.lo, static_cast<const T*>(nullptr));
                if (i + 2 < Tile::kSteps) vf[i + 2] = tile.read_transposed(vb, (i + 2) / Tile::kBlocks, (i + 2) % Tile::kBlocks);
                share(2 * i + 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            before = Tile::pack(scores);
            run.total = Tile::add_packed(run.total, before);
            run.add_exact(scores);
            scores = next;
        } else {
            floatx16 next;
            score(next, s + 1);
            values(s - 1);
            before = run.take(scores, tile);
            scores = next;
        }
    };
    const std::true_type yes{};
    const std::false_type no{};
    auto turn = [&](int s) {
        if (s % NS != NS - 1) return;
        wait_for_copies();
        lds_barrier();
        const int kt = s / NS + 2, vt = (s + NS - 1) / NS;
        k_copy.request(lds + k_tile(kt), kt * KEYS, end), v_copy.request(lds + v_tile(vt), vt * KEYS, end);
    };
    int s = 0;      // (a wavefront whose rows see fewer keys than others' still takes its part in the copies and barriers)
    if (steps > 0) {
        score(scores, 0);
        turn(0);
        if (steps == 1) {
            step(0, no, no);
        } else {
            step(0, yes, no);
            for (s = 1; s + kPhases < steps; s += kPhases) {      // always from phase 1 on
                turn(s), full_step(s, std::integral_constant<int, 1>{});
                if constexpr (NS == 2) {
                    turn(s + 1), full_step(s + 1, std::integral_constant<int, 2>{});
                    turn(s + 2), full_step(s + 2, std::integral_constant<int, 3>{});
                }
                turn(s + kPhases - 1), full_step(s + kPhases - 1, std::integral_constant<int, 0>{});
            }
            for (; s + 1 < steps; ++s) {
                turn(s);
                step(s, yes, yes);
            }
            turn(s);
            step(s, no, yes);
        }
        turn(++s);
        values(s - 1);
        ++s;
    }
    for (; s <= tiles * NS; ++s) turn(s);
    wait_for_copies();
    lds_barrier();
    const float total = add_halves(run.total);
    if constexpr (LSE) {
        const float exact = add_halves(run.exact_total());
        if (half == 0 && my_row < a.tokens) a.lse[static_cast<int64_t>(bh) * a.tokens + my_row] = exact > 0.f ? run.top + __builtin_amdgcn_logf(exact) : INFINITY;
    }
    typedef AttnOut<T, DP> Out;
    char* room = lds + wave * Out::kRoom;
    Out::park(room, run.acc, total > 0.f ? 1.0f / total : 0.f, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    T* out = static_cast<T*>(a.out) + batch * a.out_at.batch + head * a.out_at.head;
    const auto place = [&](T* base) {
        return [=](int col) -> T* {
            const int row = first_row + wave * kRows + col;
            return row < a.tokens ? base + row * a.out_at.token : nullptr;
        };
    };
    Out::write(room, a.chunks, lane, place(out));
    if constexpr (LSE && sizeof(T) == 2) {
        if (a.rest) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            Out::template park<true>(room, run.acc, total > 0.f ? 1.0f / total : 0.f, lane);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            Out::write(room, a.chunks, lane, place(static_cast<T*>(a.rest) + batch * a.out_at.batch + head * a.out_at.head));
        }
    }
}

template <typename T, int DP>
constexpr int rows_lds() {
    typedef AttnTile<T, DP> Tile;
    constexpr int tiles = 4 * keys_of_tile<T>() * Tile::kRowBytes, out = kWaves * AttnOut<T, DP>::kRoom;
    return tiles > out ? tiles : out;
}

// Few queries, many keys: the queries of all heads that share a key head (row = token x group + head in the group) in one
// wavefront, the keys dealt to `splits` workgroups and there, 32 at a time, to the four wavefronts, each with tiles of its own
// and no barrier; the four are joined through LDS, the workgroups by attention_join (or, with one split, at once).  Bound by memory where
// there are enough tiles ([64,1,32,128] bf16, 8 key heads of 2048: 104 us, 5.2 TB/s), by the latency of a few tiles and the join's
// launch where there are not ([1,1,8,128], 65536 keys of one head: 17.8 us).
// (Rows of more than 256 bytes fill the registers of a SIMD with one wavefront: 128 of them for the tiles on their way.)
template <typename T, int DP, bool LSE>
__global__ __launch_bounds__(kThreads, DP * sizeof(T) > 256 ? 1 : 2) void attention_split(const AttnArgs a) {
    typedef AttnTile<T, DP> Tile;
    typedef typename Tile::Frag Frag;
    constexpr int KEYS = 32, kTileBytes = KEYS * Tile::kRowBytes;
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane >> 5;
    const int pairs = a.batch * a.kv_heads;
    const int bk = blockIdx.x % pairs, rest_id = blockIdx.x / pairs, split = rest_id % a.splits;
    const int block = a.blocks - 1 - rest_id / a.splits;      // the last rows, which see most keys in the causal form, first
    const int batch = bk / a.kv_heads, kv_head = bk - batch * a.kv_heads;
    const int length = sequence_keys(a, batch);
    const int rows = a.tokens * a.group, first_row = block * kRows, my_row = first_row + (lane & 31);
    const int token = my_row / a.group, head = kv_head * a.group + my_row - token * a.group;
    const int seen = my_row < rows ? keys_seen(a, token, length) : 0;
    const int most = __builtin_amdgcn_readfirstlane(keys_seen(a, (min(first_row + kRows, rows) - 1) / a.group, length));
    const int least = __builtin_amdgcn_readfirstlane(keys_seen(a, first_row / a.group, length));
    // This split's keys, of those that there are: whole tiles, shared evenly.
    const int tiles = (most + KEYS - 1) / KEYS;
    constexpr bool kEarly = sizeof(T) == 2;      // of the values, too
    const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * split / a.splits), t1 = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / a.splits);
    const T* k = static_cast<const T*>(a.k) + batch * a.k_at.batch + kv_head * a.k_at.head;
    const T* v = static_cast<const T*>(a.v) + batch * a.v_at.batch + kv_head * a.v_at.head;
    const Tile tile(lds, lane);
    const int kt = wave * 2 * kTileBytes, vt = kt + kTileBytes;
    const AttnCopy<T, DP, KEYS, 1> k_copy(k, a.k_at.token, a.chunks, 0, lane), v_copy(v, a.v_at.token, a.chunks, 0, lane);
    int t = t0 + wave;
    if (t < t1) k_copy.request(lds + kt, t * KEYS, most), v_copy.request(lds + vt, t * KEYS, most);
    Frag column[Tile::kSteps];
    const T* q = static_cast<const T*>(a.q) + batch * a.q_at.batch;
#pragma unroll
    for (int s = 0; s < Tile::kSteps; ++s) {
        Frag f = {};
        if (my_row < rows && 2 * s + half < a.chunks) f = *reinterpret_cast<const Frag*>(q + token * a.q_at.token + head * a.q_at.head + (2 * s + half) * Tile::kPerChunk);
        column[s] = f;
    }
    Running<T, Tile::kBlocks, LSE && sizeof(T) == 2> run(a.scale_log2);
    for (; t < t1; t += kWaves) {
        const int after = t + kWaves;
        wait_for_copies();
        // What the products take is read out of the tiles at once, so that the next ones can come in while this one is worked on.
        Frag kf[Tile::kSteps];
#pragma unroll
        for (int s = 0; s < Tile::kSteps; ++s) kf[s] = tile.read_straight(kt, s);
        shortx8 vf[kEarly ? 2 * Tile::kBlocks : 1];
        if constexpr (kEarly) {
#pragma unroll
            for (int i = 0; i < 2 * Tile::kBlocks; ++i) vf[i] = tile.read_transposed(vt, i / Tile::kBlocks, i % Tile::kBlocks);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (after < t1) {
            k_copy.request(lds + kt, after * KEYS, most);
            if constexpr (kEarly) v_copy.request(lds + vt, after * KEYS, most);
        }
        floatx16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int i = 0; i < Tile::kSteps; ++i) mfma_chunk(s, kf[i], column[i], static_cast<const T*>(nullptr));
        if ((t + 1) * KEYS > least) mask_scores(s, seen - t * KEYS - 4 * half);
        run.follow(s, a.scale_log2, tile, nullptr);
        const typename Tile::Packed p = run.take(s, tile);
        if constexpr (kEarly) {
#pragma unroll
            for (int i = 0; i < 2 * Tile::kBlocks; ++i) mfma_chunk(run.acc[i % Tile::kBlocks], vf[i], i / Tile::kBlocks ? p.hi : p.lo, static_cast<const T*>(nullptr));
        } else {
            tile.transposed(run.acc, vt, 0, p);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (after < t1) v_copy.request(lds + vt, after * KEYS, most);
        }
    }
    wait_for_copies();
    // Joined: every wavefront's maximum and total, then its sums relative to the common maximum, added in the wavefronts' order.
    __shared__ float tops[kWaves][kRows], totals[kWaves][kRows], exacts[kWaves][kRows];
    const float own_total = add_halves(run.total), own_exact = add_halves(run.exact_total());
    if (half == 0) tops[wave][lane] = run.top, totals[wave][lane] = own_total, exacts[wave][lane] = own_exact;
    __syncthreads();
    const int col = lane & 31;
    float top = tops[0][col];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, tops[w][col]);
    const float from = top == -INFINITY ? 0.f : top;
    float total = 0.f, exact = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const float part = __builtin_amdgcn_exp2f(tops[w][col] - from);
        total += totals[w][col] * part, exact += exacts[w][col] * part;
    }
    const bool whole = a.splits == 1;
    const float factor = __builtin_amdgcn_exp2f(run.top - from) * (whole ? (total > 0.f ? 1.0f / total : 0.f) : 1.f);
    typedef AttnOut<float, DP> Out;
    if (my_row < rows) Out::park(lds + wave * Out::kRoom, run.acc, factor, lane);
    __syncthreads();
    const int dim = a.chunks * Tile::kPerChunk;
    float* partial = a.partial + (static_cast<int64_t>(split) * pairs + bk) * rows * (DP + kStats);
    for (int i = threadIdx.x; i < kRows * (DP / 4); i += kThreads) {
        const int c = i / (DP / 4), d = 4 * (i % (DP / 4)), row = first_row + c;
        if (row >= rows || d >= dim) continue;
        float4 sum = *reinterpret_cast<const float4*>(lds + c * Out::kPitch + 4 * d);
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
            const float4 more = *reinterpret_cast<const float4*>(lds + w * Out::kRoom + c * Out::kPitch + 4 * d);
            sum.x += more.x, sum.y += more.y, sum.z += more.z, sum.w += more.w;
        }
        if (whole) {
            const int tk = row / a.group, hd = kv_head * a.group + row - tk * a.group;
            const int64_t to = batch * a.out_at.batch + tk * a.out_at.token + hd * a.out_at.head + d;
            store_piece<true>(static_cast<T*>(a.out) + to, sum);
            if (LSE && sizeof(T) == 2 && a.rest) store_piece<true>(static_cast<T*>(a.rest) + to, lost<T>(sum));
        } else {
            *reinterpret_cast<float4*>(partial + row * (DP + kStats) + d) = sum;
        }
    }
    if (wave == 0 && half == 0 && my_row < rows) {
        if (whole) {
            if (LSE) a.lse[(static_cast<int64_t>(batch) * a.heads + head) * a.tokens + token] = exact > 0.f ? top + __builtin_amdgcn_logf(exact) : INFINITY;
        } else {
            *reinterpret_cast<float4*>(partial + my_row * (DP + kStats) + DP) = make_float4(top, total, exact, 0.f);
        }
    }
}

// The splits of a row: groups of DP / 4 lanes take every GROUPS-th of them (eight in flight), in one pass with a running maximum, and are
// joined in their order.  GROUPS = 1, for up to eight splits: a group has a row to itself ([1,512,8,128] bf16 to 1024 keys, two splits:
// 15.3 us for both kernels, with a workgroup for each row 20).
constexpr int kSplitsInFlight = 8;
template <int DP>
constexpr int join_lanes() { return DP == 96 ? 32 : DP / 4; }      // of a split's row, four elements each; rows of 96 leave 8 idle
template <typename T, int DP, int GROUPS>
__global__ __launch_bounds__(kThreads) void attention_join(const AttnArgs a) {
    constexpr int kLanes = join_lanes<DP>(), kAtOnce = kThreads / kLanes / GROUPS;      // rows of a workgroup
    const int pairs = a.batch * a.kv_heads, rows = a.tokens * a.group;
    const int place = threadIdx.x / kLanes, group = GROUPS == 1 ? 0 : place, lane = threadIdx.x % kLanes, d = 4 * lane;
    const int at = static_cast<int>(blockIdx.x) * kAtOnce + (GROUPS == 1 ? place : 0);
    if (GROUPS == 1 && at >= pairs * rows) return;
    const int64_t pitch = static_cast<int64_t>(pairs) * rows * (DP + kStats);
    const float* p = a.partial + static_cast<int64_t>(at) * (DP + kStats);
    const bool there = d < a.chunks * AttnElem<T>::kPerChunk;
    float top = -INFINITY, total = 0.f, exact = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    auto join = [&](float4 m, float4 v) {
        const float both = fmaxf(top, m.x), from = both == -INFINITY ? 0.f : both;
        const float f = __builtin_amdgcn_exp2f(top - from), g = __builtin_amdgcn_exp2f(m.x - from);
        top = both, total = total * f + m.y * g, exact = exact * f + m.z * g;
        sum.x = sum.x * f + v.x * g, sum.y = sum.y * f + v.y * g, sum.z = sum.z * f + v.z * g, sum.w = sum.w * f + v.w * g;
    };
    for (int s0 = group; s0 < a.splits; s0 += kSplitsInFlight * GROUPS) {
        float4 m[kSplitsInFlight], v[kSplitsInFlight];
#pragma unroll
        for (int i = 0; i < kSplitsInFlight; ++i) {
            const int s = s0 + i * GROUPS;
            m[i] = make_float4(-INFINITY, 0.f, 0.f, 0.f), v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (s < a.splits) {
                m[i] = *reinterpret_cast<const float4*>(p + s * pitch + DP);
                if (there) v[i] = *reinterpret_cast<const float4*>(p + s * pitch + d);
            }
        }
#pragma unroll
        for (int i = 0; i < kSplitsInFlight; ++i) join(m[i], v[i]);
    }
    if constexpr (GROUPS > 1) {
        __shared__ float4 stats[GROUPS];      // maximum, total, exact total
        __shared__ float4 sums[GROUPS][kLanes];
        if (lane == 0) stats[group] = make_float4(top, total, exact, 0.f);
        sums[group][lane] = sum;
        __syncthreads();
        if (group) return;
        for (int g = 1; g < GROUPS && g < a.splits; ++g) join(stats[g], sums[g][lane]);
    }
    const float inv = total > 0.f ? 1.0f / total : 0.f;
    const int bk = at / rows, row = at - bk * rows, batch = bk / a.kv_heads, kv_head = bk - batch * a.kv_heads;
    const int token = row / a.group, head = kv_head * a.group + row - token * a.group;
    if (there) {
        const int64_t to = batch * a.out_at.batch + token * a.out_at.token + head * a.out_at.head + d;
        const float4 mean = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
        store_piece<true>(static_cast<T*>(a.out) + to, mean);
        if (sizeof(T) == 2 && a.rest) store_piece<true>(static_cast<T*>(a.rest) + to, lost<T>(mean));
    }
    if (lane == 0 && a.lse) a.lse[(static_cast<int64_t>(batch) * a.heads + head) * a.tokens + token] = exact > 0.f ? top + __builtin_amdgcn_logf(exact) : INFINITY;
}

template <typename T, int DP>
constexpr int split_lds() {
    typedef AttnTile<T, DP> Tile;
    constexpr int tiles = kWaves * 2 * 32 * Tile::kRowBytes, out = kWaves * AttnOut<float, DP>::kRoom;
    return tiles > out ? tiles : out;
}

int padded_dim(int64_t dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 96 ? 96 : 128; }

// Row blocks of attention_split, times sequences and key heads.
int64_t split_units(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads) {
    return batch * kv_heads * ((tokens * (heads / kv_heads) + kRows - 1) / kRows);
}

// Does attention_split take it?  A wavefront's 32 rows cost it about twice as much as attention_rows, which has 128 in a workgroup walk over the same
// tile and overlaps the parts of a step; but its workgroups share the keys, while attention_rows takes the longest row's time however few
// workgroups there are.  So: where attention_rows would mostly have rows that do not exist, or where there are not enough workgroups to be worth it
// (measured: [1,512,16,128] bf16 to 4096 keys 41 us here and 70 there, [4,256,16,128] 80 and 81, [16,100,16,128] to 1500 115 and 46; head size 64:
// 31 and 53, 36 and 54, 48 and 29; fp32, whose matrix instructions leave little to overlap: 101 and 311, 156 and 314, 136 and 125).
bool takes_split(const AttnArgs& a, bool wide) {
    int dev;
    const int64_t cus = compute_units(dev), units = split_units(a.batch, a.tokens, a.heads, a.kv_heads);
    const int64_t whole = static_cast<int64_t>(a.batch) * a.heads * ((a.tokens + kRows * kWaves - 1) / (kRows * kWaves));
    const int64_t mean = a.causal ? a.keys - (a.tokens < a.keys ? a.tokens : a.keys) / 2 : a.keys;      // keys of a row
    return units < 2 * whole || 2 * units * mean < (!wide ? 6 : 2 * whole <= cus ? 5 : 3) * cus * a.keys;
}

// Into how many parts it splits the keys: a workgroup for each CU, with at least 256 keys (two tiles of 32 for each of its wavefronts); up to 512 stay
// together, the join costs more (2 x 512 keys, 16 heads of 64: 7.3 us, in two parts 8.5).  [16,1,8,128] bf16 to 4096 keys of one head: 13.5 us, with at
// least 512 keys 16, with 128 13.4 (but one sequence of 65536 keys 22.7 instead of 18.9: the join); two workgroups for each CU:
// [8,1,32,128] to 2048 keys 43 us instead of 39.
int splits_for(int64_t batch, int64_t tokens, int64_t keys, int64_t heads, int64_t kv_heads) {
    if (keys <= 512) return 1;
    int dev;
    const int64_t units = split_units(batch, tokens, heads, kv_heads), most = (keys + 255) / 256;
    const int64_t splits = (compute_units(dev) + units - 1) / units;
    return static_cast<int>(splits < most ? splits : most);
}

}  // namespace
}  // namespace ddl

extern "C" {

int64_t ddl_attention_workspace(int64_t batch, int64_t tokens, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim) {
    using namespace ddl;
    if (!has_work(batch, tokens, keys, heads, kv_heads, dim)) return 0;
    const int splits = splits_for(batch, tokens, keys, heads, kv_heads);
    return splits > 1 ? static_cast<int64_t>(splits) * batch * tokens * heads * (padded_dim(dim) + kStats) : 0;
}

int ddl_attention(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, int dtype,
                  int64_t batch, int64_t tokens, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim, const int32_t* lengths, int causal,
                  float scale, void* out, const int64_t* out_strides, void* out_rest, float* lse, float* workspace, int64_t workspace_elems, void* stream) {
    using namespace ddl;
    AttnArgs a{};
    bool nothing;
    if (const int rc = fill_attention(a, nothing, "ddl_attention", {{q, q_strides}, {k, k_strides}, {v, v_strides}, {out, out_strides}}, dtype, batch, tokens, keys, heads,
                                      kv_heads, dim, lengths, causal, scale))
        return rc;
    if (nothing || tokens == 0) return 0;
    if (out_rest && (dtype == DDL_DT_F32 || !lse)) return fail(DDL_E_ARG, "ddl_attention: only 16-bit results that an adjoint follows have a rest");
    if (!aligned_to(out_rest, 16)) return fail(DDL_E_ALIGN, "ddl_attention: the rest is not 16-byte aligned");
    a.out = out, a.out_at = place_of(out_strides), a.rest = out_rest, a.lse = lse;
    a.splits = splits_for(batch, tokens, keys, heads, kv_heads);
    const int64_t need = ddl_attention_workspace(batch, tokens, keys, heads, kv_heads, dim);
    if (need && (!workspace || workspace_elems < need))
        return fail(DDL_E_ARG, "ddl_attention: workspace of %lld floats, %lld are needed", static_cast<long long>(workspace ? workspace_elems : 0), static_cast<long long>(need));
    if (need && !aligned_to(workspace, 16)) return fail(DDL_E_ALIGN, "ddl_attention: workspace is not 16-byte aligned");
    a.partial = workspace;
    if (lse && !adjoint_launches(a, dtype, dim)) return fail(DDL_E_UNSUPP, "ddl_attention: 2^32 threads in its adjoint");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return with_attention_kernel(dtype, dim, [&](auto* e, auto dp) -> int {
        typedef std::remove_pointer_t<decltype(e)> T;
        constexpr int DP = decltype(dp)::value;
        const auto launch = [&](auto with_lse) {
            constexpr bool LSE = decltype(with_lse)::value;
            if (!takes_split(a, sizeof(T) == 2 && DP > 64)) {
                a.blocks = static_cast<int>(blocks_of(a.tokens));
                const int64_t grid = static_cast<int64_t>(a.blocks) * a.batch * a.heads;
                if (!launches(grid, kThreads)) return fail(DDL_E_UNSUPP, "ddl_attention: 2^32 threads");
                if (const int rc = grant_lds<attention_rows<T, DP, LSE>>(rows_lds<T, DP>(), "ddl_attention")) return rc;
                a.folded = folds(a, grid);
                hipLaunchKernelGGL((attention_rows<T, DP, LSE>), dim3(static_cast<uint32_t>(grid)), dim3(kThreads), (rows_lds<T, DP>()), s, a);
                return check_launch("ddl_attention");
            }
            const int64_t rows = static_cast<int64_t>(a.tokens) * a.group;
            a.blocks = static_cast<int>((rows + kRows - 1) / kRows);
            const int64_t grid = static_cast<int64_t>(a.batch) * a.kv_heads * a.splits * a.blocks;
            if (!launches(grid, kThreads)) return fail(DDL_E_UNSUPP, "ddl_attention: 2^32 threads");
            if (const int rc = grant_lds<attention_split<T, DP, LSE>>(split_lds<T, DP>(), "ddl_attention")) return rc;
            hipLaunchKernelGGL((attention_split<T, DP, LSE>), dim3(static_cast<uint32_t>(grid)), dim3(kThreads), (split_lds<T, DP>()), s, a);
            if (const int rc = check_launch("ddl_attention")) return rc;
            if (a.splits == 1) return 0;
            const int64_t all = static_cast<int64_t>(a.batch) * a.heads * a.tokens;
            constexpr int kGroups = kThreads / join_lanes<DP>();
            if (a.splits <= kSplitsInFlight)
                hipLaunchKernelGGL((attention_join<T, DP, 1>), dim3(static_cast<uint32_t>((all + kGroups - 1) / kGroups)), dim3(kThreads), 0, s, a);
            else
                hipLaunchKernelGGL((attention_join<T, DP, kGroups>), dim3(static_cast<uint32_t>(all)), dim3(kThreads), 0, s, a);
            return check_launch("ddl_attention");
        };
        return lse ? launch(std::true_type{}) : launch(std::false_type{});
    });
}

}  // extern "C"
