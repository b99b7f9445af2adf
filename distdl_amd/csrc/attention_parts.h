// What the attention kernels share: tiles of rows in LDS, and the two products that all of them are made of.
//
// A wavefront owns 32 columns (queries forward, keys in the gradients of keys and values), one a lane, lanes l and l + 32
// the same one, and walks over tiles of 32 rows of the other side:
//
//   straight    S[row, column]    = sum over d of tile[row, d] column[d]       scores, and dP from values or gradients
//   transposed  acc[d, column]   += sum over rows of tile[row, d] P[row, column]
//
// with v_mfma_f32_32x32x16 (16-bit types) or v_mfma_f32_32x32x2_f32.  A lane's sixteen results of the first are rows
//   (r & 3) + 8 (r >> 2) + 4 (l >> 5),  r = 0 .. 15,
// of its own column, so a column's maximum and sum need one exchange between the lanes' halves, and the second product
// takes them back as they lie: which row a reduction index stands for is free as long as both operands agree, so the tile is
// read for the rows that each lane happens to hold (16-bit: ds_read_b64_tr_b16, four rows of one column; fp32: a word a row).
// Nothing of P goes through LDS (but from one wavefront to another in attention_backward_pairs).
//
// A tile's rows are DP elements of ROWB bytes, a power of two, in chunks of 16 bytes; chunk c of row r lies at c ^ swizzle(r), a
// permutation of r's low four bits that gives 16 rows of one chunk different banks (straight reads), and the four rows
// of 64 bytes of a transposing read as well.
#ifndef DDL_ATTENTION_PARTS_H
#define DDL_ATTENTION_PARTS_H
#include "ddl_common.h"

#include "gemm_tiles.h"
#include "ln_elements.h"

#include <initializer_list>

namespace ddl {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4v __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) shortx4* lds_shortx4;

// Byte address of a place in LDS: what the reads add their immediate offsets to.
__device__ inline uint32_t lds_address(const void* p) { return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)); }
template <typename V>
__device__ inline V lds_read(uint32_t at) {
    return *(const __attribute__((address_space(3))) V*)static_cast<uintptr_t>(at);
}

template <typename T>
struct AttnElem {
    typedef shortx8 Frag;                 // 16 bytes of a row
    struct Packed {                       // 32 values of a column, for the rows that either half of the lanes holds
        shortx8 lo, hi;
    };
    static constexpr int kPerChunk = 8;
};
template <>
struct AttnElem<float> {
    typedef floatx4v Frag;
    typedef floatx16 Packed;
    static constexpr int kPerChunk = 4;
};

__device__ inline void mfma_chunk(floatx16& acc, const floatx4v& a, const floatx4v& b, const float*) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], acc, 0, 0, 0);
}
__device__ inline void mfma_chunk(floatx16& acc, const shortx8& a, const shortx8& b, const bf16_t*) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8v, a), __builtin_bit_cast(bf16x8v, b), acc, 0, 0, 0);
}
__device__ inline void mfma_chunk(floatx16& acc, const shortx8& a, const shortx8& b, const __half*) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), acc, 0, 0, 0);
}

// Eight values rounded to the 16-bit type, by at most half a step each: 2^-8 of a probability or dS in bf16, 2^-11 in fp16.  The matrix instructions of
// 16-bit types take no others, those of fp32 have a sixteenth of their rate, and keys and values carry the same rounding already; results are off by
// 1.3 to 1.5 times what rounding the exact ones gives (where they are rounded, sums of many average it out).
__device__ inline shortx8 pack8(const floatx16& v, int first, const bf16_t*) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = f32x2_to_bf16(v[first + 2 * i], v[first + 2 * i + 1]);
    shortx8 o;
    __builtin_memcpy(&o, w, 16);
    return o;
}
__device__ inline shortx8 pack8(const floatx16& v, int first, const __half*) {
    halfx8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = static_cast<_Float16>(v[first + i]);
    return __builtin_bit_cast(shortx8, o);
}

// total + two packed values, rounded as they are: a weighted mean's weights then add up to what it is divided by, and a single large one comes
// out as exactly 1.  (Half as many instructions as the sum of the unrounded ones, too.)
__device__ inline float add2(float total, uint32_t v, const bf16_t*) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, v), pair{static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)}, total, false);
}
__device__ inline float add2(float total, uint32_t v, const __half*) {
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(pair, v), pair{static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)}, total, false);
}

template <typename T>
__device__ inline float add8(float total, const shortx8& v, const T* type) {
    uint32_t w[4];
    __builtin_memcpy(w, &v, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) total = add2(total, w[i], type);
    return total;
}

// Eight values of the 16-bit type times a power of two.
__device__ inline shortx8 scale8(const shortx8& v, float factor, const bf16_t*) {
    shortx8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = static_cast<short>(f32_to_bf16(bf16_to_f32(static_cast<uint16_t>(v[i])) * factor));
    return o;
}
__device__ inline shortx8 scale8(const shortx8& v, float factor, const __half*) {
    halfx8 o = __builtin_bit_cast(halfx8, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = static_cast<_Float16>(static_cast<float>(o[i]) * factor);
    return __builtin_bit_cast(shortx8, o);
}

// `N` matrix instructions, behind each of which a share of other work is issued: matrix(i), then the parts of vector(r), r < COUNT, that fall to
// it, in this order -- left to itself the compiler puts one kind behind the other, and then one kind of unit waits.
template <int N, int COUNT, typename M, typename V>
__device__ inline void weave(M&& matrix, V&& vector) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        matrix(i);
#pragma unroll
        for (int r = COUNT * i / N; r < COUNT * (i + 1) / N; ++r) vector(r);
        __builtin_amdgcn_sched_barrier(0);
    }
}
// A value that is computed here and not where it is used.
__device__ inline float pinned(float v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Rows of DP elements of type T in LDS.
template <typename T, int DP>
struct AttnTile {
    typedef typename AttnElem<T>::Frag Frag;
    typedef typename AttnElem<T>::Packed Packed;
    static constexpr int kPerChunk = AttnElem<T>::kPerChunk;
    static constexpr int kBytes = DP * static_cast<int>(sizeof(T));
    static constexpr int kRowBytes = kBytes <= 64 ? 64 : kBytes <= 128 ? 128 : kBytes <= 256 ? 256 : 512;
    static constexpr int kSteps = kBytes / 32;         // of the straight product: a chunk from either half of the lanes
    static constexpr int kBlocks = DP / 32;            // of the transposed product
    static constexpr int kChunks = kBytes / 16;        // of a row
    static_assert(DP % 32 == 0 && kBytes <= 512, "rows of 32 to 128 elements");

    // Linear over exclusive or, so that the parts of a row number that the compiler knows and those of a lane can be permuted apart.
    static constexpr __device__ int swizzle(int row) {
        if (kRowBytes == 64) return (row >> 2) & 3;
        if (kRowBytes == 128) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
        if (sizeof(T) == 2) return ((row & 3) << 2) | ((row >> 2) & 3);
        return (((row >> 2) & 1) << 3) | (row & 3) | (((row >> 3) & 1) << 2);
    }

    // Of this lane, LDS addresses in the block of 32 rows at `base`: its chunk of every straight step; for every 32 columns of the transposed
    // product the first four rows of a lane's half (16-bit), and those eight further down, or its row 0 (fp32).
    static constexpr int kHigh = sizeof(T) == 2 ? kBlocks : 1;
    uint32_t straight_at[kSteps], trans_at[kBlocks], trans_high[kHigh];

    __device__ AttnTile(const char* lds, int lane) {
        const uint32_t base = lds_address(lds);      // of all tiles, which the products name by their byte offsets from here
        const int half = lane >> 5, col = lane & 31;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) straight_at[s] = base + col * kRowBytes + (((2 * s + half) ^ swizzle(col)) << 4);
        if constexpr (sizeof(T) == 2) {   // lane i of 16 points at row i / 4, columns 4 (i % 4) .. + 3 of 16, and receives column i of the four rows
            const int i = lane & 15, row = 4 * half + (i >> 2), chunk = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) {
                trans_at[d] = base + row * kRowBytes + (((4 * d + chunk) ^ swizzle(row)) << 4) + 8 * (i & 1);
                trans_high[d] = base + (row + 8) * kRowBytes + (((4 * d + chunk) ^ swizzle(row + 8)) << 4) + 8 * (i & 1);
            }
        } else {
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) trans_at[d] = base + 4 * half * kRowBytes + (((8 * d + (col >> 2)) ^ swizzle(4 * half)) << 4) + 4 * (col & 3);
        }
    }

    // All places `bytes` further on: to another set of tiles, whose reads then keep their immediate offsets.
    __device__ void shift(int bytes) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) straight_at[s] += bytes;
#pragma unroll
        for (int d = 0; d < kBlocks; ++d) {
            trans_at[d] += bytes;
            if (sizeof(T) == 2) trans_high[d % kHigh] += bytes;
        }
    }

    __device__ Frag read_straight(uint32_t block, int s) const { return lds_read<Frag>(straight_at[s] + block); }
    // 16-bit: what the transposed product of rows 16 k .. + 15 with 32 columns takes.
    __device__ shortx8 read_transposed(uint32_t block, int k, int d) const {
        const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4)static_cast<uintptr_t>((trans_at[d] + block) + 16 * k * kRowBytes));
        const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4)static_cast<uintptr_t>((trans_high[d] + block) + 16 * k * kRowBytes));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }

    // acc[r] += the product of rows 32 block .. + 31 of the tile with this lane's column.
    __device__ void straight(floatx16& acc, uint32_t tile, int block, const Frag (&column)[kSteps]) const {
        const uint32_t base = tile + block * 32 * kRowBytes;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) mfma_chunk(acc, read_straight(base, s), column[s], static_cast<const T*>(nullptr));
        } else {      // four matrix instructions of 64 cycles a read: the next two reads go out in front of them
            Frag a[kSteps];
            a[0] = read_straight(base, 0), a[1] = read_straight(base, 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                if (s + 2 < kSteps) a[s + 2] = read_straight(base, s + 2);
                mfma_chunk(acc, a[s], column[s], static_cast<const T*>(nullptr));
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // The same for the block at `from`, woven with COUNT calls of `vector`; nothing to weave in fp32, whose matrix instructions take most of the time.
    template <int COUNT, typename V>
    __device__ void straight_woven(floatx16& acc, uint32_t from, const Frag (&column)[kSteps], V&& vector) const {
        if constexpr (sizeof(T) == 2) {
            Frag f[kSteps];
            f[0] = read_straight(from, 0), f[1] = read_straight(from, 1);
            __builtin_amdgcn_sched_barrier(0);
            weave<kSteps, COUNT>(
                [&](int i) {
                    if (i + 2 < kSteps) f[i + 2] = read_straight(from, i + 2);
                    mfma_chunk(acc, f[i], column[i], static_cast<const T*>(nullptr));
                },
                vector);
        }
    }

    // A column's 32 values as the transposed product takes them.
    static __device__ Packed pack(const floatx16& p) {
        Packed o;
        if constexpr (sizeof(T) == 2) o.lo = pack8(p, 0, static_cast<const T*>(nullptr)), o.hi = pack8(p, 8, static_cast<const T*>(nullptr));
        else o = p;
        return o;
    }

    // total + the values as packed.
    static __device__ float add_packed(float total, const Packed& p) {
        if constexpr (sizeof(T) == 2) {
            return add8(add8(total, p.lo, static_cast<const T*>(nullptr)), p.hi, static_cast<const T*>(nullptr));
        } else {
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) sum += p[r];
            return total + sum;
        }
    }
    static __device__ void scale_packed(Packed& p, float factor) {
        if constexpr (sizeof(T) == 2) p.lo = scale8(p.lo, factor, static_cast<const T*>(nullptr)), p.hi = scale8(p.hi, factor, static_cast<const T*>(nullptr));
        else p *= factor;
    }

    template <int COUNT, typename V>
    __device__ void transposed_woven(floatx16 (&acc)[kBlocks], uint32_t from, const Packed& p, V&& vector) const {
        if constexpr (sizeof(T) == 2) {
            constexpr int kReads = 2 * kBlocks;
            shortx8 f[kReads];
            f[0] = read_transposed(from, 0, 0), f[1] = read_transposed(from, 1 / kBlocks, 1 % kBlocks);
            __builtin_amdgcn_sched_barrier(0);
            weave<kReads, COUNT>(
                [&](int i) {
                    if (i + 2 < kReads) f[i + 2] = read_transposed(from, (i + 2) / kBlocks, (i + 2) % kBlocks);
                    mfma_chunk(acc[i % kBlocks], f[i], i / kBlocks ? p.hi : p.lo, static_cast<const T*>(nullptr));
                },
                vector);
        }
    }

    // acc[d block] += tile rows 32 block .. + 31, transposed, times p of this lane's column.
    __device__ void transposed(floatx16 (&acc)[kBlocks], uint32_t tile, int block, const Packed& p) const {
        const uint32_t base = tile + block * 32 * kRowBytes;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int d = 0; d < kBlocks; ++d) mfma_chunk(acc[d], read_transposed(base, k, d), k ? p.hi : p.lo, static_cast<const T*>(nullptr));
        } else {
            float v[16][kBlocks];
            auto read = [&](int r) {
                const int row = (r & 3) + 8 * (r >> 2);      // its part of the swizzle reaches chunks by exclusive or
#pragma unroll
                for (int d = 0; d < kBlocks; ++d) v[r][d] = lds_read<float>(((trans_at[d] ^ (swizzle(row) << 4)) + base) + row * kRowBytes);
            };
            read(0), read(1), read(2), read(3);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if (r + 4 < 16) read(r + 4);
#pragma unroll
                for (int d = 0; d < kBlocks; ++d) acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[r][d], p[r], acc[d], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
};

constexpr int64_t kMaxPitch = 1 << 22;      // elements from row to row: 64 rows of 4 bytes each stay below 2^31

// ROWS rows of a tensor straight from memory into a tile, by the WAVES wavefronts of a workgroup, without passing registers: every copy instruction
// fills 1 KiB of the tile, lane after lane, so a lane takes the chunk that belongs where it writes.  Rows from the end on and chunks
// behind the head's own lie outside the buffer that the copies are told of, which gives zeros.
//
// LEAN: one offset a lane and a base for every instruction, scalar work instead of registers.
template <typename T, int DP, int ROWS, int WAVES, bool LEAN = false>
struct AttnCopy {
    typedef AttnTile<T, DP> Tile;
    static constexpr int kSlots = Tile::kRowBytes / 16, kPieces = ROWS * kSlots / (64 * WAVES);
    static_assert(ROWS * kSlots % (64 * WAVES) == 0, "whole instructions for every wavefront");
    // Rows from one instruction of a wavefront to its next; where the swizzle does not change over them, all can have one offset.
    static constexpr int kStep = 64 * WAVES / kSlots;
    static constexpr bool kSame = LEAN && kStep % 16 == 0;
    const char* base;
    int64_t pitch;             // bytes
    int row_bytes, wave;
    uint32_t offset[kSame ? 1 : kPieces];

    __device__ AttnCopy(const T* tensor, int64_t pitch_elems, int chunks, int wave, int lane)
        : base(reinterpret_cast<const char*>(tensor)), pitch(pitch_elems * static_cast<int>(sizeof(T))), row_bytes(16 * chunks), wave(wave) {
#pragma unroll
        for (int i = 0; i < (kSame ? 1 : kPieces); ++i) {
            const int at = (i * WAVES + wave) * 64 + lane, row = at / kSlots, c = (at % kSlots) ^ Tile::swizzle(row);
            offset[i] = c < chunks ? static_cast<uint32_t>(row) * static_cast<uint32_t>(pitch) + 16 * c : 0x7FFFFFF0u;
        }
    }
    // Rows first .. first + ROWS of the tensor, which ends with row `end`.
    __device__ void request(const char* tile, int first, int end) const {
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds_address(tile));
        auto buffer_from = [&](int row) {     // a tile's rows from there on; the same in all lanes, as the instruction wants it
            const int rows = end - row;
            u32x4 buffer = raw_buffer(base + row * pitch);
            buffer[2] = rows > 0 ? static_cast<uint32_t>((rows < ROWS ? rows - 1 : ROWS - 1) * static_cast<uint32_t>(pitch) + row_bytes) : 0u;
#pragma unroll
            for (int i = 0; i < 3; ++i) buffer[i] = __builtin_amdgcn_readfirstlane(buffer[i]);
            return buffer;
        };
        auto place = [&](int i) { return reinterpret_cast<const char*>(static_cast<uintptr_t>(to + (i * WAVES + wave) * 1024)); };
        if constexpr (kSame) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) dma16(buffer_from(first + i * kStep), offset[0], 0, place(i));
        } else {
            const u32x4 buffer = buffer_from(first);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) dma16(buffer, offset[i], 0, place(i));
        }
    }
};

// All requested copies of this wavefront have landed; with a barrier behind it, those of the workgroup.
__device__ inline void wait_for_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// The value of lane l ^ 32 and this lane's, combined.
template <typename Fn>
__device__ inline float both_halves(float v, Fn&& fn) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fn(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float add_halves(float v) {
    return both_halves(v, [](float a, float b) { return a + b; });
}
__device__ inline float max_halves(float v) {
    return both_halves(v, [](float a, float b) { return fmaxf(a, b); });
}

// Barrier of a workgroup whose wavefronts share LDS only: global loads stay in flight across it.
__device__ inline void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// What rounding to T takes from a value.
template <typename T>
__device__ inline float lost(float v) {
    T t;
    store1(&t, v);
    return v - load1(&t);
}
template <typename T>
__device__ inline float4 lost(const float4& v) { return make_float4(lost<T>(v.x), lost<T>(v.y), lost<T>(v.z), lost<T>(v.w)); }

// A wavefront's 32 columns of acc[d block][r] (d = 32 block + (r & 3) + 8 (r >> 2) + 4 half), times `factor`, as rows of DP elements
// in its own room of LDS, kPitch bytes apart.
template <typename T, int DP>
struct AttnOut {
    static constexpr int kPitch = DP * static_cast<int>(sizeof(T)) + 16;
    static constexpr int kRoom = 32 * kPitch;      // bytes for a wavefront
    static constexpr int kBlocks = DP / 32;
    // REST: what the rounding to T takes from them instead.
    template <bool REST = false>
    static __device__ void park(char* room, const floatx16 (&acc)[kBlocks], float factor, int lane) {
        char* row = room + (lane & 31) * kPitch;
        const int half = lane >> 5;
        auto value = [&](float v) { return REST ? lost<T>(v * factor) : v * factor; };
#pragma unroll
        for (int d = 0; d < kBlocks; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                T* at = reinterpret_cast<T*>(row) + 32 * d + 8 * q + 4 * half;
                const float a = value(acc[d][4 * q]), b = value(acc[d][4 * q + 1]), c = value(acc[d][4 * q + 2]), e = value(acc[d][4 * q + 3]);
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<float4*>(at) = make_float4(a, b, c, e);
                } else if constexpr (std::is_same_v<T, bf16_t>) {
                    *reinterpret_cast<uint2*>(at) = make_uint2(f32x2_to_bf16(a, b), f32x2_to_bf16(c, e));
                } else {
                    const __half2 lo = __floats2half2_rn(a, b), hi = __floats2half2_rn(c, e);
                    *reinterpret_cast<uint2*>(at) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
                }
            }
    }
    // Row by row to memory: `place(column)` is where a column's first element goes, null for none; `chunks` of 16 bytes each.
    template <typename Fn>
    static __device__ void write(const char* room, int chunks, int lane, Fn&& place) {
        typedef typename AttnElem<T>::Frag Frag;
        const int all = 32 * chunks;
        for (int i = lane; i < all; i += 64) {
            const int col = i / chunks, c = i - col * chunks;
            T* to = place(col);
            if (to) *reinterpret_cast<Frag*>(to + c * AttnElem<T>::kPerChunk) = *reinterpret_cast<const Frag*>(room + col * kPitch + (c << 4));
        }
    }
};

// ------------------------------------------------------------- arguments --

constexpr int kWave = 64;
constexpr int kWaves = 4;
constexpr int kThreads = kWave * kWaves;
constexpr int kRows = 32;               // columns of a wavefront: rows of the tensor that it works for
constexpr float kLog2e = 1.44269504088896340736f;

struct HeadsAt {                        // of a [batch, tokens, heads, head_dim] tensor: strides in elements
    int64_t batch, token, head;
};
inline HeadsAt place_of(const int64_t* s) { return s ? HeadsAt{s[0], s[1], s[2]} : HeadsAt{0, 0, 0}; }

struct AttnArgs {
    const void *q, *k, *v, *dout;
    void *out, *dq, *dk, *dv;
    void* rest;                         // what out lost to its rounding (as out) or null
    HeadsAt q_at, k_at, v_at, out_at, dout_at, dq_at, dk_at, dv_at;
    float* lse;                         // [batch][heads][tokens], log2
    float* delta;                       // the same, sum of dout out
    const int32_t* lengths;             // [batch] or null
    int tokens, keys, heads, kv_heads, group, batch;
    int chunks;                         // of 16 bytes of a head
    int causal;                         // 0, 1 or kOwnEnds
    float scale, scale_log2;
    int blocks;                         // of rows (or keys) of a head
    int folded;                         // order of the blocks, see block_of
    int splits;                         // of the keys (adjoint of keys: of the queries)
    float* partial;                     // sums of the splits
};

// Of the causal form: the last query sees all keys, up to the tensor's end or the sequence's own.
constexpr int kOwnEnds = 2;
__device__ inline int causal_shift(const AttnArgs& a, int length) { return (a.causal == kOwnEnds ? length : a.keys) - a.tokens; }

// Keys that the query at `token` sees of a sequence of `length`.
__device__ inline int keys_seen(const AttnArgs& a, int token, int length) {
    if (token >= a.tokens) return 0;
    if (!a.causal) return length;
    const int own = token + 1 + causal_shift(a, length);
    return min(length, max(own, 0));
}

__device__ inline int sequence_keys(const AttnArgs& a, int batch) {
    if (!a.lengths) return a.keys;
    const int n = __builtin_amdgcn_readfirstlane(a.lengths[batch]);     // the same in all lanes: into a scalar register
    return n < 0 ? 0 : n < a.keys ? n : a.keys;
}

// Workgroup `id` of `blocks` x `heads`: neighbouring numbers go to different XCDs, each of which takes its own share of the heads,
// so that what they have in common stays in its L2.  Blocks come in descending order, the longest first where a row sees the keys before it;
// `folded`: the second half of them in ascending order.
__device__ inline void block_of(int id, int heads, int blocks, bool folded, int& head, int& block, bool& late) {
    if (heads % 8 == 0) {
        const int share = heads / 8, slot = id >> 3;
        head = (id & 7) * share + slot % share, block = slot / share;
    } else {
        head = id % heads, block = id / heads;
    }
    const int down = blocks / 2;
    late = folded && block >= down;
    block = late ? block - down : blocks - 1 - block;
}

// The sequence with `rank` longer ones before it; up to 64 sequences, in every wavefront for itself.
__device__ inline int sequence_of_rank(const AttnArgs& a, int rank) {
    const int lane = threadIdx.x & (kWave - 1);
    const int n = lane < a.batch ? a.lengths[lane] : 0;
    int before = 0;
    for (int j = 0; j < a.batch; ++j) {
        const int m = __builtin_amdgcn_readlane(n, j);
        before += m > n || (m == n && j < lane) ? 1 : 0;
    }
    return __ffsll(static_cast<unsigned long long>(__ballot(lane < a.batch && before == rank))) - 1;
}

// Sequence and head of number `u` of a workgroup's, `group` heads of which share a key head.  Sequences of equal lengths one after the other, for the
// L2s; of different lengths, every XCD takes heads of all of them, the longest first, and the workgroups that come `late` to a CU the other way round
// (bf16 [8,448,16,64] to 500 .. 1500 keys: forward 37 us instead of 42, dq 45 instead of 51; [32,448,16,64] 94 instead of 106, 117 instead of 129;
// dk and dv of [4,1000,12,128] 80 instead of 112; causal [8,2048,8,128], two key heads, 85 and 85).
__device__ inline void head_of(const AttnArgs& a, int u, int heads, int group, bool late, int& batch, int& head) {
    if (!a.lengths || a.batch == 1) {
        batch = u / heads, head = u - batch * heads;
        return;
    }
    const int key_head = u / (group * a.batch), in = u - key_head * group * a.batch, at = in / group;
    head = key_head * group + in - at * group;
    batch = a.batch <= kWave ? sequence_of_rank(a, late ? a.batch - 1 - at : at) : at;
}

// More LDS than a kernel gets unasked: set once for each kernel and device.
template <auto kernel>
int grant_lds(int bytes, const char* what) {
    static std::atomic<uint64_t> granted{0};   // one bit a device
    int dev;
    compute_units(dev);
    if (granted.load(std::memory_order_relaxed) >> dev & 1) return 0;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return fail(static_cast<int>(e), "%s: %s", what, hipGetErrorString(e));
    granted.fetch_or(1ull << dev, std::memory_order_relaxed);
    return 0;
}

// Where all workgroups of a launch whose lengths differ (causal, or sequences' own) are resident at once, two on a CU, the second one on a CU is one
// of the short half that goes with the long one there (single launches, both in one run: causal, 8192 queries, 8 heads of 128, fp16 178 us instead of
// 186; [4,2048,8,128] 51 instead of 54); with more of them than that, longest first is what levels them.
inline bool folds(const AttnArgs& a, int64_t grid) {
    int dev;
    return (a.causal || a.lengths) && grid <= 2 * static_cast<int64_t>(compute_units(dev));
}

// Extents that the kernels' numbers hold, and heads that share key heads evenly: what the entry points refuse before they divide by any of them.
inline bool counts_fit(int64_t batch, int64_t tokens, int64_t keys, int64_t heads) {
    constexpr int64_t kMost = 0x3FFFFFFF;
    return heads <= kMost && keys <= kMost && (heads == 0 || (tokens <= kMost / heads && batch <= kMost / heads));
}
inline bool heads_fit(int64_t heads, int64_t kv_heads) { return heads == 0 || (kv_heads > 0 && heads % kv_heads == 0); }

// Is there any work of these extents that a workspace could be for?
inline bool has_work(int64_t batch, int64_t tokens, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim) {
    return batch > 0 && tokens > 0 && keys >= 0 && heads > 0 && dim > 0 && dim <= 128 && heads_fit(heads, kv_heads) && counts_fit(batch, tokens, keys, heads);
}

// A launch has fewer than 2^32 threads.
constexpr bool launches(int64_t workgroups, int threads) { return workgroups <= 0xFFFFFFFFll / threads; }
inline int64_t blocks_of(int64_t rows) { return (rows + kRows * kWaves - 1) / (kRows * kWaves); }

// The adjoint's kernel of keys and values takes two sets of wavefronts for 16-bit rows of more than 64 elements.
constexpr bool in_pairs(int element_bytes, int64_t dim) { return element_bytes == 2 && dim > 64; }

// Can the adjoint be launched?  (Only few workgroups are multiplied by splits.)
inline bool adjoint_launches(const AttnArgs& a, int dtype, int64_t dim) {
    return launches(blocks_of(a.tokens) * a.batch * a.heads, kThreads) &&
           launches(blocks_of(a.keys) * a.batch * a.kv_heads, in_pairs(dtype == DDL_DT_F32 ? 4 : 2, dim) ? 2 * kThreads : kThreads);
}

struct HeadsOperand {
    const void* p;
    const int64_t* strides;
};

// The checks and arguments that the entry points share: `operands` are q, k, v and others like q.  0 or a refusal;
// `nothing`: there are no queries to work for.
inline int fill_attention(AttnArgs& a, bool& nothing, const char* what, std::initializer_list<HeadsOperand> operands, int dtype, int64_t batch, int64_t tokens,
                          int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim, const int32_t* lengths, int causal, float scale) {
    if (batch < 0 || tokens < 0 || keys < 0 || heads < 0 || kv_heads < 0 || dim < 1) return fail(DDL_E_ARG, "%s: negative extent or empty heads", what);
    if (dtype != DDL_DT_F32 && dtype != DDL_DT_BF16 && dtype != DDL_DT_F16) return fail(DDL_E_ARG, "%s: dtype %d", what, dtype);
    if (dim > 128) return fail(DDL_E_UNSUPP, "%s: heads of %lld elements (at most 128)", what, static_cast<long long>(dim));
    const int per = dtype == DDL_DT_F32 ? 4 : 8;
    if (dim % per) return fail(DDL_E_ALIGN, "%s: heads of %lld elements are no multiple of 16 bytes", what, static_cast<long long>(dim));
    if (!(scale > 0.f && scale <= 1.0e38f)) return fail(DDL_E_ARG, "%s: scale %g is not positive", what, static_cast<double>(scale));
    if (!heads_fit(heads, kv_heads))
        return fail(DDL_E_SHAPE, "%s: %lld heads cannot share %lld key heads", what, static_cast<long long>(heads), static_cast<long long>(kv_heads));
    if (!counts_fit(batch, tokens, keys, heads)) return fail(DDL_E_UNSUPP, "%s: 2^30 rows or keys", what);
    if (heads == 0 && kv_heads) return fail(DDL_E_SHAPE, "%s: key heads without heads", what);
    nothing = batch == 0 || heads == 0 || (tokens == 0 && keys == 0);
    if (nothing) return 0;
    int i = 0;
    for (const HeadsOperand& o : operands) {
        const bool of_keys = i == 1 || i == 2;
        if ((of_keys ? keys : tokens) && (!o.p || !o.strides)) return fail(DDL_E_ARG, "%s: null tensor", what);
        if (o.p && o.strides) {
            if (o.strides[0] % per || o.strides[1] % per || o.strides[2] % per) return fail(DDL_E_ALIGN, "%s: strides are no multiples of 16 bytes", what);
            if (!aligned_to(o.p, 16)) return fail(DDL_E_ALIGN, "%s: operands are not 16-byte aligned", what);
            if (o.strides[1] < 0 || o.strides[1] >= kMaxPitch) return fail(DDL_E_UNSUPP, "%s: rows 2^22 elements apart", what);
        }
        HeadsAt at = place_of(o.strides);
        const int64_t rows = of_keys ? keys : tokens;
        if (rows <= 1) at.token = dim;      // nothing is ever that far away
        else if (o.p && at.token < dim) return fail(DDL_E_UNSUPP, "%s: rows that overlap", what);
        if (i == 0) a.q = o.p, a.q_at = at;
        if (i == 1) a.k = o.p, a.k_at = at;
        if (i == 2) a.v = o.p, a.v_at = at;
        ++i;
    }
    a.lengths = lengths;
    a.tokens = static_cast<int>(tokens), a.keys = static_cast<int>(keys), a.heads = static_cast<int>(heads), a.kv_heads = static_cast<int>(kv_heads);
    a.group = static_cast<int>(heads / kv_heads), a.batch = static_cast<int>(batch), a.chunks = static_cast<int>(dim / per), a.causal = causal == kOwnEnds ? kOwnEnds : causal != 0;
    a.scale = scale, a.scale_log2 = scale * kLog2e;
    return 0;
}

// Calls fn(element, head size): the element type that `dtype` names and the smallest supported row of at least `dim`.
template <typename Fn>
inline int with_attention_kernel(int dtype, int64_t dim, Fn&& fn) {
    int rc = DDL_E_ARG;
    with_ln_element(dtype, [&](auto* e) {
        if (dim <= 32) rc = fn(e, std::integral_constant<int, 32>{});
        else if (dim <= 64) rc = fn(e, std::integral_constant<int, 64>{});
        else if (dim <= 96) rc = fn(e, std::integral_constant<int, 96>{});
        else rc = fn(e, std::integral_constant<int, 128>{});
    });
    return rc;
}

}  // namespace ddl
#endif  // DDL_ATTENTION_PARTS_H
