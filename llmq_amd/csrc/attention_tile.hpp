// Building blocks of the attention kernels: bf16 matrix-instruction fragments, the LDS tile with its swizzle, staging from
// global memory, and the careful product for tiles with masked places.
//
// Everything is computed TRANSPOSED: a wave owns 32 positions of one side as the COLUMNS of v_mfma_f32_32x32x16_bf16
// results and walks tiles of the other side as rows.  Lane l = 32 h + c of a result holds column c and the 16 rows
// 8 (i / 4) + 4 h + i % 4.  Two things follow.  Softmax statistics belong to a column, that is to a lane and its partner
// c + 32: no reduction over lanes but one exchange of halves.  And a result is, after rounding to bf16, the right-hand operand
// of the next product as it stands: registers 8 u .. 8 u + 7 are the 16 inner positions 16 u + 8 (j / 4) + 4 h + j % 4, an order
// of the inner index that only has to be the same on both sides, and ds_read_b64_tr_b16 gives the left-hand operand in that
// order (four consecutive inner rows of one column per lane).
#pragma once

#include "common.hpp"

namespace llmq {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_at __attribute__((ext_vector_type(2)));
typedef float f32x2_at __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// Source of a fragment's dimensions beyond head_dim.
__device__ const uint32_t __attribute__((aligned(16))) attention_zeros[4] = {0, 0, 0, 0};

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const f32x2_at p = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2_at));
}

// max / sum over the two lanes of a column
__device__ __forceinline__ float halves_max(float x) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __builtin_fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// registers 8 u .. 8 u + 7 of a result as a right-hand operand
__device__ __forceinline__ bf16x8 operand(const f32x16& x, int u) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pack_bf16(x[8 * u + 2 * j], x[8 * u + 2 * j + 1]);
    return __builtin_bit_cast(bf16x8, w);
}

// Copies from global memory straight into LDS, 16 or 4 bytes a lane, lane i to `lds` (one address for the wave) + 16 i or 4 i, by
// the lanes of `lanes`; source: a 32-bit lane offset from a scalar base.  Inline assembly, because the
// compiler puts a wait for every outstanding copy in front of the next LDS read, whatever it reads; what a kernel reads of a copy
// it reads behind copies_landed().  All lanes are active where a kernel calls these (its branches are the wave's).  The s_nop
// covers, whoever wrote the scalars, the five wait states between a vector instruction that writes a scalar register and a memory
// instruction that reads it, and the one behind a write of M0.
__device__ __forceinline__ uint32_t lds_address(const char* p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p);
}
__device__ __forceinline__ uint32_t to_m0(uint32_t lds) {
    uint32_t m0;
    asm volatile("s_mov_b32 %0, %1" : "={m0}"(m0) : "s"(lds));
    return m0;
}
// (readfirstlane gives a signed int: its low word must not be sign-extended into the high one)
__device__ __forceinline__ uint64_t scalar(uint64_t x) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ void copy16(uint32_t lds, uint32_t offset, const char* base, uint64_t lanes) {
    asm volatile("s_mov_b64 exec, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1\n\ts_mov_b64 exec, -1"
                 : : "v"(offset), "s"(scalar(reinterpret_cast<uint64_t>(base))), "s"(scalar(lanes)), "{m0}"(to_m0(lds)) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t lds, uint32_t offset, const char* base, uint64_t lanes) {
    asm volatile("s_mov_b64 exec, %2\n\ts_nop 4\n\tglobal_load_lds_dword %0, %1\n\ts_mov_b64 exec, -1"
                 : : "v"(offset), "s"(scalar(reinterpret_cast<uint64_t>(base))), "s"(scalar(lanes)), "{m0}"(to_m0(lds)) : "memory");
}
// Waits for this wave's copies and for the other waves' to be waited for.
__device__ __forceinline__ void copies_landed() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Behind the last walk: no copy may outlive the workgroup.
__device__ __forceinline__ void all_copies_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A tile of ROWS rows of HDP bf16 in LDS, row-major, the 16-byte chunks of a row XORed with a function of the row.  A fragment
// read takes one chunk of 32 rows, 16 rows a cycle; a transposed read takes four chunks of four rows a cycle: the low bits of the
// row move the high bits of the chunk, so that the four rows' 64 bytes and the 16 rows' 16 bytes each cover all 64 banks once.
// (With the row's bits XORed in order the transposed reads took 8 cycles instead of 2.)
template <int HDP, int ROWS>
struct Tile {
    static constexpr int kChunks = HDP / 8, kRowBytes = HDP * 2, kBytes = ROWS * kRowBytes;

    static __device__ __forceinline__ int swizzle(int row) {
        return HDP == 128 ? ((row & 3) << 2 | ((row >> 2) & 3)) : ((row & 2) << 1 | ((row >> 2) & 3));
    }

    template <int THREADS>
    static __device__ __forceinline__ void clear(char* lds, int tid) {
        for (int i = tid * 16; i < kBytes; i += THREADS * 16) *reinterpret_cast<uint4*>(lds + i) = make_uint4(0, 0, 0, 0);
    }

    // Left-hand operand, rows of the tile by head dimension: lane -> row 32 rb + l % 32, chunk 2 step + l / 32.
    static __device__ __forceinline__ int row_lane(int lane) {
        return (lane & 31) * kRowBytes + (((lane >> 5) ^ swizzle(lane & 31)) << 4);
    }
    static __device__ __forceinline__ bf16x8 rows(const char* lds, int lane_ofs, int rb, int step) {
        return *reinterpret_cast<const bf16x8*>(lds + (lane_ofs ^ (step << 5)) + rb * 32 * kRowBytes);
    }
    // Left-hand operand, head dimension by rows of the tile (the transposed tile): lane -> dimension 32 db + l % 32 and the rows
    // 16 u + 8 (j / 4) + 4 (l / 32) + j % 4.
    static __device__ __forceinline__ int cols_lane(int lane) {
        const int j = (lane & 15) >> 2, row = 4 * (lane >> 5) + j;
        const int chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        return row * kRowBytes + ((chunk ^ swizzle(row)) << 4) + (lane & 1) * 8;
    }
    static __device__ __forceinline__ bf16x8 cols(char* lds, int lane_ofs, int db, int u) {
        constexpr int kFlip = 32;   // eight rows further the swizzle differs in bit 1
        const int at = lane_ofs ^ (db << 6);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(lds + at + u * 16 * kRowBytes));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(lds + (at ^ kFlip) + (u * 16 + 8) * kRowBytes));
        const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
        return __builtin_bit_cast(bf16x8, (u32x4){a.x, a.y, b.x, b.y});
    }
};

// A lane's part in copying tiles of ROWS rows by THREADS threads, in kCopies copies.  Copies land linearly in LDS, so the swizzle
// picks the source chunk.  Lanes whose chunk lies beyond head_dim copy nothing: their places are cleared once and stay zero.  Rows
// from `limit` on repeat the last one: they are masked.
template <int HDP, int ROWS, int THREADS>
struct TileCopy {
    typedef Tile<HDP, ROWS> T;
    static constexpr int kStep = THREADS / T::kChunks, kCopies = ROWS / kStep;   // rows of a copy
    static_assert(kStep % 16 == 0 && ROWS % kStep == 0, "the swizzle must repeat from copy to copy");
    int row;
    uint32_t chunk;    // bytes into the row
    uint64_t lanes;

    __device__ __forceinline__ TileCopy(int tid, int head_dim) {
        row = tid / T::kChunks;
        const int c = (tid % T::kChunks) ^ T::swizzle(row);
        chunk = c * 16;
        lanes = scalar(__ballot(c * 8 < head_dim));
    }
    // offsets from the tile's first row, row0
    __device__ __forceinline__ void offsets(uint32_t (&ofs)[kCopies], int64_t stride_bytes, int row0, int limit) const {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) ofs[i] = (uint32_t)min(row + i * kStep, limit - 1 - row0) * (uint32_t)stride_bytes + chunk;
    }
    // one copy; lds: address of the tile plus the wave's share, 1024 bytes for each of its number
    __device__ __forceinline__ void copy(int i, uint32_t lds, const uint32_t (&ofs)[kCopies], const char* base) const {
        copy16(lds + i * THREADS * 16, ofs[i], base, lanes);
    }
};

// Splits a left-hand operand into its finite values (zeros in the other places) and a 1 in each place that is not finite.
__device__ __forceinline__ void split_finite(bf16x8 v, bf16x8& finite, bf16x8& other) {
    u32x4 w = __builtin_bit_cast(u32x4, v), f, o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool lo = (w[j] & 0x7F80u) == 0x7F80u, hi = (w[j] & 0x7F800000u) == 0x7F800000u;
        f[j] = w[j] & ((lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u));
        o[j] = (lo ? 0x3F80u : 0u) | (hi ? 0x3F800000u : 0u);
    }
    finite = __builtin_bit_cast(bf16x8, f);
    other = __builtin_bit_cast(bf16x8, o);
}

// acc += a b where places of b that the mask excludes count as absent, whatever a holds there: 0 times an infinity or NaN would
// poison the sum.  `b_allowed` has a 1 in each place that counts.  A sum that meets a value that is not finite in a place that
// counts is NaN.
__device__ __forceinline__ f32x16 careful_product(bf16x8 a, bf16x8 b, bf16x8 b_allowed, f32x16 acc) {
    bf16x8 finite, other;
    split_finite(a, finite, other);
    f32x16 zero;
#pragma unroll
    for (int i = 0; i < 16; ++i) zero[i] = 0.f;
    const f32x16 met = mfma(other, b_allowed, zero);
    acc = mfma(finite, b, acc);
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = met[i] > 0.f ? __builtin_nanf("") : acc[i];
    return acc;
}

}  // namespace llmq
