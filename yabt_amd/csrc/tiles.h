// Pieces of the matrix products on the matrix cores: tiles fed through LDS, in
// steps of 128 bytes of the summed dimension, and products of few rows straight
// from memory.
#pragma once

#include "expert.h"

namespace yabt {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) float lds_float;
typedef __attribute__((address_space(3))) int lds_int;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;

constexpr int XCDS = 8;               // blocks go to the 8 dies in turn
constexpr int TILE_GROUP = 4;         // row tiles that walk the column tiles together

// 16 zero bytes for pieces past the end of the summed dimension.
__device__ const u32x4 g_zeros = {0, 0, 0, 0};

// BM x BN sums by WM x WN waves, in steps of STEP bytes of the summed dimension;
// LDS holds AS steps of the rows' operand and BS <= AS of the columns'.
template <int BM_, int BN_, int WM_, int WN_, int STEP_, int AS_, int BS_>
struct TileOf {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STEP = STEP_, AS = AS_, BS = BS_;
    static constexpr int NT = 64 * WM * WN;
    static constexpr int MI = BM / WM / 32, NI = BN / WN / 32;    // 32 x 32 blocks a wave makes
    static constexpr int ROWS = BM;                               // of the product
    static constexpr int ABYTES = BM * STEP, BBYTES = BN * STEP;
    static constexpr int LDS = AS * ABYTES + BS * BBYTES;
    static constexpr int NA = ABYTES / 16 / NT, NB = BBYTES / 16 / NT;
    static constexpr int SUMS = BM / MI * BN * 4;                 // 32 rows of every wave, as the sums leave
    static_assert(NA >= 1 && NB >= 1 && NI % 2 == 0, "whole pieces a thread, gate and up in one wave");
    static_assert(LDS <= 160 * 1024 && SUMS + BM * 8 <= LDS && BS <= AS && BM <= NT, "a block's LDS");
};

// Where piece c (16 bytes) of row r of a tile in LDS is kept: c ^ spread(r), so
// that the lanes a read serves at once (16 of 16 bytes, 32 of 8, 64 of 4: 256
// bytes, all banks) meet different banks.  ALONG: a row is STEP bytes of one
// row of the operand; across: a row is one place of the summed dimension, W
// values of the operand's rows.
template <typename T, bool ACROSS, int W, int STEP>
__device__ __forceinline__ constexpr int spread(int r) {
    if (!ACROSS) return STEP == 128 ? r >> 1 & 7 : r >> 2 & 3;
    constexpr int bytes = W * (int)sizeof(T);
    static_assert(!ACROSS || bytes >= 256 || (bytes == 128 && sizeof(T) == 2), "the places stay in their row");
    return sizeof(T) == 4 ? (r >> 2 & 1) << 3 : bytes == 128 ? (r >> 1 & 1) << 2 : (r & 3) << 2;
}

// 1 / (1 + exp(-g)), the gates' factor in silu.  fp32: right to a unit for any g.
// 16 bits: the hardware's exp2 and reciprocal, off by more the larger |g| is, as the
// rounding of g log2 e counts whole in the exponent (y at most 3 units of 2^-24 for
// g near 0, 10 to -10, 18 to -20, 59 to -60; with fp32's 3 everywhere): the rounding
// of h that follows is 2^13 or 2^16 units.  fp32's form costs 2 of 107 us of 20 000 x
// 100 -> 60 of 7, forward and backward.
template <typename T>
__device__ __forceinline__ float gate_sigmoid(float g) {
    if constexpr (sizeof(T) == 4) {
        const float x[1] = {g};
        float p[1];
        sigmoids<1>(x, p);
        return p[0];
    } else {
        return __builtin_amdgcn_rcpf(1.0f + __expf(-g));
    }
}

// 64 lanes' 16 bytes each from memory to LDS at base (the same for the wave),
// in lane order.  By hand, because the compiler waits for all LDS reads at
// every use of one where the builtin is about; it counts as a vector memory
// access, which stage_ready waits for.  m0 is the compiler's reserved register: it
// keeps nothing there from one instruction to another and refuses it as a clobber.
__device__ __forceinline__ void lds_fill(const void* g, uint32_t base) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(base));
}

// Until at most LATER of this wave's vector memory accesses are under way and
// its LDS reads are done, then for the block's other waves: what was sent to
// LDS before the last LATER accesses is there, and the places read last are free.
template <int LATER>
__device__ __forceinline__ void stage_ready() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LATER) : "memory");
}

// The block's place in a grid that is walked die by die: consecutive tiles on
// one die, whose L2 then holds the rows and weights they share.
__device__ __forceinline__ int64_t die_order(int64_t b, int64_t total) {
    const int64_t per = (total + XCDS - 1) / XCDS;
    const int64_t in = b / XCDS;
    return in < per ? (b % XCDS) * per + in : total;
}

// Four values, at an address that is a multiple of four, or (store_part) any:
// the first `have` of them.
template <typename T>
__device__ __forceinline__ void store4(T* p, const float* v) {
    typedef T VT __attribute__((ext_vector_type(4)));
    *(VT*)p = VT{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
}
template <typename T>
__device__ __forceinline__ void store_part(T* p, f32x4 v, int have) {
    typedef T VT __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (have >= 4) {
        *(VT*)p = VT{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    } else {
#pragma unroll
        for (int q = 0; q < 3; ++q)
            if (q < have) p[q] = (T)v[q];
    }
}

// Asks for the order in which MF products and RD LDS reads are issued: the reads
// spread evenly between the products.
template <int MF, int RD, int I = 0>
__device__ __forceinline__ void interleave() {
    if constexpr (I < MF) {
        constexpr int reads = RD * (I + 1) / MF - RD * I / MF;
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if constexpr (reads > 0) __builtin_amdgcn_sched_group_barrier(0x100, reads, 0);
        interleave<MF, RD, I + 1>();
    }
}

template <typename T>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (sizeof(T) == 4) {
        const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[q], fb[q], c, 0, 0, 0);
        return c;
    } else if constexpr (std::is_same_v<T, bf16>) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                      0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                     0, 0);
    }
}

// A lane's 16 bytes of block i of an operand at k-step ks (32 bytes of the
// summed dimension): row (or column) lane % 32, half lane / 32.
template <typename T, bool ACROSS, int W, int STEP>
struct Frag {
    static constexpr int READS = !ACROSS ? 1 : sizeof(T) == 4 ? 4 : 2;   // LDS reads of get()
    static constexpr int KEEP = ACROSS ? 4 : STEP / 32;
    uint32_t at[KEEP];
    __device__ __forceinline__ Frag(int first) {
        const int l = threadIdx.x & 63;
        if constexpr (!ACROSS) {
#pragma unroll
            for (int ks = 0; ks < KEEP; ++ks)
                at[ks] = (uint32_t)((first + (l & 31)) * STEP +
                                    (((ks * 2 + (l >> 5)) ^ spread<T, ACROSS, W, STEP>(l & 31)) << 4));
        } else if constexpr (sizeof(T) == 4) {
            // four rows of k, a value of each; blocks of 32 columns are 128 bytes apart
            const int r = (l >> 5) * 4;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                at[i] = (uint32_t)(r * W * 4 + ((first * 4 + i * 128 + (l & 31) * 4) ^ spread<T, ACROSS, W, STEP>(r) << 4));
        } else {
            // of four rows of k this lane fetches four values of one; blocks are 64 bytes apart
            const int r = (l & 15) >> 2, col = ((l >> 4) & 1) * 16 + (l & 3) * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                at[i] = (uint32_t)(((l >> 5) * 8 + r) * W * 2 + ((first * 2 + i * 64 + col * 2) ^ spread<T, ACROSS, W, STEP>(r) << 4));
        }
    }
    __device__ __forceinline__ u32x4 get(lds_char* tile, int i, int ks) const {
        if constexpr (!ACROSS) {
            return *(const lds_u32x4*)(tile + at[ks] + i * 32 * STEP);
        } else if constexpr (sizeof(T) == 4) {
            f32x4 v;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                v[q] = *(const lds_float*)(tile + at[i & 1] + (ks * 8 + q) * W * 4 + (i >> 1) * 256);
            return __builtin_bit_cast(u32x4, v);
        } else {
            lds_char* p = tile + at[i & 3] + (i >> 2) * 256 + ks * 16 * W * 2;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * W * 2));
            return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

extern __shared__ __attribute__((aligned(128))) char s_tiles[];

template <typename T>
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (sizeof(T) == 4) {
        const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[q], fb[q], c, 0, 0, 0);
        return c;
    } else if constexpr (std::is_same_v<T, bf16>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                      0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                     0, 0);
    }
}

// 16 bytes of a row from value k on, the row's K values alone, zeros after them.
template <typename T>
__device__ __forceinline__ u32x4 row_piece(const T* row, int k, int K) {
    typedef T VT __attribute__((ext_vector_type(VEC<T>)));
    if (k + VEC<T> <= K) return *reinterpret_cast<const u32x4_any*>(row + k);
    VT t = {};
#pragma unroll
    for (int j = 0; j < VEC<T>; ++j)
        if (k + j < K) t[j] = row[k + j];
    return __builtin_bit_cast(u32x4, t);
}

inline int up16(int v, int bytes) { return (v * bytes + 15) / 16 * 16 / bytes; }
inline int64_t over(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether rows of `width` values, ld apart, may be fetched in aligned 16-byte pieces.
inline bool pieces_ok(const void* p, int64_t ld, int width, int bytes) {
    return aligned16(p) && ld * bytes % 16 == 0 && (int64_t)width * bytes % 16 == 0;
}

}  // namespace yabt
