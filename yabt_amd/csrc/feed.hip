// The dense stage's products on the matrix cores: a gated feed-forward block,
// forward and backward, and products of 8-bit integers.
//
//   [g u] = x W_in^T,  h = act(g) u,  y = h W_out^T
//   dh = dy W_out,  du = dh act(g),  dg = dh u act'(g)
//   dx = [dg du] W_in,  dW_in = [dg du]^T x,  dW_out = dy^T h
//   8 bits:  x_ij = q_ij s_i,  w_oj = p_oj t_o  (q, p whole numbers):  (x w^T)_io = s_i t_o sum_j q_ij p_oj
//
// One kernel makes the tiles of all these products; they differ in whether an
// operand lies along the summed dimension in memory or across it, and in what
// is done with the sums:
//
//   IN, IN8     a tile's columns are gate and up alternately by 32; h = act(g) u leaves it
//   OUT, OUT8   x w^T as it is; the sums of whole numbers times their rows' and columns' scales
//   DH          dh, which becomes dg and du on the spot
//   DX, DWIN, DWOUT   the gradients, side by side in one grid
//
// Both operands pass through LDS in steps of 128 bytes of the summed dimension:
// an instruction takes 32 of them a row whatever they hold, so that 8-bit products
// are the 16-bit ones with twice the values.  Operands across the summed dimension
// are read with the transposing LDS loads.  Few rows have kernels of their own,
// which are bound by the weights' bytes.
//
// 8192 x 2048 -> 5632 -> 2048, bf16, forward and backward: h with g and u kept 366 us (378 GFLOP), y
// 150 (189), the inner gradient 284 (189), the three others 722 (945): 1030, 1260, 670 and 1310
// TFLOP/s, the matrix cores at work 54, 74, 37 and 74% of the time; the library's plain products of
// these sizes reach 980 to 1510.  What is between them: a block has its CU to itself, so that the end of
// a tile, where all CUs read and write at once (h with g and u 0.46 GB, the inner gradient 0.55 GB), is
// not covered, and neither is its first step; and h has 5.5 rounds of 256 tiles.
// 8192 x 4096 x 4096 in 8 bits: 133 us, 2070 TOP/s (the library's reaches 2110 at 8192 x 8192 x 8192).
// 4096 x 2048 -> 4096 -> 2048, fp32: 1030 us, 200 TFLOP/s (the library's fp32 product: 153).
//
// 16-bit types: h, dg and du are rounded to the inputs' type, as the matrix cores
// take them; g and u are kept in fp32 for the backward pass.  So an output has
// two roundings behind it, its own and that of one factor, and 1.41 times the error
// of its own, where many values average.  In a small block (twice_ok) one large
// value may decide, and the error was up to 2.2 times; there h, dg and du are kept in
// two parts of the type, 16 bits or more, and their products made of both.  y of
// 16 rows or fewer, whose time is the weights', takes h in two parts too, unless the
// block is so wide that y goes by tiles.  8 bits: h is kept in fp32 until its row's
// largest magnitude is known, sums of codes are whole numbers.

#include "tiles.h"
#include "yabt_hip.h"

namespace yabt {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

enum Mode { IN, IN8, OUT, OUT8, DH, DX, DWIN, DWOUT };
enum Act { SILU, GELU, GELU_TANH, RELU };

// One product of M rows by N columns (IN: N of h) over K.
struct Product {
    const void* a;                    // the rows' operand and the columns', lda and ldb values from row to row
    const void* b;
    int64_t lda, ldb;
    int M, N, K;
    int aw, bw;                       // an operand across K: its width in memory
    int F, Fp, Fi;                    // inner width; up to whole 16 bytes: the pitch of h, half of [dg du]'s; up to a
                                      // multiple of 4
    int act;
    float* pre;                       // (M, 2 Fi): g from 0, u from Fi, or NULL
    void* h;                          // (M, Fp), or NULL
    float* h32;                       // (M, Fi): h of 8-bit products and of 16 rows or fewer, or NULL
    void* dpre;                       // (M, 2 Fp): dg from 0, du from Fp
    void* out;
    int64_t ldo;
    int out_dtype;
    const float* sa;                  // scales of rows and columns (IN8: of gates, then of u)
    const float* sb;
    float* part;                      // (splits, M, N) where splits > 1: the sums in part (8 bits: as int32); IN
                                      // (splits, M, 2 Fi): of g from 0, of u from Fi; DH (splits, M, Fi)
    int splits;
    int x_dtype;                      // few rows of 8 bits: the type of a's values
    int64_t again;                    // values from h's, or dpre's, first part to its second, 0: it has one
    int64_t again_a, again_b;         // the same of an operand in two parts (TWICE); of the other 0
};

template <typename T> struct Sums { using Four = f32x4; using Block = f32x16; };
template <> struct Sums<int8_t> { using Four = i32x4; using Block = i32x16; };

__device__ __forceinline__ i32x16 mma8(u32x4 a, u32x4 b, i32x16 c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ i32x4 mma8(u32x4 a, u32x4 b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// The activation of four gates and its derivative.  16 bits: the hardware's exp2 and
// reciprocal (gate_sigmoid), and for the normal distribution function normal_tail.  8 bits too: with
// U = 2^-24, silu's and gelu_tanh's factor is off by (8 + 10 |z|) U of itself at most (z the sigmoid's argument), gelu's
// by (20 + 2 g^2) U, so that h of gates to -8 (silu: to -20) is within 2^-16 and has another code once in
// some 250 times at worst, near 0 once in thousands; the accurate functions
// made h of 16 384 x 2048 -> 5632 take 466 us instead of 415.  fp32: the accurate functions.
//
// Phi(-a) / exp(-a^2 / 2), a >= 0, is half the scaled complementary error function of x = a / sqrt(2).
// In t = 1 / (1 + 0.33 x) it is t times a polynomial, fitted here to the least largest relative error, 2^-23.5 for x to
// 9.5 (beyond, the exponential is 0): relative, because a negative gate's whole factor is this tail.
__device__ __forceinline__ float normal_tail(float a) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.23334524f, a, 1.0f));
    float p = fmaf(-0.0679644f, t, 0.23134412f);
    p = fmaf(p, t, -0.17771947f);
    p = fmaf(p, t, 0.2062708f);
    p = fmaf(p, t, 0.022505322f);
    p = fmaf(p, t, 0.100961916f);
    p = fmaf(p, t, 0.091418624f);
    p = fmaf(p, t, 0.093183056f);
    return p * t;
}
// The normal distribution function at g and exp(-g^2 / 2).
template <typename T>
__device__ __forceinline__ float gate_normal(float g, float* density) {
    const float e = -0.5f * g * g;
    float tail;                        // of the distribution, beyond |g|
    if constexpr (sizeof(T) != 4) {
        *density = __expf(e);
        tail = normal_tail(fabsf(g)) * *density;
    } else {
        *density = expf(e);
        tail = 0.5f * erfcf(fabsf(g) * 0.70710678f);
    }
    return g > 0.0f ? 1.0f - tail : tail;
}
template <typename T>
__device__ __forceinline__ void activate(int act, f32x4 g, float (&v)[4], float (&slope)[4]) {
    switch (act) {
        case SILU:
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float s = gate_sigmoid<T>(g[q]);
                v[q] = g[q] * s;
                slope[q] = s * (1.0f + g[q] * (1.0f - s));
            }
            break;
        case GELU:
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float d;
                const float p = gate_normal<T>(g[q], &d);
                v[q] = g[q] * p;
                // far out the density is 0, and an infinite g times it too
                slope[q] = p + (d > 0.0f ? g[q] * 0.39894228f * d : 0.0f);
            }
            break;
        case GELU_TANH:
            // 0.5 (1 + tanh(z)) = sigmoid(2 z); where g^2 is held at 10^8 it is 0 or 1 already
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float g2 = fminf(g[q] * g[q], 1e8f);
                const float s = gate_sigmoid<T>(1.5957691216f * g[q] * (1.0f + 0.044715f * g2));
                v[q] = g[q] * s;
                slope[q] = s + g[q] * s * (1.0f - s) * 1.5957691216f * (1.0f + 0.134145f * g2);
            }
            break;
        default:
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                v[q] = g[q] <= 0.0f ? 0.0f : g[q];
                slope[q] = g[q] > 0.0f ? 1.0f : 0.0f;
            }
    }
}

// As lds_fill, from an address that is the same for the wave and 32 bits of its lanes' own.
__device__ __forceinline__ void lds_fill_from(const char* from, uint32_t off, uint32_t base) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(from), "s"(base));
}

// The pieces of an operand that a thread brings to LDS.  Pieces past the end of the
// summed dimension are zero, rows and columns past the product's end repeat the last
// (their sums are not stored).
// PAIR: the rows' operand in two parts of the type, their rows alternately by 32.
template <typename T, int MODE, bool SIDE_B, int W, int COUNT, int NT, int STEP, bool PAIR = false>
struct Loader {
    static constexpr bool ACROSS = SIDE_B ? MODE >= DH : MODE >= DWIN;
    static constexpr bool GATED = SIDE_B && (MODE == IN || MODE == IN8);
    static constexpr int CH = VEC<T>;
    static constexpr int PER_ROW = ACROSS ? W * (int)sizeof(T) / 16 : STEP / 16;
    const T* ptr[COUNT];       // along: the row, at this piece; across: column of the piece, from row 0
    // straight to LDS: bytes from where the tile begins, which is the same for the block and moves with the step, so
    // that a step's addresses cost no vector instruction (8192 x 2048, 5632, forward and backward: 1493 us, and
    // 1609 with 64-bit addresses a lane)
    uint32_t off[COUNT];
    const char* begin;
    size_t step;               // bytes from one step to the next

    __device__ __forceinline__ static int row_of(int i) { return (i * NT + (int)threadIdx.x) / PER_ROW; }
    __device__ __forceinline__ static int piece_of(int i) {
        const int c = (i * NT + (int)threadIdx.x) % PER_ROW, r = row_of(i);
        return c ^ spread<T, ACROSS, W, STEP>(r);
    }
    __device__ __forceinline__ static int width(const Product& P) { return SIDE_B ? P.bw : P.aw; }

    // first: the tile's first row or column of the operand; lo: where its steps begin
    __device__ __forceinline__ void init(const Product& P, int first, int lo) {
        const T* const base = (const T*)(SIDE_B ? P.b : P.a);
        const size_t ld = (size_t)(SIDE_B ? P.ldb : P.lda);
        begin = (const char*)(ACROSS ? base + (size_t)lo * ld + first : base + (size_t)first * ld + lo);
        step = ACROSS ? STEP / sizeof(T) * ld * sizeof(T) : STEP;
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const int r = row_of(i), piece = piece_of(i) * CH;
            if constexpr (GATED) {
                // gate and up rows alternately by 32
                const int f = min(first + (r >> 6) * 32 + (r & 31), P.F - 1);
                ptr[i] = base + (size_t)((r >> 5 & 1 ? P.F : 0) + f) * ld + piece;
                off[i] = (uint32_t)((r >> 5 & 1 ? P.F : 0) + f - first) * (uint32_t)(ld * sizeof(T)) + piece * sizeof(T);
            } else if constexpr (PAIR) {
                static_assert(!SIDE_B && !ACROSS, "of the rows' operand along the summed dimension");
                const int row = min(first + (r >> 6) * 32 + (r & 31), P.M - 1);
                const size_t part = r >> 5 & 1 ? (size_t)P.again_a : 0;
                ptr[i] = base + (size_t)row * ld + piece + part;
                off[i] = (uint32_t)(row - first) * (uint32_t)(ld * sizeof(T)) + (piece + (uint32_t)part) * sizeof(T);
            } else if constexpr (!ACROSS) {
                const int row = min(first + r, (SIDE_B ? P.N : P.M) - 1);
                ptr[i] = base + (size_t)row * ld + piece;
                off[i] = (uint32_t)(row - first) * (uint32_t)(ld * sizeof(T)) + piece * sizeof(T);
            } else {
                const int column = min(first + piece, max(width(P) - CH, 0));
                ptr[i] = base + column;
                off[i] = (uint32_t)r * (uint32_t)(ld * sizeof(T)) + (uint32_t)(column - first) * sizeof(T);
            }
        }
    }

    // where piece i of the step from k0 on lies, or null past the end
    __device__ __forceinline__ const T* at(const Product& P, int i, int k0, int end) const {
        if constexpr (!ACROSS) {
            return k0 + piece_of(i) * CH < end ? ptr[i] + k0 : nullptr;
        } else {
            int kk = k0 + row_of(i);
            if (kk >= end) return nullptr;
            if constexpr (MODE == DX) {
                // [dg du] has du from Fp on, W_in its rows from F on
                if (kk >= P.F) {
                    if (kk < P.Fp) return nullptr;
                    kk += P.F - P.Fp;
                }
            }
            return ptr[i] + (size_t)kk * (size_t)(SIDE_B ? P.ldb : P.lda);
        }
    }

    // pieces LO .. HI - 1 of step t, which begins at k0 (at the end or before it), `again` values further on
    template <int LO = 0, int HI = COUNT>
    __device__ __forceinline__ void fill(const Product& P, int t, int k0, int end, uint32_t lds, int64_t again = 0) const {
        auto place = [&](int i) {
            return __builtin_amdgcn_readfirstlane(lds + (uint32_t)(i * NT * 16) + ((threadIdx.x & ~63u) << 4));
        };
        if (k0 + STEP / (int)sizeof(T) <= end) {
            const char* const from = begin + (size_t)t * step + (size_t)again * sizeof(T);
#pragma unroll
            for (int i = LO; i < HI; ++i) lds_fill_from(from, off[i], place(i));
        } else {
#pragma unroll
            for (int i = LO; i < HI; ++i) {
                const T* p = at(P, i, k0, end);
                lds_fill(p ? (const void*)(p + again) : (const void*)&g_zeros, place(i));
            }
        }
    }

    // the same through registers, for rows at any address: the values that
    // exist, zeros for the others
    __device__ __forceinline__ void fetch(const Product& P, int k0, int end, int first, u32x4* v, int64_t again = 0) const {
        typedef T VT __attribute__((ext_vector_type(CH)));
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const T* p = at(P, i, k0, end);
            u32x4 o = {0, 0, 0, 0};
            if (p) {
                const int piece = piece_of(i) * CH;
                int have;
                p += again;
                if constexpr (ACROSS) {
                    // the column clamp of init() does not hold pieces that end past the row
                    const int w = width(P);
                    p += first + piece - min(first + piece, max(w - CH, 0));
                    have = w - (first + piece);
                } else {
                    have = end - (k0 + piece);
                }
                if (have >= CH) o = *reinterpret_cast<const u32x4_any*>(p);
                else {
                    VT t = {};
#pragma unroll
                    for (int j = 0; j < CH; ++j)
                        if (j < have) t[j] = p[j];
                    o = __builtin_bit_cast(u32x4, t);
                }
            }
            v[i] = o;
        }
    }
    __device__ __forceinline__ static void put(lds_char* tile, const u32x4* v) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) *(lds_u32x4*)(tile + (i * NT + (int)threadIdx.x) * 16) = v[i];
    }
};

// fp32 values in three parts of bf16, 8 bits of the significand each: x = hi + mid + lo exactly, each
// part cut off, so that none is larger than x.  A product of two has nine products of parts; the
// three smallest are left out.  mid ends at 2^-7 of x and lo at 2^-15, so they are up to 2^-21 of the product
// together, 2^-24.5 on average, and have its sign: sums of terms of one sign come out low by as much (with nearest parts
// they would not, but values next to the largest would become infinite).  A part ends at bf16's least step, 2^-133:
// values below 2^-110 are taken to that.
__device__ __forceinline__ void in_parts(u32x4 a, u32x4 b, u32x4 (&part)[3]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        uint32_t x[2], r[2], l[2];
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            const int at = 2 * q + o;
            x[o] = at < 4 ? a[at] : b[at - 4];
            r[o] = __float_as_uint(__uint_as_float(x[o]) - __uint_as_float(x[o] & 0xFFFF0000u));
            l[o] = __float_as_uint(__uint_as_float(r[o]) - __uint_as_float(r[o] & 0xFFFF0000u));
        }
        part[0][q] = __builtin_amdgcn_perm(x[1], x[0], 0x07060302u);     // the upper halves of both
        part[1][q] = __builtin_amdgcn_perm(r[1], r[0], 0x07060302u);
        part[2][q] = __builtin_amdgcn_perm(l[1], l[0], 0x07060302u);
    }
}

// BM x BN sums of fp32 by WM x WN waves, in steps of 32 places of the summed dimension; LDS
// holds two steps of both operands, in three parts of bf16.
template <int BM_, int BN_, int WM_, int WN_>
struct TileParts {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STEP = 128;
    static constexpr int NT = 64 * WM * WN;
    static constexpr int MI = BM / WM / 32, NI = BN / WN / 32, ROWS = BM;
    static constexpr int APART = BM * 64, BPART = BN * 64, PLACE = 3 * (APART + BPART);   // a part's bytes, a step's
    static constexpr int LDS = 2 * PLACE;
    static constexpr int NA = APART / 16 / NT, NB = BPART / 16 / NT;                      // pieces of 8 values a thread
    static_assert(NA >= 1 && NB >= 1 && NI % 2 == 0, "whole pieces a thread, gate and up in one wave");
    static_assert(LDS <= 160 * 1024 && BM / MI * BN * 4 <= LDS, "a block's LDS");
};

// The pieces (8 values) of an fp32 operand that a thread brings to LDS in parts: laid out as bf16 in
// steps of 64 bytes.
template <int MODE, bool SIDE_B, int W, int COUNT, int NT>
struct PartsLoader {
    using Layout = Loader<bf16, MODE, SIDE_B, W, COUNT, NT, 64>;
    static constexpr bool ACROSS = Layout::ACROSS;
    const float* ptr[COUNT];
    u32x4 v[2][COUNT][2];      // two steps' pieces on their way

    __device__ __forceinline__ void init(const Product& P, int first) {
        const float* const base = (const float*)(SIDE_B ? P.b : P.a);
        const size_t ld = (size_t)(SIDE_B ? P.ldb : P.lda);
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const int r = Layout::row_of(i);
            if constexpr (Layout::GATED) {
                const int f = min(first + (r >> 6) * 32 + (r & 31), P.F - 1);
                ptr[i] = base + (size_t)((r >> 5 & 1 ? P.F : 0) + f) * ld;
            } else if constexpr (!ACROSS) {
                ptr[i] = base + (size_t)min(first + r, (SIDE_B ? P.N : P.M) - 1) * ld;
            } else {
                ptr[i] = base + min(first + Layout::piece_of(i) * 8, Layout::width(P) - 1);
            }
        }
    }
    // the step from k0 on; what does not exist is zero
    template <int SET>
    __device__ __forceinline__ void fetch(const Product& P, int k0, int end, int first) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const float* p = ptr[i];
            int have;
            if constexpr (!ACROSS) {
                const int k = k0 + Layout::piece_of(i) * 8;
                have = end - k;
                p += k;
            } else {
                int kk = k0 + Layout::row_of(i);
                have = kk < end ? Layout::width(P) - (first + Layout::piece_of(i) * 8) : 0;
                if constexpr (MODE == DX) {
                    // [dg du] has du from Fp on, W_in its rows from F on
                    if (kk >= P.F) {
                        if (kk < P.Fp) have = 0;
                        kk += P.F - P.Fp;
                    }
                }
                p += (size_t)kk * (size_t)(SIDE_B ? P.ldb : P.lda);
            }
            u32x4 a = {0, 0, 0, 0}, b = a;
            if (have >= 8) {
                a = *reinterpret_cast<const u32x4_any*>(p);
                b = *reinterpret_cast<const u32x4_any*>(p + 4);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (q < have) a[q] = __float_as_uint(p[q]);
#pragma unroll
                for (int q = 0; q < 3; ++q)
                    if (q + 4 < have) b[q] = __float_as_uint(p[q + 4]);
            }
            v[SET][i][0] = a;
            v[SET][i][1] = b;
        }
    }
    template <int SET>
    __device__ __forceinline__ void put(lds_char* tile) const {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            u32x4 part[3];
            in_parts(v[SET][i][0], v[SET][i][1], part);
#pragma unroll
            for (int o = 0; o < 3; ++o) *(lds_u32x4*)(tile + o * (W * 64) + (i * NT + (int)threadIdx.x) * 16) = part[o];
        }
    }
};

// acc += the tile's products over [lo, end) in parts.  The upper parts' products have sums of their
// own, which are rounded once a product; those of the small ones join them at the end.
template <int MODE, typename TL>
__device__ __forceinline__ void parts_sums(const Product& P, int mf, int nf, int lo, int end, int steps,
                                           f32x16 (&acc)[TL::MI][TL::NI]) {
    lds_char* const lds = (lds_char*)s_tiles;
    const int wave = threadIdx.x / 64, wm = wave / TL::WN, wn = wave % TL::WN;
    PartsLoader<MODE, false, TL::BM, TL::NA, TL::NT> la;
    PartsLoader<MODE, true, TL::BN, TL::NB, TL::NT> lb;
    la.init(P, mf);
    lb.init(P, nf);
    const Frag<bf16, decltype(la)::ACROSS, TL::BM, 64> fa(wm * TL::MI * 32);
    const Frag<bf16, decltype(lb)::ACROSS, TL::BN, 64> fb(wn * TL::NI * 32);
    auto fetch = [&](auto set, int t) {
        if (t >= steps) return;
        la.template fetch<decltype(set)::value>(P, lo + t * 32, end, mf);
        lb.template fetch<decltype(set)::value>(P, lo + t * 32, end, nf);
    };
    auto put = [&](auto set) {
        lds_char* const place = lds + decltype(set)::value * TL::PLACE;
        la.template put<decltype(set)::value>(place);
        lb.template put<decltype(set)::value>(place + 3 * TL::APART);
    };
    f32x16 small[TL::MI][TL::NI];
#pragma unroll
    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
        for (int j = 0; j < TL::NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) small[i][j][r] = 0.0f;
    auto products = [&](auto set) {
        lds_char* const ta = lds + decltype(set)::value * TL::PLACE;
        lds_char* const tb = ta + 3 * TL::APART;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            u32x4 a[3][TL::MI], b[3][TL::NI];
#pragma unroll
            for (int o = 0; o < 3; ++o) {
#pragma unroll
                for (int i = 0; i < TL::MI; ++i) a[o][i] = fa.get(ta + o * TL::APART, i, ks);
#pragma unroll
                for (int j = 0; j < TL::NI; ++j) b[o][j] = fb.get(tb + o * TL::BPART, j, ks);
            }
#pragma unroll
            for (int sum = 2; sum >= 0; --sum)
#pragma unroll
                for (int o = 0; o <= sum; ++o)
#pragma unroll
                    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
                        for (int j = 0; j < TL::NI; ++j) {
                            f32x16& to = sum ? small[i][j] : acc[i][j];
                            to = mma<bf16>(a[o][i], b[sum - o][j], to);
                        }
        }
    };
    constexpr std::integral_constant<int, 0> even;
    constexpr std::integral_constant<int, 1> odd;
    fetch(even, 0);
    fetch(odd, 1);
    put(even);
    fetch(even, 2);
    for (int t = 0; t < steps; t += 2) {
        __syncthreads();                         // step t is there, and what was read of the other place is read
        if (t + 1 < steps) put(odd);
        fetch(odd, t + 3);
        products(even);
        if (t + 1 >= steps) break;
        __syncthreads();
        if (t + 2 < steps) put(even);
        fetch(even, t + 4);
        products(odd);
    }
#pragma unroll
    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
        for (int j = 0; j < TL::NI; ++j) acc[i][j] += small[i][j];
    __syncthreads();                             // the sums leave through the same LDS
}

// What is left of v beside its first part, or beside the type's largest value where that is infinite: infinity less
// infinity would be NaN, which the product's sum then is.
template <typename T>
__device__ __forceinline__ float second_part(float v, T first) {
    constexpr float most = std::is_same_v<T, f16> ? 65504.0f : std::is_same_v<T, bf16> ? 0x1.FEp127f : 0x1.FFFFFEp127f;
    return v - __builtin_amdgcn_fmed3f((float)first, -most, most);
}

// Up to four values at p in the type that a run-time number names.
__device__ __forceinline__ void store_as(int dtype, void* p, size_t at, f32x4 v, int have) {
    if (dtype == DT_F32) store_part((float*)p + at, v, have);
    else if (dtype == DT_BF16) store_part((bf16*)p + at, v, have);
    else store_part((f16*)p + at, v, have);
}

// Four values from p on, those that exist.
__device__ __forceinline__ f32x4 four_of(const float* p, int have) {
    typedef f32x4 f32x4_any __attribute__((aligned(4)));
    if (have >= 4) return *(const f32x4_any*)p;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int q = 0; q < 3; ++q)
        if (q < have) v[q] = p[q];
    return v;
}

// The product's M in the rows of its output, and output row of tile row m, M or more if none:
// dW_in's rows lie in [dg du] with a gap behind F.
template <int MODE>
__device__ __forceinline__ int out_row(const Product& P, int m) {
    if constexpr (MODE == DWIN) return m < P.F ? m : m < P.Fp ? INT32_MAX : m + P.F - P.Fp;
    return m;
}

// The tiles of a product that a grid makes: mt x nt x splits, or `count` of them from `first` on,
// by `blocks` thread blocks (a multiple of XCDS, so that a block's number tells its die).
struct Tiles {
    int nt, mt;
    uint32_t first, count, blocks;
};

// Small tiles of a product with an operand in two parts of the type.  Of the rows' operand along the summed
// dimension both parts are rows of one tile, so that the columns' is read once (PAIR); else every step is made twice,
// of the first part and of the second, the other operand the same (TWICE: dW_in and dW_out, whose sums over a small
// block's rows have few steps).
struct TilePair : TileOf<128, 128, 2, 2, 128, 2, 2> { static constexpr int ROWS = 64; };
struct TileTwice : TileOf<64, 128, 2, 2, 128, 2, 2> {};
template <typename TL> constexpr bool PAIR = std::is_same_v<TL, TilePair>;
template <typename TL> constexpr bool TWICE = std::is_same_v<TL, TileTwice>;

// What values' roundings to T leave of them, the second parts.
template <typename T>
__device__ __forceinline__ void rest_of(const float* v, float (&rest)[4]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) rest[q] = second_part(v[q], (T)v[q]);
}

// One tile of the product MODE: that of the block with number `block` of the product's.
template <typename T, int MODE, typename TL, bool DMA>
__device__ __forceinline__ void feed_tile(const Product& P, uint32_t block, const Tiles& G) {
    using Block = typename Sums<T>::Block;
    constexpr bool GATED = MODE == IN || MODE == IN8;
    lds_char* const lds = (lds_char*)s_tiles;
    const uint32_t lds_at = (uint32_t)(uintptr_t)lds;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63;
    const int wm = wave / TL::WN, wn = wave % TL::WN;

    // column tiles together with a group of row tiles, on one die
    const int64_t place = die_order(block, G.count);
    if (place >= G.count) return;
    const uint32_t id = G.first + (uint32_t)place, per = (uint32_t)G.mt * (uint32_t)G.nt;
    const int split = (int)(id / per);
    const uint32_t in = id - split * per, whole_group = TILE_GROUP * (uint32_t)G.nt, group = in / whole_group;
    const int gin = (int)(in - group * whole_group);
    const int gm = min(TILE_GROUP, G.mt - (int)group * TILE_GROUP);
    const int mf = ((int)group * TILE_GROUP + gin % gm) * TL::ROWS;
    const int nf = gin / gm * (GATED ? TL::BN / 2 : TL::BN);

    constexpr int BK = TL::STEP / (int)sizeof(T), KS = TL::STEP / 32;
    const int part = P.splits == 1 ? P.K : ((P.K + P.splits - 1) / P.splits + BK - 1) / BK * BK;
    const int lo = (int)min((int64_t)P.K, (int64_t)split * part), end = (int)min((int64_t)P.K, (int64_t)lo + part);
    const int steps = (int)(((int64_t)end - lo + BK - 1) / BK) * (TWICE<TL> ? 2 : 1);

    Block acc[TL::MI][TL::NI];
#pragma unroll
    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
        for (int j = 0; j < TL::NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

    if constexpr (sizeof(T) == 4) {
        if (steps > 0) parts_sums<MODE, TL>(P, mf, nf, lo, end, steps, acc);
    } else if (steps > 0) {
        Loader<T, MODE, false, TL::BM, TL::NA, TL::NT, TL::STEP, PAIR<TL>> la;
        Loader<T, MODE, true, TL::BN, TL::NB, TL::NT, TL::STEP> lb;
        using LA = decltype(la);
        using LB = decltype(lb);
        la.init(P, mf, lo);
        lb.init(P, nf, lo);
        // Step t of the rows' operand lies at place t % AS, of the columns' at t % BS.  As
        // many steps as there are places are under way; a place is sent its next step as
        // soon as it is free, at the end of the step it held.  With one place more for the rows
        // than for the columns (HALVES), theirs is sent in two halves between the products of
        // step t.  Steps past the last are sent too (zeros), so that every wait is the same.
        // Without DMA there are two places, and a step waits in registers for its own.
        constexpr int AS = DMA ? TL::AS : 2, BS = DMA ? TL::BS : 2;
        constexpr bool HALVES = AS == BS + 1;
        static_assert(AS == BS || (AS == 3 && BS == 2), "places that the order of the steps is made for");
        u32x4 ra[DMA ? 1 : TL::NA], rb[DMA ? 1 : TL::NB];
        // where step t begins; past the end, from where nothing is read
        auto of = [&](int t) { return TWICE<TL> ? t >> 1 : t; };
        auto from = [&](int t) { return (int)min((int64_t)end, lo + (int64_t)of(t) * BK); };
        auto send_a = [&](int t, int place) {
            const int64_t again = TWICE<TL> && (t & 1) ? P.again_a : 0;
            if constexpr (DMA) la.fill(P, of(t), from(t), end, lds_at + (uint32_t)place * TL::ABYTES, again);
            else la.fetch(P, from(t), end, mf, ra, again);
        };
        auto send_b = [&](int t, int place) {
            const int64_t again = TWICE<TL> && (t & 1) ? P.again_b : 0;
            if constexpr (DMA)
                lb.fill(P, of(t), from(t), end, lds_at + TL::AS * TL::ABYTES + (uint32_t)place * TL::BBYTES, again);
            else lb.fetch(P, from(t), end, nf, rb, again);
        };
        auto put = [&](int t) {
            LA::put(lds + (t & 1) * TL::ABYTES, ra);
            LB::put(lds + TL::AS * TL::ABYTES + (t & 1) * TL::BBYTES, rb);
        };
        // accesses of every wave after step 0's and, in the loop, after the next step's
        constexpr int AFTER_0 = DMA ? (BS - 1) * (TL::NA + TL::NB) : 0;
        constexpr int AFTER = HALVES ? TL::NA : DMA ? (BS - 2) * (TL::NA + TL::NB) : 0;
        static_assert(AFTER_0 < 63, "what a wait can count");
        if constexpr (DMA) {
#pragma unroll
            for (int t = 0; t < BS; ++t) {
                send_a(t, t);
                send_b(t, t);
            }
        } else {
            send_a(0, 0);
            send_b(0, 0);
            put(0);
            send_a(1, 0);
            send_b(1, 0);
        }
        const Frag<T, LA::ACROSS, TL::BM, TL::STEP> fa(wm * TL::MI * 32);
        const Frag<T, LB::ACROSS, TL::BN, TL::STEP> fb(wn * TL::NI * 32);
        u32x4 a[2][TL::MI], b[2][TL::NI];
        auto read = [&](int pa, int pb, int ks) {
            lds_char* const ta = lds + pa * TL::ABYTES;
            lds_char* const tb = lds + TL::AS * TL::ABYTES + pb * TL::BBYTES;
#pragma unroll
            for (int i = 0; i < TL::MI; ++i) a[ks & 1][i] = fa.get(ta, i, ks);
#pragma unroll
            for (int j = 0; j < TL::NI; ++j) b[ks & 1][j] = fb.get(tb, j, ks);
        };
        stage_ready<AFTER_0>();
        read(0, 0, 0);
        // A k-step's operands are read while the one before is multiplied, the
        // next step's first ones too: the wait for it stands before the last
        // k-step's products, and what takes the freed places is sent there.
        int pa = 0, pb = 0;
        for (int t = 0; t < steps; ++t) {
            const int na = pa + 1 == AS ? 0 : pa + 1, nb = pb + 1 == BS ? 0 : pb + 1;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (ks + 1 < KS) {
                    if constexpr (HALVES) {
                        const uint32_t to = lds_at + (uint32_t)(na + 1 == AS ? 0 : na + 1) * TL::ABYTES;
                        if (ks == 0) la.template fill<0, TL::NA / 2>(P, t + 2, from(t + 2), end, to);
                        else if (ks == 1) la.template fill<TL::NA / 2, TL::NA>(P, t + 2, from(t + 2), end, to);
                    }
                    read(pa, pb, ks + 1);
                } else {
                    if constexpr (!DMA) put(t + 1);
                    stage_ready<AFTER>();
                    send_b(t + BS, pb);
                    if constexpr (!HALVES) send_a(t + AS, pa);
                    read(na, nb, 0);
                }
#pragma unroll
                for (int i = 0; i < TL::MI; ++i)
#pragma unroll
                    for (int j = 0; j < TL::NI; ++j) {
                        if constexpr (sizeof(T) == 1) acc[i][j] = mma8(a[ks & 1][i], b[ks & 1][j], acc[i][j]);
                        else acc[i][j] = mma<T>(a[ks & 1][i], b[ks & 1][j], acc[i][j]);
                    }
            }
            pa = na;
            pb = nb;
        }
        stage_ready<0>();                            // nothing may reach the LDS of a block that is gone
    }
    constexpr int MI = PAIR<TL> ? 1 : TL::MI;        // blocks of rows of the product
    if constexpr (PAIR<TL>) {
#pragma unroll
        for (int j = 0; j < TL::NI; ++j) acc[0][j] += acc[1][j];
    }

    // The sums go through LDS, 32 rows of a wave at a time, from the matrix
    // cores' layout (a lane has one column) to four neighbouring columns a lane,
    // so that what is read and written beside them goes in whole lines.  Of a tile that
    // lies inside the product nothing is checked.
    constexpr int W = TL::NI * 32;
    lds_float* const mine = (lds_float*)(lds + wave * 32 * W * 4);
    constexpr int LANES = GATED ? W / 8 : W / 4, PASS = 64 / LANES;    // lanes a row, rows at once
    const int c4 = lane % LANES * 4, first = nf + wn * (GATED ? W / 2 : W);   // this lane's columns: first + c4 .. + 3
    const int width = GATED || MODE == DH ? P.Fp : P.N;
    const bool inside = mf + TL::ROWS <= P.M && nf + (GATED ? TL::BN / 2 : TL::BN) <= P.N &&
                        (P.F == P.Fp || !(GATED || MODE == DH || MODE == DWIN));
    f32x4 scale[2];                   // of 8-bit products: the columns'
    if constexpr (MODE == IN8 || MODE == OUT8) {
        if (first + c4 < P.N) {
            scale[0] = four_of(P.sb + first + c4, P.N - (first + c4));
            if constexpr (MODE == IN8) scale[1] = four_of(P.sb + P.F + first + c4, P.F - (first + c4));
        }
    }
    // where the rows of block i begin in an array of this pitch, and this lane's bytes from there
    auto row0 = [&](auto* base, int i, int p, int64_t pitch) {
        return base + (size_t)(mf + (wm * MI + i) * 32 + p) * (size_t)pitch + first;
    };
    auto lane_at = [&](int64_t pitch) { return (uint32_t)(lane / LANES) * (uint32_t)pitch + (uint32_t)c4; };
    const uint32_t at_h = lane_at(P.Fp), at_pre = lane_at(2 * (int64_t)P.Fi), at_dpre = lane_at(2 * (int64_t)P.Fp),
                   at_h32 = lane_at(P.Fi), at_out = lane_at(P.splits > 1 ? P.N : 0);
    auto rows = [&](auto whole_tile, int i) {
        constexpr bool WHOLE = decltype(whole_tile)::value;
        const int f = first + c4;
#pragma unroll 4
        for (int p = 0; p < 32; p += PASS) {
            const int at = p + lane / LANES, m = mf + (wm * MI + i) * 32 + at;
            if (!WHOLE && !(m < P.M && f < width)) continue;
            auto bits = [&](int c) { return *(const lds_f32x4*)(mine + at * W + (c ^ ((at & 4) << 3))); };
            auto whole = [&](int c) {
                const i32x4 v = __builtin_bit_cast(i32x4, bits(c));
                return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
            };
            auto is = [&](int q) { return WHOLE || f + q < P.F; };
            if constexpr (GATED) {
                // columns 64 q + 0..31: gate of f 32 q + 0..31, the next 32: u
                const int c = (c4 & ~31) * 2 + (c4 & 31);
                if (P.splits > 1) {
                    if (WHOLE || f < P.Fi) {
                        float* const to = row0(P.part + (size_t)split * P.M * 2 * (size_t)P.Fi, i, p, 2 * (int64_t)P.Fi);
                        *(f32x4*)(to + at_pre) = bits(c);
                        *(f32x4*)(to + P.Fi + at_pre) = bits(c + 32);
                    }
                    continue;
                }
                f32x4 g, u;
                if constexpr (MODE == IN8) {
                    const float s = P.sa[m];
                    g = whole(c) * scale[0] * s;
                    u = whole(c + 32) * scale[1] * s;
                } else {
                    g = bits(c);
                    u = bits(c + 32);
                }
                float v[4], slope[4], h[4];
                activate<T>(P.act, g, v, slope);
#pragma unroll
                for (int q = 0; q < 4; ++q) h[q] = is(q) ? v[q] * u[q] : 0.0f;
                if constexpr (MODE == IN8) {
                    if (WHOLE || f < P.Fi) *(f32x4*)(row0(P.h32, i, p, P.Fi) + at_h32) = f32x4{h[0], h[1], h[2], h[3]};
                } else {
                    T* const to = row0((T*)P.h, i, p, P.Fp) + at_h;
                    store4(to, h);
                    if constexpr (sizeof(T) == 2 && TL::ROWS <= 64) {
                        if (P.again) {
                            float rest[4];
                            rest_of<T>(h, rest);
                            store4(to + P.again, rest);
                        }
                    }
                    if (P.pre && (WHOLE || f < P.Fi)) {
                        float* const pre = row0(P.pre, i, p, 2 * (int64_t)P.Fi);
                        *(f32x4*)(pre + at_pre) = g;
                        *(f32x4*)(pre + P.Fi + at_pre) = u;
                    }
                }
            } else if constexpr (MODE == DH) {
                if (P.splits > 1) {
                    if (WHOLE || f < P.Fi)
                        *(f32x4*)(row0(P.part + (size_t)split * P.M * (size_t)P.Fi, i, p, P.Fi) + at_h32) = bits(c4);
                    continue;
                }
                f32x4 g = {0.0f, 0.0f, 0.0f, 0.0f}, u = g;
                if (WHOLE || f < P.Fi) {
                    const float* const pre = row0(P.pre, i, p, 2 * (int64_t)P.Fi);
                    g = *(const f32x4*)(pre + at_pre);
                    u = *(const f32x4*)(pre + P.Fi + at_pre);
                }
                const f32x4 dh = bits(c4);
                float v[4], slope[4], dg[4], du[4];
                activate<T>(P.act, g, v, slope);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    dg[q] = is(q) ? dh[q] * u[q] * slope[q] : 0.0f;
                    du[q] = is(q) ? dh[q] * v[q] : 0.0f;
                }
                T* const dpre = row0((T*)P.dpre, i, p, 2 * (int64_t)P.Fp);
                store4(dpre + at_dpre, dg);
                store4(dpre + P.Fp + at_dpre, du);
                if constexpr (sizeof(T) == 2 && TL::ROWS <= 64) {
                    if (P.again) {
                        float rest[4];
                        rest_of<T>(dg, rest);
                        store4(dpre + P.again + at_dpre, rest);
                        rest_of<T>(du, rest);
                        store4(dpre + P.again + P.Fp + at_dpre, rest);
                    }
                }
            } else {
                const int M = MODE == DWIN ? 2 * P.F : P.M;
                if (WHOLE && P.splits > 1) {
                    store_part(row0(P.part + (size_t)split * M * (size_t)P.N, i, p, P.N) + at_out, bits(c4), 4);
                    continue;
                }
                const int row = out_row<MODE>(P, m), have = WHOLE ? 4 : P.N - f;
                if (!WHOLE && row >= M) continue;
                if (P.splits > 1) {
                    store_part(P.part + ((size_t)split * M + row) * (size_t)P.N + f, bits(c4), have);
                } else if constexpr (MODE == OUT8) {
                    store_as(P.out_dtype, P.out, (size_t)row * (size_t)P.ldo + f, whole(c4) * scale[0] * P.sa[row], have);
                } else {
                    store_part((T*)P.out + (size_t)row * (size_t)P.ldo + f, bits(c4), have);
                }
            }
        }
    };
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        wave_sync_lds();
        // sum r of block (i, j): row 8 (r / 4) + 4 (lane / 32) + r % 4, column 32 j + lane % 32;
        // the rows of the upper lanes are kept with their blocks in pairs swapped: other banks
#pragma unroll
        for (int j = 0; j < TL::NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const auto s = acc[i][j][r];
                mine[(8 * (r / 4) + 4 * (lane >> 5) + r % 4) * W + ((j * 32) ^ (lane & 32)) + (lane & 31)] =
                    __builtin_bit_cast(float, s);
            }
        wave_sync_lds();
        if (inside) rows(std::true_type(), i);
        else rows(std::false_type(), i);
    }
}

template <typename T, int MODE, typename TL, bool DMA>
__global__ void __launch_bounds__(TL::NT) k_feed(Product P, Tiles G) {
    feed_tile<T, MODE, TL, DMA>(P, blockIdx.x, G);
}

// Products that need nothing of each other share a grid, so that one's last tiles run beside the
// next one's first: DW_OUT, which needs h and dy alone, with DH, and DX, DW_IN and the rest of DW_OUT.
struct GradProducts {
    Product p[3];
    Tiles g[3];
};
template <typename T, typename TL, bool DMA>
__global__ void __launch_bounds__(TL::NT) k_feed_inner_grad(Product out, Tiles go, Product dh, Tiles gh) {
    if (blockIdx.x < go.blocks) feed_tile<T, DWOUT, TL, DMA>(out, blockIdx.x, go);
    else feed_tile<T, DH, TL, DMA>(dh, blockIdx.x - go.blocks, gh);
}
template <typename T, typename TL, bool DMA, typename TLX = TL>
__global__ void __launch_bounds__(TL::NT) k_feed_grads(GradProducts G) {
    static_assert(TLX::NT == TL::NT, "threads of a block");
    const uint32_t first = G.g[0].blocks, second = first + G.g[1].blocks;
    if (blockIdx.x < first) feed_tile<T, DX, TLX, DMA>(G.p[0], blockIdx.x, G.g[0]);
    else if (blockIdx.x < second) feed_tile<T, DWIN, TL, DMA>(G.p[1], blockIdx.x - first, G.g[1]);
    else feed_tile<T, DWOUT, TL, DMA>(G.p[2], blockIdx.x - second, G.g[2]);
}

// The sums of up to three products that were made in part, added in order.
struct Join {
    const float* part;
    void* out;
    int64_t ldo;
    int M, N, splits, dtype;
    const float* sa;                  // whole numbers in part: their scales
    const float* sb;
};
struct Joins {
    Join j[3];
    int count;
};
__global__ void __launch_bounds__(256) k_join(Joins A) {
    for (int o = 0; o < A.count; ++o) {
        const Join& J = A.j[o];
        const int per = (J.N + 3) / 4;
        const int64_t work = (int64_t)J.M * per;
        const size_t each = (size_t)J.M * (size_t)J.N;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < work; i += (int64_t)gridDim.x * 256) {
            const int row = (int)(i / per), c = (int)(i - (int64_t)row * per) * 4;
            const float* p = J.part + (size_t)row * (size_t)J.N + c;
            f32x4 s;
            if (J.sa) {
                i32x4 whole = {0, 0, 0, 0};
                for (int k = 0; k < J.splits; ++k) whole += __builtin_bit_cast(i32x4, four_of(p + k * each, J.N - c));
                s = f32x4{(float)whole[0], (float)whole[1], (float)whole[2], (float)whole[3]} *
                    four_of(J.sb + c, J.N - c) * J.sa[row];
            } else {
                s = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
                for (int k = 0; k < J.splits; ++k) s += four_of(p + k * each, J.N - c);
            }
            store_as(J.dtype, J.out, (size_t)row * (size_t)J.ldo + c, s, J.N - c);
        }
    }
}

// The same for IN, IN8 and DH, whose sums become h, or dg and du, here.
template <typename T, int MODE>
__global__ void __launch_bounds__(256) k_join_inner(Product P) {
    const int per = P.Fp / 4;
    const int64_t work = (int64_t)P.M * per;
    const size_t pitch = (MODE == DH ? 1 : 2) * (size_t)P.Fi, each = (size_t)P.M * pitch;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < work; i += (int64_t)gridDim.x * 256) {
        const size_t m = (size_t)(i / per);
        const int f = (int)(i - (int64_t)m * per) * 4;
        const bool there = f < P.Fi;
        f32x4 g = {0.0f, 0.0f, 0.0f, 0.0f}, u = g, dh = g;
        if (there) {
            const float* p = P.part + m * pitch + f;
            if constexpr (MODE == IN8) {
                i32x4 sg = {0, 0, 0, 0}, su = sg;
#pragma unroll 4
                for (int k = 0; k < P.splits; ++k, p += each) {
                    sg += *(const i32x4*)p;
                    su += *(const i32x4*)(p + P.Fi);
                }
                const float s = P.sa[m];
                g = f32x4{(float)sg[0], (float)sg[1], (float)sg[2], (float)sg[3]} * four_of(P.sb + f, P.F - f) * s;
                u = f32x4{(float)su[0], (float)su[1], (float)su[2], (float)su[3]} * four_of(P.sb + P.F + f, P.F - f) * s;
            } else if constexpr (MODE == IN) {
#pragma unroll 4
                for (int k = 0; k < P.splits; ++k, p += each) {
                    g += *(const f32x4*)p;
                    u += *(const f32x4*)(p + P.Fi);
                }
            } else {
#pragma unroll 4
                for (int k = 0; k < P.splits; ++k, p += each) dh += *(const f32x4*)p;
                g = *(const f32x4*)(P.pre + m * 2 * P.Fi + f);
                u = *(const f32x4*)(P.pre + m * 2 * P.Fi + P.Fi + f);
            }
        }
        float v[4], slope[4], a[4], b[4];
        activate<T>(P.act, g, v, slope);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const bool is = f + q < P.F;
            a[q] = !is ? 0.0f : MODE == DH ? dh[q] * u[q] * slope[q] : v[q] * u[q];
            b[q] = is && MODE == DH ? dh[q] * v[q] : 0.0f;
        }
        if constexpr (MODE == DH) {
            T* const to = (T*)P.dpre + m * 2 * P.Fp + f;
            store4(to, a);
            store4(to + P.Fp, b);
            if (sizeof(T) == 2 && P.again) {
                float rest[4];
                rest_of<T>(a, rest);
                store4(to + P.again, rest);
                rest_of<T>(b, rest);
                store4(to + P.again + P.Fp, rest);
            }
        } else if constexpr (MODE == IN8) {
            *(f32x4*)(P.h32 + m * P.Fi + f) = f32x4{a[0], a[1], a[2], a[3]};
        } else {
            T* const to = (T*)P.h + m * P.Fp + f;
            store4(to, a);
            if (sizeof(T) == 2 && P.again) {
                float rest[4];
                rest_of<T>(a, rest);
                store4(to + P.again, rest);
            }
            if (P.pre && there) {
                *(f32x4*)(P.pre + m * 2 * P.Fi + f) = g;
                *(f32x4*)(P.pre + m * 2 * P.Fi + P.Fi + f) = u;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Rows in 8 bits: codes of a 127th of the row's largest magnitude.
// ---------------------------------------------------------------------------

constexpr float ROW_LEAST = 0x1p-100f;           // a row whose largest magnitude is below counts as zeros

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// The scale of a row with this largest magnitude (as bits: infinities and NaN are
// larger than numbers) and what its values are multiplied by; a row that is not
// finite has zeros for codes and NaN for its scale.
__device__ __forceinline__ float row_scale(uint32_t bits, float* unit) {
    const float most = __uint_as_float(bits);
    const bool finite = bits < 0x7F800000u, some = finite && most >= ROW_LEAST;
    *unit = some ? 127.0f / most : 0.0f;
    return !finite ? __uint_as_float(0x7FC00000u) : some ? most * (1.0f / 127.0f) : 0.0f;
}
__device__ __forceinline__ int row_code(float v, float unit) {
    // unit 0: v may be infinite or NaN
    return unit == 0.0f ? 0 : (int)fminf(fmaxf(rintf(v * unit), -127.0f), 127.0f);
}
template <typename T>
__device__ __forceinline__ uint32_t chunk_most(const Chunk<T>& c) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < VEC<T>; ++i) {
        const uint32_t b = magnitude(c.get(i));
        most = most > b ? most : b;
    }
    return most;
}
// Codes of a chunk as bytes, to p (of any alignment when `have` of them exist only).
template <typename T>
__device__ __forceinline__ void chunk_codes(const Chunk<T>& c, float unit, int8_t* p, int have) {
    if (have >= VEC<T>) {
        uint32_t w[VEC<T> / 4];
#pragma unroll
        for (int i = 0; i < VEC<T> / 4; ++i) {
            w[i] = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) w[i] |= (uint32_t)(row_code(c.get(4 * i + q), unit) & 0xFF) << (8 * q);
        }
        typedef uint32_t WT __attribute__((ext_vector_type(VEC<T> / 4)));
        typedef WT WTany __attribute__((aligned(1)));
        WT o;
#pragma unroll
        for (int i = 0; i < VEC<T> / 4; ++i) o[i] = w[i];
        *(WTany*)p = o;
    } else {
#pragma unroll
        for (int q = 0; q < VEC<T>; ++q)
            if (q < have) p[q] = (int8_t)row_code(c.get(q), unit);
    }
}

// A row by LANES threads of a block (64: a wave, four rows a block; 256: the block), QUANT_CHUNKS
// pieces of 16 bytes a thread in registers; what does not fit there is read again.  Bound by its
// bytes: 16 384 x 5632 of fp32 86 us, 5.4 TB/s; 8192 x 4096 of bf16 19.3 us, 5.2 TB/s.
constexpr int QUANT_CHUNKS = 4;
template <typename T, int LANES>
__global__ void __launch_bounds__(256) k_quantize(const T* x, int64_t ldx, int64_t n, int D, int8_t* q, int64_t ldq,
                                                  float* scale) {
    __shared__ uint32_t s_most[4];
    const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const int t = threadIdx.x % LANES;
    if (LANES == 64 && row >= n) return;          // a wave by itself: no barrier below
    const T* const r = x + (size_t)row * (size_t)ldx;
    const int chunks = (D + VEC<T> - 1) / VEC<T>;
    Chunk<T> c[QUANT_CHUNKS];
    uint32_t most = 0;
    if (D % VEC<T> == 0) {
        // past the end the last piece again, which leaves the largest as it is: loads without a branch between them
#pragma unroll
        for (int i = 0; i < QUANT_CHUNKS; ++i) c[i].load(r + min(i * LANES + t, chunks - 1) * VEC<T>);
    } else {
#pragma unroll
        for (int i = 0; i < QUANT_CHUNKS; ++i) c[i].raw = row_piece<T>(r, min(i * LANES + t, chunks - 1) * VEC<T>, D);
    }
#pragma unroll
    for (int i = 0; i < QUANT_CHUNKS; ++i) most = max(most, chunk_most(c[i]));
    for (int at = QUANT_CHUNKS * LANES + t; at < chunks; at += LANES) {
        Chunk<T> d;
        d.raw = row_piece<T>(r, at * VEC<T>, D);
        most = max(most, chunk_most(d));
    }
    most = lanes_reduce<64>(most, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
    if constexpr (LANES == 256) {
        if ((threadIdx.x & 63) == 0) s_most[threadIdx.x / 64] = most;
        __syncthreads();
        most = max(max(s_most[0], s_most[1]), max(s_most[2], s_most[3]));
    }
    float unit;
    const float s = row_scale(most, &unit);
    int8_t* const o = q + (size_t)row * (size_t)ldq;
#pragma unroll
    for (int i = 0; i < QUANT_CHUNKS; ++i) {
        const int at = i * LANES + t;
        if (at < chunks) chunk_codes(c[i], unit, o + at * VEC<T>, D - at * VEC<T>);
    }
    for (int at = QUANT_CHUNKS * LANES + t; at < chunks; at += LANES) {
        Chunk<T> d;
        d.raw = row_piece<T>(r, at * VEC<T>, D);
        chunk_codes(d, unit, o + at * VEC<T>, D - at * VEC<T>);
    }
    if (t == 0) scale[row] = s;
}

// ---------------------------------------------------------------------------
// Few rows: the products are bound by the weights' bytes, each read once, and by
// the launches.  Weights go straight from memory into the matrix instructions'
// operands: a lane fetches 32 bytes in a row of one weight row, two instructions' worth, 16
// weight rows and 16 rows of x a wave.  A block has 16 columns (IN: of h) and its
// waves share the summed dimension, 128 bytes a row in turn; their sums meet in LDS.
// One row, bf16, 1024 -> 4096 -> 1024: 5.7 and 6.9 us for 17 and 8 MB, mostly launch and one round
// trip of loads; 2048 -> 5632 -> 2048: 22 us together for 69 MB.  From 16 rows on x, which every
// block reads again, costs as much as the weights.
// ---------------------------------------------------------------------------

constexpr int FEW_ROWS = 64;                     // rows of a call, up to four groups of 16
constexpr int FEW_NT = 512;
// pieces of 128 bytes a row that a wave holds, of weights and of x: with 32, the blocks of one group of rows
// would be one a CU instead of two (1024 -> 4096 -> 1024, one row: 13.7 and 12.7 us)
constexpr int few_held(int MB) { return MB > 1 ? 32 : 16; }
constexpr int FEW_VALUES = 16384;                // values of x that every block puts in 8 bits by itself

// 16 bytes of a row from value k on: all there (WHOLE), or its K values alone, zeros after them.
template <typename T, bool WHOLE>
__device__ __forceinline__ u32x4 few_piece(const T* row, int k, int K) {
    if constexpr (WHOLE) return *reinterpret_cast<const u32x4_any*>(row + k);
    else return row_piece<T>(row, k, K);
}

// Where the rows of x come from: a lane's piece of 16 bytes' worth of T from value k on, fetched
// as RAW pieces and taken apart into PARTS operands.
template <typename T>
struct FewRows {                                 // rows of T in memory
    static constexpr int RAW = 1, PARTS = 1;
    const T* base;
    size_t ld;
    int n;
    template <bool WHOLE>
    __device__ __forceinline__ void load(int mb, int k, int K, u32x4 (&raw)[RAW]) const {
        raw[0] = few_piece<T, WHOLE>(base + (size_t)min(mb * 16 + (int)(threadIdx.x & 15), n - 1) * ld, k, K);
    }
    __device__ __forceinline__ static void parts(const u32x4 (&raw)[RAW], u32x4 (&v)[PARTS]) { v[0] = raw[0]; }
};
template <typename T>
struct FewHalves {                               // fp32 rows in two parts of T: 16 bits and more of each value
    static constexpr int RAW = 2, PARTS = 2;
    const float* base;
    size_t ld;
    int n;
    template <bool WHOLE>
    __device__ __forceinline__ void load(int mb, int k, int K, u32x4 (&raw)[RAW]) const {
        const float* row = base + (size_t)min(mb * 16 + (int)(threadIdx.x & 15), n - 1) * ld;
        raw[0] = few_piece<float, WHOLE>(row, k, K);
        raw[1] = few_piece<float, WHOLE>(row, k + 4, K);
    }
    __device__ __forceinline__ static void parts(const u32x4 (&raw)[RAW], u32x4 (&v)[PARTS]) {
        typedef T VT __attribute__((ext_vector_type(8)));
        VT hi, lo;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const float f = __builtin_bit_cast(f32x4, raw[q / 4])[q % 4];
            hi[q] = (T)f;
            lo[q] = (T)second_part(f, hi[q]);
        }
        v[0] = __builtin_bit_cast(u32x4, hi);
        v[1] = __builtin_bit_cast(u32x4, lo);
    }
};
struct FewCodes {                                // codes that the block put in LDS, `ld` bytes a row, zeros to whole pieces
    static constexpr int RAW = 1, PARTS = 1;
    const lds_char* base;
    int ld, n;
    template <bool WHOLE>
    __device__ __forceinline__ void load(int mb, int k, int K, u32x4 (&raw)[RAW]) const {
        raw[0] = u32x4{0, 0, 0, 0};
        if (WHOLE || k < K) raw[0] = *(const lds_u32x4*)(base + min(mb * 16 + (int)(threadIdx.x & 15), n - 1) * ld + k);
    }
    __device__ __forceinline__ static void parts(const u32x4 (&raw)[RAW], u32x4 (&v)[PARTS]) { v[0] = raw[0]; }
};

// acc[m][b] += M matrices' 16 rows w[m] times group b of 16 rows of x, over AHEAD pieces of 128
// bytes, `by` pieces apart, the first from value k0 on.  WHOLE: they lie in the rows, and nothing
// stands between their loads; else a branch for each, which costs more than the loads.
template <typename T, int M, int MB, int AHEAD, bool WHOLE, typename Src>
__device__ __forceinline__ void few_pieces(const T* const (&w)[M], const Src& x, int K, int k0, int by,
                                           typename Sums<T>::Four (&acc)[M][MB]) {
    constexpr int CH = VEC<T>, STEP = 8 * CH;    // values in 128 bytes
    const int q = (threadIdx.x & 63) >> 4;
    u32x4 a[AHEAD][M][2], v[AHEAD][2][MB][Src::RAW];
#pragma unroll
    for (int s = 0; s < AHEAD; ++s)
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            const int k = k0 + s * by * STEP + (2 * q + o) * CH;
#pragma unroll
            for (int m = 0; m < M; ++m) a[s][m][o] = few_piece<T, WHOLE>(w[m], k, K);
#pragma unroll
            for (int b = 0; b < MB; ++b) x.template load<WHOLE>(b, k, K, v[s][o][b]);
        }
#pragma unroll
    for (int s = 0; s < AHEAD; ++s)
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                u32x4 p[Src::PARTS];
                Src::parts(v[s][o][b], p);
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int i = 0; i < Src::PARTS; ++i) {
                        if constexpr (sizeof(T) == 1) acc[m][b] = mma8(a[s][m][o], p[i], acc[m][b]);
                        else acc[m][b] = mma16<T>(a[s][m][o], p[i], acc[m][b]);
                    }
            }
}

// The same over all of a row's pieces from number `from` on, every `by`-th: eight (or what registers
// hold) under way at once, then four, two, one, and what is left of a piece.
template <typename T, int M, int MB, typename Src>
__device__ __forceinline__ void few_sums(const T* const (&w)[M], const Src& x, int K, int from, int by,
                                         typename Sums<T>::Four (&acc)[M][MB]) {
    constexpr int STEP = 8 * VEC<T>;
    int k0 = from * STEP;
    const int each = by * STEP;
    auto run = [&](auto ahead) {
        constexpr int A = decltype(ahead)::value;
        for (; k0 + (A - 1) * each + STEP <= K; k0 += A * each) few_pieces<T, M, MB, A, true>(w, x, K, k0, by, acc);
    };
    if constexpr (M + MB * Src::RAW <= few_held(MB) / 8) run(std::integral_constant<int, 8>());
    if constexpr (M + MB * Src::RAW <= few_held(MB) / 4) run(std::integral_constant<int, 4>());
    run(std::integral_constant<int, 2>());
    run(std::integral_constant<int, 1>());
    if (k0 < K) few_pieces<T, M, MB, 1, false>(w, x, K, k0, by, acc);
}

// The block's rows of x (type X) as codes in LDS, rows ld bytes apart, and their scales.
template <typename X>
__device__ __forceinline__ void few_codes(const Product& P, lds_char* codes, int ld, uint32_t* most, float* scale) {
    constexpr int CH = VEC<X>, EACH = FEW_VALUES / CH / FEW_NT;
    const int per = (P.K + 15) / 16 * (16 / CH), all = P.M * per;      // the last code piece is filled up with zeros
    Chunk<X> c[EACH + 1];                         // rows of whole 16 codes may hold a little more than FEW_VALUES
    if ((int)threadIdx.x < P.M) most[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i <= EACH; ++i) {
        const int at = i * FEW_NT + (int)threadIdx.x;
        c[i].raw = u32x4{0, 0, 0, 0};
        if (at < all) c[i].raw = row_piece<X>((const X*)P.a + (size_t)(at / per) * (size_t)P.lda, at % per * CH, P.K);
    }
#pragma unroll
    for (int i = 0; i <= EACH; ++i) {
        const int at = i * FEW_NT + (int)threadIdx.x;
        if (at < all) atomicMax(&most[at / per], chunk_most(c[i]));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i <= EACH; ++i) {
        const int at = i * FEW_NT + (int)threadIdx.x;
        if (at < all) {
            float unit;
            row_scale(most[at / per], &unit);
            chunk_codes(c[i], unit, (int8_t*)(codes + at / per * ld + at % per * CH), CH);
        }
    }
    if ((int)threadIdx.x < P.M) {
        float unit;
        scale[threadIdx.x] = row_scale(most[threadIdx.x], &unit);
    }
    __syncthreads();
}

// MODE IN or OUT with T f32, bf16, f16; IN8 or OUT8 with int8_t, FLOATS: a's values become codes here.
// OUT's rows are h, in fp32 for up to 16 of them and with FLOATS, taken in two parts of a 16-bit T, else in T.  A block
// makes R groups of 16 columns for MB groups of 16 rows.
template <typename T, int MODE, int MB, int R, bool FLOATS>
__global__ void __launch_bounds__(FEW_NT) k_few(Product P) {
    constexpr bool GATED = MODE == IN || MODE == IN8;
    constexpr int G = GATED ? 2 : 1, WAVES = FEW_NT / 64;
    using Four = typename Sums<T>::Four;
    // groups of columns and rows, and how many of their sums LDS holds: 32 KB
    constexpr int PAIRS = R * MB, AT_ONCE = PAIRS < 4 / G ? PAIRS : 4 / G;
    __shared__ Four s_sum[WAVES][AT_ONCE][G][64];
    __shared__ float s_scale[FEW_ROWS];
    __shared__ uint32_t s_most[FEW_ROWS];
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int first = blockIdx.x * (16 * R);
    const T* w[R * G];
#pragma unroll
    for (int g = 0; g < R; ++g) {
        w[g * G] = (const T*)P.b + (size_t)min(first + g * 16 + r, P.N - 1) * (size_t)P.ldb;
        if constexpr (GATED) w[g * G + 1] = w[g * G] + (size_t)P.F * (size_t)P.ldb;
    }
    Four acc[R * G][MB];
#pragma unroll
    for (int m = 0; m < R * G; ++m)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[m][b] = Four{0, 0, 0, 0};
    if constexpr (FLOATS && sizeof(T) == 1) {
        lds_char* const codes = (lds_char*)s_tiles;
        const int ld = (P.K + 15) / 16 * 16 + 16;        // rows begin at other banks
        if (P.x_dtype == DT_F32) few_codes<float>(P, codes, ld, s_most, s_scale);
        else if (P.x_dtype == DT_BF16) few_codes<bf16>(P, codes, ld, s_most, s_scale);
        else few_codes<f16>(P, codes, ld, s_most, s_scale);
        few_sums<T, R * G, MB>(w, FewCodes{codes, ld, P.M}, P.K, wave, WAVES, acc);
    } else if constexpr (MODE == OUT && sizeof(T) == 2 && (MB == 1 || FLOATS)) {
        few_sums<T, R * G, MB>(w, FewHalves<T>{(const float*)P.a, (size_t)P.lda, P.M}, P.K, wave, WAVES, acc);
    } else {
        few_sums<T, R * G, MB>(w, FewRows<T>{(const T*)P.a, (size_t)P.lda, P.M}, P.K, wave, WAVES, acc);
    }
#pragma unroll
    for (int p0 = 0; p0 < PAIRS; p0 += AT_ONCE) {
        if (p0) __syncthreads();                         // the sums before have been read
#pragma unroll
        for (int p = 0; p < AT_ONCE; ++p)
#pragma unroll
            for (int m = 0; m < G; ++m)
                if (p0 + p < PAIRS) s_sum[wave][p][m][lane] = acc[(p0 + p) / MB * G + m][(p0 + p) % MB];
        __syncthreads();
        // a wave finishes a pair of groups: a lane has row r and columns c .. c + 3
        const int pair = p0 + wave, row = pair % MB * 16 + r, c = first + pair / MB * 16 + 4 * q;
        if (wave < AT_ONCE && pair < PAIRS && row < P.M && c < P.N) {
            Four t[G];
#pragma unroll
            for (int m = 0; m < G; ++m) {
                t[m] = s_sum[0][wave][m][lane];
#pragma unroll
                for (int o = 1; o < WAVES; ++o) t[m] += s_sum[o][wave][m][lane];
            }
            f32x4 v[G];
            if constexpr (sizeof(T) == 1) {
                const float s = FLOATS ? s_scale[row] : P.sa[row];
#pragma unroll
                for (int m = 0; m < G; ++m)
                    v[m] = f32x4{(float)t[m][0], (float)t[m][1], (float)t[m][2], (float)t[m][3]} *
                           four_of(P.sb + m * P.F + c, P.N - c) * s;
            } else {
#pragma unroll
                for (int m = 0; m < G; ++m) v[m] = t[m];
            }
            if constexpr (GATED) {
                float a[4], slope[4], h[4];
                activate<T>(P.act, v[0], a, slope);
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = c + i < P.F ? a[i] * v[G - 1][i] : 0.0f;
                if (P.h32) *(f32x4*)(P.h32 + (size_t)row * (size_t)P.Fi + c) = f32x4{h[0], h[1], h[2], h[3]};
                if constexpr (sizeof(T) != 1) {
                    if (P.h) {
                        T* const to = (T*)P.h + (size_t)row * (size_t)P.Fp + c;
                        store_part(to, f32x4{h[0], h[1], h[2], h[3]}, P.Fp - c);
                        if (sizeof(T) == 2 && P.again) {
                            float rest[4];
                            rest_of<T>(h, rest);
                            store_part(to + P.again, f32x4{rest[0], rest[1], rest[2], rest[3]}, P.Fp - c);
                        }
                    }
                    if (P.pre) {
                        float* pre = P.pre + (size_t)row * 2 * (size_t)P.Fi + c;
                        *(f32x4*)pre = v[0];
                        *(f32x4*)(pre + P.Fi) = v[G - 1];
                    }
                }
            } else {
                store_as(P.out_dtype, P.out, (size_t)row * (size_t)P.ldo + c, v[0], P.N - c);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// 16384 x 2048 -> 5632 -> 2048 in 8 bits, us: 256 x 256 700, 128 x 256 (one block a CU, eight waves) 852, 128 x 128 (two
// blocks) 826; 8192 x 4096 x 4096 158, 197 and 191.
using TileSmall = TileOf<64, 128, 2, 2, 128, 2, 2>;
using TileDeep = TileOf<64, 128, 2, 2, 128, 3, 3>;
using TileLarge = TileOf<256, 256, 4, 2, 128, 3, 2>;
using PartsSmall = TileParts<64, 128, 2, 2>;     // fp32
using PartsLarge = TileParts<128, 256, 2, 4>;
// Tiles of a product of M x N sums.
inline int64_t tile_count(int bytes, bool large, int64_t M, int64_t N) {
    return over(M, large ? (bytes == 4 ? 128 : 256) : 64) * over(N, large ? 256 : 128);
}

constexpr int CUS = 256;
constexpr int PART_BLOCKS = 512;      // blocks that keep the device busy
constexpr int MOST_SPLITS = 64;
constexpr int INT8_MOST = 131071;     // terms of 128 x 128 whose sum stays in 32 bits

// Whether a tile's rows of an operand, `rows` of them ld apart, lie within 32 bits of where it begins.
inline bool near_ok(int64_t rows, int64_t ld, int bytes) { return rows <= (1ll << 31) / (ld * bytes); }
// Whether an operand's rows, of `width` values and ld apart, may go straight to LDS.
inline bool straight_ok(const void* p, int64_t ld, int width, int bytes, int64_t rows = 256) {
    return pieces_ok(p, ld, width, bytes) && near_ok(rows, ld, bytes);
}

// Whether large tiles make a product of M x K by K x N (its sums' columns) faster than small ones: they
// fetch less, or take less apart (fp32), but there have to be enough of them, and a block of theirs has
// its CU to itself, so that nothing covers its beginning and end unless K is long.  fp32, small and
// large, us: 4096 x 2048 -> 4096 -> 2048 1240 and 1020, 3000 x 700, 2000, forward and backward 634 and 590; 128 x
// 128 tiles lie between them where products are large and behind both where they are small.  16 and 8 bits, small and
// large by the number of large ones, us: bf16 n x 2048 -> 2048 -> 4096 64 tiles 55 and 87, 96 77 and 88, 128 105 and 89,
// 256 180 and 123; 8-bit products n x 2048 x 4096 96 tiles 23.8 and 31.6, 128 33.5 and 32.0, 256 55 and 41.
inline bool large_product(int bytes, int64_t M, int64_t N, int64_t K) {
    return K * bytes >= 768 && M >= 192 && N >= 192 && tile_count(bytes, true, M, N) >= (bytes == 4 ? 200 : 128);
}

// Parts of the summed dimension, so that few tiles fill the device: at least four steps each.
inline int split_count(int64_t M, int64_t N, int64_t K, bool large, int bytes) {
    if (large) return 1;
    const int64_t tiles = tile_count(bytes, false, M, N);
    int64_t s = PART_BLOCKS / (tiles < 1 ? 1 : tiles);
    const int64_t longest = K * bytes / (4 * 128);
    if (s > longest) s = longest;
    if (s > MOST_SPLITS) s = MOST_SPLITS;
    return s < 1 ? 1 : (int)s;
}

// The same of the products that become h (IN), or dg and du (DH), whose join is a launch more that reads the
// parts: where the steps that a block is spared take longer.  A step takes about 0.38 us, DH's 0.6 (0.9 where
// W_out's rows are not whole pieces), fp32's 1.1, the launch 5 and 100 parts of tiles 1.2.  Whole and in
// parts, us for the block: fp32 83 x 2520 -> 256 -> 2520 106 and 28, 1000 x 2048 -> 512 100 and 61; bf16 83 x 2520 24.5 and 15.5, but 534 x 1000 -> 760 23.5
// and 27.2 (it stays whole); 8 bits 100 x 4096 -> 1024 33.1 and 28.9, but 1000 x 2048 -> 512 27.0 and 32.9.
inline int inner_split_count(int mode, int64_t M, int64_t N, int64_t K, bool large, int bytes) {
    const int s = split_count(M, N, K, large, bytes);
    const double each = bytes == 4 ? 1.1 : mode != DH ? 0.38 : N * bytes % 16 ? 0.9 : 0.6;
    const double steps = (double)over(K * bytes, 128);
    const double spared = steps * (1.0 - 1.0 / s) * each, more = 5.0 + 0.012 * s * (double)tile_count(bytes, false, M, N);
    return spared > more ? s : 1;
}

// All tiles of a product; false: more than a grid can have.
template <typename TL>
bool all_tiles(const Product& P, bool gated, Tiles* g) {
    g->nt = (int)over(P.N, gated ? TL::BN / 2 : TL::BN);
    g->mt = (int)over(P.M, TL::ROWS);
    const double count = (double)g->nt * g->mt * P.splits;
    if (count * TL::NT > 4e9) return false;      // with the other products of a grid below 2^32 threads, checked there
    g->first = 0;
    g->count = (uint32_t)g->nt * (uint32_t)g->mt * (uint32_t)P.splits;
    g->blocks = (uint32_t)(over(g->count, XCDS) * XCDS);
    return true;
}
// The last `count` tiles in a grid of their own.
inline Tiles take_last(Tiles* g, uint32_t count) {
    Tiles last = *g;
    g->count -= count;
    g->blocks = (uint32_t)(over(g->count, XCDS) * XCDS);
    last.first += g->count;
    last.count = count;
    last.blocks = (uint32_t)(over(count, XCDS) * XCDS);
    return last;
}
inline bool grid_ok(int64_t blocks, int threads) { return blocks <= UINT32_MAX / threads; }

// fp32: in parts, whatever its rows' alignment.
template <typename T, typename F>
auto by_tile(bool large, bool dma, const F& f) {
    if constexpr (sizeof(T) == 4) {
        return large ? f(PartsLarge(), std::false_type()) : f(PartsSmall(), std::false_type());
    } else {
        if (large) return dma ? f(TileLarge(), std::true_type()) : f(TileLarge(), std::false_type());
        return dma ? f(TileSmall(), std::true_type()) : f(TileSmall(), std::false_type());
    }
}

// Makes the tiles of one product; false: the grid would be too large.
template <typename T, int MODE>
bool run_tiles(const Product& P, bool large, bool dma, hipStream_t stream) {
    auto launch = [&](auto tl, auto d) {
        using TL = decltype(tl);
        Tiles g;
        if (!all_tiles<TL>(P, MODE == IN || MODE == IN8, &g) || !grid_ok(g.blocks, TL::NT)) return false;
        // no more blocks than two a CU: three steps under way in each instead of two, which leaves room for
        // two.  Two and three, us: 128 x 2048 -> 5632 -> 2048, bf16, 37.2 and 32.4; 534 x 1000 -> 760 26.9 and
        // 23.5; steps too few to fill the places, 48 rows' y, 31.3 and 32.3.
        if constexpr (std::is_same_v<TL, TileSmall> && decltype(d)::value) {
            if (g.blocks <= 2 * CUS && (int64_t)P.K * (int)sizeof(T) / P.splits >= 8 * 128) {
                k_feed<T, MODE, TileDeep, true><<<g.blocks, TileDeep::NT, TileDeep::LDS, stream>>>(P, g);
                return true;
            }
        }
        k_feed<T, MODE, TL, decltype(d)::value><<<g.blocks, TL::NT, TL::LDS, stream>>>(P, g);
        return true;
    };
    if constexpr (MODE == OUT && sizeof(T) == 2) {
        if (P.again_a) return dma ? launch(TilePair(), std::true_type()) : launch(TilePair(), std::false_type());
    }
    return by_tile<T>(large, dma, launch);
}

inline void run_join(const Joins& J, hipStream_t stream) {
    int64_t work = 0;
    for (int i = 0; i < J.count; ++i) {
        const int64_t w = (int64_t)J.j[i].M * over(J.j[i].N, 4);
        work = w > work ? w : work;
    }
    if (J.count) k_join<<<launch_grid(work, 256, 8192), 256, 0, stream>>>(J);
}

template <typename T, int MODE>
void run_join_inner(const Product& P, hipStream_t stream) {
    const int64_t work = (int64_t)P.M * (P.Fp / 4);
    if (P.splits > 1 && work > 0) k_join_inner<T, MODE><<<launch_grid(work, 256, 8192), 256, 0, stream>>>(P);
}

template <typename T, int MODE, int MB, int R, bool FLOATS>
void launch_few(const Product& P, hipStream_t stream) {
    const size_t lds = FLOATS && sizeof(T) == 1 ? (size_t)P.M * (size_t)((P.K + 15) / 16 * 16 + 16) : 0;
    k_few<T, MODE, MB, R, FLOATS><<<(unsigned)over(P.N, 16 * R), FEW_NT, lds, stream>>>(P);
}
template <typename T, int MODE, bool FLOATS>
void run_few(const Product& P, hipStream_t stream) {
    // more columns a block read x less often, but leave fewer blocks.  One group and two, us for the block: 2048 ->
    // 5632 -> 2048, bf16, 24 rows 31.8 and 28.9, 64 rows 54.7 and 45.7; fp32 500 -> 700 -> 500, 20 rows 11.7 and
    // 16.3; of y's 2048 columns 31.8 and 36.0 (24 rows)
    auto by_rows = [&](auto r) {
        constexpr int R = decltype(r)::value;
        if (P.M <= 32) launch_few<T, MODE, 2, R, FLOATS>(P, stream);
        else if (P.M <= 48) launch_few<T, MODE, 3, R, FLOATS>(P, stream);
        else launch_few<T, MODE, 4, R, FLOATS>(P, stream);
    };
    if (P.M <= 16) return launch_few<T, MODE, 1, 1, FLOATS && sizeof(T) == 1>(P, stream);
    if constexpr (MODE == IN || MODE == IN8) {
        if (over(P.N, 32) >= 128) return by_rows(std::integral_constant<int, 2>());
    }
    by_rows(std::integral_constant<int, 1>());
}

template <typename F>
auto by_dtype(int dtype, const F& f) {
    if (dtype == DT_F32) return f((float*)nullptr);
    if (dtype == DT_BF16) return f((bf16*)nullptr);
    return f((f16*)nullptr);
}

inline bool few_rows(int64_t n) { return n <= FEW_ROWS; }
inline bool few_values(int64_t n, int64_t K) { return n * K <= FEW_VALUES; }

inline bool feed_ranges_ok(int64_t n, int D, int F, int O) {
    return n >= 0 && n < (1ll << 31) - 256 && D >= 1 && F >= 1 && O >= 1 && D <= (1 << 24) && F <= (1 << 24) &&
           O <= (1 << 24);
}

// The three gradients by large tiles, side by side, those of more steps than a CU's share of
// all in parts (of 16 steps at least).  Large and small, us for forward and backward, bf16: 8192 x 1024, 2816: 620 and
// 703; 4096 x 2048, 2048: 360 and 446; 2048 x 2048, 5632: 590 and 624.
inline bool large_gradients(int bytes, const int64_t (&M)[3], const int64_t (&N)[3], const int64_t (&K)[3],
                            int (&splits)[3]) {
    int64_t tiles[3], steps[3], all = 0, count = 0;
    for (int i = 0; i < 3; ++i) {
        if (K[i] * bytes < 768 || M[i] < 192 || N[i] < 192) return false;
        tiles[i] = tile_count(bytes, true, M[i], N[i]), steps[i] = over(K[i] * bytes, 128);
        all += tiles[i] * steps[i];
    }
    const int64_t share = all / CUS < 16 ? 16 : all / CUS;
    for (int i = 0; i < 3; ++i) {
        const int64_t s = over(steps[i], share);
        splits[i] = (int)(s < MOST_SPLITS ? s : MOST_SPLITS);
        count += tiles[i] * splits[i];
    }
    return count >= 200;
}

// y: every block of its kernel for few rows reads all of h again, 16 columns a block (16 rows or
// fewer: in fp32); tiles split over F read less but need a second launch to join them.  Few and tiles, us for
// the block: 2048 -> 5632 -> 2048, bf16, 17 rows 26.9 and 26.3, 24 28.7 and 26.8, 48 38.6 and 31.3, 64 45.7 and
// 35.4; 1024 -> 4096 -> 1024, 20 rows 19.9 and 19.0; fp32 500 -> 700 -> 500, 20 rows 16.4 and
// 23.4, 48 20.9 and 26.2.  (8 bits: 5632 -> 2048, 24 rows 27.4 and 30.1, 64 37.9 and 37.2; 4096 -> 4096, 64
// rows 15.4 and 18.2: few throughout.)
inline bool few_answer(int64_t n, int64_t F, int64_t O, int bytes) { return over(O, 16) * n * F * bytes <= (8 << 20); }

// A small block: one large value of h, or of an output, may decide the error of all, and h, dg and du are taken in
// two parts of a 16-bit type.  The error's square is that of one rounding times 1 + a weighted mean over h's values
// (their fourth moment is some 24 squares of the second) over one over the outputs' (6): a variance of 24 / (n F) +
// 6 / (n min(D, O)), up to 1 / 128 left as it is.  Of 44 500 random blocks more than 1.5 times one rounding's error
// had 19% of those below (up to 2.2 times) and 0.5% of the others.
inline bool twice_ok(int64_t n, int D, int F, int O, int bytes) {
    const double w = D < O ? D : O;
    return bytes == 2 && 128.0 * (24.0 / F + 6.0 / w) > (double)n && n * F < (1 << 28);      // parts: 32 bits apart
}

struct FeedSizes {
    int64_t n;
    int D, F, O, bytes, Fp, Fi;
    bool few, few_out, whole;         // few rows: h and y by their kernel; h is kept in fp32 for y
    bool twice;                       // h, dg and du in two parts
    bool large_in, large_out, large_dh, large_grads;
    int splits_in, splits_out;        // of [g u], of y
    int splits_dh, splits[3];         // of dh; of dx, dW_in, dW_out
};
inline FeedSizes feed_sizes(int dtype, int64_t n, int D, int F, int O) {
    FeedSizes z;
    const int b = dtype_bytes(dtype);
    z.n = n, z.D = D, z.F = F, z.O = O, z.bytes = b;
    z.Fp = up16(F, b);
    z.Fi = up16(F, 4);
    z.few = few_rows(n);
    z.large_in = large_product(b, n, 2 * (int64_t)F, D);
    z.large_out = large_product(b, n, O, F);
    z.splits_out = split_count(n, O, F, z.large_out, b);
    z.splits_in = z.few ? 1 : inner_split_count(IN, n, 2 * (int64_t)F, D, z.large_in, b);
    z.large_dh = large_product(b, n, F, O);
    z.splits_dh = inner_split_count(DH, n, F, O, z.large_dh, b);
    const int64_t M[3] = {n, (int64_t)z.Fp + F, O}, N[3] = {D, D, F}, K[3] = {(int64_t)z.Fp + F, n, n};
    z.large_grads = large_gradients(b, M, N, K, z.splits);
    z.twice = twice_ok(n, D, F, O, b) && !(z.large_in || z.large_out || z.large_dh || z.large_grads);
    z.whole = (n <= 16 || (z.few && z.twice && n * F < 16384)) && few_answer(n, F, O, 2);
    z.few_out = z.whole || (n > 16 && z.few && !z.twice && few_answer(n, F, O, b));
    if (!z.large_grads)                   // of the products whose steps are made twice, as many as of twice the length
        for (int i = 0; i < 3; ++i) z.splits[i] = split_count(M[i], N[i], K[i] * (z.twice && i ? 2 : 1), false, b);
    return z;
}

// How many tiles of dW_out are made beside dh: with large tiles, of which a CU takes one at a time, so many that
// the others' grid is whole rounds of tiles, where that round costs more than what it adds to dh's.
// 8192 x 2048, 5632 (784 tiles, dh's 704): 16 of them.
inline uint32_t beside_inner_grad(const FeedSizes& z, uint32_t dh, const Tiles (&g)[3]) {
    const uint32_t rest = (g[0].count + g[1].count + g[2].count) % CUS;
    if (!z.large_grads || rest == 0 || rest > g[2].count) return 0;
    // in steps; the end of dh's tiles, which read g and u and write dg and du, takes as long as 22
    const double each = (double)z.n * z.bytes / 128 / z.splits[2], each_dh = (double)z.O * z.bytes / 128 + 22;
    const double rounds = (double)over(dh, CUS), idle = rounds * CUS - dh;
    const double more = (rest * each - idle * each_dh) / CUS, longer = each - rounds * each_dh;
    return (more > 0 ? more : 0) + (longer > 0 ? longer : 0) < 0.9 * each ? rest : 0;
}

// A launch has fewer than 2^32 threads: whether those of the block's products have.
inline bool tiles_fit(bool large, double tiles) { return tiles * (large ? 512 : 256) < 4e9; }
inline double tiles_of(int bytes, bool large, double M, double N) {
    return (double)tile_count(bytes, large, (int64_t)M, (int64_t)N);
}
inline bool feed_grids_ok(const FeedSizes& z) {
    const int b = z.bytes;
    const double dh = tiles_of(b, z.large_dh, z.n, z.F), x = tiles_of(b, z.large_grads, z.n, z.D) * z.splits[0],
                 i = tiles_of(b, z.large_grads, (double)z.Fp + z.F, z.D) * z.splits[1],
                 o = tiles_of(b, z.large_grads, z.O, z.F) * z.splits[2];
    return tiles_fit(z.large_in, tiles_of(b, z.large_in, z.n, 2.0 * z.F)) &&
           tiles_fit(z.large_out, tiles_of(b, z.large_out, z.n, z.O) * z.splits_out) && tiles_fit(z.large_dh, dh + o) &&
           tiles_fit(z.large_grads, x + i + o);
}
inline bool feed_sizes_ok(int dtype, int64_t n, int D, int F, int O, FeedSizes* z) {
    if (!dtype_ok(dtype) || !feed_ranges_ok(n, D, F, O)) return false;
    *z = feed_sizes(dtype, n, D, F, O);
    return feed_grids_ok(*z);
}

struct FeedKept {                     // what the forward pass keeps
    float* pre;
    char* h;
};
inline size_t carve_kept(Carve& c, FeedKept* k, const FeedSizes& z) {
    k->pre = c.take<float>((size_t)z.n * 2 * z.Fi);
    k->h = c.take<char>((size_t)z.n * z.Fp * z.bytes * (z.twice ? 2 : 1));
    return c.off;
}
struct FeedSpace {
    char* h;
    float* h32;
    float* part_in;
    float* part;
};
inline size_t carve_forward(Carve& c, FeedSpace* s, const FeedSizes& z) {
    s->h = c.take<char>((size_t)z.n * z.Fp * z.bytes * (z.twice ? 2 : 1));
    s->h32 = z.whole ? c.take<float>((size_t)z.n * z.Fi) : nullptr;
    s->part_in = z.splits_in > 1 ? c.take<float>((size_t)z.splits_in * z.n * 2 * z.Fi) : nullptr;
    s->part = !z.few_out && z.splits_out > 1 ? c.take<float>((size_t)z.splits_out * z.n * z.O) : nullptr;
    return c.off;
}
struct GradSpace {
    char* dpre;
    float* part_dh;
    float* part[3];
};
inline size_t carve_backward(Carve& c, GradSpace* s, const FeedSizes& z) {
    const int64_t M[3] = {z.n, 2 * (int64_t)z.F, z.O}, N[3] = {z.D, z.D, z.F};
    s->dpre = c.take<char>((size_t)z.n * 2 * z.Fp * z.bytes * (z.twice ? 2 : 1));
    s->part_dh = z.splits_dh > 1 ? c.take<float>((size_t)z.splits_dh * z.n * z.Fi) : nullptr;
    for (int i = 0; i < 3; ++i) s->part[i] = z.splits[i] > 1 ? c.take<float>((size_t)z.splits[i] * M[i] * N[i]) : nullptr;
    return c.off;
}

template <typename T>
int run_feed(const FeedSizes& z, int act, int dtype, const void* x, int64_t ldx, const void* w_in, const void* w_out,
             void* y, int64_t ldy, const FeedKept* kept, const FeedSpace& s, hipStream_t stream) {
    Product P = {};
    P.a = x, P.lda = ldx, P.b = w_in, P.ldb = z.D;
    P.M = (int)z.n, P.N = z.F, P.K = z.D;
    P.F = z.F, P.Fp = z.Fp, P.Fi = z.Fi, P.act = act, P.splits = z.splits_in, P.part = s.part_in;
    P.pre = kept ? kept->pre : nullptr;
    P.h = kept ? kept->h : z.whole ? nullptr : s.h;
    P.h32 = s.h32;
    P.again = z.twice ? z.n * z.Fp : 0;
    const int b = z.bytes;
    if (z.few) run_few<T, IN, false>(P, stream);
    else if (!run_tiles<T, IN>(P, z.large_in,
                               straight_ok(x, ldx, z.D, b) && straight_ok(w_in, z.D, z.D, b, (int64_t)z.F + 256), stream))
        return fail(-1, "yabt_feed_forward: bad sizes");
    run_join_inner<T, IN>(P, stream);
    Product Q = {};
    Q.b = w_out, Q.ldb = z.F;
    Q.M = (int)z.n, Q.N = z.O, Q.K = z.F;
    Q.out = y, Q.ldo = ldy, Q.out_dtype = dtype, Q.splits = 1;
    Q.a = P.h, Q.lda = z.Fp;
    if (z.few_out) {
        if (z.whole) Q.a = s.h32, Q.lda = z.Fi;
        if constexpr (sizeof(T) == 2) {
            if (z.whole) run_few<T, OUT, true>(Q, stream);
            else run_few<T, OUT, false>(Q, stream);
        } else {
            run_few<T, OUT, false>(Q, stream);
        }
    } else {
        Q.splits = z.splits_out, Q.part = s.part, Q.again_a = P.again;
        if (!run_tiles<T, OUT>(Q, z.large_out, straight_ok(w_out, z.F, z.F, b) && near_ok(256, z.Fp, b), stream))
            return fail(-1, "yabt_feed_forward: bad sizes");
        if (Q.splits > 1) run_join({{{s.part, y, ldy, Q.M, Q.N, Q.splits, dtype, nullptr, nullptr}}, 1}, stream);
    }
    return launch_status("yabt_feed_forward");
}

template <typename T>
int run_feed_grad(const FeedSizes& z, int act, int dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx,
                  const void* w_in, const void* w_out, const FeedKept& kept, const GradSpace& s, void* dx, int64_t lddx,
                  void* dw_in, void* dw_out, hipStream_t stream) {
    const int b = z.bytes;
    const bool dma = straight_ok(x, ldx, z.D, b) && straight_ok(dy, lddy, z.O, b) && straight_ok(w_in, z.D, z.D, b) &&
                     straight_ok(w_out, z.F, z.F, b) && near_ok(256, 2 * (int64_t)z.Fp, b);
    Product P = {};
    P.a = dy, P.lda = lddy, P.b = w_out, P.ldb = z.F, P.bw = z.F;
    P.M = (int)z.n, P.N = z.F, P.K = z.O;
    P.F = z.F, P.Fp = z.Fp, P.Fi = z.Fi, P.act = act, P.splits = z.splits_dh, P.part = s.part_dh;
    P.pre = kept.pre, P.dpre = s.dpre, P.again = z.twice ? z.n * 2 * z.Fp : 0;
    GradProducts G = {};
    for (auto& p : G.p) p.F = z.F, p.Fp = z.Fp, p.Fi = z.Fi, p.out_dtype = dtype;
    Product &X = G.p[0], &I = G.p[1], &O = G.p[2];
    X.a = s.dpre, X.lda = 2 * (int64_t)z.Fp, X.b = w_in, X.ldb = z.D, X.bw = z.D;
    X.M = (int)z.n, X.N = z.D, X.K = z.Fp + z.F, X.out = dx, X.ldo = lddx;
    I.a = s.dpre, I.lda = 2 * (int64_t)z.Fp, I.aw = 2 * z.Fp, I.b = x, I.ldb = ldx, I.bw = z.D;
    I.M = z.Fp + z.F, I.N = z.D, I.K = (int)z.n, I.out = dw_in, I.ldo = z.D;
    O.a = dy, O.lda = lddy, O.aw = z.O, O.b = kept.h, O.ldb = z.Fp, O.bw = z.Fp;
    O.M = z.O, O.N = z.F, O.K = (int)z.n, O.out = dw_out, O.ldo = z.F;
    for (int i = 0; i < 3; ++i) G.p[i].splits = z.splits[i], G.p[i].part = s.part[i];
    X.again_a = I.again_a = P.again, O.again_b = z.twice ? z.n * z.Fp : 0;
    auto launch_with = [&](auto tl, auto d, auto tlx) {
        using TL = decltype(tl);
        using TLX = decltype(tlx);
        if (!all_tiles<TLX>(X, false, &G.g[0]) || !all_tiles<TL>(I, false, &G.g[1]) || !all_tiles<TL>(O, false, &G.g[2]))
            return false;
        if (!grid_ok((int64_t)G.g[0].blocks + G.g[1].blocks + G.g[2].blocks, TL::NT)) return false;
        bool shared = false;
        if constexpr (!TWICE<TL>) {                  // the inner gradient's own operands have one part
            if (z.large_dh == z.large_grads) {
                Tiles gh;
                if (!all_tiles<TL>(P, false, &gh)) return false;
                Tiles go = take_last(&G.g[2], beside_inner_grad(z, gh.count, G.g));
                if (!grid_ok((int64_t)go.blocks + gh.blocks, TL::NT)) return false;
                if (go.blocks + gh.blocks)
                    k_feed_inner_grad<T, TL, decltype(d)::value>
                        <<<go.blocks + gh.blocks, TL::NT, TL::LDS, stream>>>(O, go, P, gh);
                shared = true;
            }
        }
        if (!shared && z.n > 0 && !run_tiles<T, DH>(P, z.large_dh, dma, stream)) return false;
        run_join_inner<T, DH>(P, stream);
        constexpr int lds = TLX::LDS > TL::LDS ? TLX::LDS : TL::LDS;
        k_feed_grads<T, TL, decltype(d)::value, TLX>
            <<<G.g[0].blocks + G.g[1].blocks + G.g[2].blocks, TL::NT, lds, stream>>>(G);
        return true;
    };
    auto launch = [&](auto tl, auto d) { return launch_with(tl, d, tl); };
    bool ok;
    if (sizeof(T) == 4 || !z.twice) {
        ok = by_tile<T>(z.large_grads, dma, launch);
    } else if constexpr (sizeof(T) == 2) {
        // dx by pairs, whose 64 KB of LDS leave two blocks a CU, unless the grid has more of them.  In one part, by
        // pairs and with every step twice, us for forward and backward, bf16: 4 x 512 -> 2000 -> 512 27.4, 28.8 and
        // 30.4; one row of 2048 -> 2048 -> 2048 43.2, 48.5 and 45.6
        int64_t blocks = 0;
        for (int i = 0; i < 3; ++i) blocks += tile_count(b, false, G.p[i].M, G.p[i].N) * z.splits[i];
        ok = !dma                ? launch_with(TileTwice(), std::false_type(), TilePair())
             : blocks <= 2 * CUS ? launch_with(TileTwice(), std::true_type(), TilePair())
                                 : launch(TileTwice(), std::true_type());
    }
    if (!ok) return fail(-1, "yabt_feed_forward_grad: bad sizes");
    Joins J = {};
    for (int i = 0; i < 3; ++i)
        if (G.p[i].splits > 1)
            J.j[J.count++] = {G.p[i].part, G.p[i].out, G.p[i].ldo, i == 1 ? 2 * z.F : G.p[i].M, G.p[i].N, G.p[i].splits,
                              dtype, nullptr, nullptr};
    run_join(J, stream);
    return launch_status("yabt_feed_forward_grad");
}

int run_quantize(int dtype, const void* x, int64_t ldx, int64_t n, int D, int8_t* q, int64_t ldq, float* scale,
                 hipStream_t stream) {
    by_dtype(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        // rows that a wave holds in its registers, and longer ones by a block each
        if (D <= 64 * QUANT_CHUNKS * VEC<T>)
            k_quantize<T, 64><<<(unsigned)over(n, 4), 256, 0, stream>>>((const T*)x, ldx, n, D, q, ldq, scale);
        else k_quantize<T, 256><<<(unsigned)n, 256, 0, stream>>>((const T*)x, ldx, n, D, q, ldq, scale);
        return 0;
    });
    return 0;
}
inline bool quantize_ok(int64_t n, int D) { return n >= 0 && n < (1 << 24) && D >= 1 && D <= (1 << 24); }

// A product of codes: how it is made.
struct Int8Sizes {
    bool few, large;
    int splits;
};
inline Int8Sizes int8_sizes(int64_t n, int64_t N, int64_t K) {
    Int8Sizes z;
    z.few = few_rows(n);
    z.large = large_product(1, n, N, K);
    z.splits = split_count(n, N, K, z.large, 1);
    return z;
}
// y = (a b^T) scaled, a (n, K) codes; part: splits x n x N floats where it is made in parts.
bool run_int8(const Int8Sizes& z, const int8_t* a, int64_t lda, const float* sa, int64_t n, int K, const int8_t* b,
              int64_t ldb, const float* sb, int N, int out_dtype, void* y, int64_t ldy, float* part, hipStream_t stream) {
    Product P = {};
    P.a = a, P.lda = lda, P.b = b, P.ldb = ldb, P.M = (int)n, P.N = N, P.K = K, P.sa = sa, P.sb = sb;
    P.out = y, P.ldo = ldy, P.out_dtype = out_dtype, P.splits = 1;
    if (z.few) {
        run_few<int8_t, OUT8, false>(P, stream);
        return true;
    }
    P.splits = z.splits, P.part = part;
    if (!run_tiles<int8_t, OUT8>(P, z.large, straight_ok(a, lda, K, 1) && straight_ok(b, ldb, K, 1), stream)) return false;
    if (P.splits > 1) run_join({{{part, y, ldy, P.M, N, P.splits, out_dtype, sa, sb}}, 1}, stream);
    return true;
}

struct Feed8Space {
    int8_t* q;                        // codes of x, then of h
    float* scale;
    float* h32;
    float* part_in;
    float* part;
};
inline int splits_in8(int64_t n, int D, int F) {
    const int64_t N = 2 * (int64_t)F;
    return few_rows(n) ? 1 : inner_split_count(IN, n, N, D, large_product(1, n, N, D), 1);
}
inline size_t carve_feed8(Carve& c, Feed8Space* s, int64_t n, int D, int F, int O) {
    const Int8Sizes z = int8_sizes(n, O, F);
    const int64_t w = D > F ? D : F;
    s->q = c.take<int8_t>((size_t)n * up16((int)w, 1));
    s->scale = c.take<float>((size_t)n);
    const int in = splits_in8(n, D, F);
    s->h32 = c.take<float>((size_t)n * up16(F, 4));
    s->part_in = in > 1 ? c.take<float>((size_t)in * n * 2 * up16(F, 4)) : nullptr;
    s->part = !z.few && z.splits > 1 ? c.take<float>((size_t)z.splits * n * O) : nullptr;
    return c.off;
}

}  // namespace yabt

using namespace yabt;

extern "C" {

size_t yabt_feed_forward_inner_bytes(int dtype, int64_t n, int D, int F, int O) {
    FeedSizes z;
    if (!feed_sizes_ok(dtype, n, D, F, O, &z)) return 0;
    Carve c{nullptr, 0};
    FeedKept k;
    return carve_kept(c, &k, z) + 256;
}

size_t yabt_feed_forward_workspace_bytes(int dtype, int64_t n, int D, int F, int O) {
    FeedSizes z;
    if (!feed_sizes_ok(dtype, n, D, F, O, &z)) return 0;
    Carve c{nullptr, 0};
    FeedSpace s;
    return carve_forward(c, &s, z) + 256;
}

int yabt_feed_forward(int dtype, int act, const void* x, int64_t ldx, int64_t n, int D, int F, int O, const void* w_in,
                      const void* w_out, void* workspace, size_t workspace_bytes, void* out_inner, void* y, int64_t ldy,
                      yabt_stream_t stream) {
    if (!dtype_ok(dtype)) return fail(-1, "yabt_feed_forward: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (act < SILU || act > RELU) return fail(-1, "yabt_feed_forward: the activation is 0 to 3");
    FeedSizes z;
    if (!feed_sizes_ok(dtype, n, D, F, O, &z) || ldx < D || ldy < O) return fail(-1, "yabt_feed_forward: bad sizes");
    if (n == 0) return 0;
    if (!x || !w_in || !w_out || !y) return fail(-1, "yabt_feed_forward: null pointer");
    if (!workspace || workspace_bytes < yabt_feed_forward_workspace_bytes(dtype, n, D, F, O))
        return fail(-2, "yabt_feed_forward: workspace too small");
    FeedKept kept;
    if (out_inner) {
        Carve c{(char*)align_up((size_t)out_inner, 256), 0};
        carve_kept(c, &kept, z);
    }
    FeedSpace s;
    Carve c{(char*)align_up((size_t)workspace, 256), 0};
    carve_forward(c, &s, z);
    return by_dtype(dtype, [&](auto* t) {
        return run_feed<std::remove_pointer_t<decltype(t)>>(z, act, dtype, x, ldx, w_in, w_out, y, ldy,
                                                            out_inner ? &kept : nullptr, s, (hipStream_t)stream);
    });
}

int yabt_feed_forward_forms(int dtype, int64_t n, int D, int F, int O) {
    FeedSizes z;
    if (!feed_sizes_ok(dtype, n, D, F, O, &z)) return -1;
    return (int)z.few | (int)z.few_out << 1 | (int)(z.large_in && !z.few) << 2 | (int)(z.large_out && !z.few_out) << 3 |
           (int)z.large_dh << 4 | (int)z.large_grads << 5 | (int)(z.splits_in > 1) << 6 |
           (int)(!z.few_out && z.splits_out > 1) << 7 | (int)(z.splits_dh > 1) << 8 |
           (int)(z.splits[0] > 1 || z.splits[1] > 1 || z.splits[2] > 1) << 9 | (int)z.whole << 10 | (int)z.twice << 11;
}

size_t yabt_feed_forward_grad_workspace_bytes(int dtype, int64_t n, int D, int F, int O) {
    FeedSizes z;
    if (!feed_sizes_ok(dtype, n, D, F, O, &z)) return 0;
    Carve c{nullptr, 0};
    GradSpace s;
    return carve_backward(c, &s, z) + 256;
}

int yabt_feed_forward_grad(int dtype, int act, const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t n, int D,
                           int F, int O, const void* w_in, const void* w_out, const void* inner, void* workspace,
                           size_t workspace_bytes, void* dx, int64_t lddx, void* dw_in, void* dw_out, yabt_stream_t stream) {
    if (!dtype_ok(dtype)) return fail(-1, "yabt_feed_forward_grad: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (act < SILU || act > RELU) return fail(-1, "yabt_feed_forward_grad: the activation is 0 to 3");
    FeedSizes z;
    if (!feed_sizes_ok(dtype, n, D, F, O, &z) || ldx < D || lddy < O || lddx < D)
        return fail(-1, "yabt_feed_forward_grad: bad sizes");
    if (!w_in || !w_out || !dw_in || !dw_out || (n > 0 && (!x || !dy || !inner || !dx)))
        return fail(-1, "yabt_feed_forward_grad: null pointer");
    if (!workspace || workspace_bytes < yabt_feed_forward_grad_workspace_bytes(dtype, n, D, F, O))
        return fail(-2, "yabt_feed_forward_grad: workspace too small");
    FeedKept kept;
    Carve k{(char*)align_up((size_t)inner, 256), 0};
    carve_kept(k, &kept, z);
    GradSpace s;
    Carve c{(char*)align_up((size_t)workspace, 256), 0};
    carve_backward(c, &s, z);
    return by_dtype(dtype, [&](auto* t) {
        return run_feed_grad<std::remove_pointer_t<decltype(t)>>(z, act, dtype, dy, lddy, x, ldx, w_in, w_out, kept, s, dx,
                                                                 lddx, dw_in, dw_out, (hipStream_t)stream);
    });
}

int yabt_quantize_rows(int dtype, const void* x, int64_t ldx, int64_t n, int D, int8_t* out_codes, int64_t ldq,
                       float* out_scale, yabt_stream_t stream) {
    if (!dtype_ok(dtype)) return fail(-1, "yabt_quantize_rows: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (!quantize_ok(n, D) || ldx < D || ldq < D) return fail(-1, "yabt_quantize_rows: bad sizes");
    if (n == 0) return 0;
    if (!x || !out_codes || !out_scale) return fail(-1, "yabt_quantize_rows: null pointer");
    run_quantize(dtype, x, ldx, n, D, out_codes, ldq, out_scale, (hipStream_t)stream);
    return launch_status("yabt_quantize_rows");
}

static bool int8_ranges_ok(int64_t n, int K, int N) {
    if (!(n >= 0 && n < (1 << 24) && K >= 1 && K <= INT8_MOST && N >= 1 && N <= (1 << 24))) return false;
    const Int8Sizes z = int8_sizes(n, N, K);
    return tiles_fit(z.large, tiles_of(1, z.large, n, N) * z.splits);
}
static bool feed8_ranges_ok(int64_t n, int D, int F, int O) {
    if (!int8_ranges_ok(n, F, O) || D < 1 || D > INT8_MOST || F < 1 || F > INT8_MOST) return false;
    const bool large = large_product(1, n, 2 * (int64_t)F, D);
    return tiles_fit(large, tiles_of(1, large, n, 2.0 * F));
}

size_t yabt_product_int8_workspace_bytes(int64_t n, int K, int N) {
    if (!int8_ranges_ok(n, K, N)) return 0;
    const Int8Sizes z = int8_sizes(n, N, K);
    return z.few || z.splits == 1 ? 1 : (size_t)z.splits * n * N * 4 + 256;
}

int yabt_product_int8(const int8_t* a, int64_t lda, const float* a_scale, int64_t n, int K, const int8_t* b, int64_t ldb,
                      const float* b_scale, int N, int out_dtype, void* workspace, size_t workspace_bytes, void* y,
                      int64_t ldy, yabt_stream_t stream) {
    if (!dtype_ok(out_dtype)) return fail(-1, "yabt_product_int8: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (!int8_ranges_ok(n, K, N) || lda < K || ldb < K || ldy < N) return fail(-1, "yabt_product_int8: bad sizes");
    if (n == 0) return 0;
    if (!a || !a_scale || !b || !b_scale || !y) return fail(-1, "yabt_product_int8: null pointer");
    const size_t need = yabt_product_int8_workspace_bytes(n, K, N);
    if (need > 1 && (!workspace || workspace_bytes < need)) return fail(-2, "yabt_product_int8: workspace too small");
    if (!run_int8(int8_sizes(n, N, K), a, lda, a_scale, n, K, b, ldb, b_scale, N, out_dtype, y, ldy,
                  (float*)align_up((size_t)workspace, 256), (hipStream_t)stream))
        return fail(-1, "yabt_product_int8: bad sizes");
    return launch_status("yabt_product_int8");
}

size_t yabt_feed_forward_int8_workspace_bytes(int64_t n, int D, int F, int O) {
    if (!feed8_ranges_ok(n, D, F, O)) return 0;
    Carve c{nullptr, 0};
    Feed8Space s;
    return carve_feed8(c, &s, n, D, F, O) + 256;
}

int yabt_feed_forward_int8_forms(int64_t n, int D, int F, int O) {
    if (!feed8_ranges_ok(n, D, F, O)) return -1;
    const Int8Sizes z = int8_sizes(n, O, F);
    const bool few = few_rows(n), large = large_product(1, n, 2 * (int64_t)F, D);
    return (int)few | (int)few << 1 | (int)(large && !few) << 2 | (int)(z.large && !few) << 3 |
           (int)(splits_in8(n, D, F) > 1) << 6 | (int)(z.splits > 1 && !few) << 7 | (int)(few && few_values(n, D)) << 10 |
           (int)(few && few_values(n, F)) << 11;
}

int yabt_feed_forward_int8(int dtype, int act, const void* x, int64_t ldx, int64_t n, int D, int F, int O,
                           const int8_t* w_in, const float* in_scale, const int8_t* w_out, const float* out_scale, void* workspace,
                           size_t workspace_bytes, void* y, int64_t ldy, yabt_stream_t stream) {
    if (!dtype_ok(dtype)) return fail(-1, "yabt_feed_forward_int8: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (act < SILU || act > RELU) return fail(-1, "yabt_feed_forward_int8: the activation is 0 to 3");
    if (!feed8_ranges_ok(n, D, F, O) || ldx < D || ldy < O)
        return fail(-1, "yabt_feed_forward_int8: bad sizes");
    if (n == 0) return 0;
    if (!x || !w_in || !in_scale || !w_out || !out_scale || !y) return fail(-1, "yabt_feed_forward_int8: null pointer");
    if (!workspace || workspace_bytes < yabt_feed_forward_int8_workspace_bytes(n, D, F, O))
        return fail(-2, "yabt_feed_forward_int8: workspace too small");
    const hipStream_t on = (hipStream_t)stream;
    Feed8Space s;
    Carve c{(char*)align_up((size_t)workspace, 256), 0};
    carve_feed8(c, &s, n, D, F, O);
    const int Fi = up16(F, 4), dq = up16(D, 1), fq = up16(F, 1);
    Product P = {};
    P.b = w_in, P.ldb = D, P.M = (int)n, P.N = F, P.K = D, P.F = F, P.Fp = Fi, P.Fi = Fi, P.act = act, P.h32 = s.h32;
    P.sb = in_scale, P.splits = splits_in8(n, D, F), P.part = s.part_in;
    if (few_rows(n) && few_values(n, D)) {
        P.a = x, P.lda = ldx, P.x_dtype = dtype;
        run_few<int8_t, IN8, true>(P, on);
    } else {
        run_quantize(dtype, x, ldx, n, D, s.q, dq, s.scale, on);
        P.a = s.q, P.lda = dq, P.sa = s.scale;
        if (few_rows(n)) run_few<int8_t, IN8, false>(P, on);
        else if (!run_tiles<int8_t, IN8>(P, large_product(1, n, 2 * (int64_t)F, D),
                                         straight_ok(s.q, dq, D, 1) && straight_ok(w_in, D, D, 1, (int64_t)F + 256), on))
            return fail(-1, "yabt_feed_forward_int8: bad sizes");
        run_join_inner<int8_t, IN8>(P, on);
    }
    if (few_rows(n) && few_values(n, F)) {
        Product Q = {};
        Q.a = s.h32, Q.lda = Fi, Q.x_dtype = DT_F32, Q.b = w_out, Q.ldb = F, Q.M = (int)n, Q.N = O, Q.K = F;
        Q.sb = out_scale, Q.out = y, Q.ldo = ldy, Q.out_dtype = dtype, Q.splits = 1;
        run_few<int8_t, OUT8, true>(Q, on);
    } else {
        run_quantize(DT_F32, s.h32, Fi, n, F, s.q, fq, s.scale, on);
        if (!run_int8(int8_sizes(n, O, F), s.q, fq, s.scale, n, F, w_out, F, out_scale, O, dtype, y, ldy, s.part, on))
            return fail(-1, "yabt_feed_forward_int8: bad sizes");
    }
    return launch_status("yabt_feed_forward_int8");
}

}  // extern "C"
