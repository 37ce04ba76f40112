// The experts' products, forward and backward, on the matrix cores.
//
//   slot s = (row t, j), expert e:  [g u] = W_in[e] x_t,  h = silu(g) u,  z_s = W_out[e] h,  y_t = sum_j w_s z_s
//   a = W_out[e]^T dy_t,  dw_s = a . h,  dh = w_s a,  du = dh silu(g),  dg = dh u silu'(g)
//   dx_t = sum_j W_in[e]^T [dg du],  dW_in[e] = sum_s [dg du] x_t^T,  dW_out[e] = sum_s dy_t (w_s h)^T
//
// The slots come sorted by expert (yabt_expert_plan), so that every product is
// one matrix product per expert over its slots; a launch does all experts'.
// One kernel makes the tiles of all six products.  They differ in where a
// tile's rows come from (gathered rows of x or dy, or the slots' own rows), in
// whether an operand lies along the summed dimension in memory or across it,
// and in what is done with the sums:
//
//   IN     [g u] of the slots, the tile's columns gate and up alternately by 32, then h = silu(g) u
//   OUT    z = w (W_out h), by slot in fp32 (added up by k_finish), or y itself when k = 1
//   DH     a, then dg, du, w h and dw in part
//   DX     W_in^T [dg du] by slot in fp32, or dx itself when k = 1
//   DWIN, DWOUT   the weights' gradients, summed over an expert's slots
//
// Both operands pass through LDS in steps of 128 bytes of the summed dimension:
// the next steps are on their way from memory straight into LDS while the
// present one is multiplied.  16-byte pieces are stored at places that an
// xor with the row spreads over the banks; the xor is applied to the global
// address, as LDS is filled in lane order.  Operands across the summed
// dimension are read with the transposing LDS loads.  Inputs whose rows are
// not 16-byte aligned pass through registers instead.
//
// 16 384 x 2048 rows, 2 of 8 experts of 2048, bf16 (550 GFLOP for h, 275 for y and the
// inner gradient, 1375 for the other three): 0.60, 0.32, 0.51 and 1.58 ms over the
// first dozen passes, 0.57, 0.30, 0.48 and 1.46 over a hundred, the matrix
// cores at work 59, 61, 34 and 50% of the CUs' busy time; the library's plain
// product of 275 GFLOP alone takes 0.21 ms.  What is between them: a block has its
// CU to itself (its sums are 256 KB of registers), so that what a tile reads and
// writes besides (h with the kept g and u 0.67 GB, the inner gradient 0.95 GB) and its
// first loads are not covered, a quarter of what the steps take comes from behind
// L2 (h: 1.1 of 4.3 GB), the experts' last tiles are partly empty, and so is the last
// round of 256 tiles (h has 8.5, y 4.25).  Two blocks of 128 x 256 a CU, which cover
// each other, fetch half more: 0.69, 0.36, 0.52 and 1.80 ms.
//
// h, w h, dg and du are rounded to the inputs' type, as the matrix cores take
// them; g and u are kept in fp32 for the backward pass, and z and the parts of
// dx are added in fp32: so each output has two roundings behind it, its own
// and that of one factor (0.0023 from the formulas in 64 bits where its own alone
// leaves 0.0017, bf16).  In fp16 they have the type's range: an h beyond 65504 is
// infinite.  Two parts of 16 bits each would take that rounding away for
// twice the arithmetic of all products but h and dh; float32 tensors have none.

#include "expert.h"
#include "yabt_hip.h"

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

enum Mode { IN, OUT, DH, DX, DWIN, DWOUT };

constexpr int XCDS = 8;               // blocks go to the 8 dies in turn
constexpr int TILE_GROUP = 4;         // row tiles that walk the column tiles together

struct ExpertArgs {
    const void* x;
    const void* dy;
    const void* w_in;                 // (E, 2 F, D)
    const void* w_out;                // (E, D, F)
    const float* weights;             // (n, k)
    const int32_t* ids;               // (n, k)
    const int32_t* offsets;           // (E + 1), the plan
    const int32_t* slots;
    const int32_t* rows;
    int64_t ldx, lddy, n;
    int k, D, F, E;
    int Fp;                           // F up to whole 16 bytes: the pitch of h and w h, half that of [dg du]
    int Dp;                           // D up to a multiple of 4: the pitch of z
    int Fi;                           // F up to a multiple of 4: half the pitch of pre
    void* h;                          // (S, Fp)
    void* hw;                         // (S, Fp): w h
    void* dpre;                       // (S, 2 Fp): dg from 0, du from Fp
    float* pre;                       // (S, 2 Fi): g from 0, u from Fi, or NULL
    float* z;                         // (S, Dp)
    float* dwp;                       // (parts, S): dw by column tile
    void* out;                        // y or dx
    int64_t ldo;
    void* dw_in;                      // (E, 2 F, D)
    void* dw_out;                     // (E, D, F)
    float* part_in;                   // (splits_in, E, 2 F, D): dw_in in part, where splits_in > 1
    float* part_out;                  // (splits_out, E, D, F)
    int splits_in, splits_out;
    float* dweights;                  // (n, k), or NULL: not wanted
    int parts;                        // of dwp
};

// 16 zero bytes for pieces past the end of the summed dimension.
__device__ const u32x4 g_zeros = {0, 0, 0, 0};

// BM x BN sums by WM x WN waves, in steps of STEP bytes of the summed dimension;
// LDS holds AS steps of the rows' operand and BS <= AS of the columns'.
template <int BM_, int BN_, int WM_, int WN_, int STEP_, int AS_, int BS_>
struct TileOf {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STEP = STEP_, AS = AS_, BS = BS_;
    static constexpr int NT = 64 * WM * WN;
    static constexpr int MI = BM / WM / 32, NI = BN / WN / 32;    // 32 x 32 blocks a wave makes
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

// The slots' row tiles, BM slots of one expert each: a lane counts those of
// expert e0 + lane, and up to 64 experts are read once.
struct RowTiles {
    const int32_t* off;
    int E, BM;
    int first, count, upto;           // of the 64 experts in view: this lane's first slot, slots, and tiles up to it
    __device__ __forceinline__ void view(int e0) {
        const int lane = threadIdx.x & 63, e = e0 + lane;
        first = e < E ? off[e] : 0;
        count = e < E ? off[e + 1] - first : 0;
        upto = (count + BM - 1) / BM;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int o = __shfl_up(upto, m);
            if (lane >= m) upto += o;
        }
    }
    __device__ __forceinline__ int total() {
        int t = 0;
        for (int e0 = 0; e0 < E; e0 += 64) {
            view(e0);
            t += __shfl(upto, 63);
        }
        return t;
    }
    // Tile id < total(): its expert, first place and slots.
    __device__ __forceinline__ void find(int id, int* e, int* p0, int* slots) {
        int carry = 0;
        for (int e0 = 0;; e0 += 64) {
            if (E > 64) view(e0);
            const uint64_t hit = __ballot(id < carry + upto);
            if (hit) {
                const int l = __ffsll((unsigned long long)hit) - 1;
                const int c = __shfl(count, l), mi = id - carry - (__shfl(upto, l) - (c + BM - 1) / BM);
                *e = e0 + l;
                *p0 = __shfl(first, l) + mi * BM;
                *slots = min(BM, c - mi * BM);
                return;
            }
            carry += __shfl(upto, 63);
        }
    }
};

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

// The pieces of an operand that a thread brings to LDS.  The mode says where a
// row lies; pieces past the end of the summed dimension are zero, rows and
// columns past the tile's end repeat the last (their sums are not stored).
template <typename T, int MODE, bool SIDE_B, int W, int COUNT, int NT, int STEP>
struct Loader {
    static constexpr bool ACROSS = SIDE_B ? MODE >= DH : MODE >= DWIN;
    static constexpr bool GATHER = SIDE_B ? MODE == DWIN : MODE == IN || MODE == DH || MODE == DWOUT;
    static constexpr int CH = VEC<T>;
    static constexpr int PER_ROW = ACROSS ? W * (int)sizeof(T) / 16 : STEP / 16;
    const T* ptr[COUNT];       // along: the row, at this piece; across: column of the piece, from row 0
    int32_t src[COUNT], nxt[COUNT];   // across and gathered: the rows of the step to send, and of the one after

    __device__ __forceinline__ static int row_of(int i) { return (i * NT + (int)threadIdx.x) / PER_ROW; }
    __device__ __forceinline__ static int piece_of(int i) {
        const int c = (i * NT + (int)threadIdx.x) % PER_ROW, r = row_of(i);
        return c ^ spread<T, ACROSS, W, STEP>(r);
    }

    // p0: the tile's first slot place (along), or the split's (across); count:
    // how many there are; first: the tile's first row or column of the operand
    __device__ __forceinline__ void init(const ExpertArgs& P, int e, int p0, int count, int first) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const int r = row_of(i), piece = piece_of(i) * CH;
            if constexpr (!ACROSS && !SIDE_B) {
                const int p = p0 + min(r, count - 1);
                if constexpr (MODE == IN) ptr[i] = (const T*)P.x + (size_t)P.rows[p] * (size_t)P.ldx;
                else if constexpr (MODE == DH) ptr[i] = (const T*)P.dy + (size_t)P.rows[p] * (size_t)P.lddy;
                else if constexpr (MODE == OUT) ptr[i] = (const T*)P.h + (size_t)p * (size_t)P.Fp;
                else ptr[i] = (const T*)P.dpre + (size_t)p * 2 * (size_t)P.Fp;
                ptr[i] += piece;
            } else if constexpr (!ACROSS) {
                if constexpr (MODE == IN) {
                    // gate and up rows alternately by 32
                    const int f = min(first + (r >> 6) * 32 + (r & 31), P.F - 1);
                    ptr[i] = (const T*)P.w_in + ((size_t)e * 2 * P.F + (r >> 5 & 1 ? P.F : 0) + f) * (size_t)P.D;
                } else {
                    ptr[i] = (const T*)P.w_out + ((size_t)e * P.D + min(first + r, P.D - 1)) * (size_t)P.F;
                }
                ptr[i] += piece;
            } else {
                const T* base;
                int width;
                if constexpr (SIDE_B) {
                    if constexpr (MODE == DH) base = (const T*)P.w_out + (size_t)e * P.D * (size_t)P.F, width = P.F;
                    else if constexpr (MODE == DX) base = (const T*)P.w_in + (size_t)e * 2 * P.F * (size_t)P.D, width = P.D;
                    else if constexpr (MODE == DWIN) base = (const T*)P.x, width = P.D;
                    else base = (const T*)P.hw + (size_t)p0 * (size_t)P.Fp, width = P.Fp;
                } else {
                    if constexpr (MODE == DWIN) base = (const T*)P.dpre + (size_t)p0 * 2 * (size_t)P.Fp, width = 2 * P.Fp;
                    else base = (const T*)P.dy, width = P.D;
                }
                ptr[i] = base + min(first + piece, max(width - CH, 0));
            }
        }
    }

    // the summed dimension's length as this operand has it
    __device__ __forceinline__ static int length(const ExpertArgs& P, int count) {
        if constexpr (MODE == IN || MODE == DH) return P.D;
        if constexpr (MODE == OUT) return SIDE_B ? P.F : P.Fp;
        if constexpr (MODE == DX) return P.Fp + P.F;
        return count;
    }
    __device__ __forceinline__ static int width(const ExpertArgs& P) {
        if constexpr (SIDE_B) return MODE == DH ? P.F : MODE == DWOUT ? P.Fp : P.D;
        return MODE == DWIN ? 2 * P.Fp : P.D;
    }

    // rows of x or dy of the step from k0 on
    __device__ __forceinline__ void look_up(const ExpertArgs& P, int p0, int count, int k0) {
        if constexpr (ACROSS && GATHER) {
#pragma unroll
            for (int i = 0; i < COUNT; ++i) {
                const int kk = k0 + row_of(i);
                nxt[i] = kk < count ? P.rows[p0 + kk] : -1;
            }
        }
    }
    __device__ __forceinline__ void move_on() {
        if constexpr (ACROSS && GATHER) {
#pragma unroll
            for (int i = 0; i < COUNT; ++i) src[i] = nxt[i];
        }
    }

    // where piece i of the step from k0 on lies, or null past the end
    __device__ __forceinline__ const T* at(const ExpertArgs& P, int i, int k0, int len) const {
        if constexpr (!ACROSS) {
            return k0 + piece_of(i) * CH < len ? ptr[i] + k0 : nullptr;
        } else if constexpr (GATHER) {
            const size_t ld = (size_t)(SIDE_B ? P.ldx : P.lddy);
            return src[i] >= 0 ? ptr[i] + (size_t)src[i] * ld : nullptr;
        } else {
            int kk = k0 + row_of(i);
            if (kk >= len) return nullptr;
            size_t ld;
            if constexpr (MODE == DH) ld = (size_t)P.F;
            else if constexpr (MODE == DX) {
                ld = (size_t)P.D;
                if (kk >= P.F) {
                    if (kk < P.Fp) return nullptr;
                    kk += P.F - P.Fp;
                }
            } else {
                ld = (size_t)(SIDE_B ? P.Fp : 2 * P.Fp);
            }
            return ptr[i] + (size_t)kk * ld;
        }
    }

    // pieces LO .. HI - 1 of the step from k0 on
    template <int LO = 0, int HI = COUNT>
    __device__ __forceinline__ void fill(const ExpertArgs& P, int k0, int len, uint32_t lds) const {
#pragma unroll
        for (int i = LO; i < HI; ++i) {
            const T* p = at(P, i, k0, len);
            const uint32_t base = lds + (uint32_t)(i * NT * 16) + ((threadIdx.x & ~63u) << 4);
            lds_fill(p ? (const void*)p : (const void*)&g_zeros, __builtin_amdgcn_readfirstlane(base));
        }
    }

    // the same through registers, for rows at any address: the values that
    // exist, zeros for the others
    __device__ __forceinline__ void fetch(const ExpertArgs& P, int k0, int len, int first, u32x4* v) const {
        typedef T VT __attribute__((ext_vector_type(CH)));
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const T* p = at(P, i, k0, len);
            u32x4 o = {0, 0, 0, 0};
            if (p) {
                const int piece = piece_of(i) * CH;
                int have;
                if constexpr (ACROSS) {
                    // the column clamp of init() does not hold pieces that end past the row
                    const int w = width(P);
                    p += first + piece - min(first + piece, max(w - CH, 0));
                    have = w - (first + piece);
                } else {
                    have = len - (k0 + piece);
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

extern __shared__ __attribute__((aligned(128))) char s_tiles[];

// One tile of the product MODE: that of the block with number `block` of its
// product's grid of `ntiles` column tiles (and, of a weight's gradient, `mtiles`
// row tiles).
template <typename T, int MODE, typename TL, bool DMA>
__device__ __forceinline__ void expert_tile(const ExpertArgs& P, uint32_t block, int ntiles, int mtiles) {
    constexpr bool ROWS = MODE < DWIN;
    const int splits = MODE == DWIN ? P.splits_in : P.splits_out;
    lds_char* const lds = (lds_char*)s_tiles;
    const uint32_t lds_at = (uint32_t)(uintptr_t)lds;
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    const int wm = wave / TL::WN, wn = wave % TL::WN;

    // which tile: expert e, slots [p0, p0 + count), first row mf and column nf
    int e, p0, count, mf = 0, nf, split = 0, my_slot = 0;
    float my_w = 1.0f;
    if constexpr (ROWS) {
        RowTiles tiles{P.offsets, P.E, TL::BM};
        const int total = tiles.total();
        const int64_t all = (int64_t)total * ntiles, id = die_order(block, all);
        if (id >= all) return;
        const int group = (int)(id / ((int64_t)TILE_GROUP * ntiles));
        const int in = (int)(id - (int64_t)group * TILE_GROUP * ntiles);
        const int gm = min(TILE_GROUP, total - group * TILE_GROUP);
        tiles.find(group * TILE_GROUP + in % gm, &e, &p0, &count);
        nf = in / gm * (MODE == IN ? TL::BN / 2 : TL::BN);
        // a row a thread, kept until the sums are there
        if constexpr (MODE != IN) {
            if ((int)threadIdx.x < count) {
                my_slot = P.slots[p0 + threadIdx.x];
                if constexpr (MODE != DX) my_w = P.weights[my_slot];
            }
        }
    } else {
        // an expert's tiles over all dies: experts differ in how long theirs take
        const int per = mtiles * ntiles, all = per * splits, up = (all + XCDS - 1) / XCDS * XCDS;
        e = (int)(block / up);
        if (e >= P.E) return;
        const int64_t id = die_order(block - (int64_t)e * up, all);
        if (id >= all) return;
        split = (int)(id / per);
        const int in = (int)(id - (int64_t)split * per);
        // column tiles together with a group of row tiles
        const int group = in / (TILE_GROUP * ntiles), gin = in - group * TILE_GROUP * ntiles;
        const int gm = min(TILE_GROUP, mtiles - group * TILE_GROUP);
        mf = (group * TILE_GROUP + gin % gm) * TL::BM;
        nf = gin / gm * TL::BN;
        const int off = P.offsets[e], cnt = P.offsets[e + 1] - off;
        const int step = TL::STEP / (int)sizeof(T);
        const int part = ((cnt + splits - 1) / splits + step - 1) / step * step;
        const int lo = min(cnt, split * part);
        p0 = off + lo;
        count = min(part, cnt - lo);
    }

    Loader<T, MODE, false, TL::BM, TL::NA, TL::NT, TL::STEP> la;
    Loader<T, MODE, true, TL::BN, TL::NB, TL::NT, TL::STEP> lb;
    using LA = decltype(la);
    using LB = decltype(lb);
    const int ka = LA::length(P, count), kb = LB::length(P, count), K = max(ka, kb);
    constexpr int BK = TL::STEP / (int)sizeof(T), KS = TL::STEP / 32;
    const int steps = (K + BK - 1) / BK;
    f32x16 acc[TL::MI][TL::NI];
#pragma unroll
    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
        for (int j = 0; j < TL::NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

    if (steps > 0) {
        la.init(P, e, p0, count, mf);
        lb.init(P, e, p0, count, nf);
        // Step t of the rows' operand lies at place t % AS, of the columns' at t % 2.
        // The columns' step t + 2 is sent as soon as its place is free, at the end of
        // step t; the rows' step t + 2 there too, or, with a third place, in two
        // halves between the products of step t: a wave that sends waits for the
        // address units, which take a piece of 1 KB in 16 cycles for the whole CU,
        // and multiplies nothing meanwhile.  For operands whose rows are looked up
        // the rows of the step after are asked for first, so that a wait for them is
        // none for the pieces.  Steps past the last are sent too (zeros), so that
        // every wait is the same.  Without DMA a step waits in registers for its place.
        constexpr int AS = DMA ? TL::AS : 2;
        constexpr bool HALVES = AS == 3;
        static_assert(TL::BS == 2 && (AS == 2 || AS == 3), "places that the order of the steps is made for");
        u32x4 ra[DMA ? 1 : TL::NA], rb[DMA ? 1 : TL::NB];
        auto send_a = [&](int t, int place) {
            la.move_on();
            la.look_up(P, p0, count, (t + 1) * BK);
            if constexpr (DMA) la.fill(P, t * BK, ka, lds_at + (uint32_t)place * TL::ABYTES);
            else la.fetch(P, t * BK, ka, mf, ra);
        };
        auto send_b = [&](int t) {
            lb.move_on();
            lb.look_up(P, p0, count, (t + 1) * BK);
            if constexpr (DMA) lb.fill(P, t * BK, kb, lds_at + TL::AS * TL::ABYTES + (uint32_t)(t & 1) * TL::BBYTES);
            else lb.fetch(P, t * BK, kb, nf, rb);
        };
        auto put = [&](int t) {
            LA::put(lds + (t & 1) * TL::ABYTES, ra);
            LB::put(lds + TL::AS * TL::ABYTES + (t & 1) * TL::BBYTES, rb);
        };
        la.look_up(P, p0, count, 0);
        lb.look_up(P, p0, count, 0);
        // accesses of every wave after step 0's and, in the loop, after the next step's
        constexpr int AFTER_0 = DMA ? TL::NA + TL::NB : 0, AFTER = HALVES ? TL::NA : 0;
        if constexpr (DMA) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                send_a(t, t);
                send_b(t);
            }
        } else {
            send_a(0, 0);
            send_b(0);
            put(0);
            send_a(1, 0);
            send_b(1);
        }
        const Frag<T, LA::ACROSS, TL::BM, TL::STEP> fa(wm * TL::MI * 32);
        const Frag<T, LB::ACROSS, TL::BN, TL::STEP> fb(wn * TL::NI * 32);
        u32x4 a[2][TL::MI], b[2][TL::NI];
        auto read = [&](int place, int t, int ks) {
            lds_char* const ta = lds + place * TL::ABYTES;
            lds_char* const tb = lds + TL::AS * TL::ABYTES + (t & 1) * TL::BBYTES;
#pragma unroll
            for (int i = 0; i < TL::MI; ++i) a[ks & 1][i] = fa.get(ta, i, ks);
#pragma unroll
            for (int j = 0; j < TL::NI; ++j) b[ks & 1][j] = fb.get(tb, j, ks);
        };
        constexpr int READS = TL::MI * decltype(fa)::READS + TL::NI * decltype(fb)::READS;
        constexpr int PRODUCTS = TL::MI * TL::NI * (sizeof(T) == 4 ? 4 : 1);
        stage_ready<AFTER_0>();
        read(0, 0, 0);
        // A k-step's operands are read while the one before is multiplied, the
        // next step's first ones too: the wait for it stands before the last
        // k-step's products, and what takes the freed places is sent there.
        int place = 0;
        for (int t = 0; t < steps; ++t) {
            const int next = place + 1 == AS ? 0 : place + 1, free = next + 1 == AS ? 0 : next + 1;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (ks + 1 < KS) {
                    if constexpr (HALVES) {
                        const uint32_t to = lds_at + (uint32_t)free * TL::ABYTES;
                        if (ks == 0) {
                            la.move_on();
                            la.look_up(P, p0, count, (t + 3) * BK);
                            la.template fill<0, TL::NA / 2>(P, (t + 2) * BK, ka, to);
                        } else if (ks == 1) {
                            la.template fill<TL::NA / 2, TL::NA>(P, (t + 2) * BK, ka, to);
                        }
                    }
                    read(place, t, ks + 1);
                } else {
                    if constexpr (!DMA) put(t + 1);
                    stage_ready<AFTER>();
                    send_b(t + 2);
                    if constexpr (!HALVES) send_a(t + 2, place);
                    read(next, t + 1, 0);
                }
#pragma unroll
                for (int i = 0; i < TL::MI; ++i)
#pragma unroll
                    for (int j = 0; j < TL::NI; ++j) acc[i][j] = mma<T>(a[ks & 1][i], b[ks & 1][j], acc[i][j]);
                if constexpr (DMA) interleave<PRODUCTS, READS>();
            }
            place = next;
        }
        stage_ready<0>();                            // nothing may reach the LDS of a block that is gone
    }

    // The sums go through LDS, 32 rows of a wave at a time, from the matrix
    // cores' layout (a lane has one column) to four neighbouring columns a lane,
    // so that what is read and written beside them goes in whole lines.
    lds_int* const s_slot = (lds_int*)(lds + TL::SUMS);
    lds_float* const s_w = (lds_float*)(lds + TL::SUMS + TL::BM * 4);
    if constexpr (ROWS && MODE != IN) {
        if (threadIdx.x < TL::BM) {
            s_slot[threadIdx.x] = my_slot;
            s_w[threadIdx.x] = my_w;
        }
        __syncthreads();
    }
    constexpr int W = TL::NI * 32;
    lds_float* const mine = (lds_float*)(lds + wave * 32 * W * 4);
    constexpr int LANES = MODE == IN ? W / 8 : W / 4, PASS = 64 / LANES;    // lanes a row, rows at once
    const int c4 = lane % LANES * 4;
#pragma unroll
    for (int i = 0; i < TL::MI; ++i) {
        wave_sync_lds();
        // sum r of block (i, j): row 8 (r / 4) + 4 (lane / 32) + r % 4, column 32 j + lane % 32;
        // the rows of the upper lanes are kept with their blocks in pairs swapped: other banks
#pragma unroll
        for (int j = 0; j < TL::NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                mine[(8 * (r / 4) + 4 * (lane >> 5) + r % 4) * W + ((j * 32) ^ (lane & 32)) + (lane & 31)] = acc[i][j][r];
        wave_sync_lds();
#pragma unroll 4
        for (int p = 0; p < 32; p += PASS) {
            const int in = p + lane / LANES, m = (wm * TL::MI + i) * 32 + in;
            auto four = [&](int c) { return *(const lds_f32x4*)(mine + in * W + (c ^ ((in & 4) << 3))); };
            if constexpr (MODE == IN) {
                // columns 64 q + 0..31: gate of f 32 q + 0..31, the next 32: u
                const int f = nf + wn * (W / 2) + c4, c = (c4 & ~31) * 2 + (c4 & 31);
                const f32x4 g = four(c), u = four(c + 32);
                if (m < count && f < P.Fp) {
                    float h[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) h[q] = f + q < P.F ? g[q] * gate_sigmoid<T>(g[q]) * u[q] : 0.0f;
                    store4((T*)P.h + (size_t)(p0 + m) * (size_t)P.Fp + f, h);
                    if (P.pre && f < P.Fi) {
                        float* pre = P.pre + (size_t)(p0 + m) * 2 * (size_t)P.Fi + f;
                        *(f32x4*)pre = g;
                        *(f32x4*)(pre + P.Fi) = u;
                    }
                }
            } else if constexpr (MODE == OUT || MODE == DX) {
                const int d = nf + wn * W + c4;
                f32x4 v = four(c4);
                if (m < count && d < P.D) {
                    const int slot = s_slot[m];
                    if constexpr (MODE == OUT) v *= s_w[m];
                    if (P.k > 1) *(f32x4*)(P.z + (size_t)slot * (size_t)P.Dp + d) = v;
                    else store_part((T*)P.out + (size_t)slot * (size_t)P.ldo + d, v, P.D - d);
                }
            } else if constexpr (MODE == DH) {
                const int f = nf + wn * W + c4;
                const f32x4 a = four(c4);
                float dot = 0.0f;
                if (m < count && f < P.Fp) {
                    const float w = s_w[m];
                    f32x4 g = {0.0f, 0.0f, 0.0f, 0.0f}, u = g;
                    if (f < P.Fi) {
                        const float* pre = P.pre + (size_t)(p0 + m) * 2 * (size_t)P.Fi + f;
                        g = *(const f32x4*)pre;
                        u = *(const f32x4*)(pre + P.Fi);
                    }
                    float dg[4], du[4], hw[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const bool is = f + q < P.F;
                        const float s = gate_sigmoid<T>(g[q]), h = g[q] * s * u[q], dh = w * a[q];
                        dot += is ? a[q] * h : 0.0f;
                        dg[q] = is ? dh * u[q] * s * (1.0f + g[q] * (1.0f - s)) : 0.0f;
                        du[q] = is ? dh * g[q] * s : 0.0f;
                        hw[q] = is ? w * h : 0.0f;
                    }
                    T* dpre = (T*)P.dpre + (size_t)(p0 + m) * 2 * (size_t)P.Fp + f;
                    store4(dpre, dg);
                    store4(dpre + P.Fp, du);
                    store4((T*)P.hw + (size_t)(p0 + m) * (size_t)P.Fp + f, hw);
                }
                dot = lanes_sum<LANES>(dot);
                if (m < count && lane % LANES == 0)
                    P.dwp[(size_t)(nf / TL::BN * TL::WN + wn) * (size_t)(P.n * P.k) + s_slot[m]] = dot;
            } else {
                int row = mf + m;
                const int M = MODE == DWIN ? 2 * P.F : P.D, N = MODE == DWIN ? P.D : P.F, c = nf + wn * W + c4;
                if constexpr (MODE == DWIN) row = row < P.F ? row : row < P.Fp ? M : row + P.F - P.Fp;
                const f32x4 v = four(c4);
                if (row < M && c < N) {
                    const size_t at = ((size_t)e * M + row) * (size_t)N + c;
                    if (splits == 1) store_part((T*)(MODE == DWIN ? P.dw_in : P.dw_out) + at, v, N - c);
                    else store_part((MODE == DWIN ? P.part_in : P.part_out) + (size_t)split * P.E * M * N + at, v, N - c);
                }
            }
        }
    }
}

// k = 1: the rows that have no expert, to which no tile writes, become zero; a
// wave writes those among its 64 rows one after the other.
template <typename T, int NT>
__device__ __forceinline__ void zero_rows(const ExpertArgs& P) {
    for (int64_t t0 = (int64_t)blockIdx.x * NT; t0 < P.n; t0 += (int64_t)gridDim.x * NT) {
        const int64_t t = t0 + threadIdx.x;
        const int e = t < P.n ? P.ids[t] : 0;
        uint64_t left = __ballot(e < 0 || e >= P.E);
        while (left) {
            const int l = __ffsll((unsigned long long)left) - 1;
            left &= left - 1;
            T* const row = (T*)P.out + (size_t)(t0 + (threadIdx.x & ~63) + l) * (size_t)P.ldo;
            for (int d = threadIdx.x & 63; d < P.D; d += 64) row[d] = (T)0.0f;
        }
    }
}

template <typename T, int MODE, typename TL, bool DMA>
__global__ void __launch_bounds__(TL::NT) k_experts(ExpertArgs P, int ntiles) {
    // y of one slot a row is made here whole, without a launch of k_finish
    if constexpr (MODE == OUT)
        if (P.k == 1) zero_rows<T, TL::NT>(P);
    expert_tile<T, MODE, TL, DMA>(P, blockIdx.x, ntiles, 0);
}

// DX, DWIN and DWOUT need nothing of each other: one grid, so that one's last
// tiles run beside the next one's first.
struct GradGrid {
    int nt[3], mt[3];
    uint32_t first[2];                // DWIN's and DWOUT's first blocks, multiples of XCDS
};
template <typename T, typename TL, bool DMA>
__global__ void __launch_bounds__(TL::NT) k_expert_grads(ExpertArgs P, GradGrid G) {
    if (blockIdx.x < G.first[0]) expert_tile<T, DX, TL, DMA>(P, blockIdx.x, G.nt[0], 0);
    else if (blockIdx.x < G.first[1]) expert_tile<T, DWIN, TL, DMA>(P, blockIdx.x - G.first[0], G.nt[1], G.mt[1]);
    else expert_tile<T, DWOUT, TL, DMA>(P, blockIdx.x - G.first[1], G.nt[2], G.mt[2]);
}

// ---------------------------------------------------------------------------
// Few rows: the products are bound by the weights' bytes, each read once, and
// by the launches.  Weights and slots go straight from memory into the matrix
// instructions' operands: a lane fetches 32 bytes in a row of one weight row,
// two instructions' worth, 16 weight rows and 16 slots a wave.  Widths and
// addresses are free.
//   k_inner_few   h: a block has 16 gate rows and their 16 rows of u of one
//                 expert; its waves share the summed dimension, 128 bytes a row
//                 in turn, and their sums meet in LDS
//   k_answer_few  y: a block has 16 columns of all rows; its waves share the
//                 experts in use, and the weighted answers of a row's slots
//                 are added up in LDS
// One row, 6 of 64 experts, 1024 -> 512 -> 1024, bf16: 6.8 and 7.6 us, mostly launch and
// three dependent loads before the weights' first (19 MB); h of 48 rows, 2048 -> 1024,
// all of 32 experts: 62 us for 268 MB, 4.3 TB/s.
// ---------------------------------------------------------------------------

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

// The j-th of the experts that have slots, or -1.
__device__ __forceinline__ int expert_in_use(const int32_t* off, int E, int j) {
    const int lane = threadIdx.x & 63;
    for (int e0 = 0; e0 < E; e0 += 64) {
        const int e = e0 + lane;
        const bool has = e < E && off[e + 1] > off[e];
        const uint64_t all = __ballot(has);
        const int before = __popcll(all & ((1ull << lane) - 1ull));
        const uint64_t hit = __ballot(has && before == j);
        if (hit) return e0 + __ffsll((unsigned long long)hit) - 1;
        j -= __popcll(all);
    }
    return -1;
}

constexpr int FEW_NT = 256, FEW_W = FEW_NT / 64;
constexpr int FEW_AHEAD = 4;                     // 128-byte pieces of a row under way in a wave
constexpr int FEW_SLOTS = 128;                   // slots whose answers a block keeps in LDS

// acc[m] += M matrices' 16 rows w[m] times the 16 slots' x, from piece `from` on, every `by`-th.
template <typename T, int M>
__device__ __forceinline__ void few_products(const T* const (&w)[M], const T* x, int K, int from, int by, f32x4 (&acc)[M]) {
    constexpr int CH = VEC<T>, STEP = 8 * CH;    // values in 128 bytes
    const int q = (threadIdx.x & 63) >> 4;
    for (int k0 = from * STEP; k0 < K; k0 += by * FEW_AHEAD * STEP) {
        u32x4 a[FEW_AHEAD][M][2], v[FEW_AHEAD][2];
#pragma unroll
        for (int s = 0; s < FEW_AHEAD; ++s)
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                const int k = k0 + s * by * STEP + (2 * q + o) * CH;
#pragma unroll
                for (int m = 0; m < M; ++m) a[s][m][o] = row_piece<T>(w[m], k, K);
                v[s][o] = row_piece<T>(x, k, K);
            }
#pragma unroll
        for (int s = 0; s < FEW_AHEAD; ++s)
#pragma unroll
            for (int o = 0; o < 2; ++o)
#pragma unroll
                for (int m = 0; m < M; ++m) acc[m] = mma16<T>(a[s][m][o], v[s][o], acc[m]);
    }
}

template <typename T>
__global__ void __launch_bounds__(FEW_NT) k_inner_few(ExpertArgs P) {
    __shared__ f32x4 s_sum[FEW_W][2][64];
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int e = expert_in_use(P.offsets, P.E, blockIdx.y);
    if (e < 0) return;
    const int off = P.offsets[e], cnt = P.offsets[e + 1] - off, first = blockIdx.x * 16;
    const T* const gate = (const T*)P.w_in + ((size_t)e * 2 * P.F + min(first + r, P.F - 1)) * (size_t)P.D;
    const T* const w[2] = {gate, gate + (size_t)P.F * (size_t)P.D};
    for (int p0 = 0; p0 < cnt; p0 += 16) {
        const T* x = (const T*)P.x + (size_t)P.rows[off + min(p0 + r, cnt - 1)] * (size_t)P.ldx;
        f32x4 acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
        few_products<T, 2>(w, x, P.D, wave, FEW_W, acc);
        __syncthreads();                         // the sums of the slots before have been read
        s_sum[wave][0][lane] = acc[0];
        s_sum[wave][1][lane] = acc[1];
        __syncthreads();
        // a lane has slot r and f = first + 4 q .. + 3
        const int at = p0 + r, f = first + 4 * q;
        if (wave == 0 && at < cnt) {
            f32x4 g = s_sum[0][0][lane], u = s_sum[0][1][lane];
#pragma unroll
            for (int o = 1; o < FEW_W; ++o) {
                g += s_sum[o][0][lane];
                u += s_sum[o][1][lane];
            }
            const size_t p = (size_t)(off + at);
            if (f < P.Fp) {
                float h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = f + i < P.F ? g[i] * gate_sigmoid<T>(g[i]) * u[i] : 0.0f;
                store4((T*)P.h + p * (size_t)P.Fp + f, h);
            }
            if (P.pre && f < P.Fi) {
                float* pre = P.pre + p * 2 * (size_t)P.Fi + f;
                *(f32x4*)pre = g;
                *(f32x4*)(pre + P.Fi) = u;
            }
        }
    }
}

constexpr int ANSWER_NT = 512;

template <typename T>
__global__ void __launch_bounds__(ANSWER_NT) k_answer_few(ExpertArgs P, T* __restrict__ y, int64_t ldy) {
    __shared__ f32x4 s_z[FEW_SLOTS][4];          // the slots' weighted answers in the block's 16 columns
    __shared__ int s_use[FEW_SLOTS];             // the experts in use: no more than slots
    __shared__ int s_count;
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int first = blockIdx.x * 16;
    if (wave == 0) {
        int count = 0;
        for (int e0 = 0; e0 < P.E; e0 += 64) {
            const int e = e0 + lane;
            const bool has = e < P.E && P.offsets[e + 1] > P.offsets[e];
            const uint64_t all = __ballot(has);
            if (has) s_use[count + __popcll(all & ((1ull << lane) - 1ull))] = e;
            count += __popcll(all);
        }
        if (lane == 0) s_count = count;
    }
    __syncthreads();
    for (int i = wave; i < s_count; i += ANSWER_NT / 64) {
        const int e = s_use[i], off = P.offsets[e], cnt = P.offsets[e + 1] - off;
        const T* const w[1] = {(const T*)P.w_out + ((size_t)e * P.D + min(first + r, P.D - 1)) * (size_t)P.F};
        for (int p0 = 0; p0 < cnt; p0 += 16) {
            const int p = off + min(p0 + r, cnt - 1);
            f32x4 acc[1] = {{0.0f, 0.0f, 0.0f, 0.0f}};
            few_products<T, 1>(w, (const T*)P.h + (size_t)p * (size_t)P.Fp, P.F, 0, 1, acc);
            if (p0 + r < cnt) {
                const int slot = P.slots[p];
                s_z[slot][q] = acc[0] * P.weights[slot];
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < (int)P.n * 16; i += ANSWER_NT) {
        const int t = i >> 4, c = i & 15;
        float s = 0.0f;
        for (int j = 0; j < P.k; ++j) {
            const int e = P.ids[t * P.k + j];
            if (e >= 0 && e < P.E) s += ((const float*)s_z[t * P.k + j])[c];
        }
        if (first + c < P.D) y[(size_t)t * (size_t)ldy + first + c] = (T)s;
    }
}

// The parts of a weight's gradient added in order, four values a thread.
template <typename T>
__device__ __forceinline__ void add_parts(const float* part, int64_t count, int splits, T* out) {
    typedef f32x4 f32x4_any __attribute__((aligned(4)));
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < count; i += (int64_t)gridDim.x * 1024) {
        const int have = (int)min(count - i, (int64_t)4);
        f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
        if (have == 4) {
#pragma unroll 8
            for (int p = 0; p < splits; ++p) s += *(const f32x4_any*)(part + (size_t)p * (size_t)count + i);
        } else {
            for (int p = 0; p < splits; ++p)
#pragma unroll
                for (int q = 0; q < 3; ++q)
                    if (q < have) s[q] += part[(size_t)p * (size_t)count + i + q];
        }
        store_part(out + i, s, have);
    }
}

// What is left once the tiles are made: out[t] = sum_j z[t k + j] over row t's
// slots that have an expert (k = 1, dx alone: zeros for rows without one, the others
// are there), and in the backward pass dw = the sum of its parts and the weights'
// gradients of theirs.  z in fp32 because y is a sum; 16 384 x 2048, k = 2: 67 us,
// 5.0 TB/s, a copy's rate.
template <typename T>
__global__ void __launch_bounds__(256) k_finish(ExpertArgs P) {
    T* const out = (T*)P.out;
    if (P.k > 1) {
        const int per = P.Dp / 4;
        const int64_t work = P.n * per;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < work; i += (int64_t)gridDim.x * 256) {
            const int64_t t = i / per;
            const int d = (int)(i - t * per) * 4;
            f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int j = 0; j < P.k; ++j) {
                const int e = P.ids[t * P.k + j];
                if (e >= 0 && e < P.E) s += *(const f32x4*)(P.z + (size_t)(t * P.k + j) * (size_t)P.Dp + d);
            }
            store_part(out + (size_t)t * (size_t)P.ldo + d, s, P.D - d);
        }
    } else {
        zero_rows<T, 256>(P);
    }
    if (!P.dweights) return;
    const int64_t S = P.n * P.k;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < S; i += (int64_t)gridDim.x * 256) {
        const int e = P.ids[i];
        float s = 0.0f;
        if (e >= 0 && e < P.E)
            for (int p = 0; p < P.parts; ++p) s += P.dwp[(size_t)p * (size_t)S + i];
        P.dweights[i] = s;
    }
    const int64_t count = (int64_t)P.E * P.F * P.D;
    if (P.splits_in > 1) add_parts(P.part_in, 2 * count, P.splits_in, (T*)P.dw_in);
    if (P.splits_out > 1) add_parts(P.part_out, count, P.splits_out, (T*)P.dw_out);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

using TileSmall = TileOf<64, 128, 2, 2, 128, 2, 2>;
using TileLarge = TileOf<256, 256, 4, 2, 128, 3, 2>;

constexpr int PART_BLOCKS = 512;      // blocks of weight gradients that keep the device busy

inline int up16(int v, int bytes) { return (v * bytes + 15) / 16 * 16 / bytes; }
inline int64_t over(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct ExpertSizes {
    int64_t S, used;                  // slots, and the experts that can have some
    int D, F, E, bytes, Fp, Dp;
    bool large[4];                    // tiles of h, of y, of the inner gradient, of the three others
    int splits_in, splits_out, parts;
};

// Whether 256 x 256 tiles make the product of M x K by K x N of `count` experts
// faster than 64 x 128: they fetch a third of the bytes, but there have to be
// enough of them, and a block of theirs has its CU to itself, so that nothing
// covers its beginning and end unless K is long.  Large and small, bf16, us: h of
// 8000 slots, 250 an expert, 2048 -> 1024: 151 and 165, of 32 768, 256 -> 256 of 8:
// 38 and 33; dx of 8000, 1024, 16 experts: 64 and 76; dw_in of the same 84 and 107,
// of 4000, 256 x 256, 8 experts 38 and 19.  fp32 is bound by its arithmetic, of which
// small tiles waste less at the edges (6000 x 500 -> 512 of 8: 949 and 625 for all six).
inline bool large_product(int bytes, int64_t count, int64_t M, int64_t N, int64_t K) {
    return bytes == 2 && K >= 384 && M >= 192 && N >= 192 && count * over(M, 256) * over(N, 256) >= 128;
}

// Parts of the summed slots, so that an expert's few tiles fill the device: at
// least four steps each for an average expert.  With 2, 4, 8 and 16 steps, the parts'
// sum included, us: 20 000 x 100 -> 60 of 7, fp32 49, 50, 53 and 78; 3000 x 200 -> 200 of
// 2, fp16 21, 20, 23 and 33.
inline int weight_splits(int64_t S, int E, int M, int N, int bm, int bn, int bk) {
    const int64_t tiles = (int64_t)E * over(M, bm) * over(N, bn);
    int64_t s = PART_BLOCKS / tiles;
    const int64_t longest = S / E / (4 * bk);
    if (s > longest) s = longest;
    if (s > 64) s = 64;
    return s < 1 ? 1 : (int)s;
}

inline ExpertSizes expert_sizes(int dtype, int64_t n, int k, int D, int F, int E) {
    ExpertSizes z;
    const int b = dtype_bytes(dtype);
    z.S = n * k;
    z.used = z.S < E ? z.S : E;
    z.D = D, z.F = F, z.E = E, z.bytes = b;
    z.Fp = up16(F, b);
    z.Dp = up16(D, 4);
    const int64_t each = z.used ? over(z.S, z.used) : 0;
    z.large[0] = large_product(b, z.used, each, 2 * (int64_t)F, D);
    z.large[1] = large_product(b, z.used, each, D, F);
    z.large[2] = large_product(b, z.used, each, F, D);
    z.large[3] = large_product(b, z.used, each, D, 2 * (int64_t)F) && large_product(b, E, 2 * (int64_t)F, D, z.S / E);
    const int bm = z.large[3] ? 256 : 64, bn = z.large[3] ? 256 : 128;
    z.splits_in = weight_splits(z.S, E, z.Fp + F, D, bm, bn, 128 / b);
    z.splits_out = weight_splits(z.S, E, D, F, bm, bn, 128 / b);
    z.parts = (int)(z.large[2] ? over(F, TileLarge::BN) * TileLarge::WN : over(F, TileSmall::BN) * TileSmall::WN);
    return z;
}

inline size_t carve_forward(Carve& c, ExpertArgs* P, const ExpertSizes& z, int k) {
    P->h = c.take<char>((size_t)z.S * z.Fp * z.bytes);
    P->z = k > 1 ? c.take<float>((size_t)z.S * z.Dp) : nullptr;
    return c.off;
}

inline size_t carve_backward(Carve& c, ExpertArgs* P, const ExpertSizes& z, int k) {
    P->dpre = c.take<char>((size_t)z.S * 2 * z.Fp * z.bytes);
    P->hw = c.take<char>((size_t)z.S * z.Fp * z.bytes);
    P->dwp = c.take<float>((size_t)z.parts * z.S);
    P->z = k > 1 ? c.take<float>((size_t)z.S * z.Dp) : nullptr;
    const size_t count = (size_t)z.E * z.F * (size_t)z.D;
    P->part_in = z.splits_in > 1 ? c.take<float>(z.splits_in * 2 * count) : nullptr;
    P->part_out = z.splits_out > 1 ? c.take<float>(z.splits_out * count) : nullptr;
    P->splits_in = z.splits_in;
    P->splits_out = z.splits_out;
    P->parts = z.parts;
    return c.off;
}

template <typename TL, int MODE>
int64_t tile_blocks(const ExpertSizes& z, int* nt, int* mt) {
    const int N = MODE == OUT || MODE == DX || MODE == DWIN ? z.D : z.F, cols = MODE == IN ? TL::BN / 2 : TL::BN;
    const int M = MODE == DWIN ? z.Fp + z.F : z.D;
    *nt = (int)over(N, cols);
    *mt = (int)over(M, TL::BM);
    if (MODE < DWIN) return over((z.S / TL::BM + z.used) * *nt, XCDS) * XCDS;      // no plan has more tiles
    return z.E * (over((int64_t)*mt * *nt * (MODE == DWIN ? z.splits_in : z.splits_out), XCDS) * XCDS);
}

// fp32 has no large tiles (large_product).
template <typename T, typename F>
void by_tile(bool large, bool dma, const F& f) {
    if constexpr (sizeof(T) == 2) {
        if (large) return dma ? f(TileLarge(), std::true_type()) : f(TileLarge(), std::false_type());
    }
    dma ? f(TileSmall(), std::true_type()) : f(TileSmall(), std::false_type());
}

template <typename T, int MODE>
void run_tiles(const ExpertArgs& P, const ExpertSizes& z, bool large, bool dma, hipStream_t stream) {
    by_tile<T>(large, dma, [&](auto tl, auto d) {
        using TL = decltype(tl);
        int nt, mt;
        const int64_t blocks = tile_blocks<TL, MODE>(z, &nt, &mt);
        if (blocks)
            k_experts<T, MODE, TL, decltype(d)::value><<<(unsigned)blocks, TL::NT, TL::LDS, stream>>>(P, nt);
    });
}

template <typename T>
void run_grads(const ExpertArgs& P, const ExpertSizes& z, bool dma, hipStream_t stream) {
    by_tile<T>(z.large[3], dma, [&](auto tl, auto d) {
        using TL = decltype(tl);
        GradGrid G;
        const int64_t dx = tile_blocks<TL, DX>(z, &G.nt[0], &G.mt[0]);
        const int64_t in = tile_blocks<TL, DWIN>(z, &G.nt[1], &G.mt[1]);
        const int64_t out = tile_blocks<TL, DWOUT>(z, &G.nt[2], &G.mt[2]);
        G.first[0] = (uint32_t)dx;
        G.first[1] = (uint32_t)(dx + in);
        k_expert_grads<T, TL, decltype(d)::value>
            <<<(unsigned)(dx + in + out), TL::NT, TL::LDS, stream>>>(P, G);
    });
}

template <typename T>
void run_finish(const ExpertArgs& P, const ExpertSizes& z, hipStream_t stream) {
    int64_t work = P.k > 1 ? P.n * (z.Dp / 4) : P.n;
    if (P.dweights && (z.splits_in > 1 || z.splits_out > 1)) work += (int64_t)z.E * z.F * z.D / 4;
    k_finish<T><<<launch_grid(work, 256, 8192), 256, 0, stream>>>(P);
}

// The kernels for few rows by the slots an expert in use has on average.  They
// pass over the weights once per 16 slots, the tiles once per 64 with a tile's
// whole arithmetic, which fp32 does at a sixteenth of the rate.  h, few and
// tiles, us: 2048 -> 1024 of 32 experts, fp16, 6 slots each 61 and 66, 12 each 79
// and 70; 1024 -> 512 of 64, bf16, one row's 6 slots 6 and 10, 3 each 20 and 19,
// 6 each 24 and 21; of 8, fp32, 4 each 15 and 40, 32 each 22 and 42; 500 -> 101 of
// 4, fp32, 25 each 10 and 29, 50 each 17 and 29 (fp32 with as many for every expert).
inline bool few_inner(int64_t S, int E, int bytes) {
    const int64_t used = S < E ? S : E;
    return S <= used * (bytes == 4 ? 32 : 8);
}
// y, few and tiles with k_finish, us: bf16, one row's 6 slots 6.8 and 11.4, two rows'
// 12 slots 11.3 and 12.1, 8 rows' 48 slots of about 33 experts, so that a wave
// has several in turn, 26 and 15; fp32 of 8 experts 32 slots 15 and 27, 128 slots
// 26 and 27, 256 slots 44 and 27.
inline bool few_answer(int64_t S, int E, int bytes) {
    return few_inner(S, E, bytes) && S <= FEW_SLOTS && (S < E ? S : E) <= 16;
}

template <typename T>
int run_experts(const ExpertArgs& P, const ExpertSizes& z, bool dma, hipStream_t stream) {
    if (few_inner(z.S, P.E, sizeof(T)))
        k_inner_few<T><<<dim3((unsigned)over(P.F, 16), (unsigned)z.used), FEW_NT, 0, stream>>>(P);
    else
        run_tiles<T, IN>(P, z, z.large[0], dma, stream);
    if (few_answer(z.S, P.E, sizeof(T))) {
        k_answer_few<T><<<(unsigned)over(P.D, 16), ANSWER_NT, 0, stream>>>(P, (T*)P.out, P.ldo);
    } else {
        run_tiles<T, OUT>(P, z, z.large[1], dma, stream);
        if (P.k > 1) run_finish<T>(P, z, stream);
    }
    return launch_status("yabt_experts");
}

template <typename T>
int run_experts_grad(const ExpertArgs& P, const ExpertSizes& z, bool dma, hipStream_t stream) {
    run_tiles<T, DH>(P, z, z.large[2], dma, stream);
    run_grads<T>(P, z, dma, stream);
    run_finish<T>(P, z, stream);
    return launch_status("yabt_experts_grad");
}

inline bool expert_ranges_ok(int64_t n, int k, int D, int F, int E) {
    return n >= 0 && k >= 1 && D >= 1 && F >= 1 && E >= 1 && E <= 1024 && n <= INT32_MAX / k && D <= (1 << 24) &&
           F <= (1 << 24);
}

template <typename F>
auto by_dtype(int dtype, const F& f) {
    if (dtype == DT_F32) return f((float*)nullptr);
    if (dtype == DT_BF16) return f((bf16*)nullptr);
    return f((f16*)nullptr);
}

// A launch has fewer than 2^32 threads.
template <typename T>
bool forward_grids_ok(const ExpertSizes& z) {
    bool ok = true;
    auto tiles = [&](auto mode, bool large) {
        by_tile<T>(large, true, [&](auto tl, auto) {
            using TL = decltype(tl);
            int nt, mt;
            ok = ok && tile_blocks<TL, decltype(mode)::value>(z, &nt, &mt) <= UINT32_MAX / TL::NT;
        });
    };
    if (!few_inner(z.S, z.E, sizeof(T))) tiles(std::integral_constant<int, IN>(), z.large[0]);
    if (!few_answer(z.S, z.E, sizeof(T))) tiles(std::integral_constant<int, OUT>(), z.large[1]);
    return ok;
}
template <typename T>
bool backward_grids_ok(const ExpertSizes& z) {
    bool ok = true;
    int nt, mt;
    by_tile<T>(z.large[2], true, [&](auto tl, auto) {
        using TL = decltype(tl);
        ok = tile_blocks<TL, DH>(z, &nt, &mt) <= UINT32_MAX / TL::NT;
    });
    by_tile<T>(z.large[3], true, [&](auto tl, auto) {
        using TL = decltype(tl);
        ok = ok && tile_blocks<TL, DX>(z, &nt, &mt) + tile_blocks<TL, DWIN>(z, &nt, &mt) +
                           tile_blocks<TL, DWOUT>(z, &nt, &mt) <= UINT32_MAX / TL::NT;
    });
    return ok;
}

// Whether the sizes can be run, and what they lead to.
inline bool expert_sizes_ok(bool backward, int dtype, int64_t n, int k, int D, int F, int E, ExpertSizes* z) {
    if (!dtype_ok(dtype) || !expert_ranges_ok(n, k, D, F, E)) return false;
    *z = expert_sizes(dtype, n, k, D, F, E);
    return by_dtype(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return backward ? backward_grids_ok<T>(*z) : forward_grids_ok<T>(*z);
    });
}

// Whether rows of `width` values, ld apart, may be fetched in aligned 16-byte pieces.
inline bool pieces_ok(const void* p, int64_t ld, int width, int bytes) {
    return aligned16(p) && ld * bytes % 16 == 0 && (int64_t)width * bytes % 16 == 0;
}

}  // namespace yabt

using namespace yabt;

extern "C" {

size_t yabt_experts_workspace_bytes(int dtype, int64_t n, int k, int D, int F, int E) {
    ExpertSizes z;
    if (!expert_sizes_ok(false, dtype, n, k, D, F, E, &z)) return 0;
    ExpertArgs P;
    Carve c{nullptr, 0};
    return carve_forward(c, &P, z, k) + 256;
}

int yabt_experts(int dtype, const void* x, int64_t ldx, int64_t n, int k, int D, int F, int E, const int32_t* ids,
                 const int32_t* offsets, const int32_t* slots, const int32_t* rows, const float* weights,
                 const void* w_in, const void* w_out, void* workspace, size_t workspace_bytes, float* out_inner,
                 void* y, int64_t ldy, yabt_stream_t stream) {
    if (!dtype_ok(dtype)) return fail(-1, "yabt_experts: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    ExpertSizes z;
    if (!expert_sizes_ok(false, dtype, n, k, D, F, E, &z) || ldx < D || ldy < D)
        return fail(-1, "yabt_experts: bad sizes");
    if (n == 0) return 0;
    if (!x || !ids || !offsets || !slots || !rows || !weights || !w_in || !w_out || !y)
        return fail(-1, "yabt_experts: null pointer");
    if (!aligned16(out_inner)) return fail(-1, "yabt_experts: out_inner must be 16-byte aligned");
    if (!workspace || workspace_bytes < yabt_experts_workspace_bytes(dtype, n, k, D, F, E))
        return fail(-2, "yabt_experts: workspace too small");
    ExpertArgs P = {x, nullptr, w_in, w_out, weights, ids, offsets, slots, rows, ldx, 0, n, k, D, F, E, z.Fp, z.Dp, up16(F, 4)};
    P.pre = out_inner;
    P.out = y;
    P.ldo = ldy;
    Carve c{(char*)align_up((size_t)workspace, 256), 0};
    carve_forward(c, &P, z, k);
    const int b = dtype_bytes(dtype);
    const bool dma = pieces_ok(x, ldx, D, b) && pieces_ok(w_in, D, D, b) && pieces_ok(w_out, F, F, b);
    return by_dtype(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return run_experts<T>(P, z, dma, (hipStream_t)stream);
    });
}

int yabt_experts_forms(int dtype, int64_t n, int k, int D, int F, int E) {
    if (!dtype_ok(dtype) || !expert_ranges_ok(n, k, D, F, E)) return -1;
    const ExpertSizes z = expert_sizes(dtype, n, k, D, F, E);
    const bool inner = few_inner(z.S, E, z.bytes), answer = few_answer(z.S, E, z.bytes);
    int forms = (int)inner | (int)answer << 1 | (int)(z.large[0] && !inner) << 2 | (int)(z.large[1] && !answer) << 3;
    return forms | (int)z.large[2] << 4 | (int)z.large[3] << 5;
}

size_t yabt_experts_grad_workspace_bytes(int dtype, int64_t n, int k, int D, int F, int E) {
    ExpertSizes z;
    if (!expert_sizes_ok(true, dtype, n, k, D, F, E, &z)) return 0;
    ExpertArgs P;
    Carve c{nullptr, 0};
    return carve_backward(c, &P, z, k) + 256;
}

int yabt_experts_grad(int dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t n, int k, int D,
                      int F, int E, const int32_t* ids, const int32_t* offsets, const int32_t* slots,
                      const int32_t* rows, const float* weights, const void* w_in, const void* w_out,
                      const float* inner, void* workspace, size_t workspace_bytes, void* dx, int64_t lddx,
                      float* dweights, void* dw_in, void* dw_out, yabt_stream_t stream) {
    if (!dtype_ok(dtype)) return fail(-1, "yabt_experts_grad: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    ExpertSizes z;
    if (!expert_sizes_ok(true, dtype, n, k, D, F, E, &z) || ldx < D || lddy < D || lddx < D)
        return fail(-1, "yabt_experts_grad: bad sizes");
    if (!offsets || !w_in || !w_out || !dw_in || !dw_out ||
        (n > 0 && (!x || !dy || !ids || !slots || !rows || !weights || !inner || !dx || !dweights)))
        return fail(-1, "yabt_experts_grad: null pointer");
    if (!aligned16(inner)) return fail(-1, "yabt_experts_grad: inner must be 16-byte aligned");
    if (!workspace || workspace_bytes < yabt_experts_grad_workspace_bytes(dtype, n, k, D, F, E))
        return fail(-2, "yabt_experts_grad: workspace too small");
    ExpertArgs P = {x, dy, w_in, w_out, weights, ids, offsets, slots, rows, ldx, lddy, n, k, D, F, E, z.Fp, z.Dp, up16(F, 4)};
    P.pre = const_cast<float*>(inner);
    P.out = dx;
    P.ldo = lddx;
    P.dw_in = dw_in;
    P.dw_out = dw_out;
    P.dweights = dweights;
    Carve c{(char*)align_up((size_t)workspace, 256), 0};
    carve_backward(c, &P, z, k);
    const int b = dtype_bytes(dtype);
    const bool dma = pieces_ok(x, ldx, D, b) && pieces_ok(dy, lddy, D, b) && pieces_ok(w_in, D, D, b) &&
                     pieces_ok(w_out, F, F, b);
    return by_dtype(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return run_experts_grad<T>(P, z, dma, (hipStream_t)stream);
    });
}

}  // extern "C"
