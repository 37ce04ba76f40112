// Shared pieces of the expert layer's kernels: value types, 16-byte accesses,
// reductions over parts of a wave.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "host.h"

namespace yabt {

// Value types of the C ABI's `dtype` arguments.
constexpr int DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2;

using bf16 = __bf16;
using f16 = _Float16;

inline bool dtype_ok(int dt) { return dt >= DT_F32 && dt <= DT_F16; }
inline int dtype_bytes(int dt) { return dt == DT_F32 ? 4 : 2; }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at any address that is a multiple of the values' own size: rows of
// odd widths start anywhere, and this target's global loads need no alignment
typedef u32x4 u32x4_any __attribute__((aligned(2)));

template <typename T>
constexpr int VEC = 16 / (int)sizeof(T);

// VEC<T> (or, with N = 1, one) consecutive values as floats
template <typename T, int N = VEC<T>>
struct Chunk {
    static_assert(N == VEC<T> || N == 1, "16 bytes or one value");
    typedef T VT __attribute__((ext_vector_type(N)));
    union {
        u32x4 raw;
        VT v;
    };
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (N == 1) v[0] = p[0];
        else raw = *reinterpret_cast<const u32x4_any*>(p);
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (N == 1) p[0] = v[0];
        else *reinterpret_cast<u32x4_any*>(p) = raw;
    }
    __device__ __forceinline__ float get(int i) const { return (float)v[i]; }
    __device__ __forceinline__ void set(int i, float f) { v[i] = (T)f; }
};

// One value exchanged with the lane that differs in bit M of its number, or
// for M >= 4 within the rows of 16 lanes with the mirrored lane, whose run of
// M lanes is the other one: enough for reductions, where a run's lanes agree.
template <int M>
__device__ __forceinline__ uint32_t lanes_other(uint32_t v) {
    if constexpr (M == 1) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true);
    if constexpr (M == 2) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true);
    if constexpr (M == 4) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true);
    if constexpr (M == 8) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true);
    return (uint32_t)__shfl_xor((int)v, M);
}
template <int M>
__device__ __forceinline__ float lanes_other(float v) {
    return __uint_as_float(lanes_other<M>(__float_as_uint(v)));
}
template <int M>
__device__ __forceinline__ double lanes_other(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)lanes_other<M>((uint32_t)(u >> 32)) << 32 |
                                            lanes_other<M>((uint32_t)u)));
}

// Reduction over each aligned run of G lanes (G <= 64) by an operation whose
// operands may be swapped; every lane of the run gets the same bits.
template <int G, typename V, typename Op, int M = 1>
__device__ __forceinline__ V lanes_reduce(V v, const Op& op) {
    if constexpr (M < G) return lanes_reduce<G, V, Op, M * 2>(op(v, lanes_other<M>(v)), op);
    else return v;
}
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
    return lanes_reduce<(G < 64 ? G : 64)>(v, [](float a, float b) { return a + b; });
}
template <int G>
__device__ __forceinline__ float lanes_max(float v) {
    return lanes_reduce<G>(v, [](float a, float b) { return fmaxf(a, b); });
}

// p = 1 / (1 + exp(-x)) of N values, the quotient rounded correctly: the
// hardware's reciprocal (one unit off at most) and one Newton step give it for
// every divisor from 1 to 2^126 (all were tried), the compiler's division for
// what is larger, which is rare.
template <int N>
__device__ __forceinline__ void sigmoids(const float (&x)[N], float (&p)[N]) {
    float d[N], most = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        d[i] = 1.0f + expf(-x[i]);
        most = fmaxf(most, d[i]);
        const float r = __builtin_amdgcn_rcpf(d[i]);
        p[i] = fmaf(fmaf(-d[i], r, 1.0f), r, r);
    }
    if (most > 0x1p126f) {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = 1.0f / d[i];
    }
}

// Orders this wave's LDS accesses: what its lanes wrote before is read after.
__device__ __forceinline__ void wave_sync_lds() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

}  // namespace yabt
