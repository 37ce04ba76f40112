// One AdamW step over many tensors, moments in 32 bits or in 8.
//
//   m <- m + (1 - b1) (g - m),   v <- v + (1 - b2) (g^2 - v)
//   p <- p (1 - lr wd) - s m / (sqrt(v) + e),   s = lr sqrt(1 - b2^t) / (1 - b1^t),  e = eps sqrt(1 - b2^t)
//
// in fp32, every operation rounded by itself but the last product of each line,
// which is rounded with its sum: what torch's lerp_ and addcdiv_ compute.
//
// 8 bits: blocks of 256 consecutive values share a scale, the block's largest
// magnitude.  m is held as sign (c / 127)^2 of it, and sqrt(v) as (c / 255)^2 of
// its own largest: a square, because moments of one block span many powers of two, and
// equal steps would round most of them to 0.  A value that is not 0 keeps its leading
// digits down to 2^-13 (m) and 2^-16 (sqrt(v)) of the largest; the step to the next code
// is 2 / c of the value.  A v above 0 gets no code 0: m would be divided by eps alone.
// The update is made with the new moments before they are rounded.
//
// Bound by its bytes: 28 a value (26 with 16-bit gradients), 16 (14) with 8-bit
// moments: 40M fp32 values with bf16 gradients 196 us, 5.3 TB/s, a copy's rate; 120M with
// 8-bit moments 356 us, 4.7 TB/s (three square roots and a quotient a value beside the bytes),
// the values they stand for 215 us, 5.6 TB/s.  A wave takes blocks of 256 values, four a lane, so that a block's largest
// needs no LDS; a thread block takes 4096 of one tensor, which it finds by one ballot
// over the tensors' first blocks, passed by value: one launch for up to 48 tensors, and
// nothing to copy to the device first.

#include "expert.h"
#include "yabt_hip.h"

#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

namespace yabt {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int ADAMW_CAP = 48;                     // tensors of a launch: its arguments have 4 KB
constexpr int ADAMW_NT = 256;
constexpr int ADAMW_BLOCK = 256;                  // values that share a scale
constexpr int ADAMW_AHEAD = 4;                    // blocks of values a wave has under way
constexpr int ADAMW_CHUNK = ADAMW_BLOCK * ADAMW_AHEAD * (ADAMW_NT / 64);
constexpr float ADAMW_LEAST = 0x1p-100f;          // a block whose largest magnitude is below is held as zeros

struct AdamwEntry {
    void* param;                                  // values(): the first moments' values
    void* grad;                                   // values(): the second's
    void* first;
    void* second;
    float* first_scale;
    float* second_scale;
    int64_t n;
    int32_t param_dtype, grad_dtype;
};
struct AdamwTable {
    AdamwEntry t[ADAMW_CAP];
    uint32_t first_chunk[64];                     // of each tensor; behind the last the number of all
};
struct AdamwScalars {
    float w1, w2, decay, scale, eps;
    double lr, beta1, beta2, eps64;               // with the step's number on the device
    const int32_t* step;
};
static_assert(sizeof(AdamwTable) + sizeof(AdamwScalars) <= 4096, "a launch's arguments");

// Four consecutive values, of which `have` exist (all: FULL), as floats.
template <typename T, bool FULL>
__device__ __forceinline__ f32x4 load4(const void* base, int64_t at, int have) {
    typedef T VT __attribute__((ext_vector_type(4)));
    typedef VT VTany __attribute__((aligned(sizeof(T))));
    const T* p = (const T*)base + at;
    if constexpr (FULL) {
        const VT v = *(const VTany*)p;
        return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
    } else {
        f32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q < have) r[q] = (float)p[q];
        return r;
    }
}
template <typename T, bool FULL>
__device__ __forceinline__ void save4(void* base, int64_t at, int have, f32x4 v) {
    typedef T VT __attribute__((ext_vector_type(4)));
    typedef VT VTany __attribute__((aligned(sizeof(T))));
    T* p = (T*)base + at;
    if constexpr (FULL) {
        *(VTany*)p = VT{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q < have) p[q] = (T)v[q];
    }
}

// The values that a block's codes stand for.
__device__ __forceinline__ f32x4 first_values(f32x4 c, float scale) {
    const float unit = scale * (1.0f / 16129.0f);
    f32x4 m;
#pragma unroll
    for (int q = 0; q < 4; ++q) m[q] = c[q] * fabsf(c[q]) * unit;
    return m;
}
__device__ __forceinline__ f32x4 second_values(f32x4 c, float scale) {
    const float unit = scale * (1.0f / 65025.0f);
    f32x4 v;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float r = c[q] * c[q] * unit;
        v[q] = r * r;
    }
    return v;
}

// The largest of the wave's magnitudes, by their bits: an infinity or a NaN is
// larger than every number.
__device__ __forceinline__ float wave_most(f32x4 a) {
    uint32_t most = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t b = __float_as_uint(a[q]) & 0x7FFFFFFFu;
        most = most > b ? most : b;
    }
    return __uint_as_float(lanes_reduce<64>(most, [](uint32_t x, uint32_t y) { return x > y ? x : y; }));
}
// The scale that is kept for it and what the values are multiplied by; a block
// that is not finite is held as NaN.
__device__ __forceinline__ float block_scale(float most, float* unit) {
    const bool some = most >= ADAMW_LEAST, finite = most <= 3.402823466e38f;
    *unit = some && finite ? 1.0f / most : 0.0f;
    return !finite ? __uint_as_float(0x7FC00000u) : some ? most : 0.0f;
}
__device__ __forceinline__ float code_of(float steps, float part, bool finite) {
    return finite ? rintf(steps * sqrtf(part)) : 0.0f;
}

// m + w (g - m), from the nearer end as torch's lerp_ does
__device__ __forceinline__ float toward(float m, float g, float w) {
    return w < 0.5f ? fmaf(w, g - m, m) : fmaf(-(g - m), 1.0f - w, g);
}

template <typename P, typename G, int BITS, bool FULL>
__device__ __forceinline__ void adamw_groups(const AdamwEntry& T, const AdamwScalars& S, int64_t base, int64_t n) {
    const int lane = threadIdx.x & 63;
    f32x4 p[ADAMW_AHEAD], g[ADAMW_AHEAD], m[ADAMW_AHEAD], v[ADAMW_AHEAD];
    float sm[ADAMW_AHEAD], sv[ADAMW_AHEAD];
#pragma unroll
    for (int i = 0; i < ADAMW_AHEAD; ++i) {
        const int64_t at = base + i * ADAMW_BLOCK + lane * 4;
        const int have = FULL ? 4 : (int)max((int64_t)0, min((int64_t)4, n - at));
        p[i] = load4<P, FULL>(T.param, at, have);
        g[i] = load4<G, FULL>(T.grad, at, have);
        if constexpr (BITS == 32) {
            m[i] = load4<float, FULL>(T.first, at, have);
            v[i] = load4<float, FULL>(T.second, at, have);
        } else {
            const int64_t b = (base + i * ADAMW_BLOCK) / ADAMW_BLOCK;
            const bool is = FULL || base + i * ADAMW_BLOCK < n;
            m[i] = load4<int8_t, FULL>(T.first, at, have);
            v[i] = load4<uint8_t, FULL>(T.second, at, have);
            sm[i] = is ? T.first_scale[b] : 0.0f;
            sv[i] = is ? T.second_scale[b] : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < ADAMW_AHEAD; ++i) {
        const int64_t at = base + i * ADAMW_BLOCK + lane * 4;
        const int have = FULL ? 4 : (int)max((int64_t)0, min((int64_t)4, n - at));
        if constexpr (BITS == 8) {
            m[i] = first_values(m[i], sm[i]);
            v[i] = second_values(v[i], sv[i]);
        }
        f32x4 root;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            m[i][q] = toward(m[i][q], g[i][q], S.w1);
            v[i][q] = toward(v[i][q], g[i][q] * g[i][q], S.w2);
            root[q] = sqrtf(v[i][q]);
            p[i][q] = fmaf(-S.scale, m[i][q] / (root[q] + S.eps), p[i][q] * S.decay);
        }
        save4<P, FULL>(T.param, at, have, p[i]);
        if constexpr (BITS == 32) {
            save4<float, FULL>(T.first, at, have, m[i]);
            save4<float, FULL>(T.second, at, have, v[i]);
        } else {
            // values past the tensor's end are 0 here: zero moments and a zero gradient
            float um, uv;
            sm[i] = block_scale(wave_most(m[i]), &um);
            sv[i] = block_scale(wave_most(root), &uv);
            f32x4 cm, cv;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float c = code_of(127.0f, fabsf(m[i][q]) * um, sm[i] == sm[i]);
                cm[q] = m[i][q] < 0.0f ? -c : c;
                const float d = code_of(255.0f, root[q] * uv, sv[i] == sv[i]);
                cv[q] = root[q] > 0.0f && uv > 0.0f ? fmaxf(d, 1.0f) : d;
            }
            save4<int8_t, FULL>(T.first, at, have, cm);
            save4<uint8_t, FULL>(T.second, at, have, cv);
            if (lane == 0 && (FULL || base + i * ADAMW_BLOCK < n)) {
                const int64_t b = (base + i * ADAMW_BLOCK) / ADAMW_BLOCK;
                T.first_scale[b] = sm[i];
                T.second_scale[b] = sv[i];
            }
        }
    }
}

// b^t for t >= 1 by squaring
__device__ __forceinline__ double power(double b, uint32_t t) {
    double r = 1.0;
    for (; t; t >>= 1) {
        if (t & 1) r *= b;
        b *= b;
    }
    return r;
}

// Which tensor this thread block works on and where: its wave's first value.
__device__ __forceinline__ int adamw_place(const AdamwTable& A, int64_t* base) {
    const uint32_t mine = A.first_chunk[threadIdx.x & 63];
    const int i = __builtin_amdgcn_readfirstlane(__popcll(__ballot(mine <= blockIdx.x)) - 1);
    const uint32_t in = blockIdx.x - A.first_chunk[i];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    *base = (int64_t)in * ADAMW_CHUNK + wave * (ADAMW_AHEAD * ADAMW_BLOCK);
    return i;
}

template <int BITS>
__global__ void __launch_bounds__(ADAMW_NT) k_adamw(AdamwTable A, AdamwScalars S) {
    int64_t base;
    const AdamwEntry T = A.t[adamw_place(A, &base)];
    if (base >= T.n) return;
    if (S.step) {
        const int32_t t = *S.step;
        const uint32_t t1 = t < 1 ? 1u : (uint32_t)t;
        const double left = sqrt(1.0 - power(S.beta2, t1));
        S.scale = (float)(S.lr * left / (1.0 - power(S.beta1, t1)));
        S.eps = (float)(S.eps64 * left);
    }
    auto with = [&](auto* p, auto* g) {
        using P = std::remove_pointer_t<decltype(p)>;
        using G = std::remove_pointer_t<decltype(g)>;
        if (base + ADAMW_AHEAD * ADAMW_BLOCK <= T.n) adamw_groups<P, G, BITS, true>(T, S, base, T.n);
        else adamw_groups<P, G, BITS, false>(T, S, base, T.n);
    };
    auto grads = [&](auto* p) {
        if (T.grad_dtype == DT_F32) with(p, (float*)nullptr);
        else if (T.grad_dtype == DT_BF16) with(p, (bf16*)nullptr);
        else with(p, (f16*)nullptr);
    };
    if (T.param_dtype == DT_F32) grads((float*)nullptr);
    else if (T.param_dtype == DT_BF16) grads((bf16*)nullptr);
    else grads((f16*)nullptr);
}

template <bool FULL>
__device__ __forceinline__ void adamw_show(const AdamwEntry& T, int64_t base) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < ADAMW_AHEAD; ++i) {
        const int64_t start = base + i * ADAMW_BLOCK, at = start + lane * 4;
        if (!FULL && start >= T.n) return;
        const int have = FULL ? 4 : (int)max((int64_t)0, min((int64_t)4, T.n - at));
        const f32x4 m = load4<int8_t, FULL>(T.first, at, have), v = load4<uint8_t, FULL>(T.second, at, have);
        save4<float, FULL>(T.param, at, have, first_values(m, T.first_scale[start / ADAMW_BLOCK]));
        save4<float, FULL>(T.grad, at, have, second_values(v, T.second_scale[start / ADAMW_BLOCK]));
    }
}

__global__ void __launch_bounds__(ADAMW_NT) k_adamw_values(AdamwTable A) {
    int64_t base;
    const AdamwEntry T = A.t[adamw_place(A, &base)];
    if (base >= T.n) return;
    if (base + ADAMW_AHEAD * ADAMW_BLOCK <= T.n) adamw_show<true>(T, base);
    else adamw_show<false>(T, base);
}

// Calls launch(table, blocks) for up to ADAMW_CAP tensors and 2^24 - 1 blocks at a time; the launches' status.
template <typename Entry, typename Launch>
int adamw_launches(const char* what, int count, const Entry& entry, const Launch& launch) {
    constexpr int64_t MOST = (1 << 24) - 1;        // a launch has fewer than 2^32 threads
    AdamwTable A = {};
    int held = 0, launches = 0;
    int64_t blocks = 0;
    auto flush = [&] {
        for (int i = held; i < 64; ++i) A.first_chunk[i] = (uint32_t)blocks;
        if (blocks) {
            launch(A, (unsigned)blocks);
            ++launches;
        }
        held = 0;
        blocks = 0;
    };
    for (int i = 0; i < count; ++i) {
        const AdamwEntry e = entry(i);
        const int64_t need = (e.n + ADAMW_CHUNK - 1) / ADAMW_CHUNK;
        if (need == 0) continue;
        if (held == ADAMW_CAP || blocks + need > MOST) flush();
        A.t[held] = e;
        A.first_chunk[held++] = (uint32_t)blocks;
        blocks += need;
    }
    flush();
    return launches ? launch_status(what) : 0;
}

constexpr int64_t ADAMW_MOST = (int64_t)((1 << 24) - 1) * ADAMW_CHUNK;

// Bytes [lo, hi) of tensor `of`, whose values have `each` bytes.
struct Span {
    uintptr_t lo, hi;
    int of, each;
};

// Whether what a call writes overlaps, or is overlapped by what it reads: thread blocks would meet there in no
// order.  spans(i, write, read) names tensor i's, up to WRITES and READS of them.  `own_read`: a tensor's own values
// may be read where they are written, from the same place on in the same width (a thread reads what it alone
// writes, before).  0, or fails.
template <int WRITES, int READS, typename Spans>
int adamw_apart(const char* message, int count, bool own_read, const Spans& spans) {
    std::unique_ptr<Span[]> written(new (std::nothrow) Span[(size_t)count * WRITES]),
        read(new (std::nothrow) Span[(size_t)count * READS]);
    if (!written || !read) return fail(-2, "yabt_adamw: no host memory");
    Span *w = written.get(), *r = read.get();
    auto into = [](Span*& to, int i) {
        return [&to, i](const void* p, int64_t n, int each) {
            *to++ = {(uintptr_t)p, (uintptr_t)p + (size_t)n * each, i, each};
        };
    };
    for (int i = 0; i < count; ++i) spans(i, into(w, i), into(r, i));
    const Span* const first = written.get();
    std::sort(written.get(), w, [](const Span& a, const Span& b) { return a.lo < b.lo; });
    for (const Span* s = first; s + 1 < w; ++s)
        if (s->hi > s[1].lo) return fail(-3, message);
    for (const Span* s = read.get(); s < r; ++s) {
        // the written spans lie apart: those that begin below s's end, from the last one backwards
        const Span* t =
            std::lower_bound(first, (const Span*)w, s->hi, [](const Span& a, uintptr_t at) { return a.lo < at; });
        while (t > first && (--t)->hi > s->lo)
            if (!(own_read && t->of == s->of && t->lo == s->lo && t->each == s->each)) return fail(-3, message);
    }
    return 0;
}
inline int64_t adamw_scales(int64_t n) { return (n + ADAMW_BLOCK - 1) / ADAMW_BLOCK; }

}  // namespace yabt

using namespace yabt;

extern "C" {

int yabt_adamw_step(int count, const yabt_adamw_tensor* tensors, int bits, int64_t step, const int32_t* step_device,
                    double lr, double beta1, double beta2, double eps, double weight_decay, yabt_stream_t stream) {
    if (bits != 32 && bits != 8) return fail(-1, "yabt_adamw_step: moments have 32 or 8 bits");
    if (!(lr >= 0.0 && lr <= 1e30) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) ||
        !(eps >= 0.0 && eps <= 1e30) || !(weight_decay >= 0.0 && weight_decay <= 1e30))
        return fail(-1, "yabt_adamw_step: lr, eps and weight_decay are 0 or more, the betas below 1");
    if (count < 0 || (!step_device && (step < 1 || step > INT32_MAX)))
        return fail(-1, "yabt_adamw_step: bad sizes (steps count from 1 to 2^31 - 1)");
    if (count > 0 && !tensors) return fail(-1, "yabt_adamw_step: null pointer");
    for (int i = 0; i < count; ++i) {
        const yabt_adamw_tensor& t = tensors[i];
        if (!dtype_ok(t.param_dtype) || !dtype_ok(t.grad_dtype))
            return fail(-1, "yabt_adamw_step: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
        if (t.n < 0 || t.n > ADAMW_MOST) return fail(-1, "yabt_adamw_step: bad sizes");
        if (t.n > 0 && (!t.param || !t.grad || !t.first || !t.second || (bits == 8 && (!t.first_scale || !t.second_scale))))
            return fail(-1, "yabt_adamw_step: null pointer");
    }
    const int apart = adamw_apart<5, 1>(
        "yabt_adamw_step: tensors overlap", count, true, [&](int i, const auto& write, const auto& read) {
            const yabt_adamw_tensor& t = tensors[i];
            if (t.n == 0) return;
            write(t.param, t.n, dtype_bytes(t.param_dtype));
            write(t.first, t.n, bits / 8);
            write(t.second, t.n, bits / 8);
            if (bits == 8) {
                write(t.first_scale, adamw_scales(t.n), 4);
                write(t.second_scale, adamw_scales(t.n), 4);
            }
            read(t.grad, t.n, dtype_bytes(t.grad_dtype));
        });
    if (apart) return apart;
    AdamwScalars S = {(float)(1.0 - beta1), (float)(1.0 - beta2), (float)(1.0 - lr * weight_decay), 0.0f, 0.0f, lr, beta1,
                      beta2, eps, step_device};
    if (!step_device) {
        const double left = std::pow(1.0 - std::pow(beta2, (double)step), 0.5);
        S.scale = (float)(lr * left / (1.0 - std::pow(beta1, (double)step)));
        S.eps = (float)(eps * left);
    }
    return adamw_launches(
        "yabt_adamw_step", count,
        [&](int i) {
            const yabt_adamw_tensor& t = tensors[i];
            return AdamwEntry{t.param, const_cast<void*>(t.grad), t.first, t.second, t.first_scale, t.second_scale, t.n,
                              t.param_dtype, t.grad_dtype};
        },
        [&](const AdamwTable& A, unsigned blocks) {
            if (bits == 32) k_adamw<32><<<blocks, ADAMW_NT, 0, (hipStream_t)stream>>>(A, S);
            else k_adamw<8><<<blocks, ADAMW_NT, 0, (hipStream_t)stream>>>(A, S);
        });
}

int yabt_adamw_values(int count, const yabt_adamw_tensor* tensors, yabt_stream_t stream) {
    if (count < 0) return fail(-1, "yabt_adamw_values: bad sizes");
    if (count > 0 && !tensors) return fail(-1, "yabt_adamw_values: null pointer");
    for (int i = 0; i < count; ++i) {
        const yabt_adamw_tensor& t = tensors[i];
        if (t.n < 0 || t.n > ADAMW_MOST) return fail(-1, "yabt_adamw_values: bad sizes");
        if (t.n > 0 && (!t.param || !t.grad || !t.first || !t.second || !t.first_scale || !t.second_scale))
            return fail(-1, "yabt_adamw_values: null pointer");
    }
    const int apart = adamw_apart<2, 4>(
        "yabt_adamw_values: tensors overlap", count, false, [&](int i, const auto& write, const auto& read) {
            const yabt_adamw_tensor& t = tensors[i];
            if (t.n == 0) return;
            write(t.param, t.n, 4);
            write(t.grad, t.n, 4);
            read(t.first, t.n, 1);
            read(t.second, t.n, 1);
            read(t.first_scale, adamw_scales(t.n), 4);
            read(t.second_scale, adamw_scales(t.n), 4);
        });
    if (apart) return apart;
    return adamw_launches(
        "yabt_adamw_values", count,
        [&](int i) {
            const yabt_adamw_tensor& t = tensors[i];
            return AdamwEntry{t.param, const_cast<void*>(t.grad), t.first, t.second, t.first_scale, t.second_scale, t.n, 0, 0};
        },
        [&](const AdamwTable& A, unsigned blocks) {
            k_adamw_values<<<blocks, ADAMW_NT, 0, (hipStream_t)stream>>>(A);
        });
}

}  // extern "C"
