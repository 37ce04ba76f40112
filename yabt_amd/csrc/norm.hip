// Layer norm of the rows of a matrix, forward and backward.
//
//   mean = sum_d x / D, rstd = 1 / sqrt(sum_d (x - mean)^2 / D + eps),
//   y = (x - mean) rstd w + c
//   t = dy w, xh = (x - mean) rstd:
//   dx = rstd (t - sum_d t / D - xh sum_d (t xh) / D), dw = sum_n dy xh, dc = sum_n dy
//
// Both passes are bound by memory: a row is read once, kept in registers as
// 16-byte chunks over G lanes (8 lanes to a whole block, NV chunks each) and
// its sums are taken there, the variance from the centred values.  A row whose
// width is no multiple of a chunk ends in a chunk that starts earlier and
// whose first values count as another chunk's; rows need no alignment.  All
// sums are fp32, in an order that the sizes alone fix.

#include "expert.h"
#include "yabt_hip.h"

namespace yabt {

// Blocks at most: they stay and walk rows, the next row's chunks on their way
// while one is worked on, and keep the weights in registers.  16384 x 4096 bf16,
// us: forward with 512, 768, 1024, 2048 and 16384 blocks 55, 57, 59, 68 and 244 (a
// copy of as many bytes takes 52), backward with 512, 768 and 1024, the parts of
// the weights' gradients and their sum included, 106, 100 and 103 (its 403 MB as a
// copy: 78); 20000 x 500 fp32: forward with 768 and 2048 17 and 19, backward 33, 29 and 30.
constexpr int NORM_BLOCKS = 768;
constexpr int NORM_GRAD_BLOCKS = 768;

// Sum over the G threads of a row; s: 2 * (G / 64) floats in LDS when G > 64,
// `flip` alternates between its halves so that one barrier is enough.
template <int G>
__device__ __forceinline__ float row_sum(float v, float* s, int& flip) {
    v = lanes_sum<G>(v);
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        float* h = s + flip * W;
        flip ^= 1;
        if ((threadIdx.x & 63) == 0) h[threadIdx.x / 64] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) v += h[i];
    }
    return v;
}

// Where chunk c of a D-wide row starts, and how many of its first values
// belong to the chunk before.
template <int N>
__device__ __forceinline__ int chunk_at(int c, int D, int* dup) {
    const int at = c * N, off = min(at, D - N);
    *dup = at - off;
    return off;
}

template <typename T, int G, int NV, int N>
__global__ void __launch_bounds__(G < 256 ? 256 : G) k_norm(const T* __restrict__ x, int64_t ldx, int64_t n, int D,
                                                           const float* __restrict__ w, const float* __restrict__ c,
                                                           float eps, T* __restrict__ y, int64_t ldy,
                                                           float* __restrict__ mean, float* __restrict__ rstd) {
    constexpr int NT = G < 256 ? 256 : G, R = NT / G;
    __shared__ float s_red[G > 64 ? 2 * (G / 64) : 1];
    const int lane = threadIdx.x % G, C = (D + N - 1) / N;
    const float inv = 1.0f / (float)D;
    int off[NV], dup[NV];
    float wv[NV][N], cv[NV][N];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int ch = v * G + lane;
        off[v] = ch < C ? chunk_at<N>(ch, D, &dup[v]) : 0;
        if (ch >= C) dup[v] = N;             // nothing of it counts
#pragma unroll
        for (int i = 0; i < N; ++i) {
            wv[v][i] = w ? w[off[v] + i] : 1.0f;
            cv[v][i] = c ? c[off[v] + i] : 0.0f;
        }
    }
    int flip = 0;
    const int64_t step = (int64_t)gridDim.x * R;
    int64_t r = (int64_t)blockIdx.x * R + threadIdx.x / G;
    Chunk<T, N> a[NV], b[NV];
    if (r < n)
#pragma unroll
        for (int v = 0; v < NV; ++v) a[v].load(x + (size_t)r * (size_t)ldx + off[v]);
    for (; r < n; r += step) {
        const bool more = r + step < n;      // the next row's chunks are on their way meanwhile
        if (more)
#pragma unroll
            for (int v = 0; v < NV; ++v) b[v].load(x + (size_t)(r + step) * (size_t)ldx + off[v]);
        float s = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) s += i >= dup[v] ? a[v].get(i) : 0.0f;
        const float mu = row_sum<G>(s, s_red, flip) * inv;
        float q = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float d = a[v].get(i) - mu;
                q += i >= dup[v] ? d * d : 0.0f;
            }
        const float rs = 1.0f / sqrtf(row_sum<G>(q, s_red, flip) * inv + eps);
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (dup[v] < N) {
                Chunk<T, N> o;
#pragma unroll
                for (int i = 0; i < N; ++i) o.set(i, (a[v].get(i) - mu) * rs * wv[v][i] + cv[v][i]);
                o.store(y + (size_t)r * (size_t)ldy + off[v]);
            }
        if (lane == 0) {
            if (mean) mean[r] = mu;
            if (rstd) rstd[r] = rs;
        }
        if (more)
#pragma unroll
            for (int v = 0; v < NV; ++v) a[v] = b[v];
    }
}

// Backward.  A block walks its rows with the weight's and the bias's gradient
// of its columns in registers and leaves them in part (block, 2, D); with one
// block they are the result.
template <typename T, int G, int NV, int N>
__global__ void __launch_bounds__(G < 256 ? 256 : G) k_norm_grad(
    const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, int64_t n, int D,
    const float* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
    int64_t lddx, float* __restrict__ dw, float* __restrict__ dc, float* __restrict__ part) {
    constexpr int NT = G < 256 ? 256 : G, R = NT / G;
    __shared__ float s_red[G > 64 ? 2 * (G / 64) : 1];
    const int lane = threadIdx.x % G, C = (D + N - 1) / N;
    const float inv = 1.0f / (float)D;
    int off[NV], dup[NV];
    float wv[NV][N], gw[NV][N], gc[NV][N];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int ch = v * G + lane;
        off[v] = ch < C ? chunk_at<N>(ch, D, &dup[v]) : 0;
        if (ch >= C) dup[v] = N;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            wv[v][i] = w ? w[off[v] + i] : 1.0f;
            gw[v][i] = gc[v][i] = 0.0f;
        }
    }
    int flip = 0;
    const int64_t step = (int64_t)gridDim.x * R;
    int64_t r = (int64_t)blockIdx.x * R + threadIdx.x / G;
    Chunk<T, N> a[NV], b[NV], a2[NV], b2[NV];
    float mu = 0.0f, rs = 0.0f, mu2 = 0.0f, rs2 = 0.0f;
    auto load = [&](Chunk<T, N>* xa, Chunk<T, N>* ya, float& m, float& q, int64_t row) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            xa[v].load(x + (size_t)row * (size_t)ldx + off[v]);
            ya[v].load(dy + (size_t)row * (size_t)lddy + off[v]);
        }
        m = mean[row];
        q = rstd[row];
    };
    if (r < n) load(a, b, mu, rs, r);
    for (; r < n; r += step) {
        const bool more = r + step < n;
        if (more) load(a2, b2, mu2, rs2, r + step);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float g = b[v].get(i), xh = (a[v].get(i) - mu) * rs, t = g * wv[v][i];
                if (i >= dup[v]) {
                    s1 += t;
                    s2 += t * xh;
                    gw[v][i] += g * xh;
                    gc[v][i] += g;
                }
            }
        if (dx) {
            s1 = row_sum<G>(s1, s_red, flip) * inv;
            s2 = row_sum<G>(s2, s_red, flip) * inv;
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (dup[v] < N) {
                    Chunk<T, N> o;
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float xh = (a[v].get(i) - mu) * rs, t = b[v].get(i) * wv[v][i];
                        o.set(i, rs * (t - s1 - xh * s2));
                    }
                    o.store(dx + (size_t)r * (size_t)lddx + off[v]);
                }
        }
        if (more) {
#pragma unroll
            for (int v = 0; v < NV; ++v) a[v] = a2[v], b[v] = b2[v];
            mu = mu2;
            rs = rs2;
        }
    }
    if (!dw && !dc) return;
    float* ow = part ? part + (size_t)blockIdx.x * 2 * (size_t)D : dw;
    float* oc = part ? ow + D : dc;
    if constexpr (R == 1) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i >= dup[v]) {
                    if (ow) ow[off[v] + i] = gw[v][i];
                    if (oc) oc[off[v] + i] = gc[v][i];
                }
    } else {
        // the block's row groups, added in order
        __shared__ float s_g[NT * NV * N];
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            __syncthreads();
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < N; ++i) s_g[(v * N + i) * NT + threadIdx.x] = side ? gc[v][i] : gw[v][i];
            __syncthreads();
            float* o = side ? oc : ow;
            if (o && threadIdx.x < G) {
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (i >= dup[v]) {
                            float t = 0.0f;
                            for (int g = 0; g < R; ++g) t += s_g[(v * N + i) * NT + g * G + lane];
                            o[off[v] + i] = t;
                        }
            }
        }
    }
}

// Rows too long for registers: a block per row, read once per sum (the later
// reads come from the caches), by chunks as above.  4096 x 20000 bf16: 108 us forward
// (3.0 TB/s over one read and write), 193 backward, 93 and 175 back to
// back; value by value 195 and 329.
constexpr int LONG_NT = 1024;

// chunk c's values of a parameter vector, or `none` where there is no vector
template <int N>
__device__ __forceinline__ void chunk_floats(const float* p, int off, float none, float* v) {
    static_assert(N % 4 == 0, "whole 16 bytes");
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        Chunk<float, 4> f;
        if (p) f.load(p + off + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i + j] = p ? f.get(j) : none;
    }
}

template <typename T>
__global__ void __launch_bounds__(LONG_NT) k_norm_long(const T* __restrict__ x, int64_t ldx, int64_t n, int D,
                                                       const float* __restrict__ w, const float* __restrict__ c,
                                                       float eps, T* __restrict__ y, int64_t ldy,
                                                       float* __restrict__ mean, float* __restrict__ rstd) {
    constexpr int N = VEC<T>;
    __shared__ float s_red[2 * (LONG_NT / 64)];
    int flip = 0, dup;
    const int C = (D + N - 1) / N;
    const float inv = 1.0f / (float)D;
    for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
        const T* row = x + (size_t)r * (size_t)ldx;
        T* const o = y + (size_t)r * (size_t)ldy;
        Chunk<T, N> a;
        float s = 0.0f, q = 0.0f;
#pragma unroll 4
        for (int ch = threadIdx.x; ch < C; ch += LONG_NT) {
            a.load(row + chunk_at<N>(ch, D, &dup));
#pragma unroll
            for (int i = 0; i < N; ++i) s += i >= dup ? a.get(i) : 0.0f;
        }
        const float mu = row_sum<LONG_NT>(s, s_red, flip) * inv;
#pragma unroll 4
        for (int ch = threadIdx.x; ch < C; ch += LONG_NT) {
            a.load(row + chunk_at<N>(ch, D, &dup));
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float t = a.get(i) - mu;
                q += i >= dup ? t * t : 0.0f;
            }
        }
        const float rs = 1.0f / sqrtf(row_sum<LONG_NT>(q, s_red, flip) * inv + eps);
        for (int ch = threadIdx.x; ch < C; ch += LONG_NT) {
            const int off = chunk_at<N>(ch, D, &dup);
            float wv[N], cv[N];
            a.load(row + off);
            chunk_floats<N>(w, off, 1.0f, wv);
            chunk_floats<N>(c, off, 0.0f, cv);
#pragma unroll
            for (int i = 0; i < N; ++i) a.set(i, (a.get(i) - mu) * rs * wv[i] + cv[i]);
            a.store(o + off);
        }
        if (threadIdx.x == 0) {
            if (mean) mean[r] = mu;
            if (rstd) rstd[r] = rs;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(LONG_NT) k_norm_long_dx(const T* __restrict__ dy, int64_t lddy,
                                                          const T* __restrict__ x, int64_t ldx, int64_t n, int D,
                                                          const float* __restrict__ w, const float* __restrict__ mean,
                                                          const float* __restrict__ rstd, T* __restrict__ dx,
                                                          int64_t lddx) {
    constexpr int N = VEC<T>;
    __shared__ float s_red[2 * (LONG_NT / 64)];
    int flip = 0, dup;
    const int C = (D + N - 1) / N;
    const float inv = 1.0f / (float)D;
    for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
        const T* row = x + (size_t)r * (size_t)ldx;
        const T* g = dy + (size_t)r * (size_t)lddy;
        T* const o = dx + (size_t)r * (size_t)lddx;
        const float mu = mean[r], rs = rstd[r];
        Chunk<T, N> a, b;
        float wv[N], s1 = 0.0f, s2 = 0.0f;
#pragma unroll 2
        for (int ch = threadIdx.x; ch < C; ch += LONG_NT) {
            const int off = chunk_at<N>(ch, D, &dup);
            a.load(g + off);
            b.load(row + off);
            chunk_floats<N>(w, off, 1.0f, wv);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float t = i >= dup ? a.get(i) * wv[i] : 0.0f;
                s1 += t;
                s2 += i >= dup ? t * ((b.get(i) - mu) * rs) : 0.0f;
            }
        }
        s1 = row_sum<LONG_NT>(s1, s_red, flip) * inv;
        s2 = row_sum<LONG_NT>(s2, s_red, flip) * inv;
        for (int ch = threadIdx.x; ch < C; ch += LONG_NT) {
            const int off = chunk_at<N>(ch, D, &dup);
            a.load(g + off);
            b.load(row + off);
            chunk_floats<N>(w, off, 1.0f, wv);
#pragma unroll
            for (int i = 0; i < N; ++i) a.set(i, rs * (a.get(i) * wv[i] - s1 - (b.get(i) - mu) * rs * s2));
            a.store(o + off);
        }
    }
}

// Weight gradients of long rows: a block takes 256 chunks of one slice of rows.
// A row's last chunk starts earlier: two threads find the same values for its first columns.
template <typename T>
__global__ void __launch_bounds__(256) k_norm_long_dw(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x,
                                                      int64_t ldx, int64_t n, int D, const float* __restrict__ mean,
                                                      const float* __restrict__ rstd, int slices,
                                                      float* __restrict__ dw, float* __restrict__ dc,
                                                      float* __restrict__ part) {
    constexpr int N = VEC<T>;
    const int ch = blockIdx.x * 256 + threadIdx.x;
    int dup;
    if (ch >= (D + N - 1) / N) return;
    const int d = chunk_at<N>(ch, D, &dup);
    const int64_t per = (n + slices - 1) / slices, lo = blockIdx.y * per, hi = min(n, lo + per);
    float sw[N], sc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sw[i] = sc[i] = 0.0f;
#pragma unroll 4
    for (int64_t r = lo; r < hi; ++r) {
        Chunk<T, N> a, b;
        a.load(dy + (size_t)r * (size_t)lddy + d);
        b.load(x + (size_t)r * (size_t)ldx + d);
        const float mu = mean[r], rs = rstd[r];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            sw[i] += a.get(i) * ((b.get(i) - mu) * rs);
            sc[i] += a.get(i);
        }
    }
    float* ow = part ? part + (size_t)blockIdx.y * 2 * (size_t)D : dw;
    float* oc = part ? ow + D : dc;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (ow) ow[d + i] = sw[i];
        if (oc) oc[d + i] = sc[i];
    }
}

// The blocks' parts added: 64 of the 2 D columns a block, 16 threads each.
__global__ void __launch_bounds__(1024) k_norm_parts(const float* __restrict__ part, int blocks, int D,
                                                     float* __restrict__ dw, float* __restrict__ dc) {
    __shared__ float s[16][64];
    const int64_t col = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    const int g = threadIdx.x / 64;
    float t = 0.0f;
    if (col < 2 * (int64_t)D) {
#pragma unroll 8
        for (int b = g; b < blocks; b += 16) t += part[(size_t)b * 2 * (size_t)D + col];
    }
    s[g][threadIdx.x & 63] = t;
    __syncthreads();
    if (g == 0 && col < 2 * (int64_t)D) {
        t = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += s[i][threadIdx.x];
        if (col < D) {
            if (dw) dw[col] = t;
        } else if (dc) {
            dc[col - D] = t;
        }
    }
}

// (G, NV, N) for a D-wide row of T, given to f as constants; false: the row
// does not fit registers.
template <typename T, typename F>
bool norm_shape(int D, const F& f) {
    constexpr int N = VEC<T>;
    if (D < N) {
        f(std::integral_constant<int, 8>(), std::integral_constant<int, 1>(), std::integral_constant<int, 1>());
        return true;
    }
    const int C = (D + N - 1) / N;
#define YABT_SHAPE(g, nv)                                                                                     \
    if (C <= g * nv) {                                                                                        \
        f(std::integral_constant<int, g>(), std::integral_constant<int, nv>(), std::integral_constant<int, N>()); \
        return true;                                                                                          \
    }
    YABT_SHAPE(8, 1)
    YABT_SHAPE(16, 1)
    YABT_SHAPE(16, 2)
    YABT_SHAPE(64, 1)
    YABT_SHAPE(64, 2)
    YABT_SHAPE(256, 1)
    YABT_SHAPE(256, 2)
    YABT_SHAPE(512, 2)
    YABT_SHAPE(1024, 2)
#undef YABT_SHAPE
    return false;
}

template <typename T>
void run_norm(const T* x, int64_t ldx, int64_t n, int D, const float* w, const float* c, float eps, T* y, int64_t ldy,
              float* mean, float* rstd, hipStream_t stream) {
    const bool fits = norm_shape<T>(D, [&](auto g, auto nv, auto nn) {
        constexpr int G = decltype(g)::value, NV = decltype(nv)::value, N = decltype(nn)::value;
        constexpr int NT = G < 256 ? 256 : G;
        k_norm<T, G, NV, N><<<launch_grid(n, NT / G, NORM_BLOCKS), NT, 0, stream>>>(x, ldx, n, D, w, c, eps, y, ldy, mean,
                                                                           rstd);
    });
    if (!fits)
        k_norm_long<T><<<launch_grid(n, 1, 2048), LONG_NT, 0, stream>>>(x, ldx, n, D, w, c, eps, y, ldy, mean, rstd);
}

// Blocks that walk the rows in the backward pass, a part of the weights' gradients
// each: a block gets a few rows of its own before the parts' traffic (8 D bytes a
// block, written and read) counts.  Rows too long for registers: the slices of
// rows, which `across` blocks share.
template <typename T>
int norm_long_across(int D) {
    return (int)((D + 256 * (int64_t)VEC<T> - 1) / (256 * VEC<T>));
}
template <typename T>
int norm_grad_blocks(int64_t n, int D) {
    int blocks = 1;
    const bool fits = norm_shape<T>(D, [&](auto g, auto, auto) {
        constexpr int G = decltype(g)::value, R = (G < 256 ? 256 : G) / G;
        blocks = launch_grid(n, R * 4, NORM_GRAD_BLOCKS);
    });
    const int across = norm_long_across<T>(D);
    return fits ? blocks : launch_grid(n, 32, (NORM_GRAD_BLOCKS + across - 1) / across);
}

template <typename T>
void run_norm_grad(const T* dy, int64_t lddy, const T* x, int64_t ldx, int64_t n, int D, const float* w,
                   const float* mean, const float* rstd, float* part, T* dx, int64_t lddx, float* dw, float* dc,
                   hipStream_t stream) {
    const int blocks = norm_grad_blocks<T>(n, D);
    const bool fits = norm_shape<T>(D, [&](auto g, auto nv, auto nn) {
        constexpr int G = decltype(g)::value, NV = decltype(nv)::value, N = decltype(nn)::value;
        constexpr int NT = G < 256 ? 256 : G;
        k_norm_grad<T, G, NV, N><<<blocks, NT, 0, stream>>>(dy, lddy, x, ldx, n, D, w, mean, rstd, dx, lddx, dw, dc,
                                                            blocks > 1 ? part : nullptr);
    });
    if (!fits) {
        if (dx)
            k_norm_long_dx<T><<<launch_grid(n, 1, 2048), LONG_NT, 0, stream>>>(dy, lddy, x, ldx, n, D, w, mean, rstd,
                                                                             dx, lddx);
        if (dw || dc)
            k_norm_long_dw<T><<<dim3((unsigned)norm_long_across<T>(D), (unsigned)blocks), 256, 0, stream>>>(
                dy, lddy, x, ldx, n, D, mean, rstd, blocks, dw, dc, blocks > 1 ? part : nullptr);
    }
    if (blocks > 1 && (dw || dc))
        k_norm_parts<<<(unsigned)((2 * (int64_t)D + 63) / 64), 1024, 0, stream>>>(part, blocks, D, dw, dc);
}

}  // namespace yabt

using namespace yabt;

extern "C" {

int yabt_layer_norm(int dtype, const void* x, int64_t ldx, int64_t n, int D, const float* weight, const float* bias,
                    float eps, void* y, int64_t ldy, float* mean, float* rstd, yabt_stream_t stream) {
    if (!dtype_ok(dtype)) return fail(-1, "yabt_layer_norm: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (n < 0 || D < 1 || ldx < D || ldy < D || !(eps >= 0.0f)) return fail(-1, "yabt_layer_norm: bad sizes");
    if (n == 0) return 0;
    if (!x || !y) return fail(-1, "yabt_layer_norm: null pointer");
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DT_F32)
        run_norm<float>((const float*)x, ldx, n, D, weight, bias, eps, (float*)y, ldy, mean, rstd, st);
    else if (dtype == DT_BF16)
        run_norm<bf16>((const bf16*)x, ldx, n, D, weight, bias, eps, (bf16*)y, ldy, mean, rstd, st);
    else
        run_norm<f16>((const f16*)x, ldx, n, D, weight, bias, eps, (f16*)y, ldy, mean, rstd, st);
    return launch_status("yabt_layer_norm");
}

size_t yabt_layer_norm_grad_workspace_bytes(int64_t n, int D) {
    if (n < 0 || D < 1) return 0;
    // bf16 and fp16 rows have the same chunks
    const int blocks = norm_grad_blocks<float>(n, D), half = norm_grad_blocks<bf16>(n, D);
    return (size_t)(blocks > half ? blocks : half) * 2 * (size_t)D * sizeof(float);
}

int yabt_layer_norm_grad(int dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t n, int D,
                         const float* weight, const float* mean, const float* rstd, void* workspace,
                         size_t workspace_bytes, void* dx, int64_t lddx, float* dweight, float* dbias,
                         yabt_stream_t stream) {
    if (!dtype_ok(dtype)) return fail(-1, "yabt_layer_norm_grad: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (n < 0 || D < 1 || ldx < D || lddy < D || (dx && lddx < D)) return fail(-1, "yabt_layer_norm_grad: bad sizes");
    if (n > 0 && (!x || !dy || !mean || !rstd)) return fail(-1, "yabt_layer_norm_grad: null pointer");
    if (!workspace || workspace_bytes < yabt_layer_norm_grad_workspace_bytes(n, D))
        return fail(-2, "yabt_layer_norm_grad: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    float* part = (float*)workspace;
    // n = 0 launches one block, which writes zero gradients
    if (dtype == DT_F32)
        run_norm_grad<float>((const float*)dy, lddy, (const float*)x, ldx, n, D, weight, mean, rstd, part, (float*)dx,
                             lddx, dweight, dbias, st);
    else if (dtype == DT_BF16)
        run_norm_grad<bf16>((const bf16*)dy, lddy, (const bf16*)x, ldx, n, D, weight, mean, rstd, part, (bf16*)dx,
                            lddx, dweight, dbias, st);
    else
        run_norm_grad<f16>((const f16*)dy, lddy, (const f16*)x, ldx, n, D, weight, mean, rstd, part, (f16*)dx, lddx,
                           dweight, dbias, st);
    return launch_status("yabt_layer_norm_grad");
}

}  // extern "C"
