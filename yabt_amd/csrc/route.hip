// Routing rows to experts: the k best of E scores, their weights, the weights'
// gradient, and the plan that sorts the slots by expert.
//
//   p = softmax(l) or 1 / (1 + exp(-l)); an expert is chosen by its key,
//   key = l + bias (softmax, whose order is the logits') or p + bias (sigmoid),
//   in fp32; a logit of -inf or NaN closes the expert to the row.  With groups
//   the best `keep` groups stay, by their largest key (softmax) or the sum of
//   their two largest (sigmoid).  The k largest keys win, equal ones by the
//   lower index; w_j = scale p_j, or scale p_j / sum of the chosen p.
//
// A row is held by G lanes, NV consecutive experts each.  A key and its expert
// travel as one double: the key's 24 bits in front, the expert's number in low
// bits that the key leaves free, so that one v_max_f64 compares both.  A lane
// sorts its own keys once (an odd-even merge network).  Up to k = 8 of 8 and
// more a lane, the lanes then merge their best 8 pairwise (the larger of one
// list and the other reversed, sorted by three rounds of a bitonic network),
// log2 G times; else a round takes the largest of the G heads over DPP and the
// winner drops its head, k times.
//
// What bounds it is instructions, not memory: 65 536 rows of 256 bf16 logits,
// sigmoid, 8 experts in 4 of 8 groups, take 44 us, of which the VALU issues for 40
// (1258 instructions a wave of 4 rows, a third of them the exponentials; 38 MB
// are 7 us of a copy).  72 us with k rounds in place of the merge, the
// compiler's division and the groups' keys scanned in LDS.

#include "expert.h"
#include "yabt_hip.h"

#include <cfloat>

namespace yabt {

constexpr int ROUTE_NT = 256;
constexpr int ROUTE_MAX_E = 1024, ROUTE_MAX_K = 32, ROUTE_MAX_GROUPS = 64;
constexpr int SOFTMAX = 0, SIGMOID = 1;

#define YABT_NEG_INF (-__builtin_inff())

// (key, e) as one double that orders by key, then by lower e; a key of -inf
// carries no e, +inf counts as the largest number.
__device__ __forceinline__ double key_pack(float key, int e) {
    key = fminf(key, FLT_MAX) + 0.0f;               // -0 is 0
    const uint64_t u = (uint64_t)__double_as_longlong((double)key);
    // the lower e is larger in front of a positive key and smaller in front of a negative one
    const uint32_t low = (uint32_t)(ROUTE_MAX_E - 1 - e) ^ ((uint32_t)((int32_t)__float_as_uint(key) >> 31) & (ROUTE_MAX_E - 1));
    return __longlong_as_double((long long)(u | (key == YABT_NEG_INF ? 0u : low)));
}
__device__ __forceinline__ int key_expert(double m) {
    const uint64_t u = (uint64_t)__double_as_longlong(m);
    const int low = (int)(u & (ROUTE_MAX_E - 1));
    return (u >> 63) ? low : ROUTE_MAX_E - 1 - low;
}

// h sorted descending by an odd-even merge network.
template <int NV>
__device__ __forceinline__ void sort_desc(double (&h)[NV]) {
#pragma unroll
    for (int p = 1; p < NV; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j <= NV - 1 - q; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < NV && (i + j) / (p * 2) == (i + j + q) / (p * 2)) {
                        const double a = h[i + j], b = h[i + j + q];
                        h[i + j] = fmax(a, b);
                        h[i + j + q] = fmin(a, b);
                    }
}

// The best 8 of each aligned run of G lanes, descending, from the lanes' own
// (descending) lists: every lane gets them.
template <int G, int M = 1>
__device__ __forceinline__ void merge_best(double (&h)[8]) {
    if constexpr (M < G) {
        double t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = fmax(h[i], lanes_other<M>(h[7 - i]));
#pragma unroll
        for (int d = 4; d >= 1; d /= 2)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((i & d) == 0) {
                    const double a = t[i], b = t[i + d];
                    t[i] = fmax(a, b);
                    t[i + d] = fmin(a, b);
                }
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = t[i];
        merge_best<G, M * 2>(h);
    }
}

// The two largest of each run of q lanes (a power of two), from their own.
template <int G, int M = 1>
__device__ __forceinline__ void two_largest(float& a, float& b, int q) {
    if constexpr (M < G) {
        if (M < q) {
            const float a2 = lanes_other<M>(a), b2 = lanes_other<M>(b);
            b = fmaxf(fminf(a, a2), fmaxf(b, b2));
            a = fmaxf(a, a2);
            two_largest<G, M * 2>(a, b, q);
        }
    }
}

// A lane's NV consecutive logits; -inf for those past E and for NaN.
template <typename T, int NV>
__device__ __forceinline__ void load_logits(const T* row, int e0, int E, float (&x)[NV]) {
    typedef T VT __attribute__((ext_vector_type(NV), aligned(sizeof(T))));
    if constexpr (NV > 1) {
        if (e0 + NV <= E) {
            const VT v = *reinterpret_cast<const VT*>(row + e0);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const float f = (float)v[i];
                x[i] = f > YABT_NEG_INF ? f : YABT_NEG_INF;
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const float f = e0 + i < E ? (float)row[e0 + i] : YABT_NEG_INF;
        x[i] = f > YABT_NEG_INF ? f : YABT_NEG_INF;
    }
}

template <int NV>
__device__ __forceinline__ void load_any(int dtype, const void* logits, size_t at, int e0, int E, float (&x)[NV]) {
    if (dtype == DT_F32) load_logits<float, NV>((const float*)logits + at, e0, E, x);
    else if (dtype == DT_BF16) load_logits<bf16, NV>((const bf16*)logits + at, e0, E, x);
    else load_logits<f16, NV>((const f16*)logits + at, e0, E, x);
}
__device__ __forceinline__ float value_at(int dtype, const void* p, size_t i) {
    return dtype == DT_F32 ? ((const float*)p)[i] : dtype == DT_BF16 ? (float)((const bf16*)p)[i] : (float)((const f16*)p)[i];
}

// Max and sum of exp(x - max) of a row; those of a row without open experts
// count as 0 and 1, so that its scores are 0.
template <int G, int NV>
__device__ __forceinline__ void softmax_stats(const float (&x)[NV], float* top, float* sum) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < NV; ++i) m = fmaxf(m, x[i]);
    m = lanes_max<G>(m);
    if (m == YABT_NEG_INF) m = 0.0f;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) s += expf(x[i] - m);
    s = lanes_sum<G>(s);
    *top = m;
    *sum = s > 0.0f ? s : 1.0f;
}

struct RouteArgs {
    int64_t ldl, n;
    int E, k, scores, renormalise;
    int groups, keep, per_group, magic;     // magic: ceil(2^20 / per_group)
    float scale;
    int dtype;
};

// The p of the chosen experts (lane j holds slots j and j + G) turned into v:
// p / sum with `renorm`, p itself without; *total: the sum (softmax with
// renorm: of the exponentials).
template <int G, int S>
__device__ __forceinline__ void chosen_scores(const RouteArgs& A, const float (&l)[S], const bool (&on)[S], float top,
                                              float sum, float (&p)[S], float (&v)[S], float* total) {
    float t = 0.0f;
    if (A.scores == SOFTMAX && A.renormalise) {
        // over the chosen alone: the others' exponentials cancel
        float m = YABT_NEG_INF;
#pragma unroll
        for (int s = 0; s < S; ++s) m = on[s] ? fmaxf(m, l[s]) : m;
        m = lanes_max<G>(m);
#pragma unroll
        for (int s = 0; s < S; ++s) p[s] = on[s] ? expf(l[s] - m) : 0.0f;
    } else {
        if (A.scores == SIGMOID) sigmoids<S>(l, p);
#pragma unroll
        for (int s = 0; s < S; ++s) p[s] = !on[s] ? 0.0f : A.scores == SOFTMAX ? expf(l[s] - top) / sum : p[s];
    }
#pragma unroll
    for (int s = 0; s < S; ++s) t += p[s];
    t = lanes_sum<G>(t);
    *total = t;
#pragma unroll
    for (int s = 0; s < S; ++s) v[s] = !A.renormalise ? p[s] : t > 0.0f ? p[s] / t : 0.0f;
}

// GROUPS: 0 none, 1 each a power of two of lanes, 2 any.
template <int G, int NV, int SCORES, int GROUPS, bool MERGE>
__global__ void __launch_bounds__(ROUTE_NT) k_route(RouteArgs A, const void* __restrict__ logits,
                                                    const float* __restrict__ bias, int32_t* __restrict__ ids,
                                                    float* __restrict__ weights) {
    constexpr int R = ROUTE_NT / G, S = MERGE ? 1 : (ROUTE_MAX_K + G - 1) / G;
    __shared__ float s_key[GROUPS == 2 ? R : 1][GROUPS == 2 ? G * NV : 1];
    __shared__ float s_score[GROUPS ? R : 1][GROUPS ? ROUTE_MAX_GROUPS : 1];
    __shared__ int s_stay[GROUPS ? R : 1][GROUPS ? ROUTE_MAX_GROUPS : 1];
    const int lane = threadIdx.x % G, sub = threadIdx.x / G, e0 = lane * NV;
    float bv[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) bv[i] = bias && e0 + i < A.E ? bias[e0 + i] : 0.0f;
    for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < A.n; r0 += (int64_t)gridDim.x * R) {
        // rows past the end are walked as the last one, and not written
        const int64_t r = min(r0 + sub, A.n - 1);
        const size_t row = (size_t)r * (size_t)A.ldl;
        float x[NV], top = 0.0f, sum = 1.0f;
        load_any<NV>(A.dtype, logits, row, e0, A.E, x);
        if (SCORES == SOFTMAX && !A.renormalise) softmax_stats<G, NV>(x, &top, &sum);
        float key[NV];
        if constexpr (SCORES == SIGMOID) sigmoids<NV>(x, key);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const float q = (SCORES == SOFTMAX ? x[i] : key[i]) + bv[i];
            key[i] = x[i] > YABT_NEG_INF && q > YABT_NEG_INF ? q : YABT_NEG_INF;
        }
        if constexpr (GROUPS != 0) {
            if constexpr (GROUPS == 1) {
                float a = YABT_NEG_INF, b = YABT_NEG_INF;     // the lane's, then its group's two largest keys
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    b = __builtin_amdgcn_fmed3f(a, b, key[i]);        // a >= b
                    a = fmaxf(a, key[i]);
                }
                const int q = A.per_group / NV;
                two_largest<G>(a, b, q);
                // lanes past the experts are in no group
                if (e0 < A.E) s_score[sub][lane / q] = SCORES == SIGMOID && b > YABT_NEG_INF ? a + b : a;
            } else {
#pragma unroll
                for (int i = 0; i < NV; ++i) s_key[sub][e0 + i] = key[i];
                wave_sync_lds();
                for (int g = lane; g < A.groups; g += G) {
                    float a = YABT_NEG_INF, b = YABT_NEG_INF;
                    int at = g % A.per_group;                 // lanes start apart: other banks
                    for (int i = 0; i < A.per_group; ++i) {
                        const float q = s_key[sub][g * A.per_group + at];
                        b = fmaxf(b, fminf(a, q));
                        a = fmaxf(a, q);
                        at = at + 1 == A.per_group ? 0 : at + 1;
                    }
                    s_score[sub][g] = SCORES == SIGMOID && b > YABT_NEG_INF ? a + b : a;
                }
            }
            wave_sync_lds();
            // a group stays if fewer than `keep` are before it
            for (int g = lane; g < A.groups; g += G) {
                const float own = s_score[sub][g];
                int before = 0;
                for (int o = 0; o < A.groups; ++o) {
                    const float q = s_score[sub][o];
                    before += q > own || (q == own && o < g);
                }
                s_stay[sub][g] = before < A.keep;
            }
            wave_sync_lds();
            if constexpr (GROUPS == 1) {
                const bool stay = s_stay[sub][min(lane / (A.per_group / NV), A.groups - 1)];
#pragma unroll
                for (int i = 0; i < NV; ++i) key[i] = stay ? key[i] : YABT_NEG_INF;
            } else {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int g = min((int)(((uint32_t)(e0 + i) * (uint32_t)A.magic) >> 20), A.groups - 1);
                    if (!s_stay[sub][g]) key[i] = YABT_NEG_INF;
                }
            }
            wave_sync_lds();
        }
        double h[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) h[i] = key_pack(key[i], e0 + i);
        sort_desc<NV>(h);
        int mine[S];
        if constexpr (MERGE) {
            double b8[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) b8[i] = h[i];
            merge_best<G>(b8);
            double m = b8[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) m = lane == i ? b8[i] : m;
            mine[0] = lane < A.k && m > -__builtin_inf() ? key_expert(m) : -1;
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s) mine[s] = -1;
            for (int j = 0; j < A.k; ++j) {
                const double m = lanes_reduce<G>(h[0], [](double a, double b) { return fmax(a, b); });
                const int e = m > -__builtin_inf() ? key_expert(m) : -1;
#pragma unroll
                for (int s = 0; s < S; ++s)
                    if (j == s * G + lane) mine[s] = e;
                const bool won = h[0] == m;
#pragma unroll
                for (int i = 0; i < NV; ++i) h[i] = won ? i + 1 < NV ? h[i + 1] : -__builtin_inf() : h[i];
            }
        }
        float l[S], p[S], v[S], total;
        bool on[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            on[s] = mine[s] >= 0;
            l[s] = on[s] ? value_at(A.dtype, logits, row + mine[s]) : 0.0f;
        }
        chosen_scores<G, S>(A, l, on, top, sum, p, v, &total);
        if (r0 + sub < A.n) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const int j = s * G + lane;
                if (j < A.k) {
                    ids[(size_t)r * A.k + j] = mine[s];
                    weights[(size_t)r * A.k + j] = A.scale * v[s];
                }
            }
        }
    }
}

// d(weights) to d(logits), the choice held fixed (ids as k_route left them;
// one outside [0, E) takes no part):
//   softmax, renormalised: v = softmax over the chosen, dl_j = v_j (dw_j - sum v dw)
//   softmax:  dl_i = p_i ([i chosen] dw_i - sum_chosen p dw)
//   sigmoid, renormalised: v = p / t, dl_j = (dw_j - sum v dw) / t p_j (1 - p_j)
//   sigmoid:  dl_j = dw_j p_j (1 - p_j)                    with dw scaled by `scale`
// A row's gradient is put together in LDS, so that it leaves in whole lines
// whatever experts were chosen.  8191 x 60 fp32, k = 4: 4.8 us, a launch's length
// and its loads' latency (4 MB).
template <typename T, int G, int NV>
__global__ void __launch_bounds__(ROUTE_NT) k_route_grad(RouteArgs A, const float* __restrict__ dweights, int64_t lddw,
                                                         const T* __restrict__ logits,
                                                         const int32_t* __restrict__ ids, T* __restrict__ dlogits,
                                                         int64_t lddl) {
    constexpr int R = ROUTE_NT / G, S = (ROUTE_MAX_K + G - 1) / G;
    __shared__ float s_d[R][G * NV];
    const int lane = threadIdx.x % G, sub = threadIdx.x / G, e0 = lane * NV;
    for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < A.n; r0 += (int64_t)gridDim.x * R) {
        const int64_t r = min(r0 + sub, A.n - 1);
        const T* row = logits + (size_t)r * (size_t)A.ldl;
        const bool whole = A.scores == SOFTMAX && !A.renormalise;
        float x[NV], top = 0.0f, sum = 1.0f;
        if (whole) {
            load_logits<T, NV>(row, e0, A.E, x);
            softmax_stats<G, NV>(x, &top, &sum);
        }
        int id[S];
        float l[S], dw[S], p[S], v[S], total, mean = 0.0f;
        bool on[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int j = s * G + lane;
            id[s] = j < A.k ? ids[(size_t)r * A.k + j] : -1;
            on[s] = id[s] >= 0 && id[s] < A.E;
            l[s] = on[s] ? (float)row[id[s]] : 0.0f;
            dw[s] = on[s] ? dweights[(size_t)r * (size_t)lddw + j] * A.scale : 0.0f;
        }
        chosen_scores<G, S>(A, l, on, top, sum, p, v, &total);
#pragma unroll
        for (int s = 0; s < S; ++s) mean += v[s] * dw[s];
        mean = lanes_sum<G>(mean);
#pragma unroll
        for (int i = 0; i < NV; ++i) s_d[sub][e0 + i] = whole ? -(expf(x[i] - top) / sum) * mean : 0.0f;
        wave_sync_lds();
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (on[s]) {
                float d;
                if (A.scores == SOFTMAX) d = v[s] * (whole ? dw[s] : dw[s] - mean);
                else if (A.renormalise) d = total > 0.0f ? (dw[s] - mean) / total * p[s] * (1.0f - p[s]) : 0.0f;
                else d = dw[s] * p[s] * (1.0f - p[s]);
                atomicAdd(&s_d[sub][id[s]], d);
            }
        wave_sync_lds();
        if (r0 + sub < A.n) {
            T* o = dlogits + (size_t)r * (size_t)lddl;
            for (int e = lane; e < A.E; e += G) o[e] = (T)s_d[sub][e];
        }
        wave_sync_lds();
    }
}

// ---------------------------------------------------------------------------
// The plan: a stable counting sort of the slots (row, j) by expert.  A wave
// takes 64 R slots in a row, all loaded at once, and counts them 64 at a time:
// a slot's rank is its wave's count so far plus the lanes before it with the
// same expert, which one ballot per bit of the expert's number finds.  Up to
// PLAN_ONE slots are sorted in one block's LDS, in one launch; more are counted
// by blocks, then ranked and placed: 32 764 slots of 60 experts take 12.6 us with a
// launch between that takes the counts' prefix per expert, and 30 in one block,
// whose CU alone is bound by the ballots.  Few blocks take the prefix each by
// itself, without the launch between, us of kernels with and without it: 20 000
// slots of 7 experts 13.1 and 9.3, 131 072 of 64 13.9 and 11.0, 65 536 of 1024 17.4 and
// 16.1; many do not, 524 288 of 256 18.8 and 24.3.
// ---------------------------------------------------------------------------

constexpr int PLAN_NT = 512, PLAN_R = 4;
constexpr int PLAN_TILE = PLAN_NT * PLAN_R;      // slots a block ranks at a time
constexpr int PLAN_BLOCKS = 1024;                // blocks at most
constexpr int PLAN_ONE = 8192;                   // slots one block sorts, at most
constexpr int PLAN_FEW = 64;                     // blocks that add up each other's counts, at most,
constexpr int PLAN_FEW_COUNTS = 32768;           // and their counts
constexpr size_t PLAN_LDS = 156 * 1024;

// LDS of one block of nt threads that sorts S slots.
inline size_t plan_one_lds(int nt, int64_t S, int E) { return ((size_t)(nt / 64 + 1) * E + (size_t)S) * sizeof(uint32_t); }

struct PlanArgs {
    const int32_t* ids;
    int64_t S;
    int k, E;
    int64_t chunk;                      // slots per block, a multiple of PLAN_TILE
    int blocks;
};

// The block's slots [lo, lo + NT R): experts (-1: none) and ranks within the
// wave; s_cnt[wave][expert] (zero before) gets the waves' counts.
template <int NT, int R, int BITS>
__device__ __forceinline__ void plan_rank(const PlanArgs& A, int64_t lo, int64_t hi, uint32_t* s_cnt, int (&e)[R],
                                          uint32_t (&rank)[R]) {
    const int lane = threadIdx.x & 63;
    uint32_t* own = s_cnt + threadIdx.x / 64 * A.E;
    const int64_t s0 = lo + (int64_t)(threadIdx.x / 64) * 64 * R + lane;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        e[r] = s0 + r * 64 < hi ? A.ids[s0 + r * 64] : -1;
        if (e[r] >= A.E) e[r] = -1;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const bool ok = e[r] >= 0;
        uint64_t same = __ballot(ok);
#pragma unroll
        for (int i = 0; i < BITS; ++i) {
            const uint64_t one = __ballot(e[r] >> i & 1);
            same &= one ^ ((uint64_t)(e[r] >> i & 1) - 1ull);
        }
        // the last of the lanes with one expert counts them; a wave's LDS
        // accesses are done in order, so the R counts need not wait for each other
        const int last = ok ? 63 - __clzll((long long)same) : lane;
        uint32_t so_far = 0;
        if (ok && lane == last) so_far = atomicAdd(&own[e[r]], (uint32_t)__popcll(same));
        rank[r] = (uint32_t)__shfl((int)so_far, last) + (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
    }
}

// Exclusive prefix of v over the block's threads; s: NT / 64 words.
template <int NT>
__device__ __forceinline__ uint32_t plan_scan(uint32_t v, uint32_t* s, uint32_t* total) {
    constexpr int W = NT / 64;
    const int lane = threadIdx.x & 63, w = threadIdx.x / 64;
    uint32_t t = v;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const uint32_t o = (uint32_t)__shfl_up((int)t, m);
        if (lane >= m) t += o;
    }
    __syncthreads();
    if (lane == 63) s[w] = t;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        before += i < w ? s[i] : 0u;
        all += s[i];
    }
    *total = all;
    return before + t - v;
}

__global__ void __launch_bounds__(PLAN_NT) k_plan_count(PlanArgs A, uint32_t* __restrict__ cnt) {
    extern __shared__ uint32_t s_cnt[];
    const int64_t lo = blockIdx.x * A.chunk, hi = min(A.S, lo + A.chunk);
    for (int e = threadIdx.x; e < A.E; e += PLAN_NT) s_cnt[e] = 0;
    __syncthreads();
    for (int64_t s = lo + threadIdx.x; s < hi; s += PLAN_TILE) {
        int e[PLAN_R];
#pragma unroll
        for (int r = 0; r < PLAN_R; ++r) e[r] = s + r * PLAN_NT < hi ? A.ids[s + r * PLAN_NT] : -1;
#pragma unroll
        for (int r = 0; r < PLAN_R; ++r)
            if (e[r] >= 0 && e[r] < A.E) atomicAdd(&s_cnt[e[r]], 1u);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < A.E; e += PLAN_NT) cnt[(size_t)e * A.blocks + blockIdx.x] = s_cnt[e];
}

// Expert e = blockIdx.x: its counts over the blocks become a prefix, tot[e] their sum.
__global__ void __launch_bounds__(PLAN_NT) k_plan_scan(PlanArgs A, uint32_t* __restrict__ cnt,
                                                       uint32_t* __restrict__ tot) {
    __shared__ uint32_t s_w[PLAN_NT / 64];
    uint32_t* c = cnt + (size_t)blockIdx.x * A.blocks;
    uint32_t carry = 0;
    for (int b0 = 0; b0 < A.blocks; b0 += PLAN_NT) {
        const int b = b0 + threadIdx.x;
        const uint32_t v = b < A.blocks ? c[b] : 0u;
        uint32_t all;
        const uint32_t p = plan_scan<PLAN_NT>(v, s_w, &all);
        if (b < A.blocks) c[b] = carry + p;
        carry += all;
    }
    if (threadIdx.x == 0) tot[blockIdx.x] = carry;
}

// ONE: the only block, whose own counts are all there is; else after k_plan_scan,
// or, tot NULL, from all blocks' counts as they are.
template <int NT, int R, int BITS, bool ONE>
__global__ void __launch_bounds__(NT) k_plan_place(PlanArgs A, const uint32_t* __restrict__ cnt,
                                                   const uint32_t* __restrict__ tot, int32_t* __restrict__ offsets,
                                                   int32_t* __restrict__ slots, int32_t* __restrict__ rows) {
    extern __shared__ uint32_t s_cnt[];          // [waves][E], then the experts' next places [E]
    __shared__ uint32_t s_w[NT / 64];
    constexpr int W = NT / 64;
    uint32_t* s_next = s_cnt + W * A.E;
    int32_t* s_out = (int32_t*)(s_next + A.E);   // ONE: the sorted slots, which leave in whole lines
    const int64_t lo = blockIdx.x * A.chunk, hi = min(A.S, lo + A.chunk);
    uint32_t carry = 0;
    auto experts_places = [&]() {
        for (int e0 = 0; e0 < A.E; e0 += NT) {
            const int e = e0 + threadIdx.x;
            uint32_t mine = 0, before = 0, all;
            if (e < A.E) {
                if (ONE) {
                    for (int w = 0; w < W; ++w) mine += s_cnt[w * A.E + e];
                } else {
                    const uint32_t* c = cnt + (size_t)e * A.blocks;
                    if (tot) {
                        mine = tot[e];
                        before = c[blockIdx.x];
                    } else {
#pragma unroll 8
                        for (int b = 0; b < A.blocks; ++b) {
                            mine += c[b];
                            before += b < (int)blockIdx.x ? c[b] : 0u;
                        }
                    }
                }
            }
            const uint32_t at = carry + plan_scan<NT>(mine, s_w, &all);
            carry += all;
            if (e < A.E) {
                if (blockIdx.x == 0) offsets[e] = (int32_t)at;
                s_next[e] = at + before;
            }
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) offsets[A.E] = (int32_t)carry;
    };
    if (!ONE) experts_places();
    int64_t t0 = lo;
    do {
        __syncthreads();
        for (int i = threadIdx.x; i < W * A.E; i += NT) s_cnt[i] = 0;
        __syncthreads();
        int e[R];
        uint32_t rank[R];
        plan_rank<NT, R, BITS>(A, t0, hi, s_cnt, e, rank);
        __syncthreads();
        if (ONE) {
            experts_places();
            __syncthreads();
        }
        for (int x = threadIdx.x; x < A.E; x += NT) {
            uint32_t at = s_next[x];
            for (int w = 0; w < W; ++w) {
                const uint32_t c = s_cnt[w * A.E + x];
                s_cnt[w * A.E + x] = at;
                at += c;
            }
            s_next[x] = at;
        }
        __syncthreads();
        const int64_t s0 = t0 + (int64_t)(threadIdx.x / 64) * 64 * R + (threadIdx.x & 63);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (e[r] >= 0) {
                const uint32_t at = s_cnt[threadIdx.x / 64 * A.E + e[r]] + rank[r];
                const int32_t s = (int32_t)(s0 + r * 64);
                if (ONE) {
                    s_out[at] = s;
                } else {
                    slots[at] = s;
                    rows[at] = (int32_t)((uint32_t)s / (uint32_t)A.k);
                }
            }
        t0 += NT * R;
    } while (t0 < hi);
    if (ONE) {
        __syncthreads();
        for (int i = threadIdx.x; i < (int)carry; i += NT) {
            slots[i] = s_out[i];
            rows[i] = (int32_t)((uint32_t)s_out[i] / (uint32_t)A.k);
        }
    }
    // the places that no slot takes
    for (int64_t i = max(lo, (int64_t)carry) + threadIdx.x; i < hi; i += NT) slots[i] = rows[i] = -1;
}

inline PlanArgs plan_args(int64_t S, int k, int E) {
    PlanArgs A = {};
    A.S = S;
    A.k = k;
    A.E = E;
    if (S <= PLAN_ONE && plan_one_lds(1024, S, E) <= PLAN_LDS) {
        A.chunk = PLAN_ONE;
        A.blocks = 1;
        return A;
    }
    const int64_t chunk = (S + PLAN_BLOCKS - 1) / PLAN_BLOCKS;
    A.chunk = (chunk + PLAN_TILE - 1) / PLAN_TILE * PLAN_TILE;
    A.blocks = (int)((S + A.chunk - 1) / A.chunk);
    return A;
}

template <int BITS>
void run_plan(const PlanArgs& A, uint32_t* cnt, int32_t* offsets, int32_t* slots, int32_t* rows, hipStream_t st) {
    auto lds = [&](int nt) { return (size_t)(nt / 64 + 1) * A.E * sizeof(uint32_t); };
    if (A.blocks > 1) {
        uint32_t* tot = cnt + (size_t)A.blocks * A.E;
        k_plan_count<<<A.blocks, PLAN_NT, (size_t)A.E * sizeof(uint32_t), st>>>(A, cnt);
        const bool scan = A.blocks > PLAN_FEW || A.blocks * A.E > PLAN_FEW_COUNTS;
        if (scan) k_plan_scan<<<A.E, PLAN_NT, 0, st>>>(A, cnt, tot);
        k_plan_place<PLAN_NT, PLAN_R, BITS, false>
            <<<A.blocks, PLAN_NT, lds(PLAN_NT), st>>>(A, cnt, scan ? tot : nullptr, offsets, slots, rows);
    } else {
        auto one = [&](auto nt, auto r) {
            constexpr int NT = decltype(nt)::value, R = decltype(r)::value;
            k_plan_place<NT, R, BITS, true><<<1, NT, plan_one_lds(NT, A.S, A.E), st>>>(A, nullptr, nullptr, offsets, slots, rows);
        };
        if (A.S <= 256) one(std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
        else one(std::integral_constant<int, 1024>(), std::integral_constant<int, PLAN_ONE / 1024>());
    }
}

// f with (G, NV) as constants for E experts.
template <typename F>
void route_shape(int E, const F& f) {
#define YABT_SHAPE(g, nv) \
    if (E <= g * nv) return f(std::integral_constant<int, g>(), std::integral_constant<int, nv>());
    YABT_SHAPE(16, 1)
    YABT_SHAPE(16, 2)
    YABT_SHAPE(16, 4)
    YABT_SHAPE(16, 8)
    YABT_SHAPE(16, 16)
    YABT_SHAPE(64, 8)
    YABT_SHAPE(64, 16)
#undef YABT_SHAPE
}

template <int SCORES>
void run_route(const RouteArgs& A, const void* logits, const float* bias, int32_t* ids, float* weights,
               hipStream_t stream) {
    route_shape(A.E, [&](auto g, auto nv) {
        constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
        const int grid = launch_grid(A.n, ROUTE_NT / G, 4096);
        auto go = [&](auto groups, auto merge) {
            k_route<G, NV, SCORES, decltype(groups)::value, decltype(merge)::value>
                <<<grid, ROUTE_NT, 0, stream>>>(A, logits, bias, ids, weights);
        };
        const int q = A.per_group % NV == 0 ? A.per_group / NV : 0;
        const int kind = A.groups == 1 ? 0 : q >= 1 && q <= G && (q & (q - 1)) == 0 ? 1 : 2;
        auto by_groups = [&](auto merge) {
            if (kind == 0) go(std::integral_constant<int, 0>(), merge);
            else if (kind == 1) go(std::integral_constant<int, 1>(), merge);
            else go(std::integral_constant<int, 2>(), merge);
        };
        if constexpr (NV >= 8) {
            if (A.k <= 8) return by_groups(std::true_type());
        }
        by_groups(std::false_type());
    });
}

template <typename T>
void run_route_grad(const RouteArgs& A, const float* dweights, int64_t lddw, const T* logits, const int32_t* ids,
                    T* dlogits, int64_t lddl, hipStream_t stream) {
    route_shape(A.E, [&](auto g, auto nv) {
        constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
        k_route_grad<T, G, NV><<<launch_grid(A.n, ROUTE_NT / G, 4096), ROUTE_NT, 0, stream>>>(
            A, dweights, lddw, logits, ids, dlogits, lddl);
    });
}

}  // namespace yabt

using namespace yabt;

extern "C" {

int yabt_route(int dtype, const void* logits, int64_t ldl, int64_t n, int E, int k, int scores, const float* bias,
               int groups, int keep_groups, int renormalise, float scale, int32_t* out_ids, float* out_weights,
               yabt_stream_t stream) {
    if (!dtype_ok(dtype)) return fail(-1, "yabt_route: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (n < 0 || E < 1 || E > ROUTE_MAX_E || ldl < E) return fail(-1, "yabt_route: bad sizes (1 <= E <= 1024)");
    if (k < 1 || k > ROUTE_MAX_K || k > E) return fail(-1, "yabt_route: 1 <= k <= min(E, 32)");
    if (scores != SOFTMAX && scores != SIGMOID) return fail(-1, "yabt_route: scores is 0 (softmax) or 1 (sigmoid)");
    if (groups < 1 || groups > ROUTE_MAX_GROUPS || E % groups != 0 || keep_groups < 1 || keep_groups > groups)
        return fail(-1, "yabt_route: groups (at most 64) divide E, 1 <= keep_groups <= groups");
    if (n == 0) return 0;
    if (!logits || !out_ids || !out_weights) return fail(-1, "yabt_route: null pointer");
    RouteArgs A = {ldl, n, E, k, scores, renormalise, keep_groups < groups ? groups : 1, keep_groups, E / groups, 0, scale, dtype};
    A.magic = ((1 << 20) + A.per_group - 1) / A.per_group;
    hipStream_t st = (hipStream_t)stream;
    if (scores == SOFTMAX) run_route<SOFTMAX>(A, logits, bias, out_ids, out_weights, st);
    else run_route<SIGMOID>(A, logits, bias, out_ids, out_weights, st);
    return launch_status("yabt_route");
}

int yabt_route_grad(int dtype, const float* dweights, int64_t lddw, const void* logits, int64_t ldl,
                    const int32_t* ids, int64_t n, int E, int k, int scores, int renormalise, float scale,
                    void* out_dlogits, int64_t lddl, yabt_stream_t stream) {
    if (!dtype_ok(dtype)) return fail(-1, "yabt_route_grad: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (n < 0 || E < 1 || E > ROUTE_MAX_E || ldl < E || lddl < E)
        return fail(-1, "yabt_route_grad: bad sizes (1 <= E <= 1024)");
    if (k < 1 || k > ROUTE_MAX_K || k > E || lddw < k) return fail(-1, "yabt_route_grad: 1 <= k <= min(E, 32)");
    if (scores != SOFTMAX && scores != SIGMOID)
        return fail(-1, "yabt_route_grad: scores is 0 (softmax) or 1 (sigmoid)");
    if (n == 0) return 0;
    if (!dweights || !logits || !ids || !out_dlogits) return fail(-1, "yabt_route_grad: null pointer");
    RouteArgs A = {ldl, n, E, k, scores, renormalise, 1, 1, E, 0, scale, dtype};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DT_F32)
        run_route_grad<float>(A, dweights, lddw, (const float*)logits, ids, (float*)out_dlogits, lddl, st);
    else if (dtype == DT_BF16)
        run_route_grad<bf16>(A, dweights, lddw, (const bf16*)logits, ids, (bf16*)out_dlogits, lddl, st);
    else
        run_route_grad<f16>(A, dweights, lddw, (const f16*)logits, ids, (f16*)out_dlogits, lddl, st);
    return launch_status("yabt_route_grad");
}

size_t yabt_expert_plan_workspace_bytes(int64_t n, int k, int E) {
    if (n < 0 || k < 1 || E < 1 || E > ROUTE_MAX_E || n > INT32_MAX / k) return 0;
    const PlanArgs A = plan_args(n * k, k, E);
    return ((size_t)A.blocks + 1) * (size_t)E * sizeof(uint32_t);
}

int yabt_expert_plan(const int32_t* ids, int64_t n, int k, int E, void* workspace, size_t workspace_bytes,
                     int32_t* out_offsets, int32_t* out_slots, int32_t* out_rows, yabt_stream_t stream) {
    const size_t need = yabt_expert_plan_workspace_bytes(n, k, E);
    if (need == 0) return fail(-1, "yabt_expert_plan: bad sizes (1 <= E <= 1024, n k < 2^31)");
    if (!workspace || workspace_bytes < need) return fail(-2, "yabt_expert_plan: workspace too small");
    if (!out_offsets || (n > 0 && (!ids || !out_slots || !out_rows)))
        return fail(-1, "yabt_expert_plan: null pointer");
    PlanArgs A = plan_args(n * k, k, E);
    A.ids = ids;
    hipStream_t st = (hipStream_t)stream;
    if (E <= 16) run_plan<4>(A, (uint32_t*)workspace, out_offsets, out_slots, out_rows, st);
    else if (E <= 64) run_plan<6>(A, (uint32_t*)workspace, out_offsets, out_slots, out_rows, st);
    else if (E <= 256) run_plan<8>(A, (uint32_t*)workspace, out_offsets, out_slots, out_rows, st);
    else run_plan<10>(A, (uint32_t*)workspace, out_offsets, out_slots, out_rows, st);
    return launch_status("yabt_expert_plan");
}

}  // extern "C"
