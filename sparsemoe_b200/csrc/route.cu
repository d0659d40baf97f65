// Expert routing from given logits: scores, balance bias, expert groups, top-k, weights.
//
// Per token, x_e the logit of expert e (converted to f32 exactly):
//   s_e = 1 / (1 + exp(-x_e))  or  exp(x_e - max) / sum_j exp(x_j - max);
//   v_e = s_e + b_e with a selection bias, else x_e (both scores grow with
//         the logit, so the logits give the same order and never saturate);
//   groups of E/G neighbours, each scored by its largest v (no bias: x) or by
//         the sum of its two largest v (no bias: s); the `kept` best stay;
//   the k largest v of the kept groups, equal values by the lower index;
//   w_l = s / sum over the chosen of s (renormalised; where every chosen
//         sigmoid is tiny, exp(x - max) in its place, its limit) or s, times scale.
// Masked experts (NaN, logits <= -1e20 or f16's lowest value, a bias that is
// NaN or <= -1e20) are never chosen; slots that stay empty hold (-1, 0).
//
// The order is that of f64 arithmetic.  The selection runs on 32-bit keys, the
// value's order-preserving bits with the expert's index in the low ones, which
// makes every key unique and a tie fall to the lower index.  f32 scores carry an
// error bound and the index takes low bits of the value, so where two neighbours
// of the order are closer than both, the candidates (the chosen and what is that
// close behind them) are ranked again, one a lane, by their f64 values; where the
// last kept and the first left group are, the whole row is selected in f64, and
// group sums that agree to 2^-49 of what they are summed from are ties (sigmoid(x) +
// sigmoid(-x) is 1 for every x).  16-bit logits without a bias give up only zeros and need neither.
//
// One warp per token, lane l holding experts l*NV .. l*NV + NV - 1.  Each lane
// sorts its keys once; a round of the selection is one redux.sync over the
// lanes' first keys and a pop in the lane that has it.
#include "moe_internal.h"
#include "common.cuh"

namespace moe {
namespace {

constexpr int kRouteWarps = 4;
constexpr unsigned kFull = 0xffffffffu;

struct RouteParams {
    const void* x;
    int64_t T, ld;
    int E, k;
    int sigmoid;            // else softmax
    int G, per, kept, group_top;
    int lanes;              // > 0: a group is this many whole lanes (a power of two)
    int sub;                // else: lanes that share the pass over one group (0: G > 32, left to the f64 path)
    int renorm;
    float scale;
    const float* bias;
    int* idx;
    float* w;
    int vec, vec_bias;      // rows / the bias allow the vector loads
};

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

constexpr float kMasked = -1e20f;   // as in the layer's own gate
template <typename T> __device__ __forceinline__ bool selectable(float x) {
    return x > (sizeof(T) == 2 && std::is_same<T, __half>::value ? -65504.0f : kMasked);
}

__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);   // -0 and +0 are a tie
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}
__device__ __forceinline__ unsigned long long order_key(double v) {
    const unsigned long long u = __double_as_longlong(v + 0.0);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double key_value(unsigned long long key) {
    return __longlong_as_double((key >> 63) ? (key & 0x7FFFFFFFFFFFFFFFull) : ~key);
}

__device__ __forceinline__ float warp_max(float v) { return key_value(__reduce_max_sync(kFull, order_key(v))); }
__device__ __forceinline__ double warp_max(double v) {
    const unsigned long long k = order_key(v);
    const uint32_t hi = __reduce_max_sync(kFull, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(kFull, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return key_value((unsigned long long)hi << 32 | lo);
}
template <typename V> __device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

// Two largest of a set, merged with another set's (a >= b in each).
template <typename V> __device__ __forceinline__ void merge2(V& a, V& b, V c, V d) {
    const V lo = fmin(a, c);
    a = fmax(a, c);
    b = fmax(lo, fmax(b, d));
}

// Descending in-register sort (odd-even merge network, NV a power of two).
template <int NV> __device__ __forceinline__ void sort_desc(uint32_t (&k)[NV]) {
#pragma unroll
    for (int p = 1; p < NV; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < NV; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < NV && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const uint32_t hi = max(k[i + j], k[i + j + q]);
                        k[i + j + q] = min(k[i + j], k[i + j + q]);
                        k[i + j] = hi;
                    }
}

template <typename T, int NV>
__device__ __forceinline__ void load_row(const T* row, int e0, int E, bool vec, float (&x)[NV]) {
    constexpr int kBytes = NV * (int)sizeof(T);
    constexpr int kVec = kBytes % 16 == 0 ? 16 : kBytes % 8 == 0 ? 8 : kBytes % 4 == 0 ? 4 : 2;
    if (kVec > (int)sizeof(T) && vec && e0 + NV <= E) {
        union { T v[NV]; uint4 q[(kBytes + 15) / 16]; uint2 d[(kBytes + 7) / 8]; uint32_t u[(kBytes + 3) / 4]; } r;
        if constexpr (kVec == 16) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) r.q[i] = reinterpret_cast<const uint4*>(row + e0)[i];
        } else if constexpr (kVec == 8) {
#pragma unroll
            for (int i = 0; i < kBytes / 8; ++i) r.d[i] = reinterpret_cast<const uint2*>(row + e0)[i];
        } else if constexpr (kVec == 4) {
#pragma unroll
            for (int i = 0; i < kBytes / 4; ++i) r.u[i] = reinterpret_cast<const uint32_t*>(row + e0)[i];
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) x[i] = to_f32<T>(r.v[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = e0 + i < E ? to_f32<T>(row[e0 + i]) : -INFINITY;
}

// The f64 passes of single rows, rare and therefore small in code and registers
// (a function that is called takes its registers in every warp of the kernel):
// values lie in shared memory, lane l looks at experts l, l + 32, ...

// buf[e] = what orders expert e (members: what scores its group), -infinity if masked.
template <typename T>
__device__ __forceinline__ void values_f64(const RouteParams& p, const T* row, double* buf, int lane, bool members) {
    const bool scores = p.bias || (members && p.group_top == 2);
    double top = -INFINITY, sum = 0.0;
#pragma unroll 1
    for (int e = lane; e < p.E; e += 32) {
        const float x = to_f32<T>(row[e]);
        const double v = selectable<T>(x) ? (double)x : -INFINITY;
        top = fmax(top, v);
        buf[e] = v;
    }
    if (!scores) return;
    top = warp_max(top);
#pragma unroll 1
    for (int e = lane; e < p.E; e += 32) {
        const double x = buf[e];
        const double u = p.sigmoid ? exp(-x) : x == top ? 1.0 : exp(x - top);
        sum += x == -INFINITY ? 0.0 : u;
        buf[e] = x == -INFINITY ? x : u;
    }
    sum = warp_sum(sum);
#pragma unroll 1
    for (int e = lane; e < p.E; e += 32) {
        const double u = buf[e];
        if (u == -INFINITY) continue;
        double v = p.sigmoid ? 1.0 / (1.0 + u) : u / sum;
        if (p.bias) {
            const float b = p.bias[e];
            v = b > kMasked ? v + (double)b : -INFINITY;
        }
        buf[e] = v;
    }
}

// Group sums of two are equal where they agree to 2^-49 of what they are summed
// from, the members' values and biases: sigmoid(x) + sigmoid(-x) is 1 for every x,
// which f64 leaves within a few 2^-53 of their sizes, while the order of scores of
// any size stands.  a, b: the two best members, bias: the largest magnitude of
// theirs.
__device__ __forceinline__ double group_tie(bool pair, double a, double b, float bias) {
    if (!pair || isinf(a)) return 0.0;
    return 0x1p-49 * (fabs(a) + (b == -INFINITY ? 0.0 : fabs(b)) + 2.0 * fabs((double)bias));
}

// Best members a, b of group g and the largest bias of theirs, from lanes lane % sub
// of sub that share it (all get them).
__device__ __forceinline__ void group_best(const RouteParams& p, const double* buf, int g, int first, int sub, double& a,
                                           double& b, float& bias) {
    a = b = -INFINITY;
    bias = 0.0f;
    if (g < p.G)
#pragma unroll 1
        for (int i = first; i < p.per; i += sub) merge2(a, b, buf[g * p.per + i], (double)-INFINITY);
#pragma unroll 1
    for (int o = sub >> 1; o > 0; o >>= 1) {
        const double c = __shfl_xor_sync(kFull, a, o), d = __shfl_xor_sync(kFull, b, o);
        merge2(a, b, c, d);
    }
    if (p.bias == nullptr || p.group_top != 2) return;
    if (g < p.G)
#pragma unroll 1
        for (int i = first; i < p.per; i += sub) {
            const double v = buf[g * p.per + i];
            if (v >= b && v != -INFINITY) bias = fmaxf(bias, fabsf(p.bias[g * p.per + i]));
        }
#pragma unroll 1
    for (int o = sub >> 1; o > 0; o >>= 1) bias = fmaxf(bias, __shfl_xor_sync(kFull, bias, o));
}

// Which of up to 32 groups of a row stay: bit g.  buf: E doubles of this warp's
// shared memory.  Chosen one by one: the lowest of those that equal the largest.
template <typename T>
__device__ __noinline__ uint32_t groups_f64(const RouteParams& p, const T* row, double* buf, int lane) {
    __syncwarp();
    values_f64<T>(p, row, buf, lane, true);
    __syncwarp();
    const bool pair = p.group_top == 2;
    int sub = 32;
    while (32 / sub < p.G) sub >>= 1;
    double a, b;
    float bias;
    group_best(p, buf, lane / sub, lane % sub, sub, a, b, bias);
    double tie = group_tie(pair, a, b, bias);
    if (pair && b != -INFINITY) a += b;
    a = __shfl_sync(kFull, a, (lane * sub) & 31);   // lane g: group g
    tie = __shfl_sync(kFull, tie, (lane * sub) & 31);
    if (lane >= p.G) a = -INFINITY;
    uint32_t stay = 0;
#pragma unroll 1
    for (int r = 0; r < p.kept; ++r) {
        const double m = warp_max(a);
        if (m == -INFINITY) break;
        const double from = -warp_max(a == m ? tie - a : -INFINITY);
        const uint32_t at = __reduce_min_sync(kFull, a != -INFINITY && a + tie >= from ? lane : 32);
        stay |= 1u << at;
        if (lane == (int)at) a = -INFINITY;
    }
    __syncwarp();
    return stay;
}

// The whole selection of one row.  Returns the lane's choice (lane l: the l-th) or -1.
template <typename T>
__device__ __noinline__ int route_row_f64(const RouteParams& p, const T* row, double* buf, int lane) {
    uint32_t keep = kFull;   // lane l, bit i: group l + 32 i
    if (p.G > 32) {
        __syncwarp();
        values_f64<T>(p, row, buf, lane, true);
        __syncwarp();
        const bool pair = p.group_top == 2;
        double gs[32], ties[32];
        const int gn = (p.G + 31) / 32;
#pragma unroll 1
        for (int i = 0; i < gn; ++i) {
            double a, b;
            float bias;
            group_best(p, buf, lane + 32 * i, 0, 1, a, b, bias);
            ties[i] = group_tie(pair, a, b, bias);
            gs[i] = pair && b != -INFINITY ? a + b : a;
        }
        keep = 0;
#pragma unroll 1
        for (int r = 0; r < p.kept; ++r) {
            double a = -INFINITY;
            for (int i = 0; i < gn; ++i) a = fmax(a, gs[i]);
            const double m = warp_max(a);
            if (m == -INFINITY) break;
            double from = -INFINITY;
            for (int i = 0; i < gn; ++i)
                if (gs[i] == m) from = fmax(from, ties[i] - m);
            from = -warp_max(from);
            uint32_t at = 0xFFFFFFFFu;
            for (int i = gn - 1; i >= 0; --i)
                if (gs[i] != -INFINITY && gs[i] + ties[i] >= from) at = lane + 32 * i;
            at = __reduce_min_sync(kFull, at);
            if ((at & 31) == lane) {
                keep |= 1u << (at >> 5);
                gs[at >> 5] = -INFINITY;
            }
        }
    } else if (p.G > 1) {
        keep = groups_f64<T>(p, row, buf, lane) >> lane & 1;
    }
    __syncwarp();
    values_f64<T>(p, row, buf, lane, false);
    if (p.G > 1)
#pragma unroll 1
        for (int e0 = 0; e0 < p.E; e0 += 32) {
            const int e = e0 + lane, g = min(e, p.E - 1) / p.per;
            if (!(__shfl_sync(kFull, keep, g & 31) >> (g >> 5) & 1) && e < p.E) buf[e] = -INFINITY;
        }
    int mine = -1;
#pragma unroll 1
    for (int l = 0; l < p.k; ++l) {
        double a = -INFINITY;
        for (int e = lane; e < p.E; e += 32) a = fmax(a, buf[e]);
        const double m = warp_max(a);
        if (m == -INFINITY) break;
        uint32_t at = 0xFFFFFFFFu;
        for (int e = lane; e < p.E; e += 32)
            if (buf[e] == m && at == 0xFFFFFFFFu) at = e;
        at = __reduce_min_sync(kFull, at);
        if ((int)(at & 31) == lane) buf[at] = -INFINITY;
        if (lane == l) mine = (int)at;
    }
    return mine;
}

// exp(x): ex2.approx of the rounded x log2(e), (2 + 1.2 |x|) 2^-23 relative
// (results below 2^-126 become 0).
__device__ __forceinline__ float exp_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
    return r;
}
__device__ __forceinline__ float rcp_fast(float x) {   // 1 ulp
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 1 / (1 + exp(-x)), its small values (exp(x) / (1 + exp(x))) down to the subnormal ones.
__device__ __forceinline__ float sigmoid(float x) {
    const float t = expf(-fabsf(x)), r = rcp_fast(1.0f + t);
    return x < 0.0f ? t * r : r;
}
// Up to this sum of sigmoids exp(x - max) stands for them: sigmoid(x) is exp(x)
// (1 - exp(x) + ..), off by less than 2^-26, and no score that counts beside the
// largest underflows.
constexpr float kSmallSum = 0x1p-26f;

// The candidates in lanes 0 .. n-1 (n >= k, or fewer where nothing else is
// left) ranked by value, equal values by the lower index: lane l gets the l-th.
// f32 values decide where those that follow each other, down to the first behind
// the k-th, are further apart than their error (logits themselves are exact);
// else f64 values do.  top, inv_sum: the softmax's statistics; buf: 64 words.
template <typename T>
__device__ __noinline__ int rank_candidates(const RouteParams& p, const T* row, float top, float inv_sum, float err2,
                                            int cand, int n, int* buf, int lane) {
    const float x = lane < n ? to_f32<T>(row[cand]) : 0.0f;
    const float b = p.bias && lane < n ? p.bias[cand] : 0.0f;
    float f = x;
    if (p.bias) f = (p.sigmoid ? rcp_fast(1.0f + exp_fast(-x)) : (x == top ? 1.0f : exp_fast(x - top)) * inv_sum) + b;
    int rank = 0;
    for (int j = 0; j < n; ++j) {
        const float o = __shfl_sync(kFull, f, j);
        const int e = __shfl_sync(kFull, cand, j);
        rank += o > f || (o == f && e < cand) ? 1 : 0;
    }
    __syncwarp();
    if (lane < n) {
        buf[rank] = cand;
        buf[32 + rank] = __float_as_int(f);
    }
    __syncwarp();
    if (!p.bias) return lane < n ? buf[lane] : -1;
    const float hi = __int_as_float(buf[32 + min(lane, n - 1)]), lo = __int_as_float(buf[32 + min(lane + 1, n - 1)]);
    const bool close = !(hi - lo > err2 + 3e-7f * fmaxf(fabsf(hi), fabsf(lo)));
    if (!__any_sync(kFull, lane + 1 < n && lane < p.k && close)) return lane < n ? buf[lane] : -1;
    double v;
    if (p.sigmoid) {
        v = 1.0 / (1.0 + exp(-(double)x)) + (double)b;
    } else {
        double sum = 0.0;
#pragma unroll 1
        for (int e = lane; e < p.E; e += 32) {
            const float o = to_f32<T>(row[e]);
            if (selectable<T>(o)) sum += o == top ? 1.0 : exp((double)o - (double)top);
        }
        sum = warp_sum(sum);
        v = (x == top ? 1.0 : exp((double)x - (double)top)) / sum + (double)b;
    }
    rank = 0;
    for (int j = 0; j < n; ++j) {
        const double o = __shfl_sync(kFull, v, j);
        const int e = __shfl_sync(kFull, cand, j);
        rank += o > v || (o == v && e < cand) ? 1 : 0;
    }
    __syncwarp();
    if (lane < n) buf[rank] = cand;
    __syncwarp();
    return lane < n ? buf[lane] : -1;
}

// What a group's score, a or the sum of its two best members a and b, may be off
// by in f32: err2 for the members' scores, 2^-24 each for the members (of their
// own sizes, which biases of both signs leave in a small sum), the sum, and the
// addition of this slack to it.
__device__ __forceinline__ float group_slack(float a, float b, float err2) {
    const float size = fabsf(a) + (b == -INFINITY ? 0.0f : fabsf(b));
    return size < INFINITY ? err2 + 2.5e-7f * size : 0.0f;
}

template <typename T, int NV>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const __grid_constant__ RouteParams p) {
    constexpr uint32_t kIdx = 32 * NV - 1;      // the key bits that hold the index
    __shared__ double sv[kRouteWarps][NV * 32];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t t = (int64_t)blockIdx.x * kRouteWarps + warp;
    if (t >= p.T) return;
    const T* row = static_cast<const T*>(p.x) + t * p.ld;
    const int e0 = lane * NV;
    float v[NV];
    load_row<T, NV>(row, e0, p.E, p.vec != 0, v);
#pragma unroll
    for (int q = 0; q < NV; ++q) v[q] = selectable<T>(v[q]) ? v[q] : -INFINITY;

    const bool pair = p.group_top == 2;         // (one group has group_top 1)
    // 16-bit logits without a bias: at most 10 of 13 zero bits are given up
    const bool exact = p.bias == nullptr && sizeof(T) == 2;
    float top = 0.0f, inv_sum = 1.0f;
    float s[NV];
    if (p.sigmoid) {
        if (p.bias || pair)
#pragma unroll
            for (int q = 0; q < NV; ++q) s[q] = rcp_fast(1.0f + exp_fast(-v[q]));
    } else if (p.bias || pair || !p.renorm) {
        top = v[0];
#pragma unroll
        for (int q = 1; q < NV; ++q) top = fmaxf(top, v[q]);
        top = warp_max(top);
        float sum = 0.0f;
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            s[q] = v[q] == top ? 1.0f : exp_fast(v[q] - top);
            sum += s[q];
        }
        sum = warp_sum(sum);
        inv_sum = 1.0f / sum;
#pragma unroll
        for (int q = 0; q < NV; ++q) s[q] *= inv_sum;
    }
    if (p.bias) {
        float b[NV];
        load_row<float, NV>(p.bias, e0, p.E, p.vec_bias != 0, b);
#pragma unroll
        for (int q = 0; q < NV; ++q) v[q] = v[q] > -INFINITY && b[q] > kMasked ? s[q] + b[q] : -INFINITY;
    }
    // Bound of the error in a difference of two scores, in units of 2^-23.  The
    // sigmoid's error is at most 0.65 (of exp, times s (1 - s)) + 0.5 + 1 (of 1 + e
    // and rcp), 5 units for two.  The softmax's is in units of its largest score
    // 35: the sum's relative error, 18 (36 additions of half a unit) + 7 (of its
    // exps, 2 + 1.2 d for a logit d below the largest: weighted by e^-d over 1024
    // experts their mean is at most 7) + 0.5 (1 / sum), is one factor of the whole
    // row and counts once; the two scores' own exps add at most 2 each (e^-d (2 +
    // 1.2 d) falls with d), their products half each.  30.5 in all.
    const float err2 = p.sigmoid ? 6e-7f : 4.2e-6f * inv_sum;

    bool redo = false;                          // the whole row in f64
    if (p.G > 1) {
        const bool scored = p.bias || pair;
        float m[NV];
#pragma unroll
        for (int q = 0; q < NV; ++q) m[q] = v[q];
        if (pair && !p.bias)
#pragma unroll
            for (int q = 0; q < NV; ++q) m[q] = v[q] == -INFINITY ? v[q] : s[q];
        float a = -INFINITY, b = -INFINITY;
        int g;
        if (p.lanes > 0) {
            g = lane / p.lanes;
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                b = fmaxf(b, fminf(a, m[q]));
                a = fmaxf(a, m[q]);
            }
            for (int o = p.lanes >> 1; o > 0; o >>= 1) {
                const float c = __shfl_xor_sync(kFull, a, o), d = __shfl_xor_sync(kFull, b, o);
                merge2(a, b, c, d);
            }
        } else {
            float* buf = reinterpret_cast<float*>(sv[warp]);
#pragma unroll
            for (int q = 0; q < NV; ++q) buf[e0 + q] = m[q];
            __syncwarp();
            const int sub = max(p.sub, 1);
            g = lane / sub;
            if (p.sub > 0 && g < p.G)
                for (int i = lane % sub; i < p.per; i += sub) merge2(a, b, buf[g * p.per + i], -INFINITY);
            for (int o = sub >> 1; o > 0; o >>= 1) {
                const float c = __shfl_xor_sync(kFull, a, o), d = __shfl_xor_sync(kFull, b, o);
                merge2(a, b, c, d);
            }
            redo = p.sub == 0;
            __syncwarp();
        }
        bool near = false;
        const float slack = scored ? group_slack(a, b, err2) : 0.0f;
        if (pair && b != -INFINITY) a += b;
        if (g >= p.G) a = -INFINITY;
        const uint32_t gk = a != -INFINITY ? (order_key(a) & ~31u) | (31 - g) : 0u;
        uint32_t cur = gk;
        for (int r = 0; r < p.kept; ++r) {
            const uint32_t best = __reduce_max_sync(kFull, cur);
            if (best == 0) break;
            if (cur == best) cur = 0;
        }
        bool stay = gk != 0 && cur == 0;
        const uint32_t out = __reduce_max_sync(kFull, cur);
        if (out != 0 && (scored || !exact)) {
            // close with the index in the low bits: the scores themselves, as far off as they may be, decide
            const float worst = key_value(__reduce_min_sync(kFull, stay ? order_key(a - slack) : 0xFFFFFFFFu));
            const float other = key_value(__reduce_max_sync(kFull, stay || gk == 0 ? 0u : order_key(a + slack)));
            near = !(worst > other);
        }
        if (near && !redo) {
            const uint32_t mask = groups_f64<T>(p, row, sv[warp], lane);
            stay = g < p.G && (mask >> g & 1);
        }
        if (p.lanes > 0) {
#pragma unroll
            for (int q = 0; q < NV; ++q) v[q] = stay ? v[q] : -INFINITY;
        } else {
            const uint32_t kept = __ballot_sync(kFull, stay);
            int gg = e0 / p.per, r = e0 - gg * p.per;
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                if (e0 + q >= p.E || !((kept >> (gg * p.sub & 31)) & 1)) v[q] = -INFINITY;
                if (++r == p.per) { r = 0; ++gg; }
            }
        }
    }

    uint32_t key[NV];
#pragma unroll
    for (int q = 0; q < NV; ++q) key[q] = v[q] == -INFINITY ? 0u : (order_key(v[q]) & ~kIdx) | (kIdx - (e0 + q));
    sort_desc<NV>(key);
    uint32_t mine = 0;
    int n = 0;
    auto pop = [&](uint32_t best) {
        if (key[0] == best) {
#pragma unroll
            for (int q = 0; q + 1 < NV; ++q) key[q] = key[q + 1];
            key[NV - 1] = 0;
        }
        if (lane == n) mine = best;
    };
    uint32_t best = __reduce_max_sync(kFull, key[0]);
    for (; n < p.k && best != 0; ++n) {
        pop(best);
        best = __reduce_max_sync(kFull, key[0]);
    }
    int my_i = mine != 0 ? (int)(kIdx - (mine & kIdx)) : -1;
    if (!exact && !redo) {
        auto close = [&](uint32_t a, uint32_t b) {   // a >= b, keys that follow each other
            const float hi = key_value(a & ~kIdx), lo = key_value(b & ~kIdx);
            return p.bias ? !(hi - lo > err2 + (32 * NV * 1.2e-7f + 3e-7f) * fmaxf(fabsf(hi), fabsf(lo))) : !(hi > lo);
        };
        uint32_t next = __shfl_down_sync(kFull, mine, 1);
        if (lane == n - 1) next = best;
        if (__any_sync(kFull, lane < n && next != 0 && close(mine, next))) {
            // all that is close behind the last chosen is a candidate too
            uint32_t last = __shfl_sync(kFull, mine, n - 1);
            while (best != 0 && close(last, best) && n < 32) {
                pop(best);
                ++n;
                last = best;
                best = __reduce_max_sync(kFull, key[0]);
            }
            redo = best != 0 && close(last, best);
            if (!redo)
                my_i = rank_candidates<T>(p, row, top, inv_sum, err2, mine != 0 ? (int)(kIdx - (mine & kIdx)) : -1, n,
                                              reinterpret_cast<int*>(sv[warp]), lane);
        }
    }
    if (redo) my_i = route_row_f64<T>(p, row, sv[warp], lane);
    if (lane >= p.k) my_i = -1;

    const float xs = my_i >= 0 ? to_f32<T>(row[my_i]) : -INFINITY;
    float e = 0.0f;
    if (p.sigmoid) {
        e = sigmoid(xs);
    } else if (!p.renorm) {
        e = my_i < 0 ? 0.0f : (xs == top ? 1.0f : expf(xs - top)) * inv_sum;
    }
    if (p.renorm) {
        float sum = 0.0f;
        if (p.sigmoid) sum = warp_sum(e);
        if (!(sum > kSmallSum)) {   // softmax, or sigmoids so small that their ratios are exp of the differences
            const float mx = warp_max(xs);
            e = my_i < 0 ? 0.0f : xs == mx ? 1.0f : expf(xs - mx);
            sum = warp_sum(e);
        }
        e = sum > 0.0f ? e * rcp_fast(sum) : 0.0f;
    }
    if (lane < p.k) {
        p.idx[t * p.k + lane] = my_i;
        p.w[t * p.k + lane] = e * p.scale;
    }
}

// Many tokens: four to a warp, eight lanes each, lane l of a token holding its
// experts l*per .. l*per + per - 1 (per = E / 8: one group, where there are
// eight).  Everything that a round costs a warp is then paid for four tokens, and
// a group's score needs no shuffle.  A lane keeps the eight best of its experts
// in order (sorting networks of eight, merged); k <= 8.  500 warp instructions a
// token for the 880 of a warp a token (256 experts, bias, groups), half of them
// on the half-rate ALU pipe, which bounds both; the chain that a warp runs
// through is longer.  Measured (us, a warp a token / four a warp): 256 experts in
// groups 8192 tokens 11.9 / 14.5, 16384 19.4 / 16.5, 32768 32.3 / 26.7; 64 experts 4096
// tokens 3.2 / 2.9, 16384 7.6 / 4.9, 32768 13.0 / 7.5.
__device__ __forceinline__ uint32_t max8(uint32_t v) {   // over a token's eight lanes
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(kFull, v, o));
    return v;
}
__device__ __forceinline__ float fmax8(float v) {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
    return v;
}
__device__ __forceinline__ double fmax8(double v) {
#pragma unroll 1
    for (int o = 4; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(kFull, v, o));
    return v;
}
__device__ __forceinline__ float sum8(float v) {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

// Four consecutive elements (rows allow it: the host checks).
__device__ __forceinline__ void load4(const float* p, float* x) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
}
template <typename T16> __device__ __forceinline__ void load4(const T16* p, float* x) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    const float2 lo = F16Traits<T16>::unpack2(a.x), hi = F16Traits<T16>::unpack2(a.y);
    x[0] = lo.x; x[1] = lo.y; x[2] = hi.x; x[3] = hi.y;
}

// The eight largest of NV keys, descending, in key[0..8).
template <int NV> __device__ __forceinline__ void top8(uint32_t (&key)[NV]) {
#pragma unroll
    for (int b = 0; b < NV; b += 8) {
        uint32_t t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = key[b + i];
        sort_desc<8>(t);
        if (b == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) key[i] = t[i];
        } else {
            // the larger of a_i and b_(7-i) are the eight largest, in bitonic order
#pragma unroll
            for (int i = 0; i < 8; ++i) key[i] = max(key[i], t[7 - i]);
#pragma unroll
            for (int q = 4; q > 0; q >>= 1)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!(i & q)) {
                        const uint32_t hi = max(key[i], key[i + q]);
                        key[i + q] = min(key[i], key[i + q]);
                        key[i] = hi;
                    }
        }
    }
}

template <typename T, int NV, bool kWhole>   // kWhole: per == NV
__global__ void __launch_bounds__(kRouteWarps * 32, 7) route_many_kernel(const __grid_constant__ RouteParams p) {
    constexpr uint32_t kIdx = NV - 1;           // the key bits that hold the place in the lane
    // per warp: the four rows on their way to the lanes' parts, each part padded by
    // 16 bytes (eight lanes' 16-byte reads fall into different banks); later the
    // f64 passes' space.  Loading the parts directly touched 32 lines an instruction.
    constexpr int kRowFloats = 8 * (NV + 4);
    __shared__ __align__(16) float sx[kRouteWarps][4 * kRowFloats];
    __shared__ __align__(16) float sb[kRowFloats];    // the bias, as a row
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & 7;
    pdl_wait();
    pdl_trigger();
    const int per = kWhole ? NV : p.E / 8, e0 = sub * per;
    const float inv_chunks = 4.0f / (float)per;       // chunks of four: of part (c + 1/2) / (per / 4)
    auto place = [&](int c) { return 4 * c + 4 * (int)(((float)c + 0.5f) * inv_chunks); };
    if (p.bias) {
        for (int c = threadIdx.x; c < 2 * per; c += kRouteWarps * 32) {
            float b[4];
            load4(p.bias + 4 * c, b);
            *reinterpret_cast<float4*>(sb + place(c)) = make_float4(b[0], b[1], b[2], b[3]);
        }
        __syncthreads();
    }
    const int64_t tw = ((int64_t)blockIdx.x * kRouteWarps + warp) * 4, t = tw + (lane >> 3);
    if (tw >= p.T) return;
    const bool live = t < p.T;                  // the last warp's lanes without a token work on its last one
    const T* row = static_cast<const T*>(p.x) + (live ? t : p.T - 1) * p.ld;
    float* const rows = sx[warp] + (lane >> 3) * kRowFloats;
    double* const wide = reinterpret_cast<double*>(sx[warp]);
    float v[NV];
#pragma unroll
    for (int q = 0; q < NV; q += 4)
        if (q < per) load4(row + 4 * (2 * q + sub), v + q);   // chunks sub, sub + 8, ..: 128 bytes of f32 a row
#pragma unroll
    for (int q = 0; q < NV; q += 4)
        if (q < per) *reinterpret_cast<float4*>(rows + place(2 * q + sub)) = make_float4(v[q], v[q + 1], v[q + 2], v[q + 3]);
    __syncwarp();
#pragma unroll
    for (int q = 0; q < NV; q += 4) {
        float4 x = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (q < per) x = *reinterpret_cast<const float4*>(rows + sub * (per + 4) + q);
        v[q] = x.x; v[q + 1] = x.y; v[q + 2] = x.z; v[q + 3] = x.w;
    }
    __syncwarp();
    // Rows without masked experts (the whole warp's) skip the tests of every element.
    float low = INFINITY, sum_all = 0.0f;
#pragma unroll
    for (int q = 0; q < NV; ++q)
        if (q < per) {
            low = fminf(low, v[q]);
            sum_all += v[q];
        }
    bool clean = __all_sync(kFull, selectable<T>(low) && sum_all == sum_all);
    if (!clean) {
#pragma unroll
        for (int q = 0; q < NV; ++q) v[q] = selectable<T>(v[q]) ? v[q] : -INFINITY;
    }

    const bool pair = p.group_top == 2;
    const bool exact = p.bias == nullptr && sizeof(T) == 2;
    float top = 0.0f, inv_sum = 1.0f;
    float a = -INFINITY, b = -INFINITY;         // the lane's two best members (the group's, where there are eight)
    if (!p.sigmoid && (p.bias || pair || !p.renorm)) {
        top = v[0];
#pragma unroll
        for (int q = 1; q < NV; ++q) top = fmaxf(top, v[q]);
        top = fmax8(top);
        float sum = 0.0f;
#pragma unroll
        for (int q = 0; q < NV; ++q) sum += v[q] == top ? 1.0f : exp_fast(v[q] - top);
        inv_sum = 1.0f / sum8(sum);
    }
    auto score = [&](float x) {
        return p.sigmoid ? rcp_fast(1.0f + exp_fast(-x)) : (x == top ? 1.0f : exp_fast(x - top)) * inv_sum;
    };
    if (p.bias) {
        low = INFINITY;
        sum_all = 0.0f;
#pragma unroll
        for (int q = 0; q < NV; q += 4) {
            if (q >= per) continue;
            const float4 b4 = *reinterpret_cast<const float4*>(sb + sub * (per + 4) + q);
            const float bias[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (clean) {
                    v[q + i] = score(v[q + i]) + bias[i];
                    low = fminf(low, v[q + i]);
                    sum_all += v[q + i];
                } else {
                    v[q + i] = v[q + i] > -INFINITY && bias[i] > kMasked ? score(v[q + i]) + bias[i] : -INFINITY;
                }
            }
        }
        if (clean && !__all_sync(kFull, low > 0.1f * kMasked && sum_all == sum_all)) {   // a masking bias
            clean = false;
#pragma unroll
            for (int q = 0; q < NV; ++q)
                if (q < per && !(p.bias[e0 + q] > kMasked)) v[q] = -INFINITY;
        }
    }
    const float err2 = p.sigmoid ? 6e-7f : 4.2e-6f * inv_sum;   // as above
    uint32_t keep = ~kIdx;
    if (p.G > 1) {
        if (!pair) {
#pragma unroll
            for (int q = 0; q < NV; ++q) a = fmaxf(a, v[q]);
        } else {
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                if (q >= per) continue;
                const float m = p.bias || v[q] == -INFINITY ? v[q] : score(v[q]);
                b = fmaxf(b, fminf(a, m));
                a = fmaxf(a, m);
            }
        }
        const float least = pair ? b : a;       // of the members that score the group
        const float slack = group_slack(a, b, err2);
        if (pair && b != -INFINITY) a += b;
        const uint32_t mine = a != -INFINITY ? order_key(a) : 0u;
        int rank = 0;
        bool near = false;
#pragma unroll
        for (int h = 1; h < 8; ++h) {
            const uint32_t other = __shfl_xor_sync(kFull, mine, h);
            rank += other > mine || (other == mine && (sub ^ h) < sub) ? 1 : 0;
        }
        bool stay = mine != 0 && rank < p.kept;
        const uint32_t worst = ~max8(stay ? ~order_key(a - slack) : 0u);
        const uint32_t other = max8(stay || mine == 0 ? 0u : order_key(a + slack));
        near = other != 0 && (p.bias || pair) && !(key_value(worst) > key_value(other));
        unsigned bad = __ballot_sync(kFull, near);
        if (bad != 0 && p.sigmoid) {
            // every lane its group's one or two members in f64, where f32 values tell them from the others
            const float from = least - (err2 + 3e-7f * fabsf(least));
            int first = -1, second = -1, count = 0;
#pragma unroll 4
            for (int q = 0; q < NV; ++q) {
                if (q >= per) break;
                const float x = to_f32<T>(row[e0 + q]);
                float m = selectable<T>(x) ? rcp_fast(1.0f + exp_fast(-x)) : -INFINITY;
                if (p.bias) {
                    const float pb = p.bias[e0 + q];
                    m = pb > kMasked ? m + pb : -INFINITY;
                }
                if (m > -INFINITY && m >= from) {
                    second = count == 1 ? q : second;
                    first = count == 0 ? q : first;
                    ++count;
                }
            }
            double m1 = -INFINITY, m2 = -INFINITY;
            float bias = 0.0f;
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
                const int q = h == 0 ? first : second;
                if (q < 0) continue;
                double m = 1.0 / (1.0 + exp(-(double)to_f32<T>(row[e0 + q])));
                if (p.bias) {
                    m += (double)p.bias[e0 + q];
                    bias = fmaxf(bias, fabsf(p.bias[e0 + q]));
                }
                m2 = m1;
                m1 = m;
            }
            const double tie = group_tie(pair, m1, m2, bias);
            double sum = m2 == -INFINITY ? m1 : m1 + m2;
            // as groups_f64, in the token's eight lanes
            bool among = false;
#pragma unroll 1
            for (int r = 0; r < p.kept; ++r) {
                const double m = fmax8(sum);
                const double from = -fmax8(sum == m ? tie - sum : -INFINITY);
                const uint32_t equal = sum != -INFINITY && sum + tie >= from ? 8 - sub : 0;
                if (max8(equal) == equal && equal != 0) {
                    among = true;
                    sum = -INFINITY;
                }
            }
            const bool sure = count <= (pair ? 2 : 1) && least < INFINITY;
            const unsigned unsure = __ballot_sync(kFull, near && !sure);
            const bool settled = near && (unsure >> (lane & 24) & 255) == 0;
            if (settled) stay = among;
            bad = __ballot_sync(kFull, near && !settled);
        }
        if (bad != 0)
            for (int r = 0; r < 4; ++r) {
                if ((bad >> (8 * r) & 255) == 0 || tw + r >= p.T) continue;
                const uint32_t mask = groups_f64<T>(p, static_cast<const T*>(p.x) + (tw + r) * p.ld, wide, lane);
                if (lane >> 3 == r) stay = mask >> sub & 1;
            }
        keep = stay ? ~kIdx : 0u;
    }

    // keys: a lane that does not stay, masked and missing experts keep the place alone (<= kIdx)
    uint32_t key[NV];
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        key[q] = 0;
        if (q < per) key[q] = (order_key(v[q]) & keep) | (kIdx - q);
        if (!clean && v[q] == -INFINITY) key[q] = 0;
    }
    top8<NV>(key);
    // rounds: the largest value, then the lowest lane (in the bits of the place), whose first key is popped
    uint32_t val = 0;                           // lane l: the value bits of the l-th choice
    int my_i = -1, extra = -1, n = 0, taken = 0;
    auto best = [&]() { return max8(key[0] > kIdx ? (key[0] & ~kIdx) | (7 - sub) : 0u); };
    auto pop = [&](uint32_t m, int last) {      // the expert of the winner; key[0..last) are wanted afterwards
        const int wl = 7 - (int)(m & kIdx);
        const int e = __shfl_sync(kFull, e0 + (int)(kIdx - (key[0] & kIdx)), (lane & 24) | wl);
        if (m != 0 && sub == wl) {
#pragma unroll
            for (int q = 0; q < 7; ++q)
                if (q < last) key[q] = key[q + 1];
            if (last >= 7) key[7] = 0;
            ++taken;
        }
        return e;
    };
#pragma unroll
    for (int l = 0; l < 8; ++l) {               // (the four tokens go together)
        if (l >= p.k) break;
        const uint32_t m = best();
        const int e = pop(m, 7);
        n += m != 0 ? 1 : 0;
        if (sub == l && m != 0) {
            val = m & ~kIdx;
            my_i = e;
        }
    }
    if (!exact) {
        auto close = [&](uint32_t x, uint32_t y) {   // value bits that follow each other
            const float hi = key_value(x), lo = key_value(y);
            return p.bias ? !(hi - lo > err2 + (NV * 1.2e-7f + 3e-7f) * fmaxf(fabsf(hi), fabsf(lo))) : !(hi > lo);
        };
        // a list whose eight are all chosen goes on with the best of the lane's others
        auto refill = [&](bool empty) {
            if (!__any_sync(kFull, empty)) return;
            uint32_t used = 0, more = 0;
            for (int l = 0; l < 9; ++l) {
                const int q = (l < 8 ? __shfl_sync(kFull, my_i, (lane & 24) | l) : extra) - e0;
                if (q >= 0 && q < per) used |= 1u << q;
            }
#pragma unroll 4
            for (int q = 0; q < NV; ++q) {
                if (q >= per) break;
                const float x = to_f32<T>(row[e0 + q]);
                float m = selectable<T>(x) ? x : -INFINITY;
                if (p.bias) {
                    const float pb = p.bias[e0 + q];
                    m = m > -INFINITY && pb > kMasked ? score(x) + pb : -INFINITY;
                }
                const uint32_t k = m == -INFINITY ? 0u : (order_key(m) & ~kIdx) | (kIdx - q);
                if (!(used >> q & 1)) more = max(more, k);
            }
            if (empty) key[0] = more;
        };
        if (per > 8) refill(taken == 8);
        const uint32_t out = best();            // the first that was left
        uint32_t next = __shfl_down_sync(kFull, val, 1, 8);
        if (sub == n - 1) next = out & ~kIdx;
        const bool near = sub < n && next != 0 && close(val, next);
        const unsigned bad = __ballot_sync(kFull, near);
        if (bad != 0) {
            // the last choice and the first left are close: the latter is a candidate too, if the one behind it is not
            const bool border = near && sub == n - 1;
            const bool grow = (__ballot_sync(kFull, border) >> (lane & 24) & 255) != 0;
            const int before = taken;
            const int e = pop(grow ? out : 0u, 7);
            if (grow) extra = e;
            if (per > 8) refill(taken > before && taken >= 8);
            const uint32_t after = best() & ~kIdx;
            // of the token: the whole row in f64
            const bool redo = grow && after != 0 && close(out & ~kIdx, after);
            const unsigned again = __ballot_sync(kFull, redo);
            for (int r = 0; r < 4; ++r) {
                if ((bad >> (8 * r) & 255) == 0 || tw + r >= p.T) continue;
                const T* rr = static_cast<const T*>(p.x) + (tw + r) * p.ld;
                int got;
                if ((again >> (8 * r) & 255) != 0) {
                    got = route_row_f64<T>(p, rr, wide, lane);
                } else {
                    const int count = __shfl_sync(kFull, n, 8 * r), ex = __shfl_sync(kFull, extra, 8 * r);
                    const int c = __shfl_sync(kFull, my_i, 8 * r + (lane & 7));
                    const float tp = __shfl_sync(kFull, top, 8 * r), is = __shfl_sync(kFull, inv_sum, 8 * r);
                    const float er = __shfl_sync(kFull, err2, 8 * r);
                    got = rank_candidates<T>(p, rr, tp, is, er, lane < count ? c : ex, count + (ex >= 0 ? 1 : 0),
                                                     reinterpret_cast<int*>(wide), lane);
                    __syncwarp();
                }
                got = __shfl_sync(kFull, got, sub);
                if (lane >> 3 == r) my_i = got;
            }
        }
    }
    if (sub >= p.k) my_i = -1;

    const float xs = my_i >= 0 ? to_f32<T>(row[my_i]) : -INFINITY;
    float e = 0.0f;
    if (p.sigmoid) e = sigmoid(xs);
    else if (!p.renorm) e = my_i < 0 ? 0.0f : (xs == top ? 1.0f : expf(xs - top)) * inv_sum;
    if (p.renorm) {
        float sum = p.sigmoid ? sum8(e) : 0.0f;
        if (!__all_sync(kFull, sum > kSmallSum)) {   // as above; a token whose sum stands keeps it
            const float mx = fmax8(xs);
            const float f = my_i < 0 ? 0.0f : xs == mx ? 1.0f : expf(xs - mx);
            const float g = sum8(f);
            if (!(sum > kSmallSum)) {
                e = f;
                sum = g;
            }
        }
        e = sum > 0.0f ? e * rcp_fast(sum) : 0.0f;
    }
    if (live && sub < p.k) {
        p.idx[t * p.k + sub] = my_i;
        p.w[t * p.k + sub] = e * p.scale;
    }
}

cudaError_t launch_kernel(void (*kern)(RouteParams), int64_t blocks, const RouteParams& p, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kRouteWarps * 32);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // (see pdl_wait)
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

template <typename T, int NV>
cudaError_t launch_many(const RouteParams& p, cudaStream_t st) {
    auto kern = p.E == 8 * NV ? route_many_kernel<T, NV, true> : route_many_kernel<T, NV, false>;
    return launch_kernel(kern, (p.T + 4 * kRouteWarps - 1) / (4 * kRouteWarps), p, st);
}

// True (and launched) where the shape fits: 8 parts of a multiple of 4 experts,
// at most 256 in all, no groups or eight, rows that allow loads of four.
template <typename T>
bool try_many(RouteParams p, cudaStream_t st, cudaError_t* err) {
    const int per = p.E / 8;
    if (p.T < (per <= 8 ? 4096 : 16384) || p.E % 32 != 0 || p.E > 256 || p.k > 8 || (p.G != 1 && p.G != 8) ||
        reinterpret_cast<uintptr_t>(p.x) % (4 * sizeof(T)) != 0 || p.ld % 4 != 0 ||
        reinterpret_cast<uintptr_t>(p.bias) % 16 != 0)
        return false;
    p.vec = p.vec_bias = 0;   // (for the whole-warp pass)
    *err = per <= 8 ? launch_many<T, 8>(p, st) : per <= 16 ? launch_many<T, 16>(p, st) : launch_many<T, 32>(p, st);
    return true;
}

template <typename T, int NV>
cudaError_t launch_nv(RouteParams p, cudaStream_t st) {
    constexpr int kBytes = NV * (int)sizeof(T);
    constexpr int kVec = kBytes % 16 == 0 ? 16 : kBytes % 8 == 0 ? 8 : kBytes % 4 == 0 ? 4 : 2;
    p.vec = reinterpret_cast<uintptr_t>(p.x) % kVec == 0 && (p.ld * (int64_t)sizeof(T)) % kVec == 0;
    constexpr int kVecB = NV >= 4 ? 16 : NV * 4;
    p.vec_bias = reinterpret_cast<uintptr_t>(p.bias) % kVecB == 0;
    const int whole = p.per % NV == 0 ? p.per / NV : 0;
    p.lanes = p.G > 1 && (whole & (whole - 1)) == 0 ? whole : 0;
    return launch_kernel(route_kernel<T, NV>, (p.T + kRouteWarps - 1) / kRouteWarps, p, st);
}

template <typename T>
cudaError_t launch_typed(const RouteParams& p, cudaStream_t st) {
    cudaError_t err;
    if (try_many<T>(p, st, &err)) return err;
    if (p.E <= 32) return launch_nv<T, 1>(p, st);
    if (p.E <= 64) return launch_nv<T, 2>(p, st);
    if (p.E <= 128) return launch_nv<T, 4>(p, st);
    if (p.E <= 256) return launch_nv<T, 8>(p, st);
    if (p.E <= 512) return launch_nv<T, 16>(p, st);
    return launch_nv<T, 32>(p, st);
}

}  // namespace

int check_routing(const MoeRouting* r, int E, int k) {
    if (!r) { set_error("routing is null"); return MOE_ERR_INVALID_ARG; }
    if (E < 1 || E > kRouteMaxExperts) {
        set_error("num_experts=%d: routing takes 1 to %d", E, kRouteMaxExperts);
        return E < 1 ? MOE_ERR_INVALID_ARG : MOE_ERR_UNSUPPORTED;
    }
    if (k < 1 || k > 32 || k > E) {
        set_error("top_k=%d must be in 1..32 and <= num_experts=%d", k, E);
        return MOE_ERR_INVALID_ARG;
    }
    if (r->score != MOE_SCORE_SOFTMAX && r->score != MOE_SCORE_SIGMOID) {
        set_error("routing score %d unknown", r->score);
        return MOE_ERR_INVALID_ARG;
    }
    if (r->num_groups < 1 || E % r->num_groups != 0 || r->groups_kept < 1 || r->groups_kept > r->num_groups) {
        set_error("num_groups=%d must divide num_experts=%d, and groups_kept=%d be in 1..num_groups", r->num_groups, E,
                  r->groups_kept);
        return MOE_ERR_INVALID_ARG;
    }
    if (r->group_top != 1 && r->group_top != 2) {
        set_error("group_top=%d must be 1 or 2", r->group_top);
        return MOE_ERR_INVALID_ARG;
    }
    if (!(r->scale > -INFINITY && r->scale < INFINITY)) {
        set_error("routing scale must be finite");
        return MOE_ERR_INVALID_ARG;
    }
    return MOE_OK;
}

cudaError_t launch_route(const void* logits, int type, int64_t T, int E, int64_t ld, int k, const MoeRouting& r,
                         const float* bias, int* idx, float* w, cudaStream_t st) {
    if (T == 0) return cudaSuccess;
    RouteParams p{};
    p.x = logits;
    p.T = T;
    p.ld = ld;
    p.E = E;
    p.k = k;
    p.sigmoid = r.score == MOE_SCORE_SIGMOID;
    // every group kept is no grouping at all
    p.G = r.groups_kept == r.num_groups ? 1 : r.num_groups;
    p.per = E / p.G;
    p.kept = p.G == 1 ? 1 : r.groups_kept;
    p.group_top = p.G == 1 ? 1 : r.group_top;
    p.sub = 32;
    while (p.sub > 0 && 32 / p.sub < p.G) p.sub >>= 1;
    p.renorm = r.renormalise != 0;
    p.scale = r.scale;
    p.bias = bias;
    p.idx = idx;
    p.w = w;
    switch (type) {
        case MOE_TYPE_F32: return launch_typed<float>(p, st);
        case MOE_TYPE_F16: return launch_typed<__half>(p, st);
        default: return launch_typed<__nv_bfloat16>(p, st);
    }
}

}  // namespace moe

using namespace moe;

extern "C" int moe_route_experts(const void* logits, int logits_type, int64_t tokens, int num_experts,
                                 int64_t row_stride, int top_k, const MoeRouting* routing, const float* select_bias,
                                 int* indices, float* weights, cudaStream_t stream) {
    int rc = check_routing(routing, num_experts, top_k);
    if (rc != MOE_OK) return rc;
    if (logits_type != MOE_TYPE_F32 && logits_type != MOE_TYPE_F16 && logits_type != MOE_TYPE_BF16) {
        set_error("moe_route_experts: logits type %d unknown", logits_type);
        return MOE_ERR_INVALID_ARG;
    }
    if (tokens < 0 || row_stride < num_experts) {
        set_error("moe_route_experts: tokens=%lld must be >= 0 and row_stride=%lld >= num_experts=%d",
                  (long long)tokens, (long long)row_stride, num_experts);
        return MOE_ERR_INVALID_ARG;
    }
    if (tokens >= (int64_t)1 << 32) {
        set_error("moe_route_experts: %lld tokens, at most 2^32 - 1 in a call", (long long)tokens);
        return MOE_ERR_UNSUPPORTED;
    }
    if (tokens == 0) return MOE_OK;
    if (!logits || !indices || !weights) {
        set_error("moe_route_experts: a buffer is null");
        return MOE_ERR_INVALID_ARG;
    }
    const int size = logits_type == MOE_TYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) % size != 0 || reinterpret_cast<uintptr_t>(indices) % 4 != 0 ||
        reinterpret_cast<uintptr_t>(weights) % 4 != 0 || reinterpret_cast<uintptr_t>(select_bias) % 4 != 0) {
        set_error("moe_route_experts: a buffer is not aligned to its type");
        return MOE_ERR_INVALID_ARG;
    }
    const Span rows{logits, row_stride * size, (int64_t)num_experts * size, tokens};
    const Span outs[2] = {vector_span(indices, tokens * top_k * 4), vector_span(weights, tokens * top_k * 4)};
    for (const Span& o : outs)
        if (overlap(rows, o) || overlap(vector_span(select_bias, num_experts * 4), o) || overlap(outs[0], outs[1])) {
            set_error("moe_route_experts: an output shares memory with the logits, the bias or the other output");
            return MOE_ERR_INVALID_ARG;
        }
    int dev = 0, num_sms = 0;
    rc = current_device(&dev, &num_sms);
    if (rc != MOE_OK) return rc;
    const cudaError_t e = launch_route(logits, logits_type, tokens, num_experts, row_stride, top_k, *routing,
                                       select_bias, indices, weights, stream);
    if (e != cudaSuccess) {
        set_error("moe_route_experts: %s", cudaGetErrorString(e));
        return MOE_ERR_CUDA;
    }
    return MOE_OK;
}
