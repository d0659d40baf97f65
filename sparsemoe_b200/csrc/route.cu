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
//         sigmoid underflows, exp(x - max) in its place, its limit) or s, times scale.
// Masked experts (NaN, logits <= -1e20 or f16's lowest value, a bias that is
// NaN or <= -1e20) are never chosen; slots that stay empty hold (-1, 0).
//
// The order is that of exact arithmetic: the f32 scores carry an error bound,
// and a row in which two values that follow each other in the order (or the
// last kept and the first left group) are closer than twice that is selected
// again in f64, where group sums that agree to 2^-49 are ties.  Rows that need
// it are about 1 in 10^4 for continuous logits.
//
// One warp per token, lane l holding experts l*NV .. l*NV + NV - 1, so the
// lowest lane of a ballot is the lowest index of a tie.  A round of the
// selection is one redux.sync over the lanes' best keys and a ballot.
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
    int sub;                // lanes that share one group of the fast group pass (0: G > 32, f64 path)
    int renorm;
    float scale;
    const float* bias;
    int* idx;
    float* w;
    int vec;                // rows allow the vector loads
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
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
    return v;
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

template <typename T, int NV>
__device__ __forceinline__ void load_row(const T* row, int e0, int E, bool vec, float (&x)[NV]) {
    constexpr int kBytes = NV * (int)sizeof(T);
    constexpr int kVec = kBytes % 16 == 0 ? 16 : kBytes % 8 == 0 ? 8 : kBytes % 4 == 0 ? 4 : 2;
    if (kVec > (int)sizeof(T) && vec && e0 + NV <= E) {
        union { T v[NV]; uint4 q[(kBytes + 15) / 16]; uint2 d[(kBytes + 7) / 8]; uint32_t u[(kBytes + 3) / 4]; } r;
        if constexpr (kVec == 16) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) r.q[i] = __ldg(reinterpret_cast<const uint4*>(row + e0) + i);
        } else if constexpr (kVec == 8) {
#pragma unroll
            for (int i = 0; i < kBytes / 8; ++i) r.d[i] = __ldg(reinterpret_cast<const uint2*>(row + e0) + i);
        } else if constexpr (kVec == 4) {
#pragma unroll
            for (int i = 0; i < kBytes / 4; ++i) r.u[i] = __ldg(reinterpret_cast<const uint32_t*>(row + e0) + i);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) x[i] = to_f32<T>(r.v[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = e0 + i < E ? to_f32<T>(row[e0 + i]) : -INFINITY;
}

// The whole selection of one row in f64: lane l looks at experts l, l + 32, ..
// (E <= 1024).  Returns the lane's choice (lane l: the l-th) or -1.
template <typename T>
__device__ __noinline__ int route_row_f64(const RouteParams& p, const T* row, int lane) {
    const int n = (p.E + 31) / 32;
    double v[32], s[32];
    double top = -INFINITY;
    for (int i = 0; i < n; ++i) {
        const int e = lane + 32 * i;
        const float x = e < p.E ? to_f32<T>(row[e]) : -INFINITY;
        v[i] = selectable<T>(x) ? (double)x : -INFINITY;
        top = fmax(top, v[i]);
    }
    if (p.bias || p.group_top == 2) {
        double sum = 0.0;
        if (!p.sigmoid)
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(kFull, top, o));
        for (int i = 0; i < n; ++i) {
            if (p.sigmoid) s[i] = 1.0 / (1.0 + exp(-v[i]));
            else s[i] = v[i] == -INFINITY ? 0.0 : v[i] == top ? 1.0 : exp(v[i] - top);
            sum += s[i];
        }
        sum = p.sigmoid ? 1.0 : warp_sum(sum);
        for (int i = 0; i < n; ++i) {
            const int e = lane + 32 * i;
            s[i] = p.sigmoid ? s[i] : s[i] / sum;
            if (v[i] == -INFINITY) s[i] = -INFINITY;
            if (p.bias && e < p.E) {
                const float b = __ldg(p.bias + e);
                v[i] = b > kMasked ? s[i] + (double)b : -INFINITY;
                s[i] = v[i];
            }
        }
    }
    // a round over d[0..m): the largest value, then the lowest index of those
    // that reach it (within `tie` of it, relative to 1 + |value|)
    auto best_of = [&](const double* d, int m, double tie) {
        double a = -INFINITY;
        for (int i = 0; i < m; ++i) a = fmax(a, d[i]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a = fmax(a, __shfl_xor_sync(kFull, a, o));
        if (a == -INFINITY) return -1;
        const double from = isinf(a) ? a : a - tie * (1.0 + fabs(a));
        uint32_t at = 0xFFFFFFFFu;
        for (int i = m - 1; i >= 0; --i)
            if (d[i] >= from) at = lane + 32 * i;
        return (int)__reduce_min_sync(kFull, at);
    };
    if (p.G > 1) {
        double gs[32];   // lane l: groups l, l + 32, ..
        const int gn = (p.G + 31) / 32;
        for (int i = 0; i < gn; ++i) gs[i] = -INFINITY;
        for (int g = 0; g < p.G; ++g) {
            double a = -INFINITY, b = -INFINITY;
            for (int i = 0; i < n; ++i) {
                const int e = lane + 32 * i;
                if (e < p.E && e / p.per == g) merge2(a, b, p.group_top == 2 ? s[i] : v[i], (double)-INFINITY);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const double c = __shfl_xor_sync(kFull, a, o), d = __shfl_xor_sync(kFull, b, o);
                merge2(a, b, c, d);
            }
            if (p.group_top == 2 && b != -INFINITY) a += b;
            if ((g & 31) == lane) gs[g >> 5] = a;
        }
        uint32_t keep = 0;
        // sums that agree to 2^-49 are ties: sigmoid(x) + sigmoid(-x) is 1 for every x
        const double tie = p.group_top == 2 ? 0x1p-49 : 0.0;
        for (int r = 0; r < p.kept; ++r) {
            const int g = best_of(gs, gn, tie);
            if (g < 0) break;
            if ((g & 31) == lane) {
                keep |= 1u << (g >> 5);
                gs[g >> 5] = -INFINITY;
            }
        }
        for (int i = 0; i < n; ++i) {
            const int e = lane + 32 * i, g = e < p.E ? e / p.per : 0;
            if (!((__shfl_sync(kFull, keep, g & 31) >> (g >> 5)) & 1)) v[i] = -INFINITY;
        }
    }
    int mine = -1;
    for (int l = 0; l < p.k; ++l) {
        const int e = best_of(v, n, 0.0);
        if (e < 0) break;
        if (lane == l) mine = e;
        if ((e & 31) == lane) v[e >> 5] = -INFINITY;
    }
    return mine;
}

template <typename T, int NV>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const RouteParams p) {
    __shared__ float sv[kRouteWarps][NV * 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t t = (int64_t)blockIdx.x * kRouteWarps + warp;
    if (t >= p.T) return;
    const T* row = static_cast<const T*>(p.x) + t * p.ld;
    const int e0 = lane * NV;
    float v[NV];
    load_row<T, NV>(row, e0, p.E, p.vec != 0, v);
    uint32_t seen = 0;
#pragma unroll
    for (int q = 0; q < NV; ++q)
        if (selectable<T>(v[q])) seen |= 1u << q;
        else v[q] = -INFINITY;

    // softmax statistics, where a score or an unnormalised weight needs them
    const bool pair = p.G > 1 && p.group_top == 2;
    const bool scores = p.bias != nullptr || pair;
    float top = 0.0f, inv_sum = 1.0f;
    float s[NV];
    if (!p.sigmoid && (scores || !p.renorm)) {
        top = -INFINITY;
#pragma unroll
        for (int q = 0; q < NV; ++q) top = fmaxf(top, v[q]);
        top = warp_max(top);
        float sum = 0.0f;
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            s[q] = !((seen >> q) & 1) ? 0.0f : v[q] == top ? 1.0f : __expf(v[q] - top);
            sum += s[q];
        }
        sum = warp_sum(sum);
        inv_sum = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
        for (int q = 0; q < NV; ++q) s[q] *= inv_sum;
    } else if (p.sigmoid && scores) {
#pragma unroll
        for (int q = 0; q < NV; ++q) s[q] = __fdividef(1.0f, 1.0f + __expf(-v[q]));
    }
    if (p.bias) {
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const float b = e0 + q < p.E ? __ldg(p.bias + e0 + q) : -INFINITY;
            v[q] = ((seen >> q) & 1) && b > kMasked ? s[q] + b : -INFINITY;
        }
    }
    // Error bounds: |s - exact| <= 4e-7 for the sigmoid (__expf: (2 + 1.2|x|)
    // 2^-23 relative, times s(1-s); __fdividef 2 ulp) and <= 2e-6 for the
    // softmax (the sum's relative error times s); two values compared, each of
    // one or (groups) two scores, plus the roundings of the sums.
    const float err = p.sigmoid ? 4e-7f : 2e-6f;
    bool near = p.sub == 0 && p.G > 1;   // more than 32 groups: the f64 pass does them

    if (p.G > 1 && !near) {
        float* buf = sv[warp];
        const bool from_scores = pair && !p.bias;
#pragma unroll
        for (int q = 0; q < NV; ++q) buf[e0 + q] = !from_scores ? v[q] : ((seen >> q) & 1) ? s[q] : -INFINITY;
        __syncwarp();
        const int g = lane / p.sub, j = lane % p.sub;
        float a = -INFINITY, b = -INFINITY;
        if (g < p.G)
            for (int i = j; i < p.per; i += p.sub) merge2(a, b, buf[g * p.per + i], -INFINITY);
        for (int o = p.sub >> 1; o > 0; o >>= 1) {
            const float c = __shfl_xor_sync(kFull, a, o), d = __shfl_xor_sync(kFull, b, o);
            merge2(a, b, c, d);
        }
        if (pair && b != -INFINITY) a += b;
        const uint32_t key = g < p.G && a != -INFINITY ? order_key(a) : 0u;
        int rank = 0;
        for (int h = 0; h < p.G; ++h) {
            const uint32_t other = __shfl_sync(kFull, key, h * p.sub);
            rank += other > key || (other == key && h < g) ? 1 : 0;
        }
        const bool stay = key != 0 && rank < p.kept;
        if (scores) {
            const uint32_t last = __reduce_min_sync(kFull, stay ? key : 0xFFFFFFFFu);
            const uint32_t out = __reduce_max_sync(kFull, stay ? 0u : key);
            if (out != 0) {
                const float lo = key_value(last), hi = key_value(out);
                near = !(lo - hi > 4.0f * err + 6e-7f * fmaxf(fabsf(lo), fabsf(hi)));
            }
        }
        const uint32_t kept = __ballot_sync(kFull, stay);
        int gg = e0 / p.per, r = e0 - gg * p.per;
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            if (e0 + q >= p.E || !((kept >> (gg * p.sub & 31)) & 1)) v[q] = -INFINITY;
            if (++r == p.per) { r = 0; ++gg; }
        }
    }

    int my_i = -1;
    if (!near) {
        uint32_t key[NV], bk = 0;
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            key[q] = v[q] == -INFINITY ? 0u : order_key(v[q]);
            bk = max(bk, key[q]);
        }
        float prev = INFINITY;
        for (int l = 0; l <= p.k; ++l) {
            const uint32_t m = __reduce_max_sync(kFull, bk);
            if (m == 0) break;
            if (p.bias) {
                const float val = key_value(m);
                if (l > 0) near |= !(prev - val > 2.0f * err + 3e-7f * fmaxf(fabsf(prev), fabsf(val)));
                prev = val;
            }
            if (l == p.k) break;
            const int wl = __ffs(__ballot_sync(kFull, bk == m)) - 1;
            int bq = 0;
            if (lane == wl) {
#pragma unroll
                for (int q = NV - 1; q >= 0; --q) bq = key[q] == m ? q : bq;
                bk = 0;
#pragma unroll
                for (int q = 0; q < NV; ++q) {
                    if (q == bq) key[q] = 0;
                    bk = max(bk, key[q]);
                }
            }
            bq = __shfl_sync(kFull, bq, wl);
            if (lane == l) my_i = wl * NV + bq;
        }
    }
    if (near) my_i = route_row_f64<T>(p, row, lane);

    const float xs = my_i >= 0 ? to_f32<T>(row[my_i]) : -INFINITY;
    float e;
    if (p.renorm) {
        const float mx = warp_max(xs);
        if (p.sigmoid && mx > -80.0f) e = my_i >= 0 ? 1.0f / (1.0f + expf(-xs)) : 0.0f;
        else e = my_i < 0 ? 0.0f : xs == mx ? 1.0f : expf(xs - mx);
        const float sum = warp_sum(e);
        e = sum > 0.0f ? e / sum : 0.0f;
    } else if (p.sigmoid) {
        e = my_i >= 0 ? 1.0f / (1.0f + expf(-xs)) : 0.0f;
    } else {
        e = my_i < 0 ? 0.0f : (xs == top ? 1.0f : expf(xs - top)) * inv_sum;
    }
    if (lane < p.k) {
        p.idx[t * p.k + lane] = my_i;
        p.w[t * p.k + lane] = e * p.scale;
    }
}

template <typename T, int NV>
cudaError_t launch_nv(RouteParams p, cudaStream_t st) {
    constexpr int kBytes = NV * (int)sizeof(T);
    constexpr int kVec = kBytes % 16 == 0 ? 16 : kBytes % 8 == 0 ? 8 : kBytes % 4 == 0 ? 4 : 2;
    p.vec = reinterpret_cast<uintptr_t>(p.x) % kVec == 0 && (p.ld * (int64_t)sizeof(T)) % kVec == 0;
    const int64_t blocks = (p.T + kRouteWarps - 1) / kRouteWarps;
    route_kernel<T, NV><<<(unsigned)blocks, kRouteWarps * 32, 0, st>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_typed(const RouteParams& p, cudaStream_t st) {
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
