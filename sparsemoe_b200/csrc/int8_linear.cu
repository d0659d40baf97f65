// Dense int8 products with a scale per token and per output channel, the
// per-token quantiser in front of them, and the shared expert built from both.
//
//   quantise   s_t = max_k |x_tk| * f32(1/127), one f32 product (1 for a zero row),
//              q_tk = round-half-even(x_tk / s_t) of the exact quotient;
//   product    y_tn = (sum_k q_tk w_kn) * s_t * s_n (+ bias_n) (+ residual_tn),
//              the sum exact in s32 (K <= 131071), the rest in f32, one
//              rounding to the output type;
//   shared     g = product(x, Wg), u = product(x, Wu), h = u * g / (1 + exp(-g))
//   expert     kept in f32, quantised per token, y = product(h, Wd) + residual.
// A row holding a NaN or an infinity gets s_t = NaN, so its outputs are NaN.
#include "moe_internal.h"
#include "common.cuh"
#include "sm100.cuh"

#include <cudaTypedefs.h>
#include <cuda.h>
#include <algorithm>

namespace moe {

// expert_gemm.cu: [outer, inner] bytes, rows `stride` bytes apart, boxes of box_inner (64 or 128, the swizzle span)
// bytes x box_outer rows
bool make_map_u8_strided(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer, uint64_t stride,
                         uint32_t box_inner, uint32_t box_outer);

namespace {

using namespace sm100;

// Report of a wait that ran out, for the host alone: read and cleared by
// moe_check_device_status.  No kernel reads it, so what one launch reports
// stops no other.
__device__ int g_linear_status;

// ---- per-token quantisation --------------------------------------------------------

// Rows of up to TPR * 32 elements stay in registers (four vectors of eight a
// thread); longer ones are read twice, the second time from L1 / L2.
constexpr int kQVec = 4;

// Eight elements.  Plain loads: the values may come from the kernel before
// (griddepcontrol.wait), and a load through the read-only path could be moved
// ahead of the wait.
template <typename T> struct In8;
template <> struct In8<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* p) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    __device__ __forceinline__ void load_part(const float* p, int n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.0f;
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
    // largest magnitude as f32 bits: NaN > infinity > every finite value
    __device__ __forceinline__ uint32_t amax_bits() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
        return m;
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = v[i];
    }
};
template <typename T16> struct In8_16 {
    uint4 raw;
    __device__ __forceinline__ void load(const T16* p) { raw = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void load_part(const T16* p, int n) {
        uint32_t u[4] = {0u, 0u, 0u, 0u};
        const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) u[i >> 1] |= (uint32_t)s[i] << (16 * (i & 1));
        raw = make_uint4(u[0], u[1], u[2], u[3]);
    }
    __device__ __forceinline__ void zero() { raw = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ uint32_t amax_bits() const {
        const uint32_t m = __vmaxu2(__vmaxu2(raw.x & 0x7FFF7FFFu, raw.y & 0x7FFF7FFFu),
                                    __vmaxu2(raw.z & 0x7FFF7FFFu, raw.w & 0x7FFF7FFFu));
        const float2 f = F16Traits<T16>::unpack2(max(m & 0xFFFFu, m >> 16));
        return __float_as_uint(f.x) & 0x7FFFFFFFu;
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 p = F16Traits<T16>::unpack2(u[i]);
            f[2 * i] = p.x;
            f[2 * i + 1] = p.y;
        }
    }
};
template <> struct In8<__half> : In8_16<__half> {};
template <> struct In8<__nv_bfloat16> : In8_16<__nv_bfloat16> {};

// Two fused multiply-adds in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// Codes of eight values: round-half-even of the exact x / s.  x * (1/s) is within
// 127 * 2^-23 of the quotient, so its nearest integer n (which one fma leaves in
// the low bits of 1.5 * 2^23 + n) is right or the other neighbour of a border.
// e = x - n s, exact in one fma (both are multiples of the smaller of their last
// places, and |e| <= s), tells: past s / 2 the neighbour is nearer, at s / 2 the
// even one is taken.  bf16 rows meet a border in most warps (x / s is 127 times a
// quotient of two 8-bit numbers), so the correction is a few instructions, not a
// division.  Tiny and huge rows are scaled by a power of two first (pre != 1),
// which changes no quotient and keeps the arithmetic in the normal range; a
// subnormal scale has few bits, so there the codes are clamped.
__device__ __forceinline__ uint2 quant8(float (&f)[8], float s, float inv, float pre) {
    constexpr float kMagic = 12582912.0f;
    uint32_t t[8];
    float e[8], far = 0.0f;
    if (pre != 1.0f)
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= pre;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2 x = make_float2(f[i], f[i + 1]);
        const float2 m = fma2(x, make_float2(inv, inv), make_float2(kMagic, kMagic));
        const float2 n = fma2(m, make_float2(-1.0f, -1.0f), make_float2(kMagic, kMagic));
        const float2 d = fma2(n, make_float2(s, s), x);
        e[i] = d.x;
        e[i + 1] = d.y;
        far = fmaxf(far, fmaxf(fabsf(d.x), fabsf(d.y)));
        t[i] = __float_as_uint(m.x);
        t[i + 1] = __float_as_uint(m.y);
    }
    const float half = 0.5f * s;
    if (far >= half) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float ae = fabsf(e[i]);
            if (ae > half || (ae == half && (t[i] & 1u))) t[i] += e[i] > 0.0f ? 1u : 0xFFFFFFFFu;
        }
    }
    if (pre != 1.0f)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            t[i] = (uint32_t)max(-127, min(127, (int)(t[i] - __float_as_uint(kMagic))));
    uint2 w;
    w.x = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
    w.y = __byte_perm(__byte_perm(t[4], t[5], 0x0040), __byte_perm(t[6], t[7], 0x0040), 0x5410);
    return w;
}

// Scale of a row from the bits of its largest magnitude, and what quant8 needs.
struct RowScale {
    float s;          // the scale as it is handed out: NaN for a row with a NaN or an infinity
    float ss, inv;    // scale x pre, its reciprocal
    float pre;        // 2^100 or 2^-100 for tiny and huge rows (s is rounded before: a subnormal one keeps its few bits)
    bool bad;
    __device__ __forceinline__ explicit RowScale(uint32_t m) {
        const float amax = __uint_as_float(m);
        bad = m >= 0x7F800000u;
        s = bad ? __uint_as_float(0x7FFFFFFFu) : __fmul_rn(amax, 1.0f / 127.0f);
        if (s == 0.0f) s = 1.0f;   // a zero row, or one whose scale rounds to zero
        pre = amax < 5.4e-20f && s != 1.0f ? 1.2676506e30f : amax > 1.8e19f ? 7.8886091e-31f : 1.0f;
        ss = s * pre;
        inv = bad ? 0.0f : __fdiv_rn(1.0f, ss);
    }
    __device__ __forceinline__ uint2 codes(float (&f)[8]) const {
        return bad ? make_uint2(0u, 0u) : quant8(f, ss, inv, pre);
    }
};

// The first n of eight codes, at an 8-byte boundary.
__device__ __forceinline__ void store8(int8_t* q, uint2 w, int n) {
    if (n >= 8) {
        *reinterpret_cast<uint2*>(q) = w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) q[i] = (int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
}

__device__ __forceinline__ float silu(float g) { return g / (1.0f + __expf(-g)); }

// kPair (T = float): x holds gate values, the up values start `up` elements
// behind them, and the row that is quantised is up * gate / (1 + exp(-gate)).
// For many rows instruction issue (four fifths of the slots) and the HBM both
// count: 8192 x 7168 bf16 takes 34.1 us (5.2 TB/s of reads and writes), 8192 x 2048
// f32 15.3 (5.5 TB/s).  The registers are held to 32 a thread where 256 share a
// row (eight blocks an SM; 40 and six took 34.8 us) and to 40 below, where 32
// spill (8192 x 2048 bf16 12.0 us, 13.3 with 32); to 48 for f32.
template <typename T, int TPR, bool kPair>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 5 : TPR == 256 ? 8 : 6)
    quantize_tokens_kernel(const T* x, int64_t rows, int K, int64_t ldx, int64_t up, int8_t* q, int64_t ldq,
                           float* scale, int vec) {
    pdl_wait();
    pdl_trigger();
    constexpr int kRows = 256 / TPR;
    __shared__ uint32_t red[8];
    const int tr = threadIdx.x % TPR;
    const int64_t t = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
    const bool live = t < rows;
    const T* src = x + t * ldx;
    const bool keep = K <= TPR * 8 * kQVec;
    In8<T> v[kQVec];
    uint32_t m = 0;
    auto fetch = [&](In8<T>& d, int k) {
        if (!live || k >= K) d.zero();
        else if (vec && k + 8 <= K) d.load(src + k);
        else d.load_part(src + k, K - k);
        if constexpr (kPair) {
            if (live && k < K) {
                In8<T> u;
                if (vec && k + 8 <= K) u.load(src + up + k);
                else u.load_part(src + up + k, K - k);
#pragma unroll
                for (int i = 0; i < 8; ++i) d.v[i] = u.v[i] * silu(d.v[i]);
            }
        }
    };
    if (keep) {
#pragma unroll
        for (int i = 0; i < kQVec; ++i) fetch(v[i], (i * TPR + tr) * 8);
#pragma unroll
        for (int i = 0; i < kQVec; ++i) m = max(m, v[i].amax_bits());
    } else {
        for (int k = tr * 8; k < K; k += TPR * 8) {
            fetch(v[0], k);
            m = max(m, v[0].amax_bits());
        }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (TPR > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
        __syncthreads();
        const int w0 = threadIdx.x / TPR * (TPR / 32);
#pragma unroll
        for (int i = 0; i < TPR / 32; ++i) m = max(m, red[w0 + i]);
    }
    if (!live) return;
    const RowScale rs(m);
    if (tr == 0) scale[t] = rs.s;
    int8_t* dst = q + t * ldq;
    auto put = [&](const In8<T>& d, int k) {
        if (k >= K) return;
        float f[8];
        d.get(f);
        store8(dst + k, rs.codes(f), K - k);
    };
    if (keep) {
#pragma unroll
        for (int i = 0; i < kQVec; ++i) put(v[i], (i * TPR + tr) * 8);
    } else {
        for (int k = tr * 8; k < K; k += TPR * 8) {
            fetch(v[0], k);
            put(v[0], k);
        }
    }
}

// ---- product -----------------------------------------------------------------------

constexpr int kBM = 128;       // tokens of a tile
constexpr int kBK = 128;       // K of a stage: one 128-byte swizzle span
constexpr int kEpiThreads = 256;  // eight epilogue warps: two for each quarter of the TMEM lanes
constexpr int kThreads = 64 + kEpiThreads;  // behind the TMA and the MMA warp
constexpr int kMaxSplit = 8;

struct LinearParams {
    int T, N, K;               // N: output columns
    int m_tiles, n_tiles, kblocks;
    int n0_tiles;              // column tiles of the first matrix; the others are of the second (plain product of two)
    int64_t out1;              // elements from the first matrix's outputs to the second's
    int split;                 // CTAs of a cluster that share a tile's K
    int a_rows;                // rows of the A box
    int b_nk;                  // weights [N, K] (K-contiguous) rather than [K, N]
    int ahead;                 // weights may be loaded before the wait
    const float* s_tok;
    const float* s_ch0;        // channel scales (swiglu: gate)
    const float* s_ch1;        // swiglu: up
    const float* bias;
    const void* residual;
    int64_t ld_res;
    int res_type;
    void* out;
    int64_t ld_out;
    int out_type;
    int vec_out, vec_res;      // rows allow 16-byte accesses of eight columns
    int row_end16;             // a row of outputs is a whole number of 16-byte units
    int staged;                // outputs leave through shared memory (all but split tiles and unlike residuals)
    int tma_out;               // and from there by TMA (rows on 16-byte boundaries)
    uint32_t idesc;
};

// Eight columns of the parts of a split tile: 128 rows x 8 s32, and 16 bytes that
// put consecutive units into different banks.
constexpr int kUnitBytes = kBM * 32 + 16;

template <int kBN, bool kPair>
struct LinearCfg {
    static constexpr int kStages = kPair ? 6 : 4;
    static constexpr int kABytes = kBM * kBK;
    static constexpr int kBBytes = (kPair ? kBN / 2 : kBN) * kBK;   // a pair's CTAs hold half of the columns each
    static constexpr int kStageBytes = kABytes + kBBytes;
    // split sums (kBN = 128 only), or a staged chunk of 32 rows x 64 bytes for each epilogue warp
    static constexpr int kRecvBytes = kBN == 128 ? kBN / 8 * kUnitBytes : 8 * 2048;
    static constexpr size_t kSmem = 1024 + (size_t)kStages * kStageBytes + kRecvBytes + 256;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_cluster4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_32x32b_x8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}

// 2-D tiled store from shared memory, and the bulk groups that track its reads.
__device__ __forceinline__ void tma_store_2d(const void* tmap, const void* src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(tmap)),
                 "r"(smem_u32(src)), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int kPending> __device__ __forceinline__ void bulk_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- CTA pairs (tcgen05 cta_group::2) ----
__device__ __forceinline__ void tmem_alloc2(uint32_t* dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc2(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void mma_i8_ss2(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives on this barrier of the CTAs in `ctas` (both) when the tcgen05 operations issued so far are done.
__device__ __forceinline__ void mma_commit2(uint64_t* bar, uint16_t ctas = 3) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(ctas)
        : "memory");
}
// A load into this CTA whose bytes count on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const void* tmap, uint32_t bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A CTA's bounded waits.  One that runs out is reported to the host and sets
// `stop` (shared memory), which ends the waits of the CTA's other roles and, of
// a pair, the other CTA's.  Most waits end in their first try, which may last;
// the others are in line in the small kernel (1 x 7168 x 2048 7.37 us, 7.47 with
// a call) and a call in the tiles (512 x 2048 x 7168 15.12, 15.35 in line).
template <bool kInline> struct Waits {
    uint32_t* stop;
    uint32_t peer;   // the other CTA's word (0: none)
    uint64_t limit_ns;

    __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) const {
        if (mbar_try_wait(smem_u32(bar), parity)) return true;
        return kInline ? tries(smem_u32(bar), parity, stop, peer, limit_ns) : called(smem_u32(bar), parity, stop, peer, limit_ns);
    }
    static __device__ __noinline__ bool called(uint32_t bar, uint32_t parity, uint32_t* stop, uint32_t peer,
                                               uint64_t limit_ns) {
        return tries(bar, parity, stop, peer, limit_ns);
    }
    static __device__ __forceinline__ bool tries(uint32_t bar, uint32_t parity, uint32_t* stop, uint32_t peer,
                                                 uint64_t limit_ns) {
        const uint64_t t0 = globaltimer_ns();
        for (uint32_t it = 1;; ++it) {
            if (mbar_try_wait(bar, parity)) return true;
            if ((it & 15) == 0) {   // (the clock and the word not at every try, as mbar_wait)
                if (*(volatile uint32_t*)stop != 0) return false;
                if (globaltimer_ns() - t0 > limit_ns) {
                    atomicCAS(&g_linear_status, 0, kDevErrTimeout);
                    *(volatile uint32_t*)stop = 1;
                    if (peer) asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(peer), "r"(1u) : "memory");
                    return false;
                }
            }
        }
    }
    // For roles that go on with warp-collective operations: one answer for the warp.
    __device__ __forceinline__ bool warp(uint64_t* bar, uint32_t parity) const {
        return __all_sync(0xffffffffu, (*this)(bar, parity));
    }
    __device__ __forceinline__ bool stopped() const { return *(volatile uint32_t*)stop != 0; }
    // For arrivals from the cluster.
    __device__ __forceinline__ bool cluster(uint64_t* bar, uint32_t parity) const {
        const bool ok = (*this)(bar, parity);
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
        return ok;
    }
};

// Tells the CTAs of a cluster of `ctas` that this one has given up, ahead of the
// cluster barrier behind which their sums take its parts (all of them have
// started: an earlier phase of the barrier is behind).  The epilogue's warps call
// it: where another role gives up, theirs is the wait that runs out or is ended.
__device__ __noinline__ void tell_cluster(uint32_t stop, int ctas) {
    for (int r = 0; r < ctas; ++r)
        asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(mapa(stop, r)), "r"(1u) : "memory");
}

// After a wait that ran out, by the thread that issues the MMAs: up to 1 ms each
// for the copies that may be in flight (the next one of each stage; a copy takes
// microseconds) and for the MMAs issued so far, so that none of them reaches
// memory that the CTA has left.  (The producers run at most that far ahead.)
constexpr uint64_t kDrainNs = 1000000;
template <bool kPair> __device__ __noinline__ void drain(uint64_t* full, int s, uint32_t ph, int stages, uint64_t* bail) {
    if (kPair) mma_commit2(bail, 1);
    else mma_commit(bail);
    for (int i = 0; i <= stages; ++i) {
        const uint32_t bar = smem_u32(i < stages ? &full[s] : bail), parity = i < stages ? ph : 0;
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(bar, parity) && globaltimer_ns() - t0 < kDrainNs) {}
        if (++s == stages) { s = 0; ph ^= 1u; }
    }
}

__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int type) {
    if (type == MOE_TYPE_F32) return static_cast<const float*>(p)[i];
    if (type == MOE_TYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// A sum's value, rounded before bias or residual are added: no fused multiply-add
// in one epilogue that another lacks, so that a token's result is the same bits
// in any batch.
__device__ __forceinline__ float dequant(uint32_t sum, float s_tok, float s_ch) {
    return __fmul_rn((float)(int)sum * s_tok, s_ch);
}

// Eight consecutive outputs of row t from column n on (those below N) of the first or second matrix.
__device__ __forceinline__ void emit8(const LinearParams& p, int64_t t, bool second, int n, float (&v)[8]) {
    const int left = p.N - n;
    if (p.residual) {   // plain loads: it may be the output itself
        const int64_t at = t * p.ld_res + n;
        if (p.vec_res && left >= 8) {
            if (p.res_type == MOE_TYPE_F32) {
                const float4* r = reinterpret_cast<const float4*>(static_cast<const float*>(p.residual) + at);
                const float4 a = r[0], b = r[1];
                v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w; v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
            } else {
                const uint4 r = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.residual) + at);
                const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = p.res_type == MOE_TYPE_F16 ? F16Traits<__half>::unpack2(u[i])
                                                                : F16Traits<__nv_bfloat16>::unpack2(u[i]);
                    v[2 * i] += f.x;
                    v[2 * i + 1] += f.y;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) v[i] += load_as_f32(p.residual, at + i, p.res_type);
        }
    }
    const int64_t at = t * p.ld_out + n + (second ? p.out1 : 0);
    if (p.out_type == MOE_TYPE_F32) {
        float* o = static_cast<float*>(p.out) + at;
        if (p.vec_out && left >= 8) {
            reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) o[i] = v[i];
        }
        return;
    }
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        u[i] = p.out_type == MOE_TYPE_F16 ? F16Traits<__half>::pack2(v[2 * i], v[2 * i + 1])
                                          : F16Traits<__nv_bfloat16>::pack2(v[2 * i], v[2 * i + 1]);
    uint16_t* o = static_cast<uint16_t*>(p.out) + at;
    if (p.vec_out && left >= 8) {
        *reinterpret_cast<uint4*>(o) = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) o[i] = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
    }
}

// One arrival a warp: its reads of the accumulator are done.
__device__ __forceinline__ void release_acc(uint32_t bar, int lane) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) arrive_cluster(bar);
}

template <int kC> __device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[kC]) {
    if constexpr (kC == 32) tmem_ld_32x32b_x32(taddr, r);
    else tmem_ld_32x32b_x16(taddr, r);
}

// One epilogue warp's 32 rows and kCols output columns of a tile, staged: chunks
// of kC columns (64 bytes a row) go from TMEM through the arithmetic into the
// warp's 2 KB of shared memory (64-byte swizzle: 16-byte unit j of row r at
// j ^ ((r >> 1) & 3)) and from there by a TMA store, which leaves out rows and
// columns outside the tensor.  Storing one row a thread instead touched 32 rows
// an instruction.  A 16-bit residual is read coalesced, a chunk ahead (its lines
// are asked into L2 before the accumulator is waited for), and meets its row's
// thread in the same buffer.
template <int kCols, int kOutN, bool kSwiglu, bool kF32>
struct StagedEpilogue {
    static constexpr int kC = kF32 ? 16 : 32;
    static constexpr bool kRes = !kF32 && !kSwiglu;

    static __device__ __forceinline__ void prefetch_residual(const LinearParams& p, int row, int col0) {
        if (row >= p.T) return;
        const uint16_t* src = static_cast<const uint16_t*>(p.residual) + (int64_t)row * p.ld_res;
#pragma unroll
        for (int c = 0; c < kCols; c += 64)
            if (col0 + c < p.N) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + col0 + c));
    }
    // rows (lane / 4) + 8 i, 16-byte unit lane % 4 of a chunk
    static __device__ __forceinline__ void fetch(const LinearParams& p, int row0, int col0, int lane, uint4 (&res)[4]) {
        const int col = col0 + 8 * (lane % 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = row0 + lane / 4 + 8 * i;
            res[i] = make_uint4(0u, 0u, 0u, 0u);
            if (row >= p.T || col >= p.N) continue;
            const uint16_t* src = static_cast<const uint16_t*>(p.residual) + (int64_t)row * p.ld_res + col;
            if (p.vec_res && col + 8 <= p.N) {
                res[i] = *reinterpret_cast<const uint4*>(src);
            } else {
                uint32_t u[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (col + j < p.N) u[j >> 1] |= (uint32_t)src[j] << (16 * (j & 1));
                res[i] = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
    }

    // Rows that TMA cannot store (not on 16-byte boundaries, or a last tile that
    // ends inside 16 bytes): consecutive lanes write consecutive columns.
    static __device__ __forceinline__ void store_rows(const LinearParams& p, const uint8_t* stage, int64_t base, int row0,
                                                      int col0, int lane) {
        using E = typename std::conditional<kF32, float, uint16_t>::type;
        constexpr int kStep = 32 / kC, kBatch = 8;   // rows an instruction, instructions at once
        const int c = lane % kC, first = lane / kC, rows = p.T - row0;
        if (col0 + c >= p.N) return;
        const int unit = c / (kC / 4), in = c % (kC / 4);
        const uint8_t* src = stage + first * 64 + in * (int)sizeof(E);
        E* dst = static_cast<E*>(p.out) + base + (int64_t)(row0 + first) * p.ld_out + col0 + c;
#pragma unroll 1
        for (int r = 0; r < 32; r += kStep * kBatch) {
            E v[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i)         // row r + kStep * i + first
                v[i] = *reinterpret_cast<const E*>(src + (r + kStep * i) * 64 + ((unit ^ ((kStep * i) >> 1 & 3)) * 16));
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                if (r + kStep * i + first < rows) *dst = v[i];
                dst += kStep * p.ld_out;
            }
        }
    }

    template <bool kHalf>
    static __device__ __forceinline__ void run(const LinearParams& p, const CUtensorMap* map, int64_t base,
                                               uint8_t* stage, uint32_t taddr, float st, const float* sc, const float* sb, int row0,
                                               int col0, uint32_t release, int lane) {
        using T16 = typename std::conditional<kHalf, __half, __nv_bfloat16>::type;
        uint4* const mine = reinterpret_cast<uint4*>(stage + lane * 64);
        const int sw = (lane >> 1) & 3;
        const bool add = kRes && p.residual != nullptr;
        const bool biased = !kSwiglu && p.bias != nullptr;
        uint4 next[4];
        if (add) fetch(p, row0, col0, lane, next);
#pragma unroll 1
        for (int n = 0; n < kCols; n += kC) {
            uint32_t a[kC], b[kSwiglu ? kC : 1];
            tmem_ld<kC>(taddr + n, a);
            if constexpr (kSwiglu) tmem_ld<kC>(taddr + kOutN + n, b);
            tmem_wait_ld();
            if (n + kC == kCols) release_acc(release, lane);
            if (row0 >= p.T || col0 + n >= p.N) continue;   // the same for the whole warp
            uint4 r[4];
            if (add) {
                if (lane == 0) bulk_wait_read<0>();         // the last chunk has been read
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int q = lane / 4 + 8 * i;
                    reinterpret_cast<uint4*>(stage + q * 64)[(lane % 4) ^ ((q >> 1) & 3)] = next[i];
                }
                if (n + kC < kCols) fetch(p, row0, col0 + n + kC, lane, next);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 4; ++j) r[j] = mine[j ^ sw];
            }
            uint4 out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                constexpr int kU = kC / 4;                  // columns of a 16-byte unit
                float v[kU];
#pragma unroll
                for (int i = 0; i < kU; i += 4) {
                    const int k = j * kU + i;
                    const float4 w = *reinterpret_cast<const float4*>(sc + n + k);
                    v[i] = dequant(a[k], st, w.x);
                    v[i + 1] = dequant(a[k + 1], st, w.y);
                    v[i + 2] = dequant(a[k + 2], st, w.z);
                    v[i + 3] = dequant(a[k + 3], st, w.w);
                    if constexpr (kSwiglu) {
                        const float4 g = *reinterpret_cast<const float4*>(sc + kOutN + n + k);
                        const float u[4] = {dequant(b[k], st, g.x), dequant(b[k + 1], st, g.y),
                                            dequant(b[k + 2], st, g.z), dequant(b[k + 3], st, g.w)};
#pragma unroll
                        for (int h = 0; h < 4; ++h) v[i + h] = u[h] * silu(v[i + h]);
                    }
                }
                if (biased) {
#pragma unroll
                    for (int i = 0; i < kU; ++i) v[i] += sb[n + j * kU + i];
                }
                if constexpr (kF32) {
                    out[j] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                                        __float_as_uint(v[3]));
                } else {
                    if (add) {
                        const uint32_t u[4] = {r[j].x, r[j].y, r[j].z, r[j].w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 f = F16Traits<T16>::unpack2(u[i]);
                            v[2 * i] += f.x;
                            v[2 * i + 1] += f.y;
                        }
                    }
                    out[j] = make_uint4(F16Traits<T16>::pack2(v[0], v[1]), F16Traits<T16>::pack2(v[2], v[3]),
                                        F16Traits<T16>::pack2(v[4], v[5]), F16Traits<T16>::pack2(v[6], v[7]));
                }
            }
            if (!add) {
                if (lane == 0) bulk_wait_read<0>();
                __syncwarp();
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) mine[j ^ sw] = out[j];
            if (map) {
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    tma_store_2d(map, stage, (col0 + n) * (64 / kC), row0);
                    bulk_commit();
                }
            } else {
                __syncwarp();
                store_rows(p, stage, base, row0, col0 + n, lane);
                __syncwarp();
            }
        }
    }
};

// Tiles of 128 tokens x kBN weight columns (kSwiglu, kBN = 256: 128 gate
// columns, then the same 128 up columns, one output column each).
// split == 1: every CTA walks the tiles with a double-buffered accumulator.
// split > 1 (kBN = 128): a cluster shares one tile, each CTA a part of K; the
// s32 parts meet in shared memory, where CTA r adds up the r-th slice of the
// columns -- integer sums, so the split changes no bit of the result.
// kPair (kBN = 256): two CTAs on a tile of 256 tokens, each with its 128 tokens
// and half of the columns in shared memory; the first one issues the MMAs
// (cta_group::2, M = 256) and every CTA drains its own 128 rows.  A K block then
// brings 32 KB into an SM for the 48 KB of a CTA alone, which is what bounds the
// latter: an SM takes in 64 B/clk, 768 clocks for 512 clocks of MMA.
template <int kBN, bool kSwiglu, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB0,
                  const __grid_constant__ CUtensorMap tmB1, const __grid_constant__ CUtensorMap tmO0,
                  const __grid_constant__ CUtensorMap tmO1, const __grid_constant__ LinearParams p) {
    using C = LinearCfg<kBN, kPair>;
    static_assert(!kPair || kBN == 256, "a pair shares 256 columns");
    static_assert(!kSwiglu || kBN == 256, "the gate and up halves are whole 128-column boxes");
    constexpr int kOutN = kSwiglu ? kBN / 2 : kBN;
    constexpr int kTmemCols = 2 * kBN;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(16) float s_scale[2][kBN];
    __shared__ __align__(16) float s_bias[2][kBN];
    __shared__ uint32_t s_stop;

    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = smem + C::kStages * C::kABytes;
    uint8_t* recv = sB + C::kStages * C::kBBytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(recv + C::kRecvBytes);
    uint64_t* empty = full + C::kStages;
    uint64_t* tfull = empty + C::kStages;
    uint64_t* tempty = tfull + 2;
    uint64_t* bail = tempty + 2;   // of MMAs that were given up
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bail + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    const Waits<false> wait{&s_stop, kPair ? mapa(smem_u32(&s_stop), rank ^ 1) : 0u, kWaitTimeoutNs};

    if (threadIdx.x == 0) {
        s_stop = 0;
        for (int s = 0; s < C::kStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(&tfull[a], 1); mbar_init(&tempty[a], (kPair ? 2 : 1) * kEpiThreads / 32); }
        mbar_init(bail, 1);
        fence_mbar_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB0);
        tma_prefetch_desc(&tmB1);
    }
    if (warp == 1) {
        if (kPair) {
            tmem_alloc2(tmem_slot, kTmemCols);
        } else {
            tmem_alloc(tmem_slot, kTmemCols);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (kPair) {   // the barriers of both CTAs stand before anything arrives on them
        cluster_arrive();
        cluster_wait();
    }
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    // first phase of the cluster barrier: every CTA has started before anything is sent to it
    if (p.split > 1) cluster_arrive();

    const int total = p.m_tiles * p.n_tiles;
    const int ctas = kPair ? 2 : p.split;   // of a tile
    const int tile0 = (int)blockIdx.x / ctas, step = (int)gridDim.x / ctas;
    // this CTA's part of K, in blocks (the host leaves no part empty)
    const int part = kPair ? 0 : rank;
    const int kb0 = (int)((int64_t)p.kblocks * part / p.split);
    const int kb1 = (int)((int64_t)p.kblocks * (part + 1) / p.split);
    const uint32_t stage_bytes = (kPair ? 2u : 1u) * (uint32_t)(p.a_rows * kBK + C::kBBytes);
    const bool leads = !kPair || rank == 0;
    // tile row m of the tokens: this CTA's 128
    auto token_row = [&](int m) { return (kPair ? 2 * m + rank : m) * kBM; };

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- TMA producer ----------------
            auto expect = [&](int s) {
                if (leads) mbar_arrive_expect_tx(&full[s], stage_bytes);   // the loads of both CTAs
            };
            auto load = [&](void* dst, const CUtensorMap* map, int s, int x, int y) {
                if (kPair) tma_load_2d_pair(dst, map, mapa(smem_u32(&full[s]), 0), x, y);
                else tma_load_2d(dst, map, &full[s], x, y);
            };
            auto load_b = [&](int s, int n, int kb) {
                uint8_t* dst = sB + s * C::kBBytes;
                const int k0 = kb * kBK;
                const bool second = !kSwiglu && n >= p.n0_tiles;
                const CUtensorMap* b0 = second ? &tmB1 : &tmB0;
                const CUtensorMap* b1 = kSwiglu || second ? &tmB1 : &tmB0;
                const int col = (second ? n - p.n0_tiles : n) * kOutN;
                if (kPair) {    // this CTA's half, one box (gate or up columns of the fused pass)
                    const int mine = kSwiglu ? col : col + rank * 128;
                    load(dst, rank == 0 ? b0 : b1, s, p.b_nk ? k0 : mine, p.b_nk ? mine : k0);
                } else if (p.b_nk) {   // a box is kBN / 2 rows of N x 128 of K
                    load(dst, b0, s, k0, col);
                    load(dst + C::kBBytes / 2, b1, s, k0, kSwiglu ? col : col + kBN / 2);
                } else {               // a box is 128 rows of K x 128 of N
                    load(dst, b0, s, col, k0);
                    if (kBN == 256) load(dst + C::kBBytes / 2, b1, s, kSwiglu ? col : col + 128, k0);
                }
            };
            // ahead: the kernel before this one is this call's quantiser, which lets this one start after its own
            // wait; whoever wrote the weights came before it and has ended
            int ahead = 0;
            if (p.ahead) {
                for (int kb = kb0; tile0 < total && kb < kb1 && ahead < C::kStages; ++kb, ++ahead) {
                    expect(ahead);
                    load_b(ahead, tile0 / p.m_tiles, kb);
                }
            }
            // No trigger: the kernel behind is mostly a quantiser, whose CTAs would all settle on the SMs that this
            // grid leaves idle (the shared expert of 512 tokens took 54.7 us with one here, 50.1 without).
            pdl_wait();
            int s = 0;
            uint32_t ph = 0;
            for (int t = tile0; t < total; t += step) {
                const int n = t / p.m_tiles, m = t - n * p.m_tiles;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (ahead > 0) {
                        --ahead;
                    } else {
                        if (!wait(&empty[s], ph ^ 1u)) goto producer_done;
                        expect(s);
                        load_b(s, n, kb);
                    }
                    load(sA + s * C::kABytes, &tmA, s, kb * kBK, token_row(m));
                    if (++s == C::kStages) { s = 0; ph ^= 1u; }
                }
            }
        producer_done:;
        }
    } else if (warp == 1) {
        if (lane == 0 && leads) {
            // ---------------- MMA issuer (of a pair, its first CTA's) ----------------
            pdl_wait();   // the bounds of the waits below count from here
            int s = 0;
            uint32_t ph = 0;
            bool gave_up = false;
            // blocks yet to come; a stage is released only for a fill that comes and waits for it, so that no release
            // (of a pair's MMAs, one in the other CTA's memory) can arrive behind the CTA's end
            int64_t left = (int64_t)(total - tile0 + step - 1) / step * (kb1 - kb0);
            int acc = 0;
            uint32_t aph = 0;
            for (int t = tile0; t < total; t += step) {
                if (!wait.cluster(&tempty[acc], aph ^ 1u)) { gave_up = true; break; }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * kBN;
                bool ok = true;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!wait(&full[s], ph)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t a_base = smem_u32(sA + s * C::kABytes);
                    const uint32_t b_base = smem_u32(sB + s * C::kBBytes);
#pragma unroll
                    for (int kk = 0; kk < kBK / 32; ++kk) {
                        // A, and B of [N, K] weights: K-major, 8-row groups 1 KB apart, K step 32 bytes.
                        // B of [K, N] weights: MN-major, 128-column chunks 16 KB apart, K step 32 rows.
                        const uint64_t adesc = smem_desc_sw128(a_base + kk * 32, 16, 1024);
                        const uint64_t bdesc = p.b_nk ? smem_desc_sw128(b_base + kk * 32, 16, 1024)
                                                      : smem_desc_sw128(b_base + kk * 32 * 128, kBK * 128, 1024);
                        if (kPair) mma_i8_ss2(d_tmem, adesc, bdesc, p.idesc, (kb != kb0 || kk != 0) ? 1u : 0u);
                        else mma_i8_ss(d_tmem, adesc, bdesc, p.idesc, (kb != kb0 || kk != 0) ? 1u : 0u);
                    }
                    if (left-- > C::kStages) {
                        if (kPair) mma_commit2(&empty[s]);
                        else mma_commit(&empty[s]);
                    }
                    if (++s == C::kStages) { s = 0; ph ^= 1u; }
                }
                gave_up = !ok;
                if (gave_up) break;
                if (kPair) mma_commit2(&tfull[acc]);
                else mma_commit(&tfull[acc]);
                acc ^= 1;
                if (acc == 0) aph ^= 1u;
            }
            if (gave_up) drain<kPair>(full, s, ph, C::kStages, bail);
        }
    } else {
        // ---------------- epilogue (warps 2..9) ----------------
        pdl_wait();
        if (p.split > 1) cluster_wait();
        constexpr int kCols = kOutN / 2;          // output columns of a warp
        const int q = warp & 3, half = (warp - 2) >> 2;
        const int etid = threadIdx.x - 64;
        uint8_t* const stage = recv + (warp - 2) * 2048;
        int acc = 0;
        uint32_t aph = 0;
        bool ok = true;   // a wait that ran out: the warp keeps to its barriers and writes nothing more
        for (int t = tile0; t < total; t += step) {
            const int n = t / p.m_tiles, m = t - n * p.m_tiles;
            const bool second = !kSwiglu && n >= p.n0_tiles;
            const int tile_col = (second ? n - p.n0_tiles : n) * kOutN, col0 = tile_col + half * kCols;
            // channel scales of the tile, in the order of the accumulator's columns
            float* const scales = s_scale[acc];
            float* const biases = s_bias[acc];
            for (int c = etid; c < kBN; c += kEpiThreads) {
                const int col = tile_col + (kSwiglu ? c % kOutN : c);
                const float* src = second || (kSwiglu && c >= kOutN) ? p.s_ch1 : p.s_ch0;
                scales[c] = col < p.N ? src[col] : 0.0f;
                biases[c] = !kSwiglu && p.bias && col < p.N ? p.bias[col] : 0.0f;
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float* const sc = scales + half * kCols;
            const float* const sb = biases + half * kCols;
            const int row0 = token_row(m) + q * 32, row = row0 + lane;
            const bool valid = row < p.T;
            const uint32_t release = mapa(smem_u32(&tempty[acc]), kPair ? 0 : rank);
            const float st = valid ? p.s_tok[row] : 0.0f;
            const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + acc * kBN + half * kCols;
            if (p.staged && p.residual) StagedEpilogue<kCols, kOutN, false, false>::prefetch_residual(p, row, col0);
            if (ok) ok = wait.warp(&tfull[acc], aph);
            tc_fence_after();
            if (ok && p.staged) {
                // TMA stores clip rows at 16-byte units: not for a last tile that ends inside one
                const CUtensorMap* map =
                    !p.tma_out || !(p.row_end16 || tile_col + kOutN <= p.N) ? nullptr : second ? &tmO1 : &tmO0;
                const int64_t base = second ? p.out1 : 0;
                if (kSwiglu || p.out_type == MOE_TYPE_F32)
                    StagedEpilogue<kCols, kOutN, kSwiglu, true>::template run<false>(p, map, base, stage, taddr, st, sc, sb,
                                                                                     row0, col0, release, lane);
                else if (p.out_type == MOE_TYPE_F16)
                    StagedEpilogue<kCols, kOutN, false, kSwiglu>::template run<true>(p, map, base, stage, taddr, st, sc, sb,
                                                                                     row0, col0, release, lane);
                else
                    StagedEpilogue<kCols, kOutN, false, kSwiglu>::template run<false>(p, map, base, stage, taddr, st, sc, sb,
                                                                                      row0, col0, release, lane);
            } else if (ok && p.split == 1) {
#pragma unroll 1
                for (int c = 0; c < kCols; c += 16) {
                    uint32_t a[16], b[16];
                    tmem_ld_32x32b_x16(taddr + c, a);
                    if (kSwiglu) tmem_ld_32x32b_x16(taddr + kOutN + c, b);
                    tmem_wait_ld();
                    if (c + 16 == kCols) release_acc(release, lane);
                    if (!valid) continue;
#pragma unroll
                    for (int h = 0; h < 16; h += 8) {
                        float v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            v[i] = dequant(a[h + i], st, sc[c + h + i]);
                            if (kSwiglu) v[i] = dequant(b[h + i], st, sc[kOutN + c + h + i]) * silu(v[i]);
                            else v[i] += sb[c + h + i];
                        }
                        if (col0 + c + h < p.N) emit8(p, row, second, col0 + c + h, v);
                    }
                }
            } else if (ok) {
                if constexpr (kBN == 128) {
                    // send the parts in units of eight columns: [source][unit of the slice][row][8]
                    if (row0 < p.T) {   // a warp without a token has nothing to send
                        const int units = kBN / 8 / p.split;
#pragma unroll 1
                        for (int u = half * 8; u < half * 8 + 8; u += 4) {
                            uint32_t a[32];
                            tmem_ld_32x32b_x32(taddr + 8 * (u - half * 8), a);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int at = u + i;
                                const uint32_t dst = mapa(
                                    smem_u32(recv) +
                                        (uint32_t)((rank * units + at % units) * kUnitBytes + (q * 32 + lane) * 32),
                                    at / units);
                                st_cluster4(dst, a[8 * i], a[8 * i + 1], a[8 * i + 2], a[8 * i + 3]);
                                st_cluster4(dst + 16, a[8 * i + 4], a[8 * i + 5], a[8 * i + 6], a[8 * i + 7]);
                            }
                        }
                    }
                }
            }
            acc ^= 1;
            if (acc == 0) aph ^= 1u;
        }
        if (p.split > 1 && !ok) tell_cluster(smem_u32(&s_stop), p.split);
        if (lane == 0) bulk_wait_read<0>();   // the staged chunks are read before the CTA's memory goes
    }
    if (p.split > 1) {
        __syncwarp();
        if (warp < 2) cluster_wait();   // the first phase, which the epilogue warps have waited for above
        cluster_arrive();               // second phase: every part has been sent
        cluster_wait();
        if constexpr (kBN == 128 && !kSwiglu) {
            const int n = tile0 / p.m_tiles, m = tile0 - n * p.m_tiles;   // one tile a cluster
            const bool second = n >= p.n0_tiles;
            const int col0 = (second ? n - p.n0_tiles : n) * kOutN;
            // this CTA's 128 / split columns: consecutive lanes take consecutive units of a row
            const int units = kBN / 8 / p.split, rows = min(kBM, p.T - m * kBM);
            const bool all = !wait.stopped();   // else a part is missing
            for (int i = threadIdx.x - 64; i >= 0 && i < units * rows; i += kEpiThreads) {
                const int u = i % units, r = i / units, c = (rank * units + u) * 8;
                if (col0 + c >= p.N) continue;
                int sum[8] = {};
                for (int src = 0; src < p.split; ++src) {
                    const int4* a = reinterpret_cast<const int4*>(recv + (src * units + u) * kUnitBytes + r * 32);
                    const int4 x = a[0], y = a[1];
                    sum[0] += x.x; sum[1] += x.y; sum[2] += x.z; sum[3] += x.w;
                    sum[4] += y.x; sum[5] += y.y; sum[6] += y.z; sum[7] += y.w;
                }
                const int64_t row = (int64_t)m * kBM + r;
                const float st = p.s_tok[row];
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = dequant(sum[j], st, s_scale[0][c + j]) + s_bias[0][c + j];
                if (all) emit8(p, row, second, col0 + c, v);
            }
        }
    }
    if (kPair) {   // the first CTA's MMAs read both CTAs' memory, and both release into the first's barriers
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        if (kPair) tmem_dealloc2(tmem_base, kTmemCols);
        else tmem_dealloc(tmem_base, kTmemCols);
    }
}

// ---- product of a few tokens ---------------------------------------------------------

// Up to kNT tokens in one launch, quantiser included.  The product is turned
// round: the 128 weight columns of a tile are the rows of the MMA (M = 128) and
// the tokens its columns (N = kNT), so a thread of the epilogue holds one
// channel's sums of all tokens and consecutive lanes write consecutive columns.
// A cluster of `split` CTAs shares a tile, each a part of K.  Each CTA asks for
// its weights at once, reads the tokens for their amax (short rows whole; of long
// ones its part, the cluster exchanging what it finds), then its part again for
// the codes, written where the MMA reads them, and hands the s32 sums of each
// slice of the channels to the CTA that adds them up.
// kSwiglu: the tile is 128 features, their gate and up columns are multiplied in
// turn (two accumulators), and h = up * silu(gate) is written.
// What bounds it is latency: 512 x 2048 takes 4.5 us (3.1 with codes given), an
// exchange of a cluster about 1, and the MMAs, 128 clocks each whatever their
// columns, 0.27 us for each block of K; the 14.7 MB of weights of 1 x 7168 x 2048
// (6.8 us, 8.7 when none of them is in the L2) are 2.2 us at the HBM's rate.
// Kept short for one reason more: a code path that a CTA runs once is fetched as
// slowly as it is long (the quantiser of gate / up pairs, 96 times silu in line,
// cost the down product 17 us).
struct SmallParams {
    const void* x;             // tokens, rows ld_x elements apart
    int64_t ld_x;
    const float* s_tok;        // codes given: their scales
    int T, K, N;
    int kblocks, split, stages;
    int b_nk, ahead, vec_x;
    int exchange;              // each CTA takes its part's amax and the cluster exchanges them; else every CTA the rows'
    const float* s_ch0;
    const float* s_ch1;
    const float* bias;
    const void* residual;
    int64_t ld_res;
    int res_type;
    void* out;
    int64_t ld_out;
    int out_type;
    uint32_t idesc;
};

enum SmallInput { kInF32, kInF16, kInBF16, kInCodes };
template <int kIn> struct SmallIn { using T = float; };
template <> struct SmallIn<kInF16> { using T = __half; };
template <> struct SmallIn<kInBF16> { using T = __nv_bfloat16; };
template <> struct SmallIn<kInCodes> { using T = int8_t; };

constexpr int kSmallWorkers = 256;
constexpr int kSmallThreads = 64 + kSmallWorkers;
constexpr int kSmallStageBytes = 128 * kBK;

// Shared memory behind the aligned base: weight stages, code blocks, parts, barriers.
template <int kNT> __host__ __device__ constexpr size_t small_smem(int stages, int blocks, int split, int mats) {
    return 1024 + (size_t)stages * kSmallStageBytes + (size_t)blocks * kNT * kBK +
           (split > 1 ? (size_t)mats * 128 * kNT * 4 : 0) + 256;
}

template <int kNT, int kIn, bool kSwiglu>
__global__ void __launch_bounds__(kSmallThreads, 2)
    small_linear_kernel(const __grid_constant__ CUtensorMap tmW0, const __grid_constant__ CUtensorMap tmW1,
                        const __grid_constant__ SmallParams p) {
    using T = typename SmallIn<kIn>::T;
    constexpr int kMats = kSwiglu ? 2 : 1;
    constexpr int kTmemCols = 32;
    static_assert(kMats * kNT <= kTmemCols, "one accumulator for each matrix");
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t s_amax[kMaxSplit][kNT];   // [source CTA][token]: bits of the largest magnitude
    __shared__ float s_tok[kNT];
    __shared__ uint32_t s_stop;

    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int rank = p.split > 1 ? (int)cluster_rank() : 0;
    const int kb0 = (int)((int64_t)p.kblocks * rank / p.split);
    const int kb1 = (int)((int64_t)p.kblocks * (rank + 1) / p.split);
    const int max_blocks = (p.kblocks + p.split - 1) / p.split;
    uint8_t* const sW = smem;
    uint8_t* const sQ = sW + p.stages * kSmallStageBytes;
    uint8_t* const recv = sQ + (size_t)max_blocks * kNT * kBK;
    uint64_t* const full = reinterpret_cast<uint64_t*>(recv + (p.split > 1 ? kMats * 128 * kNT * 4 : 0));
    uint64_t* const empty = full + 8;
    uint64_t* const ready = empty + 8;   // the codes are written
    uint64_t* const tfull = ready + 1;
    uint64_t* const bail = tfull + 1;    // of MMAs that were given up
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bail + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Waits<true> wait{&s_stop, 0u, kWaitTimeoutNs};
    if (threadIdx.x == 0) {
        s_stop = 0;
        for (int s = 0; s < p.stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_init(ready, kSmallWorkers);
        mbar_init(tfull, 1);
        mbar_init(bail, 1);
        fence_mbar_init();
        tma_prefetch_desc(&tmW0);
        tma_prefetch_desc(&tmW1);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const bool split = p.split > 1, exchange = split && kIn != kInCodes && p.exchange;
    if (split) cluster_arrive();   // phase 1: every CTA has started

    const int col0 = (int)blockIdx.x / p.split * 128;
    const int loads = (kb1 - kb0) * kMats;   // weight boxes of this CTA: block by block, gate before up

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        auto load = [&](int s, int i) {
            const CUtensorMap* map = kSwiglu && (i & 1) ? &tmW1 : &tmW0;
            const int k = (kb0 + i / kMats) * kBK;
            mbar_arrive_expect_tx(&full[s], kSmallStageBytes);
            if (p.b_nk) tma_load_2d(sW + s * kSmallStageBytes, map, &full[s], k, col0);
            else tma_load_2d(sW + s * kSmallStageBytes, map, &full[s], col0, k);
        };
        const int first = min(p.stages, loads);
        if (lane == 0) {
            if (!p.ahead) pdl_wait();
            for (int i = 0; i < first; ++i) load(i, i);
            if (p.ahead) pdl_wait();
            pdl_trigger();
        }
        __syncwarp();
        if (split) cluster_wait();   // phase 1; and 2, before any wait that the other warps' progress ends
        if (exchange) {
            cluster_arrive();
            cluster_wait();
        }
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            for (int i = first; i < loads; ++i) {
                if (!wait(&empty[s], ph)) break;
                load(s, i);
                if (++s == p.stages) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        if (split) cluster_wait();
        if (exchange) {
            cluster_arrive();
            cluster_wait();
        }
        if (lane == 0) {
            pdl_wait();   // the bounds of the waits below count from here
            bool ok = wait(ready, 0);
            int s = 0;
            uint32_t ph = 0;
            for (int i = 0; ok && i < loads; ++i) {
                if (!wait(&full[s], ph)) { ok = false; break; }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + (kSwiglu ? (i & 1) * kNT : 0);
                const uint32_t w_base = smem_u32(sW + s * kSmallStageBytes);
                const uint32_t q_base = smem_u32(sQ + (size_t)(i / kMats) * kNT * kBK);
#pragma unroll
                for (int kk = 0; kk < kBK / 32; ++kk) {
                    // weights [N, K]: K-major rows; [K, N]: MN-major, a K step is 32 rows of 128 bytes
                    const uint64_t wdesc = p.b_nk ? smem_desc_sw128(w_base + kk * 32, 16, 1024)
                                                  : smem_desc_sw128(w_base + kk * 32 * 128, kBK * 128, 1024);
                    mma_i8_ss(d_tmem, wdesc, smem_desc_sw128(q_base + kk * 32, 16, 1024), p.idesc,
                              (i >= kMats || kk != 0) ? 1u : 0u);
                }
                if (i + p.stages < loads) mma_commit(&empty[s]);   // (as the tiles: only for a load that waits for it)
                if (++s == p.stages) { s = 0; ph ^= 1u; }
            }
            if (ok) mma_commit(tfull);
            else drain<false>(full, s, ph, p.stages, bail);
        }
    } else {
        // ---------------- quantiser, then epilogue (warps 2..9) ----------------
        pdl_wait();
        const int w = warp - 2;
        const int k0 = kb0 * kBK, k1 = min(p.K, kb1 * kBK);
        const T* const x = static_cast<const T*>(p.x);
        if constexpr (kIn != kInCodes) {
            // a warp takes tokens w, w + 8; with up to 4 the warps share a token's units of eight
            const int share = p.T > 4 ? 1 : p.T > 2 ? 2 : p.T > 1 ? 4 : 8;   // warps of a token
            const int tok0 = w / share, tstep = 8 / share;
            const int u0 = (w % share) * 32 + lane, ustep = 32 * share * 8;
            constexpr int kBatch = 4;
            // units k, k + ustep, .. of token t below `end`, all asked for before any is used
            auto fetch = [&](In8<T> (&d)[kBatch], int t, int k, int end) {
                const T* src = x + t * p.ld_x;
                if (p.vec_x && end % 8 == 0) {
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {
                        d[i].zero();
                        if (t < p.T && k + i * ustep < end) d[i].load(src + k + i * ustep);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {
                        d[i].zero();
                        if (t < p.T && k + i * ustep < end) d[i].load_part(src + k + i * ustep, end - k - i * ustep);
                    }
                }
            };
            const int from = exchange ? k0 : 0, to = exchange ? k1 : p.K, slot = exchange ? rank : 0;   // of the amax
            if (threadIdx.x - 64 < kNT) s_amax[slot][threadIdx.x - 64] = 0u;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            for (int t = tok0; t < p.T; t += 2 * tstep) {
                uint32_t m[2] = {0u, 0u};
                for (int k = from + u0 * 8; k - u0 * 8 < to; k += kBatch * ustep) {
                    In8<T> d[2][kBatch];
                    fetch(d[0], t, k, to);
                    fetch(d[1], t + tstep, k, to);
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {
                        m[0] = max(m[0], d[0][i].amax_bits());
                        m[1] = max(m[1], d[1][i].amax_bits());
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    m[h] = __reduce_max_sync(0xffffffffu, m[h]);
                    if (lane == 0 && t + h * tstep < p.T) atomicMax(&s_amax[slot][t + h * tstep], m[h]);
                }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (exchange) {
                cluster_wait();   // phase 1
                for (int i = threadIdx.x - 64; i < p.T * p.split; i += kSmallWorkers) {
                    const int cta = i / p.T, t = i % p.T;
                    if (cta != rank)
                        asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(mapa(smem_u32(&s_amax[rank][t]), cta)),
                                     "r"(s_amax[rank][t])
                                     : "memory");
                }
                __syncwarp();
                cluster_arrive();   // phase 2: every part's amax is here
                cluster_wait();
            }
            for (int t = tok0; t < p.T; t += tstep) {
                uint32_t m = s_amax[0][t];
                if (exchange)
                    for (int r = 1; r < p.split; ++r) m = max(m, s_amax[r][t]);
                const RowScale rs(m);
                if (u0 == 0) s_tok[t] = rs.s;
                for (int k = k0 + u0 * 8; k - u0 * 8 < k1; k += kBatch * ustep) {
                    In8<T> d[kBatch];
                    fetch(d, t, k, k1);
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {
                        const int kk = k + i * ustep - k0;
                        if (kk >= k1 - k0) continue;
                        float f[8];
                        d[i].get(f);
                        // K-major, 128-byte swizzle: 16-byte unit j of row t at j ^ (t & 7)
                        uint8_t* dst = sQ + (size_t)(kk / kBK) * kNT * kBK + t * 128 +
                                       ((((kk & 127) >> 4) ^ (t & 7)) << 4) + (kk & 8);
                        *reinterpret_cast<uint2*>(dst) = rs.codes(f);
                    }
                }
            }
        } else {
            if (threadIdx.x - 64 < p.T) s_tok[threadIdx.x - 64] = p.s_tok[threadIdx.x - 64];
            const int units = (k1 - k0 + 15) / 16;   // rows start on 16-byte boundaries
            for (int i = threadIdx.x - 64; i < units * p.T; i += kSmallWorkers) {
                const int t = i / units, kk = (i - t * units) * 16;
                const int8_t* src = x + t * p.ld_x + k0 + kk;
                union { uint4 v; int8_t b[16]; } q;
                if (k0 + kk + 16 <= k1) {
                    q.v = *reinterpret_cast<const uint4*>(src);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) q.b[j] = k0 + kk + j < k1 ? src[j] : (int8_t)0;
                }
                *reinterpret_cast<uint4*>(sQ + (size_t)(kk / kBK) * kNT * kBK + t * 128 +
                                          ((((kk & 127) >> 4) ^ (t & 7)) << 4)) = q.v;
            }
        }
        fence_async_smem();
        mbar_arrive(ready);
        asm volatile("bar.sync 1, 256;" ::: "memory");   // s_tok

        // a thread: channel c, half of the tokens
        constexpr int kHalfTok = kNT / 2;
        const int q = warp & 3, half = w >> 2, c = q * 32 + lane, tok = half * kHalfTok;
        if (split && !exchange) cluster_wait();   // phase 1
        const bool ok = wait.warp(tfull, 0);
        tc_fence_after();
        const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + tok;
        auto put = [&](int sum, int sum1, int t, int ch) {   // channel ch of the tile
            const int col = col0 + ch;
            if (col >= p.N) return;
            float v = dequant(sum, s_tok[t], p.s_ch0[col]);
            if (kSwiglu) v = dequant(sum1, s_tok[t], p.s_ch1[col]) * silu(v);
            if (p.bias) v += p.bias[col];
            if (p.residual) v += load_as_f32(p.residual, t * p.ld_res + col, p.res_type);
            const int64_t at = t * p.ld_out + col;
            if (p.out_type == MOE_TYPE_F32) static_cast<float*>(p.out)[at] = v;
            else if (p.out_type == MOE_TYPE_F16) static_cast<__half*>(p.out)[at] = __float2half_rn(v);
            else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
        };
        const int wch = 128 / p.split;              // channels of a slice
        static_assert(kHalfTok == 8, "a thread reads its tokens at once");
        if (ok && tok < p.T) {                      // the same for the whole warp
            uint32_t a[kMats][8];
#pragma unroll
            for (int j = 0; j < kMats; ++j) tmem_ld_32x32b_x8(taddr + j * kNT, a[j]);
            tmem_wait_ld();
            if (!split) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (tok + i < p.T) put((int)a[0][i], (int)a[kMats - 1][i], tok + i, c);
            } else {
                // parts: [matrix][source][token / 4][channel of the slice][4 tokens]
#pragma unroll
                for (int j = 0; j < kMats; ++j)
#pragma unroll
                    for (int i = 0; i < 8; i += 4) {
                        if (tok + i >= p.T) break;
                        const uint32_t at = (uint32_t)(j * 128 * kNT * 4 +
                                                       ((rank * (kNT / 4) + (tok + i) / 4) * wch + c % wch) * 16);
                        st_cluster4(mapa(smem_u32(recv) + at, c / wch), a[j][i], a[j][i + 1], a[j][i + 2], a[j][i + 3]);
                    }
            }
        }
        if (split) {
            if (!ok) tell_cluster(smem_u32(&s_stop), p.split);
            __syncwarp();
            cluster_arrive();   // phase 3: every part has been sent
            cluster_wait();
            const int* parts = reinterpret_cast<const int*>(recv);
            const bool all = !wait.stopped();   // else a part is missing
            for (int i = threadIdx.x - 64; i < wch * p.T; i += kSmallWorkers) {
                const int t = i / wch, ch = i % wch;
                int sum[kMats] = {};
                for (int r = 0; r < p.split; ++r)
#pragma unroll
                    for (int j = 0; j < kMats; ++j)
                        sum[j] += parts[j * 128 * kNT + ((r * (kNT / 4) + t / 4) * wch + ch) * 4 + t % 4];
                if (all) put(sum[0], sum[kMats - 1], t, rank * wch + ch);
            }
        }
    }
    if (split && warp < 2) {
        __syncwarp();
        cluster_arrive();       // phase 3
        cluster_wait();
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

// ---- self-test of the waits ------------------------------------------------------------

// A cluster of two whose second CTA waits for what nothing completes; then each
// CTA writes its word, unless it has been told to stop.
__global__ void __launch_bounds__(32) waits_selftest_kernel(uint64_t limit_ns, int* written) {
    __shared__ __align__(8) uint64_t bar;
    __shared__ uint32_t s_stop;
    const int rank = (int)cluster_rank();
    if (threadIdx.x == 0) {
        s_stop = 0;
        mbar_init(&bar, 1);
        fence_mbar_init();
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    const Waits<true> wait{&s_stop, 0u, limit_ns};
    if (rank == 1 && !wait.warp(&bar, 0)) tell_cluster(smem_u32(&s_stop), 2);
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (threadIdx.x == 0 && !wait.stopped()) written[rank] = 1;
}

// ---- host side -----------------------------------------------------------------------

// SMs the tile rules count on (B200).
constexpr int kRuleSms = 148;
constexpr int kMaxK = 131071;   // 128 * 128 * K stays below 2^31

int elem_bytes(int type) { return type == MOE_TYPE_F32 ? 4 : 2; }
bool is_type(int t) { return t == MOE_TYPE_F32 || t == MOE_TYPE_F16 || t == MOE_TYPE_BF16; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }
size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

template <typename... P, typename... A>
cudaError_t launch_ex(void (*kern)(P...), unsigned grid, unsigned threads, size_t smem, int cluster, cudaStream_t st,
                      A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (cluster > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim = {(unsigned)cluster, 1, 1};
        ++n;
    }
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // (see pdl_wait)
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
    cfg.attrs = at;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kern, P(args)...);
}

template <typename T, bool kPair>
cudaError_t launch_quantize_typed(const T* x, int64_t rows, int K, int64_t ldx, int64_t up, int8_t* q, int64_t ldq,
                                  float* s, int num_sms, cudaStream_t st) {
    const int vec = aligned(x, 16) && (ldx * (int64_t)sizeof(T)) % 16 == 0;
    // As many threads a row as hold it in registers, four vectors of eight each; one each for few rows, where the
    // chain through a row counts and not the CTAs on an SM.  Measured (us, four / one): 64 x 2048 bf16 2.6 / 1.7,
    // 512 x 2048 2.8 / 2.6, 1024 x 2048 3.4 / 3.9; f32 256 x 2048 2.4 / 1.9, 512 x 2048 2.4 / 3.0.
    const int span = rows <= (sizeof(T) == 2 || kPair ? 4 : 2) * num_sms ? 256 : 1024;
    const int tpr = K <= span ? 32 : K <= 2 * span ? 64 : K <= 4 * span ? 128 : 256;
    const int64_t blocks = (rows * tpr + 255) / 256;
    auto kern = tpr == 32    ? quantize_tokens_kernel<T, 32, kPair>
                : tpr == 64  ? quantize_tokens_kernel<T, 64, kPair>
                : tpr == 128 ? quantize_tokens_kernel<T, 128, kPair>
                             : quantize_tokens_kernel<T, 256, kPair>;
    return launch_ex(kern, (unsigned)blocks, 256u, 0, 1, st, x, rows, K, ldx, up, q, ldq, s, vec);
}

// up != 0: x holds f32 gate values with the up values `up` elements behind.
cudaError_t launch_quantize(const void* x, int type, int64_t rows, int K, int64_t ldx, int64_t up, int8_t* q,
                            int64_t ldq, float* s, int num_sms, cudaStream_t st) {
    if (up != 0)
        return launch_quantize_typed<float, true>(static_cast<const float*>(x), rows, K, ldx, up, q, ldq, s, num_sms, st);
    switch (type) {
        case MOE_TYPE_F32:
            return launch_quantize_typed<float, false>(static_cast<const float*>(x), rows, K, ldx, 0, q, ldq, s, num_sms, st);
        case MOE_TYPE_F16:
            return launch_quantize_typed<__half, false>(static_cast<const __half*>(x), rows, K, ldx, 0, q, ldq, s, num_sms, st);
        default:
            return launch_quantize_typed<__nv_bfloat16, false>(static_cast<const __nv_bfloat16*>(x), rows, K, ldx, 0, q,
                                                               ldq, s, num_sms, st);
    }
}

template <int kBN, bool kSwiglu, bool kPair>
cudaError_t launch_linear_cfg(const CUtensorMap& a, const CUtensorMap (&b)[2], const CUtensorMap (&o)[2],
                              const LinearParams& p, int clusters, cudaStream_t st) {
    auto kern = linear_kernel<kBN, kSwiglu, kPair>;
    static SmemAttr attr;
    const size_t smem = LinearCfg<kBN, kPair>::kSmem;
    const int ctas = kPair ? 2 : p.split;
    cudaError_t err = ensure_smem(kern, smem, attr);
    if (err != cudaSuccess) return err;
    return launch_ex(kern, (unsigned)(clusters * ctas), (unsigned)kThreads, smem, ctas, st, a, b[0], b[1],
                     o[0], o[1], p);
}

// Tiles and split of K, by the estimated time of a launch: rounds of tiles over
// the SMs x K blocks of a tile x the time of a block, plus what a launch costs
// besides.  A block takes 0.34 us at 128 x 128, 0.43 at 128 x 256 and 0.36 at 256 x
// 256 on two SMs (a CTA alone is bound by what an SM takes in, 64 B/clk: 32 and 48
// KB); a launch 3.5 us, a pair's 4.5, a split one 4.8 and up to 4 more for sending
// the parts of 128 tokens.  Clusters of 4 and 8 CTAs of this size fit 33 and 15
// times at once.  Measured (us; T x K x N: pair, 128 x 256, 128 x 128 with K split
// 1 / 2 / 4 / 8 times): 16x7168x2048 21.5, 21.2, 19.3 / 13.0 / 9.8 / 15.2;
// 128x7168x2048 22.5, 22.2, 20.3 / 16.3 / 13.6 / 22.5; 512x7168x2048 22.8, 22.8,
// 20.9 / 17.6 / 28.7 / 59; 512x2048x7168 12.5, 12.1, 16.0 / 41.6 / 75.6 / 155;
// 1024x2048x2048 12.1, 11.7, 10.8 / 22.4 / 44.5 / 92; 2048x7168x2048 25.0, 26.6,
// 39.4 / 66 / 109 / 205; 8192x7168x4096 159, 201, 270 / 455 / 791 / 1577.  The
// estimate leaves out the epilogue, which a CTA's only tile does not hide: at
// 512x2048x7168 it puts the pair 1 % ahead of 128 x 256, which measured 3 % faster.
struct Tiles {
    bool wide, pair;
    int split;
};
Tiles pick_tiles(int T, int N, int kblocks, int mats, bool swiglu, int num_sms) {
    auto rounds = [](int64_t n, int64_t at_once) { return (double)((n + at_once - 1) / at_once); };
    const int64_t m128 = (T + 127) / 128, m256 = (T + 255) / 256;
    const int64_t n128 = (int64_t)((N + 127) / 128) * mats, n256 = swiglu ? n128 : (int64_t)((N + 255) / 256) * mats;
    double best = 3.5 + rounds(m128 * n256, num_sms) * kblocks * 0.43;
    Tiles pick{true, false, 1};
    const double pair = 4.5 + rounds(m256 * n256, num_sms / 2) * kblocks * 0.36;
    if (num_sms >= 2 && pair < best) {
        best = pair;
        pick.pair = true;
    }
    for (int s = 1; !swiglu && s <= kMaxSplit && s <= kblocks; s *= 2) {
        const int64_t at_once = s == 1 ? num_sms : s == 2 ? num_sms / 2 : s == 4 ? num_sms * 33 / 148 : num_sms * 15 / 148;
        if (at_once < 1 || (s > 1 && m128 * n128 > at_once)) break;   // a split tile's CTAs run one tile each
        const double t = (s == 1 ? 3.5 : 4.8 + 4.0 * std::min(T, kBM) / kBM) +
                         rounds(m128 * n128, at_once) * ((kblocks + s - 1) / s) * 0.34;
        if (t < best) {
            best = t;
            pick = Tiles{false, false, s};
        }
    }
    return pick;
}

struct Matrix {
    const int8_t* w;
    int64_t ld;
    const float* scale;
};

// One product over one matrix, two of the same shape side by side (w1: the
// second's outputs start out1 elements behind the first's), or (swiglu) the
// gate and up matrices of h.
cudaError_t launch_linear(const int8_t* q, int64_t ldq, LinearParams p, const Matrix& w0, const Matrix* w1, bool swiglu,
                          int num_sms, cudaStream_t st) {
    p.kblocks = (p.K + kBK - 1) / kBK;
    const int mats = w1 && !swiglu ? 2 : 1;
    const Tiles tiles = pick_tiles(p.T, p.N, p.kblocks, mats, swiglu, num_sms);
    const bool pair = tiles.pair;
    p.split = tiles.split;
    p.m_tiles = pair ? (p.T + 2 * kBM - 1) / (2 * kBM) : (p.T + kBM - 1) / kBM;
    p.a_rows = pair || p.T >= kBM ? kBM : (p.T + 7) / 8 * 8;
    const int bn = tiles.wide ? 256 : 128;
    const int out_n = swiglu ? bn / 2 : bn;
    p.n0_tiles = (p.N + out_n - 1) / out_n;
    p.n_tiles = p.n0_tiles * mats;
    p.s_ch0 = w0.scale;
    p.s_ch1 = w1 ? w1->scale : w0.scale;
    p.idesc = idesc_i8(pair ? 2 * kBM : kBM, bn, !p.b_nk);
    CUtensorMap ta, tb[2], to[2] = {};
    if (!make_map_u8_strided(&ta, q, p.K, p.T, ldq, 128, p.a_rows)) return cudaErrorInvalidValue;
    const Matrix* ws[2] = {&w0, w1 ? w1 : &w0};
    for (int i = 0; i < 2; ++i) {
        const bool ok = p.b_nk ? make_map_u8_strided(&tb[i], ws[i]->w, p.K, p.N, ws[i]->ld, 128, bn / 2)
                               : make_map_u8_strided(&tb[i], ws[i]->w, p.N, p.K, ws[i]->ld, 128, kBK);
        if (!ok) return cudaErrorInvalidValue;
    }
    const int size = elem_bytes(p.out_type);
    p.row_end16 = (int64_t)p.N * size % 16 == 0;
    p.staged = p.split == 1 && (!p.residual || (size == 2 && p.res_type == p.out_type));
    p.tma_out = p.staged && p.vec_out;
    for (int i = 0; p.tma_out && i < mats; ++i)
        if (!make_map_u8_strided(&to[i], static_cast<uint8_t*>(p.out) + i * p.out1 * size, (uint64_t)p.N * size, p.T,
                                 (uint64_t)p.ld_out * size, 64, 32))
            return cudaErrorInvalidValue;
    const int64_t count = (int64_t)p.m_tiles * p.n_tiles;
    const int clusters = (int)(p.split > 1 ? count : std::min<int64_t>(count, pair ? num_sms / 2 : num_sms));
    if (pair)
        return swiglu ? launch_linear_cfg<256, true, true>(ta, tb, to, p, clusters, st)
                      : launch_linear_cfg<256, false, true>(ta, tb, to, p, clusters, st);
    if (swiglu) return launch_linear_cfg<256, true, false>(ta, tb, to, p, clusters, st);
    if (tiles.wide) return launch_linear_cfg<256, false, false>(ta, tb, to, p, clusters, st);
    return launch_linear_cfg<128, false, false>(ta, tb, to, p, clusters, st);
}

// Up to this many tokens small_linear_kernel is used: with its own quantiser, or
// on codes (given, or of the quantiser's launch).  Measured (us a call; one launch,
// quantiser + small kernel, quantiser + tiles): int8_linear 7168 -> 2048 of 1 token
// 7.3, 8.4, 11.1, 4 tokens 8.2, 8.4, 10.6, 8 tokens 8.9, 8.9, 10.7, 16 tokens 11.0,
// 9.5, 10.8; 2048 -> 7168 of 8 tokens 8.4, 8.1, 8.9, 16 tokens 10.4, 9.3, 9.2;
// int8_matmul 7168 -> 2048 of 16 codes 6.7, by tiles 9.5; shared expert 7168 / 2048
// of 1 token 20.2, 22.0, 22.8, 4 tokens 21.1, 21.5, 22.6, 8 tokens 22.7, 22.6, 22.7,
// 16 tokens 26.8, 24.4, 23.1.
constexpr int kSmallLinear = 4, kSmallCodes = 16;   // gate / up: its own quantiser as the linear's
constexpr int kSmallPairs = 8;                      // gate / up on codes
constexpr int kSmallN = 16;
constexpr int kSmallStages = 5, kSmallMinStages = 3;
constexpr size_t kSmallSmem = 112 * 1024;   // two CTAs an SM

template <int kIn, bool kSwiglu>
cudaError_t launch_small_typed(const CUtensorMap (&w)[2], const SmallParams& p, int tiles, size_t smem, cudaStream_t st) {
    auto kern = small_linear_kernel<kSmallN, kIn, kSwiglu>;
    static SmemAttr attr;
    cudaError_t err = ensure_smem(kern, kSmallSmem, attr);   // one limit: threads may call at once
    if (err != cudaSuccess) return err;
    return launch_ex(kern, (unsigned)(tiles * p.split), (unsigned)kSmallThreads, smem, p.split, st, w[0], w[1],
                     p);
}

// Whether a call's codes fit beside the weight stages at some split with all of
// its CTAs resident at once (two an SM); the largest such split.  More CTAs are
// left to the persistent tiles (us, here / there, 1 token: 7168 x 8192 14.1 / 17.7,
// all at once; 7168 x 14336 26.7 / 25.8, 7168 x 28672 51.3 / 37.1, in rounds).
// The counts are a whole B200's: the scratch sizes follow the choice and are asked
// for without a device.  With fewer SMs the CTAs run in rounds, slower.
bool plan_small(int64_t T, int limit, int K, int N, int mats, int* split, int* stages, size_t* smem) {
    if (T > limit) return false;
    const int kblocks = (K + kBK - 1) / kBK, tiles = (N + 127) / 128;
    *split = 0;
    for (int s = 1; s <= kMaxSplit && s <= kblocks; s *= 2) {
        const int blocks = (kblocks + s - 1) / s;
        int st = std::min(kSmallStages, blocks * mats);
        while (st > kSmallMinStages && small_smem<kSmallN>(st, blocks, s, mats) > kSmallSmem) --st;
        const size_t need = small_smem<kSmallN>(st, blocks, s, mats);
        if (need > kSmallSmem) continue;
        // clusters of 1, 2, 4 and 8 CTAs of up to half an SM's memory fit 296, 148, 71 and 33 times
        if (tiles > (s == 1 ? 2 * kRuleSms : s == 2 ? kRuleSms : s == 4 ? 71 : 33)) break;
        *split = s;
        *stages = st;
        *smem = need;
    }
    return *split != 0;
}

// A product of few tokens in one launch (w1: gate and up, h written); x_type:
// MOE_TYPE_* of x, or -1 for codes.  False where the shape needs the tiles.
bool try_small(int limit, const void* x, int x_type, int64_t ld_x, const LinearParams& l, const Matrix& w0, const Matrix* w1,
               cudaStream_t st, cudaError_t* err) {
    int split, stages;
    size_t smem;
    const int mats = w1 ? 2 : 1;
    if (!plan_small(l.T, limit, l.K, l.N, mats, &split, &stages, &smem)) return false;
    SmallParams p{};
    p.x = x;
    p.ld_x = ld_x;
    p.s_tok = l.s_tok;
    p.T = l.T;
    p.K = l.K;
    p.N = l.N;
    p.kblocks = (l.K + kBK - 1) / kBK;
    p.split = split;
    p.stages = stages;
    p.b_nk = l.b_nk;
    p.ahead = l.ahead;
    p.s_ch0 = w0.scale;
    p.s_ch1 = w1 ? w1->scale : w0.scale;
    p.bias = l.bias;
    p.residual = l.residual;
    p.ld_res = l.ld_res;
    p.res_type = l.res_type;
    p.out = l.out;
    p.ld_out = l.ld_out;
    p.out_type = l.out_type;
    const int size = x_type < 0 ? 1 : elem_bytes(x_type);
    p.vec_x = aligned(x, 16) && (ld_x * size) % 16 == 0;
    // (us, exchanged / read by each: 1 x 7168 x 2048 7.8 / 7.2, 2 tokens 7.9 / 7.9, 4 tokens 8.1 / 10.0)
    p.exchange = (int64_t)l.T * l.K * size > 32 * 1024;
    // weights are the A operand (M = 128 channels): MN-major for [K, N]
    p.idesc = idesc_i8(128, kSmallN, false) | (p.b_nk ? 0u : 1u << 15);
    CUtensorMap w[2];
    const Matrix* ws[2] = {&w0, w1 ? w1 : &w0};
    for (int i = 0; i < mats; ++i) {
        const bool ok = p.b_nk ? make_map_u8_strided(&w[i], ws[i]->w, p.K, p.N, ws[i]->ld, 128, 128)
                               : make_map_u8_strided(&w[i], ws[i]->w, p.N, p.K, ws[i]->ld, 128, kBK);
        if (!ok) {
            *err = cudaErrorInvalidValue;
            return true;
        }
    }
    if (mats == 1) w[1] = w[0];
    const int tiles = (l.N + 127) / 128;
    if (x_type < 0)
        *err = w1 ? launch_small_typed<kInCodes, true>(w, p, tiles, smem, st)
                  : launch_small_typed<kInCodes, false>(w, p, tiles, smem, st);
    else if (x_type == MOE_TYPE_F32)
        *err = w1 ? launch_small_typed<kInF32, true>(w, p, tiles, smem, st)
                  : launch_small_typed<kInF32, false>(w, p, tiles, smem, st);
    else if (x_type == MOE_TYPE_F16)
        *err = w1 ? launch_small_typed<kInF16, true>(w, p, tiles, smem, st)
                  : launch_small_typed<kInF16, false>(w, p, tiles, smem, st);
    else
        *err = w1 ? launch_small_typed<kInBF16, true>(w, p, tiles, smem, st)
                  : launch_small_typed<kInBF16, false>(w, p, tiles, smem, st);
    return true;
}

int bad(const char* who, const char* what) {
    set_error("%s: %s", who, what);
    return MOE_ERR_INVALID_ARG;
}

// Shape checks that every entry point here shares.
int check_dims(const char* who, int64_t T, int64_t K, int64_t N) {
    if (T < 0 || K < 1 || N < 1) return bad(who, "tokens must be >= 0, dimensions >= 1");
    if (K > kMaxK) {
        set_error("%s: K = %lld, s32 sums are exact up to %d", who, (long long)K, kMaxK);
        return MOE_ERR_UNSUPPORTED;
    }
    if (T > 0x7FFFFF00ll || N > (1ll << 28) || ((T + 127) / 128) * ((N + 127) / 128) * 2 > 0x7FFFFFFFll) {
        set_error("%s: %lld x %lld outputs are too many for one call", who, (long long)T, (long long)N);
        return MOE_ERR_UNSUPPORTED;
    }
    return MOE_OK;
}

int check_matrix(const char* who, const MoeInt8Weight* w, int64_t K, int64_t N) {
    if (!w || !w->w || !w->scale) return bad(who, "a weight matrix or its scales are null");
    if (w->order != MOE_WEIGHT_KN && w->order != MOE_WEIGHT_NK) return bad(who, "weight order unknown");
    if (!aligned(w->w, 16) || w->row_stride % 16 != 0 || w->row_stride < (w->order == MOE_WEIGHT_KN ? N : K))
        return bad(who, "weight rows must start on 16-byte boundaries and hold a whole row (row_stride % 16 == 0)");
    if (!aligned(w->scale, 4)) return bad(who, "weight scales are not aligned to f32");
    return MOE_OK;
}

int check_x(const char* who, const void* x, int type, int64_t T, int64_t K, int64_t ldx) {
    if (!is_type(type)) return bad(who, "activation type unknown");
    if (ldx < K) return bad(who, "activation row stride is smaller than a row");
    if (T > 0 && (!x || !aligned(x, elem_bytes(type)))) return bad(who, "activations are null or not aligned to their type");
    return MOE_OK;
}

int check_out(const char* who, const void* out, int type, int64_t T, int64_t N, int64_t ldo) {
    if (!is_type(type)) return bad(who, "output type unknown");
    if (ldo < N) return bad(who, "output row stride is smaller than a row");
    if (T > 0 && (!out || !aligned(out, elem_bytes(type)))) return bad(who, "output is null or not aligned to its type");
    return MOE_OK;
}

int check_scratch(const char* who, const void* scratch, size_t have, size_t need) {
    if (need == 0) return MOE_OK;
    if (!scratch || !aligned(scratch, 256)) return bad(who, "scratch is null or not 256-byte aligned");
    if (have < need) {
        set_error("%s: scratch of %zu bytes is smaller than the %zu this call needs", who, have, need);
        return MOE_ERR_INVALID_ARG;
    }
    return MOE_OK;
}

// An output in the memory of what other blocks still read: a matrix, its scales, the bias or the scratch.
int check_apart(const char* who, const Span& out, const MoeInt8Weight& w, int64_t K, int64_t N, const float* bias,
                const void* scratch, size_t scratch_bytes) {
    const Span m{w.w, w.row_stride, w.order == MOE_WEIGHT_KN ? N : K, w.order == MOE_WEIGHT_KN ? K : N};
    if (overlap(out, m) || overlap(out, vector_span(w.scale, N * 4)) || overlap(out, vector_span(bias, N * 4)))
        return bad(who, "the output shares memory with a weight matrix, its scales or the bias");
    if (overlap(out, vector_span(scratch, (int64_t)scratch_bytes))) return bad(who, "the output shares memory with the scratch");
    return MOE_OK;
}

int cuda_error(const char* who, cudaError_t e) {
    set_error("%s: %s", who, cudaGetErrorString(e));
    return MOE_ERR_CUDA;
}

LinearParams out_params(int64_t T, int K, int N, const float* s_tok, const float* bias, void* out, int out_type,
                        int64_t ldo, int order) {
    LinearParams p{};
    p.T = (int)T;
    p.K = K;
    p.N = N;
    p.b_nk = order == MOE_WEIGHT_NK;
    p.s_tok = s_tok;
    p.bias = bias;
    p.out = out;
    p.out_type = out_type;
    p.ld_out = ldo;
    p.vec_out = aligned(out, 16) && (ldo * elem_bytes(out_type)) % 16 == 0;
    return p;
}

// Whether the gate and up products run as one fused launch (h written), or as
// two plain products whose SwiGLU the quantiser of h applies: fused tiles are
// 128 tokens x 128 features, and too few of them leave SMs idle that the plain
// product's split of K fills.
bool fused_swiglu(int64_t T, int64_t f) { return (T + 127) / 128 * ((f + 127) / 128) * 4 >= kRuleSms * 3; }

// Whether the small kernel takes a call.
bool is_small(int64_t T, int limit, int K, int N, int mats = 1) {
    int split, stages;
    size_t smem;
    return plan_small(T, limit, K, N, mats, &split, &stages, &smem);
}

size_t linear_scratch(int64_t T, int K, int N) {
    return is_small(T, kSmallLinear, K, N) ? 0 : up256((size_t)T * up16(K)) + up256((size_t)T * sizeof(float));
}

struct SharedScratch {
    size_t qx, sx, h, qh, sh, total;
    int64_t ldh;
};
SharedScratch shared_scratch(int64_t T, int64_t d, int64_t f) {
    SharedScratch s;
    s.ldh = (f + 3) / 4 * 4;
    size_t at = 0;
    s.qx = at; at += up256((size_t)T * up16(d));
    s.sx = at; at += up256((size_t)T * sizeof(float));
    const bool one = fused_swiglu(T, f) || is_small(T, kSmallPairs, (int)d, (int)f, 2);
    s.h = at;  at += up256((size_t)T * s.ldh * sizeof(float)) * (one ? 1 : 2);
    s.qh = at; at += up256((size_t)T * up16(f));
    s.sh = at; at += up256((size_t)T * sizeof(float));
    s.total = at;
    return s;
}

}  // namespace

// Devices on which a product has run (only there is the status word read).
std::atomic<bool> g_linear_used[64];

int linear_status_collect(int dev) {
    if (dev < 0 || dev >= 64 || !g_linear_used[dev].load()) return MOE_OK;
    int host = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&host, g_linear_status, sizeof(int));
    if (e != cudaSuccess) return cuda_error("moe_check_device_status", e);
    if (host == 0) return MOE_OK;
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_linear_status, &zero, sizeof(int));
    if (e != cudaSuccess) return cuda_error("moe_check_device_status", e);
    set_error("device-side wait timed out (int8 product, status %d)", host);
    return MOE_ERR_TIMEOUT;
}

int run_shared_expert(const char* who, const void* x, int x_type, int64_t tokens, int d_model, int64_t row_stride,
                      const MoeInt8Weight* gate, const MoeInt8Weight* up, const MoeInt8Weight* down, int d_ff,
                      const void* residual, int64_t residual_stride, void* out, int out_type, int64_t out_stride,
                      void* scratch, size_t scratch_bytes, bool check_only, cudaStream_t stream) {
    int rc = check_dims(who, tokens, d_model, d_ff);
    if (rc == MOE_OK) rc = check_dims(who, tokens, d_ff, d_model);
    if (rc == MOE_OK) rc = check_x(who, x, x_type, tokens, d_model, row_stride);
    if (rc == MOE_OK) rc = check_matrix(who, gate, d_model, d_ff);
    if (rc == MOE_OK) rc = check_matrix(who, up, d_model, d_ff);
    if (rc == MOE_OK) rc = check_matrix(who, down, d_ff, d_model);
    if (rc == MOE_OK) rc = check_out(who, out, out_type, tokens, d_model, out_stride);
    if (rc != MOE_OK) return rc;
    if (gate->order != up->order) return bad(who, "gate and up weights must have the same order");
    if (residual && (residual_stride < d_model || !aligned(residual, elem_bytes(x_type))))
        return bad(who, "residual rows are shorter than d_model or not aligned to their type");
    if (tokens == 0) return MOE_OK;
    const SharedScratch sc = shared_scratch(tokens, d_model, d_ff);
    rc = check_scratch(who, scratch, scratch_bytes, sc.total);
    if (rc != MOE_OK) return rc;
    const int in = elem_bytes(x_type), size = elem_bytes(out_type);
    const bool same = residual == out && x_type == out_type && (tokens == 1 || residual_stride == out_stride);
    const Span rows{out, out_stride * size, (int64_t)d_model * size, tokens},
        act{x, row_stride * in, (int64_t)d_model * in, tokens}, res{residual, residual_stride * in, (int64_t)d_model * in, tokens},
        temp = vector_span(scratch, (int64_t)sc.total);
    if (!same && overlap(res, rows)) return bad(who, "the output shares memory with the residual without being it");
    if (overlap(act, temp) || overlap(res, temp)) return bad(who, "the scratch shares memory with the activations or the residual");
    rc = check_apart(who, rows, *gate, d_model, d_ff, nullptr, scratch, sc.total);
    if (rc == MOE_OK) rc = check_apart(who, rows, *up, d_model, d_ff, nullptr, nullptr, 0);
    if (rc == MOE_OK) rc = check_apart(who, rows, *down, d_ff, d_model, nullptr, nullptr, 0);
    if (rc != MOE_OK) return rc;
    if (check_only) return MOE_OK;
    int dev = 0, num_sms = 0;
    rc = current_device(&dev, &num_sms);
    if (rc != MOE_OK) return rc;
    g_linear_used[dev] = true;
    uint8_t* base = static_cast<uint8_t*>(scratch);
    int8_t *qx = reinterpret_cast<int8_t*>(base + sc.qx), *qh = reinterpret_cast<int8_t*>(base + sc.qh);
    float *sx = reinterpret_cast<float*>(base + sc.sx), *sh = reinterpret_cast<float*>(base + sc.sh);
    float* h = reinterpret_cast<float*>(base + sc.h);
    const bool fused = fused_swiglu(tokens, d_ff);
    const int64_t behind = (int64_t)(up256((size_t)tokens * sc.ldh * sizeof(float)) / sizeof(float));
    const Matrix mg{gate->w, gate->row_stride, gate->scale}, mu{up->w, up->row_stride, up->scale},
        md{down->w, down->row_stride, down->scale};
    LinearParams ph = out_params(tokens, d_model, d_ff, sx, nullptr, h, MOE_TYPE_F32, sc.ldh, gate->order);
    ph.out1 = behind;
    LinearParams py = out_params(tokens, d_ff, d_model, sh, nullptr, out, out_type, out_stride, down->order);
    py.ahead = 1;
    py.residual = residual;
    py.ld_res = residual_stride;
    py.res_type = x_type;
    py.vec_res = aligned(residual, 16) && (residual_stride * elem_bytes(x_type)) % 16 == 0;
    cudaError_t e = cudaSuccess;
    // gate and up: h, or (too few tiles to fuse) g and u
    const bool small = is_small(tokens, kSmallPairs, d_model, d_ff, 2);
    if (!try_small(kSmallLinear, x, x_type, row_stride, ph, mg, &mu, stream, &e)) {
        ph.ahead = 1;
        e = launch_quantize(x, x_type, tokens, d_model, row_stride, 0, qx, up16(d_model), sx, num_sms, stream);
        if (e == cudaSuccess && !try_small(kSmallPairs, qx, -1, up16(d_model), ph, mg, &mu, stream, &e))
            e = launch_linear(qx, up16(d_model), ph, mg, &mu, fused, num_sms, stream);
    }
    if (e != cudaSuccess) return cuda_error(who, e);
    const bool pairs = !fused && !small;
    if (pairs || !try_small(kSmallLinear, h, MOE_TYPE_F32, sc.ldh, py, md, nullptr, stream, &e)) {
        e = launch_quantize(h, MOE_TYPE_F32, tokens, d_ff, sc.ldh, pairs ? behind : 0, qh, up16(d_ff), sh, num_sms, stream);
        if (e == cudaSuccess && !try_small(kSmallCodes, qh, -1, up16(d_ff), py, md, nullptr, stream, &e))
            e = launch_linear(qh, up16(d_ff), py, md, nullptr, false, num_sms, stream);
    }
    return e == cudaSuccess ? MOE_OK : cuda_error(who, e);
}

}  // namespace moe

using namespace moe;

extern "C" int moe_selftest_int8_wait_timeout(int64_t timeout_ns, int* written, cudaStream_t stream) {
    const char* who = "moe_selftest_int8_wait_timeout";
    if (timeout_ns <= 0 || timeout_ns > 10000000000ll) return bad(who, "timeout_ns must be in (0, 10 s]");
    if (!written || !aligned(written, 4)) return bad(who, "written is null or not aligned to int");
    int dev = 0, num_sms = 0;
    const int rc = current_device(&dev, &num_sms);
    if (rc != MOE_OK) return rc;
    g_linear_used[dev] = true;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2);
    cfg.blockDim = dim3(32);
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {2, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, waits_selftest_kernel, (uint64_t)timeout_ns, written);
    return e == cudaSuccess ? MOE_OK : cuda_error(who, e);
}

extern "C" size_t moe_int8_linear_scratch_bytes(int64_t tokens, int K, int N) {
    return tokens < 0 || K < 1 || N < 1 ? 0 : linear_scratch(tokens, K, N);
}

extern "C" size_t moe_int8_shared_expert_scratch_bytes(int64_t tokens, int d_model, int d_ff) {
    return tokens < 0 || d_model < 1 || d_ff < 1 ? 0 : shared_scratch(tokens, d_model, d_ff).total;
}

extern "C" int moe_int8_quantize_tokens(const void* x, int x_type, int64_t tokens, int K, int64_t row_stride, int8_t* q,
                                        int64_t q_stride, float* scale, cudaStream_t stream) {
    const char* who = "moe_int8_quantize_tokens";
    int rc = check_dims(who, tokens, K, 1);
    if (rc == MOE_OK) rc = check_x(who, x, x_type, tokens, K, row_stride);
    if (rc != MOE_OK) return rc;
    if (tokens == 0) return MOE_OK;
    if (!q || !scale || !aligned(q, 16) || q_stride % 16 != 0 || q_stride < K || !aligned(scale, 4))
        return bad(who, "codes must be rows on 16-byte boundaries (q_stride % 16 == 0, >= K) and scales f32");
    const int in = elem_bytes(x_type);
    const Span rows{x, row_stride * in, (int64_t)K * in, tokens}, codes{q, q_stride, K, tokens},
        scales = vector_span(scale, tokens * 4);
    if (overlap(rows, codes) || overlap(rows, scales) || overlap(codes, scales))
        return bad(who, "an output shares memory with the activations or the other output");
    int dev = 0, num_sms = 0;
    rc = current_device(&dev, &num_sms);
    if (rc != MOE_OK) return rc;
    const cudaError_t e = launch_quantize(x, x_type, tokens, K, row_stride, 0, q, q_stride, scale, num_sms, stream);
    return e == cudaSuccess ? MOE_OK : cuda_error(who, e);
}

extern "C" int moe_int8_matmul(const int8_t* q, int64_t q_stride, const float* scale, int64_t tokens, int K,
                               const MoeInt8Weight* w, int N, const float* bias, void* out, int out_type,
                               int64_t out_stride, cudaStream_t stream) {
    const char* who = "moe_int8_matmul";
    int rc = check_dims(who, tokens, K, N);
    if (rc == MOE_OK) rc = check_matrix(who, w, K, N);
    if (rc == MOE_OK) rc = check_out(who, out, out_type, tokens, N, out_stride);
    if (rc != MOE_OK) return rc;
    if (tokens == 0) return MOE_OK;
    if (!q || !scale || !aligned(q, 16) || q_stride % 16 != 0 || q_stride < K || !aligned(scale, 4))
        return bad(who, "codes must be rows on 16-byte boundaries (q_stride % 16 == 0, >= K) and scales f32");
    if (!aligned(bias, 4)) return bad(who, "bias is not aligned to f32");
    const int size = elem_bytes(out_type);
    const Span rows{out, out_stride * size, (int64_t)N * size, tokens};
    if (overlap({q, q_stride, K, tokens}, rows) || overlap(vector_span(scale, tokens * 4), rows))
        return bad(who, "the output shares memory with the codes or their scales");
    rc = check_apart(who, rows, *w, K, N, bias, nullptr, 0);
    if (rc != MOE_OK) return rc;
    int dev = 0, num_sms = 0;
    rc = current_device(&dev, &num_sms);
    if (rc != MOE_OK) return rc;
    g_linear_used[dev] = true;
    const LinearParams p = out_params(tokens, K, N, scale, bias, out, out_type, out_stride, w->order);
    const Matrix m{w->w, w->row_stride, w->scale};
    cudaError_t e;
    if (!try_small(kSmallCodes, q, -1, q_stride, p, m, nullptr, stream, &e))
        e = launch_linear(q, q_stride, p, m, nullptr, false, num_sms, stream);
    return e == cudaSuccess ? MOE_OK : cuda_error(who, e);
}

extern "C" int moe_int8_linear(const void* x, int x_type, int64_t tokens, int K, int64_t row_stride,
                               const MoeInt8Weight* w, int N, const float* bias, void* out, int out_type,
                               int64_t out_stride, void* scratch, size_t scratch_bytes, cudaStream_t stream) {
    const char* who = "moe_int8_linear";
    int rc = check_dims(who, tokens, K, N);
    if (rc == MOE_OK) rc = check_x(who, x, x_type, tokens, K, row_stride);
    if (rc == MOE_OK) rc = check_matrix(who, w, K, N);
    if (rc == MOE_OK) rc = check_out(who, out, out_type, tokens, N, out_stride);
    if (rc != MOE_OK) return rc;
    if (!aligned(bias, 4)) return bad(who, "bias is not aligned to f32");
    if (tokens == 0) return MOE_OK;
    const size_t need = linear_scratch(tokens, K, N);
    rc = check_scratch(who, scratch, scratch_bytes, need);
    if (rc != MOE_OK) return rc;
    const int in = elem_bytes(x_type), size = elem_bytes(out_type);
    const Span rows{out, out_stride * size, (int64_t)N * size, tokens}, act{x, row_stride * in, (int64_t)K * in, tokens};
    if (overlap(act, rows)) return bad(who, "the output shares memory with the activations");
    if (overlap(act, vector_span(scratch, (int64_t)need))) return bad(who, "the scratch shares memory with the activations");
    rc = check_apart(who, rows, *w, K, N, bias, scratch, need);
    if (rc != MOE_OK) return rc;
    int dev = 0, num_sms = 0;
    rc = current_device(&dev, &num_sms);
    if (rc != MOE_OK) return rc;
    g_linear_used[dev] = true;
    int8_t* q = static_cast<int8_t*>(scratch);   // (null where the small kernel needs none)
    float* s = q ? reinterpret_cast<float*>(q + up256((size_t)tokens * up16(K))) : nullptr;
    LinearParams p = out_params(tokens, K, N, s, bias, out, out_type, out_stride, w->order);
    const Matrix m{w->w, w->row_stride, w->scale};
    cudaError_t e;
    if (!try_small(kSmallLinear, x, x_type, row_stride, p, m, nullptr, stream, &e)) {
        p.ahead = 1;
        e = launch_quantize(x, x_type, tokens, K, row_stride, 0, q, up16(K), s, num_sms, stream);
        if (e == cudaSuccess && !try_small(kSmallCodes, q, -1, up16(K), p, m, nullptr, stream, &e))
            e = launch_linear(q, up16(K), p, m, nullptr, false, num_sms, stream);
    }
    return e == cudaSuccess ? MOE_OK : cuda_error(who, e);
}

extern "C" int moe_int8_shared_expert(const void* x, int x_type, int64_t tokens, int d_model, int64_t row_stride,
                                      const MoeInt8Weight* gate, const MoeInt8Weight* up, const MoeInt8Weight* down,
                                      int d_ff, const void* residual, int64_t residual_stride, void* out, int out_type,
                                      int64_t out_stride, void* scratch, size_t scratch_bytes, cudaStream_t stream) {
    return run_shared_expert("moe_int8_shared_expert", x, x_type, tokens, d_model, row_stride, gate, up, down, d_ff,
                             residual, residual_stride, out, out_type, out_stride, scratch, scratch_bytes, false, stream);
}
