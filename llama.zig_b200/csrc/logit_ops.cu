// logit_ops.cu -- operators on rows of logits beside the sampler: the
// log-probabilities of given tokens (with their gradient), the top logits of
// a row, and two training losses with their gradients.  CUDA kernels for
// sm_100a and their C ABI (include/b200_sampler.h).
//
// A row of V logits v is seen through the sampler's prologue and temperature,
//     z_j = c(v_j) m,  c(v) = cap tanh(v / cap) or v,  m = 1 / (logit_scale T),
//     p_j = exp(z_j) / sum_i exp(z_i),
// computed relative to the row's maximum M of c(v) and in base 2:
//     d_j = (c(v_j) - M) m log2e <= 0,  S = sum_j 2^d_j,
//     U = sum_j 2^d_j d_j,  log2 p_j = d_j - log2 S,  H = ln2 (log2 S - U / S).
// The difference is taken before the product, so rows at the edge of the
// float range (masks of the type's lowest value) do not overflow.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstdio>

#include "b200_sampler.h"

namespace bs {
namespace ops {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_CLUSTER = 16;      // CTAs of a row (8 is the portable limit; 16 where a row needs it)
constexpr float LN2 = 0.6931471805599453f;
constexpr double LN2_D = 0.6931471805599453;
// 2^d is zero in f32 below this; products with d stop here, so that a logit
// of -inf adds 0 to the entropy and not 0 * inf.
constexpr float D_MIN = -200.0f;

enum Op { OP_LOGPROB, OP_POLICY, OP_POLICY_ENT, OP_DISTILL, OP_DISTILL_TAIL };

struct Scale {
    float k;         // m log2(e)
    float m;         // 1 / (logit_scale T)
    float cap, icap; // soft-cap and its reciprocal
    float k2, k2_lo; // -2 log2(e) / cap, and what f32 leaves off it
    float most;      // c(v) is +-cap from here on
    double md;       // m in 64 bits
    double inv_t;    // 1 / T
    double dk;       // what rounding left off k, relative
};

struct RowArgs {
    const void *x;
    size_t ld;
    uint32_t vocab;
    uint32_t keep;              // 16-byte chunks of a CTA's slice that stay in shared memory
    uint32_t log_ranks;         // CTAs of a row
    uint32_t bit_words;         // with a teacher: words of one bit per element of a slice
    Scale sc;
    const int32_t *tokens;
    uint32_t zero;              // 0, which the compiler does not know
    long long wait_limit;       // clock cycles
    uint32_t gone_rank, gone_row;   // (for tests) the CTA of a row whose waits give up, from a cluster's i-th row on
    // outputs (null where not asked for)
    float *logprobs, *entropy, *kl, *row_loss;
    float2 *stats;
    void *grad;
    size_t ld_grad;
    // losses
    const float *weights;       // null: 1 / rows each
    float w_all;
    const float *old_lp, *adv, *ref_lp;
    double clip_lo, clip_hi;
    float kl_coef, ent_coef;
    const int32_t *t_ids;       // rows x n_ids
    const float *t_logits, *t_lse;
    uint32_t n_ids;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// Two f32 in one 64-bit register: Blackwell's FMA pipe does both halves in
// one issue slot, and issue slots are what the 16-bit types run short of.
typedef float2 f2;
__device__ __forceinline__ f2 pair(float a, float b) { return make_float2(a, b); }
__device__ __forceinline__ f2 both(float a) { return make_float2(a, a); }
__device__ __forceinline__ void halves(f2 v, float &a, float &b) { a = v.x; b = v.y; }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ f2 ex2_2(f2 v) {
    float a, b;
    halves(v, a, b);
    return pair(ex2(a), ex2(b));
}
__device__ __forceinline__ f2 floor2(f2 v) {   // at least D_MIN; a NaN stays
    float a, b;
    halves(v, a, b);
    return pair(max_nan(a, D_MIN), max_nan(b, D_MIN));
}

// The soft-cap c(v) = cap tanh(v / cap).  Up to |v| = cap, where nearly all
// logits are, c = v + v y W(y) with y = (v / cap)^2 and W a polynomial: the least
// largest relative error of c over y in [0, 1] with f32 coefficients, 4.7e-9.
// The last fused step rounds once, what comes before it is at most 0.31 of c: at
// most 3.3 half steps in all, 0.45 root mean square on the workloads' logits, where
// cap * tanhf(v / cap) has 1.3.  Ten FMA-pipe slots for two logits.  Beyond, c = cap - cap 2 e / (1 + e) with
// e = exp(-2 |v| / cap), the exponent rounded once: at most 3.9 half steps.
__constant__ const float TANH_W[7] = {-0.33333295583724976f, 0.13332347571849823f, -0.0538799911737442f, 0.021487198770046234f,
                                      -0.007946893572807312f, 0.0023019297514110804f, -0.00035861122887581587f};
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ f2 cap_near(f2 v, const Scale &sc) {
    const f2 x = mul2(v, both(sc.icap)), y = mul2(x, x);
    f2 w = both(TANH_W[6]);
#pragma unroll
    for (int i = 5; i >= 0; i--) w = fma2(w, y, both(TANH_W[i]));
    return fma2(mul2(v, y), w, v);
}
__device__ __forceinline__ float cap_far(float v, const Scale &sc, float *slope = nullptr) {
    const float a = fminf(fabsf(v), sc.most);
    const float e = isinf(v) ? 0.0f : ex2(fmaf(a, sc.k2, a * sc.k2_lo));
    const float r = rcp(1.0f + e), q = 2.0f * e * r;
    if (slope) *slope = 2.0f * q * r;
    return copysignf(fmaf(-sc.cap, q, sc.cap), v);
}
template <bool CAP> __device__ __forceinline__ float capped(float v, const Scale &sc) {
    if (!CAP) return v;
    if (fabsf(v) > sc.cap) return cap_far(v, sc);
    return cap_near(both(v), sc).x;
}

// The soft-cap's slope: 1 - (c / cap)^2 up to |v| = cap, where at least 0.42 is
// left of it; beyond, where less and less would be, 4 e / (1 + e)^2.
__device__ __forceinline__ f2 slope2(f2 c, const Scale &sc) {
    const f2 t = mul2(c, both(sc.icap));
    return fma2(mul2(t, both(-1.0f)), t, both(1.0f));
}
// The slope at one logit, and c(v) with it.
__device__ __forceinline__ float cap_slope(float c, float v, const Scale &sc) {
    float slope = slope2(both(c), sc).x;
    if (fabsf(v) > sc.cap) cap_far(v, sc, &slope);
    return slope;
}
template <bool CAP> __device__ __forceinline__ float2 cap_both(float v, const Scale &sc) {
    if (!CAP) return make_float2(v, 1.0f);
    float2 r = make_float2(cap_near(both(v), sc).x, 0.0f);
    r.y = slope2(both(r.x), sc).x;
    if (fabsf(v) > sc.cap) r.x = cap_far(v, sc, &r.y);
    return r;
}

// Two at once, the same operations.
template <bool SLOPE> __device__ __forceinline__ f2 cap_far2(f2 v, const Scale &sc, f2 &slope) {
    const f2 a = pair(fminf(fabsf(v.x), sc.most), fminf(fabsf(v.y), sc.most));
    const f2 e = ex2_2(fma2(a, both(sc.k2), mul2(a, both(sc.k2_lo))));
    const f2 n = add2(e, both(1.0f)), r = pair(rcp(n.x), rcp(n.y)), q = mul2(add2(e, e), r);
    if (SLOPE) slope = mul2(add2(q, q), r);
    const f2 c = fma2(both(-sc.cap), q, both(sc.cap));
    return pair(copysignf(c.x, v.x), copysignf(c.y, v.y));
}

// A streaming read: not kept in L1.
__device__ __forceinline__ uint4 ld_stream(const void *p) {
    uint4 q;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "l"(p) : "memory");
    return q;
}
__device__ __forceinline__ f2 widen(uint32_t w, __nv_bfloat16) {
    return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ f2 widen(uint32_t w, __half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    return pair(f.x, f.y);
}
__device__ __forceinline__ uint32_t narrow(f2 v, __nv_bfloat16) {
    float a, b;
    halves(v, a, b);
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t narrow(f2 v, __half) {
    float a, b;
    halves(v, a, b);
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b, __nv_bfloat16) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b, __half) {
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// A 16-byte chunk of E logits as pairs, and back.
template <typename T> __device__ __forceinline__ void unpack(const uint4 &q, f2 (&v)[8 / sizeof(T)]) {
    if constexpr (sizeof(T) == 4) {
        v[0] = pair(__uint_as_float(q.x), __uint_as_float(q.y));
        v[1] = pair(__uint_as_float(q.z), __uint_as_float(q.w));
    } else {
        v[0] = widen(q.x, T());
        v[1] = widen(q.y, T());
        v[2] = widen(q.z, T());
        v[3] = widen(q.w, T());
    }
}
template <typename T> __device__ __forceinline__ uint4 pack(const f2 (&v)[8 / sizeof(T)]) {
    if constexpr (sizeof(T) == 4) {
        float a, b, c, d;
        halves(v[0], a, b);
        halves(v[1], c, d);
        return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d));
    } else {
        return make_uint4(narrow(v[0], T()), narrow(v[1], T()), narrow(v[2], T()), narrow(v[3], T()));
    }
}
// The largest logit of a chunk (a NaN is passed over).
template <typename T> __device__ __forceinline__ float max_of(const uint4 &q) {
    if constexpr (sizeof(T) == 4) {
        return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
    } else {
        float a, b;
        halves(widen(max_pair(max_pair(q.x, q.y, T()), max_pair(q.z, q.w, T()), T()), T()), a, b);
        return fmaxf(a, b);
    }
}
template <typename T, int N> __device__ __forceinline__ float max_of(const uint4 (&q)[N]) {
    uint4 m = q[0];
#pragma unroll
    for (int i = 1; i < N; i++) {
        if constexpr (sizeof(T) == 4) {
            m.x = __float_as_uint(fmaxf(__uint_as_float(m.x), __uint_as_float(q[i].x)));
            m.y = __float_as_uint(fmaxf(__uint_as_float(m.y), __uint_as_float(q[i].y)));
            m.z = __float_as_uint(fmaxf(__uint_as_float(m.z), __uint_as_float(q[i].z)));
            m.w = __float_as_uint(fmaxf(__uint_as_float(m.w), __uint_as_float(q[i].w)));
        } else {
            m.x = max_pair(m.x, q[i].x, T());
            m.y = max_pair(m.y, q[i].y, T());
            m.z = max_pair(m.z, q[i].z, T());
            m.w = max_pair(m.w, q[i].w, T());
        }
    }
    return max_of<T>(m);
}
// The largest |logit| of a chunk (a NaN is passed over).
template <typename T> __device__ __forceinline__ float max_abs(uint4 q) {
    if constexpr (sizeof(T) == 4) {
        return fmaxf(fmaxf(fabsf(__uint_as_float(q.x)), fabsf(__uint_as_float(q.y))),
                     fmaxf(fabsf(__uint_as_float(q.z)), fabsf(__uint_as_float(q.w))));
    } else {
        const uint32_t m = 0x7FFF7FFFu;
        return max_of<T>(make_uint4(q.x & m, q.y & m, q.z & m, q.w & m));
    }
}
// Who wants to know of a logit above the soft-cap: `stamp` goes to *at.
struct Note {
    uint32_t *at;
    uint32_t stamp;
    __device__ __forceinline__ void put() const {
        if (at) *at = stamp;
    }
};
// A chunk's logits after the soft-cap, and (SLOPE) its slopes there.  LEFT: q
// holds c(v) where |v| <= cap and v beyond (|c| is below 0.77 cap on the one side).
template <typename T, bool CAP, bool SLOPE = false, bool LEFT = false>
__device__ __forceinline__ void cap_chunk(const uint4 &q, f2 (&v)[8 / sizeof(T)], const Scale &sc, const Note &note, f2 *slopes = nullptr) {
    unpack<T>(q, v);
    if (!CAP) return;
    constexpr int N = 8 / sizeof(T);
    const bool far = max_abs<T>(q) > sc.cap;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (!LEFT) v[i] = cap_near(v[i], sc);
        if (SLOPE) slopes[i] = slope2(v[i], sc);
    }
    if (far) {
        note.put();
        f2 raw[N];
        unpack<T>(q, raw);
#pragma unroll
        for (int i = 0; i < N; i++) {
            f2 slope;
            const f2 c = cap_far2<SLOPE>(raw[i], sc, slope);
            const bool x = fabsf(raw[i].x) > sc.cap, y = fabsf(raw[i].y) > sc.cap;
            v[i] = pair(x ? c.x : v[i].x, y ? c.y : v[i].y);
            if (SLOPE) slopes[i] = pair(x ? slope.x : slopes[i].x, y ? slope.y : slopes[i].y);
        }
    }
}
// What a thread writes of a chunk where 16-byte stores do not fit.
template <typename T> __device__ __forceinline__ void store_each(T *g, const uint4 &q) {
    const T *e = reinterpret_cast<const T *>(&q);
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); i++) g[i] = e[i];
}

// Logits of a chunk that count for nothing: -inf in place of those in `marks`.
template <typename T> __device__ __forceinline__ void mask_out(f2 (&v)[8 / sizeof(T)], uint32_t marks) {
#pragma unroll
    for (int i = 0; i < (int)(8 / sizeof(T)); i++) {
        if (marks >> (2 * i) & 1u) v[i].x = -INFINITY;
        if (marks >> (2 * i) & 2u) v[i].y = -INFINITY;
    }
}
template <typename T> __device__ __forceinline__ void mask_out(uint4 &q, uint32_t marks) {
    f2 v[8 / sizeof(T)];
    unpack<T>(q, v);
    mask_out<T>(v, marks);
    q = pack<T>(v);
}

// A row as its body, the 16-byte aligned chunks that lie wholly inside it,
// and at most E - 1 single elements before and behind the body.
template <typename T> struct Row {
    static constexpr int E = 16 / sizeof(T);
    const T *x;              // element 0
    uint32_t vocab;
    uint32_t lead;           // elements before the body
    uint32_t chunks;         // of the body
    uint32_t trail;          // elements behind it
    __device__ Row(const void *base, size_t ld, uint32_t row, uint32_t v) : x((const T *)base + (size_t)row * ld), vocab(v) {
        uint32_t head = (uint32_t)(((uintptr_t)x & 15u) / sizeof(T));
        lead = head ? min(E - head, v) : 0u;
        chunks = (v - lead) / E;
        trail = v - lead - chunks * E;
    }
    // the single element of thread tid (tid < 32): leading ones in lanes
    // 0.., trailing ones in lanes 8..; -1 where there is none
    __device__ int32_t edge(uint32_t tid) const {
        if (tid < lead) return (int32_t)tid;
        if (tid >= 8 && tid - 8 < trail) return (int32_t)(vocab - trail + tid - 8);
        return -1;
    }
    __device__ const T *at(uint32_t chunk) const { return x + lead + (size_t)chunk * E; }
};

// Running (M, S, U) of a set of logits.
// S is kept in 64 bits from a warp's lanes on: the dozen additions that
// fold a row would each round off half a step of 1 beside its largest logit.
struct __align__(16) Stat {
    double s;
    float m, u;
};
// A maximum of -inf (all of the set masked) is replaced by 0 in differences,
// so that the masked logits give 2^-inf = 0.
__device__ __forceinline__ float anchor(float m) { return m == -INFINITY ? 0.0f : m; }

// What a thread gathers of the logits it reads, on the scale of its running
// maximum m: s = sum 2^d and (ENT) u = sum 2^d d in pairs (even and odd logits).
// Terms are added up by chunks and steps of chunks (`part`) before they meet s:
// once the row's largest logit is in s, every addition to it rounds off half a
// step of 1, however small the term.
template <typename T, bool CAP, bool ENT> struct Gather {
    static constexpr int E = 16 / sizeof(T);
    float m = -INFINITY;
    f2 s = {0.0f, 0.0f}, u = {0.0f, 0.0f}, part = {0.0f, 0.0f};
    __device__ __forceinline__ void step() {
        s = add2(s, part);
        part = both(0.0f);
    }
    __device__ __forceinline__ void raise(float to, float k) {
        if (to > m) {   // (fmaxf: from -inf there is nothing to rescale)
            const float d = fmaxf((m - to) * k, D_MIN), f = ex2(d);
            if (ENT) u = mul2(both(f), fma2(both(d), s, u));
            s = mul2(s, both(f));
            m = to;
        }
    }
    // logits after the soft-cap, none above m (but for the soft-cap's rounding)
    __device__ __forceinline__ void chunk(const f2 (&v)[E / 2], float k) {
        const f2 base = both(-anchor(m)), kk = both(k);
        f2 sum;
#pragma unroll
        for (int i = 0; i < E / 2; i++) {
            const f2 d = mul2(add2(v[i], base), kk);
            const f2 e = ex2_2(d);
            sum = i ? add2(sum, e) : e;
            if (ENT) u = fma2(e, floor2(d), u);
        }
        part = add2(part, sum);
    }
    // (those in `marks` are left out)
    __device__ __forceinline__ void chunk(const uint4 &q, const Scale &sc, uint32_t marks = 0, Note note = {}) {
        f2 v[E / 2];
        cap_chunk<T, CAP>(q, v, sc, note);
        if (CAP && marks) mask_out<T>(v, marks);
        chunk(v, sc.k);
    }
    __device__ __forceinline__ void one(float c, float k) {   // a single logit
        raise(c, k);
        const float d = (c - anchor(m)) * k, e = ex2(d);
        s = add2(s, pair(e, 0.0f));
        if (ENT) u = fma2(pair(e, 0.0f), both(max_nan(d, D_MIN)), u);
    }
    __device__ __forceinline__ Stat stat() const {
        float a, b, c, d;
        halves(s, a, b);
        halves(u, c, d);
        return Stat{(double)a + (double)b, m, c + d};
    }
};

// The CTAs of a row form a cluster.
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The address, in CTA `rank` of the cluster, of a shared variable of this one.
__device__ __forceinline__ uint32_t remote(const void *p, uint32_t rank) {
    uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
// A Stat into a shared variable of another CTA.
__device__ __forceinline__ void st_remote(uint32_t addr, const Stat &a) {
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(__double2loint(a.s)),
                 "r"(__double2hiint(a.s)), "r"(__float_as_uint(a.m)), "r"(__float_as_uint(a.u))
                 : "memory");
}

// The gradient of one row: c'(v_j) p_j (ca + cb log2 p_j), log2 p_j = d_j - log2 S.
template <bool ENT> struct GradRow {
    float m, k, l2s, ca, cb;
    __device__ __forceinline__ float one(float c) const {
        const float l = fmaf(c - m, k, -l2s), p = ex2(l);
        return ENT ? p * fmaf(cb, max_nan(l, D_MIN), ca) : p * ca;
    }
    // A chunk of it (LEFT: as cap_chunk).
    template <typename T, bool CAP, bool LEFT = false> __device__ __forceinline__ uint4 chunk(const uint4 &q, const Scale &sc) const {
        constexpr int N = 8 / sizeof(T);
        f2 v[N], slopes[N];
        cap_chunk<T, CAP, CAP, LEFT>(q, v, sc, Note{}, slopes);
        return from<T, CAP>(v, slopes);
    }
    // The same where no logit lies above the soft-cap; DONE: q holds c(v) already.
    template <typename T, bool CAP, bool DONE = false>
    __device__ __forceinline__ uint4 near(const uint4 &q, const Scale &sc) const {
        constexpr int N = 8 / sizeof(T);
        f2 v[N], slopes[N];
        unpack<T>(q, v);
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (CAP && !DONE) v[i] = cap_near(v[i], sc);
            if (CAP) slopes[i] = slope2(v[i], sc);
        }
        return from<T, CAP>(v, slopes);
    }
    template <typename T, bool CAP>
    __device__ __forceinline__ uint4 from(const f2 (&v)[8 / sizeof(T)], const f2 (&slopes)[8 / sizeof(T)]) const {
        f2 o[8 / sizeof(T)];
#pragma unroll
        for (int i = 0; i < (int)(8 / sizeof(T)); i++) {
            const f2 l = fma2(add2(v[i], both(-m)), both(k), both(-l2s));
            o[i] = mul2(ex2_2(l), ENT ? fma2(both(cb), floor2(l), both(ca)) : both(ca));
            if (CAP) o[i] = mul2(o[i], slopes[i]);
        }
        return pack<T>(o);
    }
};

// ---------------------------------------------------------------------------
// The losses' kernel: statistics, results and gradient of whole rows, each
// logit read from memory once.
//
// Its floor is HBM: V s bytes read and V s written a row, against some 14
// issue slots and two ex2 a logit.  A row must be known whole before its
// gradient starts, so it is kept on chip: a cluster of CTAs (one per SM) takes
// a row, each CTA a slice of up to 1/3 of its shared memory, and the three
// buffers hold the row whose gradient is being written, the row being summed
// and the row being loaded.  So that no SM waits while a row's sums travel
// between its CTAs, the sums of row i travel while the gradient of row i - 1
// is written and row i + 1 is loaded:
//
//   warps S             sum row i as soon as its copy is there,
//   warps A             (two, taking turns) add up the CTA's sums and exchange
//                       them with the row's other CTAs; the row's results and
//                       its gradient's coefficients; the single elements
//                       before and behind the 16-byte chunks,
//   warps G             write the gradient (without one, these sum too),
//   warp C              starts the copy of row i + 3 into row i's buffer,
//   warps B             losses with a teacher (four, one for each set of slots,
//                       with every fourth row): prepare a row's slots (shares
//                       q, the student's logits there) and, after the row's
//                       gradient, write the tokens that its teacher names.
//
// Summing and gradient each need one ex2 a logit, so half of the warps do
// either, and the special-function unit always has work while a row's sums
// travel.  A warp that shares the SM with these issues an instruction in some
// ten cycles, so B's 64-bit work is spread over four rows and meets no barrier
// of its own: with the four warps together on one row 512 x 256000 f32 with 128
// ids took 262 us, so 219; 4000 x 8000 bf16 with 64 ids, where a row is short,
// 71 and 89.  Barriers, in as many copies as rows can be between the two sides:
// X (S -> A: row i summed), Y (A -> G: its coefficients), Z (-> C, B: done
// with; from G, or without a gradient from S and A); and mbarriers: full_bar
// (copy -> S), slots_bar (B -> S), mail_bar (A -> A of the other CTAs).
//
// Measured (policy loss and gradient, of the copy bandwidth for one read and
// one write): 777 x 151936 f32 157 us, 92 %; 2048 x 128256 bf16 214 us, 75 %,
// where the sums are what takes longest (4,700 cycles a slice of 32,000 logits
// beside the gradient's 4,200; the copies take 4,900 a row on the 132 SMs that
// clusters of four find, their own sum with nothing beside it 2,600).  A row's
// scalars and folds in 64 bits, its checked waits and sums by steps are 4 % of
// that: 205 us without.  Steps on the way, 4096 x 128256 bf16: one CTA a row, read twice 523 us; clusters of
// small CTAs that keep the row 543; this pipeline with one set of warps for
// both passes and copies by the threads 488, with bulk copies 441 (the threads'
// copies stalled on the memory system's queue), sums and gradient by different
// warps 390, two exchange warps and more threads 380.  Two CTAs to an SM with
// half the slice each: 504.  A quarter of the ex2 as polynomials on the FMA
// pipe: 399.
constexpr uint32_t COPY = 512;       // chunks of one copy
constexpr int MAX_CWARPS = 24;       // most warps S and G together
constexpr int BTHREADS = 128;        // a warp for each of the four sets of slots
constexpr int AHEAD = 4;             // slots of a lane that are loaded ahead
enum Bar { BAR_X = 1, BAR_Y = 5, BAR_Z = 9 };
__device__ __forceinline__ void bar_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void bar_arrive(int id, int threads) {
    asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void copy_bulk(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     (uint32_t)__cvta_generic_to_shared(dst)),
                 "l"(src), "r"(bytes), "r"((uint32_t)__cvta_generic_to_shared(bar))
                 : "memory");
}

__host__ __device__ constexpr bool is_distill(int op) { return op == OP_DISTILL || op == OP_DISTILL_TAIL; }
__host__ __device__ constexpr bool is_policy(int op) { return op == OP_POLICY || op == OP_POLICY_ENT; }
__host__ __device__ constexpr int row_threads(int op, int compute) { return compute + 96 + (is_distill(op) ? BTHREADS : 0); }

// Row i's results as the gradient needs them.
struct Coef {
    float m, l2s;        // maximum, log2 S
    float ca, cb;        // dv_j = c'(v_j) p_j (ca + cb log2 p_j)
    float ct;            // the token's dv
    uint32_t live;       // 0: the row is left out; 2: lost, a wait gave up
    double lse, q_all, wm;   // teacher's ids: wm c'(v_j) (p_j q_all - q_j), log p_j = (c(v_j) - U) m - lse
};
// What the warps B sum of a row's slots, in 64 bits.
struct Teacher {
    double cross, mass;  // sum of q (log q - (c - U) m), sum of q
    double scale;        // q = scale x what the slots hold
    double top;          // with a tail: sum of exp((c - U) m) over the CTA's own ids, each once
    float u;             // U: the largest c(v) of the slots
    uint32_t live;       // 0: no slot, or no share to give
};
// Threads of S and G, and of S alone where there is a gradient to write.  The
// 16-bit types have twice the logits a byte and want more of both: 4096 x 128256
// bf16 390 us with 512, 380 with 640, 389 with 768; 777 x 151936 f32 152 with
// 512, 155 with 640.  Other shares than half: 394 with 352 of 640.  f32 under a
// soft-cap leaves most of the work to S (see LEAVE): policy loss 777 x 151936
// 197 us with 384 of 512, 208 with 352, 249 with 416.
template <typename T> __host__ __device__ constexpr int compute_threads() { return sizeof(T) == 4 ? 512 : 640; }
template <typename T, bool CAP> __host__ __device__ constexpr int sum_threads_of() {
    return CAP && sizeof(T) == 4 ? 384 : compute_threads<T>() / 2;
}
struct RowsShared {
    Stat part[4][MAX_CWARPS];        // of the warps S; m is NaN where one gave up on its copy
    uint4 mail[4][MAX_CLUSTER];      // and of the row's CTAs; two for each warp A
    Coef coef[4];
    uint32_t far[4];                 // i + 1: row i has a logit above the soft-cap in the slice
    uint32_t gone;                   // a wait of this CTA gave up
    uint32_t passed;                 // rows that C has seen through Z
    uint32_t sent[2][MAX_CLUSTER];   // at the end: exchanges that the CTAs' warps A have sent into,
    uint32_t failed[2];              // and whether this CTA's gave up on its last
    int32_t code[16];                // the row's token (0 for a teacher's row); -1: left out
    Teacher teacher[4];
    uint32_t edge_marks[4];          // the teacher's ids among the row's single elements
    uint64_t mail_bar[4], full_bar[3], slots_bar[4];
};

// The sum of a warp's (or of each group of W lanes') Stats, the same in all its
// lanes: the largest maximum first, then every lane's sums on that scale.
template <bool ENT, int W> __device__ __forceinline__ Stat fold_lanes(Stat a, float k) {
    float m = a.m;
#pragma unroll
    for (int o = W / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    const float d = fmaxf((a.m - m) * k, D_MIN), f = ex2(d);
    if (ENT) a.u = f * fmaf(d, (float)a.s, a.u);
    a.s *= (double)f;
#pragma unroll
    for (int o = W / 2; o; o >>= 1) {
        a.s += __shfl_xor_sync(~0u, a.s, o);
        if (ENT) a.u += __shfl_xor_sync(~0u, a.u, o);
    }
    a.m = m;
    return a;
}

// The exchange between a row's CTAs: 16 bytes into every CTA's mail, which
// count on its mbarrier.
__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t *bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive_local(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void mail_send(const uint4 *slot, const uint64_t *bar, uint32_t rank, const uint4 &v) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %5}, [%4];" ::"r"(
                     remote(slot, rank)),
                 "r"(v.x), "r"(v.y), "r"(v.z), "r"(remote(bar, rank)), "r"(v.w)
                 : "memory");
}
// Takes bytes off what a phase waits for: those that nobody will send.
__device__ __forceinline__ void bar_forgo(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
// Waits for a phase; false if it gave up, after `limit` clock cycles or because
// another wait of the CTA had (`gone`).
__device__ __forceinline__ bool bar_wait(const uint64_t *bar, uint32_t parity, long long limit, const volatile uint32_t *gone) {
    long long start = 0;
    for (uint32_t tries = 0;; tries++) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(smem_addr(bar)), "r"(parity) : "memory");
        if (done) return true;
        const long long now = clock64();
        if (tries == 0) start = now;
        if (now - start > limit || (gone && *gone)) return false;
    }
}
constexpr long long WAIT_LIMIT = 1ll << 32;   // two seconds
// Set by a wait that gave up, until the host asks (bs_logit_ops_status).
__device__ uint32_t wait_gave_up;

// Results and coefficients of a row with a token.  A few values a row, so all
// in 64 bits from the f32 sums: a ratio near 1, a KL near 0 and a loss whose
// terms cancel leave the sums' rounding and not their own.
struct TokenIn {
    float w, adv, old_lp, ref_lp, c_tok;
    float slope;         // the soft-cap's, at the token
};
// The gradient at the token itself, before the soft-cap's slope, from those of
// log-probability and entropy: g (1 - p) - h p (log p + H), with 1 - p as
// -expm1(log p), whose bits a p near 1 in f32 has lost.
__device__ __forceinline__ double token_slope(double lp, double pm1, double H, double g, double h) {
    return -g * pm1 - (h != 0.0 ? h * (1.0 + pm1) * (fmax(lp, -1e4) + H) : 0.0);
}
// e^x to 2^-41: 2^n by the exponent's bits times the exponential series of the
// rest, |r| <= ln 2 / 2, whose eleventh power over 11! is 2^-42.  0 below e^-700
// (-inf too), +inf above e^700; a NaN stays.
__device__ __forceinline__ double exp_d(double x) {
    const double magic = 6755399441055744.0, n = fma(x, 1.0 / LN2_D, magic), r = fma(n - magic, -LN2_D, x);
    double y = 1.0 / 3628800;
    y = fma(y, r, 1.0 / 362880);
    y = fma(y, r, 1.0 / 40320);
    y = fma(y, r, 1.0 / 5040);
    y = fma(y, r, 1.0 / 720);
    y = fma(y, r, 1.0 / 120);
    y = fma(y, r, 1.0 / 24);
    y = fma(y, r, 1.0 / 6);
    y = fma(y, r, 0.5);
    y = fma(y, r, 1.0);
    y = fma(y, r, 1.0);
    y *= __hiloint2double((__double2loint(n) + 1023) << 20, 0);
    return x < -700.0 ? 0.0 : x > 700.0 ? INFINITY : y;
}
// The exchange between a row's sums and its gradient waits for these few
// values, so a warp works them out side by side: lane e has the function at the
// e-th argument, and every lane gets all results.
template <int N> __device__ __forceinline__ void by_lanes(double (&v)[N], double (*f)(double)) {
    double mine = v[0];
#pragma unroll
    for (int e = 1; e < N; e++) mine = (threadIdx.x & 31) == e ? v[e] : mine;
    mine = f(mine);
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = __shfl_sync(~0u, mine, e);
}
template <int OP>
__device__ __forceinline__ Coef token_row(const RowArgs &A, uint32_t row, const Stat &st, const TokenIn &in, bool write) {
    // (u / s by one Newton step on the f32 reciprocal: 2^-46)
    const double m = st.m, rs = (double)(1.0f / (float)st.s), ratio = (double)st.u * (rs * (2.0 - st.s * rs));
    // k is m log2 e in f32: to first order, what its rounding did to the sum
    const double ln_s = log(st.s) + LN2_D * A.sc.dk * ratio;
    const double lp = ((double)in.c_tok - m) * A.sc.md - ln_s;
    const double H = ln_s - LN2_D * (1.0 + A.sc.dk) * ratio;
    Coef c{st.m, (float)(ln_s * (1.0 / LN2_D)), 0.0f, 0.0f, 0.0f, 1u, 0.0, 0.0, 0.0};
    double kl = 0.0, loss = 0.0;
    if (is_policy(OP)) {
        const double adv = in.adv, dr = (double)in.ref_lp - lp;
        double x1[3] = {lp - (double)in.old_lp, dr, lp};
        by_lanes(x1, [](double v) { return expm1(v); });
        // (1 + expm1 has the exponential's bits but where it is small)
        const double r = x1[0] < -0.5 ? exp(lp - (double)in.old_lp) : 1.0 + x1[0];
        // min(r A, clip(r) A) is the clipped one only beyond the bound that A favours
        const bool over = adv > 0.0 && r > A.clip_hi, under = adv < 0.0 && r < A.clip_lo;
        loss = -adv * (over ? A.clip_hi : under ? A.clip_lo : r);
        double g = over || under ? 0.0 : -r * adv;
        if (A.ref_lp) {
            kl = x1[1] - dr;
            if (A.kl_coef != 0.0f) {
                loss += (double)A.kl_coef * kl;
                g -= (double)A.kl_coef * x1[1];
            }
        }
        const double ent = OP == OP_POLICY_ENT ? (double)A.ent_coef : 0.0, wm = (double)in.w * A.sc.md;
        if (OP == OP_POLICY_ENT) loss -= ent * H;
        c.ct = (float)(wm * token_slope(lp, x1[2], H, g, -ent)) * in.slope;
        c.ca = (float)(wm * (OP == OP_POLICY_ENT ? ent * H - g : -g));
        c.cb = OP == OP_POLICY_ENT ? (float)(wm * ent * LN2_D) : 0.0f;
    }
    if (write) {
        if (is_policy(OP)) A.row_loss[row] = (float)loss;
        if (A.logprobs) A.logprobs[row] = (float)lp;
        if (A.entropy) A.entropy[row] = (float)H;
        if (A.kl) A.kl[row] = (float)kl;
        if (A.stats) A.stats[row] = make_float2(st.m, (float)ln_s);
    }
    return c;
}

// The teacher's slots of a row, in one of four sets.
struct Slots {
    double *q;        // the slot's share, but for the row's scale
    int32_t *id;      // -1: empty; padded to a multiple of 4 with empty ones
    float *c, *v;     // the student's c(v) there and (under a soft-cap) v
    uint32_t *bits;   // one bit per element of the CTA's slice: named by the teacher
};
template <bool CAP> __host__ __device__ constexpr uint32_t slot_words() { return CAP ? 5 : 4; }
__host__ __device__ __forceinline__ uint32_t slots_padded(uint32_t n_ids) { return (n_ids + 3u) & ~3u; }

// Results and coefficients of a row with a teacher, in 64 bits as those of a
// row with a token: a student near its teacher has a loss near 0.  With TAIL,
// st is of the tokens that the teacher does not name, the rest R, on a scale of
// its own: however far it lies below the others (or above), log p_R and the
// shares p_j / p_R that its gradient goes by are finite,
//     dv_j = w m c'(v_j) (p_j / p_R) (Q p_R - q_R)  in R,
// and `top` is the sum of exp((c - U) m) over the named ones.
template <bool TAIL>
__device__ __forceinline__ Coef teacher_row(const RowArgs &A, uint32_t row, const Stat &st, double top, const Teacher &t, float w,
                                            bool write) {
    const double wm = (double)w * A.sc.md, u = (double)anchor(t.u);
    double s = st.s, big = (double)st.m, below = 1.0;
    if (TAIL) {
        const double d = ((double)st.m - (double)t.u) * A.sc.md, e = exp_d(-fabs(d));
        if (d >= 0.0) {
            s += top * e;
        } else {
            below = e;
            s = s * e + top;
            big = (double)t.u;
        }
    }
    const double qr = 1.0 - t.mass;
    double ln[3] = {s, st.s, qr};
    if (TAIL) by_lanes(ln, [](double v) { return log(v); });
    else ln[0] = log(s);
    const double lse = (big - u) * A.sc.md + ln[0];   // relative to U
    double loss = t.cross + t.mass * lse, mass = t.mass;
    Coef c{st.m, (float)(ln[TAIL ? 1 : 0] * (1.0 / LN2_D)), 0.0f, 0.0f, 0.0f, 1u, lse, 0.0, wm};
    if (TAIL) {   // the rest as one outcome
        if (st.s == 0.0) {
            c.m = c.l2s = 0.0f;
        } else {
            const bool has = !(qr <= 0.0);
            if (has) {
                loss += qr * (ln[2] - (((double)st.m - big) * A.sc.md + ln[1] - ln[0]));
                mass += qr;
            }
            c.ca = (float)(wm * (mass * (st.s * below / s) - (has ? qr : 0.0)));
        }
    } else {
        c.ca = (float)(wm * mass);
    }
    c.q_all = mass;
    if (write) A.row_loss[row] = (float)loss;
    return c;
}

template <typename T, int OP, bool CAP>
__global__ void __launch_bounds__(row_threads(OP, compute_threads<T>()), 1) k_rows(RowArgs A, uint32_t rows, uint32_t clusters) {
    constexpr bool DIST = is_distill(OP), TAIL = OP == OP_DISTILL_TAIL;
    constexpr uint32_t COMPUTE = compute_threads<T>();
    constexpr int E = Row<T>::E;
    extern __shared__ uint4 dyn[];
    __shared__ __align__(16) RowsShared sh;
    const uint32_t ranks = 1u << A.log_ranks, rank = cluster_rank();
    const uint32_t cluster = blockIdx.x >> A.log_ranks, tid = threadIdx.x, lane = tid & 31, V = A.vocab;
    const uint32_t n = (rows - cluster + clusters - 1) / clusters;   // rows of this cluster
    const float k = A.sc.k;
    const bool grad = A.grad != nullptr;
    // threads of S and G, and of the barriers
    constexpr uint32_t ST = sum_threads_of<T, CAP>(), GT = COMPUTE - ST;
    const uint32_t sum_threads = grad ? ST : COMPUTE, x_threads = sum_threads + 32;
    const uint32_t y_threads = GT + 32;
    const uint32_t z_threads = (grad ? GT : COMPUTE + 32) + 32 + (DIST ? 32 : 0);
    // f32 logits under a soft-cap: S leaves c(v) in the buffer, so that G need not work it out again (v above the cap)
    constexpr bool LEAVE = CAP && sizeof(T) == 4;
    // Chunks of a thread summed at a time.  Under a soft-cap, with 4 and 2: distillation 512 x 256000 f32 326 and 291 us,
    // 2048 x 128256 bf16 409 and 387; policy loss 777 x 151936 f32 197 and 195, 2048 x 128256 bf16 388 and 398.
    constexpr int STEP = CAP && (DIST || sizeof(T) == 4) ? 2 : 4;
    auto row_of = [&](uint32_t i) { return cluster + i * clusters; };
    auto weight = [&](uint32_t row) { return A.weights ? A.weights[row] : A.w_all; };
    // the slice [c0, c1) of a row's chunks
    struct Slice {
        uint32_t c0, c1;
    };
    auto slice_of = [&](const Row<T> &R) {
        const uint32_t per = (R.chunks + ranks - 1) >> A.log_ranks, c0 = min(rank * per, R.chunks);
        return Slice{c0, min(c0 + per, R.chunks)};
    };
    const uint32_t pad = DIST ? slots_padded(A.n_ids) : 0u;
    auto slots = [&](uint32_t i) {
        const uint32_t set = i & 3;
        char *base = (char *)(dyn + 3 * (size_t)A.keep);
        Slots s;
        s.q = (double *)base + set * pad;
        s.id = (int32_t *)base + (8 + set) * pad;
        s.c = (float *)base + (12 + set) * pad;
        s.v = (float *)base + (16 + set) * pad;
        s.bits = (uint32_t *)base + 4 * slot_words<CAP>() * pad + set * A.bit_words;
        return s;
    };

    // rows' codes, four ahead
    if (tid >= COMPUTE && tid < COMPUTE + 32) {
        if (lane < 4 && lane < n) {
            const uint32_t row = row_of(lane);
            const int32_t tok = DIST ? 0 : A.tokens[row];
            sh.code[lane] = weight(row) != 0.0f && (uint32_t)tok < V ? tok : -1;
        }
    } else if (DIST && tid >= COMPUTE) {
        for (uint32_t i = tid - COMPUTE - 32; i < 4 * A.bit_words; i += BTHREADS + 64) slots(0).bits[i] = 0;
    }
    if (tid == 0) {
        for (int i = 0; i < 4; i++) bar_init(&sh.mail_bar[i]), bar_init(&sh.slots_bar[i]);
        for (int i = 0; i < 3; i++) bar_init(&sh.full_bar[i]);
        sh.gone = sh.passed = 0u;
        for (int i = 0; i < 4; i++) sh.far[i] = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (ranks > 1) {   // every CTA of the row runs, its mail barriers ready
        cluster_arrive();
        cluster_wait();
    }

    // A wait that gives up is the CTA's last: from there on it starts no copies and no exchanges, and its rows are NaN.
    // (The other CTAs of the row then miss its mail, and give up too.)  All warps still go through all rows and meet at
    // the barriers, so that none is left waiting.
    const volatile uint32_t *const gone = &sh.gone;
    const uint32_t give_up = rank == A.gone_rank ? A.gone_row : 0xFFFFFFFFu;
    auto wait = [&](const uint64_t *bar, uint32_t parity, uint32_t i) {
        if (i < give_up && bar_wait(bar, parity, A.wait_limit, gone)) return true;
        *const_cast<volatile uint32_t *>(gone) = 1u;
        *const_cast<volatile uint32_t *>(&wait_gave_up) = 1u;
        return false;
    };

    if (tid < sum_threads) {
        // ---- warps S; thread tid has the chunks tid, tid + sum_threads, ... of the slice
        uint32_t at = 0, phase = 0;   // the buffers take turns
        bool there = true;
        for (uint32_t i = 0; i < n; i++) {
            const Row<T> R(A.x, A.ld, row_of(i), V);
            const Slice sl = slice_of(R);
            const uint32_t count = sl.c1 - sl.c0, copied = min(count, A.keep);
            uint4 *buf = dyn + at * A.keep + tid;
            there = there && wait(&sh.full_bar[at], phase, i);
            if (++at == 3) at = 0, phase ^= 1;
            if (DIST) there = there && wait(&sh.slots_bar[i & 3], i >> 2 & 1, i);
            if (!there) {
                // without copies to wait for: not further ahead of the other warps than with them
                const volatile uint32_t *const passed = &sh.passed;
                const long long start = clock64();
                while (*passed + 2 < i && clock64() - start < WAIT_LIMIT) __nanosleep(200);
            }
            there = __all_sync(~0u, there);
            Gather<T, CAP, !DIST> G;
            const Note note{CAP && grad ? &sh.far[i & 3] : nullptr, i + 1}, none{};
            if (there && sh.code[i & 15] >= 0) {
                const uint32_t *bits = TAIL ? slots(i).bits : nullptr;
                auto marks = [&](uint32_t c) -> uint32_t {
                    if (!TAIL) return 0u;
                    const uint32_t b = c * E;
                    return bits[b >> 5] >> (b & 31) & ((1u << E) - 1u);
                };
                // (LEAVE: c(v), and into the buffer what G starts from: v itself beyond the cap, for its slope)
                auto capped_chunk = [&](const uint4 &q, uint4 *left) {
                    f2 v[E / 2];
                    cap_chunk<T, CAP>(q, v, A.sc, note);
                    const uint4 c = pack<T>(v);
                    if (grad) {
                        *left = c;
                        if (max_abs<T>(q) > A.sc.cap) {
                            const float cap = A.sc.cap;
                            *left = make_uint4(fabsf(__uint_as_float(q.x)) > cap ? q.x : c.x, fabsf(__uint_as_float(q.y)) > cap ? q.y : c.y,
                                               fabsf(__uint_as_float(q.z)) > cap ? q.z : c.z, fabsf(__uint_as_float(q.w)) > cap ? q.w : c.w);
                        }
                    }
                    return c;
                };
                // (a chunk's named tokens left out)
                auto leave_out = [&](uint4 &q, uint32_t mk) {
                    if (CAP && max_abs<T>(q) > A.sc.cap) note.put();
                    mask_out<T>(q, mk);
                };
                // several chunks at a time, for one comparison with the running maximum
                uint32_t c = tid;
                for (; c + (STEP - 1) * sum_threads < copied; c += STEP * sum_threads, buf += STEP * sum_threads) {
                    uint4 q[STEP];
                    uint32_t mk[STEP];
#pragma unroll
                    for (int u = 0; u < STEP; u++) q[u] = buf[u * sum_threads], mk[u] = marks(c + u * sum_threads);
                    if constexpr (LEAVE) {
                        // (the soft-cap of all of them first: that of the largest alone would be waited for)
#pragma unroll
                        for (int u = 0; u < STEP; u++) {
                            q[u] = capped_chunk(q[u], buf + u * sum_threads);
                            if (mk[u]) mask_out<T>(q[u], mk[u]);
                        }
                        G.raise(max_of<T>(q), k);
#pragma unroll
                        for (int u = 0; u < STEP; u++) {
                            f2 v[E / 2];
                            unpack<T>(q[u], v);
                            G.chunk(v, k);
                        }
                        G.step();
                    } else {
#pragma unroll
                        for (int u = 0; u < STEP; u++)
                            if (mk[u]) leave_out(q[u], mk[u]);
                        G.raise(capped<CAP>(max_of<T>(q), A.sc), k);
#pragma unroll
                        for (int u = 0; u < STEP; u++) G.chunk(q[u], A.sc, mk[u], mk[u] ? none : note);
                        G.step();
                    }
                }
                for (; c < copied; c += sum_threads, buf += sum_threads) {
                    uint4 q = buf[0];
                    const uint32_t mk = marks(c);
                    if constexpr (LEAVE) capped_chunk(q, buf);
                    if (mk) leave_out(q, mk);
                    G.raise(capped<CAP>(max_of<T>(q), A.sc), k);
                    G.chunk(q, A.sc, mk, mk ? none : note);
                    G.step();
                }
                // what did not fit
                const T *x = R.at(sl.c0);
                for (c = copied + tid; c < count; c += STEP * sum_threads) {
                    uint4 q[STEP];
#pragma unroll
                    for (int u = 0; u < STEP; u++)
                        if (c + u * sum_threads < count) q[u] = ld_stream(x + (size_t)(c + u * sum_threads) * E);
#pragma unroll
                    for (int u = 0; u < STEP; u++)
                        if (c + u * sum_threads < count) {
                            const uint32_t mk = marks(c + u * sum_threads);
                            if (mk) leave_out(q[u], mk);
                            G.raise(capped<CAP>(max_of<T>(q[u]), A.sc), k);
                            G.chunk(q[u], A.sc, mk, mk ? none : note);
                            G.step();
                        }
                }
            }
            // (the buffer is written by copies again)
            if (LEAVE && grad) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            Stat st{0.0, -INFINITY, 0.0f};
            if (there && sh.code[i & 15] >= 0) st = fold_lanes<!DIST, 32>(G.stat(), k);
            if (lane == 0) sh.part[i & 3][tid >> 5] = Stat{st.s, there ? st.m : NAN, st.u};
            bar_arrive(BAR_X + (i & 3), x_threads);
            if (!grad) bar_arrive(BAR_Z + (i & 3), z_threads);
        }
    } else if (tid < COMPUTE) {
        // ---- warps G
        const uint32_t g = tid - ST;
        uint32_t at = 0;
        for (uint32_t i = 0; i < n; i++) {
            const uint32_t row = row_of(i);
            const Row<T> R(A.x, A.ld, row, V);
            const Slice sl = slice_of(R);
            const uint32_t count = sl.c1 - sl.c0, copied = min(count, A.keep);
            const uint4 *buf = dyn + at * A.keep + g;
            at = at == 2 ? 0 : at + 1;
            T *out = (T *)A.grad + (size_t)row * A.ld_grad + R.lead + (size_t)sl.c0 * E;
            const bool wide = ((uintptr_t)out & 15u) == 0;   // aligned like the logits
            auto store = [&](uint32_t c, const uint4 &q) {
                if (wide) *reinterpret_cast<uint4 *>(out + (size_t)c * E) = q;
                else store_each<T>(out + (size_t)c * E, q);
            };
            bar_sync(BAR_Y + (i & 3), y_threads);
            const Coef cf = sh.coef[i & 3];
            if (cf.live == 1u) {
                const GradRow<OP == OP_POLICY_ENT> gr{cf.m, k, cf.l2s, cf.ca, cf.cb};
                const T *x = R.at(sl.c0);
                if (CAP && __builtin_expect(sh.far[i & 3] == i + 1, 0)) {
                    // logits above the soft-cap (777 x 151936 f32, cap 30: 198 us without, 249 with 16 a row, 405 with half of
                    // all; 2048 x 128256 bf16 401, 430, 682)
#pragma unroll 2
                    for (uint32_t c = g; c < copied; c += GT, buf += GT) store(c, gr.template chunk<T, CAP, LEAVE>(*buf, A.sc));
                    for (uint32_t c = copied + g; c < count; c += GT) store(c, gr.template chunk<T, CAP>(ld_stream(x + (size_t)c * E), A.sc));
                } else {
                    if (wide) {
                        uint4 *o = reinterpret_cast<uint4 *>(out) + g;
#pragma unroll 4
                        for (uint32_t c = g; c < copied; c += GT, buf += GT, o += GT)
                            *o = gr.template near<T, CAP, LEAVE>(*buf, A.sc);
                    } else {
                        for (uint32_t c = g; c < copied; c += GT, buf += GT)
                            store(c, gr.template near<T, CAP, LEAVE>(*buf, A.sc));
                    }
                    for (uint32_t c = copied + g; c < count; c += STEP * GT) {
                        uint4 q[STEP];
#pragma unroll
                        for (int u = 0; u < STEP; u++)
                            if (c + u * GT < count) q[u] = ld_stream(x + (size_t)(c + u * GT) * E);
#pragma unroll
                        for (int u = 0; u < STEP; u++)
                            if (c + u * GT < count) store(c + u * GT, gr.template near<T, CAP>(q[u], A.sc));
                    }
                }
                if (!DIST) {
                    // the token's own element, written again by the thread that wrote its chunk (where the token
                    // is a single element, warp A has it)
                    const uint32_t t_at = (uint32_t)sh.code[i & 15] - R.lead - sl.c0 * E;
                    const uint32_t t = t_at / E, mine = t < copied ? t : t - copied;
                    if (t < count && mine % GT == g) out[t_at] = from_f<T>(cf.ct);
                }
            } else {   // the row is left out: zeros; or lost: NaN
                f2 v[E / 2];
                for (int e = 0; e < E / 2; e++) v[e] = both(cf.live ? NAN : 0.0f);
                const uint4 fill = pack<T>(v);
                for (uint32_t c = g; c < count; c += GT) store(c, fill);
            }
            bar_arrive(BAR_Z + (i & 3), z_threads);
        }
    } else if (tid < COMPUTE + 64) {
        // ---- warps A; this one has every other row
        const uint32_t which = (tid - COMPUTE) >> 5;
        struct Params {
            TokenIn in;
            T tok, edge;   // as loaded: a conversion here would wait for the load
        };
        auto edge_of = [&](uint32_t i) {
            return rank == 0 ? Row<T>(A.x, A.ld, row_of(i), V).edge(lane) : -1;
        };
        auto params = [&](uint32_t i) {   // loads only; used an iteration later
            Params p{};
            const int32_t code = sh.code[i & 15];
            if (i < n && code >= 0) {
                const uint32_t row = row_of(i);
                const T *x = (const T *)A.x + (size_t)row * A.ld;
                p.in.w = weight(row);
                if (!DIST) p.tok = x[code];
                if (is_policy(OP)) {
                    p.in.adv = A.adv[row];
                    p.in.old_lp = A.old_lp[row];
                    p.in.ref_lp = A.ref_lp ? A.ref_lp[row] : 0.0f;
                }
                const int32_t e = edge_of(i);
                if (e >= 0) p.edge = x[e];
            }
            return p;
        };
        Params next = params(which);
        float w4 = 0.0f;          // weight and token of row i + 4
        int32_t t4 = -1;
        auto load4 = [&](uint32_t i) {
            if (i + 4 < n && lane == 0) {
                w4 = weight(row_of(i + 4));
                t4 = DIST ? 0 : A.tokens[row_of(i + 4)];
            }
        };
        load4(which);
        uint32_t sent = 0;        // exchanges of this warp so far
        bool failed = false, stopped = false;   // its last one gave up; or what S waited for did
        for (uint32_t i = which; i < n; i += 2) {
            const Params cur = next;
            const uint32_t row = row_of(i);
            if (i + 2 < n) next = params(i + 2);
            if (lane == 0 && i + 4 < n) sh.code[(i + 4) & 15] = w4 != 0.0f && (uint32_t)t4 < V ? t4 : -1;
            load4(i + 2);
            bar_sync(BAR_X + (i & 3), x_threads);
            const int32_t edge = edge_of(i);
            const float c_edge = capped<CAP>(to_f(cur.edge), A.sc);
            const float c_tok = DIST ? 0.0f : capped<CAP>(to_f(cur.tok), A.sc);
            Stat st{0.0, -INFINITY, 0.0f};
            if (lane < sum_threads / 32) st = sh.part[i & 3][lane];
            stopped = __any_sync(~0u, st.m != st.m || stopped);
            const bool wanted = sh.code[i & 15] >= 0;
            bool lost = wanted && stopped, live = wanted && !lost;
            if (DIST && live) live = sh.teacher[i & 3].live != 0u;
            if (!grad && !DIST) bar_arrive(BAR_Z + (i & 3), z_threads);   // the sums are read: S may go on
            if (live && edge >= 0 && !(TAIL && (sh.edge_marks[i & 3] >> lane & 1u))) {
                // one logit: 2^0 at itself, nothing where it is -inf (or a sum of NaN)
                const float one = c_edge == -INFINITY ? 0.0f : c_edge - c_edge == 0.0f ? 1.0f : NAN;
                const float m = c_edge != c_edge ? st.m : fmaxf(st.m, c_edge);
                const float da = fmaxf((st.m - m) * k, D_MIN), db = fmaxf((c_edge - m) * k, D_MIN), fa = ex2(da), fb = ex2(db);
                st = Stat{st.s * fa + (double)(one * fb), m, fa * fmaf(da, (float)st.s, st.u) + fb * (db * one)};
            }
            st = fold_lanes<!DIST, 32>(st, k);
            double top = TAIL && live ? sh.teacher[i & 3].top : 0.0;
            if (ranks > 1 && wanted && !lost) {
                // The rows that take part in an exchange count the same in every CTA.  A warp's exchanges take turns
                // with two boxes: a CTA sends into one only after all have sent into the other, so have read what
                // was in this one.  The token's logit goes along so that it has been read before another CTA may
                // write the gradient over it.
                const uint32_t box = which * 2 + (sent & 1), turn = sent >> 1 & 1;
                sent++;
                const double big = TAIL ? top : st.s;   // (with a tail the named ids' sum has the 64 bits, the rest's 32)
                const float small = TAIL ? (float)st.s : st.u;
                uint4 out = make_uint4(__double2loint(big), __double2hiint(big), __float_as_uint(st.m), __float_as_uint(small));
                if (!DIST) out.x |= __float_as_uint(c_tok) & A.zero;
                if (lane < ranks) mail_send(&sh.mail[box][rank], &sh.mail_bar[box], lane, out);
                if (lane == 0) bar_expect(&sh.mail_bar[box], ranks * 16);
                lost = !__all_sync(~0u, wait(&sh.mail_bar[box], turn, i));
                live = live && !lost;
                failed = stopped = lost;
                st = Stat{0.0, -INFINITY, 0.0f};
                top = 0.0;
                if (lane < ranks) {
                    const uint4 f = sh.mail[box][lane];
                    const double big = __hiloint2double(f.y, f.x);
                    const float small = __uint_as_float(f.w);
                    st = Stat{TAIL ? (double)small : big, __uint_as_float(f.z), TAIL ? 0.0f : small};
                    if (TAIL) top = big;
                }
                if (TAIL) {
                    for (int o = MAX_CLUSTER / 2; o; o >>= 1) top += __shfl_xor_sync(~0u, top, o);
                    top = __shfl_sync(~0u, top, 0);
                }
                st = fold_lanes<!DIST, MAX_CLUSTER>(st, k);
                st.m = __shfl_sync(~0u, st.m, 0);
                st.s = __shfl_sync(~0u, st.s, 0);
                st.u = __shfl_sync(~0u, st.u, 0);
            }
            const bool write = rank == 0 && lane == 0;
            Coef cf{};
            if (live) {
                if constexpr (DIST) {
                    cf = teacher_row<TAIL>(A, row, st, top, sh.teacher[i & 3], cur.in.w, write);
                } else {
                    TokenIn in = cur.in;
                    in.c_tok = c_tok;
                    in.slope = cap_both<CAP>(to_f(cur.tok), A.sc).y;
                    cf = token_row<OP>(A, row, st, in, write);
                }
            } else {
                const float none = lost ? NAN : 0.0f;
                if (write) {
                    if (A.logprobs) A.logprobs[row] = none;
                    if (A.entropy) A.entropy[row] = none;
                    if (A.kl) A.kl[row] = none;
                    A.row_loss[row] = none;
                }
                if (lost) cf.live = 2u;
            }
            if (grad && edge >= 0) {
                float o = lost ? NAN : 0.0f;
                if (live) {
                    const GradRow<OP == OP_POLICY_ENT> gr{cf.m, k, cf.l2s, cf.ca, cf.cb};
                    o = !DIST && edge == sh.code[i & 15] ? cf.ct : gr.one(c_edge) * cap_both<CAP>(to_f(cur.edge), A.sc).y;
                }
                ((T *)A.grad)[(size_t)row * A.ld_grad + edge] = from_f<T>(o);
            }
            if (lane == 0) sh.coef[i & 3] = cf;
            __syncwarp();
            if (grad) bar_arrive(BAR_Y + (i & 3), y_threads);
            else if (DIST) bar_arrive(BAR_Z + (i & 3), z_threads);   // (done with the slots)
        }
        if (lane < ranks)
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote(&sh.sent[which][rank], lane)), "r"(sent) : "memory");
        if (lane == 0) sh.failed[which] = failed;
    } else if (tid < COMPUTE + 96) {
        // ---- warp C: row i + 3 into row i's buffer
        auto copy = [&](uint32_t i) {
            uint64_t *bar = &sh.full_bar[i % 3];
            const Row<T> R(A.x, A.ld, row_of(i), V);
            const Slice sl = slice_of(R);
            const uint32_t copied = sh.code[i & 15] < 0 ? 0u : min(sl.c1 - sl.c0, A.keep);
            if (lane == 0) bar_expect(bar, copied * 16);
            __syncwarp();
            uint4 *buf = dyn + (i % 3) * A.keep;
            for (uint32_t c = lane * COPY; c < copied; c += 32 * COPY)
                copy_bulk(buf + c, R.at(sl.c0 + c), min(copied - c, COPY) * 16, bar);
        };
        uint32_t started = 0;
        for (; started < 3 && started < n; started++) copy(started);
        for (uint32_t i = 0; i < n; i++) {
            bar_sync(BAR_Z + (i & 3), z_threads);
            if (lane == 0) *const_cast<volatile uint32_t *>(&sh.passed) = i + 1;
            if (i + 3 < n && !__any_sync(~0u, *gone != 0u)) copy(started++);
        }
        // (S has seen every copy land; were it to have given up on one, it still lands before the CTA's memory goes)
        for (uint32_t i = started > 3 ? started - 3 : 0; i < started; i++) bar_wait(&sh.full_bar[i % 3], i / 3 & 1, WAIT_LIMIT, nullptr);
    } else if constexpr (DIST) {
        // ---- warps B; warp w has the rows w, w + 4, ..., and the set w of slots
        const uint32_t set = (tid - COMPUTE - 96) >> 5;
        const Slots sl = slots(set);
        // (f32 as a whole number of the same order; a NaN is the largest, 0 is below all)
        auto order = [](float v) {
            const uint32_t u = __float_as_uint(v);
            return v != v ? ~0u : u & 0x80000000u ? ~u : u | 0x80000000u;
        };
        auto value = [](uint32_t key) {
            return key == ~0u ? NAN : __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
        };
        // A row's weight and lse and a lane's first slots, loaded while the row four before is worked on; the student's
        // logits there once the ids have come.
        struct Ahead {
            float w, lse, t[AHEAD];
            int32_t id[AHEAD];
            T x[AHEAD];
        } f;
        auto fetch_slots = [&](uint32_t row, uint32_t j0) {
#pragma unroll
            for (int a = 0; a < AHEAD; a++) {
                const uint32_t j = j0 + lane + 32 * a;
                f.id[a] = -1;
                if (j < A.n_ids) {
                    f.id[a] = A.t_ids[(size_t)row * A.n_ids + j];
                    f.t[a] = A.t_logits[(size_t)row * A.n_ids + j];
                }
            }
        };
        auto fetch_logits = [&](uint32_t row) {
#pragma unroll
            for (int a = 0; a < AHEAD; a++)
                if ((uint32_t)f.id[a] < V) f.x[a] = ((const T *)A.x)[(size_t)row * A.ld + (uint32_t)f.id[a]];
        };
        auto fetch = [&](uint32_t i) {
            if (i < n) {
                f.w = weight(row_of(i));
                if (TAIL) f.lse = A.t_lse[row_of(i)];
                fetch_slots(row_of(i), 0);
            }
        };
        auto fetch_row_logits = [&](uint32_t i) {
            if (i < n && f.w != 0.0f) fetch_logits(row_of(i));
        };
        // in the CTA's slice, or (rank 0) a single element
        auto mine = [&](int32_t id, const Row<T> &R, uint32_t e0, uint32_t span) {
            const bool single = (uint32_t)id < R.lead || (uint32_t)id >= V - R.trail;
            return single ? rank == 0 : (uint32_t)id - e0 < span;
        };
        bool twice = false;   // an id of the slice comes twice
        auto prepare = [&](uint32_t i) {
            const uint32_t row = row_of(i);
            const Row<T> R(A.x, A.ld, row, V);
            const Slice part = slice_of(R);
            const uint32_t e0 = R.lead + part.c0 * E, span = (part.c1 - part.c0) * E;
            const bool wanted = f.w != 0.0f;
            uint32_t most_t = 0u, most_c = 0u;   // the largest of the teacher's logits and of c(v); 0 without a slot
            if (lane == 0) sh.edge_marks[set] = 0u;
            if (wanted) {
                for (uint32_t j0 = 0; j0 < pad; j0 += 32 * AHEAD) {
                    if (j0) {
                        fetch_slots(row, j0);
                        fetch_logits(row);
                    }
#pragma unroll
                    for (int a = 0; a < AHEAD; a++) {
                        const uint32_t j = j0 + lane + 32 * a;
                        if (j >= pad) continue;
                        const bool valid = (uint32_t)f.id[a] < V;
                        sl.id[j] = valid ? f.id[a] : -1;
                        if (valid) {
                            const float c = capped<CAP>(to_f(f.x[a]), A.sc);
                            sl.q[j] = (double)f.t[a];
                            sl.c[j] = c;
                            if (CAP) sl.v[j] = to_f(f.x[a]);
                            most_t = max(most_t, order(f.t[a]));
                            most_c = max(most_c, order(c));
                        }
                    }
                }
                most_t = __reduce_max_sync(~0u, most_t);
                most_c = __reduce_max_sync(~0u, most_c);
            }
            __syncwarp();
            // (without a teacher's lse there may be no share to give: as without ids)
            const bool live = wanted && most_c != 0u && (TAIL || most_t != order(-INFINITY));
            if (live) {
                const double ref = TAIL ? (double)f.lse : (double)value(most_t) * A.sc.inv_t, u = (double)anchor(value(most_c));
                double sum = 0.0, cross = 0.0;   // of q, of q (log q - (c - U) m); without an lse, q is not yet divided by its sum
                bool again = false;
                for (uint32_t j = lane; j < pad; j += 32) {
                    const int32_t id = sl.id[j];
                    if (id < 0) continue;
                    const double a = sl.q[j] * A.sc.inv_t - ref, q = exp_d(a);
                    sl.q[j] = q;
                    if (!(q <= 0.0)) {
                        sum += q;
                        cross += q * (a - ((double)sl.c[j] - u) * A.sc.md);
                    }
                    const uint32_t e = (uint32_t)id - e0;
                    uint32_t *word = &sl.bits[e >> 5], bit = 1u << (e & 31);
                    if (e >= span) {
                        word = &sh.edge_marks[set];
                        bit = (uint32_t)id < R.lead ? 1u << id : (uint32_t)id >= V - R.trail ? 256u << (id - (V - R.trail)) : 0u;
                    }
                    if (bit && (atomicOr(word, bit) & bit)) again = true;
                }
                twice = __any_sync(~0u, again);
                __syncwarp();   // all of sl.id is there
                double top = 0.0;
                if (TAIL) {
                    for (uint32_t j = lane; j < pad; j += 32) {
                        const int32_t id = sl.id[j];
                        if (id < 0 || !mine(id, R, e0, span)) continue;
                        bool first = true;
                        for (uint32_t o = 0; twice && o < j; o++) first = first && sl.id[o] != id;
                        if (first) top += exp_d(((double)sl.c[j] - u) * A.sc.md);
                    }
                }
                for (int o = 16; o; o >>= 1) {
                    sum += __shfl_xor_sync(~0u, sum, o);
                    cross += __shfl_xor_sync(~0u, cross, o);
                    if (TAIL) top += __shfl_xor_sync(~0u, top, o);
                }
                const double scale = TAIL ? 1.0 : 1.0 / sum;
                if (!TAIL) cross = cross * scale - log(sum);
                if (lane == 0) sh.teacher[set] = Teacher{cross, sum * scale, scale, top, value(most_c), 1u};
            } else if (lane == 0) {
                sh.teacher[set].live = 0u;
            }
            __syncwarp();
        };
        auto finish = [&](uint32_t i) {
            const uint32_t row = row_of(i);
            const Coef cf = sh.coef[set];
            const Row<T> R(A.x, A.ld, row, V);
            const Slice part = slice_of(R);
            const uint32_t e0 = R.lead + part.c0 * E, span = (part.c1 - part.c0) * E;
            if (!sh.teacher[set].live) return;
            const double u = (double)anchor(sh.teacher[set].u), scale = sh.teacher[set].scale;
            T *out = (T *)A.grad + (size_t)row * A.ld_grad;
            for (uint32_t j = lane; j < A.n_ids; j += 32) {
                const int32_t id = sl.id[j];
                if (id < 0) continue;
                const uint32_t e = (uint32_t)id - e0;
                if (!mine(id, R, e0, span)) continue;
                if (e < span) sl.bits[e >> 5] = 0u;
                if (!grad || cf.live != 1u) continue;
                // p Q - q, where q is the sum over the slots that hold the id (the first of them writes)
                double q = sl.q[j];
                bool first = true;
                if (twice) q = 0.0;
                for (uint32_t o = 0; twice && o < pad; o += 4) {
                    const int4 v = *reinterpret_cast<const int4 *>(sl.id + o);
                    if (v.x == id) q += sl.q[o], first = first && o >= j;
                    if (v.y == id) q += sl.q[o + 1], first = first && o + 1 >= j;
                    if (v.z == id) q += sl.q[o + 2], first = first && o + 2 >= j;
                    if (v.w == id) q += sl.q[o + 3], first = first && o + 3 >= j;
                }
                if (!first) continue;
                const float c = sl.c[j], slope = CAP ? cap_slope(c, sl.v[j], A.sc) : 1.0f;
                const double p = exp_d(((double)c - u) * A.sc.md - cf.lse);
                out[id] = from_f<T>((float)(cf.wm * (p * cf.q_all - q * scale)) * slope);
            }
        };
        fetch(set);
        fetch_row_logits(set);
        for (uint32_t i = set; i < n; i += 4) {
            prepare(i);
            if (lane == 0) bar_arrive_local(&sh.slots_bar[set]);
            fetch(i + 4);
            bar_sync(BAR_Z + set, z_threads);          // row i's gradient is written
            fetch_row_logits(i + 4);
            finish(i);
            __syncwarp();
        }
    }
    // No CTA's memory goes while another's mail may be on its way: all have sent what they will, and who gave up waits for
    // what was sent all the same (who did not has seen it).
    if (ranks > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (tid >= COMPUTE && tid < COMPUTE + 4 && *gone) {
            const uint32_t box = tid - COMPUTE, which = box >> 1, odd = box & 1;
            auto into = [&](uint32_t sent) { return (sent + 1 - odd) / 2; };   // of a warp's exchanges, those in this box
            const uint32_t mine = sh.sent[which][rank];
            const bool armed = sh.failed[which] && ((mine - 1) & 1) == odd;    // the one it gave up on
            const uint32_t seen = into(mine) - (armed ? 1 : 0);
            uint32_t left = 0;
            for (uint32_t r = 0; r < ranks; r++) left += (into(sh.sent[which][r]) - seen) * 16;
            if (armed && left < ranks * 16) bar_forgo(&sh.mail_bar[box], ranks * 16 - left);
            if (!armed && left) bar_expect(&sh.mail_bar[box], left);
            if (armed || left) bar_wait(&sh.mail_bar[box], seen & 1, WAIT_LIMIT, nullptr);
        }
    }
}

// The logits' gradient from those of log-probability and entropy, with the
// forward pass's statistics:
//   dv_j = m c'(v_j) [g (d_jt - p_j) - h p_j (log p_j + H)]
// Grid: rows x slices of GRAD_SLICE chunks.  A pure stream, one read and one
// write a logit: 1024 x 151936 bf16 98 us, 97 % of the copy bandwidth; under a
// soft-cap 124.
// The token's element is worked out again in 64 bits (token_slope).
__device__ __noinline__ float token_grad(const Scale &sc, float c, float2 st, float H, float g, float h) {
    const double lp = ((double)c - (double)st.x) * sc.md - (double)st.y;
    return (float)(sc.md * token_slope(lp, expm1(lp), H, g, h));
}
constexpr int GRAD_BATCH = 4;
constexpr uint32_t GRAD_SLICE = THREADS * GRAD_BATCH * 2;   // chunks of a CTA
template <typename T, bool CAP, bool ENT>
__global__ void __launch_bounds__(THREADS) k_logprob_grad(RowArgs A, uint32_t slices, const float2 *stats,
                                                          const float *d_lp, const float *d_ent, const float *entropy) {
    constexpr int E = Row<T>::E;
    const uint32_t row = blockIdx.x / slices, slice = blockIdx.x % slices, tid = threadIdx.x, V = A.vocab;
    Row<T> R(A.x, A.ld, row, V);
    T *gout = (T *)A.grad + (size_t)row * A.ld_grad;
    const bool wide = (((uintptr_t)(gout + R.lead)) & 15u) == 0;
    const uint32_t c0 = slice * GRAD_SLICE, c1 = min(c0 + GRAD_SLICE, R.chunks);
    const int32_t edge = slice == 0 && tid < 32 ? R.edge(tid) : -1;
    const int32_t tok = A.tokens[row];
    const bool live = (uint32_t)tok < V;
    const uint32_t t = ((uint32_t)tok - R.lead) / E;                          // the token's chunk,
    const bool own = live && t - c0 < c1 - c0 && (t - c0) % THREADS == tid;   // and whether this thread has it
    float m = 0.0f, l2s = 0.0f, ca = 0.0f, cb = 0.0f, v_tok = 0.0f;
    const float k = A.sc.k;
    if (live) {
        if (own) v_tok = to_f(R.x[tok]);
        const float2 st = stats[row];
        m = st.x;
        l2s = st.y * (float)(1.0 / LN2_D);
        const float g = d_lp ? d_lp[row] * A.sc.m : 0.0f;
        const float h = ENT ? d_ent[row] * A.sc.m : 0.0f;
        ca = ENT ? -g - h * entropy[row] : -g;
        cb = ENT ? -h * LN2 : 0.0f;
    }
    const GradRow<ENT> gr{m, k, l2s, ca, cb};
    auto store = [&](uint32_t c, const uint4 &q) {
        T *o = gout + R.lead + (size_t)c * E;
        if (wide) *reinterpret_cast<uint4 *>(o) = q;
        else store_each<T>(o, q);
    };
    if (!live) {
        for (uint32_t c = c0 + tid; c < c1; c += THREADS) store(c, make_uint4(0, 0, 0, 0));
        if (edge >= 0) gout[edge] = from_f<T>(0.0f);
        return;
    }
    const T *body = R.at(0);
    for (uint32_t c = c0 + tid; c < c1; c += GRAD_BATCH * THREADS) {
        uint4 q[GRAD_BATCH];
#pragma unroll
        for (int u = 0; u < GRAD_BATCH; u++)
            if (c + u * THREADS < c1) q[u] = ld_stream(body + (size_t)(c + u * THREADS) * E);
#pragma unroll
        for (int u = 0; u < GRAD_BATCH; u++) {
            const uint32_t cu = c + u * THREADS;
            if (cu < c1) store(cu, gr.template chunk<T, CAP>(q[u], A.sc));
        }
    }
    auto at_token = [&](float2 c) {
        return token_grad(A.sc, c.x, stats[row], ENT ? entropy[row] : 0.0f, d_lp ? d_lp[row] : 0.0f, ENT ? d_ent[row] : 0.0f) * c.y;
    };
    // the token's own element, written again by the thread that wrote its chunk
    if (own) gout[tok] = from_f<T>(at_token(cap_both<CAP>(v_tok, A.sc)));
    if (edge >= 0) {
        const float2 c = cap_both<CAP>(to_f(R.x[edge]), A.sc);
        gout[edge] = from_f<T>(edge == tok ? at_token(c) : gr.one(c.x) * c.y);
    }
}

// loss = sum_i w_i L_i in a fixed order, in 64 bits; a row of weight 0 adds
// nothing whatever its loss.
__global__ void __launch_bounds__(1024) k_loss(const float *row_loss, const float *weights, float w_all, uint32_t rows,
                                               float *loss) {
    __shared__ double part[32];
    double s = 0.0;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the rows' losses are there
    for (uint32_t i = threadIdx.x; i < rows; i += 1024) {
        const float w = weights ? weights[i] : w_all;
        if (w != 0.0f) s += (double)w * (double)row_loss[i];
    }
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = part[threadIdx.x];
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        if (threadIdx.x == 0) *loss = (float)s;
    }
}

// Order of the logits as whole numbers: larger logit, larger key; +0 and -0
// alike; a NaN below everything (it never wins, as in the argmax).
__device__ __forceinline__ uint32_t order_key(float v) {
    if (v != v) return 0u;
    uint32_t u = __float_as_uint(v + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t key) {
    if (key == 0u) return NAN;
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// The digit of a radix selection: with `need` elements wanted from the top of
// a 256-bin histogram, the bin that holds the last of them; `need` becomes
// the number wanted from that bin.
__device__ __forceinline__ uint32_t pick_bin(const uint32_t *hist, uint32_t &need) {
    for (int b = 255; b > 0; b--) {
        if (hist[b] >= need) return (uint32_t)b;
        need -= hist[b];
    }
    return 0u;
}

constexpr int TOP_TILE = 8;          // chunks of a tile
constexpr int TOP_CAND = 2048;       // candidates of a row
constexpr uint32_t TOP_EACH = 40960; // most logits whose keys are searched in shared memory
constexpr int TOP_MORE = 16;          // candidate tiles that are not worth another step of the search
struct TopShared {
    unsigned long long cand[TOP_CAND];   // key << 32 | ~id
    union {
        uint16_t tiles[TOP_CAND];
        uint32_t hist[256];
    };
    uint32_t warp[2][WARPS];
    uint32_t chunks[TOP_CAND];
    uint32_t bin, need, n, n_tiles, n_chunks;
};
static_assert(BS_MAX_VOCAB / (16 / 4) / TOP_TILE + 2 <= 65536, "tile numbers fit 16 bits");

// Selection over the whole row by its keys' digits (four passes over the row
// in L2; ties are cut by the same selection over the ids): for rows whose
// candidates do not fit, as those of a few distinct values.
template <typename T> __device__ __noinline__ void select_whole_row(const T *x, uint32_t vocab, uint32_t top, TopShared &sh) {
    const uint32_t tid = threadIdx.x;
    uint32_t need = top, kth = 0, mask = 0, id_floor = 0, id_mask = 0;
    for (int part = 0; part < 2; part++) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            for (uint32_t i = tid; i < 256; i += THREADS) sh.hist[i] = 0;
            __syncthreads();
            for (uint32_t j = tid; j < vocab; j += THREADS) {
                const uint32_t key = order_key(to_f(x[j]));
                if (part == 0 ? (key & mask) == kth : key == kth && (~j & id_mask) == id_floor)
                    atomicAdd(&sh.hist[(part == 0 ? key : ~j) >> shift & 255u], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                sh.bin = pick_bin(sh.hist, need);
                sh.need = need;
            }
            __syncthreads();
            need = sh.need;
            (part == 0 ? kth : id_floor) |= sh.bin << shift;
            (part == 0 ? mask : id_mask) |= 255u << shift;
        }
    }
    if (tid == 0) sh.n = 0;
    __syncthreads();
    for (uint32_t j = tid; j < vocab; j += THREADS) {
        const uint32_t key = order_key(to_f(x[j]));
        if (key > kth || (key == kth && ~j >= id_floor)) {
            const uint32_t at = atomicAdd(&sh.n, 1u);
            if (at < TOP_CAND) sh.cand[at] = (unsigned long long)key << 32 | (uint32_t)~j;
        }
    }
    __syncthreads();
}

// The top logits of one row from its tile maxima; one CTA.  A value that at
// least `top` tile maxima reach is a floor that all of the `top` largest
// logits reach, so only the few tiles above it are read again (mostly from L2)
// and only their logits above it sorted.  Latency bound: the search for the
// floor counts keys in shared memory (a histogram's atomics would meet in a
// few bins), the tiles' loads are under way together, and the sort is one of
// 64 elements in a warp's registers and a rank by binary searches in the other
// warps' runs.  Where there are hardly more tiles than wanted logits (`each`),
// the logits themselves are searched.  A floor below very many equal values is
// left where it is: the larger logits are taken and the rest filled up with the
// lowest ids that have the value.  Measured, with k_stream before it: top 64 of
// 256 x 128256 f32 38 us (10 of them here), top 256 of 1024 x 256000 bf16 136;
// by a radix selection over the whole row 515 and 2015.
struct TopArgs {
    uint32_t top;
    float out_scale;
    bool each, fused;    // fused: k_stream's CTA 0 of a row selects; else k_select
    float *values;
    int32_t *ids;
    float *lse, *maxima;
    uint32_t max_ld;
};
template <typename T, bool CAP>
__device__ __forceinline__ void select_top(const Row<T> &R, uint32_t row, const Scale &sc, const TopArgs &P, TopShared &ts,
                                           uint32_t *keys) {   // keys: of the tile maxima, or (each) of the logits; padded with 0
    constexpr int E = Row<T>::E;
    const uint32_t top = P.top, vocab = R.vocab;
    const bool each = P.each;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t tiles = (R.chunks + TOP_TILE - 1) / TOP_TILE, n_max = each ? vocab : tiles + 1;
    const int32_t edge = tid < 32 ? R.edge(tid) : -1;
    const T *body = R.at(0);
    const float *tile_max = P.maxima + (size_t)row * P.max_ld;
    const float v_edge = edge >= 0 ? to_f(R.x[edge]) : -INFINITY;
    if (tid == 0) ts.n = ts.n_tiles = ts.n_chunks = 0;

    const uint32_t quads = (n_max + 3) / 4;
    uint4 *const key4 = reinterpret_cast<uint4 *>(keys);
    uint32_t hi_key = 0;
    if (each) {
        for (uint32_t i = tid; i < quads * 4; i += 8 * THREADS) {
            float m[8];
#pragma unroll
            for (int u = 0; u < 8; u++) m[u] = i + u * THREADS < n_max ? to_f(R.x[i + u * THREADS]) : NAN;
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const uint32_t key = order_key(m[u]);
                hi_key = max(hi_key, key);
                if (i + u * THREADS < quads * 4) keys[i + u * THREADS] = key;
            }
        }
    } else {
        for (uint32_t i = tid; i < quads; i += 4 * THREADS) {
            float4 m[4];
#pragma unroll
            for (int u = 0; u < 4; u++)
                m[u] = i + u * THREADS < quads ? __ldcg(reinterpret_cast<const float4 *>(tile_max) + i + u * THREADS)
                                               : make_float4(NAN, NAN, NAN, NAN);
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const uint32_t j = (i + u * THREADS) * 4;   // (behind the last maximum the scratch holds nothing)
                const uint4 key = make_uint4(order_key(m[u].x), j + 1 < n_max ? order_key(m[u].y) : 0u,
                                             j + 2 < n_max ? order_key(m[u].z) : 0u, j + 3 < n_max ? order_key(m[u].w) : 0u);
                hi_key = max(max(max(hi_key, key.x), max(key.y, key.z)), key.w);
                if (i + u * THREADS < quads) key4[i + u * THREADS] = key;
            }
        }
    }
    hi_key = __reduce_max_sync(~0u, hi_key);
    if (lane == 0) ts.warp[0][warp] = hi_key;
    __syncthreads();
    for (int i = 0; i < WARPS; i++) hi_key = max(hi_key, ts.warp[0][i]);

    // The largest floor that `top` keys reach, or a little below it: down from
    // the largest key in steps that grow, then by halves.
    uint32_t turn = 1;
    auto reach = [&](uint32_t key) {   // keys of at least `key`
        uint32_t c = 0;
        for (uint32_t i = tid; i < quads; i += 4 * THREADS) {
            uint4 q[4];
#pragma unroll
            for (int u = 0; u < 4; u++) q[u] = i + u * THREADS < quads ? key4[i + u * THREADS] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int u = 0; u < 4; u++) c += (q[u].x >= key) + (q[u].y >= key) + (q[u].z >= key) + (q[u].w >= key);
        }
        c = __reduce_add_sync(~0u, c);
        if (lane == 0) ts.warp[turn][warp] = c;
        __syncthreads();
        c = 0;
        for (int i = 0; i < WARPS; i++) c += ts.warp[turn][i];
        turn ^= 1u;
        return c;
    };
    uint32_t lo = 0, count = n_max;
    bool exact = false;     // no key between lo and the next larger floor, which too few reach
    if (n_max > top) {
        uint32_t hi = hi_key;
        const uint32_t enough = top + top / 8 + TOP_MORE;
        for (uint32_t step = 1u << 22;; step = step < 1u << 30 ? step << 2 : ~0u) {
            lo = hi_key > step ? hi_key - step : 0u;
            count = reach(lo);
            if (count >= top) break;
            hi = lo - 1;                   // (too few reach lo, so lo > 0)
        }
        // `top` keys reach lo; the answer is at most hi
        while (count > enough && lo < hi) {
            const uint32_t mid = lo + (hi - lo + 1) / 2, c = reach(mid);
            if (c >= top) lo = mid, count = c;
            else hi = mid - 1;
        }
        exact = count > enough;
    }
    // the tiles above the floor, then their logits above it; many tiles that
    // just reach it are left to the search for ties below
    const uint32_t floor_key = exact ? lo + 1 : lo;
    // (one place in the list per warp and round; a lane's own by a prefix sum)
    auto place = [&](uint32_t *n, uint32_t mine) {
        uint32_t sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(~0u, sum, o);
            if (lane >= (uint32_t)o) sum += t;
        }
        uint32_t at = 0;
        if (lane == 31 && sum) at = atomicAdd(n, sum);
        return __shfl_sync(~0u, at, 31) + sum - mine;
    };
    for (uint32_t i0 = tid - lane; i0 < quads; i0 += 4 * THREADS) {
        uint4 q[4];
        uint32_t mine = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const uint32_t i = i0 + lane + u * THREADS;
            q[u] = i < quads ? key4[i] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (i * 4 + e < n_max && (&q[u].x)[e] >= floor_key) mine |= 1u << (u * 4 + e);
        }
        uint32_t at = place(each ? &ts.n : &ts.n_tiles, __popc(mine));
#pragma unroll
        for (int b = 0; b < 16; b++)
            if (mine >> b & 1u) {
                const uint32_t i = (i0 + lane + (b / 4) * THREADS) * 4 + b % 4;
                if (at < TOP_CAND) {
                    if (each) ts.cand[at] = (unsigned long long)(&q[b / 4].x)[b % 4] << 32 | (uint32_t)~i;
                    else ts.tiles[at] = (uint16_t)i;
                }
                at++;
            }
    }
    __syncthreads();
    const uint32_t n_tiles = min(ts.n_tiles, (uint32_t)TOP_CAND);   // (fewer than 1024 + 1024 / 8 + TOP_MORE, in fact)
    // first the chunks of these tiles that hold one (about one a tile), then those chunks' logits
    constexpr int SOME = 8;
    for (uint32_t i0 = (tid - lane) >> 3; i0 < n_tiles; i0 += SOME * (THREADS / 8)) {
        uint4 q[SOME];
        uint32_t c[SOME], mine = 0;
#pragma unroll
        for (int u = 0; u < SOME; u++) {
            const uint32_t j = i0 + (lane >> 3) + u * (THREADS / 8), t = j < n_tiles ? ts.tiles[j] : tiles;
            c[u] = t < tiles ? t * TOP_TILE + (lane & 7) : R.chunks;
            if (c[u] < R.chunks) q[u] = ld_stream(body + (size_t)c[u] * E);
        }
#pragma unroll
        for (int u = 0; u < SOME; u++)
            if (c[u] < R.chunks && order_key(max_of<T>(q[u])) >= floor_key) mine |= 1u << u;
        uint32_t at = place(&ts.n_chunks, __popc(mine));
#pragma unroll
        for (int u = 0; u < SOME; u++)
            if (mine >> u & 1u) {
                if (at < TOP_CAND) ts.chunks[at] = c[u];
                at++;
            }
    }
    __syncthreads();
    const uint32_t n_chunks = min(ts.n_chunks, (uint32_t)TOP_CAND);
    for (uint32_t i0 = tid - lane; i0 < n_chunks; i0 += THREADS) {
        const uint32_t c = i0 + lane < n_chunks ? ts.chunks[i0 + lane] : R.chunks;
        uint32_t key[E], mine = 0;
        if (c < R.chunks) {
            f2 v[E / 2];
            unpack<T>(*reinterpret_cast<const uint4 *>(body + (size_t)c * E), v);
#pragma unroll
            for (int e = 0; e < E; e++) {
                key[e] = order_key(e & 1 ? v[e / 2].y : v[e / 2].x);
                if (key[e] >= floor_key) mine |= 1u << e;
            }
        }
        uint32_t at = place(&ts.n, __popc(mine));
#pragma unroll
        for (int e = 0; e < E; e++)
            if (mine >> e & 1u) {
                if (at < TOP_CAND) ts.cand[at] = (unsigned long long)key[e] << 32 | (uint32_t)~(R.lead + c * E + e);
                at++;
            }
    }
    if (edge >= 0 && !each && order_key(v_edge) >= floor_key) {
        const uint32_t at = atomicAdd(&ts.n, 1u);
        if (at < TOP_CAND) ts.cand[at] = (unsigned long long)order_key(v_edge) << 32 | (uint32_t)~edge;
    }
    __syncthreads();
    uint32_t n = ts.n;
    if (ts.n_chunks > TOP_CAND) n = TOP_CAND + 1;   // (too many: as with too many logits)
    if (exact && n < top) {
        // the rest are ties at lo: the lowest ids that have it, in order
        for (uint32_t j0 = 0; n < top && j0 < vocab; j0 += THREADS) {
            const uint32_t j = j0 + tid;
            const bool is = j < vocab && order_key(to_f(R.x[j])) == lo;
            const uint32_t who = __ballot_sync(~0u, is);
            if (lane == 0) ts.warp[turn][warp] = __popc(who);
            __syncthreads();
            uint32_t at = n + __popc(who & ((1u << lane) - 1u));
            for (uint32_t i = 0; i < WARPS; i++) {
                if (i < warp) at += ts.warp[turn][i];
                n += ts.warp[turn][i];
            }
            turn ^= 1u;
            if (is && at < TOP_CAND) ts.cand[at] = (unsigned long long)lo << 32 | (uint32_t)~j;
        }
        n = min(n, (uint32_t)TOP_CAND);
        __syncthreads();
    } else if (n > TOP_CAND || n < top) {
        select_whole_row(R.x, vocab, top, ts);
        n = top;
    }

    // sort by (key, lower id): runs of 64 in a warp's registers, two a lane
    const uint32_t runs = (n + 63) / 64;
    for (uint32_t i = n + tid; i < runs * 64; i += THREADS) ts.cand[i] = 0ull;
    __syncthreads();
    for (uint32_t r = warp; r < runs; r += WARPS) {
        unsigned long long a = ts.cand[r * 64 + lane], b = ts.cand[r * 64 + 32 + lane];   // elements lane, lane + 32
#pragma unroll
        for (uint32_t size = 2; size <= 64; size <<= 1)
#pragma unroll
            for (uint32_t stride = size >> 1; stride; stride >>= 1) {
                if (stride == 32) {
                    if (a < b) {
                        const unsigned long long t = a;
                        a = b;
                        b = t;
                    }
                } else {
                    const unsigned long long pa = __shfl_xor_sync(~0u, a, stride), pb = __shfl_xor_sync(~0u, b, stride);
                    const bool low = (lane & stride) == 0;
                    // falling where (index & size) == 0; for size 32 that parts a from b, for 64 all fall
                    const bool fa = size >= 32 || (lane & size) == 0, fb = size == 64 || (size < 32 && (lane & size) == 0);
                    a = (low == fa) == (a > pa) ? a : pa;
                    b = (low == fb) == (b > pb) ? b : pb;
                }
            }
        ts.cand[r * 64 + lane] = a;
        ts.cand[r * 64 + 32 + lane] = b;
    }
    __syncthreads();
    // an element's rank: its place in its run and, by binary search, the larger elements of the others
    for (uint32_t i = tid; i < n; i += THREADS) {
        const unsigned long long c = ts.cand[i];
        uint32_t rank = i & 63;
        for (uint32_t r = 0; r < runs; r += 4) {
            uint32_t m[4] = {};
#pragma unroll
            for (uint32_t h = 32; h; h >>= 1)
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (r + u < runs && ts.cand[(r + u) * 64 + m[u] + h - 1] > c) m[u] += h;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (r + u >= runs || r + u == i >> 6) continue;
                rank += m[u] + (m[u] == 63 && ts.cand[(r + u) * 64 + 63] > c);
            }
        }
        if (rank < top) {
            P.values[(size_t)row * top + rank] = capped<CAP>(key_value((uint32_t)(c >> 32)), sc) * P.out_scale;
            P.ids[(size_t)row * top + rank] = (int32_t)~(uint32_t)c;
        }
    }
}

// ---------------------------------------------------------------------------
// One pass over the rows without a gradient: log-probability and entropy of
// the rows' tokens, or (TOP) the rows' lse and the largest logit of each
// 128-byte tile, from which CTA 0 of the row then selects.  Bound by HBM reads,
// so many small CTAs with their loads under way at once; few rows are split
// over clusters of CTAs.  Measured: 1792 rows of 151936 bf16 94 us, 89 % of
// the copy bandwidth (the persistent form of the losses' kernel took 129: one
// CTA an SM has too few warps for a pass that only reads); 256 x 128256 f32
// 27 us, 74 %, two waves of CTAs with their start and end.  Three or five CTAs
// an SM: 97 and 95 us.
constexpr int BATCH = 8;             // 16-byte loads of a thread under way before the first is used
struct StreamShared {
    Stat warp[WARPS], cta[8];
};
template <typename T, bool CAP, bool TOP>
__global__ void __launch_bounds__(THREADS, 4) k_stream(RowArgs A, TopArgs P) {
    constexpr int E = Row<T>::E;
    extern __shared__ __align__(16) uint32_t keys[];
    __shared__ __align__(16) StreamShared sh;
    const uint32_t ranks = 1u << A.log_ranks, rank = ranks > 1 ? cluster_rank() : 0u;
    const uint32_t row = blockIdx.x >> A.log_ranks, tid = threadIdx.x, lane = tid & 31;
    const float k = A.sc.k;
    Row<T> R(A.x, A.ld, row, A.vocab);
    if (ranks > 1) cluster_arrive();             // (waited for before the first remote store)
    const int32_t tok = TOP ? 0 : A.tokens[row];
    if ((uint32_t)tok >= A.vocab) {              // left out: not read
        if (rank == 0 && tid == 0) {
            A.logprobs[row] = 0.0f;
            if (A.entropy) A.entropy[row] = 0.0f;
            if (A.stats) A.stats[row] = make_float2(0.0f, 0.0f);
        }
        if (ranks > 1) cluster_wait();
        return;
    }
    // slices of whole tiles; rank 0 also has the single elements
    const uint32_t tiles = (R.chunks + TOP_TILE - 1) / TOP_TILE;
    const uint32_t per = ((tiles + ranks - 1) >> A.log_ranks) * TOP_TILE;
    const uint32_t c0 = min(rank * per, R.chunks), c1 = min(c0 + per, R.chunks);
    const int32_t edge = rank == 0 && tid < 32 ? R.edge(tid) : -1;
    const T *body = R.at(0);
    const float v_edge = edge >= 0 ? to_f(R.x[edge]) : -INFINITY;
    const T v_tok = !TOP && rank == 0 && tid == 0 ? R.x[tok] : from_f<T>(0.0f);
    float *tile_max = TOP ? P.maxima + (size_t)row * P.max_ld : nullptr;
    Gather<T, CAP, !TOP> G;

    // whole batches of the CTA, so that a warp's lanes stay together
    for (uint32_t b = c0; b < c1; b += BATCH * THREADS) {
        uint4 q[BATCH];
        if (b + BATCH * THREADS <= c1) {
#pragma unroll
            for (int u = 0; u < BATCH; u++) q[u] = ld_stream(body + (size_t)(b + u * THREADS + tid) * E);
            if (!TOP) {
                G.raise(capped<CAP>(max_of<T>(q), A.sc), k);
#pragma unroll
                for (int u = 0; u < BATCH; u++) {
                    G.chunk(q[u], A.sc);
                    if (u == BATCH / 2 - 1) G.step();
                }
                G.step();
                continue;
            }
        } else {
#pragma unroll
            for (int u = 0; u < BATCH; u++)
                if (b + u * THREADS + tid < c1) q[u] = ld_stream(body + (size_t)(b + u * THREADS + tid) * E);
        }
        float mx[BATCH], big = -INFINITY;
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            mx[u] = b + u * THREADS + tid < c1 ? max_of<T>(q[u]) : -INFINITY;
            big = fmaxf(big, mx[u]);
        }
        G.raise(capped<CAP>(big, A.sc), k);
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            if (b + u * THREADS + tid < c1) G.chunk(q[u], A.sc);
            if (u == BATCH / 2 - 1) G.step();
        }
        G.step();
        if (TOP) {
            // 8 x 8 transposing maximum: lane l of an 8-lane group ends up with
            // the maximum of batch step l & 7 over the group, one tile
            static_assert(BATCH == 8 && TOP_TILE == 8, "one tile per lane and batch");
#pragma unroll
            for (int o = 4; o; o >>= 1) {
#pragma unroll
                for (int u = 0; u < o; u++) {
                    const bool up = lane & o;
                    const float keep = up ? mx[u + o] : mx[u], give = up ? mx[u] : mx[u + o];
                    mx[u] = fmaxf(keep, __shfl_xor_sync(~0u, give, o));
                }
            }
            const uint32_t first = b + (lane & 7) * THREADS + (tid & ~7u);   // the tile's first chunk
            if (first < c1) tile_max[first / TOP_TILE] = mx[0];
        }
    }
    if (edge >= 0) G.one(capped<CAP>(v_edge, A.sc), k);
    if (TOP && rank == 0 && tid < 32) {          // the single elements as one more tile
        float m = v_edge;
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        if (tid == 0) tile_max[tiles] = m;
    }
    Stat st = fold_lanes<!TOP, 32>(G.stat(), k);
    if (lane == 0) sh.warp[tid >> 5] = st;
    __syncthreads();
    if (tid < 32) {
        st = lane < WARPS ? sh.warp[lane] : Stat{0.0, -INFINITY, 0.0f};
        st = fold_lanes<!TOP, 32>(st, k);
    }
    if (ranks > 1) {
        cluster_wait();
        if (tid == 0) st_remote(remote(&sh.cta[rank], 0), st);
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (tid < 32) {
            st = fold_lanes<!TOP, 32>(lane < ranks ? sh.cta[lane] : Stat{0.0, -INFINITY, 0.0f}, k);
        }
    }
    if (rank != 0) return;
    if constexpr (TOP) {
        // (the barriers above also made the tile maxima of all CTAs visible to this one)
        __shared__ TopShared ts;
        if (tid == 0) P.lse[row] = (float)((double)st.m * A.sc.md + log(st.s));
        if (P.fused) select_top<T, CAP>(R, row, A.sc, P, ts, keys);
    } else if (tid == 0) {
        token_row<OP_LOGPROB>(A, row, st, TokenIn{1.0f, 0.0f, 0.0f, 0.0f, capped<CAP>(to_f(v_tok), A.sc), 1.0f}, true);
    }
}

template <typename T, bool CAP> __global__ void __launch_bounds__(THREADS) k_select(RowArgs A, TopArgs P) {
    extern __shared__ __align__(16) uint32_t keys[];
    __shared__ TopShared ts;
    const Row<T> R(A.x, A.ld, blockIdx.x, A.vocab);
    asm volatile("griddepcontrol.wait;" ::: "memory");   // k_stream is done
    select_top<T, CAP>(R, blockIdx.x, A.sc, P, ts, keys);
}

// ---------------------------------------------------------------------------
// Host side

static bs_status launched(const char *what) {
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return BS_OK;
    fprintf(stderr, "b200_sampler: %s: launch failed: %s\n", what, cudaGetErrorString(e));
    return BS_ECUDA;
}

static size_t elem_size(uint32_t dtype) { return dtype == BS_F32 ? 4 : 2; }

// Checks a descriptor and works out its factors.
static bs_status check_logits(const bs_logits *x, Scale *sc, float *out_scale, bool *cap) {
    if (!x || (!x->data && x->rows) || x->vocab == 0 || x->ld < x->vocab || x->dtype > BS_F16) return BS_EINVAL;
    if (x->vocab > BS_MAX_VOCAB || (uintptr_t)x->data % elem_size(x->dtype)) return BS_EINVAL;
    if (x->rows > 0x7FFFFFFFu) return BS_EINVAL;
    if (!(x->temperature > 0.0f) || std::isinf(x->temperature)) return BS_EINVAL;
    if (std::isnan(x->final_logit_softcapping) || std::isinf(x->final_logit_softcapping)) return BS_EINVAL;
    if (!(x->logit_scale >= 0.0f) || std::isinf(x->logit_scale)) return BS_EINVAL;
    const double scale = x->logit_scale == 0.0f ? 1.0 : (double)x->logit_scale;   // 0: off, as in the sampler
    const double m = 1.0 / (scale * (double)x->temperature);
    const double k = m * 1.4426950408889634;
    if (!(k >= 1.2e-38) || !(k <= 3.0e38)) return BS_EINVAL;
    sc->m = (float)m;
    sc->md = m;
    sc->k = (float)k;
    sc->dk = k / (double)sc->k - 1.0;
    sc->inv_t = 1.0 / (double)x->temperature;
    *cap = x->final_logit_softcapping > 0.0f;
    sc->cap = *cap ? x->final_logit_softcapping : 1.0f;
    // (a cap below 2^-126 has reciprocals past f32)
    sc->icap = (float)fmin(1.0 / (double)sc->cap, 3.4e38);
    const double k2 = fmax(-2.0 * 1.4426950408889634 / (double)sc->cap, -3.4e38);
    sc->k2 = (float)k2;
    sc->k2_lo = (float)(k2 - (double)sc->k2);
    sc->most = (float)fmin(fmax(64.0 * (double)sc->cap, 6e-37), 3.4e38);   // (2^(most k2) is 0)
    *out_scale = (float)(1.0 / scale);
    return BS_OK;
}

static bs_status check_grad(const bs_logits *x, const void *grad, size_t ld_grad) {
    if (grad && (ld_grad < x->vocab || (uintptr_t)grad % elem_size(x->dtype))) return BS_EINVAL;
    return BS_OK;
}

constexpr int MAX_DEVICES = 64;
constexpr int SMEM_MAX = 227 * 1024;

// What a kernel needs to know of a device, found out by the first launch there
// (twice does no harm).
struct DeviceInfo {
    std::atomic<int> sms{0};
    std::atomic<int> clusters[5] = {};   // clusters of 1, 2, 4, 8, 16 CTAs that run at once
    std::atomic<bool> ready{false};
};

template <auto K, typename... Q>
static cudaError_t launch_clusters(uint32_t grid, uint32_t ranks, uint32_t threads, size_t smem, cudaStream_t st, Q... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, K, args...);
}

// A launch that may overlap the end of the stream's previous kernel (the kernel
// waits for that one before it reads its results).
template <auto K, typename... Q>
static cudaError_t launch_after(uint32_t grid, uint32_t threads, size_t smem, cudaStream_t st, Q... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, K, args...);
}

// The current device's entry of kernel K's table, with K allowed all of an
// SM's shared memory (per device, as kernel attributes are) and, if `wide`,
// clusters of 16.
template <auto K> static cudaError_t device_info(DeviceInfo **out, bool wide) {
    static DeviceInfo table[MAX_DEVICES];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= MAX_DEVICES) return cudaErrorInvalidDevice;
    DeviceInfo &d = table[dev];
    if (!d.ready.load(std::memory_order_acquire)) {
        cudaFuncAttributes fa;
        int sms = 0;
        e = cudaFuncGetAttributes(&fa, K);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX - (int)fa.sharedSizeBytes);
        if (e == cudaSuccess && wide) e = cudaFuncSetAttribute(K, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return e;
        d.sms.store(sms);
        d.ready.store(true, std::memory_order_release);
    }
    *out = &d;
    return cudaSuccess;
}

static bs_status failed(const char *what, cudaError_t e) {
    cudaGetLastError();
    fprintf(stderr, "b200_sampler: %s: launch failed: %s\n", what, cudaGetErrorString(e));
    return BS_ECUDA;
}

constexpr uint32_t STREAM_CTAS = 148 * 4;   // of k_stream that run at once

// CTAs per row of k_stream: few rows still fill the GPU (four to an SM), no CTA
// has less than two chunks a thread.  Measured, split against one CTA a row:
// 1 x 128256 f32 6.2 and 12.8 us (the first is the launch), 64 rows 11.1 and
// 20.6; at 256 rows it no longer matters (27.2 and 26.7).
static uint32_t stream_log_ranks(uint32_t rows, uint32_t chunks) {
    uint32_t l = 0;
    while (l < 3 && ((uint64_t)rows << l) < STREAM_CTAS && (chunks >> (l + 1)) >= 2 * THREADS) l++;
    return l;
}

// Whether k_stream itself selects.  With many rows (one CTA each) that overlaps
// other rows' streaming, with few it saves a launch; in between all rows would
// select at the kernel's end, several to an SM.  Measured, separate against
// fused: 8 x 128256 f32 16.3 and 14.5 us, 256 rows 37.9 and 44.6, 2048 rows
// 217 and 210; 512 x 32000 bf16 24.7 and 30.9, 4096 rows 115 and 111.
static bool top_fused(uint32_t rows) { return rows < 64 || rows >= STREAM_CTAS; }

template <typename T, bool CAP, bool TOP>
static bs_status launch_stream(const char *what, RowArgs A, uint32_t rows, TopArgs P, cudaStream_t st) {
    constexpr auto K = k_stream<T, CAP, TOP>;
    DeviceInfo *dev;
    cudaError_t e = device_info<K>(&dev, false);
    size_t smem = 0;
    A.log_ranks = stream_log_ranks(rows, A.vocab / (16 / sizeof(T)));
    if (TOP) {
        // The logits themselves where the tiles are few and all keys fit (the tiles would let through more logits than
        // can be sorted): top 256 of 512 x 8000 bf16 34.8 us, by tiles 75.5; top 1000 of 64 x 32000 f32 63 and 161.
        P.each = A.vocab <= TOP_EACH && P.max_ld < P.top + P.top / 2;
        P.fused = top_fused(rows);
        smem = (size_t)(((P.each ? A.vocab : P.max_ld) + 3) & ~3u) * 4;
    }
    if (((uint64_t)rows << A.log_ranks) > 0x7FFFFFFFull) return BS_EINVAL;
    if (e == cudaSuccess)
        e = launch_clusters<K>(rows << A.log_ranks, 1u << A.log_ranks, THREADS, P.fused ? smem : 0, st, A, P);
    if constexpr (TOP) {
        constexpr auto S = k_select<T, CAP>;
        if (e == cudaSuccess && !P.fused) e = device_info<S>(&dev, false);
        if (e == cudaSuccess && !P.fused) e = launch_after<S>(rows, THREADS, smem, st, A, P);   // (its launch overlaps k_stream's end)
    }
    return e == cudaSuccess ? BS_OK : failed(what, e);
}
template <bool TOP>
static bs_status launch_stream_typed(const char *what, const bs_logits *x, const RowArgs &A, bool cap, const TopArgs &P,
                                     cudaStream_t st) {
    switch (x->dtype) {
        case BS_F32:
            return cap ? launch_stream<float, true, TOP>(what, A, x->rows, P, st)
                       : launch_stream<float, false, TOP>(what, A, x->rows, P, st);
        case BS_BF16:
            return cap ? launch_stream<__nv_bfloat16, true, TOP>(what, A, x->rows, P, st)
                       : launch_stream<__nv_bfloat16, false, TOP>(what, A, x->rows, P, st);
        default:
            return cap ? launch_stream<__half, true, TOP>(what, A, x->rows, P, st)
                       : launch_stream<__half, false, TOP>(what, A, x->rows, P, st);
    }
}

// Shared memory of k_rows: three buffers of a slice, the teacher's slots.
constexpr size_t ROWS_SMEM = SMEM_MAX - sizeof(RowsShared) - 256;
// No row is split into slices below this many chunks for the sake of more SMs
// (8 x 128256 bf16 10.3 us with eight CTAs a row, 12.2 with four).
constexpr uint32_t SLICE_MIN = 1024;

template <typename T, int OP, bool CAP>
static bs_status launch_row(RowArgs A, uint32_t rows, cudaStream_t st) {
    constexpr auto K = k_rows<T, OP, CAP>;
    constexpr uint32_t E = 16 / sizeof(T);
    DeviceInfo *dev;
    cudaError_t e = device_info<K>(&dev, true);
    if (e != cudaSuccess) return failed("logit_ops", e);
    const uint32_t chunks = A.vocab / E;
    uint32_t ranks = 1, log_ranks = 0, slice = 0;
    size_t slots = 0, room = 0;
    for (;; ranks *= 2, log_ranks++) {
        slice = (chunks + ranks - 1) / ranks;
        A.bit_words = is_distill(OP) ? (slice * E + 31) / 32 : 0;
        slots = is_distill(OP) ? (size_t)slots_padded(A.n_ids) * 16 * slot_words<CAP>() + (size_t)A.bit_words * 16 : 0;
        room = slots < ROWS_SMEM ? (ROWS_SMEM - slots) / 48 : 0;
        // Enough CTAs to hold the row, and to use the GPU where the rows are few.  Sixteen only where eight cannot
        // hold it (seven such clusters fit the GPU, 112 SMs): 512 x 256000 f32 424 us, with eight and the rest of
        // the slices read again from L2 495.
        if (ranks == MAX_CLUSTER ||
            (slice <= room && !(ranks < 8 && (uint64_t)rows * ranks * 2 <= (uint64_t)dev->sms.load() && slice / 2 >= SLICE_MIN)))
            break;
    }
    if (slots >= ROWS_SMEM) return BS_ENOTSUP;
    A.keep = slice < room ? slice : (uint32_t)room;
    A.log_ranks = log_ranks;
    // one CTA per SM: all of its shared memory is asked for
    int most = dev->clusters[log_ranks].load(std::memory_order_relaxed);
    if (most == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ranks);
        cfg.blockDim = dim3(row_threads(OP, compute_threads<T>()));
        cfg.dynamicSmemBytes = ROWS_SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ranks;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&most, K, &cfg);
        if (e == cudaSuccess && most <= 0) e = cudaErrorInvalidConfiguration;
        if (e != cudaSuccess) return failed("logit_ops", e);
        dev->clusters[log_ranks].store(most, std::memory_order_relaxed);
    }
    const uint32_t clusters = rows < (uint32_t)most ? rows : (uint32_t)most;
    e = launch_clusters<K>(clusters * ranks, ranks, row_threads(OP, compute_threads<T>()), ROWS_SMEM, st, A, rows, clusters);
    return e == cudaSuccess ? BS_OK : failed("logit_ops", e);
}

template <int OP>
static bs_status launch_row_typed(const bs_logits *x, const RowArgs &A, bool cap, cudaStream_t st) {
    switch (x->dtype) {
        case BS_F32: return cap ? launch_row<float, OP, true>(A, x->rows, st) : launch_row<float, OP, false>(A, x->rows, st);
        case BS_BF16:
            return cap ? launch_row<__nv_bfloat16, OP, true>(A, x->rows, st)
                       : launch_row<__nv_bfloat16, OP, false>(A, x->rows, st);
        default: return cap ? launch_row<__half, OP, true>(A, x->rows, st) : launch_row<__half, OP, false>(A, x->rows, st);
    }
}

static std::atomic<long long> wait_limit{WAIT_LIMIT};
static std::atomic<uint32_t> gone_rank{0xFFFFFFFFu}, gone_row{0};

static RowArgs row_args(const bs_logits *x, const Scale &sc) {
    RowArgs A = {};
    A.wait_limit = wait_limit.load(std::memory_order_relaxed);
    A.gone_rank = gone_rank.load(std::memory_order_relaxed);
    A.gone_row = gone_row.load(std::memory_order_relaxed);
    A.x = x->data;
    A.ld = x->ld;
    A.vocab = x->vocab;
    A.sc = sc;
    A.w_all = x->rows ? 1.0f / (float)x->rows : 0.0f;
    return A;
}

static bs_status total_loss(const RowArgs &A, uint32_t rows, float *loss, cudaStream_t st) {
    cudaError_t e = launch_after<k_loss>(1, 1024, 0, st, (const float *)A.row_loss, A.weights, A.w_all, rows, loss);
    return e == cudaSuccess ? BS_OK : failed("logit_ops loss", e);
}

static bs_status no_rows(float *d_loss, void *stream) {
    if (cudaMemsetAsync(d_loss, 0, sizeof(float), (cudaStream_t)stream) != cudaSuccess) {
        cudaGetLastError();
        return BS_ECUDA;
    }
    return BS_OK;
}

}  // namespace ops
}  // namespace bs

using namespace bs::ops;

extern "C" bs_status bs_logit_ops_status(void) {
    uint32_t gave_up = 0;
    const uint32_t zero = 0;
    if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyFromSymbol(&gave_up, wait_gave_up, sizeof(gave_up)) != cudaSuccess ||
        (gave_up && cudaMemcpyToSymbol(wait_gave_up, &zero, sizeof(zero)) != cudaSuccess)) {
        cudaGetLastError();
        return BS_ECUDA;
    }
    return gave_up ? BS_ETIMEOUT : BS_OK;
}

// For tests of what follows a wait that gives up: the waits' limit in clock
// cycles (0: as it is without this call), and a CTA of the clusters whose waits
// give up at once from its row-th row on (rank 0xFFFFFFFF: none).
extern "C" void bs_debug_logit_ops_waits(uint64_t cycles, uint32_t rank, uint32_t row) {
    wait_limit.store(cycles && cycles < (uint64_t)WAIT_LIMIT ? (long long)cycles : WAIT_LIMIT);
    gone_rank.store(rank);
    gone_row.store(row);
}

extern "C" bs_status bs_token_logprobs(const bs_logits *x, const int32_t *d_tokens, float *d_logprobs, float *d_entropy,
                                       float *d_stats, void *stream) {
    Scale sc;
    float os;
    bool cap;
    bs_status st = check_logits(x, &sc, &os, &cap);
    if (st != BS_OK) return st;
    if (x->rows == 0) return BS_OK;
    if (!d_tokens || !d_logprobs || (uintptr_t)d_stats % 8) return BS_EINVAL;
    RowArgs A = row_args(x, sc);
    A.tokens = d_tokens;
    A.logprobs = d_logprobs;
    A.entropy = d_entropy;
    A.stats = (float2 *)d_stats;
    return launch_stream_typed<false>("bs_token_logprobs", x, A, cap, TopArgs{}, (cudaStream_t)stream);
}

template <typename T>
static bs_status launch_logprob_grad(const RowArgs &A, uint32_t rows, bool cap, const float2 *stats, const float *d_lp,
                                     const float *d_ent, const float *entropy, cudaStream_t st) {
    auto kern = cap ? (d_ent ? k_logprob_grad<T, true, true> : k_logprob_grad<T, true, false>)
                    : (d_ent ? k_logprob_grad<T, false, true> : k_logprob_grad<T, false, false>);
    const uint32_t chunks = A.vocab / (16 / sizeof(T));
    const uint32_t slices = chunks ? (chunks + GRAD_SLICE - 1) / GRAD_SLICE : 1;
    if ((uint64_t)rows * slices > 0x7FFFFFFFull) return BS_EINVAL;
    kern<<<rows * slices, THREADS, 0, st>>>(A, slices, stats, d_lp, d_ent, entropy);
    return launched("bs_token_logprobs_grad");
}

extern "C" bs_status bs_token_logprobs_grad(const bs_logits *x, const int32_t *d_tokens, const float *d_stats,
                                            const float *d_entropy, const float *d_grad_logprobs,
                                            const float *d_grad_entropy, void *d_grad, size_t ld_grad, void *stream) {
    Scale sc;
    float os;
    bool cap;
    bs_status st = check_logits(x, &sc, &os, &cap);
    if (st != BS_OK) return st;
    if (x->rows == 0) return BS_OK;
    if (!d_tokens || !d_stats || (uintptr_t)d_stats % 8 || !d_grad || (!d_grad_logprobs && !d_grad_entropy) ||
        (d_grad_entropy && !d_entropy))
        return BS_EINVAL;
    st = check_grad(x, d_grad, ld_grad);
    if (st != BS_OK) return st;
    RowArgs A = row_args(x, sc);
    A.tokens = d_tokens;
    A.grad = d_grad;
    A.ld_grad = ld_grad;
    const float2 *stats = (const float2 *)d_stats;
    cudaStream_t s = (cudaStream_t)stream;
    switch (x->dtype) {
        case BS_F32:
            return launch_logprob_grad<float>(A, x->rows, cap, stats, d_grad_logprobs, d_grad_entropy, d_entropy, s);
        case BS_BF16:
            return launch_logprob_grad<__nv_bfloat16>(A, x->rows, cap, stats, d_grad_logprobs, d_grad_entropy, d_entropy, s);
        default:
            return launch_logprob_grad<__half>(A, x->rows, cap, stats, d_grad_logprobs, d_grad_entropy, d_entropy, s);
    }
}

extern "C" bs_status bs_policy_loss(const bs_logits *x, const int32_t *d_tokens, const float *d_old_logprobs,
                                    const float *d_advantages, const float *d_ref_logprobs, const float *d_weights,
                                    const bs_policy_config *cfg, float *d_loss, float *d_row_loss, float *d_logprobs,
                                    float *d_entropy, float *d_kl, void *d_grad, size_t ld_grad, void *stream) {
    Scale sc;
    float os;
    bool cap;
    bs_status st = check_logits(x, &sc, &os, &cap);
    if (st != BS_OK) return st;
    if (!cfg || !d_loss) return BS_EINVAL;
    if (!(cfg->clip_low >= 0.0f) || !(cfg->clip_high >= 0.0f) || !std::isfinite(cfg->kl_coef) ||
        !std::isfinite(cfg->entropy_coef))
        return BS_EINVAL;
    if (x->rows == 0) return no_rows(d_loss, stream);
    if (!d_tokens || !d_old_logprobs || !d_advantages || !d_row_loss) return BS_EINVAL;
    if (cfg->kl_coef != 0.0f && !d_ref_logprobs) return BS_EINVAL;
    st = check_grad(x, d_grad, ld_grad);
    if (st != BS_OK) return st;
    RowArgs A = row_args(x, sc);
    A.tokens = d_tokens;
    A.old_lp = d_old_logprobs;
    A.adv = d_advantages;
    A.ref_lp = d_ref_logprobs;
    A.weights = d_weights;
    A.clip_lo = 1.0 - (double)cfg->clip_low;
    A.clip_hi = 1.0 + (double)cfg->clip_high;
    A.kl_coef = cfg->kl_coef;
    A.ent_coef = cfg->entropy_coef;
    A.row_loss = d_row_loss;
    A.logprobs = d_logprobs;
    A.entropy = d_entropy;
    A.kl = d_kl;
    A.grad = d_grad;
    A.ld_grad = ld_grad;
    cudaStream_t s = (cudaStream_t)stream;
    st = cfg->entropy_coef != 0.0f ? launch_row_typed<OP_POLICY_ENT>(x, A, cap, s)
                                   : launch_row_typed<OP_POLICY>(x, A, cap, s);
    return st != BS_OK ? st : total_loss(A, x->rows, d_loss, s);
}

extern "C" bs_status bs_distill_loss(const bs_logits *x, const int32_t *d_teacher_ids, const float *d_teacher_logits,
                                     const float *d_teacher_lse, uint32_t n_ids, const float *d_weights, float *d_loss,
                                     float *d_row_loss, void *d_grad, size_t ld_grad, void *stream) {
    Scale sc;
    float os;
    bool cap;
    bs_status st = check_logits(x, &sc, &os, &cap);
    if (st != BS_OK) return st;
    if (!d_loss || n_ids == 0) return BS_EINVAL;
    if (n_ids > BS_MAX_TOP) return BS_ENOTSUP;
    if (x->rows == 0) return no_rows(d_loss, stream);
    if (!d_teacher_ids || !d_teacher_logits || !d_row_loss) return BS_EINVAL;
    st = check_grad(x, d_grad, ld_grad);
    if (st != BS_OK) return st;
    RowArgs A = row_args(x, sc);
    A.t_ids = d_teacher_ids;
    A.t_logits = d_teacher_logits;
    A.t_lse = d_teacher_lse;
    A.n_ids = n_ids;
    A.weights = d_weights;
    A.row_loss = d_row_loss;
    A.grad = d_grad;
    A.ld_grad = ld_grad;
    cudaStream_t s = (cudaStream_t)stream;
    st = d_teacher_lse ? launch_row_typed<OP_DISTILL_TAIL>(x, A, cap, s)
                       : launch_row_typed<OP_DISTILL>(x, A, cap, s);
    return st != BS_OK ? st : total_loss(A, x->rows, d_loss, s);
}

// Floats of tile maxima per row: the body's tiles and one more.
// (a multiple of 4: rows of 16-byte loads)
static uint32_t top_tiles(const bs_logits *x) {
    return (x->vocab / (16 / (uint32_t)elem_size(x->dtype)) / TOP_TILE + 2 + 3) & ~3u;
}

extern "C" size_t bs_top_logits_workspace(const bs_logits *x) {
    if (!x || x->dtype > BS_F16 || x->vocab > BS_MAX_VOCAB) return 0;
    return (size_t)x->rows * top_tiles(x) * 4;
}

extern "C" bs_status bs_top_logits(const bs_logits *x, uint32_t k, float *d_values, int32_t *d_ids, float *d_lse,
                                   void *d_work, size_t work_bytes, void *stream) {
    Scale sc;
    float os;
    bool cap;
    bs_status st = check_logits(x, &sc, &os, &cap);
    if (st != BS_OK) return st;
    if (k == 0 || k > x->vocab) return BS_EINVAL;
    if (k > BS_MAX_TOP) return BS_ENOTSUP;
    if (x->rows == 0) return BS_OK;
    if (!d_values || !d_ids || !d_lse || !d_work || (uintptr_t)d_work % 16 || work_bytes < bs_top_logits_workspace(x))
        return BS_EINVAL;
    const TopArgs P{k, os, false, false, d_values, d_ids, d_lse, (float *)d_work, top_tiles(x)};
    return launch_stream_typed<true>("bs_top_logits", x, row_args(x, sc), cap, P, (cudaStream_t)stream);
}
