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

#include <cmath>
#include <cstdint>
#include <cstdio>

#include "b200_sampler.h"

namespace bs {
namespace ops {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_K = 1024;          // most teacher ids of a row, most top logits
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
    double inv_t;    // 1 / T
};

struct RowArgs {
    const void *x;
    size_t ld;
    uint32_t vocab;
    Scale sc;
    const int32_t *tokens;
    // outputs (null where not asked for)
    float *logprobs, *entropy, *kl, *row_loss;
    float2 *stats;
    void *grad;
    size_t ld_grad;
    // losses
    const float *weights;       // null: 1 / rows each
    float w_all;
    const float *old_lp, *adv, *ref_lp;
    float clip_lo, clip_hi, kl_coef, ent_coef;
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

// c(v) and its slope 1 - (c / cap)^2.
template <bool CAP> __device__ __forceinline__ float capped(float v, const Scale &sc) {
    return CAP ? sc.cap * tanhf(v * sc.icap) : v;
}
template <bool CAP> __device__ __forceinline__ float slope(float c, const Scale &sc) {
    if (!CAP) return 1.0f;
    float t = c * sc.icap;
    return fmaf(-t, t, 1.0f);
}

// A row as 16-byte chunks of its memory.  The row may start anywhere, so
// chunk 0 begins up to 15 bytes before it and the last one may end behind it;
// `head` is the number of elements before the row in chunk 0.
template <typename T> struct Row {
    static constexpr int E = 16 / sizeof(T);
    const T *x;          // element 0
    uint32_t head, vocab, chunks;
    __device__ Row(const void *base, size_t ld, uint32_t row, uint32_t v) {
        x = (const T *)base + (size_t)row * ld;
        head = (uint32_t)(((uintptr_t)x & 15u) / sizeof(T));
        vocab = v;
        chunks = (uint32_t)(((uint64_t)head + v + E - 1) / E);
    }
    __device__ int64_t first(uint32_t c) const { return (int64_t)c * E - head; }
    __device__ bool whole(uint32_t c) const { return first(c) >= 0 && first(c) + E <= (int64_t)vocab; }
    // the chunk's logits after the soft-cap; -inf outside the row
    template <bool CAP> __device__ void load(uint32_t c, const Scale &sc, float (&v)[E]) const {
        int64_t j0 = first(c);
        if (whole(c)) {
            uint4 q = *reinterpret_cast<const uint4 *>(x + j0);
            const T *e = reinterpret_cast<const T *>(&q);
#pragma unroll
            for (int i = 0; i < E; i++) v[i] = capped<CAP>(to_f(e[i]), sc);
        } else {
#pragma unroll
            for (int i = 0; i < E; i++) {
                int64_t j = j0 + i;
                v[i] = j >= 0 && j < (int64_t)vocab ? capped<CAP>(to_f(x[j]), sc) : -INFINITY;
            }
        }
    }
};

// Running (M, S, U) of a set of logits.
struct Stat {
    float m, s, u;
};
__device__ __forceinline__ void rebase(Stat &a, float m, float k) {
    // factor 2^((a.m - m) k); fmaxf also turns -inf - -inf into "nothing there"
    float d = fmaxf((a.m - m) * k, D_MIN);
    float f = ex2(d);
    a.u = f * fmaf(d, a.s, a.u);
    a.s *= f;
    a.m = m;
}
// A maximum of -inf (all of the set masked) is replaced by 0 in differences,
// so that the masked logits give 2^-inf = 0.
__device__ __forceinline__ float anchor(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ __forceinline__ Stat merge(Stat a, const Stat &b, float k) {
    float m = fmaxf(a.m, b.m);
    Stat c = b;
    rebase(a, m, k);
    rebase(c, m, k);
    a.s += c.s;
    a.u += c.u;
    return a;
}

// log2 S as exponent + log2 of the mantissa: exact to 2^-24 for any S.
__device__ __forceinline__ double log2_d(float s) {
    if (!(s > 0.0f) || isinf(s)) return (double)log2f(s);
    int e;
    float f = frexpf(s, &e);
    return (double)e + (double)log2f(f);
}

template <typename V> __device__ __forceinline__ V block_sum(V v, V *scratch) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    V r = 0;
    for (int w = 0; w < WARPS; w++) r += scratch[w];
    return r;
}

// One CTA per row: the row's statistics in one pass over its logits, the
// row's results, then (if asked for) the gradient in a second pass, which
// finds the row in L2.
template <typename T, int OP, bool CAP>
__global__ void __launch_bounds__(THREADS) k_row(RowArgs A) {
    constexpr bool DIST = OP == OP_DISTILL || OP == OP_DISTILL_TAIL;
    constexpr bool TAIL = OP == OP_DISTILL_TAIL;
    constexpr bool POLICY = OP == OP_POLICY || OP == OP_POLICY_ENT;
    constexpr int E = Row<T>::E;
    extern __shared__ uint32_t dyn[];
    __shared__ Stat sh_stat[WARPS];
    __shared__ float sh_f[WARPS];
    __shared__ double sh_d[WARPS];
    const uint32_t row = blockIdx.x, tid = threadIdx.x, V = A.vocab;
    const float k = A.sc.k;
    Row<T> R(A.x, A.ld, row, V);
    T *gout = A.grad ? (T *)A.grad + (size_t)row * A.ld_grad : nullptr;

    const float w = DIST || POLICY ? (A.weights ? A.weights[row] : A.w_all) : 1.0f;
    bool live = w != 0.0f;
    const int32_t tok = DIST ? -1 : A.tokens[row];
    if (!DIST) live = live && (uint32_t)tok < V;

    // the teacher's slots
    int32_t *s_id = (int32_t *)dyn;              // n_ids; -1: empty
    float *s_q = (float *)(s_id + A.n_ids);      // share q of the slot
    float *s_c = s_q + A.n_ids;                  // the student's c(v) there
    uint32_t *s_bits = (uint32_t *)(s_c + A.n_ids);  // tail: one bit per element of the row's chunks
    if (DIST && live) {
        const size_t at = (size_t)row * A.n_ids;
        float umax = -INFINITY;
        bool any = false;
        if (TAIL)
            for (uint32_t i = tid; i < (R.chunks * E + 31) / 32; i += THREADS) s_bits[i] = 0;
        for (uint32_t i = tid; i < A.n_ids; i += THREADS) {
            int32_t id = A.t_ids[at + i];
            if ((uint32_t)id >= V) id = -1;
            s_id[i] = id;
            if (id >= 0) {
                any = true;
                umax = max_nan(umax, A.t_logits[at + i]);
                s_c[i] = capped<CAP>(to_f(R.x[id]), A.sc);
            }
        }
        live = __syncthreads_or(any);
        if (live) {
            if (!TAIL) {
                for (int o = 16; o; o >>= 1) umax = max_nan(umax, __shfl_xor_sync(~0u, umax, o));
                if ((tid & 31) == 0) sh_f[tid >> 5] = umax;
                __syncthreads();
                for (int i = 0; i < WARPS; i++) umax = max_nan(umax, sh_f[i]);
                live = umax != -INFINITY;   // no share to give: as without ids
            }
        }
        if (live) {
            const double ref = TAIL ? (double)A.t_lse[row] : (double)umax * A.sc.inv_t;
            float q_sum = 0.0f;
            for (uint32_t i = tid; i < A.n_ids; i += THREADS) {
                float q = 0.0f;
                if (s_id[i] >= 0) {
                    q = expf((float)((double)A.t_logits[at + i] * A.sc.inv_t - ref));
                    if (TAIL) atomicOr(&s_bits[(R.head + s_id[i]) >> 5], 1u << ((R.head + s_id[i]) & 31));
                }
                s_q[i] = q;
                q_sum += q;
            }
            if (!TAIL) {
                const float total = (float)block_sum((double)q_sum, sh_d);
                for (uint32_t i = tid; i < A.n_ids; i += THREADS) s_q[i] /= total;
            }
            __syncthreads();
        }
    }

    if (!live) {  // the row is left out: zeros, and its logits are not read
        if (tid == 0) {
            if (A.logprobs) A.logprobs[row] = 0.0f;
            if (A.entropy) A.entropy[row] = 0.0f;
            if (A.stats) A.stats[row] = make_float2(0.0f, 0.0f);
            if (A.kl) A.kl[row] = 0.0f;
            if (A.row_loss) A.row_loss[row] = 0.0f;
        }
        if (gout)
            for (uint32_t j = tid; j < V; j += THREADS) gout[j] = from_f<T>(0.0f);
        return;
    }

    const float c_tok = DIST ? 0.0f : capped<CAP>(to_f(R.x[tok]), A.sc);

    // statistics; with a tail, s is the rest's sum and `top` that of the teacher's ids
    Stat a{-INFINITY, 0.0f, 0.0f};
    float top = 0.0f;
    for (uint32_t c = tid; c < R.chunks; c += THREADS) {
        float v[E];
        R.template load<CAP>(c, A.sc, v);
        float m = v[0];
#pragma unroll
        for (int i = 1; i < E; i++) m = fmaxf(m, v[i]);
        if (m > a.m) {
            if (TAIL) top *= ex2(fmaxf((a.m - m) * k, D_MIN));
            rebase(a, m, k);
        }
        const float base = anchor(a.m);
        uint32_t marked = 0;
        if (TAIL) marked = s_bits[(c * E) >> 5] >> ((c * E) & 31) & ((1u << E) - 1u);
#pragma unroll
        for (int i = 0; i < E; i++) {
            float d = (v[i] - base) * k;
            float e = ex2(d);
            if (TAIL && (marked >> i & 1u)) {
                top += e;
            } else {
                a.s += e;
                if (!DIST) a.u = fmaf(e, max_nan(d, D_MIN), a.u);
            }
        }
    }
    // block: the maximum first, then the sums on one scale
    float m = a.m;
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if ((tid & 31) == 0) sh_f[tid >> 5] = m;
    __syncthreads();
    for (int i = 0; i < WARPS; i++) m = fmaxf(m, sh_f[i]);
    if (TAIL) top *= ex2(fmaxf((a.m - m) * k, D_MIN));
    rebase(a, m, k);
    if (TAIL) a.u = top;
    for (int o = 16; o; o >>= 1) {
        a.s += __shfl_xor_sync(~0u, a.s, o);
        a.u += __shfl_xor_sync(~0u, a.u, o);
    }
    if ((tid & 31) == 0) sh_stat[tid >> 5] = a;
    __syncthreads();
    float s = 0.0f, u = 0.0f;
    for (int i = 0; i < WARPS; i++) {
        s += sh_stat[i].s;
        u += sh_stat[i].u;
    }
    const float rest = s;
    if (TAIL) s += u;
    const double l2s = log2_d(s);

    // the row's results and the gradient's coefficients:
    //   dv_j = c'(v_j) p_j (ca + cb log2 p_j), + c'(v_t) ct at the token
    float ca = 0.0f, cb = 0.0f, ct = 0.0f, q_all = 0.0f;
    if (!DIST) {
        const double lp = LN2_D * (((double)c_tok - (double)m) * (double)k - l2s);
        const float H = (float)(LN2_D * (l2s - (double)u / (double)s));
        float g = 0.0f, kl = 0.0f;
        if (POLICY) {
            const float adv = A.adv[row];
            const float r = expf((float)(lp - (double)A.old_lp[row]));
            // min(r A, clip(r) A) is the clipped one only beyond the bound that A favours
            const bool over = adv > 0.0f && r > A.clip_hi, under = adv < 0.0f && r < A.clip_lo;
            float loss = -adv * (over ? A.clip_hi : under ? A.clip_lo : r);
            g = over || under ? 0.0f : -r * adv;
            if (A.ref_lp) {
                const float dr = (float)((double)A.ref_lp[row] - lp);
                const float x1 = expm1f(dr);
                kl = x1 - dr;
                if (A.kl_coef != 0.0f) {
                    loss += A.kl_coef * kl;
                    g -= A.kl_coef * x1;
                }
            }
            if (OP == OP_POLICY_ENT) loss -= A.ent_coef * H;
            if (tid == 0) A.row_loss[row] = loss;
            const float wm = w * A.sc.m;
            ct = wm * g;
            ca = wm * (OP == OP_POLICY_ENT ? A.ent_coef * H - g : -g);
            cb = OP == OP_POLICY_ENT ? wm * A.ent_coef * LN2 : 0.0f;
        }
        if (tid == 0) {
            if (A.logprobs) A.logprobs[row] = (float)lp;
            if (A.entropy) A.entropy[row] = H;
            if (A.kl) A.kl[row] = kl;
            if (A.stats) A.stats[row] = make_float2(m, (float)(LN2_D * l2s));
        }
    } else {
        // sum q (log q - log p) over the slots, and the rest as one outcome
        double loss = 0.0, mass = 0.0;
        for (uint32_t i = tid; i < A.n_ids; i += THREADS) {
            const float q = s_q[i];
            if (s_id[i] >= 0 && !(q <= 0.0f)) {
                const double l2p = ((double)s_c[i] - (double)m) * (double)k - l2s;
                loss += (double)q * (log2_d(q) - l2p);
                mass += (double)q;
            }
        }
        loss = block_sum(loss, sh_d);
        mass = block_sum(mass, sh_d);
        float share = 0.0f;
        if (TAIL) {
            const float qr = mass >= 1.0 ? 0.0f : (float)(1.0 - mass);
            if (!(qr <= 0.0f) && !(rest == 0.0f)) {
                const double l2r = log2_d(rest) - l2s;
                loss += (double)qr * (log2_d(qr) - l2r);
                mass += (double)qr;
                share = (float)((double)qr * (double)s / (double)rest);
            }
        }
        if (tid == 0) A.row_loss[row] = (float)(LN2_D * loss);
        q_all = w * A.sc.m * (float)mass;
        ca = w * A.sc.m * ((float)mass - share);
    }
    if (!gout) return;

    const float l2f = (float)l2s;
    for (uint32_t c = tid; c < R.chunks; c += THREADS) {
        float v[E];
        R.template load<CAP>(c, A.sc, v);
        const int64_t j0 = R.first(c);
#pragma unroll
        for (int i = 0; i < E; i++) {
            const float lp2 = (v[i] - m) * k - l2f;
            const float p = ex2(lp2);
            float g = OP == OP_POLICY_ENT ? p * fmaf(cb, max_nan(lp2, D_MIN), ca) : p * ca;
            if (!DIST && j0 + i == (int64_t)tok) g += ct;
            v[i] = g * slope<CAP>(v[i], A.sc);
        }
        if (R.whole(c) && (((uintptr_t)(gout + j0)) & 15u) == 0) {
            uint4 q;
            T *e = reinterpret_cast<T *>(&q);
#pragma unroll
            for (int i = 0; i < E; i++) e[i] = from_f<T>(v[i]);
            *reinterpret_cast<uint4 *>(gout + j0) = q;
        } else {
#pragma unroll
            for (int i = 0; i < E; i++)
                if (j0 + i >= 0 && j0 + i < (int64_t)V) gout[j0 + i] = from_f<T>(v[i]);
        }
    }
    if (DIST) {
        // the teacher's ids: p Q - q, where q is the sum over the slots that
        // hold the id (the first of them writes)
        __syncthreads();
        for (uint32_t i = tid; i < A.n_ids; i += THREADS) {
            const int32_t id = s_id[i];
            if (id < 0) continue;
            float q = 0.0f;
            bool first = true;
            for (uint32_t j = 0; j < A.n_ids; j++)
                if (s_id[j] == id) {
                    if (j < i) first = false;
                    q += s_q[j];
                }
            if (!first) continue;
            const float p = ex2((s_c[i] - m) * k - l2f);
            gout[id] = from_f<T>((p * q_all - w * A.sc.m * q) * slope<CAP>(s_c[i], A.sc));
        }
    }
}

// The logits' gradient from those of log-probability and entropy, with the
// forward pass's statistics:
//   dv_j = m c'(v_j) [g (d_jt - p_j) - h p_j (log p_j + H)]
template <typename T, bool CAP, bool ENT>
__global__ void __launch_bounds__(THREADS) k_logprob_grad(RowArgs A, const float2 *stats, const float *d_lp,
                                                          const float *d_ent, const float *entropy) {
    constexpr int E = Row<T>::E;
    const uint32_t row = blockIdx.x, tid = threadIdx.x, V = A.vocab;
    Row<T> R(A.x, A.ld, row, V);
    T *gout = (T *)A.grad + (size_t)row * A.ld_grad;
    const int32_t tok = A.tokens[row];
    if ((uint32_t)tok >= V) {
        for (uint32_t j = tid; j < V; j += THREADS) gout[j] = from_f<T>(0.0f);
        return;
    }
    const float2 st = stats[row];
    const float m = st.x, k = A.sc.k, l2s = st.y * (float)(1.0 / LN2_D);
    const float g = d_lp ? d_lp[row] * A.sc.m : 0.0f;
    const float h = ENT ? d_ent[row] * A.sc.m : 0.0f;
    const float ca = ENT ? -g - h * entropy[row] : -g, cb = ENT ? -h * LN2 : 0.0f;
    for (uint32_t c = tid; c < R.chunks; c += THREADS) {
        float v[E];
        R.template load<CAP>(c, A.sc, v);
        const int64_t j0 = R.first(c);
#pragma unroll
        for (int i = 0; i < E; i++) {
            const float lp2 = (v[i] - m) * k - l2s;
            const float p = ex2(lp2);
            float o = ENT ? p * fmaf(cb, max_nan(lp2, D_MIN), ca) : p * ca;
            if (j0 + i == (int64_t)tok) o += g;
            v[i] = o * slope<CAP>(v[i], A.sc);
        }
        if (R.whole(c) && (((uintptr_t)(gout + j0)) & 15u) == 0) {
            uint4 q;
            T *e = reinterpret_cast<T *>(&q);
#pragma unroll
            for (int i = 0; i < E; i++) e[i] = from_f<T>(v[i]);
            *reinterpret_cast<uint4 *>(gout + j0) = q;
        } else {
#pragma unroll
            for (int i = 0; i < E; i++)
                if (j0 + i >= 0 && j0 + i < (int64_t)V) gout[j0 + i] = from_f<T>(v[i]);
        }
    }
}

// loss = sum_i w_i L_i in a fixed order, in 64 bits; a row of weight 0 adds
// nothing whatever its loss.
__global__ void __launch_bounds__(1024) k_loss(const float *row_loss, const float *weights, float w_all, uint32_t rows,
                                               float *loss) {
    __shared__ double part[32];
    double s = 0.0;
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

// One CTA per row: statistics, then a radix selection over the whole row
// (four passes over the key's digits; ties are cut by the same selection over
// the ids), then a sort of the k winners by (key, lower id).
template <typename T, bool CAP>
__global__ void __launch_bounds__(THREADS) k_top_row(const void *x, size_t ld, uint32_t vocab, Scale sc, float out_scale,
                                                     uint32_t top, float *values, int32_t *ids, float *lse) {
    constexpr int E = Row<T>::E;
    __shared__ Stat sh_stat[WARPS];
    __shared__ uint32_t hist[256];
    __shared__ uint32_t sh_bin, sh_need, sh_n;
    __shared__ unsigned long long best[MAX_K];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    Row<T> R(x, ld, row, vocab);

    Stat a{-INFINITY, 0.0f, 0.0f};
    for (uint32_t c = tid; c < R.chunks; c += THREADS) {
        float v[E];
        R.template load<CAP>(c, sc, v);
        float m = v[0];
#pragma unroll
        for (int i = 1; i < E; i++) m = fmaxf(m, v[i]);
        if (m > a.m) rebase(a, m, sc.k);
        const float base = anchor(a.m);
#pragma unroll
        for (int i = 0; i < E; i++) a.s += ex2((v[i] - base) * sc.k);
    }
    for (int o = 16; o; o >>= 1) {
        Stat b;
        b.m = __shfl_xor_sync(~0u, a.m, o);
        b.s = __shfl_xor_sync(~0u, a.s, o);
        b.u = 0.0f;
        a = merge(a, b, sc.k);
    }
    if ((tid & 31) == 0) sh_stat[tid >> 5] = a;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < WARPS; i++) a = merge(a, sh_stat[i], sc.k);
        lse[row] = (float)((double)a.m * (double)sc.m + LN2_D * log2_d(a.s));
        sh_n = 0;
    }

    // the k-th largest key
    uint32_t need = top, prefix = 0, mask = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (uint32_t i = tid; i < 256; i += THREADS) hist[i] = 0;
        __syncthreads();
        for (uint32_t j = tid; j < vocab; j += THREADS) {
            uint32_t key = order_key(to_f(R.x[j]));
            if ((key & mask) == prefix) atomicAdd(&hist[key >> shift & 255u], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            sh_bin = pick_bin(hist, need);
            sh_need = need;
        }
        __syncthreads();
        need = sh_need;
        prefix |= sh_bin << shift;
        mask |= 255u << shift;
    }
    const uint32_t kth = prefix;
    // of the elements that equal it, the `need` with the lowest ids: the
    // need-th largest ~id
    uint32_t id_floor = 0, id_mask = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (uint32_t i = tid; i < 256; i += THREADS) hist[i] = 0;
        __syncthreads();
        for (uint32_t j = tid; j < vocab; j += THREADS)
            if (order_key(to_f(R.x[j])) == kth && (~j & id_mask) == id_floor) atomicAdd(&hist[~j >> shift & 255u], 1u);
        __syncthreads();
        if (tid == 0) {
            sh_bin = pick_bin(hist, need);
            sh_need = need;
        }
        __syncthreads();
        need = sh_need;
        id_floor |= sh_bin << shift;
        id_mask |= 255u << shift;
    }
    for (uint32_t i = tid; i < MAX_K; i += THREADS) best[i] = 0ull;
    __syncthreads();
    for (uint32_t j = tid; j < vocab; j += THREADS) {
        uint32_t key = order_key(to_f(R.x[j]));
        if (key > kth || (key == kth && ~j >= id_floor)) {
            uint32_t at = atomicAdd(&sh_n, 1u);
            if (at < MAX_K) best[at] = (unsigned long long)key << 32 | (uint32_t)~j;
        }
    }
    uint32_t n = 1;
    while (n < top) n <<= 1;
    for (uint32_t size = 2; size <= n; size <<= 1)
        for (uint32_t stride = size >> 1; stride; stride >>= 1) {
            __syncthreads();
            for (uint32_t i = tid; i < n / 2; i += THREADS) {
                uint32_t lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
                bool down = (lo & size) == 0;
                unsigned long long p = best[lo], q = best[hi];
                if ((p < q) == down) {
                    best[lo] = q;
                    best[hi] = p;
                }
            }
        }
    __syncthreads();
    for (uint32_t i = tid; i < top; i += THREADS) {
        unsigned long long b = best[i];
        values[(size_t)row * top + i] = capped<CAP>(key_value((uint32_t)(b >> 32)), sc) * out_scale;
        ids[(size_t)row * top + i] = (int32_t)~(uint32_t)b;
    }
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
    sc->k = (float)k;
    sc->inv_t = 1.0 / (double)x->temperature;
    *cap = x->final_logit_softcapping > 0.0f;
    sc->cap = *cap ? x->final_logit_softcapping : 1.0f;
    sc->icap = 1.0f / sc->cap;
    *out_scale = (float)(1.0 / scale);
    return BS_OK;
}

static bs_status check_grad(const bs_logits *x, const void *grad, size_t ld_grad) {
    if (grad && (ld_grad < x->vocab || (uintptr_t)grad % elem_size(x->dtype))) return BS_EINVAL;
    return BS_OK;
}

template <typename T, int OP>
static bs_status launch_row(const RowArgs &A, uint32_t rows, bool cap, size_t smem, cudaStream_t st) {
    auto kern = cap ? k_row<T, OP, true> : k_row<T, OP, false>;
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) {
            fprintf(stderr, "b200_sampler: logit_ops: shared memory of %zu bytes: %s\n", smem, cudaGetErrorString(e));
            return BS_ECUDA;
        }
    }
    kern<<<rows, THREADS, smem, st>>>(A);
    return launched("logit_ops");
}

template <int OP>
static bs_status launch_row_typed(const bs_logits *x, const RowArgs &A, bool cap, size_t smem, cudaStream_t st) {
    switch (x->dtype) {
        case BS_F32: return launch_row<float, OP>(A, x->rows, cap, smem, st);
        case BS_BF16: return launch_row<__nv_bfloat16, OP>(A, x->rows, cap, smem, st);
        default: return launch_row<__half, OP>(A, x->rows, cap, smem, st);
    }
}

static RowArgs row_args(const bs_logits *x, const Scale &sc) {
    RowArgs A = {};
    A.x = x->data;
    A.ld = x->ld;
    A.vocab = x->vocab;
    A.sc = sc;
    A.w_all = x->rows ? 1.0f / (float)x->rows : 0.0f;
    return A;
}

static bs_status total_loss(const RowArgs &A, uint32_t rows, float *loss, cudaStream_t st) {
    k_loss<<<1, 1024, 0, st>>>(A.row_loss, A.weights, A.w_all, rows, loss);
    return launched("logit_ops loss");
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
    return launch_row_typed<OP_LOGPROB>(x, A, cap, 0, (cudaStream_t)stream);
}

template <typename T>
static bs_status launch_logprob_grad(const RowArgs &A, uint32_t rows, bool cap, const float2 *stats, const float *d_lp,
                                     const float *d_ent, const float *entropy, cudaStream_t st) {
    auto kern = cap ? (d_ent ? k_logprob_grad<T, true, true> : k_logprob_grad<T, true, false>)
                    : (d_ent ? k_logprob_grad<T, false, true> : k_logprob_grad<T, false, false>);
    kern<<<rows, THREADS, 0, st>>>(A, stats, d_lp, d_ent, entropy);
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
    A.clip_lo = 1.0f - cfg->clip_low;
    A.clip_hi = 1.0f + cfg->clip_high;
    A.kl_coef = cfg->kl_coef;
    A.ent_coef = cfg->entropy_coef;
    A.row_loss = d_row_loss;
    A.logprobs = d_logprobs;
    A.entropy = d_entropy;
    A.kl = d_kl;
    A.grad = d_grad;
    A.ld_grad = ld_grad;
    cudaStream_t s = (cudaStream_t)stream;
    st = cfg->entropy_coef != 0.0f ? launch_row_typed<OP_POLICY_ENT>(x, A, cap, 0, s)
                                   : launch_row_typed<OP_POLICY>(x, A, cap, 0, s);
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
    size_t smem = (size_t)n_ids * 12;
    if (d_teacher_lse) smem += ((size_t)x->vocab + 16 + 31) / 32 * 4 + 16;
    cudaStream_t s = (cudaStream_t)stream;
    st = d_teacher_lse ? launch_row_typed<OP_DISTILL_TAIL>(x, A, cap, smem, s)
                       : launch_row_typed<OP_DISTILL>(x, A, cap, smem, s);
    return st != BS_OK ? st : total_loss(A, x->rows, d_loss, s);
}

template <typename T>
static bs_status launch_top(const bs_logits *x, const Scale &sc, float os, bool cap, uint32_t k, float *values,
                            int32_t *ids, float *lse, cudaStream_t st) {
    auto kern = cap ? k_top_row<T, true> : k_top_row<T, false>;
    kern<<<x->rows, THREADS, 0, st>>>(x->data, x->ld, x->vocab, sc, os, k, values, ids, lse);
    return launched("bs_top_logits");
}

extern "C" bs_status bs_top_logits(const bs_logits *x, uint32_t k, float *d_values, int32_t *d_ids, float *d_lse,
                                   void *stream) {
    Scale sc;
    float os;
    bool cap;
    bs_status st = check_logits(x, &sc, &os, &cap);
    if (st != BS_OK) return st;
    if (k == 0 || k > x->vocab) return BS_EINVAL;
    if (k > BS_MAX_TOP) return BS_ENOTSUP;
    if (x->rows == 0) return BS_OK;
    if (!d_values || !d_ids || !d_lse) return BS_EINVAL;
    cudaStream_t s = (cudaStream_t)stream;
    switch (x->dtype) {
        case BS_F32: return launch_top<float>(x, sc, os, cap, k, d_values, d_ids, d_lse, s);
        case BS_BF16: return launch_top<__nv_bfloat16>(x, sc, os, cap, k, d_values, d_ids, d_lse, s);
        default: return launch_top<__half>(x, sc, os, cap, k, d_values, d_ids, d_lse, s);
    }
}
