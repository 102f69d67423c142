// Losses of a training step and the gradients they start the backward pass with (include/rlcu_losses.h).
//
// Mathematics, per row z of logits (t: inv_temperature, c = t * log2 e, y: target):
//   E  = ceil(c * max z)            an integer, so that x_j = fma(z_j, c, -E) is rounded once
//   s  = sum 2^x_j                  one pass with a running E per thread, partial sums rescaled by powers of two
//   logp = (x_y - log2 s) ln 2,     lse = (E + log2 s) ln 2
//   dz_j = coef * S * t * ([j == y] - 2^x_j / s)
#include "rlcu_losses.h"

#include <cfloat>
#include <cmath>

#include "host_util.h"
#include "typed.cuh"

namespace rlcu {
namespace {

constexpr int kRowThreads = 512;
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Where the running maximum starts: logits below it (-inf, and masks of a type's lowest value) add nothing,
// and a row without any other has s = 0.
constexpr float kNoLogit = -1e30f;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct LogitsArgs {
    const void* data;
    uint64_t rows, row_stride;
    uint32_t vocab;
    float inv_temperature;
    const int32_t* targets;
    float* logp;
    float* lse;
    void* grad;
    uint64_t grad_stride;
    const rlcu_scaler_state* scaler;
};

struct PolicyArgs {
    const float* old_logp;
    const float* ref_logp;
    const float* advantage;
    const float* weight;      // NULL outside the policy loss
    rlcu_policy_hparams hp;
};

struct PolicyTerm {
    float l, k, coef, ratio;
    bool cut;
};

// One token of the policy loss.
__device__ __forceinline__ PolicyTerm policy_term(float logp, const PolicyArgs& p, uint64_t t) {
    const float a = p.advantage[t], w = p.weight[t];
    PolicyTerm o;
    o.ratio = p.old_logp ? expf(logp - p.old_logp[t]) : 1.0f;
    const float lo = 1.0f - p.hp.clip_low, hi = 1.0f + p.hp.clip_high;
    const float kept = o.ratio * a;
    float best = kept, slope = kept;
    // a comparison with NaN is false: a NaN ratio stays in `best`, `slope` and so in the gradient
    const float held = (o.ratio < lo ? lo : (o.ratio > hi ? hi : o.ratio)) * a;
    o.cut = false;
    if (held < kept) {
        best = held;
        slope = 0.0f;
        o.cut = true;
    }
    if (p.hp.dual_clip > 0.0f && a < 0.0f && best < p.hp.dual_clip * a) {
        best = p.hp.dual_clip * a;
        slope = 0.0f;
        o.cut = true;
    }
    o.l = -best;
    o.k = 0.0f;
    float dk = 0.0f;
    if (p.hp.kl_coef != 0.0f) {
        const float d = logp - p.ref_logp[t];
        if (p.hp.kl_kind == RLCU_KL_K1) {
            o.k = d;
            dk = 1.0f;
        } else if (p.hp.kl_kind == RLCU_KL_K2) {
            o.k = 0.5f * d * d;
            dk = d;
        } else {
            const float e = expm1f(-d);          // exp(-d) - 1 without the cancellation at small d
            o.k = e + d;
            dk = -e;
        }
    }
    o.coef = w * (p.hp.kl_coef * dk - slope);
    return o;
}

// ---------------------------------------------------------------------------
// logits
// ---------------------------------------------------------------------------

// Sum of 2^(c z - ceil(c max)) with its running maximum.
struct Online {
    float top = kNoLogit;   // largest logit so far
    float e;                // ceil(c * top)
    float s = 0.0f;

    __device__ __forceinline__ explicit Online(float c) : e(ceilf(kNoLogit * c)) {}
    __device__ __forceinline__ void raise(float top_new, float c) {
        if (top_new > top) {
            const float e_new = ceilf(top_new * c);
            s *= exp2_fast(e - e_new);
            top = top_new;
            e = e_new;
        }
    }
    __device__ __forceinline__ void add(float z, float c) {
        raise(z, c);
        s += exp2_fast(fmaf(z, c, -e));
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&z)[N], float largest, float c) {
        raise(largest, c);
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            a += exp2_fast(fmaf(z[i], c, -e));
            b += exp2_fast(fmaf(z[i + 1], c, -e));
        }
        s += a + b;
    }
    __device__ __forceinline__ void merge(float top2, float s2, float c) {
        const float e2 = ceilf(top2 * c);
        if (top2 > top) {
            s = s * exp2_fast(e - e2) + s2;
            top = top2;
            e = e2;
        } else {
            s = s + s2 * exp2_fast(e2 - e);
        }
    }
};

enum { kModeLogprob = 0, kModeGrad = 1, kModePolicy = 2 };

__device__ __forceinline__ bool row_takes_part(const LogitsArgs& a, const PolicyArgs& p, uint64_t row, int32_t y) {
    if (y < 0 || (uint32_t)y >= a.vocab) return false;
    return !p.weight || p.weight[row] != 0.0f;
}

template <uint32_t DT>
__device__ __forceinline__ void zero_row(void* grad, uint64_t at, uint32_t vocab, int tid, int threads) {
    using E = Elem<DT>;
    typename E::T* out = static_cast<typename E::T*>(grad) + at;
    const RowCut cut = cut_row(out, vocab);
    if (tid < (int)cut.head) out[tid] = E::down(0.0f);
    uint4* body = reinterpret_cast<uint4*>(out + cut.head);
    for (uint32_t i = tid; i < cut.groups; i += threads) __stcs(body + i, make_uint4(0u, 0u, 0u, 0u));
    for (uint32_t i = cut.head + cut.groups * E::kVec + tid; i < vocab; i += threads) out[i] = E::down(0.0f);
}

// One CTA per row, two passes: the running sum, then the gradient.  The second pass finds the row in L2 (148
// rows of 300 KB are 44 MB of its 126).
template <uint32_t DT, int MODE>
__global__ void __launch_bounds__(kRowThreads)
logits_row_kernel(LogitsArgs a, PolicyArgs p, const float* lse_in, const float* coef_in) {
    using E = Elem<DT>;
    using T = typename E::T;
    __shared__ float tops[kRowThreads / 32], sums[kRowThreads / 32];
    __shared__ float row_e, row_scale, row_k;
    const float c = a.inv_temperature * kLog2E;
    const float S = a.scaler ? a.scaler->scale : 1.0f;

    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int32_t y = a.targets[row];
        bool takes = row_takes_part(a, p, row, y);
        if (MODE == kModeGrad) takes = takes && coef_in[row] != 0.0f;
        if (!takes) {
            if (MODE != kModeGrad && threadIdx.x == 0) {
                a.logp[row] = 0.0f;
                if (a.lse) a.lse[row] = 0.0f;
            }
            if (a.grad) zero_row<DT>(a.grad, row * a.grad_stride, a.vocab, threadIdx.x, kRowThreads);
            continue;
        }
        const T* x = static_cast<const T*>(a.data) + row * a.row_stride;
        const RowCut cut = cut_row(x, a.vocab);
        const uint4* body = reinterpret_cast<const uint4*>(x + cut.head);
        const uint32_t tail = cut.head + cut.groups * E::kVec;

        if (MODE != kModeGrad) {
            Online o(c);
            for (uint32_t i = threadIdx.x; i < cut.groups; i += kRowThreads) {
                const uint4 v = body[i];
                float f[E::kVec];
                E::unpack(v, f);
                o.add(f, E::largest(v), c);
            }
            if (threadIdx.x < cut.head) o.add(E::up(x[threadIdx.x]), c);
            for (uint32_t i = tail + threadIdx.x; i < a.vocab; i += kRowThreads) o.add(E::up(x[i]), c);
#pragma unroll
            for (int mask = 16; mask >= 1; mask >>= 1)
                o.merge(__shfl_xor_sync(0xFFFFFFFFu, o.top, mask), __shfl_xor_sync(0xFFFFFFFFu, o.s, mask), c);
            if ((threadIdx.x & 31) == 0) {
                tops[threadIdx.x >> 5] = o.top;
                sums[threadIdx.x >> 5] = o.s;
            }
            __syncthreads();
            if (threadIdx.x == 0) {
                Online all(c);
                for (int w = 0; w < kRowThreads / 32; w++) all.merge(tops[w], sums[w], c);
                if (all.e == INFINITY) all.s = NAN;      // logits whose product with c is beyond FP32
                const float l2 = log2f(all.s);
                // s = 0: nothing but -inf in the row
                const float logp = all.s == 0.0f ? -INFINITY : (fmaf(E::up(x[y]), c, -all.e) - l2) * kLn2;
                a.logp[row] = logp;
                if (a.lse) a.lse[row] = (all.e + l2) * kLn2;
                if (MODE == kModePolicy) {
                    row_e = all.e;
                    row_scale = all.s == 0.0f ? 0.0f : 1.0f / all.s;
                    row_k = policy_term(logp, p, row).coef * S * a.inv_temperature;
                    tops[0] = -expm1f(logp);     // 1 - p_y
                }
            }
            __syncthreads();
        }
        if (MODE == kModeLogprob) continue;

        // gradient
        float e, scale, k, rest;
        if (MODE == kModePolicy) {
            e = row_e;
            scale = row_scale;
            k = row_k;
            rest = tops[0];
        } else {
            const float lse = lse_in[row];
            // 2^(c z - log2e lse) = 2^(c z - e) * 2^(e - log2e lse), e an integer
            e = lse == -INFINITY ? 0.0f : rintf(lse * kLog2E);
            scale = lse == -INFINITY ? 0.0f : exp2f(-fmaf(lse, kLog2E, -e));
            k = coef_in[row] * S * a.inv_temperature;
            rest = lse == -INFINITY ? 1.0f : -expm1f(fmaf(E::up(x[y]), a.inv_temperature, -lse));
        }
        const float kn = -k * scale, ky = k * rest;
        if (MODE == kModeGrad) __syncthreads();          // x[y] is read before it is overwritten in place
        T* g = static_cast<T*>(a.grad) + row * a.grad_stride;
        const bool vec = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(x)) & 15u) == 0;
        if (vec) {
            uint4* out = reinterpret_cast<uint4*>(g + cut.head);
            for (uint32_t i = threadIdx.x; i < cut.groups; i += kRowThreads) {
                float f[E::kVec];
                E::unpack(body[i], f);
                const uint32_t at = (uint32_t)y - (cut.head + i * E::kVec);
#pragma unroll
                for (int j = 0; j < E::kVec; j++) f[j] = (uint32_t)j == at ? ky : kn * exp2_fast(fmaf(f[j], c, -e));
                __stcs(out + i, E::pack(f));
            }
            if (threadIdx.x < cut.head)
                g[threadIdx.x] = E::down(threadIdx.x == (uint32_t)y ? ky : kn * exp2_fast(fmaf(E::up(x[threadIdx.x]), c, -e)));
            for (uint32_t i = tail + threadIdx.x; i < a.vocab; i += kRowThreads)
                g[i] = E::down(i == (uint32_t)y ? ky : kn * exp2_fast(fmaf(E::up(x[i]), c, -e)));
        } else {
            for (uint32_t i = threadIdx.x; i < a.vocab; i += kRowThreads)
                g[i] = E::down(i == (uint32_t)y ? ky : kn * exp2_fast(fmaf(E::up(x[i]), c, -e)));
        }
        __syncthreads();                                  // row_* and tops are written again for the next row
    }
}

// ---------------------------------------------------------------------------
// policy loss of log-probabilities
// ---------------------------------------------------------------------------

constexpr int kVectorThreads = 1024;

__device__ __forceinline__ double block_sum_d(double x, double* smem) {
#pragma unroll
    for (int mask = 16; mask >= 1; mask >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, mask);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = x;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) s += smem[w];
    return s;
}

// Weighted sums of the policy loss over all tokens, and the gradient by log-probability.  `targets` (with vocab):
// tokens whose target is out of range take no part.
__global__ void __launch_bounds__(kVectorThreads)
policy_kernel(const float* logp, uint64_t tokens, const int32_t* targets, uint32_t vocab, PolicyArgs p, float* coef,
              rlcu_policy_stat* stat, uint32_t flags) {
    __shared__ double smem[kVectorThreads / 32];
    double sum_l = 0.0, sum_k = 0.0, sum_w = 0.0, n = 0.0, cuts = 0.0;
    float ratio = 0.0f;
    for (uint64_t t = threadIdx.x; t < tokens; t += kVectorThreads) {
        const float w = p.weight[t];
        const bool takes = w != 0.0f && (!targets || (targets[t] >= 0 && (uint32_t)targets[t] < vocab));
        float co = 0.0f;
        if (takes) {
            const PolicyTerm o = policy_term(logp[t], p, t);
            sum_l += (double)w * o.l;
            sum_k += (double)w * o.k;
            sum_w += w;
            n += 1.0;
            cuts += o.cut ? 1.0 : 0.0;
            ratio = fmaxf(ratio, o.ratio);
            co = o.coef;
        }
        if (coef) coef[t] = co;
    }
    sum_l = block_sum_d(sum_l, smem);
    sum_k = block_sum_d(sum_k, smem);
    sum_w = block_sum_d(sum_w, smem);
    n = block_sum_d(n, smem);
    cuts = block_sum_d(cuts, smem);
#pragma unroll
    for (int mask = 16; mask >= 1; mask >>= 1) ratio = fmaxf(ratio, __shfl_xor_sync(0xFFFFFFFFu, ratio, mask));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = ratio;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 0; w < kVectorThreads / 32; w++) ratio = fmaxf(ratio, (float)smem[w]);
        rlcu_policy_stat r = {};
        if (flags & RLCU_LOSS_ACCUMULATE) r = *stat;
        const double kl = p.hp.kl_coef != 0.0f ? (double)p.hp.kl_coef * sum_k : 0.0;
        r.loss = (float)((double)r.loss + sum_l + kl);
        r.policy = (float)((double)r.policy + sum_l);
        r.kl = (float)((double)r.kl + sum_k);
        r.weight = (float)((double)r.weight + sum_w);
        r.tokens += (uint32_t)n;
        r.clipped += (uint32_t)cuts;
        r.ratio_max = fmaxf(r.ratio_max, ratio);
        *stat = r;
    }
}

// ---------------------------------------------------------------------------
// preference loss
// ---------------------------------------------------------------------------

struct PreferenceArgs {
    const float* logp;
    const float* ref_logp;
    const uint8_t* mask;
    const int32_t* offsets;
    const float* pair_weight;
    uint64_t tokens, pairs;
    rlcu_preference_hparams hp;
    float* coef;
    float* rewards;
    rlcu_preference_stat* stat;
    uint32_t flags;
};

__device__ __forceinline__ uint64_t offset_at(const PreferenceArgs& a, uint64_t q) {
    const int32_t o = a.offsets[q];
    return o < 0 ? 0ull : ((uint64_t)o < a.tokens ? (uint64_t)o : a.tokens);
}

__device__ __forceinline__ void preference_term(const rlcu_preference_hparams& hp, double c, double r, double& h,
                                                double& loss, double& slope) {
    const double beta = hp.beta;
    h = beta * (c - r) - (double)hp.margin;
    if (hp.kind == RLCU_PREF_SIGMOID) {
        const double e = hp.label_smoothing, tail = log1p(exp(-fabs(h)));
        // -log sigmoid(h) = max(-h, 0) + log(1 + exp(-|h|))
        loss = (1.0 - e) * (fmax(-h, 0.0) + tail) + e * (fmax(h, 0.0) + tail);
        slope = e / (1.0 + exp(-h)) - (1.0 - e) / (1.0 + exp(h));
    } else if (hp.kind == RLCU_PREF_HINGE) {
        loss = fmax(0.0, 1.0 - h);
        slope = h < 1.0 ? -1.0 : 0.0;
        if (isnan(h)) loss = slope = h;
    } else {
        const double d = h / beta - 0.5 / beta;
        loss = d * d;
        slope = 2.0 * d / beta;
    }
    slope *= beta;
}

__global__ void __launch_bounds__(kVectorThreads)
preference_kernel(PreferenceArgs a) {
    __shared__ double smem[kVectorThreads / 32];
    double loss_sum = 0.0, margin_sum = 0.0;
    uint32_t correct = 0;
    const uint64_t first = offset_at(a, 0);
    if (a.coef)
        for (uint64_t t = threadIdx.x; t < first; t += kVectorThreads) a.coef[t] = 0.0f;
    uint64_t lo = first;
    for (uint64_t i = 0; i < a.pairs; i++) {
        double s[2], share[2];
        uint64_t at[3] = {lo, 0, 0};
        for (int q = 0; q < 2; q++) {
            at[q + 1] = offset_at(a, 2 * i + q + 1);
            if (at[q + 1] < at[q]) at[q + 1] = at[q];
            double sum = 0.0, n = 0.0;
            for (uint64_t t = at[q] + threadIdx.x; t < at[q + 1]; t += kVectorThreads) {
                if (a.mask && !a.mask[t]) continue;
                sum += (double)(a.ref_logp ? a.logp[t] - a.ref_logp[t] : a.logp[t]);
                n += 1.0;
            }
            s[q] = block_sum_d(sum, smem);
            n = a.hp.length_mean ? block_sum_d(n, smem) : 1.0;
            share[q] = n > 0.0 ? 1.0 / n : 0.0;
            s[q] *= share[q];
        }
        double h, loss, slope;
        preference_term(a.hp, s[0], s[1], h, loss, slope);
        const double w = a.pair_weight ? (double)a.pair_weight[i] : 1.0 / (double)a.pairs;
        loss_sum += w * loss;
        margin_sum += w * h;
        correct += s[0] > s[1];
        if (threadIdx.x == 0 && a.rewards) {
            a.rewards[2 * i] = (float)((double)a.hp.beta * s[0]);
            a.rewards[2 * i + 1] = (float)((double)a.hp.beta * s[1]);
        }
        if (a.coef)
            for (int q = 0; q < 2; q++) {
                const float co = (float)((q ? -slope : slope) * w * share[q]);
                for (uint64_t t = at[q] + threadIdx.x; t < at[q + 1]; t += kVectorThreads)
                    a.coef[t] = !a.mask || a.mask[t] ? co : 0.0f;
            }
        lo = at[2];
    }
    if (a.coef)
        for (uint64_t t = lo + threadIdx.x; t < a.tokens; t += kVectorThreads) a.coef[t] = 0.0f;
    if (threadIdx.x == 0) {
        rlcu_preference_stat r = {};
        if (a.flags & RLCU_LOSS_ACCUMULATE) r = *a.stat;
        r.loss = (float)((double)r.loss + loss_sum);
        r.margin = (float)((double)r.margin + margin_sum);
        r.pairs += (uint32_t)a.pairs;
        r.correct += correct;
        *a.stat = r;
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

int check_logits(const void* logits, uint32_t dtype, uint64_t rows, uint64_t vocab, uint64_t& row_stride,
                 float inv_temperature, const int32_t* targets) {
    if (!dtype_known(dtype)) return set_error(RLCU_ERR_INVALID, "unknown dtype %u", dtype);
    if (vocab < 1 || vocab > 0x7FFFFFFFull) return set_error(RLCU_ERR_INVALID, "vocab must be in [1, 2^31)");
    if (row_stride == 0) row_stride = vocab;
    if (row_stride < vocab) return set_error(RLCU_ERR_INVALID, "row stride below vocab");
    if (rows > 0x7FFFFFFFull || too_large(rows, row_stride)) return set_error(RLCU_ERR_INVALID, "rows or row stride out of range");
    if (!(inv_temperature > 0.0f && inv_temperature <= 1e6f)) return set_error(RLCU_ERR_INVALID, "inv_temperature must be in (0, 1e6]");
    if (rows && (!logits || !targets)) return set_error(RLCU_ERR_INVALID, "null logits or targets");
    if (reinterpret_cast<uintptr_t>(logits) % dtype_bytes(dtype)) return set_error(RLCU_ERR_INVALID, "logits not aligned to their element size");
    return RLCU_OK;
}

int check_grad(const void* logits, uint32_t dtype, uint64_t rows, uint64_t vocab, uint64_t row_stride, const void* grad,
               uint64_t& grad_stride) {
    if (grad_stride == 0) grad_stride = vocab;
    if (grad_stride < vocab || too_large(rows, grad_stride)) return set_error(RLCU_ERR_INVALID, "gradient stride below vocab or out of range");
    if (rows && !grad) return set_error(RLCU_ERR_INVALID, "null gradient");
    const size_t esz = dtype_bytes(dtype);
    if (reinterpret_cast<uintptr_t>(grad) % esz) return set_error(RLCU_ERR_INVALID, "gradient not aligned to its element size");
    if (grad == logits && (grad_stride == row_stride || rows <= 1)) return RLCU_OK;
    if (overlap(span_of(logits, rows, vocab, row_stride, esz), span_of(grad, rows, vocab, grad_stride, esz)))
        return set_error(RLCU_ERR_INVALID, "gradient and logits overlap without being the same buffer");
    return RLCU_OK;
}

int check_policy(const rlcu_policy_hparams* hp, const float* ref_logp, const float* advantage, const float* weight,
                 const rlcu_policy_stat* stat, uint64_t tokens, uint32_t flags) {
    if (!hp) return set_error(RLCU_ERR_INVALID, "null hyper-parameters");
    if (!(hp->clip_low >= 0.0f) || !(hp->clip_low <= 1.0f) || !(hp->clip_high >= 0.0f))
        return set_error(RLCU_ERR_INVALID, "clip_low must be in [0, 1] and clip_high at least 0");
    if (!(hp->dual_clip == 0.0f || (hp->dual_clip > 1.0f && !std::isinf(hp->dual_clip))))
        return set_error(RLCU_ERR_INVALID, "dual_clip must be 0 or above 1");
    if (!std::isfinite(hp->kl_coef)) return set_error(RLCU_ERR_INVALID, "kl_coef must be finite");
    if (hp->kl_coef != 0.0f && hp->kl_kind != RLCU_KL_K1 && hp->kl_kind != RLCU_KL_K2 && hp->kl_kind != RLCU_KL_K3)
        return set_error(RLCU_ERR_INVALID, "unknown kl_kind %u", hp->kl_kind);
    if (flags & ~(uint32_t)RLCU_LOSS_ACCUMULATE) return set_error(RLCU_ERR_INVALID, "unknown flags");
    if (tokens > 0x7FFFFFFFull) return set_error(RLCU_ERR_INVALID, "too many tokens");
    if (!stat || reinterpret_cast<uintptr_t>(stat) % 16) return set_error(RLCU_ERR_INVALID, "the record must be given and 16-byte aligned");
    if (tokens && (!advantage || !weight)) return set_error(RLCU_ERR_INVALID, "null advantage or weight");
    if (tokens && hp->kl_coef != 0.0f && !ref_logp) return set_error(RLCU_ERR_INVALID, "a KL term needs ref_logp");
    return RLCU_OK;
}

int sm_count(int* out) {
    int dev = 0;
    RLCU_CUDA(cudaGetDevice(&dev));
    RLCU_CUDA(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev));
    return RLCU_OK;
}

template <int MODE>
int launch_rows(const LogitsArgs& a, const PolicyArgs& p, uint32_t dtype, const float* lse, const float* coef, cudaStream_t s) {
    int sms = 0;
    if (const int rc = sm_count(&sms)) return rc;
    const uint64_t most = (uint64_t)sms * 4;
    const int grid = (int)(a.rows < most ? a.rows : most);
    if (dtype == RLCU_F16) logits_row_kernel<RLCU_F16, MODE><<<grid, kRowThreads, 0, s>>>(a, p, lse, coef);
    else if (dtype == RLCU_BF16) logits_row_kernel<RLCU_BF16, MODE><<<grid, kRowThreads, 0, s>>>(a, p, lse, coef);
    else logits_row_kernel<RLCU_F32, MODE><<<grid, kRowThreads, 0, s>>>(a, p, lse, coef);
    RLCU_CUDA(cudaGetLastError());
    return RLCU_OK;
}

int launch_policy(const float* logp, uint64_t tokens, const int32_t* targets, uint32_t vocab, const PolicyArgs& p,
                  float* coef, rlcu_policy_stat* stat, uint32_t flags, cudaStream_t s) {
    policy_kernel<<<1, kVectorThreads, 0, s>>>(logp, tokens, targets, vocab, p, coef, stat, flags);
    RLCU_CUDA(cudaGetLastError());
    return RLCU_OK;
}

}  // namespace
}  // namespace rlcu

using namespace rlcu;

extern "C" int rlcu_token_logprob(const void* logits, uint32_t dtype, uint64_t rows, uint64_t vocab, uint64_t row_stride,
                                  float inv_temperature, const int32_t* targets, float* logp, float* lse, void* stream) {
    if (const int rc = check_logits(logits, dtype, rows, vocab, row_stride, inv_temperature, targets)) return rc;
    if (rows && !logp) return set_error(RLCU_ERR_INVALID, "null logp");
    if (!rows) return RLCU_OK;
    LogitsArgs a = {logits, rows, row_stride, (uint32_t)vocab, inv_temperature, targets, logp, lse, nullptr, 0, nullptr};
    return launch_rows<kModeLogprob>(a, PolicyArgs{}, dtype, nullptr, nullptr, (cudaStream_t)stream);
}

extern "C" int rlcu_token_logprob_grad(const void* logits, uint32_t dtype, uint64_t rows, uint64_t vocab,
                                       uint64_t row_stride, float inv_temperature, const int32_t* targets,
                                       const float* lse, const float* coef, const rlcu_scaler_state* scaler, void* grad,
                                       uint64_t grad_stride, void* stream) {
    if (const int rc = check_logits(logits, dtype, rows, vocab, row_stride, inv_temperature, targets)) return rc;
    if (const int rc = check_grad(logits, dtype, rows, vocab, row_stride, grad, grad_stride)) return rc;
    if (rows && (!lse || !coef)) return set_error(RLCU_ERR_INVALID, "null lse or coef");
    if (!rows) return RLCU_OK;
    LogitsArgs a = {logits, rows, row_stride, (uint32_t)vocab, inv_temperature, targets, nullptr, nullptr, grad, grad_stride, scaler};
    return launch_rows<kModeGrad>(a, PolicyArgs{}, dtype, lse, coef, (cudaStream_t)stream);
}

extern "C" int rlcu_policy_loss_logp(const float* logp, uint64_t tokens, const float* old_logp, const float* ref_logp,
                                     const float* advantage, const float* weight, const rlcu_policy_hparams* hp,
                                     float* coef, rlcu_policy_stat* stat, uint32_t flags, void* stream) {
    if (const int rc = check_policy(hp, ref_logp, advantage, weight, stat, tokens, flags)) return rc;
    if (tokens && !logp) return set_error(RLCU_ERR_INVALID, "null logp");
    PolicyArgs p = {old_logp, ref_logp, advantage, weight, *hp};
    return launch_policy(logp, tokens, nullptr, 0, p, coef, stat, flags, (cudaStream_t)stream);
}

extern "C" int rlcu_policy_loss(const void* logits, uint32_t dtype, uint64_t rows, uint64_t vocab, uint64_t row_stride,
                                float inv_temperature, const int32_t* targets, const float* old_logp,
                                const float* ref_logp, const float* advantage, const float* weight,
                                const rlcu_policy_hparams* hp, const rlcu_scaler_state* scaler, float* logp, void* grad,
                                uint64_t grad_stride, rlcu_policy_stat* stat, uint32_t flags, void* stream) {
    if (const int rc = check_logits(logits, dtype, rows, vocab, row_stride, inv_temperature, targets)) return rc;
    if (const int rc = check_policy(hp, ref_logp, advantage, weight, stat, rows, flags)) return rc;
    if (grad)
        if (const int rc = check_grad(logits, dtype, rows, vocab, row_stride, grad, grad_stride)) return rc;
    if (rows && !logp) return set_error(RLCU_ERR_INVALID, "null logp");
    LogitsArgs a = {logits, rows, row_stride, (uint32_t)vocab, inv_temperature, targets, logp, nullptr, grad, grad_stride, scaler};
    PolicyArgs p = {old_logp, ref_logp, advantage, weight, *hp};
    if (rows) {
        const int rc = grad ? launch_rows<kModePolicy>(a, p, dtype, nullptr, nullptr, (cudaStream_t)stream)
                            : launch_rows<kModeLogprob>(a, p, dtype, nullptr, nullptr, (cudaStream_t)stream);
        if (rc) return rc;
    }
    return launch_policy(logp, rows, targets, (uint32_t)vocab, p, nullptr, stat, flags, (cudaStream_t)stream);
}

extern "C" int rlcu_preference_loss(const float* logp, uint64_t tokens, const float* ref_logp, const uint8_t* mask,
                                    const int32_t* offsets, uint64_t pairs, const float* pair_weight,
                                    const rlcu_preference_hparams* hp, float* coef, float* rewards,
                                    rlcu_preference_stat* stat, uint32_t flags, void* stream) {
    if (!hp) return set_error(RLCU_ERR_INVALID, "null hyper-parameters");
    if (!(hp->beta > 0.0f) || std::isinf(hp->beta) || !std::isfinite(hp->margin))
        return set_error(RLCU_ERR_INVALID, "beta must be positive and finite, margin finite");
    if (hp->kind > RLCU_PREF_IPO) return set_error(RLCU_ERR_INVALID, "unknown kind %u", hp->kind);
    if (!(hp->label_smoothing >= 0.0f && hp->label_smoothing <= 0.5f) || (hp->label_smoothing != 0.0f && hp->kind != RLCU_PREF_SIGMOID))
        return set_error(RLCU_ERR_INVALID, "label_smoothing must be in [0, 0.5], and 0 for other kinds than the sigmoid");
    if (hp->length_mean > 1) return set_error(RLCU_ERR_INVALID, "length_mean must be 0 or 1");
    if (flags & ~(uint32_t)RLCU_LOSS_ACCUMULATE) return set_error(RLCU_ERR_INVALID, "unknown flags");
    if (tokens > 0x7FFFFFFFull || pairs > 0x3FFFFFFFull) return set_error(RLCU_ERR_INVALID, "too many tokens or pairs");
    if (!stat || reinterpret_cast<uintptr_t>(stat) % 16) return set_error(RLCU_ERR_INVALID, "the record must be given and 16-byte aligned");
    if (!offsets) return set_error(RLCU_ERR_INVALID, "null offsets");
    if (tokens && !logp) return set_error(RLCU_ERR_INVALID, "null logp");
    PreferenceArgs a = {logp, ref_logp, mask, offsets, pair_weight, tokens, pairs, *hp, coef, rewards, stat, flags};
    preference_kernel<<<1, kVectorThreads, 0, (cudaStream_t)stream>>>(a);
    RLCU_CUDA(cudaGetLastError());
    return RLCU_OK;
}
