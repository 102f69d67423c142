// Losses of a training step and the gradients they start the backward pass with (include/rlcu_losses.h).
//
// Mathematics, per row z of logits (t: inv_temperature, c = t * log2 e, y: target):
//   E  = ceil(c * max z)            an integer, so that x_j = fma(z_j, c, -E) is rounded once (within 2^31: see Top)
//   s  = sum 2^x_j                  one pass with a running E per thread, partial sums rescaled by powers of two
//   logp = (x_y - log2 s) ln 2,     lse = (E + log2 s) ln 2
//   dz_j = coef * S * t * ([j == y] - 2^x_j / s)
#include "rlcu_losses.h"

#include <cooperative_groups.h>

#include <atomic>
#include <cfloat>
#include <cmath>

#include "host_util.h"
#include "typed.cuh"

namespace rlcu {
namespace {

constexpr int kRowThreads = 512;
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Logits of this and less (-inf, and masks of a type's lowest value) add nothing, and a row without any other has s = 0.
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
    uint32_t tries;           // of a wait before it counts as given up
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

// One token of the policy loss: advantage a, weight w, log-probabilities logp, old (p.old_logp given) and ref
// (a KL term given).
__device__ __forceinline__ PolicyTerm policy_term(const PolicyArgs& p, float logp, float a, float w, float old, float ref) {
    PolicyTerm o;
    const float since = p.old_logp ? logp - old : 0.0f;
    o.ratio = expf(since);
    const float lo = 1.0f - p.hp.clip_low, hi = 1.0f + p.hp.clip_high;
    // (a ratio beyond FP32 is still a number, and nothing of it is left where there is no advantage)
    const float kept = a == 0.0f && o.ratio == INFINITY && since < INFINITY ? 0.0f : o.ratio * a;
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
        const float d = logp - ref;
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

__device__ __forceinline__ PolicyTerm policy_term(const PolicyArgs& p, float logp, uint64_t t) {
    return policy_term(p, logp, p.advantage[t], p.weight[t], p.old_logp ? p.old_logp[t] : 0.0f,
                       p.hp.kl_coef != 0.0f ? p.ref_logp[t] : 0.0f);
}

// ---------------------------------------------------------------------------
// logits
// ---------------------------------------------------------------------------

// Sum of 2^(c z - e) for an integer e that follows the largest c z: raised when terms pass 2^kSlack, so after a
// thread's first group hardly ever.  The sum is a float: how far e lies below the largest term costs nothing.
// It stays within 2^31: a larger one would be so coarse that the largest term itself is inf or 0 beside it.  Terms below
// 2^-2^31 are zeros then, as they have to be beside any other, and a row without any other ends with s = 0; a term above
// 2^2^31 makes s inf.  Such rows are looked at again (Top).
constexpr float kSlack = 1099511627776.0f;            // 2^40
constexpr float kFar = 2147483648.0f;                 // 2^31

struct Online {
    float e;
    float s = 0.0f;

    __device__ __forceinline__ explicit Online(float c) : e(fmaxf(ceilf(kNoLogit * c), -kFar)) {}
    __device__ __forceinline__ void raise(float largest, float c) {
        const float e_new = ceilf(fminf(largest * c, kFar));
        if (e_new > e) {
            s *= exp2_fast(e - e_new);
            e = e_new;
        }
    }
    __device__ __forceinline__ void add(float z, float c) {
        raise(z, c);
        s += exp2_fast(fmaf(z, c, -e));
    }
    template <int N>
    __device__ __forceinline__ float terms(const float (&f)[N], float c) const {
        const F2 cc(c, c), ee(-e, -e);
        F2 sum;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            float x, y;
            fma2(F2(f[i], f[i + 1]), cc, ee).get(x, y);
            const F2 term(exp2_fast(x), exp2_fast(y));
            sum = i ? add2(sum, term) : term;
        }
        float x, y;
        sum.get(x, y);
        return x + y;
    }
    // a group of 16 bytes
    template <uint32_t DT>
    __device__ __forceinline__ void add(uint4 v, float c) {
        using E = Elem<DT>;
        float f[E::kVec];
        E::unpack(v, f);
        float sum = terms(f, c);
        if (sum > kSlack) {                            // (NaN is not: it goes into the sum)
            raise(E::largest(v), c);
            sum = terms(f, c);
        }
        s += sum;
    }
    __device__ __forceinline__ void merge(float e2, float s2) {
        const float most = fmaxf(e, e2);
        s = s * exp2_fast(e - most) + s2 * exp2_fast(e2 - most);
        e = most;
    }
    __device__ __forceinline__ void merge_warp() {
        float most;
        asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(most) : "f"(e));      // (sm_100a; NaN is passed over)
        s *= exp2_fast(e - most);
        e = most;
#pragma unroll
        for (int mask = 16; mask >= 1; mask >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, mask);
    }
    // the sum says nothing of the row's largest logit
    __device__ __forceinline__ bool says_nothing() const { return s == 0.0f || s == INFINITY; }
};

// The other look at a row: its largest logit m and how many there are of it.  With c m beyond 2^31 two different logits of
// a type are 2^7 apart after the product with c, so that all but the largest add nothing to a float.
struct Top {
    float e = -INFINITY;           // m
    float s = 0.0f;                // their number

    __device__ __forceinline__ Top() {}
    __device__ __forceinline__ explicit Top(float) {}
    __device__ __forceinline__ void add(float z) { merge(z, z > kNoLogit ? 1.0f : 0.0f); }
    __device__ __forceinline__ void merge(float e2, float s2) {
        const float most = fmaxf(e, e2);
        s = (e == most ? s : 0.0f) + (e2 == most ? s2 : 0.0f);
        e = most;
    }
    __device__ __forceinline__ void merge_warp() {
#pragma unroll
        for (int mask = 16; mask >= 1; mask >>= 1) {
            const float e2 = __shfl_xor_sync(0xFFFFFFFFu, e, mask), s2 = __shfl_xor_sync(0xFFFFFFFFu, s, mask);
            merge(e2, s2);
        }
    }
};

// What one thread makes of a row's sum.
struct RowAnswer {
    float logp, lse;
    float e, by, inv;  // p_j = 2^(by z_j - e) * inv
};

// e is exact to 1 and more: rows of any usual logits
constexpr float kExact = 8388608.0f;                  // 2^23

// (o.s is neither 0 nor inf)
template <bool NEAR>
__device__ __forceinline__ RowAnswer row_answer(const Online& o, float z_y, float c) {
    // s = s' 2^k with s' in [1, 2).  k goes into e, so that x_y = c z_y - e is no larger than its own logarithm, or, where
    // that sum would be rounded, into x_y.
    float e = o.e, t = o.s;
    int k = 0;
    if (o.s > 0.0f && o.s < INFINITY) {
        k = (int)((__float_as_uint(o.s) >> 23) & 0xFFu) - 127;
        t *= __uint_as_float((uint32_t)(127 - k) << 23);
        if (NEAR || fabsf(e) < kExact) {
            e += (float)k;
            k = 0;
        }
    }
    const float l2 = log2f(t), x_y = fmaf(z_y, c, -e);
    RowAnswer r;
    r.by = c;
    r.e = e;
    r.logp = ((NEAR ? x_y : x_y - (float)k) - l2) * kLn2;
    r.lse = ((NEAR ? e : e + (float)k) + l2) * kLn2;
    r.inv = 1.0f / (NEAR || k == 0 ? t : o.s);
    return r;
}

__device__ __forceinline__ RowAnswer row_answer(const Top& o, float z_y, float c, float inv_temperature) {
    RowAnswer r;
    if (o.s == 0.0f) {             // nothing but -inf in the row
        r.logp = r.lse = -INFINITY;
        r.e = INFINITY;
        r.by = c;
        r.inv = 0.0f;
        return r;
    }
    // 2^31 <= |by m| < 2^32: exact, and any other logit is at least 2^7 away
    const uint32_t exponent = (__float_as_uint(o.e) >> 23) & 0xFFu;
    r.by = __uint_as_float((127u + 31u + 127u - exponent) << 23);
    r.e = o.e * r.by;
    r.inv = 1.0f / o.s;
    r.logp = fmaf(z_y - o.e, inv_temperature, -logf(o.s));
    r.lse = fmaf(o.e, inv_temperature, logf(o.s));
    if (isinf(o.e * c)) r.logp = r.lse = r.inv = NAN;      // +inf, or logits whose product with c is beyond FP32
    return r;
}

// 16 bytes of gradient away from the target: kn 2^(by z - e)
template <uint32_t DT>
__device__ __forceinline__ uint4 grad_group(uint4 v, float by, float e, float kn) {
    using E = Elem<DT>;
    float f[E::kVec];
    E::unpack(v, f);
    const F2 cc(by, by), ee(-e, -e), kk(kn, kn);
#pragma unroll
    for (int i = 0; i < E::kVec; i += 2) {
        float x, y;
        fma2(F2(f[i], f[i + 1]), cc, ee).get(x, y);
        mul2(F2(exp2_fast(x), exp2_fast(y)), kk).get(f[i], f[i + 1]);
    }
    return E::pack(f);
}

// An FP32 log-sum-exp of more than this is off by up to a factor of e, and a probability taken from it is worth nothing:
// the row's gradient is NaN.
constexpr float kMostLse = 16777216.0f;               // 2^24
__device__ __forceinline__ float usable(float lse) { return fabsf(lse) > kMostLse && lse != -INFINITY ? NAN : lse; }

// Top of a row, by a warp (a call, so that its registers are not taken from those who hardly ever make it)
template <uint32_t DT>
__device__ __noinline__ Top top_by_warp(const typename Elem<DT>::T* x, uint32_t n) {
    using E = Elem<DT>;
    const RowCut cut = cut_row(x, n);
    const uint32_t lane = threadIdx.x & 31;
    Top o;
#pragma unroll 4
    for (uint32_t i = lane; i < cut.groups; i += 32) {
        float f[E::kVec];
        E::unpack(reinterpret_cast<const uint4*>(x + cut.head)[i], f);
#pragma unroll
        for (int q = 0; q < E::kVec; q++) o.add(f[q]);
    }
    if (lane < cut.head) o.add(E::up(x[lane]));
    for (uint32_t i = cut.head + cut.groups * E::kVec + lane; i < n; i += 32) o.add(E::up(x[i]));
    o.merge_warp();
    return o;
}

// The sum over a CTA of up to 32 warps, in every thread.  Another call with the same parts needs a barrier before it.
template <typename Sum>
__device__ __forceinline__ Sum add_in_block(Sum o, float2* parts, float c) {
    o.merge_warp();
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = make_float2(o.e, o.s);
    __syncthreads();
    Sum all(c);
    if ((threadIdx.x & 31) < blockDim.x >> 5) all.merge(parts[threadIdx.x & 31].x, parts[threadIdx.x & 31].y);
    all.merge_warp();
    return all;
}

constexpr uint32_t kNoTarget = 0xFFFFFFFFu;
// log-probability (a NaN that no arithmetic makes) of a row whose sum says nothing, until policy_kernel has looked again
constexpr uint32_t kLookAgain = 0x7FC5EEDu << 4;
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

// One CTA per row, two passes: the running sum, then the gradient.  For what the kernels below do not take: a gradient
// whose rows lie at other 16-byte offsets than the logits', vocabularies of less than 64 groups of 16 bytes, rows beyond
// sixteen CTAs' registers.  4096 x 151936 bf16 takes 627 us this way.
template <uint32_t DT, int MODE>
__global__ void __launch_bounds__(kRowThreads)
logits_row_kernel(LogitsArgs a, PolicyArgs p, const float* lse_in, const float* logp_in, const float* coef_in) {
    using E = Elem<DT>;
    using T = typename E::T;
    __shared__ float2 warp_part[kRowThreads / 32];
    __shared__ float4 answer;                         // e, -k / s, k (1 - p_y), factor of z
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
            for (uint32_t i = threadIdx.x; i < cut.groups; i += kRowThreads) o.add<DT>(body[i], c);
            if (threadIdx.x < cut.head) o.add(E::up(x[threadIdx.x]), c);
            for (uint32_t i = tail + threadIdx.x; i < a.vocab; i += kRowThreads) o.add(E::up(x[i]), c);
            o = add_in_block(o, warp_part, c);
            if (threadIdx.x < 32) {
                const float z_y = E::up(x[y]);
                RowAnswer r;
                if (__any_sync(0xFFFFFFFFu, o.says_nothing())) r = row_answer(top_by_warp<DT>(x, a.vocab), z_y, c, a.inv_temperature);
                else r = row_answer<false>(o, z_y, c);
                if (threadIdx.x == 0) {
                    a.logp[row] = r.logp;
                    if (a.lse) a.lse[row] = r.lse;
                    if (MODE == kModePolicy) {
                        const float k = policy_term(p, r.logp, row).coef * S * a.inv_temperature;
                        answer = make_float4(r.e, -k * r.inv, -k * expm1f(r.logp), r.by);
                    }
                }
            }
            __syncthreads();
        }
        if (MODE == kModeLogprob) continue;

        // gradient
        float e, kn, ky, by = c;
        if (MODE == kModePolicy) {
            e = answer.x;
            kn = answer.y;
            ky = answer.z;
            by = answer.w;
        } else {
            // 2^(c z - log2e lse) = 2^(c z - e) * 2^(e - log2e lse), e an integer
            const float lse = usable(lse_in[row]), k = coef_in[row] * S * a.inv_temperature;
            const bool empty = lse == -INFINITY;
            e = empty ? 0.0f : rintf(lse * kLog2E);
            kn = empty ? 0.0f * k : -k * exp2f(-fmaf(lse, kLog2E, -e));
            ky = empty ? k : -k * expm1f(logp_in ? logp_in[row] + 0.0f * lse : fmaf(E::up(x[y]), a.inv_temperature, -lse));
        }
        if (MODE == kModeGrad) __syncthreads();          // x[y] is read before it is overwritten in place
        T* g = static_cast<T*>(a.grad) + row * a.grad_stride;
        const bool vec = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(x)) & 15u) == 0;
        if (vec) {
            uint4* out = reinterpret_cast<uint4*>(g + cut.head);
            for (uint32_t i = threadIdx.x; i < cut.groups; i += kRowThreads) __stcs(out + i, grad_group<DT>(body[i], by, e, kn));
            if ((uint32_t)y - cut.head < cut.groups * E::kVec && ((uint32_t)y - cut.head) / E::kVec % kRowThreads == threadIdx.x)
                g[y] = E::down(ky);              // behind this thread's own store of the group
            if (threadIdx.x < cut.head)
                g[threadIdx.x] = E::down(threadIdx.x == (uint32_t)y ? ky : kn * exp2_fast(fmaf(E::up(x[threadIdx.x]), by, -e)));
            for (uint32_t i = tail + threadIdx.x; i < a.vocab; i += kRowThreads)
                g[i] = E::down(i == (uint32_t)y ? ky : kn * exp2_fast(fmaf(E::up(x[i]), by, -e)));
        } else {
            for (uint32_t i = threadIdx.x; i < a.vocab; i += kRowThreads)
                g[i] = E::down(i == (uint32_t)y ? ky : kn * exp2_fast(fmaf(E::up(x[i]), by, -e)));
        }
        __syncthreads();                                  // the shared values are written again for the next row
    }
}

// CTAs that may share a row or a record.  More than 8 need the kernel's consent (non-portable cluster size).
constexpr int kMostCluster = 16;

// A row's share of one thread of a CTA: every THREADS-th group of the CTA's run, and perhaps one of the single
// elements at the row's ends.
template <uint32_t DT, int THREADS>
struct RowShare {
    using E = Elem<DT>;
    using T = typename E::T;
    const T* x;
    const uint4* in;          // first group
    uint32_t y;
    uint32_t groups;
    uint32_t end_at;          // index of the single element, or vocab
    bool owns_y;              // the target is in one of the groups

    // y_: the target, below vocab where the row takes part; a row that does not has nothing
    __device__ __forceinline__ RowShare(const LogitsArgs& a, uint32_t row, uint32_t y_, uint32_t rank, uint32_t C) {
        y = y_;
        x = static_cast<const T*>(a.data) + (uint64_t)row * a.row_stride;
        in = nullptr;
        groups = 0;
        end_at = a.vocab;
        owns_y = false;
        if (y >= a.vocab) return;
        const RowCut cut = cut_row(x, a.vocab);
        const uint32_t tid = threadIdx.x, tail = cut.head + cut.groups * E::kVec;
        const uint32_t share = (cut.groups + C - 1) / C;
        const uint32_t lo = min(rank * share, cut.groups), n = min(share, cut.groups - lo);
        groups = n > tid ? (n - tid + THREADS - 1) / THREADS : 0;
        in = reinterpret_cast<const uint4*>(x + cut.head) + lo + tid;
        if (rank == 0 && tid < cut.head + (a.vocab - tail)) end_at = tid < cut.head ? tid : tail + (tid - cut.head);
        const uint32_t group = (y - cut.head) / E::kVec - lo;
        owns_y = y >= cut.head && y < tail && group < n && group % THREADS == tid;
    }
};

// Set when a bounded wait below gave up; read by policy_kernel, read and cleared by rlcu_losses_check.  In host code this
// name is only a handle for cudaMemcpyFromSymbol.
static __device__ unsigned int losses_error_word;
constexpr uint32_t kWaitTries = 1u << 18;

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// bounded wait for a phase of an mbarrier of this CTA
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t phase, uint32_t tries = kWaitTries) {
    uint32_t done = 0;
    for (uint32_t i = 0; i < tries && !done; i++)
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(done) : "r"(bar), "r"(phase) : "memory");
    return done;
}

// A wait that gave up says so and is taken up again, once: what is on its way to this CTA should not arrive after it has
// left.  False: it has not arrived in that time either.
__device__ __forceinline__ bool wait_or_say(uint32_t bar, uint32_t phase, uint32_t tries) {
    if (wait_phase(bar, phase, tries)) return true;
    atomicExch(&losses_error_word, 1u);
    return wait_phase(bar, phase);
}

// Sums of all threads of a cluster, in warp 0 of each of its CTAs.  The CTAs hand each other their sums with st.async,
// whose arrival the receiver's mbarrier counts in bytes: unlike a cluster barrier with release semantics this does not
// wait for the gradient stores that are still on their way (an earlier form of the policy kernel took 667 us with the
// barrier and 629 us with this, 4096 x 151936 bf16).
template <int WARPS>
struct ClusterSum {
    float2 part[2][kMostCluster * WARPS];  // (e, s) of each warp of the cluster, by exchange parity: a CTA may be one ahead
    uint2 next[2];                         // what warp 0 of the first CTA passes on
    unsigned long long bar[2];

    __device__ __forceinline__ void init(uint32_t C) {
        if (C == 1) return;
        if (threadIdx.x == 0) {
            for (int i = 0; i < 2; i++)
                asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(smem_at(&bar[i])) : "memory");
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        cluster_barrier();
    }
    // a CTA leaves when no other one of its cluster can still write to it
    __device__ __forceinline__ void finish(uint32_t C) {
        if (C > 1) cluster_barrier();
    }
    // (not .aligned: the threads of a warp come from different branches)
    static __device__ __forceinline__ void cluster_barrier() {
        asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    }
    // every warp, exchange n (counted from 0): hands what it has of the sum to warp 0 of every CTA
    template <typename Sum>
    __device__ __forceinline__ void give(Sum o, uint2 pass_on, uint32_t n, uint32_t rank, uint32_t C) {
        const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, parity = n & 1;
        o.merge_warp();
        if (C == 1) {
            if (lane == 0) part[parity][warp] = make_float2(o.e, o.s);
            if (threadIdx.x == 0) next[parity] = pass_on;
            return;
        }
        const uint32_t here = smem_at(&bar[parity]);
        if (threadIdx.x == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(here), "r"(C * WARPS * 8u + 8u) : "memory");
        if (lane < C) {
            uint32_t to, to_bar;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_at(&part[parity][rank * WARPS + warp])), "r"(lane));
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to_bar) : "r"(here), "r"(lane));
            asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];"
                         :: "r"(to), "f"(o.e), "f"(o.s), "r"(to_bar) : "memory");
            if (rank == 0 && warp == 0) {
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_at(&next[parity])), "r"(lane));
                asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.u32 [%0], {%1, %2}, [%3];"
                             :: "r"(to), "r"(pass_on.x), "r"(pass_on.y), "r"(to_bar) : "memory");
            }
        }
    }
    // warp 0 (C = 1: behind a barrier with all that give): the sum over the cluster
    template <typename Sum>
    __device__ __forceinline__ Sum take(float c, uint32_t n, uint32_t C, uint32_t tries) {
        const uint32_t lane = threadIdx.x & 31, parity = n & 1, phase = (n >> 1) & 1;
        const bool done = C == 1 || __all_sync(0xFFFFFFFFu, wait_or_say(smem_at(&bar[parity]), phase, tries));
        Sum o(c);
        if (!done) {                                         // no more rows for this CTA
            if (lane == 0) next[parity] = make_uint2(0xFFFFFFFFu, 0u);
            o.s = NAN;
        } else {
            for (uint32_t i = lane; i < C * WARPS; i += 32) o.merge(part[parity][i].x, part[parity][i].y);
        }
        __syncwarp();
        o.merge_warp();
        return o;
    }
};

// The rows of a grid with one cluster per row, for clusters that stay: instead of leaving, a cluster takes over the
// next one that has not been launched.  So rows are worked on in order, by whoever is free, and the addresses in use
// stay close together: DRAM moves a copy of this shape in 338 us that way and in 394 us when each cluster takes every
// n-th row and they drift apart.  One thread of the cluster asks.
struct RowFeed {
    ulonglong2 response;
    unsigned long long bar;

    __device__ __forceinline__ void init() {
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(smem_at(&bar)) : "memory");
    }
    __device__ __forceinline__ void ask() {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the last response has been read
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], 16;" :: "r"(smem_at(&bar)) : "memory");
        asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                     :: "r"(smem_at(&response)), "r"(smem_at(&bar)) : "memory");
    }
    // first CTA of the cluster taken over by request n (counted from 0), or -1: none was left
    __device__ __forceinline__ int answer(uint32_t n, uint32_t tries) {
        if (!wait_or_say(smem_at(&bar), n & 1, tries)) return -1;
        unsigned long long lo, hi;
        int first;
        asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(lo), "=l"(hi) : "r"(smem_at(&response)) : "memory");
        asm volatile(
            "{\n"
            ".reg .b128 h;\n"
            ".reg .pred p;\n"
            "mov.b128 h, {%1, %2};\n"
            "mov.b32 %0, -1;\n"
            "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
            "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n"
            "}\n"
            : "=r"(first) : "l"(lo), "l"(hi) : "memory");
        return first;
    }
};

// The policy loss of most calls.  A row belongs to a cluster of C CTAs, each of which has a run of its 16-byte groups
// and keeps it in registers between the sum and the gradient: the logits are read once, the gradient is written once.
// Several clusters share an SM (four CTAs of 256 threads with up to ten groups each: 160 KB of its registers), so that
// one row's loads and stores run under another's arithmetic.
// Measured (B200, a tenth of the rows without part): 4096 x 151936 bf16 457 to 469 us on different GPUs, 0.79 to 0.77 of the
// copy rate (6.55 TB/s) for the bytes it cannot do without; 1000 x 151936 f32, all with part, 217 to 223 us, 0.86 to 0.83.
// (With ten groups of a 16-bit type a thread keeps 8 bytes in local memory.)  A row takes a CTA about 14,500 cycles: 3,500
// until its loads are there, 3,000 for the sum, 3,000 to 4,500 to exchange it, 1,100 for the row's factors, 2,000 for the
// gradient; with four CTAs per SM the special-function units and the issue slots are each a little over half busy.  The same
// kernel without any arithmetic takes 421 us, a plain copy of the same bytes 335 us.  Fetching the next row ahead (into L2,
// into shared memory by cp.async or by a bulk copy), a second row in the same loop, and five or six CTAs per SM with part of
// the row in shared memory were all slower (453 to 720 us; L2 prefetch gained 2 % here and lost 20 % for f32).
template <uint32_t DT, int THREADS, int NV>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
logits_policy_kernel(LogitsArgs a, PolicyArgs p) {
    using E = Elem<DT>;
    using T = typename E::T;
    __shared__ ClusterSum<THREADS / 32> sums;
    __shared__ RowFeed feed;
    __shared__ float inputs[8];
    __shared__ float4 answer;                         // e, -k / s, k (1 - p_y), 0 for a row to be looked at again
    const uint32_t C = cooperative_groups::this_cluster().num_blocks(), rank = cooperative_groups::this_cluster().block_rank();
    const int tid = threadIdx.x;
    const bool asks = rank == 0 && tid == 0;
    const float c = a.inv_temperature * kLog2E;
    if (asks) feed.init();
    sums.init(C);
    uint32_t row = blockIdx.x / C;
    uint32_t y = row_takes_part(a, p, row, a.targets[row]) ? (uint32_t)a.targets[row] : kNoTarget;
    for (uint32_t n = 0; n < a.rows; n++) {          // (ends at the break; the bound holds whatever the feed answers)
        if (asks) feed.ask();
        const RowShare<DT, THREADS> now(a, row, y, rank, C);
        T* g = static_cast<T*>(a.grad) + (uint64_t)row * a.grad_stride;
        uint4 v[NV];
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (j < (int)now.groups) v[j] = __ldcs(now.in + j * THREADS);
        float end = 0.0f, input = 0.0f;
        if (now.end_at < a.vocab) end = E::up(now.x[now.end_at]);
        if (y < a.vocab) {
            if (tid == 32) input = E::up(now.x[y]);
            if (tid == 33) input = p.advantage[row];
            if (tid == 34) input = p.weight[row];
            if (tid == 35 && p.old_logp) input = p.old_logp[row];
            if (tid == 36 && p.hp.kl_coef != 0.0f) input = p.ref_logp[row];
        } else {
            zero_row<DT>(a.grad, (uint64_t)row * a.grad_stride, a.vocab, rank * THREADS + tid, C * THREADS);
        }
        Online o(c);
        uint2 next = make_uint2(0xFFFFFFFFu, kNoTarget);
        float next_weight = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (j < (int)now.groups) o.add<DT>(v[j], c);
            if (j == 0 && asks) {
                const int first = feed.answer(n, a.tries);
                if (first >= 0) {
                    next.x = (uint32_t)first / C;
                    next.y = (uint32_t)a.targets[next.x];
                    next_weight = p.weight[next.x];
                }
            }
        }
        if (asks && next_weight == 0.0f) next.y = kNoTarget;
        if (now.end_at < a.vocab) o.add(end, c);
        if (tid >= 32 && tid < 37) inputs[tid - 32] = input;
        if (tid < 32) {
            next.x = __shfl_sync(0xFFFFFFFFu, next.x, 0);
            next.y = __shfl_sync(0xFFFFFFFFu, next.y, 0);
        }
        sums.give(o, next, n, rank, C);
        __syncthreads();
        if (tid < 32) {
            o = sums.template take<Online>(c, n, C, a.tries);
            if (tid == 0 && y < a.vocab) {
                const RowAnswer r = row_answer<true>(o, inputs[0], c);
                const bool again = fabsf(o.e) >= kExact || o.says_nothing();
                if (rank == 0) a.logp[row] = again ? __uint_as_float(kLookAgain) : r.logp;
                const float S = a.scaler ? a.scaler->scale : 1.0f;
                const float k = policy_term(p, r.logp, inputs[1], inputs[2], inputs[3], inputs[4]).coef * S * a.inv_temperature;
                answer = make_float4(r.e, -k * r.inv, -k * expm1f(r.logp), again ? 0.0f : c);
            } else if (asks) {
                a.logp[row] = 0.0f;
            }
        }
        __syncthreads();
        const float e = answer.x, kn = answer.y, ky = answer.z;
        if (answer.w != 0.0f) {                       // (0: the row is left to the kernel behind this one)
            // the gradient's groups lie where the logits' do
            uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(now.in) + reinterpret_cast<uintptr_t>(g) -
                                                  reinterpret_cast<uintptr_t>(now.x));
#pragma unroll
            for (int j = 0; j < NV; j++) {
                // the packed group is what stays in registers, not what the sum unpacked from it
                asm volatile("" : "+r"(v[j].x), "+r"(v[j].y), "+r"(v[j].z), "+r"(v[j].w));
                if (j < (int)now.groups) __stcs(out + j * THREADS, grad_group<DT>(v[j], c, e, kn));
            }
            if (now.end_at < a.vocab) g[now.end_at] = E::down(now.end_at == y ? ky : kn * exp2_fast(fmaf(end, c, -e)));
            if (now.owns_y) g[y] = E::down(ky);           // behind this thread's own store of the group
        }
        row = sums.next[n & 1].x;
        y = sums.next[n & 1].y;
        if (row >= a.rows) break;
    }
    sums.finish(C);
}

// Log-probabilities alone: a cluster (one CTA, unless rows are few) per row, kDepth groups per thread on their way in
// registers.  Bound by HBM: 2048 x 151936 bf16 95 to 102 us on different GPUs, 0.90 to 0.84 of the copy rate; on one of them
// 97, with the groups on their way by cp.async through shared memory 106, with CTAs that stay and take over rows 110.
constexpr int kDepth = 5;

template <uint32_t DT, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
logits_sum_kernel(LogitsArgs a, PolicyArgs p) {
    using E = Elem<DT>;
    __shared__ ClusterSum<THREADS / 32> sums;
    __shared__ float z_y;
    const uint32_t C = cooperative_groups::this_cluster().num_blocks(), rank = cooperative_groups::this_cluster().block_rank();
    const int tid = threadIdx.x;
    const float c = a.inv_temperature * kLog2E;
    const uint32_t row = blockIdx.x / C;
    const int32_t y = a.targets[row];
    if (!row_takes_part(a, p, row, y)) {              // (the whole cluster)
        if (rank == 0 && tid == 0) {
            a.logp[row] = 0.0f;
            if (a.lse) a.lse[row] = 0.0f;
        }
        return;
    }
    const RowShare<DT, THREADS> now(a, row, (uint32_t)y, rank, C);
    uint4 next[kDepth];
#pragma unroll
    for (int d = 0; d < kDepth; d++)
        if ((uint32_t)d < now.groups) next[d] = __ldcs(now.in + d * THREADS);
    float end = 0.0f;
    if (now.end_at < a.vocab) end = E::up(now.x[now.end_at]);
    if (tid == 32) z_y = E::up(now.x[y]);
    sums.init(C);
    Online o(c);
    const uint4* in = now.in + kDepth * THREADS;
    for (uint32_t j = 0; j < now.groups; j += kDepth) {
        uint4 v[kDepth];
#pragma unroll
        for (int d = 0; d < kDepth; d++) {
            v[d] = next[d];
            if (j + kDepth + d < now.groups) next[d] = __ldcs(in + d * THREADS);
        }
#pragma unroll
        for (int d = 0; d < kDepth; d++)
            if (j + d < now.groups) o.add<DT>(v[d], c);
        in += kDepth * THREADS;
    }
    if (now.end_at < a.vocab) o.add(end, c);
    sums.give(o, make_uint2(0u, 0u), 0, rank, C);
    __syncthreads();
    if (tid < 32) {
        o = sums.template take<Online>(c, 0, C, a.tries);
        if (rank == 0) {
            RowAnswer r;
            if (__any_sync(0xFFFFFFFFu, o.says_nothing())) r = row_answer(top_by_warp<DT>(now.x, a.vocab), z_y, c, a.inv_temperature);
            else r = row_answer<false>(o, z_y, c);
            if (tid == 0) {
                a.logp[row] = r.logp;
                if (a.lse) a.lse[row] = r.lse;
            }
        }
    }
    sums.finish(C);
}

// The gradient alone (the sum is known): elementwise, a CTA per run of kGradGroups groups of a row, so that the grid
// moves through memory in order.  Bound by HBM: with the sum before it, 1000 x 50001 f32 95 to 97 us for 560 MB (the logits
// are read twice), 0.90 to 0.88 of the copy rate.
constexpr int kGradThreads = 256, kGradPer = 4, kGradGroups = kGradThreads * kGradPer;

template <uint32_t DT>
__global__ void __launch_bounds__(kGradThreads)
logits_grad_kernel(LogitsArgs a, const float* lse_in, const float* logp_in, const float* coef_in, uint32_t runs) {
    using E = Elem<DT>;
    using T = typename E::T;
    const uint32_t row = blockIdx.x / runs, run = blockIdx.x - row * runs;
    const uint32_t tid = threadIdx.x;
    const int32_t y = a.targets[row];
    const float coef = coef_in[row], lse = usable(lse_in[row]), S = a.scaler ? a.scaler->scale : 1.0f;
    const T* x = static_cast<const T*>(a.data) + (uint64_t)row * a.row_stride;
    T* g = static_cast<T*>(a.grad) + (uint64_t)row * a.grad_stride;
    const RowCut cut = cut_row(x, a.vocab);
    const uint32_t tail = cut.head + cut.groups * E::kVec, ends = cut.head + (a.vocab - tail);
    const uint32_t end_at = tid < cut.head ? tid : tail + (tid - cut.head);
    const bool has_end = run == 0 && tid < ends, takes = y >= 0 && (uint32_t)y < a.vocab && coef != 0.0f;
    const uint4* in = reinterpret_cast<const uint4*>(x + cut.head);
    uint4* out = reinterpret_cast<uint4*>(g + cut.head);
    const uint32_t lo = run * kGradGroups + tid;
    if (!takes) {
#pragma unroll
        for (int j = 0; j < kGradPer; j++)
            if (lo + j * kGradThreads < cut.groups) __stcs(out + lo + j * kGradThreads, make_uint4(0u, 0u, 0u, 0u));
        if (has_end) g[end_at] = E::down(0.0f);
        return;
    }
    uint4 v[kGradPer];
#pragma unroll
    for (int j = 0; j < kGradPer; j++)
        if (lo + j * kGradThreads < cut.groups) v[j] = __ldcs(in + lo + j * kGradThreads);
    const float c = a.inv_temperature * kLog2E, k = coef * S * a.inv_temperature;
    // 2^(c z - log2e lse) = 2^(c z - e) * 2^(e - log2e lse), e an integer
    const bool empty = lse == -INFINITY;
    const float e = empty ? 0.0f : rintf(lse * kLog2E), kn = empty ? 0.0f * k : -k * exp2f(-fmaf(lse, kLog2E, -e));
    // the target's logit is read by the thread that overwrites it.  1 - p of a confident target comes from its
    // log-probability where that is given: lse has lost those digits.  (A NaN lse is one of the whole row.)
    const uint32_t group = ((uint32_t)y - cut.head) / E::kVec;
    const bool in_groups = (uint32_t)y >= cut.head && (uint32_t)y < tail;
    const bool owns_y = in_groups ? group / kGradGroups == run && group % kGradThreads == tid : has_end && end_at == (uint32_t)y;
    float ky = 0.0f;
    if (owns_y) ky = empty ? k : -k * expm1f(logp_in ? logp_in[row] + 0.0f * lse : fmaf(E::up(x[y]), a.inv_temperature, -lse));
    if (has_end) g[end_at] = E::down(kn * exp2_fast(fmaf(E::up(x[end_at]), c, -e)));
#pragma unroll
    for (int j = 0; j < kGradPer; j++)
        if (lo + j * kGradThreads < cut.groups) __stcs(out + lo + j * kGradThreads, grad_group<DT>(v[j], c, e, kn));
    if (owns_y) g[y] = E::down(ky);
}

// ---------------------------------------------------------------------------
// policy loss of log-probabilities
// ---------------------------------------------------------------------------

constexpr int kVectorThreads = 1024;

// A CTA may store into the shared memory of another one of its cluster only when that one has started: every thread says
// so first thing in a kernel, and waits for all others before the first such store.
__device__ __forceinline__ void cluster_started() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void wait_cluster_started() { asm volatile("barrier.cluster.wait;" ::: "memory"); }

// What a part of the tokens makes of the record.
struct PolicySums {
    double l = 0.0, k = 0.0, w = 0.0;
    uint32_t tokens = 0, clipped = 0;
    float ratio = 0.0f;

    __device__ __forceinline__ void add_warp() {
#pragma unroll
        for (int mask = 16; mask >= 1; mask >>= 1) {
            l += __shfl_xor_sync(0xFFFFFFFFu, l, mask);
            k += __shfl_xor_sync(0xFFFFFFFFu, k, mask);
            w += __shfl_xor_sync(0xFFFFFFFFu, w, mask);
            ratio = fmaxf(ratio, __shfl_xor_sync(0xFFFFFFFFu, ratio, mask));
        }
        tokens = __reduce_add_sync(0xFFFFFFFFu, tokens);
        clipped = __reduce_add_sync(0xFFFFFFFFu, clipped);
    }
};

// A row that logits_policy_kernel has marked, by the whole CTA: log-probability and gradient.  It happens to rows of nothing
// but masks and to logits beyond 2^31, so it is written to be short; in the kernel that marks it, it cost registers and with
// them 7 to 14 % of every call.
template <uint32_t DT>
__device__ __noinline__ void look_again(const LogitsArgs& a, const PolicyArgs& p, uint64_t row) {
    using E = Elem<DT>;
    using T = typename E::T;
    __shared__ float2 parts[kVectorThreads / 32];
    __shared__ RowAnswer answer;
    const T* x = static_cast<const T*>(a.data) + row * a.row_stride;
    T* g = static_cast<T*>(a.grad) + row * a.grad_stride;
    const uint32_t y = (uint32_t)a.targets[row];
    const float c = a.inv_temperature * kLog2E;
    Online o(c);
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kVectorThreads) o.add(E::up(x[i]), c);
    o = add_in_block(o, parts, c);
    if (o.says_nothing()) {
        __syncthreads();
        Top top;
        for (uint32_t i = threadIdx.x; i < a.vocab; i += kVectorThreads) top.add(E::up(x[i]));
        top = add_in_block(top, parts, c);
        if (threadIdx.x == 0) answer = row_answer(top, E::up(x[y]), c, a.inv_temperature);
    } else if (threadIdx.x == 0) {
        answer = row_answer<false>(o, E::up(x[y]), c);
    }
    __syncthreads();
    const RowAnswer r = answer;
    const float k = policy_term(p, r.logp, row).coef * (a.scaler ? a.scaler->scale : 1.0f) * a.inv_temperature;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kVectorThreads)
        g[i] = E::down(i == y ? -k * expm1f(r.logp) : -k * r.inv * exp2_fast(fmaf(E::up(x[i]), r.by, -r.e)));
    if (threadIdx.x == 0) a.logp[row] = r.logp;
    __syncthreads();
}

// log-probability and first gradient of a row as NaN
__device__ __forceinline__ void spoil(const LogitsArgs& a, uint32_t dtype, uint64_t row) {
    a.logp[row] = NAN;
    if (!a.grad) return;
    const uint64_t at = row * a.grad_stride;
    if (dtype == RLCU_F32) static_cast<float*>(a.grad)[at] = NAN;
    else static_cast<uint16_t*>(a.grad)[at] = 0x7FFFu;           // (in both 16-bit types)
}

// Weighted sums of the policy loss over all tokens, and the gradient by log-probability.  `a` (with targets): tokens whose
// target is out of range take no part; rows marked by logits_policy_kernel are done first; and after a wait of that kernel
// has given up, when rows may have been left out, nothing of the call is left that looks like a result.  One cluster: its
// CTAs hand their sums to the first one, so the record needs no scratch memory and no second launch.  Bound by latency:
// 16384 tokens 4.7 us in a graph.
__global__ void __launch_bounds__(kVectorThreads)
policy_kernel(const float* logp, uint64_t tokens, const __grid_constant__ LogitsArgs a, uint32_t dtype,
              const __grid_constant__ PolicyArgs p, float* coef, rlcu_policy_stat* stat, uint32_t flags) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ PolicySums warps[kVectorThreads / 32], ctas[kMostCluster];
    const uint32_t C = cluster.num_blocks(), rank = cluster.block_rank();
    cluster_started();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const bool gave_up = a.targets && *const_cast<const volatile unsigned int*>(&losses_error_word);
sums:
    PolicySums mine;
    bool marked = false;                              // a row that logits_policy_kernel has left is among the CTA's
    for (uint64_t t = rank * kVectorThreads + threadIdx.x; t < tokens; t += C * kVectorThreads) {
        const float w = p.weight[t];
        const bool takes = w != 0.0f && (!a.targets || (a.targets[t] >= 0 && (uint32_t)a.targets[t] < a.vocab));
        float co = 0.0f;
        if (takes) {
            const float lp = logp[t];
            if (a.grad) marked |= __float_as_uint(lp) == kLookAgain;
            const PolicyTerm o = policy_term(p, lp, t);
            mine.l += (double)w * o.l;
            mine.k += (double)w * o.k;
            mine.w += w;
            mine.tokens++;
            mine.clipped += o.cut;
            mine.ratio = fmaxf(mine.ratio, o.ratio);
            co = o.coef;
        }
        if (coef) coef[t] = co;
    }
    mine.add_warp();
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = mine;
    if (__syncthreads_or(marked || gave_up)) {
        if (__syncthreads_or(gave_up)) {
            for (uint64_t t = rank * kVectorThreads + threadIdx.x; t < tokens; t += C * kVectorThreads) spoil(a, dtype, t);
            if (threadIdx.x == 0) warps[0].l = warps[0].w = NAN;
            __syncthreads();
        } else {
            for (uint64_t base = rank * kVectorThreads; base < tokens; base += C * kVectorThreads)
                for (uint64_t t = base; t < tokens && t < base + kVectorThreads; t++) {
                    if (__float_as_uint(logp[t]) != kLookAgain) continue;       // (one thread changes it, behind a barrier)
                    if (dtype == RLCU_F16) look_again<RLCU_F16>(a, p, t);
                    else if (dtype == RLCU_BF16) look_again<RLCU_BF16>(a, p, t);
                    else look_again<RLCU_F32>(a, p, t);
                }
            goto sums;
        }
    }
    wait_cluster_started();
    if (threadIdx.x < 32) {
        mine = warps[threadIdx.x];
        mine.add_warp();
        if (threadIdx.x == 0) *cluster.map_shared_rank(&ctas[rank], 0) = mine;
    }
    cluster.sync();
    if (rank != 0 || threadIdx.x >= 32) return;
    mine = threadIdx.x < C ? ctas[threadIdx.x] : PolicySums();
    mine.add_warp();
    if (threadIdx.x == 0) {
        rlcu_policy_stat r = {};
        if (flags & RLCU_LOSS_ACCUMULATE) r = *stat;
        const double kl = p.hp.kl_coef != 0.0f ? (double)p.hp.kl_coef * mine.k : 0.0;
        r.loss = (float)((double)r.loss + mine.l + kl);
        r.policy = (float)((double)r.policy + mine.l);
        r.kl = (float)((double)r.kl + mine.k);
        r.weight = (float)((double)r.weight + mine.w);
        r.tokens += mine.tokens;
        r.clipped += mine.clipped;
        r.ratio_max = fmaxf(r.ratio_max, mine.ratio);
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
        loss = (1.0 - e) * (fmax(-h, 0.0) + tail);
        if (e > 0.0) loss += e * (fmax(h, 0.0) + tail);                // (not 0 times an infinite h)
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

// One cluster, so that the record needs no scratch memory and no second launch.  CTA r has the pairs r, r + C, ... and
// works on kBatch of them at a time, whatever their lengths: their tokens are cut into at most kSegments segments of
// equal length, a warp sums a segment, and the segments of a sequence are added in order.  Bound by latency, that of
// loads of 4 bytes a lane and of five barriers of 1024 threads per batch: 128 pairs of 2048 tokens 16 us (a CTA per pair in
// turn: 706 us; 16 SMs could read them in 2 to 3), one pair of 200 7 us in a graph.
constexpr int kBatch = 16, kSegments = 512;

__global__ void __launch_bounds__(kVectorThreads)
preference_kernel(PreferenceArgs a) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    constexpr int kWarps = kVectorThreads / 32;
    __shared__ uint32_t begin[2 * kBatch], length[2 * kBatch], first_segment[2 * kBatch + 1], segment;
    __shared__ double part[kSegments + 2 * kBatch], sums[2 * kBatch];
    __shared__ uint32_t counted[kSegments + 2 * kBatch], counts[2 * kBatch];
    __shared__ float coefs[2 * kBatch];
    __shared__ double totals[kMostCluster][2];
    __shared__ uint32_t corrects[kMostCluster];
    const uint32_t C = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    cluster_started();
    double loss_sum = 0.0, margin_sum = 0.0;          // of threads 0 to kBatch - 1
    uint32_t correct = 0;

    for (uint64_t base = 0; base * C + rank < a.pairs; base += kBatch) {
        if (warp == 0) {
            // lane q: sequence q of the batch
            static_assert(2 * kBatch == 32, "a lane per sequence");
            const uint64_t pair = (base + lane / 2) * C + rank;
            uint32_t lo = 0, n = 0;
            if (pair < a.pairs) {
                const uint64_t chosen = offset_at(a, 2 * pair), rejected = max(chosen, offset_at(a, 2 * pair + 1));
                const uint64_t behind = max(rejected, offset_at(a, 2 * pair + 2));
                lo = (uint32_t)(lane & 1 ? rejected : chosen);
                n = (uint32_t)(lane & 1 ? behind : rejected) - lo;
            }
            unsigned long long all = n;
#pragma unroll
            for (int mask = 16; mask >= 1; mask >>= 1) all += __shfl_xor_sync(0xFFFFFFFFu, all, mask);
            const uint32_t seg = max(256u, (uint32_t)((all + kSegments - 1) / kSegments));
            uint32_t before = (n + seg - 1) / seg;
            const uint32_t own = before;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t left = __shfl_up_sync(0xFFFFFFFFu, before, d);
                if ((int)lane >= d) before += left;
            }
            begin[lane] = lo;
            length[lane] = n;
            first_segment[lane] = before - own;
            if (lane == 31) first_segment[32] = before;
            if (lane == 0) segment = seg;
        }
        __syncthreads();
        const uint32_t segments = first_segment[2 * kBatch], seg = segment;
        for (uint32_t s = warp; s < segments; s += kWarps) {
            const uint32_t q = 31 - __clz(__ballot_sync(0xFFFFFFFFu, first_segment[lane] <= s));      // last sequence that begins by s
            const uint32_t at = (s - first_segment[q]) * seg, hi = min(at + seg, length[q]);
            const uint32_t t0 = begin[q];
            double sum = 0.0;
            uint32_t n = 0;
#pragma unroll 8
            for (uint32_t t = at + lane; t < hi; t += 32) {
                const float ref = a.ref_logp ? a.ref_logp[t0 + t] : 0.0f, lp = a.logp[t0 + t];
                const bool counts_here = !a.mask || a.mask[t0 + t];
                if (counts_here) {
                    sum += (double)(lp - ref);
                    n++;
                }
            }
#pragma unroll
            for (int mask = 16; mask >= 1; mask >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, mask);
            n = __reduce_add_sync(0xFFFFFFFFu, n);
            if (lane == 0) {
                part[s] = sum;
                counted[s] = n;
            }
        }
        __syncthreads();
        for (uint32_t q = warp; q < 2 * kBatch; q += kWarps) {
            double sum = 0.0;
            uint32_t n = 0;
            for (uint32_t s = first_segment[q] + lane; s < first_segment[q + 1]; s += 32) {
                sum += part[s];
                n += counted[s];
            }
#pragma unroll
            for (int mask = 16; mask >= 1; mask >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, mask);
            n = __reduce_add_sync(0xFFFFFFFFu, n);
            if (lane == 0) {
                sums[q] = sum;
                counts[q] = n;
            }
        }
        __syncthreads();
        const uint64_t pair = (base + tid) * C + rank;
        if (tid < kBatch && pair < a.pairs) {
            double s[2], share[2];
            for (int q = 0; q < 2; q++) {
                share[q] = a.hp.length_mean ? (counts[2 * tid + q] ? 1.0 / counts[2 * tid + q] : 0.0) : 1.0;
                s[q] = sums[2 * tid + q] * share[q];
            }
            double h, loss, slope;
            preference_term(a.hp, s[0], s[1], h, loss, slope);
            const double w = a.pair_weight ? (double)a.pair_weight[pair] : 1.0 / (double)a.pairs;
            if (w != 0.0) {                           // (not 0 times an infinite margin or NaN)
                loss_sum += w * loss;
                margin_sum += w * h;
            }
            correct += s[0] > s[1];
            for (int q = 0; q < 2; q++) {
                if (a.rewards) a.rewards[2 * pair + q] = (float)((double)a.hp.beta * s[q]);
                coefs[2 * tid + q] = w != 0.0 ? (float)((q ? -slope : slope) * w * share[q]) : 0.0f;
            }
        }
        __syncthreads();
        if (a.coef)
            for (uint32_t s = warp; s < segments; s += kWarps) {
                const uint32_t q = 31 - __clz(__ballot_sync(0xFFFFFFFFu, first_segment[lane] <= s));
                const uint32_t at = (s - first_segment[q]) * seg, hi = min(at + seg, length[q]);
                const uint32_t t0 = begin[q];
                const float co = coefs[q];
#pragma unroll 8
                for (uint32_t t = at + lane; t < hi; t += 32) a.coef[t0 + t] = !a.mask || a.mask[t0 + t] ? co : 0.0f;
            }
        __syncthreads();                              // the batch's tables are written again
    }
    if (a.coef) {
        // tokens of no sequence
        const uint64_t first = offset_at(a, 0);
        uint64_t behind = first;
        if (a.pairs) behind = max(max(offset_at(a, 2 * a.pairs - 2), offset_at(a, 2 * a.pairs - 1)), offset_at(a, 2 * a.pairs));
        for (uint64_t t = rank * kVectorThreads + tid; t < first; t += C * kVectorThreads) a.coef[t] = 0.0f;
        for (uint64_t t = behind + rank * kVectorThreads + tid; t < a.tokens; t += C * kVectorThreads) a.coef[t] = 0.0f;
    }
    wait_cluster_started();
    if (warp == 0) {
#pragma unroll
        for (int mask = 16; mask >= 1; mask >>= 1) {
            loss_sum += __shfl_xor_sync(0xFFFFFFFFu, loss_sum, mask);
            margin_sum += __shfl_xor_sync(0xFFFFFFFFu, margin_sum, mask);
        }
        correct = __reduce_add_sync(0xFFFFFFFFu, correct);
        if (lane == 0) {
            *cluster.map_shared_rank(&totals[rank][0], 0) = loss_sum;
            *cluster.map_shared_rank(&totals[rank][1], 0) = margin_sum;
            *cluster.map_shared_rank(&corrects[rank], 0) = correct;
        }
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
        rlcu_preference_stat r = {};
        if (a.flags & RLCU_LOSS_ACCUMULATE) r = *a.stat;
        loss_sum = margin_sum = 0.0;
        correct = 0;
        for (uint32_t i = 0; i < C; i++) {
            loss_sum += totals[i][0];
            margin_sum += totals[i][1];
            correct += corrects[i];
        }
        r.loss = (float)((double)r.loss + loss_sum);
        r.margin = (float)((double)r.margin + margin_sum);
        r.pairs += (uint32_t)a.pairs;
        r.correct += correct;
        *a.stat = r;
    }
}

// Waits for a barrier that nothing completes, as the kernels above would, with few tries.
__global__ void wait_probe_kernel() {
    __shared__ unsigned long long bar;
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(smem_at(&bar)) : "memory");
    if (!wait_phase(smem_at(&bar), 0, 64)) atomicExch(&losses_error_word, 1u);
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
    if (rows_overlap({logits, vocab * esz, row_stride * esz}, {grad, vocab * esz, grad_stride * esz}, rows))
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

const char* const kUnaligned = "a vector of 4-byte values is not aligned to them";

// `out` (n FP32 values) shares none of its bytes with the inputs, or (with `same`) all of them
bool out_apart(const float* out, uint64_t n, std::initializer_list<const float*> inputs, bool same) {
    for (const float* in : inputs)
        if (out && in && !(same && in == out) && overlap(span_of(out, 1, n, n, 4), span_of(in, 1, n, n, 4))) return false;
    return true;
}

// a vector of 4-byte values
Span words(const void* p, uint64_t n) { return bytes_of(p, n * 4); }

std::atomic<uint32_t> wait_tries{kWaitTries};

int sm_count(int* out) {
    int dev = 0;
    RLCU_CUDA(cudaGetDevice(&dev));
    RLCU_CUDA(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev));
    return RLCU_OK;
}

template <int MODE>
int launch_rows(const LogitsArgs& a, const PolicyArgs& p, uint32_t dtype, const float* lse, const float* logp, const float* coef, cudaStream_t s) {
    int sms = 0;
    if (const int rc = sm_count(&sms)) return rc;
    const uint64_t most = (uint64_t)sms * 4;
    const int grid = (int)(a.rows < most ? a.rows : most);
    if (dtype == RLCU_F16) logits_row_kernel<RLCU_F16, MODE><<<grid, kRowThreads, 0, s>>>(a, p, lse, logp, coef);
    else if (dtype == RLCU_BF16) logits_row_kernel<RLCU_BF16, MODE><<<grid, kRowThreads, 0, s>>>(a, p, lse, logp, coef);
    else logits_row_kernel<RLCU_F32, MODE><<<grid, kRowThreads, 0, s>>>(a, p, lse, logp, coef);
    RLCU_CUDA(cudaGetLastError());
    return RLCU_OK;
}

// one cluster of `cluster` CTAs
cudaLaunchConfig_t cluster_launch(cudaLaunchAttribute* attr, int cluster, int threads, cudaStream_t s) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster);
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

template <typename Kernel>
int launch_clusters(Kernel kernel, const LogitsArgs& a, const PolicyArgs& p, int cluster, int threads, cudaStream_t s) {
    if (cluster > 8) RLCU_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = cluster_launch(attr, cluster, threads, s);
    cfg.gridDim = dim3((unsigned)(a.rows * cluster));
    RLCU_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, p));
    return RLCU_OK;
}

constexpr int kWide = 256, kNarrow = 128, kMostHeld = 10;

template <uint32_t DT, int THREADS>
int launch_policy_rows(const LogitsArgs& a, const PolicyArgs& p, int cluster, uint32_t held, cudaStream_t s) {
#define RLCU_HELD(NV) \
    if (held <= NV) return launch_clusters(logits_policy_kernel<DT, THREADS, NV>, a, p, cluster, THREADS, s)
    RLCU_HELD(2);
    RLCU_HELD(4);
    RLCU_HELD(6);
    RLCU_HELD(8);
    RLCU_HELD(10);
#undef RLCU_HELD
    return set_error(RLCU_ERR_UNSUPPORTED, "row too long");
}

template <uint32_t DT, int MODE>
int launch_logits_dt(const LogitsArgs& a, const PolicyArgs& p, int sms, uint64_t groups, cudaStream_t s) {
    // a row of up to kNarrow * kMostHeld groups fits one narrow CTA, and twice as many rows an SM
    const int threads = groups > (MODE == kModePolicy ? kNarrow * kMostHeld : 1024) ? kWide : kNarrow;
    int cluster = 1;
    if (MODE == kModePolicy)
        while (cluster < kMostCluster && groups > (uint64_t)cluster * threads * kMostHeld) cluster *= 2;
    // few rows: spread each over more SMs, as long as every thread keeps a group
    while (cluster < 8 && a.rows * cluster < (uint64_t)sms && groups > (uint64_t)cluster * threads) cluster *= 2;
    if (MODE == kModePolicy) {
        const uint32_t held = (uint32_t)(((groups + cluster - 1) / cluster + threads - 1) / threads);
        return threads == kWide ? launch_policy_rows<DT, kWide>(a, p, cluster, held, s) : launch_policy_rows<DT, kNarrow>(a, p, cluster, held, s);
    }
    return threads == kWide ? launch_clusters(logits_sum_kernel<DT, kWide>, a, p, cluster, kWide, s)
                          : launch_clusters(logits_sum_kernel<DT, kNarrow>, a, p, cluster, kNarrow, s);
}

// every row of the gradient starts at the same place of a 16-byte group as its logits do
bool alike(const LogitsArgs& a, size_t esz) {
    return ((reinterpret_cast<uintptr_t>(a.grad) ^ reinterpret_cast<uintptr_t>(a.data)) & 15) == 0 && (a.grad_stride - a.row_stride) * esz % 16 == 0;
}

template <int MODE>
int launch_logits(const LogitsArgs& a, const PolicyArgs& p, uint32_t dtype, cudaStream_t s) {
    int sms = 0;
    if (const int rc = sm_count(&sms)) return rc;
    const size_t esz = dtype_bytes(dtype);
    const uint64_t groups = a.vocab / (16 / esz);
    const bool fits = MODE != kModePolicy || groups <= (uint64_t)kMostCluster * kWide * kMostHeld;
    if ((MODE == kModePolicy && !alike(a, esz)) || !fits || groups < 64 || a.rows > 0x7FFFFFFFull / kMostCluster)
        return launch_rows<MODE>(a, p, dtype, nullptr, nullptr, nullptr, s);
    if (dtype == RLCU_F16) return launch_logits_dt<RLCU_F16, MODE>(a, p, sms, groups, s);
    if (dtype == RLCU_BF16) return launch_logits_dt<RLCU_BF16, MODE>(a, p, sms, groups, s);
    return launch_logits_dt<RLCU_F32, MODE>(a, p, sms, groups, s);
}

int launch_grad(const LogitsArgs& a, uint32_t dtype, const float* lse, const float* logp, const float* coef, cudaStream_t s) {
    const size_t esz = dtype_bytes(dtype);
    const uint64_t groups = a.vocab / (16 / esz), runs = (groups + kGradGroups - 1) / kGradGroups;
    if (!alike(a, esz) || groups < 64 || a.rows * runs > 0x7FFFFFFFull) return launch_rows<kModeGrad>(a, PolicyArgs{}, dtype, lse, logp, coef, s);
    const unsigned grid = (unsigned)(a.rows * runs);
    if (dtype == RLCU_F16) logits_grad_kernel<RLCU_F16><<<grid, kGradThreads, 0, s>>>(a, lse, logp, coef, (uint32_t)runs);
    else if (dtype == RLCU_BF16) logits_grad_kernel<RLCU_BF16><<<grid, kGradThreads, 0, s>>>(a, lse, logp, coef, (uint32_t)runs);
    else logits_grad_kernel<RLCU_F32><<<grid, kGradThreads, 0, s>>>(a, lse, logp, coef, (uint32_t)runs);
    RLCU_CUDA(cudaGetLastError());
    return RLCU_OK;
}

// behind: its launch is prepared while the call's own kernel before it still runs; it starts when that one's last CTA has
// left, since none of them triggers it sooner, and waits for what they wrote
int launch_policy(const float* logp, uint64_t tokens, const LogitsArgs& a, uint32_t dtype, const PolicyArgs& p, float* coef,
                  rlcu_policy_stat* stat, uint32_t flags, bool behind, cudaStream_t s) {
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = cluster_launch(attr, tokens <= kVectorThreads ? 1 : tokens <= 4 * kVectorThreads ? 4 : 8, kVectorThreads, s);
    if (behind) {
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    RLCU_CUDA(cudaLaunchKernelEx(&cfg, policy_kernel, logp, tokens, a, dtype, p, coef, stat, flags));
    return RLCU_OK;
}

}  // namespace
}  // namespace rlcu

using namespace rlcu;

extern "C" int rlcu_token_logprob(const void* logits, uint32_t dtype, uint64_t rows, uint64_t vocab, uint64_t row_stride,
                                  float inv_temperature, const int32_t* targets, float* logp, float* lse, void* stream) {
    if (const int rc = check_logits(logits, dtype, rows, vocab, row_stride, inv_temperature, targets)) return rc;
    if (rows && !logp) return set_error(RLCU_ERR_INVALID, "null logp");
    if (!words_aligned({targets, logp, lse})) return set_error(RLCU_ERR_INVALID, "%s", kUnaligned);
    if (!rows) return RLCU_OK;
    for (const float* out : {logp, lse})
        if (overlaps_any(words(out, rows), {words(targets, rows), words(out == logp ? lse : logp, rows)}) ||
            overlaps_rows(words(out, rows), logits, rows, vocab, row_stride, dtype_bytes(dtype)))
            return set_error(RLCU_ERR_INVALID, "logp or lse overlaps another buffer of the call");
    LogitsArgs a = {logits, rows, row_stride, (uint32_t)vocab, inv_temperature, targets, logp, lse, nullptr, 0, nullptr, wait_tries};
    return launch_logits<kModeLogprob>(a, PolicyArgs{}, dtype, (cudaStream_t)stream);
}

extern "C" int rlcu_token_logprob_grad_logp(const void* logits, uint32_t dtype, uint64_t rows, uint64_t vocab,
                                            uint64_t row_stride, float inv_temperature, const int32_t* targets,
                                            const float* lse, const float* logp, const float* coef,
                                            const rlcu_scaler_state* scaler, void* grad, uint64_t grad_stride, void* stream) {
    if (const int rc = check_logits(logits, dtype, rows, vocab, row_stride, inv_temperature, targets)) return rc;
    if (const int rc = check_grad(logits, dtype, rows, vocab, row_stride, grad, grad_stride)) return rc;
    if (rows && (!lse || !coef)) return set_error(RLCU_ERR_INVALID, "null lse or coef");
    if (!words_aligned({targets, lse, logp, coef, scaler})) return set_error(RLCU_ERR_INVALID, "%s", kUnaligned);
    if (!rows) return RLCU_OK;
    for (const Span& in : {words(targets, rows), words(lse, rows), words(logp, rows), words(coef, rows), bytes_of(scaler, sizeof *scaler)})
        if (overlaps_rows(in, grad, rows, vocab, grad_stride, dtype_bytes(dtype)))
            return set_error(RLCU_ERR_INVALID, "gradient overlaps a vector that the call reads");
    LogitsArgs a = {logits, rows, row_stride, (uint32_t)vocab, inv_temperature, targets, nullptr, nullptr, grad, grad_stride, scaler, wait_tries};
    return launch_grad(a, dtype, lse, logp, coef, (cudaStream_t)stream);
}

extern "C" int rlcu_token_logprob_grad(const void* logits, uint32_t dtype, uint64_t rows, uint64_t vocab,
                                       uint64_t row_stride, float inv_temperature, const int32_t* targets,
                                       const float* lse, const float* coef, const rlcu_scaler_state* scaler, void* grad,
                                       uint64_t grad_stride, void* stream) {
    return rlcu_token_logprob_grad_logp(logits, dtype, rows, vocab, row_stride, inv_temperature, targets, lse, nullptr, coef, scaler, grad,
                                        grad_stride, stream);
}

extern "C" int rlcu_policy_loss_logp(const float* logp, uint64_t tokens, const float* old_logp, const float* ref_logp,
                                     const float* advantage, const float* weight, const rlcu_policy_hparams* hp,
                                     float* coef, rlcu_policy_stat* stat, uint32_t flags, void* stream) {
    if (const int rc = check_policy(hp, ref_logp, advantage, weight, stat, tokens, flags)) return rc;
    if (tokens && !logp) return set_error(RLCU_ERR_INVALID, "null logp");
    if (!words_aligned({logp, old_logp, ref_logp, advantage, weight, coef})) return set_error(RLCU_ERR_INVALID, "%s", kUnaligned);
    if (!out_apart(coef, tokens, {logp, old_logp, ref_logp, advantage, weight}, true))
        return set_error(RLCU_ERR_INVALID, "coef overlaps an input without being the same buffer");
    if (overlaps_any(bytes_of(stat, sizeof *stat), {words(logp, tokens), words(old_logp, tokens), words(ref_logp, tokens),
                                                    words(advantage, tokens), words(weight, tokens), words(coef, tokens)}))
        return set_error(RLCU_ERR_INVALID, "the record overlaps a vector of the call");
    PolicyArgs p = {old_logp, ref_logp, advantage, weight, *hp};
    return launch_policy(logp, tokens, LogitsArgs{}, RLCU_F32, p, coef, stat, flags, false, (cudaStream_t)stream);
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
    if (!words_aligned({targets, old_logp, ref_logp, advantage, weight, logp, scaler})) return set_error(RLCU_ERR_INVALID, "%s", kUnaligned);
    // logp is written before the record is formed from the inputs
    if (!out_apart(logp, rows, {old_logp, ref_logp, advantage, weight}, false))
        return set_error(RLCU_ERR_INVALID, "logp overlaps another input of the loss");
    const size_t esz = dtype_bytes(dtype);
    const Span record = bytes_of(stat, sizeof *stat), out = words(logp, rows), scale = bytes_of(scaler, sizeof *scaler);
    if (overlaps_any(out, {words(targets, rows), scale, record}) || overlaps_rows(out, logits, rows, vocab, row_stride, esz))
        return set_error(RLCU_ERR_INVALID, "logp overlaps another buffer of the call");
    for (const Span& v : {words(targets, rows), words(old_logp, rows), words(ref_logp, rows), words(advantage, rows), words(weight, rows), scale, out})
        if (overlap(v, record) || (grad && overlaps_rows(v, grad, rows, vocab, grad_stride, esz)))
            return set_error(RLCU_ERR_INVALID, "gradient or record overlaps a vector of the call");
    if (overlaps_rows(record, logits, rows, vocab, row_stride, esz) || (grad && overlaps_rows(record, grad, rows, vocab, grad_stride, esz)))
        return set_error(RLCU_ERR_INVALID, "the record overlaps logits or gradient");
    LogitsArgs a = {logits, rows, row_stride, (uint32_t)vocab, inv_temperature, targets, logp, nullptr, grad, grad_stride, scaler, wait_tries};
    PolicyArgs p = {old_logp, ref_logp, advantage, weight, *hp};
    if (rows) {
        const int rc = grad ? launch_logits<kModePolicy>(a, p, dtype, (cudaStream_t)stream)
                            : launch_logits<kModeLogprob>(a, p, dtype, (cudaStream_t)stream);
        if (rc) return rc;
    }
    return launch_policy(logp, rows, a, dtype, p, nullptr, stat, flags, rows > 0, (cudaStream_t)stream);
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
    if (!words_aligned({logp, ref_logp, offsets, pair_weight, coef, rewards})) return set_error(RLCU_ERR_INVALID, "%s", kUnaligned);
    if (!out_apart(coef, tokens, {logp, ref_logp}, true)) return set_error(RLCU_ERR_INVALID, "coef overlaps an input without being the same buffer");
    const Span read = bytes_of(mask, tokens), starts = words(offsets, 2 * pairs + 1), weights = words(pair_weight, pairs);
    const Span record = bytes_of(stat, sizeof *stat), coefs = words(coef, tokens), reward = words(rewards, 2 * pairs);
    if (overlaps_any(coefs, {read, starts, weights, reward, record}) ||
        overlaps_any(reward, {words(logp, tokens), words(ref_logp, tokens), read, starts, weights, record}) ||
        overlaps_any(record, {words(logp, tokens), words(ref_logp, tokens), read, starts, weights}))
        return set_error(RLCU_ERR_INVALID, "coef, rewards or the record overlaps another buffer of the call");
    PreferenceArgs a = {logp, ref_logp, mask, offsets, pair_weight, tokens, pairs, *hp, coef, rewards, stat, flags};
    // more CTAs than pairs would idle; below a few thousand tokens each, the cluster costs more than it saves
    int cluster = 1;
    while (cluster < kMostCluster && (uint64_t)cluster < pairs && tokens > (uint64_t)cluster * 4096) cluster *= 2;
    if (cluster > 8) RLCU_CUDA(cudaFuncSetAttribute(preference_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = cluster_launch(attr, cluster, kVectorThreads, (cudaStream_t)stream);
    RLCU_CUDA(cudaLaunchKernelEx(&cfg, preference_kernel, a));
    return RLCU_OK;
}

extern "C" int rlcu_losses_check(void) {
    RLCU_CUDA(cudaDeviceSynchronize());
    unsigned int word = 0, none = 0;
    RLCU_CUDA(cudaMemcpyFromSymbol(&word, losses_error_word, sizeof word));
    if (!word) return RLCU_OK;
    RLCU_CUDA(cudaMemcpyToSymbol(losses_error_word, &none, sizeof none));
    return set_error(RLCU_ERR_TIMEOUT, "a bounded wait inside a loss kernel gave up: its results are incomplete");
}

extern "C" uint32_t rlcu_losses_selftest_tries(uint32_t tries) { return wait_tries.exchange(tries < kWaitTries ? tries : kWaitTries); }

extern "C" int rlcu_losses_selftest_wait(void* stream) {
    wait_probe_kernel<<<1, 1, 0, (cudaStream_t)stream>>>();
    RLCU_CUDA(cudaGetLastError());
    return rlcu_losses_check();
}
