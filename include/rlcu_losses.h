/*
 * rlcu_losses.h -- C ABI of the losses a training step starts its backward pass with, on B200 (sm_100a):
 * token log-probabilities of a block of logits, the clipped policy loss (GRPO / PPO) and the preference
 * loss (DPO), each with its gradient.  They stand where RL.cu has log_softmax_gather_kernel and its backward
 * (src/model/qwen3.cu:91-234), nll_loss_* (include/training/SFT_trainer.h:21-53) and grpo_loss_kernel
 * (include/training/GRPO_trainer.h:44-65).
 *
 * Conventions are those of rlcu_adamw.h: an int status, device pointers unless a parameter is documented as a
 * host pointer, `stream` a cudaStream_t as void*, no allocation and no synchronisation.  Calls keep no state
 * and no scratch of their own: calls on different buffers may overlap on the GPU, and every call can be
 * captured into a CUDA graph.  The same inputs give the same bits.
 *
 * Logits are `rows` rows of `vocab` values (F16, BF16 or F32), `row_stride` elements from row to row (0: vocab).
 * The loss is that of logits * inv_temperature (in (0, 1e6]).  Values between the rows are neither read nor written.
 * A row takes part when its target is in [0, vocab) (and, in the policy loss, its weight is not zero); of a row
 * that takes no part the logits are not read, its log-probability is 0 and its gradient row is written as
 * zeros.  Logits of -inf, and finite ones of -1e30 and below, are tokens of probability zero; a row with nothing else
 * has lse = logp = -inf and probabilities of zero.  (Other masks, -1e9 or -1e20, are logits like any other: a row of
 * nothing but one of them is uniform.)  NaN and +inf, and logits whose product with inv_temperature * log2 e is beyond
 * FP32, make their row's results NaN, which the statistics pass (rlcu_gradstat) then finds in the gradients.
 *
 * Gradients are those of the loss times scaler->scale (the loss scale the statistics pass later divides out;
 * no scaler: 1), rounded once to the logits' type.  A gradient buffer may be the logits' own
 * (same pointer, same stride).  What a call writes may share no other byte with what it reads or writes elsewhere, unless a
 * parameter says so; such calls are refused.
 */
#ifndef RLCU_LOSSES_H
#define RLCU_LOSSES_H

#include "rlcu_adamw.h"

#ifdef __cplusplus
extern "C" {
#endif

/* -------- token log-probabilities ---------------------------------------- */
/* logp[t] = log softmax(logits[t] * inv_temperature)[targets[t]], lse[t] = log sum exp (lse may be NULL; both
 * are 0 for a row that takes no part).  Old and reference log-probabilities of rollouts come from here, and
 * with rlcu_token_logprob_grad any loss of them. */
int rlcu_token_logprob(const void* logits, uint32_t dtype, uint64_t rows, uint64_t vocab, uint64_t row_stride,
                       float inv_temperature, const int32_t* targets, float* logp, float* lse, void* stream);
/* grad[t][j] = coef[t] * S * inv_temperature * ([j == targets[t]] - softmax_j), with coef[t] = dLoss/dlogp[t]
 * (coef = -1/tokens: the SFT loss of RL.cu) and S the loss scale; `lse` is what rlcu_token_logprob wrote for the
 * same logits.  A row with coef 0 takes no part.
 * FP32 holds lse to 2^-24 of itself, so probabilities taken from it are off by up to 2^-23 |lse| of themselves, and 1 - p
 * of the target by that much in absolute terms: with logits around 1e4, 1e-3, more than a confident target has.  A row
 * whose |lse| is above 2^24 has a gradient of NaN. */
int rlcu_token_logprob_grad(const void* logits, uint32_t dtype, uint64_t rows, uint64_t vocab, uint64_t row_stride,
                            float inv_temperature, const int32_t* targets, const float* lse, const float* coef,
                            const rlcu_scaler_state* scaler, void* grad, uint64_t grad_stride, void* stream);
/* The same with the log-probabilities that rlcu_token_logprob wrote beside lse (NULL: without): the target's 1 - p is
 * taken from them, right to a few 2^-24 of itself whatever lse. */
int rlcu_token_logprob_grad_logp(const void* logits, uint32_t dtype, uint64_t rows, uint64_t vocab, uint64_t row_stride,
                                 float inv_temperature, const int32_t* targets, const float* lse, const float* logp,
                                 const float* coef, const rlcu_scaler_state* scaler, void* grad, uint64_t grad_stride,
                                 void* stream);

/* -------- clipped policy loss --------------------------------------------- */
/* estimator of KL(policy || reference) per token, d = logp - ref_logp */
enum {
    RLCU_KL_K1 = 1,   /* d                     */
    RLCU_KL_K2 = 2,   /* d^2 / 2               */
    RLCU_KL_K3 = 3    /* exp(-d) + d - 1       */
};

/* ratio r = exp(logp - old_logp), advantage A:
 *   l = -min(r A, clamp(r, 1 - clip_low, 1 + clip_high) A)
 *   and, with dual_clip = c > 1, l = min(l, -c A) where A < 0 (0: off)
 *   loss = sum over tokens of weight * (l + kl_coef * k)                                                   */
typedef struct rlcu_policy_hparams {
    float    clip_low, clip_high;  /* >= 0, clip_low <= 1; +inf (clip_high) and 1 (clip_low) leave a side open */
    float    dual_clip;            /* 0 or > 1                                                               */
    float    kl_coef;              /* 0: no KL term, ref_logp is not read                                     */
    uint32_t kl_kind;              /* RLCU_KL_*                                                               */
} rlcu_policy_hparams;

/* Device memory, 32 bytes, 16-byte aligned. */
typedef struct rlcu_policy_stat {
    float    loss;        /* sum of weight * (l + kl_coef k), without the loss scale                          */
    float    policy;      /* sum of weight * l                                                                */
    float    kl;          /* sum of weight * k                                                                */
    float    weight;      /* sum of the weights of the tokens that take part                                  */
    uint32_t tokens;      /* tokens that take part                                                            */
    uint32_t clipped;     /* of them, those whose gradient a clip cut                                          */
    float    ratio_max;   /* largest r (0 without tokens)                                                      */
    uint32_t reserved;
} rlcu_policy_stat;

/* flags of the losses */
enum {
    RLCU_LOSS_ACCUMULATE = 1u  /* add to the record instead of overwriting it (micro-batches of one step)     */
};

/* The loss of `tokens` log-probabilities that are there already.
 *   advantage, weight : one per token (weight = mask / number of tokens: DAPO's normalisation, which RL.cu
 *                       uses; mask / (sequences * tokens of the sequence): GRPO's).  Weight 0: the token takes
 *                       no part and none of its other values matter.
 *   old_logp          : NULL: the policy that sampled is the one that is trained (r = 1, with its gradient)
 *   ref_logp          : NULL only with kl_coef 0
 *   coef              : dloss/dlogp per token, without the loss scale (rlcu_token_logprob_grad applies it);
 *                       0 for tokens that take no part; may be NULL, and may be the buffer of logp        */
int rlcu_policy_loss_logp(const float* logp, uint64_t tokens, const float* old_logp, const float* ref_logp,
                          const float* advantage, const float* weight, const rlcu_policy_hparams* hp /* host */,
                          float* coef, rlcu_policy_stat* stat, uint32_t flags, void* stream);
/* The loss of a block of logits and its gradient in one call: the logits are read from memory once and the
 * gradient is written once.  `logp` receives the log-probabilities and is a buffer of its own, not that of old_logp.
 * `grad` may be NULL: the loss alone. */
int rlcu_policy_loss(const void* logits, uint32_t dtype, uint64_t rows, uint64_t vocab, uint64_t row_stride,
                     float inv_temperature, const int32_t* targets, const float* old_logp, const float* ref_logp,
                     const float* advantage, const float* weight, const rlcu_policy_hparams* hp /* host */,
                     const rlcu_scaler_state* scaler, float* logp, void* grad, uint64_t grad_stride,
                     rlcu_policy_stat* stat, uint32_t flags, void* stream);

/* -------- preference loss -------------------------------------------------- */
enum {
    RLCU_PREF_SIGMOID = 0,  /* -(1 - e) log sigmoid(h) - e log sigmoid(-h), e = label_smoothing               */
    RLCU_PREF_HINGE = 1,    /* max(0, 1 - h)                                                                   */
    RLCU_PREF_IPO = 2       /* (h / beta - 1 / (2 beta))^2                                                     */
};

/* h = beta * (s_chosen - s_rejected) - margin, s the sum (length_mean: the mean) over a sequence's tokens of
 * logp - ref_logp */
typedef struct rlcu_preference_hparams {
    float    beta;             /* > 0                                                                          */
    float    margin;
    float    label_smoothing;  /* [0, 0.5], RLCU_PREF_SIGMOID only                                             */
    uint32_t kind;             /* RLCU_PREF_*                                                                  */
    uint32_t length_mean;      /* 0 or 1                                                                       */
} rlcu_preference_hparams;

/* Device memory, 32 bytes, 16-byte aligned. */
typedef struct rlcu_preference_stat {
    float    loss;        /* sum over pairs of weight * loss (weight 1/pairs where pair_weight is NULL)        */
    float    margin;      /* sum over pairs of weight * h                                                      */
    uint32_t pairs;
    uint32_t correct;     /* pairs with s_chosen > s_rejected                                                  */
    uint32_t reserved[4];
} rlcu_preference_stat;

/* `tokens` log-probabilities of packed sequences: sequence q has tokens [offsets[q], offsets[q+1]), pair i is
 * sequences 2i (chosen) and 2i + 1 (rejected).  offsets has 2*pairs + 1 entries that do not fall; entries
 * outside [0, tokens] are read as the nearer end.  A padded batch has its row starts in offsets and its padding
 * in the mask.
 *   ref_logp    : NULL: without a reference
 *   mask        : one byte per token, 0 takes no part (NULL: all do); what a masked place holds does not matter
 *   pair_weight : NULL: 1/pairs each.  A pair of weight 0 has no loss, no margin and a coef of 0, whatever its tokens hold
 *   coef        : dloss/dlogp, 0 for masked tokens and for tokens of no sequence; may be NULL, and may be the buffer of logp
 *   rewards     : beta * s of each sequence; may be NULL
 * A sequence without tokens has s = 0. */
int rlcu_preference_loss(const float* logp, uint64_t tokens, const float* ref_logp, const uint8_t* mask,
                         const int32_t* offsets, uint64_t pairs, const float* pair_weight,
                         const rlcu_preference_hparams* hp /* host */, float* coef, float* rewards,
                         rlcu_preference_stat* stat, uint32_t flags, void* stream);

/* -------- bounded waits ------------------------------------------------------ */
/* The CTAs that share a row of logits wait for one another, for a bounded time.  When such a wait gives up
 *   - rlcu_token_logprob: log-probability (and lse) of the rows concerned may be NaN;
 *   - rlcu_policy_loss: rows may have been left out.  All log-probabilities of the call, the first value of each row of its
 *     gradient (which rlcu_gradstat finds) and loss, policy and weight of its record are NaN; so are those of later
 *     calls of rlcu_policy_loss on the device until the condition is cleared.
 * Waits for every stream of the device (cudaDeviceSynchronize), reports whether a wait gave up since the last check
 * (RLCU_ERR_TIMEOUT) and clears the condition. */
int rlcu_losses_check(void);
/* Runs a one-thread kernel whose bounded wait is certain to run out and reports it through the same path: the
 * expected return value is RLCU_ERR_TIMEOUT, and the device stays usable. */
int rlcu_losses_selftest_wait(void* stream);
/* For tests: how often the waits of kernels launched later by this process try before they count as given up (they wait on
 * after that, so that nothing is left on its way; the results are spoilt all the same).  0: at once.  More than the
 * number they start with counts as that number.  Returns the number that held before. */
uint32_t rlcu_losses_selftest_tries(uint32_t tries);

#ifdef __cplusplus
}
#endif
#endif /* RLCU_LOSSES_H */
