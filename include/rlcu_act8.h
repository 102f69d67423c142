/*
 * rlcu_act8.h -- C ABI of 8-bit activation checkpoints on B200 (sm_100a): what a layer's forward pass keeps for
 * its backward pass, at half of FP16's bytes, and the RMSNorm (forward again, and backward) that reads it
 * without a decoded copy.  RL.cu keeps each layer's input in FP16 and recomputes the layer from it
 * (src/model/qwen3.cu:784-855); the norm is the first thing it recomputes and the last thing it
 * differentiates (src/kernels/rmsnorm.cu:3-158).
 *
 * Conventions are those of rlcu_adamw.h.  Calls keep no state: calls on different buffers may overlap on the
 * GPU and every call can be captured into a CUDA graph.  The same inputs give the same bits.
 *
 * Format: `rows` x `cols` values.  Each run of RLCU_ACT8_BLOCK consecutive columns of a row (the last one may be
 * shorter) has one byte s of scale, 2^e with e = s - 127, and one e4m3 code per value: value = code * 2^e.
 * e is the smallest exponent (of -127 and up) with max|x| <= 448 * 2^e, so a code is x * 2^-e rounded to nearest
 * even: off by at most 2^-4 of the value where that is at least 2^-6 * 2^e (2^-15 of the block's largest), by at most
 * 2^-10 * 2^e below.  The product with the scale is exact.  inf and NaN are kept as NaN; they do not enter max|x|.  A
 * block of zeros has s = 0.
 *   codes  : row r at codes + r * code_stride bytes (0: cols); bytes behind a row's last code are left alone
 *   scales : row r at scales + r * rlcu_act8_blocks(cols), one byte per block
 * Decoded values are rounded to the output's type once and, where they are finite, stay finite
 * (RLCU_F16: at most 65504).
 * What a call writes may share no byte with what it reads or writes elsewhere, unless a parameter says so; such calls are
 * refused.
 */
#ifndef RLCU_ACT8_H
#define RLCU_ACT8_H

#include "rlcu_adamw.h"

#ifdef __cplusplus
extern "C" {
#endif

#define RLCU_ACT8_BLOCK 128

/* scale bytes of one row */
uint64_t rlcu_act8_blocks(uint64_t cols);

/* x (F16, BF16 or F32; x_stride elements from row to row, 0: cols) into a checkpoint */
int rlcu_act8_store(const void* x, uint32_t dtype, uint64_t rows, uint64_t cols, uint64_t x_stride,
                    uint8_t* codes, uint64_t code_stride, uint8_t* scales, void* stream);
/* a checkpoint into x */
int rlcu_act8_load(const uint8_t* codes, uint64_t code_stride, const uint8_t* scales, uint64_t rows, uint64_t cols,
                   void* x, uint32_t dtype, uint64_t x_stride, void* stream);

/* The norm again: y = x * rstd * weight with rstd = 1 / sqrt(mean(x^2) + eps) per row, x the checkpoint's values.
 * weight has `cols` values of weight_dtype (RL.cu: F32); rstd may be NULL.  Squares are summed in FP32: a row whose sum is
 * beyond it (values above 1e18 or so) has rstd = 0. */
int rlcu_act8_rmsnorm(const uint8_t* codes, uint64_t code_stride, const uint8_t* scales, uint64_t rows, uint64_t cols,
                      const void* weight, uint32_t weight_dtype, float eps, void* y, uint32_t dtype, uint64_t y_stride,
                      float* rstd, void* stream);

enum {
    RLCU_ACT8_ACCUMULATE = 1u  /* dweight += instead of = (micro-batches of one step: the FP32 gradient pool)   */
};

/* Its gradient: with g = dy * weight,
 *   dx = rstd * (g - x * rstd^2 * mean(g x)) + dresidual,    dweight = sum over rows of dy * x * rstd
 * dy, dresidual (NULL: none) and dx are of `dtype`, each with its own row stride (0: cols); dx may be the buffer of
 * dy or of dresidual (same pointer and stride).  rstd is computed again from the checkpoint.  dweight may be NULL.
 * `workspace` (16-byte aligned device memory) holds partial sums of dweight; rlcu_act8_rmsnorm_grad_workspace says
 * how much, calls that overlap on the GPU need one each. */
uint64_t rlcu_act8_rmsnorm_grad_workspace(uint64_t rows, uint64_t cols);
int rlcu_act8_rmsnorm_grad(const uint8_t* codes, uint64_t code_stride, const uint8_t* scales, uint64_t rows,
                           uint64_t cols, const void* weight, uint32_t weight_dtype, float eps,
                           const void* dy, uint64_t dy_stride, const void* dresidual, uint64_t dresidual_stride,
                           void* dx, uint64_t dx_stride, uint32_t dtype, float* dweight, void* workspace,
                           uint64_t workspace_bytes, uint32_t flags, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* RLCU_ACT8_H */
