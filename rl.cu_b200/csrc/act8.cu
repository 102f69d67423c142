// 8-bit activation checkpoints and the RMSNorm that reads them (include/rlcu_act8.h).
//
// A block of 128 values shares a scale 2^e.  For a floating-point code a power of two loses nothing against a
// finer scale, and it makes both x * 2^-e and code * 2^e exact: the one rounding is that to e4m3.
#include "rlcu_act8.h"

#include <cfloat>
#include <cmath>

#include <cuda_fp8.h>

#include "host_util.h"
#include "typed.cuh"

namespace rlcu {
namespace {

constexpr int kAct8Threads = 256;
constexpr uint32_t kBlock = RLCU_ACT8_BLOCK;

// 2^e for e in [-149, 127]
__device__ __forceinline__ float pow2(int e) {
    return e >= -126 ? __uint_as_float((uint32_t)(e + 127) << 23) : __uint_as_float(1u << (e + 149));
}

// e + 127 of a block whose largest finite |x| is `top`: 448 = 1.75 * 2^8, so with top = f * 2^k, f in [1, 2),
// e = k - 8, one more where f > 1.75
__device__ __forceinline__ uint32_t scale_byte(float top) {
    const uint32_t bits = __float_as_uint(top);
    const int k = (int)(bits >> 23) - 127;               // a subnormal top gives -127: e stays above its own
    const int e = k - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return top == 0.0f || e < -127 ? 0u : (uint32_t)(e + 127);
}

__device__ __forceinline__ uint8_t encode(float x, float inv) {
    // inf stays inf under the exact product; the conversion would turn it into the largest finite code
    const float q = x * inv;
    if (!(fabsf(x) <= FLT_MAX)) return 0x7F;
    return (uint8_t)__nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float decode(uint8_t code, float scale) {
    const __half h = __half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3));
    // the product is exact, or beyond FP32 by the rounding to e4m3 (max|x| near FLT_MAX)
    const float v = __half2float(h) * scale;
    return fabsf(v) > FLT_MAX ? copysignf(FLT_MAX, v) : v;      // NaN compares false and stays
}

// one rounding to the output's type, finite values staying finite
template <uint32_t DT>
__device__ __forceinline__ float keep_finite(float v) {
    constexpr float most = DT == RLCU_F16 ? 65504.0f : DT == RLCU_BF16 ? 3.3895313892515355e38f : FLT_MAX;
    return fabsf(v) > most ? copysignf(most, v) : v;
}

// One warp per block of 128 columns.
template <uint32_t DT>
__global__ void __launch_bounds__(kAct8Threads)
act8_store_kernel(const void* x, uint64_t rows, uint32_t cols, uint64_t x_stride, uint8_t* codes, uint64_t code_stride,
                  uint8_t* scales) {
    using E = Elem<DT>;
    const uint32_t blocks = (cols + kBlock - 1) / kBlock;
    const uint64_t total = rows * blocks, step = (uint64_t)gridDim.x * (kAct8Threads / 32);
    const uint32_t lane = threadIdx.x & 31;
    for (uint64_t b = (uint64_t)blockIdx.x * (kAct8Threads / 32) + (threadIdx.x >> 5); b < total; b += step) {
        const uint64_t row = b / blocks;
        const uint32_t col = (uint32_t)(b - row * blocks) * kBlock;
        const typename E::T* in = static_cast<const typename E::T*>(x) + row * x_stride;
        float v[4], top = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t j = col + i * 32 + lane;
            v[i] = j < cols ? E::up(in[j]) : 0.0f;
            if (fabsf(v[i]) <= FLT_MAX) top = fmaxf(top, fabsf(v[i]));
        }
#pragma unroll
        for (int mask = 16; mask >= 1; mask >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, mask));
        const uint32_t byte = scale_byte(top);
        const float inv = pow2(127 - (int)byte);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t j = col + i * 32 + lane;
            if (j < cols) codes[row * code_stride + j] = encode(v[i], inv);
        }
        if (lane == 0) scales[b] = (uint8_t)byte;
    }
}

template <uint32_t DT>
__global__ void __launch_bounds__(kAct8Threads)
act8_load_kernel(const uint8_t* codes, uint64_t code_stride, const uint8_t* scales, uint64_t rows, uint32_t cols, void* x,
                 uint64_t x_stride) {
    using E = Elem<DT>;
    const uint32_t blocks = (cols + kBlock - 1) / kBlock;
    const uint64_t total = rows * blocks, step = (uint64_t)gridDim.x * (kAct8Threads / 32);
    const uint32_t lane = threadIdx.x & 31;
    for (uint64_t b = (uint64_t)blockIdx.x * (kAct8Threads / 32) + (threadIdx.x >> 5); b < total; b += step) {
        const uint64_t row = b / blocks;
        const uint32_t col = (uint32_t)(b - row * blocks) * kBlock;
        typename E::T* out = static_cast<typename E::T*>(x) + row * x_stride;
        const float scale = pow2((int)scales[b] - 127);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t j = col + i * 32 + lane;
            if (j < cols) out[j] = E::down(keep_finite<DT>(decode(codes[row * code_stride + j], scale)));
        }
    }
}

// ---------------------------------------------------------------------------
// RMSNorm
// ---------------------------------------------------------------------------

struct NormArgs {
    const uint8_t* codes;
    uint64_t code_stride;
    const uint8_t* scales;
    uint64_t rows;
    uint32_t cols, blocks;
    const void* weight;
    uint32_t weight_dtype;
    float eps;
    const void* dy;
    uint64_t dy_stride;
    const void* dres;
    uint64_t dres_stride;
    void* out;            // y or dx
    uint64_t out_stride;
    float* rstd;
    float* partial;       // [gridDim.x][cols] sums of dy * x * rstd
};

__device__ __forceinline__ float value_at(const NormArgs& a, uint64_t row, uint32_t j) {
    return decode(a.codes[row * a.code_stride + j], pow2((int)a.scales[row * a.blocks + j / kBlock] - 127));
}

__device__ __forceinline__ float weight_at(const NormArgs& a, uint32_t j) {
    if (a.weight_dtype == RLCU_F32) return static_cast<const float*>(a.weight)[j];
    const uint16_t w = static_cast<const uint16_t*>(a.weight)[j];
    return a.weight_dtype == RLCU_BF16 ? Elem<RLCU_BF16>::up(w) : Elem<RLCU_F16>::up(w);
}

// both sums over the CTA, in every thread
__device__ __forceinline__ float2 block_sum2(float x, float y, float2* smem) {
#pragma unroll
    for (int mask = 16; mask >= 1; mask >>= 1) {
        x += __shfl_xor_sync(0xFFFFFFFFu, x, mask);
        y += __shfl_xor_sync(0xFFFFFFFFu, y, mask);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = make_float2(x, y);
    __syncthreads();
    x = y = 0.0f;
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) {
        x += smem[w].x;
        y += smem[w].y;
    }
    return make_float2(x, y);
}

// One CTA per row at a time, the row decoded twice: any width.
template <uint32_t DT>
__global__ void __launch_bounds__(kAct8Threads)
norm_kernel(NormArgs a) {
    using E = Elem<DT>;
    __shared__ float2 smem[kAct8Threads / 32];
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float sq = 0.0f;
        for (uint32_t j = threadIdx.x; j < a.cols; j += kAct8Threads) {
            const float v = value_at(a, row, j);
            sq = fmaf(v, v, sq);
        }
        const float mean = block_sum2(sq, 0.0f, smem).x / (float)a.cols;
        const float rstd = 1.0f / sqrtf(mean + a.eps);
        if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
        typename E::T* out = static_cast<typename E::T*>(a.out) + row * a.out_stride;
        for (uint32_t j = threadIdx.x; j < a.cols; j += kAct8Threads)
            out[j] = E::down(value_at(a, row, j) * rstd * weight_at(a, j));
    }
}

template <uint32_t DT>
__global__ void __launch_bounds__(kAct8Threads)
norm_grad_kernel(NormArgs a) {
    using E = Elem<DT>;
    using T = typename E::T;
    __shared__ float2 smem[kAct8Threads / 32];
    float* part = a.partial ? a.partial + (uint64_t)blockIdx.x * a.cols : nullptr;
    if (part)
        for (uint32_t j = threadIdx.x; j < a.cols; j += kAct8Threads) part[j] = 0.0f;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
        const T* dres = a.dres ? static_cast<const T*>(a.dres) + row * a.dres_stride : nullptr;
        T* dx = static_cast<T*>(a.out) + row * a.out_stride;
        float sq = 0.0f, dot = 0.0f;
        for (uint32_t j = threadIdx.x; j < a.cols; j += kAct8Threads) {
            const float v = value_at(a, row, j);
            sq = fmaf(v, v, sq);
            dot = fmaf(E::up(dy[j]) * weight_at(a, j), v, dot);
        }
        const float2 sums = block_sum2(sq, dot, smem);
        const float rstd = 1.0f / sqrtf(sums.x / (float)a.cols + a.eps);
        const float pull = sums.y / (float)a.cols * rstd * rstd;
        for (uint32_t j = threadIdx.x; j < a.cols; j += kAct8Threads) {
            const float v = value_at(a, row, j), d = E::up(dy[j]);
            float g = rstd * fmaf(-v, pull, d * weight_at(a, j));
            if (dres) g += E::up(dres[j]);
            dx[j] = E::down(g);
            if (part) part[j] = fmaf(d, v * rstd, part[j]);
        }
    }
}

__global__ void __launch_bounds__(kAct8Threads)
norm_weight_kernel(const float* partial, uint32_t parts, uint32_t cols, float* dweight, uint32_t flags) {
    for (uint32_t j = blockIdx.x * kAct8Threads + threadIdx.x; j < cols; j += gridDim.x * kAct8Threads) {
        float s = 0.0f;
        for (uint32_t p = 0; p < parts; p++) s += partial[(uint64_t)p * cols + j];
        dweight[j] = flags & RLCU_ACT8_ACCUMULATE ? dweight[j] + s : s;
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

constexpr uint64_t kMostParts = 296;      // rows are dealt to at most this many CTAs where dweight is asked for

uint64_t norm_parts(uint64_t rows) { return rows < kMostParts ? rows : kMostParts; }

int check_matrix(const char* what, const void* p, uint32_t dtype, uint64_t rows, uint64_t cols, uint64_t& stride) {
    if (!dtype_known(dtype)) return set_error(RLCU_ERR_INVALID, "unknown dtype %u", dtype);
    if (stride == 0) stride = cols;
    if (stride < cols || too_large(rows, stride)) return set_error(RLCU_ERR_INVALID, "%s: row stride below cols or out of range", what);
    if (rows && cols && !p) return set_error(RLCU_ERR_INVALID, "%s: null pointer", what);
    if (reinterpret_cast<uintptr_t>(p) % dtype_bytes(dtype)) return set_error(RLCU_ERR_INVALID, "%s: not aligned to its element size", what);
    return RLCU_OK;
}

int check_held(const uint8_t* codes, uint64_t& code_stride, const uint8_t* scales, uint64_t rows, uint64_t cols) {
    if (cols > 0x7FFFFFFFull || rows > 0x7FFFFFFFull) return set_error(RLCU_ERR_INVALID, "rows or cols out of range");
    if (code_stride == 0) code_stride = cols;
    if (code_stride < cols || too_large(rows, code_stride)) return set_error(RLCU_ERR_INVALID, "code stride below cols or out of range");
    if (rows && cols && (!codes || !scales)) return set_error(RLCU_ERR_INVALID, "null codes or scales");
    return RLCU_OK;
}

// the same buffer, or none of it
bool same_or_apart(const void* p, uint64_t ps, const void* q, uint64_t qs, uint64_t rows, uint64_t cols, size_t esz) {
    if (p == q && (ps == qs || rows <= 1)) return true;
    return !overlap(span_of(p, rows, cols, ps, esz), span_of(q, rows, cols, qs, esz));
}

int grid_for(uint64_t units, int per_sm, int* out) {
    int dev = 0, sms = 0;
    RLCU_CUDA(cudaGetDevice(&dev));
    RLCU_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    const uint64_t most = (uint64_t)sms * per_sm;
    *out = (int)(units < most ? units : most);
    return RLCU_OK;
}

}  // namespace
}  // namespace rlcu

using namespace rlcu;

extern "C" uint64_t rlcu_act8_blocks(uint64_t cols) { return (cols + kBlock - 1) / kBlock; }

extern "C" uint64_t rlcu_act8_rmsnorm_grad_workspace(uint64_t rows, uint64_t cols) { return norm_parts(rows) * cols * sizeof(float); }

extern "C" int rlcu_act8_store(const void* x, uint32_t dtype, uint64_t rows, uint64_t cols, uint64_t x_stride,
                               uint8_t* codes, uint64_t code_stride, uint8_t* scales, void* stream) {
    if (const int rc = check_held(codes, code_stride, scales, rows, cols)) return rc;
    if (const int rc = check_matrix("x", x, dtype, rows, cols, x_stride)) return rc;
    if (!rows || !cols) return RLCU_OK;
    if (overlap(span_of(x, rows, cols, x_stride, dtype_bytes(dtype)), span_of(codes, rows, cols, code_stride, 1)))
        return set_error(RLCU_ERR_INVALID, "x and codes overlap");
    int grid = 0;
    if (const int rc = grid_for((rows * rlcu_act8_blocks(cols) + 7) / 8, 8, &grid)) return rc;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == RLCU_F16) act8_store_kernel<RLCU_F16><<<grid, kAct8Threads, 0, s>>>(x, rows, (uint32_t)cols, x_stride, codes, code_stride, scales);
    else if (dtype == RLCU_BF16) act8_store_kernel<RLCU_BF16><<<grid, kAct8Threads, 0, s>>>(x, rows, (uint32_t)cols, x_stride, codes, code_stride, scales);
    else act8_store_kernel<RLCU_F32><<<grid, kAct8Threads, 0, s>>>(x, rows, (uint32_t)cols, x_stride, codes, code_stride, scales);
    RLCU_CUDA(cudaGetLastError());
    return RLCU_OK;
}

extern "C" int rlcu_act8_load(const uint8_t* codes, uint64_t code_stride, const uint8_t* scales, uint64_t rows, uint64_t cols,
                              void* x, uint32_t dtype, uint64_t x_stride, void* stream) {
    if (const int rc = check_held(codes, code_stride, scales, rows, cols)) return rc;
    if (const int rc = check_matrix("x", x, dtype, rows, cols, x_stride)) return rc;
    if (!rows || !cols) return RLCU_OK;
    if (overlap(span_of(x, rows, cols, x_stride, dtype_bytes(dtype)), span_of(codes, rows, cols, code_stride, 1)))
        return set_error(RLCU_ERR_INVALID, "x and codes overlap");
    int grid = 0;
    if (const int rc = grid_for((rows * rlcu_act8_blocks(cols) + 7) / 8, 8, &grid)) return rc;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == RLCU_F16) act8_load_kernel<RLCU_F16><<<grid, kAct8Threads, 0, s>>>(codes, code_stride, scales, rows, (uint32_t)cols, x, x_stride);
    else if (dtype == RLCU_BF16) act8_load_kernel<RLCU_BF16><<<grid, kAct8Threads, 0, s>>>(codes, code_stride, scales, rows, (uint32_t)cols, x, x_stride);
    else act8_load_kernel<RLCU_F32><<<grid, kAct8Threads, 0, s>>>(codes, code_stride, scales, rows, (uint32_t)cols, x, x_stride);
    RLCU_CUDA(cudaGetLastError());
    return RLCU_OK;
}

extern "C" int rlcu_act8_rmsnorm(const uint8_t* codes, uint64_t code_stride, const uint8_t* scales, uint64_t rows,
                                 uint64_t cols, const void* weight, uint32_t weight_dtype, float eps, void* y,
                                 uint32_t dtype, uint64_t y_stride, float* rstd, void* stream) {
    uint64_t one = 0;
    if (const int rc = check_held(codes, code_stride, scales, rows, cols)) return rc;
    if (const int rc = check_matrix("y", y, dtype, rows, cols, y_stride)) return rc;
    if (const int rc = check_matrix("weight", weight, weight_dtype, 1, cols, one)) return rc;
    if (!(eps >= 0.0f) || std::isinf(eps)) return set_error(RLCU_ERR_INVALID, "eps must be finite and not negative");
    if (!rows || !cols) return RLCU_OK;
    if (overlap(span_of(y, rows, cols, y_stride, dtype_bytes(dtype)), span_of(codes, rows, cols, code_stride, 1)))
        return set_error(RLCU_ERR_INVALID, "y and codes overlap");
    NormArgs a = {codes, code_stride, scales, rows, (uint32_t)cols, (uint32_t)rlcu_act8_blocks(cols), weight, weight_dtype, eps,
                  nullptr, 0, nullptr, 0, y, y_stride, rstd, nullptr};
    int grid = 0;
    if (const int rc = grid_for(rows, 8, &grid)) return rc;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == RLCU_F16) norm_kernel<RLCU_F16><<<grid, kAct8Threads, 0, s>>>(a);
    else if (dtype == RLCU_BF16) norm_kernel<RLCU_BF16><<<grid, kAct8Threads, 0, s>>>(a);
    else norm_kernel<RLCU_F32><<<grid, kAct8Threads, 0, s>>>(a);
    RLCU_CUDA(cudaGetLastError());
    return RLCU_OK;
}

extern "C" int rlcu_act8_rmsnorm_grad(const uint8_t* codes, uint64_t code_stride, const uint8_t* scales, uint64_t rows,
                                      uint64_t cols, const void* weight, uint32_t weight_dtype, float eps,
                                      const void* dy, uint64_t dy_stride, const void* dresidual,
                                      uint64_t dresidual_stride, void* dx, uint64_t dx_stride, uint32_t dtype,
                                      float* dweight, void* workspace, uint64_t workspace_bytes, uint32_t flags,
                                      void* stream) {
    uint64_t one = 0;
    if (const int rc = check_held(codes, code_stride, scales, rows, cols)) return rc;
    if (const int rc = check_matrix("dy", dy, dtype, rows, cols, dy_stride)) return rc;
    if (const int rc = check_matrix("dx", dx, dtype, rows, cols, dx_stride)) return rc;
    if (dresidual)
        if (const int rc = check_matrix("dresidual", dresidual, dtype, rows, cols, dresidual_stride)) return rc;
    if (const int rc = check_matrix("weight", weight, weight_dtype, 1, cols, one)) return rc;
    if (!(eps >= 0.0f) || std::isinf(eps)) return set_error(RLCU_ERR_INVALID, "eps must be finite and not negative");
    if (flags & ~(uint32_t)RLCU_ACT8_ACCUMULATE) return set_error(RLCU_ERR_INVALID, "unknown flags");
    const size_t esz = dtype_bytes(dtype);
    if (!same_or_apart(dx, dx_stride, dy, dy_stride, rows, cols, esz) ||
        (dresidual && !same_or_apart(dx, dx_stride, dresidual, dresidual_stride, rows, cols, esz)) ||
        overlap(span_of(dx, rows, cols, dx_stride, esz), span_of(codes, rows, cols, code_stride, 1)))
        return set_error(RLCU_ERR_INVALID, "dx overlaps another buffer without being the same");
    const uint64_t need = rlcu_act8_rmsnorm_grad_workspace(rows, cols);
    if (dweight && need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < need))
        return set_error(RLCU_ERR_INVALID, "workspace: %llu bytes, 16-byte aligned, are needed", (unsigned long long)need);
    if (!cols) return RLCU_OK;
    cudaStream_t s = (cudaStream_t)stream;
    NormArgs a = {codes, code_stride, scales, rows, (uint32_t)cols, (uint32_t)rlcu_act8_blocks(cols), weight, weight_dtype, eps,
                  dy, dy_stride, dresidual, dresidual_stride, dx, dx_stride, nullptr,
                  dweight ? static_cast<float*>(workspace) : nullptr};
    const int grid = (int)norm_parts(rows);
    if (grid) {
        if (dtype == RLCU_F16) norm_grad_kernel<RLCU_F16><<<grid, kAct8Threads, 0, s>>>(a);
        else if (dtype == RLCU_BF16) norm_grad_kernel<RLCU_BF16><<<grid, kAct8Threads, 0, s>>>(a);
        else norm_grad_kernel<RLCU_F32><<<grid, kAct8Threads, 0, s>>>(a);
        RLCU_CUDA(cudaGetLastError());
    }
    if (dweight) {
        norm_weight_kernel<<<(int)((cols + kAct8Threads - 1) / kAct8Threads), kAct8Threads, 0, s>>>(a.partial, (uint32_t)grid,
                                                                                                  (uint32_t)cols, dweight, flags);
        RLCU_CUDA(cudaGetLastError());
    }
    return RLCU_OK;
}
