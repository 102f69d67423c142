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

// Element by element, for rows that start anywhere: a warp per kWarpBlocks blocks of a row, lane i with every 32nd column,
// all of its loads in flight at once.
constexpr int kWarpBlocks = 4, kPerLane = kWarpBlocks * (int)kBlock / 32;

// where the calling warp works: false if there is nothing
__device__ __forceinline__ bool warp_place(uint64_t rows, uint32_t blocks, uint64_t& row, uint32_t& block) {
    const uint32_t per_row = (blocks + kWarpBlocks - 1) / kWarpBlocks;
    const uint64_t unit = (uint64_t)blockIdx.x * (kAct8Threads / 32) + (threadIdx.x >> 5);
    row = unit <= 0xFFFFFFFFull ? (uint32_t)unit / per_row : unit / per_row;
    block = (uint32_t)(unit - row * per_row) * kWarpBlocks;
    return row < rows;
}

template <uint32_t DT>
__global__ void __launch_bounds__(kAct8Threads)
act8_store_kernel(const void* x, uint64_t rows, uint32_t cols, uint64_t x_stride, uint8_t* codes, uint64_t code_stride,
                  uint8_t* scales) {
    using E = Elem<DT>;
    const uint32_t blocks = (cols + kBlock - 1) / kBlock, lane = threadIdx.x & 31;
    uint64_t row;
    uint32_t block;
    if (!warp_place(rows, blocks, row, block)) return;
    const uint32_t col = block * kBlock + lane;
    const typename E::T* in = static_cast<const typename E::T*>(x) + row * x_stride + col;
    uint8_t* out = codes + row * code_stride + col;
    float v[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane; i++) v[i] = col + i * 32 < cols ? E::up(in[i * 32]) : 0.0f;
#pragma unroll
    for (int b = 0; b < kWarpBlocks; b++) {
        float top = 0.0f;
#pragma unroll
        for (int i = 4 * b; i < 4 * b + 4; i++)
            if (fabsf(v[i]) <= FLT_MAX) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
        for (int mask = 16; mask >= 1; mask >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, mask));
        const uint32_t byte = scale_byte(top);
        const float inv = pow2(127 - (int)byte);
#pragma unroll
        for (int i = 4 * b; i < 4 * b + 4; i++)
            if (col + i * 32 < cols) out[i * 32] = encode(v[i], inv);
        if (lane == 0 && block + b < blocks) scales[row * blocks + block + b] = (uint8_t)byte;
    }
}

template <uint32_t DT>
__global__ void __launch_bounds__(kAct8Threads)
act8_load_kernel(const uint8_t* codes, uint64_t code_stride, const uint8_t* scales, uint64_t rows, uint32_t cols, void* x,
                 uint64_t x_stride) {
    using E = Elem<DT>;
    const uint32_t blocks = (cols + kBlock - 1) / kBlock, lane = threadIdx.x & 31;
    uint64_t row;
    uint32_t block;
    if (!warp_place(rows, blocks, row, block)) return;
    const uint32_t col = block * kBlock + lane;
    const uint8_t* in = codes + row * code_stride + col;
    typename E::T* out = static_cast<typename E::T*>(x) + row * x_stride + col;
    uint8_t v[kPerLane], byte[kWarpBlocks];
#pragma unroll
    for (int i = 0; i < kPerLane; i++) v[i] = col + i * 32 < cols ? in[i * 32] : 0;
#pragma unroll
    for (int b = 0; b < kWarpBlocks; b++) byte[b] = block + b < blocks ? scales[row * blocks + block + b] : 0;
#pragma unroll
    for (int i = 0; i < kPerLane; i++)
        if (col + i * 32 < cols) out[i * 32] = E::down(keep_finite<DT>(decode(v[i], pow2((int)byte[i / 4] - 127))));
}

// The same in 16- and 32-byte accesses, for rows that start on 16-byte boundaries: eight threads per block of 128, 16
// columns each (one 16-byte group of codes).  Pure streaming, bound by HBM; a CTA takes kVecBlocks consecutive blocks and
// the grid goes through memory in order.  16384 x 4096 bf16, store and load: 67 us, 0.92 of the copy rate (16-byte accesses
// alone: 74 us; element by element: 179 to 230 us).
constexpr int kRun = 16;                                   // columns per thread and step
constexpr int kVecSteps = 2;
constexpr uint32_t kVecBlocks = kAct8Threads / (kBlock / kRun) * kVecSteps;

// 32 bytes in one access where the address allows it (sm_100): a thread's 16 columns of 16 bits
__device__ __forceinline__ void load32(const void* p, uint4& a, uint4& b) {
    if ((reinterpret_cast<uintptr_t>(p) & 31u) == 0) {
        asm volatile("ld.global.cs.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "l"(p));
    } else {
        a = __ldcs(static_cast<const uint4*>(p));
        b = __ldcs(static_cast<const uint4*>(p) + 1);
    }
}
__device__ __forceinline__ void store32(void* p, uint4 a, uint4 b) {
    if ((reinterpret_cast<uintptr_t>(p) & 31u) == 0) {
        asm volatile("st.global.cs.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                     :: "l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
    } else {
        __stcs(static_cast<uint4*>(p), a);
        __stcs(static_cast<uint4*>(p) + 1, b);
    }
}

// 16 columns as they are in memory
template <uint32_t DT>
struct Run {
    static constexpr int kGroups = kRun / Elem<DT>::kVec;
    uint4 v[kGroups];

    __device__ __forceinline__ void load(const void* p) {
#pragma unroll
        for (int i = 0; i < kGroups; i += 2) load32(static_cast<const uint4*>(p) + i, v[i], v[i + 1]);
    }
    __device__ __forceinline__ void store(void* p) const {
#pragma unroll
        for (int i = 0; i < kGroups; i += 2) store32(static_cast<uint4*>(p) + i, v[i], v[i + 1]);
    }
    // the first n of them, one by one
    __device__ __forceinline__ void load_part(const typename Elem<DT>::T* p, int n) {
        float f[kRun];
#pragma unroll
        for (int i = 0; i < kRun; i++) f[i] = i < n ? Elem<DT>::up(p[i]) : 0.0f;
        set(f);
    }
    __device__ __forceinline__ void store_part(typename Elem<DT>::T* p, int n) const {
        float f[kRun];
        get(f);
#pragma unroll
        for (int i = 0; i < kRun; i++)
            if (i < n) p[i] = Elem<DT>::down(f[i]);
    }
    __device__ __forceinline__ void get(float (&f)[kRun]) const {
#pragma unroll
        for (int i = 0; i < kGroups; i++) {
            float g[Elem<DT>::kVec];
            Elem<DT>::unpack(v[i], g);
#pragma unroll
            for (int q = 0; q < Elem<DT>::kVec; q++) f[i * Elem<DT>::kVec + q] = g[q];
        }
    }
    __device__ __forceinline__ void set(const float (&f)[kRun]) {
#pragma unroll
        for (int i = 0; i < kGroups; i++) {
            float g[Elem<DT>::kVec];
#pragma unroll
            for (int q = 0; q < Elem<DT>::kVec; q++) g[q] = f[i * Elem<DT>::kVec + q];
            v[i] = Elem<DT>::pack(g);
        }
    }
};
constexpr int kPairs = kRun / 2;

// 16 columns as pairs of FP32 (for the packed arithmetic)
template <uint32_t DT>
__device__ __forceinline__ void to_pairs(const Run<DT>& r, F2 (&p)[kPairs]) {
    float f[kRun];
    r.get(f);
#pragma unroll
    for (int i = 0; i < kPairs; i++) p[i] = F2(f[2 * i], f[2 * i + 1]);
}
template <uint32_t DT>
__device__ __forceinline__ Run<DT> from_pairs(const F2 (&p)[kPairs]) {
    float f[kRun];
#pragma unroll
    for (int i = 0; i < kPairs; i++) p[i].get(f[2 * i], f[2 * i + 1]);
    Run<DT> r;
    r.set(f);
    return r;
}
__device__ __forceinline__ float add_pairs(F2 a) {
    float x, y;
    a.get(x, y);
    return x + y;
}

// the codes of 16 columns, the first n of them where the row ends sooner
__device__ __forceinline__ uint4 load_codes(const uint8_t* p, int n) {
    if (n >= kRun) return __ldcs(reinterpret_cast<const uint4*>(p));
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < kRun; i++)
        if (i < n) w[i / 4] |= (uint32_t)p[i] << (i % 4 * 8);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// four codes of finite values (or NaN)
__device__ __forceinline__ uint32_t encode4(const float* q) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(q[1]), "f"(q[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(q[3]), "f"(q[2]));
    return (uint32_t)lo | (uint32_t)hi << 16;
}
__device__ __forceinline__ void decode4(uint32_t w, float* f) {
    uint32_t a, b;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(a) : "h"((uint16_t)w));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"((uint16_t)(w >> 16)));
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    f[0] = x.x;
    f[1] = x.y;
    f[2] = y.x;
    f[3] = y.y;
}
// 16 codes without their scale
__device__ __forceinline__ void code_pairs(uint4 v, F2 (&p)[kPairs]) {
    float f[kRun];
    decode4(v.x, f);
    decode4(v.y, f + 4);
    decode4(v.z, f + 8);
    decode4(v.w, f + 12);
#pragma unroll
    for (int i = 0; i < kPairs; i++) p[i] = F2(f[2 * i], f[2 * i + 1]);
}
// 16 codes as values, before any rounding; finite ones stay finite
__device__ __forceinline__ void decode_run(uint4 v, uint32_t byte, float (&f)[kRun]) {
    decode4(v.x, f);
    decode4(v.y, f + 4);
    decode4(v.z, f + 8);
    decode4(v.w, f + 12);
    const float scale = pow2((int)byte - 127);
#pragma unroll
    for (int i = 0; i < kRun; i++) f[i] *= scale;
    if (byte >= 127 + 119) {                               // 448 * 2^119 < 2^128
#pragma unroll
        for (int i = 0; i < kRun; i++) f[i] = fabsf(f[i]) > FLT_MAX ? copysignf(FLT_MAX, f[i]) : f[i];
    }
}
// where a thread's step k of a CTA's blocks lies
struct Place {
    uint32_t block, row, col;
    int n;                       // columns of its 16 that the row has

    __device__ __forceinline__ Place(int k, uint32_t total, uint32_t blocks, uint32_t cols) {
        block = blockIdx.x * kVecBlocks + k * (kVecBlocks / kVecSteps) + threadIdx.x / (kBlock / kRun);
        row = block / blocks;
        col = (block - row * blocks) * kBlock + threadIdx.x % (kBlock / kRun) * kRun;
        n = block < total ? (int)cols - (int)col : 0;
    }
};

template <uint32_t DT>
__global__ void __launch_bounds__(kAct8Threads)
act8_store_vec_kernel(const void* x, uint32_t total, uint32_t blocks, uint32_t cols, uint64_t x_stride, uint8_t* codes,
                      uint64_t code_stride, uint8_t* scales) {
    using T = typename Elem<DT>::T;
    Run<DT> runs[kVecSteps];
#pragma unroll
    for (int k = 0; k < kVecSteps; k++) {
        const Place at(k, total, blocks, cols);
        const T* in = static_cast<const T*>(x) + at.row * x_stride + at.col;
        if (at.n >= kRun) runs[k].load(in);
        else runs[k].load_part(in, at.n);
    }
#pragma unroll
    for (int k = 0; k < kVecSteps; k++) {
        const Place at(k, total, blocks, cols);
        float f[kRun], top = 0.0f;
        runs[k].get(f);
#pragma unroll
        for (int i = 0; i < kRun; i++) top = fmaxf(top, fabsf(f[i]));             // NaN is passed over
#pragma unroll
        for (int mask = 4; mask >= 1; mask >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, mask));
        if (__any_sync(0xFFFFFFFFu, top > FLT_MAX)) {                              // an infinity somewhere: finite values count
            top = 0.0f;
#pragma unroll
            for (int i = 0; i < kRun; i++) {
                if (fabsf(f[i]) <= FLT_MAX) top = fmaxf(top, fabsf(f[i]));
                else f[i] = NAN;
            }
#pragma unroll
            for (int mask = 4; mask >= 1; mask >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, mask));
        }
        if (at.n <= 0) {
            // (a block's last threads may have no column; the first one has)
            continue;
        }
        const uint32_t byte = scale_byte(top);
        const float inv = pow2(127 - (int)byte);
#pragma unroll
        for (int i = 0; i < kRun; i++) f[i] *= inv;
        const uint4 q = make_uint4(encode4(f), encode4(f + 4), encode4(f + 8), encode4(f + 12));
        uint8_t* out = codes + at.row * code_stride + at.col;
        if (at.n >= kRun) {
            *reinterpret_cast<uint4*>(out) = q;
        } else {
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < kRun; i++)
                if (i < at.n) out[i] = (uint8_t)(w[i / 4] >> (i % 4 * 8));
        }
        if (threadIdx.x % (kBlock / kRun) == 0) scales[at.block] = (uint8_t)byte;
    }
}

template <uint32_t DT>
__global__ void __launch_bounds__(kAct8Threads)
act8_load_vec_kernel(const uint8_t* codes, uint64_t code_stride, const uint8_t* scales, uint32_t total, uint32_t blocks,
                     uint32_t cols, void* x, uint64_t x_stride) {
    using T = typename Elem<DT>::T;
    uint4 v[kVecSteps];
    uint32_t byte[kVecSteps];
#pragma unroll
    for (int k = 0; k < kVecSteps; k++) {
        const Place at(k, total, blocks, cols);
        if (at.n > 0) {
            v[k] = load_codes(codes + at.row * code_stride + at.col, at.n);
            byte[k] = scales[at.block];
        }
    }
#pragma unroll
    for (int k = 0; k < kVecSteps; k++) {
        const Place at(k, total, blocks, cols);
        if (at.n <= 0) continue;
        float f[kRun];
        decode_run(v[k], byte[k], f);
        if (DT == RLCU_F16 ? byte[k] >= 127 + 7 : DT == RLCU_BF16 && byte[k] >= 127 + 119) {      // 448 * 2^7 < 65504
#pragma unroll
            for (int i = 0; i < kRun; i++) f[i] = keep_finite<DT>(f[i]);
        }
        Run<DT> run;
        run.set(f);
        T* out = static_cast<T*>(x) + at.row * x_stride + at.col;
        if (at.n >= kRun) run.store(out);
        else run.store_part(out, at.n);
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
    float* dweight;       // given where the grid is one cluster, which adds the partial sums itself
    uint32_t flags;
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

// One CTA per row at a time, the row decoded twice, a code per access: rows wider than the kernels below hold.  Not fast:
// 4096 x 16384 bf16 154 us, its gradient (whose partial sums are in memory) 1231 us; the bytes alone would take 31 and 72.
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

// Rows that start on 16-byte boundaries: TPR threads per row, each with the same run of 16 columns of every row it works
// on (so their weights stay in registers), a CTA with THREADS / TPR rows at a time.  The row is decoded once; the sums
// over it go through one barrier (none where a warp has the row).
template <int TPR, int THREADS>
struct RowSum {
    float2 part[2][THREADS / 32];              // by step parity
    // of the TPR threads that have the row
    __device__ __forceinline__ float2 operator()(float x, float y, uint32_t step) {
#pragma unroll
        for (int mask = 16; mask >= 1; mask >>= 1) {
            x += __shfl_xor_sync(0xFFFFFFFFu, x, mask);
            y += __shfl_xor_sync(0xFFFFFFFFu, y, mask);
        }
        if constexpr (TPR > 32) {
            const uint32_t warp = threadIdx.x >> 5, group = threadIdx.x / TPR;
            if ((threadIdx.x & 31) == 0) part[step & 1][warp] = make_float2(x, y);
            if constexpr (TPR == THREADS) {
                __syncthreads();
            } else {
                // each group its own barrier, by constant numbers (a number in a register would claim all sixteen)
                static_assert(THREADS / TPR <= 4, "barriers");
                if (group == 0) asm volatile("barrier.cta.sync 1, %0;" :: "n"(TPR) : "memory");
                else if (group == 1) asm volatile("barrier.cta.sync 2, %0;" :: "n"(TPR) : "memory");
                else if (group == 2) asm volatile("barrier.cta.sync 3, %0;" :: "n"(TPR) : "memory");
                else asm volatile("barrier.cta.sync 4, %0;" :: "n"(TPR) : "memory");
            }
            x = y = 0.0f;
#pragma unroll
            for (int w = 0; w < TPR / 32; w++) {
                x += part[step & 1][group * (TPR / 32) + w].x;
                y += part[step & 1][group * (TPR / 32) + w].y;
            }
        }
        return make_float2(x, y);
    }
};

template <uint32_t DT>
__device__ __forceinline__ void load_weight_run(const void* weight, uint32_t col, int n, float (&w)[kRun]) {
    using E = Elem<DT>;
    const typename E::T* p = static_cast<const typename E::T*>(weight) + col;
    if (n >= kRun && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
#pragma unroll
        for (int i = 0; i < kRun / E::kVec; i++) {
            float g[E::kVec];
            E::unpack(__ldg(reinterpret_cast<const uint4*>(p) + i), g);
#pragma unroll
            for (int q = 0; q < E::kVec; q++) w[i * E::kVec + q] = g[q];
        }
    } else {
#pragma unroll
        for (int i = 0; i < kRun; i++) w[i] = i < n ? E::up(p[i]) : 0.0f;
    }
}

__device__ __forceinline__ void load_weights(const NormArgs& a, uint32_t col, int n, F2 (&w)[kPairs]) {
    float f[kRun];
    if (a.weight_dtype == RLCU_F32) load_weight_run<RLCU_F32>(a.weight, col, n, f);
    else if (a.weight_dtype == RLCU_BF16) load_weight_run<RLCU_BF16>(a.weight, col, n, f);
    else load_weight_run<RLCU_F16>(a.weight, col, n, f);
#pragma unroll
    for (int i = 0; i < kPairs; i++) w[i] = F2(f[2 * i], f[2 * i + 1]);
}

// A thread's 16 columns lie in one block, so their scale s comes out of the sums: sum x^2 = s^2 sum c^2 and so on, with
// c the codes, and x itself is never formed.  Bound by HBM and, a row at a time, by the latency of its sum: 16384 x 4096
// bf16 39 to 41 us on different GPUs, 0.79 to 0.75 of the copy rate (one row per barrier 43 us, scalar arithmetic 54 us).
template <uint32_t DT, int TPR, int THREADS>
__global__ void __launch_bounds__(THREADS)
norm_vec_kernel(NormArgs a, uint32_t rows_per_cta) {
    using T = typename Elem<DT>::T;
    __shared__ RowSum<TPR, THREADS> sum;
    const uint32_t lane = threadIdx.x % TPR, rows = (uint32_t)a.rows, col = lane * kRun;
    const int n = (int)a.cols - (int)col;
    const uint32_t first = blockIdx.x * rows_per_cta + threadIdx.x / TPR, last = min(rows, (blockIdx.x + 1) * rows_per_cta);
    F2 w[kPairs];
    load_weights(a, col, n, w);
    struct Held {
        uint4 codes;
        uint32_t byte;
    } next[2];
    constexpr uint32_t at_once = THREADS / TPR;
    // two rows per step: one barrier for both
    auto fetch = [&](uint32_t row) {
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const uint32_t at = row + r * at_once;
            next[r].byte = 0;
            next[r].codes = make_uint4(0u, 0u, 0u, 0u);
            if (at < last && n > 0) {
                next[r].codes = load_codes(a.codes + at * a.code_stride + col, n);
                next[r].byte = a.scales[(uint64_t)at * a.blocks + col / kBlock];
            }
        }
    };
    fetch(first);
    uint32_t step = 0;
    for (uint32_t row = first; row < last; row += 2 * at_once, step++) {
        Held now[2] = {next[0], next[1]};
        float sq[2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const float s = pow2((int)now[r].byte - 127);
            F2 c[kPairs];
            code_pairs(now[r].codes, c);
            F2 acc = mul2(c[0], c[0]);
#pragma unroll
            for (int i = 1; i < kPairs; i++) acc = fma2(c[i], c[i], acc);
            sq[r] = n > 0 ? s * (s * add_pairs(acc)) : 0.0f;
        }
        fetch(row + 2 * at_once);
        const float2 sums = sum(sq[0], sq[1], step);
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const uint32_t at = row + r * at_once;
            if (at >= last) continue;
            const float rstd = 1.0f / sqrtf((r ? sums.y : sums.x) / (float)a.cols + a.eps);
            if (a.rstd && lane == 0) a.rstd[at] = rstd;
            if (n <= 0) continue;
            const float s = pow2((int)now[r].byte - 127) * rstd;
            const F2 k(s, s);
            // decoded again: packed, two rows fit the registers
            asm volatile("" : "+r"(now[r].codes.x), "+r"(now[r].codes.y), "+r"(now[r].codes.z), "+r"(now[r].codes.w));
            F2 c[kPairs];
            code_pairs(now[r].codes, c);
#pragma unroll
            for (int i = 0; i < kPairs; i++) c[i] = mul2(mul2(c[i], k), w[i]);
            const Run<DT> run = from_pairs<DT>(c);
            T* out = static_cast<T*>(a.out) + at * a.out_stride + col;
            if (n >= kRun) run.store(out);
            else run.store_part(out, n);
        }
    }
}

// four columns of a run as two pairs, and back
template <uint32_t DT>
__device__ __forceinline__ void get_four(const Run<DT>& r, int i, F2 (&p)[2]) {
    if constexpr (DT == RLCU_F32) {
        const uint4 v = r.v[i];
        p[0] = F2(__uint_as_float(v.x), __uint_as_float(v.y));
        p[1] = F2(__uint_as_float(v.z), __uint_as_float(v.w));
    } else {
        const uint4 v = r.v[i / 2];
        float a, b, c, d;
        Elem<DT>::up2(i % 2 ? v.z : v.x, a, b);
        Elem<DT>::up2(i % 2 ? v.w : v.y, c, d);
        p[0] = F2(a, b);
        p[1] = F2(c, d);
    }
}
template <uint32_t DT>
__device__ __forceinline__ void set_four(Run<DT>& r, int i, const F2 (&p)[2]) {
    float a, b, c, d;
    p[0].get(a, b);
    p[1].get(c, d);
    if constexpr (DT == RLCU_F32) {
        r.v[i] = make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d));
    } else {
        uint4& v = r.v[i / 2];
        (i % 2 ? v.z : v.x) = Elem<DT>::down2(a, b);
        (i % 2 ? v.w : v.y) = Elem<DT>::down2(c, d);
    }
}

// The end of a gradient kernel whose grid is one cluster: partial sums added in order, the columns dealt to all threads.
__device__ __forceinline__ void add_parts_in_cluster(const NormArgs& a) {
    // (not .aligned: the threads of a warp come from different branches)
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    for (uint32_t j = blockIdx.x * blockDim.x + threadIdx.x; j < a.cols; j += gridDim.x * blockDim.x) {
        float s = 0.0f;
        for (uint32_t p = 0; p < gridDim.x; p++) s += __ldcg(a.partial + (uint64_t)p * a.cols + j);
        a.dweight[j] = a.flags & RLCU_ACT8_ACCUMULATE ? a.dweight[j] + s : s;
    }
}

// What a thread reads of one row.  It stays packed between its two uses: unpacked it would not fit the registers.
template <uint32_t DT>
struct GradRow {
    uint4 codes;
    uint32_t byte;
    Run<DT> dy, dres;

    __device__ __forceinline__ void four(int i, F2 (&c)[2], F2 (&d)[2]) const {
        float f[4];
        decode4(i == 0 ? codes.x : i == 1 ? codes.y : i == 2 ? codes.z : codes.w, f);
        c[0] = F2(f[0], f[1]);
        c[1] = F2(f[2], f[3]);
        get_four(dy, i, d);
    }
    __device__ __forceinline__ void four_dres(int i, F2 (&r)[2]) const { get_four(dres, i, r); }
    __device__ __forceinline__ void keep_packed() {
        asm volatile("" : "+r"(codes.x), "+r"(codes.y), "+r"(codes.z), "+r"(codes.w));
#pragma unroll
        for (int i = 0; i < Run<DT>::kGroups; i++)
            asm volatile("" : "+r"(dy.v[i].x), "+r"(dy.v[i].y), "+r"(dy.v[i].z), "+r"(dy.v[i].w));
    }
};

// The gradient: rows are dealt to the CTAs in a fixed order, so that dweight's partial sums are the same in every run;
// the next row is on its way in registers.  16384 x 4096 bf16 with a residual: 86 to 91 us on different GPUs with the
// second kernel, 0.83 to 0.79 of the copy rate; f32, without the row ahead, 160 us, 0.83.  Issue slots were 69 % busy with
// scalar arithmetic (95 us); packed pairs and the scale taken out of the sums left 86 us.  More CTAs per SM spill (177 to 255
// us); the next row by cp.async is slower (112 us).  With 512 threads a row (more than 4096 columns) a thread keeps 8 to 24
// bytes in local memory as it is.
template <uint32_t DT, int TPR, int THREADS>
__global__ void __launch_bounds__(THREADS, 512 / THREADS)
norm_grad_vec_kernel(NormArgs a) {
    using T = typename Elem<DT>::T;
    constexpr bool kAhead = DT != RLCU_F32;    // FP32 rows take twice the registers: two of them would spill
    __shared__ RowSum<TPR, THREADS> sum;
    const uint32_t lane = threadIdx.x % TPR, rows = (uint32_t)a.rows, at_once = THREADS / TPR, jump = gridDim.x * at_once;
    const uint32_t col = lane * kRun;
    const int n = (int)a.cols - (int)col;
    F2 w[kPairs], dw[kPairs];
    load_weights(a, col, n, w);
#pragma unroll
    for (int i = 0; i < kPairs; i++) dw[i] = F2(0.0f, 0.0f);
    uint32_t row = blockIdx.x * at_once + threadIdx.x / TPR;
    const uint8_t* codes_at = a.codes + row * a.code_stride + col;
    const uint8_t* scale_at = a.scales + (uint64_t)row * a.blocks + col / kBlock;
    const T* dy_at = static_cast<const T*>(a.dy) + row * a.dy_stride + col;
    const T* dres_at = static_cast<const T*>(a.dres) + row * a.dres_stride + col;
    T* out = static_cast<T*>(a.out) + row * a.out_stride + col;
    GradRow<DT> next;
    auto fetch = [&]() {
        if (n >= kRun) {
            next.codes = __ldcs(reinterpret_cast<const uint4*>(codes_at));
            next.dy.load(dy_at);
            if (a.dres) next.dres.load(dres_at);
        } else if (n > 0) {
            next.codes = load_codes(codes_at, n);
            next.dy.load_part(dy_at, n);
            if (a.dres) next.dres.load_part(dres_at, n);
        }
        next.byte = n > 0 ? *scale_at : 0u;
        codes_at += (uint64_t)jump * a.code_stride;
        scale_at += (uint64_t)jump * a.blocks;
        dy_at += (uint64_t)jump * a.dy_stride;
        dres_at += (uint64_t)jump * a.dres_stride;
    };
    if (kAhead && row < rows) fetch();
    // (the TPR threads that share a barrier take the same number of steps)
    for (uint32_t step = 0; row < rows; row += jump, step++) {
        if (!kAhead) fetch();
        GradRow<DT> now = next;
        const float s = pow2((int)now.byte - 127);
        float sq = 0.0f, dot = 0.0f;
        if (n > 0) {
            F2 acc(0.0f, 0.0f), acc2(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < kPairs; i += 2) {
                F2 c[2], d[2];
                now.four(i / 2, c, d);
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    acc = fma2(c[q], c[q], acc);
                    acc2 = fma2(mul2(d[q], w[i + q]), c[q], acc2);
                }
            }
            sq = s * (s * add_pairs(acc));
            dot = s * add_pairs(acc2);
        }
        if (kAhead && row + jump < rows) fetch();
        const float2 sums = sum(sq, dot, step);
        const float rstd = 1.0f / sqrtf(sums.x / (float)a.cols + a.eps);
        const float pull = sums.y / (float)a.cols * rstd * rstd;
        if (n > 0) {
            const F2 to_dw(s * rstd, s * rstd), from_x(-(s * pull) * rstd, -(s * pull) * rstd), from_dy(rstd, rstd);
            now.keep_packed();
            Run<DT> run;
#pragma unroll
            for (int i = 0; i < kPairs; i += 2) {
                F2 c[2], d[2], r[2];
                now.four(i / 2, c, d);
                if (a.dres) now.four_dres(i / 2, r);
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    dw[i + q] = fma2(d[q], mul2(c[q], to_dw), dw[i + q]);
                    const F2 g = fma2(mul2(d[q], w[i + q]), from_dy, mul2(c[q], from_x));
                    r[q] = a.dres ? add2(g, r[q]) : g;
                }
                set_four(run, i / 2, r);
            }
            if (n >= kRun) run.store(out);
            else run.store_part(out, n);
        }
        out += (uint64_t)jump * a.out_stride;
    }
    if (!a.partial) return;
    float* part = a.partial + (uint64_t)blockIdx.x * a.cols;
    float f[kRun];
#pragma unroll
    for (int i = 0; i < kPairs; i++) dw[i].get(f[2 * i], f[2 * i + 1]);
    if constexpr (TPR < THREADS) {
        // the CTA's groups have the same columns: the first to the last, in turn
        __shared__ float shared[TPR * kRun];
        for (int turn = 0; turn < (int)at_once; turn++) {
            if (threadIdx.x / TPR == turn)
#pragma unroll
                for (int i = 0; i < kRun; i++) shared[i * TPR + lane] = turn ? shared[i * TPR + lane] + f[i] : f[i];
            __syncthreads();
        }
        for (uint32_t j = threadIdx.x; j < a.cols; j += THREADS) part[j] = shared[j % kRun * TPR + j / kRun];
    } else if (n >= kRun && a.cols % 4 == 0) {
#pragma unroll
        for (int i = 0; i < kRun; i += 4) *reinterpret_cast<float4*>(part + col + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < kRun; i++)
            if (i < n) part[col + i] = f[i];
    }
    if (a.dweight) add_parts_in_cluster(a);
}

// Rows that start anywhere: thread t of the TPR that have a row takes columns t, t + TPR, ..., K at most, one element per
// access (a warp's 32 are side by side); the next row's are on their way.  Bound by its many accesses.  TPR and K by the
// width, as measured (bf16; eight columns of every thread beside it): gradient, 20000 x 300 38 us (89), 20000 x 1001 70 (96),
// 16384 x 4001 264 (289), 9000 x 6001 364 (458, less room per SM); forward, 20000 x 300 23 (31), 9000 x 1501 38 (55).
// There eight are better where four would be added up over more warps: 20000 x 1001 37 (39 of four), 16384 x 4001 103 (191).

// one code without its scale
__device__ __forceinline__ float code_value(uint8_t code) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)code));
    return __half2float(__ushort_as_half((uint16_t)h));
}

// A thread's columns of one row: codes, and the scales of the blocks they lie in.
template <int TPR, int K>
struct Columns {
    uint8_t code[K], byte[K];

    __device__ __forceinline__ void load(const NormArgs& a, uint32_t row, uint32_t lane) {
        const uint8_t* c = a.codes + row * a.code_stride + lane;
        const uint8_t* s = a.scales + (uint64_t)row * a.blocks + lane / kBlock;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const bool in = lane + k * TPR < a.cols;
            code[k] = in ? c[k * TPR] : 0;
            byte[k] = in ? s[k * TPR / (int)kBlock] : 0;          // TPR = 32: a warp's columns lie in one block
        }
    }
    __device__ __forceinline__ float scale(int k) const { return pow2((int)byte[k] - 127); }
};

template <uint32_t DT, int TPR, int THREADS, int K>
__global__ void __launch_bounds__(THREADS)
norm_col_kernel(NormArgs a, uint32_t rows_per_cta) {
    using E = Elem<DT>;
    __shared__ RowSum<TPR, THREADS> sum;
    const uint32_t lane = threadIdx.x % TPR, rows = (uint32_t)a.rows;
    const uint32_t first = blockIdx.x * rows_per_cta + threadIdx.x / TPR, last = min(rows, (blockIdx.x + 1) * rows_per_cta);
    float w[K];
#pragma unroll
    for (int k = 0; k < K; k++) w[k] = lane + k * TPR < a.cols ? weight_at(a, lane + k * TPR) : 0.0f;
    Columns<TPR, K> next;
    if (first < last) next.load(a, first, lane);
    uint32_t step = 0;
    for (uint32_t row = first; row < last; row += THREADS / TPR, step++) {
        const Columns<TPR, K> x = next;
        if (row + THREADS / TPR < last) next.load(a, row + THREADS / TPR, lane);
        float c[K], sq = 0.0f;
#pragma unroll
        for (int k = 0; k < K; k++) {
            c[k] = code_value(x.code[k]);
            const float v = c[k] * x.scale(k);
            sq = fmaf(v, v, sq);
        }
        const float rstd = 1.0f / sqrtf(sum(sq, 0.0f, step).x / (float)a.cols + a.eps);
        if (a.rstd && lane == 0) a.rstd[row] = rstd;
        typename E::T* out = static_cast<typename E::T*>(a.out) + row * a.out_stride + lane;
#pragma unroll
        for (int k = 0; k < K; k++)
            if (lane + k * TPR < a.cols) out[k * TPR] = E::down(c[k] * (x.scale(k) * rstd) * w[k]);
    }
}

template <uint32_t DT, int TPR, int K>
struct GradColumns {
    Columns<TPR, K> x;
    typename Elem<DT>::T d[K], r[K];

    __device__ __forceinline__ void load(const NormArgs& a, uint32_t row, uint32_t lane) {
        using T = typename Elem<DT>::T;
        const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride + lane;
        const T* dres = static_cast<const T*>(a.dres) + row * a.dres_stride + lane;
        x.load(a, row, lane);
#pragma unroll
        for (int k = 0; k < K; k++) {
            const bool in = lane + k * TPR < a.cols;
            d[k] = in ? dy[k * TPR] : (T)0;
            r[k] = in && a.dres ? dres[k * TPR] : (T)0;
        }
    }
};

template <uint32_t DT, int TPR, int THREADS, int K>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
norm_grad_col_kernel(NormArgs a) {
    using E = Elem<DT>;
    using T = typename E::T;
    constexpr bool kAhead = K <= 4;            // two rows of eight columns would spill
    __shared__ RowSum<TPR, THREADS> sum;
    const uint32_t lane = threadIdx.x % TPR, rows = (uint32_t)a.rows, at_once = THREADS / TPR, jump = gridDim.x * at_once;
    float w[K], dw[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        w[k] = lane + k * TPR < a.cols ? weight_at(a, lane + k * TPR) : 0.0f;
        dw[k] = 0.0f;
    }
    uint32_t step = 0, row = blockIdx.x * at_once + threadIdx.x / TPR;
    GradColumns<DT, TPR, K> next;
    if (kAhead && row < rows) next.load(a, row, lane);
    for (; row < rows; row += jump, step++) {
        if (!kAhead) next.load(a, row, lane);
        const GradColumns<DT, TPR, K> now = next;
        if (kAhead && row + jump < rows) next.load(a, row + jump, lane);
        T* out = static_cast<T*>(a.out) + row * a.out_stride + lane;
        float sq = 0.0f, dot = 0.0f;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const float v = code_value(now.x.code[k]) * now.x.scale(k);
            sq = fmaf(v, v, sq);
            dot = fmaf(E::up(now.d[k]) * w[k], v, dot);
        }
        const float2 sums = sum(sq, dot, step);
        const float rstd = 1.0f / sqrtf(sums.x / (float)a.cols + a.eps);
        const float pull = sums.y / (float)a.cols * rstd * rstd;
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (lane + k * TPR >= a.cols) continue;
            const float c = code_value(now.x.code[k]), s = now.x.scale(k), dk = E::up(now.d[k]);
            dw[k] = fmaf(dk, c * (s * rstd), dw[k]);
            out[k * TPR] = E::down(fmaf(rstd, fmaf(-c, s * pull, dk * w[k]), a.dres ? E::up(now.r[k]) : 0.0f));
        }
    }
    if (!a.partial) return;
    float* part = a.partial + (uint64_t)blockIdx.x * a.cols;
    if constexpr (TPR < THREADS) {
        // the CTA's groups have the same columns: the first to the last, in turn
        __shared__ float shared[TPR * K];
        for (int turn = 0; turn < (int)at_once; turn++) {
            if (threadIdx.x / TPR == turn)
#pragma unroll
                for (int k = 0; k < K; k++) shared[lane + k * TPR] = turn ? shared[lane + k * TPR] + dw[k] : dw[k];
            __syncthreads();
        }
        for (uint32_t j = threadIdx.x; j < a.cols; j += THREADS) part[j] = shared[j];
    } else {
#pragma unroll
        for (int k = 0; k < K; k++)
            if (lane + k * TPR < a.cols) part[lane + k * TPR] = dw[k];
    }
    if (a.dweight) add_parts_in_cluster(a);
}

// dweight from the CTAs' partial sums: a CTA per 32 columns, each warp every 32nd part, then the warps in order.  Its
// launch is prepared while the gradient kernel still runs; it starts when that one's last CTA has left.
constexpr int kWeightThreads = 1024;

__global__ void __launch_bounds__(kWeightThreads)
norm_weight_kernel(const float* partial, uint32_t parts, uint32_t cols, float* dweight, uint32_t flags) {
    __shared__ float sums[kWeightThreads / 32][33];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = blockIdx.x * 32 + lane;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float s = 0.0f;
    if (j < cols)
#pragma unroll 8
        for (uint32_t p = warp; p < parts; p += kWeightThreads / 32) s += partial[(uint64_t)p * cols + j];
    sums[warp][lane] = s;
    __syncthreads();
    // warp w: columns w of the 32, a lane per warp that summed
    s = sums[lane][warp];
#pragma unroll
    for (int mask = 16; mask >= 1; mask >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, mask);
    const uint32_t out = blockIdx.x * 32 + warp;
    if (lane == 0 && out < cols) dweight[out] = flags & RLCU_ACT8_ACCUMULATE ? dweight[out] + s : s;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// CTAs the rows of a gradient are dealt to, at most: what the registers of 148 SMs hold of the kernels for that width
uint64_t norm_parts(uint64_t rows, uint64_t cols) {
    const uint64_t most = 148 * (cols <= 1024 ? 4 : 2);
    return rows < most ? rows : most;
}

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

Span scales_of(const uint8_t* scales, uint64_t rows, uint64_t cols) { return bytes_of(scales, rows * rlcu_act8_blocks(cols)); }

// the same buffer, or none of it
bool same_or_apart(const void* p, uint64_t ps, const void* q, uint64_t qs, uint64_t rows, uint64_t cols, size_t esz) {
    if (p == q && (ps == qs || rows <= 1)) return true;
    return !rows_overlap({p, cols * esz, ps * esz}, {q, cols * esz, qs * esz}, rows);
}

// every row starts on a 16-byte boundary
bool rows16(const void* p, uint64_t stride, size_t esz, uint64_t rows) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows <= 1 || stride * esz % 16 == 0);
}

int grid_for(uint64_t units, int per_sm, int* out) {
    int dev = 0, sms = 0;
    RLCU_CUDA(cudaGetDevice(&dev));
    RLCU_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    const uint64_t most = (uint64_t)sms * per_sm;
    *out = (int)(units < most ? units : most);
    return RLCU_OK;
}

constexpr uint64_t kMostVecCols = 8192;

template <uint32_t DT, int TPR, int THREADS>
int launch_norm_vec(const NormArgs& a, cudaStream_t s) {
    // a few rows per CTA, so that their weights are read once for them; the grid moves through memory in order
    uint32_t per = THREADS / TPR * 8;
    while (per > THREADS / TPR * 2 && a.rows / per < 148 * 2048 / THREADS) per /= 2;
    norm_vec_kernel<DT, TPR, THREADS><<<(unsigned)((a.rows + per - 1) / per), THREADS, 0, s>>>(a, per);
    RLCU_CUDA(cudaGetLastError());
    return RLCU_OK;
}

template <uint32_t DT, int TPR, int THREADS, int K>
int launch_norm_col(const NormArgs& a, cudaStream_t s) {
    uint32_t per = THREADS / TPR * 8;
    while (per > THREADS / TPR && a.rows / per < 148 * 2048 / THREADS) per /= 2;
    norm_col_kernel<DT, TPR, THREADS, K><<<(unsigned)((a.rows + per - 1) / per), THREADS, 0, s>>>(a, per);
    RLCU_CUDA(cudaGetLastError());
    return RLCU_OK;
}

template <uint32_t DT>
int launch_norm(const NormArgs& a, bool vec, cudaStream_t s) {
    if (vec) {
        if (a.cols <= 512) return launch_norm_vec<DT, 32, 256>(a, s);
        if (a.cols <= 1024) return launch_norm_vec<DT, 64, 64>(a, s);
        if (a.cols <= 2048) return launch_norm_vec<DT, 128, 128>(a, s);
        if (a.cols <= 4096) return launch_norm_vec<DT, 256, 256>(a, s);
        return launch_norm_vec<DT, 512, 512>(a, s);
    }
    if (a.cols <= 128) return launch_norm_col<DT, 32, 256, 4>(a, s);
    if (a.cols <= 512) return launch_norm_col<DT, 128, 256, 4>(a, s);
    if (a.cols <= 1024) return launch_norm_col<DT, 128, 256, 8>(a, s);
    if (a.cols <= 2048) return launch_norm_col<DT, 512, 512, 4>(a, s);
    if (a.cols <= 4096) return launch_norm_col<DT, 512, 512, 8>(a, s);
    if (a.cols <= kMostVecCols) return launch_norm_col<DT, 1024, 1024, 8>(a, s);
    int grid = 0;
    if (const int rc = grid_for(a.rows, 8, &grid)) return rc;
    norm_kernel<DT><<<grid, kAct8Threads, 0, s>>>(a);
    RLCU_CUDA(cudaGetLastError());
    return RLCU_OK;
}

// A few steps of rows (kClusterSteps of 256 threads, fewer of more) are one cluster's work, which adds the partial sums
// itself.  Per call through the binding: 77 x 1001 f32 12.0 us, 13.7 with the second launch; 64 x 4096 bf16 12.5, 15.2; 96 x
// 8192 would take 16.9, 14.3 with it.
constexpr uint64_t kClusterSteps = 96;

template <typename Kernel>
int launch_grad_kernel(Kernel kernel, NormArgs a, int threads, uint64_t steps, uint64_t most, float* dweight, uint32_t flags, int* parts, cudaStream_t s) {
    *parts = (int)(steps < most ? steps : most);
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = {};
    if (dweight && steps * threads <= kClusterSteps * 256) {
        int cluster = 1;
        while (cluster < 16 && (uint64_t)cluster * 2 <= steps) cluster *= 2;
        if (cluster > 8) RLCU_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = cluster;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        a.dweight = dweight;
        a.flags = flags;
        *parts = cluster;
    }
    cfg.gridDim = dim3(*parts);
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    RLCU_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
    if (a.dweight) *parts = -1;                        // nothing is left to add
    return RLCU_OK;
}

template <uint32_t DT, int TPR, int THREADS>
int launch_norm_grad_vec(const NormArgs& a, float* dweight, uint32_t flags, int* parts, cudaStream_t s) {
    constexpr uint64_t kAtOnce = THREADS / TPR;
    return launch_grad_kernel(norm_grad_vec_kernel<DT, TPR, THREADS>, a, THREADS, (a.rows + kAtOnce - 1) / kAtOnce, 148 * (THREADS <= 256 ? 2 : 1), dweight, flags, parts, s);
}

template <uint32_t DT, int TPR, int THREADS, int K>
int launch_norm_grad_col(const NormArgs& a, float* dweight, uint32_t flags, int* parts, cudaStream_t s) {
    constexpr uint64_t kAtOnce = THREADS / TPR;
    return launch_grad_kernel(norm_grad_col_kernel<DT, TPR, THREADS, K>, a, THREADS, (a.rows + kAtOnce - 1) / kAtOnce, 148 * 1024 / THREADS, dweight, flags, parts, s);
}

template <uint32_t DT>
int launch_norm_grad(const NormArgs& a, bool vec, float* dweight, uint32_t flags, int* parts, cudaStream_t s) {
    if (vec) {
        if (a.cols <= 512) return launch_norm_grad_vec<DT, 32, 256>(a, dweight, flags, parts, s);
        if (a.cols <= 1024) return launch_norm_grad_vec<DT, 64, 256>(a, dweight, flags, parts, s);
        if (a.cols <= 2048) return launch_norm_grad_vec<DT, 128, 256>(a, dweight, flags, parts, s);
        if (a.cols <= 4096) return launch_norm_grad_vec<DT, 256, 256>(a, dweight, flags, parts, s);
        return launch_norm_grad_vec<DT, 512, 512>(a, dweight, flags, parts, s);
    }
    if (a.cols <= 128) return launch_norm_grad_col<DT, 32, 256, 4>(a, dweight, flags, parts, s);
    if (a.cols <= 512) return launch_norm_grad_col<DT, 128, 256, 4>(a, dweight, flags, parts, s);
    if (a.cols <= 1024) return launch_norm_grad_col<DT, 256, 256, 4>(a, dweight, flags, parts, s);
    if (a.cols <= 2048) return launch_norm_grad_col<DT, 512, 512, 4>(a, dweight, flags, parts, s);
    if (a.cols <= 4096) return launch_norm_grad_col<DT, 1024, 1024, 4>(a, dweight, flags, parts, s);
    if (a.cols <= kMostVecCols) return launch_norm_grad_col<DT, 1024, 1024, 8>(a, dweight, flags, parts, s);
    *parts = (int)norm_parts(a.rows, a.cols);
    norm_grad_kernel<DT><<<*parts, kAct8Threads, 0, s>>>(a);
    RLCU_CUDA(cudaGetLastError());
    return RLCU_OK;
}

}  // namespace
}  // namespace rlcu

using namespace rlcu;

extern "C" uint64_t rlcu_act8_blocks(uint64_t cols) { return (cols + kBlock - 1) / kBlock; }

extern "C" uint64_t rlcu_act8_rmsnorm_grad_workspace(uint64_t rows, uint64_t cols) { return norm_parts(rows, cols) * cols * sizeof(float); }

extern "C" int rlcu_act8_store(const void* x, uint32_t dtype, uint64_t rows, uint64_t cols, uint64_t x_stride,
                               uint8_t* codes, uint64_t code_stride, uint8_t* scales, void* stream) {
    if (const int rc = check_held(codes, code_stride, scales, rows, cols)) return rc;
    if (const int rc = check_matrix("x", x, dtype, rows, cols, x_stride)) return rc;
    if (!rows || !cols) return RLCU_OK;
    if (rows_overlap({x, cols * dtype_bytes(dtype), x_stride * dtype_bytes(dtype)}, {codes, cols, code_stride}, rows))
        return set_error(RLCU_ERR_INVALID, "x and codes overlap");
    const Span held = scales_of(scales, rows, cols);
    if (overlaps_rows(held, x, rows, cols, x_stride, dtype_bytes(dtype)) || overlaps_rows(held, codes, rows, cols, code_stride, 1))
        return set_error(RLCU_ERR_INVALID, "scales overlap x or codes");
    cudaStream_t s = (cudaStream_t)stream;
    const uint64_t blocks = rlcu_act8_blocks(cols), total = rows * blocks;
    if (rows16(x, x_stride, dtype_bytes(dtype), rows) && rows16(codes, code_stride, 1, rows) && total <= 0x7FFFFFFFull) {
        const unsigned grid = (unsigned)((total + kVecBlocks - 1) / kVecBlocks);
#define RLCU_STORE(DT) act8_store_vec_kernel<DT><<<grid, kAct8Threads, 0, s>>>(x, (uint32_t)total, (uint32_t)blocks, (uint32_t)cols, x_stride, codes, code_stride, scales)
        if (dtype == RLCU_F16) RLCU_STORE(RLCU_F16);
        else if (dtype == RLCU_BF16) RLCU_STORE(RLCU_BF16);
        else RLCU_STORE(RLCU_F32);
#undef RLCU_STORE
    } else {
        const uint64_t warps = rows * ((blocks + kWarpBlocks - 1) / kWarpBlocks), ctas = (warps + kAct8Threads / 32 - 1) / (kAct8Threads / 32);
        if (ctas > 0x7FFFFFFFull) return set_error(RLCU_ERR_INVALID, "too many rows for rows that are not 16-byte aligned");
        const unsigned grid = (unsigned)ctas;
        if (dtype == RLCU_F16) act8_store_kernel<RLCU_F16><<<grid, kAct8Threads, 0, s>>>(x, rows, (uint32_t)cols, x_stride, codes, code_stride, scales);
        else if (dtype == RLCU_BF16) act8_store_kernel<RLCU_BF16><<<grid, kAct8Threads, 0, s>>>(x, rows, (uint32_t)cols, x_stride, codes, code_stride, scales);
        else act8_store_kernel<RLCU_F32><<<grid, kAct8Threads, 0, s>>>(x, rows, (uint32_t)cols, x_stride, codes, code_stride, scales);
    }
    RLCU_CUDA(cudaGetLastError());
    return RLCU_OK;
}

extern "C" int rlcu_act8_load(const uint8_t* codes, uint64_t code_stride, const uint8_t* scales, uint64_t rows, uint64_t cols,
                              void* x, uint32_t dtype, uint64_t x_stride, void* stream) {
    if (const int rc = check_held(codes, code_stride, scales, rows, cols)) return rc;
    if (const int rc = check_matrix("x", x, dtype, rows, cols, x_stride)) return rc;
    if (!rows || !cols) return RLCU_OK;
    if (rows_overlap({x, cols * dtype_bytes(dtype), x_stride * dtype_bytes(dtype)}, {codes, cols, code_stride}, rows))
        return set_error(RLCU_ERR_INVALID, "x and codes overlap");
    if (overlaps_rows(scales_of(scales, rows, cols), x, rows, cols, x_stride, dtype_bytes(dtype)))
        return set_error(RLCU_ERR_INVALID, "scales and x overlap");
    cudaStream_t s = (cudaStream_t)stream;
    const uint64_t blocks = rlcu_act8_blocks(cols), total = rows * blocks;
    if (rows16(x, x_stride, dtype_bytes(dtype), rows) && rows16(codes, code_stride, 1, rows) && total <= 0x7FFFFFFFull) {
        const unsigned grid = (unsigned)((total + kVecBlocks - 1) / kVecBlocks);
#define RLCU_LOAD(DT) act8_load_vec_kernel<DT><<<grid, kAct8Threads, 0, s>>>(codes, code_stride, scales, (uint32_t)total, (uint32_t)blocks, (uint32_t)cols, x, x_stride)
        if (dtype == RLCU_F16) RLCU_LOAD(RLCU_F16);
        else if (dtype == RLCU_BF16) RLCU_LOAD(RLCU_BF16);
        else RLCU_LOAD(RLCU_F32);
#undef RLCU_LOAD
    } else {
        const uint64_t warps = rows * ((blocks + kWarpBlocks - 1) / kWarpBlocks), ctas = (warps + kAct8Threads / 32 - 1) / (kAct8Threads / 32);
        if (ctas > 0x7FFFFFFFull) return set_error(RLCU_ERR_INVALID, "too many rows for rows that are not 16-byte aligned");
        const unsigned grid = (unsigned)ctas;
        if (dtype == RLCU_F16) act8_load_kernel<RLCU_F16><<<grid, kAct8Threads, 0, s>>>(codes, code_stride, scales, rows, (uint32_t)cols, x, x_stride);
        else if (dtype == RLCU_BF16) act8_load_kernel<RLCU_BF16><<<grid, kAct8Threads, 0, s>>>(codes, code_stride, scales, rows, (uint32_t)cols, x, x_stride);
        else act8_load_kernel<RLCU_F32><<<grid, kAct8Threads, 0, s>>>(codes, code_stride, scales, rows, (uint32_t)cols, x, x_stride);
    }
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
    if (!words_aligned({rstd})) return set_error(RLCU_ERR_INVALID, "rstd: not aligned to its element size");
    if (!rows || !cols) return RLCU_OK;
    if (rows_overlap({y, cols * dtype_bytes(dtype), y_stride * dtype_bytes(dtype)}, {codes, cols, code_stride}, rows))
        return set_error(RLCU_ERR_INVALID, "y and codes overlap");
    const Span read[] = {scales_of(scales, rows, cols), bytes_of(weight, cols * dtype_bytes(weight_dtype))}, out = bytes_of(rstd, rows * 4);
    for (const Span& v : {read[0], read[1], out})
        if (overlaps_rows(v, y, rows, cols, y_stride, dtype_bytes(dtype))) return set_error(RLCU_ERR_INVALID, "y overlaps another buffer of the call");
    if (overlaps_any(out, {read[0], read[1]}) || overlaps_rows(out, codes, rows, cols, code_stride, 1))
        return set_error(RLCU_ERR_INVALID, "rstd overlaps another buffer of the call");
    NormArgs a = {codes, code_stride, scales, rows, (uint32_t)cols, (uint32_t)rlcu_act8_blocks(cols), weight, weight_dtype, eps,
                  nullptr, 0, nullptr, 0, y, y_stride, rstd, nullptr, nullptr, 0};
    cudaStream_t s = (cudaStream_t)stream;
    const bool vec = rows16(codes, code_stride, 1, rows) && rows16(y, y_stride, dtype_bytes(dtype), rows) && cols <= kMostVecCols;
    if (dtype == RLCU_F16) return launch_norm<RLCU_F16>(a, vec, s);
    if (dtype == RLCU_BF16) return launch_norm<RLCU_BF16>(a, vec, s);
    return launch_norm<RLCU_F32>(a, vec, s);
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
    if (!words_aligned({dweight})) return set_error(RLCU_ERR_INVALID, "dweight: not aligned to its element size");
    if (flags & ~(uint32_t)RLCU_ACT8_ACCUMULATE) return set_error(RLCU_ERR_INVALID, "unknown flags");
    const size_t esz = dtype_bytes(dtype);
    if (!same_or_apart(dx, dx_stride, dy, dy_stride, rows, cols, esz) ||
        (dresidual && !same_or_apart(dx, dx_stride, dresidual, dresidual_stride, rows, cols, esz)) ||
        rows_overlap({dx, cols * esz, dx_stride * esz}, {codes, cols, code_stride}, rows))
        return set_error(RLCU_ERR_INVALID, "dx overlaps another buffer without being the same");
    const uint64_t need = rlcu_act8_rmsnorm_grad_workspace(rows, cols);
    if (dweight && need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < need))
        return set_error(RLCU_ERR_INVALID, "workspace: %llu bytes, 16-byte aligned, are needed", (unsigned long long)need);
    if (!cols) return RLCU_OK;
    const Span held = scales_of(scales, rows, cols), w = bytes_of(weight, cols * dtype_bytes(weight_dtype));
    const Span sums = bytes_of(dweight, cols * 4), parts_at = bytes_of(dweight ? workspace : nullptr, need);
    for (const Span& v : {held, w, sums, parts_at})
        if (overlaps_rows(v, dx, rows, cols, dx_stride, esz)) return set_error(RLCU_ERR_INVALID, "dx overlaps another buffer of the call");
    for (const Span& v : {sums, parts_at})
        if (overlaps_any(v, {held, w}) || overlaps_rows(v, codes, rows, cols, code_stride, 1) || overlaps_rows(v, dy, rows, cols, dy_stride, esz) ||
            (dresidual && overlaps_rows(v, dresidual, rows, cols, dresidual_stride, esz)))
            return set_error(RLCU_ERR_INVALID, "dweight or workspace overlaps what the call reads");
    if (overlap(sums, parts_at)) return set_error(RLCU_ERR_INVALID, "dweight and workspace overlap");
    cudaStream_t s = (cudaStream_t)stream;
    NormArgs a = {codes, code_stride, scales, rows, (uint32_t)cols, (uint32_t)rlcu_act8_blocks(cols), weight, weight_dtype, eps,
                  dy, dy_stride, dresidual, dresidual_stride, dx, dx_stride, nullptr,
                  dweight ? static_cast<float*>(workspace) : nullptr, nullptr, 0};
    const bool vec = rows16(codes, code_stride, 1, rows) && rows16(dy, dy_stride, esz, rows) && rows16(dx, dx_stride, esz, rows) &&
                     (!dresidual || rows16(dresidual, dresidual_stride, esz, rows)) && cols <= kMostVecCols;
    int parts = 0;
    if (rows) {
        const int rc = dtype == RLCU_F16    ? launch_norm_grad<RLCU_F16>(a, vec, dweight, flags, &parts, s)
                       : dtype == RLCU_BF16 ? launch_norm_grad<RLCU_BF16>(a, vec, dweight, flags, &parts, s)
                                            : launch_norm_grad<RLCU_F32>(a, vec, dweight, flags, &parts, s);
        if (rc) return rc;
    }
    if (dweight && parts >= 0) {
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)((cols + 31) / 32));
        cfg.blockDim = dim3(kWeightThreads);
        cfg.stream = s;
        cfg.attrs = attr;
        cfg.numAttrs = parts ? 1 : 0;
        RLCU_CUDA(cudaLaunchKernelEx(&cfg, norm_weight_kernel, (const float*)a.partial, (uint32_t)parts, (uint32_t)cols, dweight, flags));
    }
    return RLCU_OK;
}
