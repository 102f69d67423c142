// Element types of the operators that take FP16, bfloat16 or FP32 tensors: 16-byte groups unpacked to FP32
// and back (one rounding), single elements, and the alignment arithmetic of rows that start anywhere.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>

#include "rlcu_adamw.h"

namespace rlcu {

// Two FP32 values in a register pair: sm_100 multiplies and adds such pairs with one instruction.
struct F2 {
    unsigned long long v;
    __device__ __forceinline__ F2() {}
    __device__ __forceinline__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

template <uint32_t DT>
struct Elem {                                   // RLCU_F16 and RLCU_BF16
    using T = uint16_t;
    static constexpr int kVec = 8;              // elements of 16 bytes
    static constexpr bool kBF = DT == RLCU_BF16;

    static __device__ __forceinline__ float up(T x) {
        return kBF ? __uint_as_float((uint32_t)x << 16) : __half2float(__ushort_as_half(x));
    }
    static __device__ __forceinline__ T down(float x) {
        return kBF ? __bfloat16_as_ushort(__float2bfloat16_rn(x)) : __half_as_ushort(__float2half_rn(x));
    }
    static __device__ __forceinline__ void up2(uint32_t w, float& a, float& b) {
        if (kBF) {
            a = __uint_as_float(w << 16);
            b = __uint_as_float(w & 0xFFFF0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
            a = f.x;
            b = f.y;
        }
    }
    static __device__ __forceinline__ uint32_t down2(float a, float b) {
        if (kBF) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            return *reinterpret_cast<const uint32_t*>(&h);
        }
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ void unpack(uint4 x, float (&f)[kVec]) {
        up2(x.x, f[0], f[1]);
        up2(x.y, f[2], f[3]);
        up2(x.z, f[4], f[5]);
        up2(x.w, f[6], f[7]);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[kVec]) {
        return make_uint4(down2(f[0], f[1]), down2(f[2], f[3]), down2(f[4], f[5]), down2(f[6], f[7]));
    }
    // largest element of 16 bytes (NaN is passed over)
    static __device__ __forceinline__ float largest(uint4 x) {
        float a, b;
        if (kBF) {
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&x);
            const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            up2(*reinterpret_cast<const uint32_t*>(&m), a, b);
        } else {
            const __half2* h = reinterpret_cast<const __half2*>(&x);
            const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            up2(*reinterpret_cast<const uint32_t*>(&m), a, b);
        }
        return fmaxf(a, b);
    }
};

template <>
struct Elem<RLCU_F32> {
    using T = float;
    static constexpr int kVec = 4;
    static __device__ __forceinline__ float up(T x) { return x; }
    static __device__ __forceinline__ T down(float x) { return x; }
    static __device__ __forceinline__ void unpack(uint4 x, float (&f)[kVec]) {
        f[0] = __uint_as_float(x.x);
        f[1] = __uint_as_float(x.y);
        f[2] = __uint_as_float(x.z);
        f[3] = __uint_as_float(x.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[kVec]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
    static __device__ __forceinline__ float largest(uint4 x) {
        return fmaxf(fmaxf(__uint_as_float(x.x), __uint_as_float(x.y)), fmaxf(__uint_as_float(x.z), __uint_as_float(x.w)));
    }
};

// A row of n elements cut at 16-byte boundaries: `head` single elements, `groups` groups, then the rest.
struct RowCut {
    uint32_t head, groups;
};

template <typename T>
__device__ __forceinline__ RowCut cut_row(const T* row, uint32_t n) {
    const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15u) / (uint32_t)sizeof(T);
    constexpr uint32_t kVec = 16 / sizeof(T);
    uint32_t head = off ? kVec - off : 0u;
    if (head > n) head = n;
    return {head, (n - head) / kVec};
}

__host__ inline size_t dtype_bytes(uint32_t dtype) { return dtype == RLCU_F32 ? 4 : 2; }
__host__ inline bool dtype_known(uint32_t dtype) { return dtype == RLCU_F16 || dtype == RLCU_F32 || dtype == RLCU_BF16; }

// rows of `stride` elements that no address space could hold are refused before any product of the two is formed
__host__ inline bool too_large(uint64_t rows, uint64_t stride) { return rows && stride > (1ull << 48) / rows; }

// a rows x cols matrix with `stride` elements from row to row, as the bytes from its first to its last element
struct Span {
    uintptr_t lo, hi;
};
__host__ inline Span span_of(const void* p, uint64_t rows, uint64_t cols, uint64_t stride, size_t esz) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    return {lo, rows && cols ? lo + ((rows - 1) * stride + cols) * esz : lo};
}
__host__ inline bool overlap(Span a, Span b) { return a.lo < a.hi && b.lo < b.hi && a.lo < b.hi && b.lo < a.hi; }

__host__ inline Span bytes_of(const void* p, uint64_t bytes) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    return {lo, p ? lo + bytes : lo};
}
__host__ inline bool overlaps_any(Span a, std::initializer_list<Span> others) {
    for (const Span& o : others)
        if (overlap(a, o)) return true;
    return false;
}
// whether v shares a byte with one of the rows of a matrix (what lies between the rows is not the matrix's)
__host__ inline bool overlaps_rows(Span v, const void* p, uint64_t rows, uint64_t cols, uint64_t stride, size_t esz) {
    const Span all = span_of(p, rows, cols, stride, esz);
    if (!overlap(v, all)) return false;
    if (v.lo <= all.lo) return true;
    const uint64_t at = v.lo - all.lo, row = at / (stride * esz);
    return at < row * stride * esz + cols * esz || (row + 1 < rows && v.hi - all.lo > (row + 1) * stride * esz);
}

// Whether two matrices of `rows` rows share a byte.  With the same stride in bytes they may lie beside each other, column
// by column, in one buffer: row j of q then starts `in` bytes into row j + k of p's.  With other strides their extents decide.
struct RowBytes {
    const void* p;
    uint64_t row, stride;     // bytes
};
__host__ inline bool rows_overlap(RowBytes p, RowBytes q, uint64_t rows) {
    if (!rows || !p.row || !q.row) return false;
    if (p.stride != q.stride || rows == 1) return overlap(span_of(p.p, rows, p.row, p.stride, 1), span_of(q.p, rows, q.row, q.stride, 1));
    const int64_t d = (int64_t)(reinterpret_cast<uintptr_t>(q.p) - reinterpret_cast<uintptr_t>(p.p)), s = (int64_t)p.stride, n = (int64_t)rows;
    const int64_t k = d >= 0 ? d / s : -((-d + s - 1) / s), in = d - k * s;
    return (k > -n && k < n && (uint64_t)in < p.row) || (k + 1 > -n && k + 1 < n && (uint64_t)in + q.row > p.stride);
}

// vectors of 4-byte values (null: none), each aligned to them
__host__ inline bool words_aligned(std::initializer_list<const void*> vectors) {
    for (const void* p : vectors)
        if (reinterpret_cast<uintptr_t>(p) % 4) return false;
    return true;
}

}  // namespace rlcu
