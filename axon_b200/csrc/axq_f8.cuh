// Element types of the float tensors the 8-bit floating point and
// mixture-of-experts entry points take, and their conversions.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "../../include/axq.h"

namespace axq {

template <typename T> struct Elem;
template <> struct Elem<float> {
    __device__ __forceinline__ static float get(float v) { return v; }
    __device__ __forceinline__ static float put(float v) { return v; }
};
template <> struct Elem<__half> {
    __device__ __forceinline__ static float get(__half v) { return __half2float(v); }
    __device__ __forceinline__ static __half put(float v) { return __float2half_rn(v); }
};
template <> struct Elem<__nv_bfloat16> {
    __device__ __forceinline__ static float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    __device__ __forceinline__ static __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

inline int host_dtype_size(int dtype) {
    return dtype == AXQ_DT_F32 ? 4 : (dtype == AXQ_DT_F16 || dtype == AXQ_DT_BF16) ? 2 : 0;
}

// f.template operator()<T>() for the C type of `dtype` (already checked).
template <class Fn>
cudaError_t with_dtype(int dtype, Fn&& f) {
    switch (dtype) {
        case AXQ_DT_F32: return f(static_cast<float*>(nullptr));
        case AXQ_DT_F16: return f(static_cast<__half*>(nullptr));
        default: return f(static_cast<__nv_bfloat16*>(nullptr));
    }
}

// Eight consecutive elements at p (16-byte aligned) as floats.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
        T h[8];
        memcpy(h, w, 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = Elem<T>::get(h[i]);
    }
}

constexpr float kF8Max = 448.0f;  // largest e4m3 value
constexpr int kF8Block = 128;     // columns (and, for weights, rows) that share one scale

// Two e4m3 codes (RNE, saturating; NaN stays NaN): a in the low byte.
__device__ __forceinline__ uint32_t cvt_e4m3x2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}

// a / b rounded to nearest from y = RN(1/b): with q = RN(a*y) and r = q*b - a
// (exact in one FMA), RN(q - r*y) is the correctly rounded quotient unless b's
// significand is all ones (Markstein, "Computation of elementary functions on
// the IBM RISC System/6000 processor", 1990) and as long as r is exact and
// nothing overflows.  -0 stays -0 in this order.
__device__ __forceinline__ float div_by(float a, float b, float y) {
    const float q = __fmul_rn(a, y);
    return __fmaf_rn(-__fmaf_rn(q, b, -a), y, q);
}

// The cases that div_by does not cover, out of line: they are rare and their
// code, inlined at each element, filled the instruction cache.
static __device__ __noinline__ float div_slow(float a, float b) {
    if (b == 0.0f) return a != a ? a : 0.0f;
    return __fdiv_rn(a, b);
}

// Scale of a block with maximum m: RN(m / 448).
__device__ __forceinline__ float f8_scale(float m) {
    // outside 2^-100 .. 2^126 (0 and infinity among them) r might not be exact
    if (m > 7.8886091e-31f && m < 8.5070592e37f) return div_by(m, kF8Max, 1.0f / kF8Max);
    return __fdiv_rn(m, kF8Max);
}

// Codes of N elements under the scale s: two FMAs, a product and half a
// conversion each.  Where s is outside 2^-90 .. 2^90 or its significand is all
// ones the division itself is used; |x| < 2^-100 otherwise gives a quotient
// below 2^-10, whose code is 0 whether r is exact or not.
template <int N>
__device__ __forceinline__ void f8_codes(const float (&v)[N], float s, uint32_t (&w)[N / 4]) {
    float q[N];
    if (s > 8.0779357e-28f && s < 1.2379400e27f && (__float_as_uint(s) & 0x7FFFFFu) != 0x7FFFFFu) {
        const float y = __frcp_rn(s);
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = div_by(v[i], s, y);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = div_slow(v[i], s);
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
        w[i] = cvt_e4m3x2(q[4 * i], q[4 * i + 1]) | (cvt_e4m3x2(q[4 * i + 2], q[4 * i + 3]) << 16);
}

// Elements c0 .. c0+7 of a row of `cols` (zero past them).
template <typename T, bool VEC>
__device__ __forceinline__ void load_row8(const T* row, int64_t c0, int64_t cols, float (&v)[8]) {
    if (VEC && c0 + 8 <= cols) {
        load8(row + c0, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c0 + i < cols ? Elem<T>::get(row[c0 + i]) : 0.0f;
    }
}

// A 1 x 128 block held by 16 lanes, 8 elements each (all 32 lanes of the warp
// call it): its scale, and the lane's 8 codes.
__device__ __forceinline__ float pack_block16(const float (&v)[8], uint32_t (&w)[2]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
#pragma unroll
    for (int d = 8; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
    const float s = f8_scale(m);
    f8_codes(v, s, w);
    return s;
}

}  // namespace axq
