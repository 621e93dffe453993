// b3x_train_common.cuh -- element types and arithmetic shared by the training
// operators (include/b3x_train.h).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "b3x_train.h"

namespace b3t {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_huge_valf();

template <class T> __device__ __forceinline__ float to_float(T x) { return (float)x; }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <class T> __device__ __forceinline__ T from_float(float x) { return (T)x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }

// 2^x; about 2 ulp, results under the normal range are 0.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Two floats in one register pair, for the two-wide 32-bit arithmetic of sm_100.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Square roots of two numbers in [2^-96, 2^100], rounded as sqrtf rounds them:
// Newton's step from s = v y, y an approximate 1 / sqrt(v), with the residual
// v - s^2 formed by a fused operation (Markstein 1990).  What is left of the
// error before the last rounding, about 2^-45, decides no rounding of a 24-bit
// number (the tests compare all significands of two octaves with sqrtf).
// sqrtf's own cases for other numbers cost a branch a number.
__device__ __forceinline__ uint64_t sqrt2(uint64_t v) {
    const float2 x = unpack2(v);
    float2 y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(x.x));
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(x.y));
    const uint64_t y2 = pack2(y.x, y.y), s = mul2(v, y2), minus = mul2(s, pack2(-1.0f, -1.0f));
    const uint64_t half = mul2(y2, pack2(0.5f, 0.5f));
    return fma2(fma2(minus, s, v), half, s);
}

// Whether (rows, cols) elements at these strides are apart from one another.
inline bool apart(long long rows, long long cols, long long rs, long long cs) {
    if (rows < 2 && cols < 2) return true;
    if (rows < 2) return cs > 0;
    if (cols < 2) return rs > 0;
    if (rs <= 0 || cs <= 0) return false;
    return rs >= cs ? (rs - 1) / cs >= cols - 1 : (cs - 1) / rs >= rows - 1;
}

}  // namespace b3t
