// Two fp32 values in a register pair: one instruction of the packed fp32 pipe for both; and the
// special-function units' exponential (base 2) and reciprocal, each within a few ulp.
#pragma once

namespace nb {

typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2(float lo, float hi) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(f2 v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f2 dup2(float v) { return pack2(v, v); }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rcp(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
constexpr float LOG2E = 1.4426950408889634f;

// 1 / (1 + e^-v): below v = -87.3, where it is less than 2^-126, it is 0; a NaN stays one
__device__ __forceinline__ float sigmoid_fast(float v) { return rcp(1.0f + ex2(v * -LOG2E)); }
__device__ __forceinline__ f2 sigmoid2(f2 v) {
    float a, b;
    unpack2(mul2(v, dup2(-LOG2E)), a, b);
    unpack2(add2(pack2(ex2(a), ex2(b)), dup2(1.0f)), a, b);
    return pack2(rcp(a), rcp(b));
}

}  // namespace nb
