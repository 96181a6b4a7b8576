// Element types of the operators whose activations may be fp32, bf16 or fp16 (NEMO_ELT_*): the
// arithmetic is fp32 throughout, a value is rounded once (to nearest even) where it is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"
#include "f32x2.cuh"

namespace nb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// N consecutive elements as one aligned vector (N * sizeof(T) = 4, 8 or 16 bytes; 32 as two of 16).
template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Vec {
    T v[N];
};

inline int elt_size(int elt) { return elt == NEMO_ELT_F32 ? 4 : 2; }
inline bool elt_ok(int elt) { return elt == NEMO_ELT_F32 || elt == NEMO_ELT_BF16 || elt == NEMO_ELT_F16; }

}  // namespace nb

// Runs the statement with T as the element type of `elt`.
#define NB_ELT_SWITCH(elt, T, ...)                                        \
    switch (elt) {                                                        \
        case NEMO_ELT_F32: { using T = float; __VA_ARGS__; } break;          \
        case NEMO_ELT_BF16: { using T = __nv_bfloat16; __VA_ARGS__; } break; \
        default: { using T = __half; __VA_ARGS__; } break;                   \
    }
