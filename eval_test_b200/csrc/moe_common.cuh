// Shared by the mixture-of-experts kernels: element types by their code in the C ABI, and vector access to them.
//
// T tokens choose k of E experts each; a copy i = t*k + j is one choice.  Sorted stably by expert the copies fill the
// rows 0 .. live-1 of a buffer of T*k rows; copies whose expert id lies outside [0, E) have no row.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "nvfp4_internal.h"
#include "ptx_sm100.cuh"

namespace nvfp4 {

constexpr int MOE_MAX_EXPERTS = 1024;
constexpr int MOE_MAX_CHOICES = 32;

// KIND: the element type codes of the C ABI (NVFP4_F32 / NVFP4_F16 / NVFP4_BF16).
template <int KIND> struct ElemOf { using type = float; };
template <> struct ElemOf<NVFP4_F16> { using type = __half; };
template <> struct ElemOf<NVFP4_BF16> { using type = __nv_bfloat16; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements, read or written as one access (N * sizeof(T) = 2 .. 32 bytes, aligned to its size, at most 16).
template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Vec {
    T v[N];
};

inline int elem_bytes(int kind) { return kind == NVFP4_F32 ? 4 : 2; }
inline bool kind_ok(int kind) { return kind == NVFP4_F32 || kind == NVFP4_F16 || kind == NVFP4_BF16; }

}  // namespace nvfp4
