// Shared by the mixture-of-experts kernels: element types by their code in the C ABI, and vector access to them.
//
// T tokens choose k of E experts each; a copy i = t*k + j is one choice.  Sorted stably by expert the copies fill the
// rows 0 .. live-1 of a buffer of T*k rows; copies whose expert id lies outside [0, E) have no row.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "nvfp4_internal.h"
#include "ptx_sm100.cuh"

namespace nvfp4 {

constexpr int MOE_MAX_EXPERTS = 1024;
constexpr int MOE_MAX_CHOICES = 32;
// Copies, and elements of a row: a loop's stride (at most 148 x 8 x 8 warps of four tokens) or 128 rows for each of 1024
// experts may be added to an index without leaving 31 bits.
constexpr long long MOE_MOST = (1ll << 31) - (1ll << 20);

// KIND: the element type codes of the C ABI (NVFP4_F32 / NVFP4_F16 / NVFP4_BF16).
template <int KIND> struct ElemOf { using type = float; };
template <> struct ElemOf<NVFP4_F16> { using type = __half; };
template <> struct ElemOf<NVFP4_BF16> { using type = __nv_bfloat16; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
// Unsigned word of a size: what is moved without being looked at.
template <int BYTES> struct Bits;
template <> struct Bits<16> { using type = uint4; };
template <> struct Bits<8> { using type = uint2; };
template <> struct Bits<4> { using type = uint32_t; };
template <> struct Bits<2> { using type = uint16_t; };

// 16 bytes that are read once (no line of L1 is kept for them).  A volatile asm stays behind the pdl_wait() before it.
__device__ __forceinline__ uint4 load_once(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// N consecutive elements (2, 4, 8, 16 or 32 bytes) kept as they lie in memory, two 16-bit elements to a register, until
// they are looked at: as arrays of 16-bit values the compiler gave each element a register of its own, and the kernels
// with eight vectors in flight fell to a quarter of the SM's threads.  Aligned to its size, at most 16 bytes.
template <typename T, int N>
struct Vec {
    static constexpr int BYTES = N * (int)sizeof(T), WORDS = (BYTES + 3) / 4;
    uint32_t w[WORDS];

    template <bool ONCE = false>
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (BYTES >= 16) {
#pragma unroll
            for (int i = 0; i < WORDS / 4; i++) {
                const uint4* at = reinterpret_cast<const uint4*>(p) + i;
                const uint4 v = ONCE ? load_once(at) : *at;
                w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
        } else if constexpr (BYTES == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x; w[1] = v.y;
        } else if constexpr (BYTES == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (BYTES >= 16) {
#pragma unroll
            for (int i = 0; i < WORDS / 4; i++)
                reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else if constexpr (BYTES == 8) {
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        } else if constexpr (BYTES == 4) {
            *reinterpret_cast<uint32_t*>(p) = w[0];
        } else {
            *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
        }
    }
    __device__ __forceinline__ float get(int q) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[q]);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(q & 1 ? w[q / 2] & 0xffff0000u : w[q / 2] << 16);
        else return __half2float(__ushort_as_half((unsigned short)(q & 1 ? w[q / 2] >> 16 : w[q / 2])));
    }
    // from fp32, one rounding to the nearest
    __device__ __forceinline__ void set(const float (&f)[N]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int q = 0; q < N; q++) w[q] = __float_as_uint(f[q]);
        } else if constexpr (N == 1) {
            if constexpr (std::is_same_v<T, __half>) w[0] = __half_as_ushort(__float2half_rn(f[0]));
            else w[0] = __bfloat16_as_ushort(__float2bfloat16_rn(f[0]));
        } else {
#pragma unroll
            for (int q = 0; q < N / 2; q++) {
                if constexpr (std::is_same_v<T, __half>) {
                    const __half2 h = __floats2half2_rn(f[2 * q], f[2 * q + 1]);
                    w[q] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * q], f[2 * q + 1]);
                    w[q] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
        }
    }
};

// Whether the addresses are those of 32-bit words (NULL is).
template <typename... P> bool words(const P*... p) { return ((0 | ... | (uintptr_t)p) & 3) == 0; }
inline int elem_bytes(int kind) { return kind == NVFP4_F32 ? 4 : 2; }
inline bool kind_ok(int kind) { return kind == NVFP4_F32 || kind == NVFP4_F16 || kind == NVFP4_BF16; }

}  // namespace nvfp4
