// Element types of the operators that take float32, float16 and bfloat16 tensors: conversions (round to nearest even) and groups of four.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

enum { LG_F32 = 0, LG_F16 = 1, LG_BF16 = 2 };

typedef _Float16 LgHalf;
struct LgBf16 { uint16_t bits; };

template <typename T> struct alignas(4 * sizeof(T)) LgVec4 { T v[4]; };

__device__ __forceinline__ float lg_to_float(float v) { return v; }
__device__ __forceinline__ float lg_to_float(LgHalf v) { return (float)v; }
__device__ __forceinline__ float lg_to_float(LgBf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }

template <typename T> __device__ __forceinline__ T lg_from_float(float v);
template <> __device__ __forceinline__ float lg_from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ LgHalf lg_from_float<LgHalf>(float v) { return (LgHalf)v; }
template <> __device__ __forceinline__ LgBf16 lg_from_float<LgBf16>(float v)
{
    const uint32_t b = __float_as_uint(v);
    if ((b & 0x7fffffffu) > 0x7f800000u) return LgBf16{ (uint16_t)((b >> 16) | 0x40u) };         // NaN stays NaN
    return LgBf16{ (uint16_t)((b + 0x7fffu + ((b >> 16) & 1u)) >> 16) };
}
