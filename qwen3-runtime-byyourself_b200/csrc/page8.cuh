// Rows of a cache that is kept in 8 bits: a row (one token's key or value of one kv head) is held as e4m3 codes and one
// scale, a power of two.
//
// The scale 2^k is the smallest one by which the row's largest value fits into e4m3's largest, 448; k lies in -60 .. 60
// (smaller rows lose their small values, larger ones saturate) and is stored as the byte k + 127.  A power of two costs
// no accuracy beside any other scale - the steps of e4m3 are relative to a value, not to the row's largest one - and
// makes x / 2^k and code * 2^k exact, the latter in bfloat16 too: what a row stands for does not hang on how it is computed.
// A value that is no number (infinity or NaN) becomes the NaN code; the largest value is taken over the others.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

constexpr int Q3_SCALE_LOW = -60, Q3_SCALE_HIGH = 60, Q3_SCALE_BIAS = 127;

__device__ __forceinline__ bool q3_is_number(float x) { return fabsf(x) <= 3.402823466e38f; }

// The exponent of the scale of a row whose largest value is `top` (finite, >= 0).
__device__ __forceinline__ int q3_scale_exponent(float top) {
    const uint32_t bits = __float_as_uint(top);
    const int k = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);      // 448 = 1.75 * 2^8
    return min(max(k, Q3_SCALE_LOW), Q3_SCALE_HIGH);
}
__device__ __forceinline__ float q3_exp2i(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }   // |k| <= 126

// Two values, divided by the scale, as codes (NaN stays NaN; an infinity has to be one already).
__device__ __forceinline__ uint32_t q3_codes2(float2 v, float inv_scale) {
    return __nv_cvt_float2_to_fp8x2(make_float2(v.x * inv_scale, v.y * inv_scale), __NV_SATFINITE, __NV_E4M3);
}
// Two codes (the low 16 bits) as the numbers they stand for, exact in half precision.
__device__ __forceinline__ __half2 q3_half2_of(uint32_t codes) {
    return __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3));
}
