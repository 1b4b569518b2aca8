// Rows of four-bit codes for the KV ring (gfx950): the quantiser and its inverse, shared by the
// ring's write, read and attention kernels.
//
// A row is the dk features of one token and KV head, in T (bf16 or fp16). With lo and hi its
// smallest and largest feature,
//   s = T((hi - lo) / 15),   code = clamp(round((x - lo) / s), 0, 15),   value = lo + s code,
// every operation one float32 rounding (the division is correctly rounded, ties to even), formed on
// halves so that hi - lo stays finite for all finite T. lo is a feature of the row, so T holds it
// exactly; s is rounded to T first and the codes are taken against the rounded one, so the pair
// (s, lo) that is stored is the pair the codes belong to (T's half step in s moves the top value by
// at most 15 s eps / 2: 6 % of a step in bf16, less than the half step of the codes themselves).
// s = 0 (equal features, or a range below T's smallest number) gives codes 0. A row with an infinity
// or a NaN is stored as s = lo = NaN with codes 0, so it reads back, and is attended, as NaN.
//
// Two codes a byte, the even feature in the low half: dword i of a row holds features 8 i .. 8 i + 7,
// feature 8 i + e in bits 4 e .. 4 e + 3. The pair (s, lo) is one dword, s in its low half.
#pragma once

#include "common.h"

namespace vsp {

constexpr float kInf = __builtin_inff();

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(T s, T lo) {
  return (uint32_t)__builtin_bit_cast(uint16_t, s) | ((uint32_t)__builtin_bit_cast(uint16_t, lo) << 16);
}
template <typename T>
__device__ __forceinline__ float pair_scale(uint32_t pair) {
  return to_f32(__builtin_bit_cast(T, (uint16_t)(pair & 0xffffu)));
}
template <typename T>
__device__ __forceinline__ float pair_low(uint32_t pair) {
  return to_f32(__builtin_bit_cast(T, (uint16_t)(pair >> 16)));
}

// The least and the greatest of three (one instruction, gfx950's): NaN where one of them is NaN.
__device__ __forceinline__ float min3(float x, float y, float z) {
  float r = x;
#if defined(__HIP_DEVICE_COMPILE__)
  asm("v_minimum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
#endif
  return r;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r = x;
#if defined(__HIP_DEVICE_COMPILE__)
  asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
#endif
  return r;
}
struct MinNanOp {
  __device__ __forceinline__ float operator()(float x, float y) const { return min3(x, y, y); }
};
struct MaxNanOp {
  __device__ __forceinline__ float operator()(float x, float y) const { return max3(x, y, y); }
};

// n / d correctly rounded for finite n and a normal d of at most 11 significant bits (15, or a scale rounded to bf16
// or fp16) with a normal 1 / d: a reciprocal within one unit and one Newton step on the residual, which fma forms
// exactly, are within 2^-46 of n / d before the last rounding, and no n / d lies within 2^-36 of the middle between two
// floats (a middle has 25 bits; its product with d is never n's 24 and is a whole unit of it away).
__device__ __forceinline__ float quotient(float n, float d, float reciprocal) {
  const float t = n * reciprocal;
  return __builtin_fmaf(__builtin_fmaf(-t, d, n), reciprocal, t);
}

// Eight features of a row held by L adjacent lanes (a lane past the row's width holds features of the row
// again, which change nothing): the lane's dword of codes, and the row's pair in every lane.
template <typename T, int L>
__device__ __forceinline__ uint32_t quantize_row8(const float (&x)[8], uint32_t& pair) {
  float lo = min3(min3(x[0], x[1], x[2]), min3(x[3], x[4], x[5]), min3(x[6], x[7], x[7]));
  float hi = max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max3(x[6], x[7], x[7]));
  lo = 0.5f * group_reduce<L>(lo, MinNanOp{});
  hi = 0.5f * group_reduce<L>(hi, MaxNanOp{});
  const float range = hi - lo;  // finite for finite features; infinite or NaN with an infinity or a NaN
  const bool fine = range < kInf;
  const T s = from_f32<T>(2.f * quotient(range, 15.f, 1.f / 15.f));
  const float half = 0.5f * to_f32(s);
  // Small steps are scaled up first (exactly), so that the reciprocal and the residual stay normal numbers;
  // the largest step, 2^124, has a normal reciprocal.
  // Not a step of 0, whose features may be of any size: it finds every quotient 0.
  const float up = __float_as_uint(half) - 1u < __float_as_uint(0x1p-60f) - 1u ? 0x1p80f : 1.f;
  const float step = half * up, low = lo * up, inv = half > 0.f ? __builtin_amdgcn_rcpf(step) : 0.f;
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float q = __builtin_fminf(quotient(__builtin_fmaf(x[e], 0.5f * up, -low), step, inv), 15.f);
    // 2^23 + 2^22 more: the sum's rounding is that of q to a whole number, ties to even, in its low bits
    codes += __float_as_uint(q + 12582912.f) << (4 * e);
  }
  codes -= 0x4B400000u * 0x11111111u;  // the sum's exponent bits of all eight
  const T nan = from_f32<T>(__builtin_nanf(""));
  pair = fine ? pack_pair<T>(s, from_f32<T>(2.f * lo)) : pack_pair<T>(nan, nan);
  return fine ? codes : 0u;
}

template <typename T> constexpr float kFiniteMax = 0.f;
template <> constexpr float kFiniteMax<__bf16> = 3.38953139e38f;
template <> constexpr float kFiniteMax<_Float16> = 65504.f;

// An average of numbers of T, formed as a / b: among them, so one that passes T's largest number, by the rounding of a
// scale, is brought back to it; an infinity or a NaN in the sum is kept.
template <typename T>
__device__ __forceinline__ float average(float a, float b) {
  const float x = a / b;
  const bool past = __builtin_fabsf(a) < kInf && __builtin_fabsf(x) > kFiniteMax<T>;
  return past ? __builtin_copysignf(kFiniteMax<T>, x) : x;
}

// A lane's eight features from its dword of codes. The top code may land past T's largest number by
// the rounding of s: it is brought back to it.
template <typename T, typename V8>
__device__ __forceinline__ V8 dequantize_row8(uint32_t codes, uint32_t pair) {
  const float s = pair_scale<T>(pair), lo = pair_low<T>(pair);
  const uint32_t even = codes & 0x0f0f0f0fu, odd = (codes >> 4) & 0x0f0f0f0fu;  // bytes: one instruction a float
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __builtin_fmaf(s, (float)((even >> (8 * i)) & 255u), lo);
    f[2 * i + 1] = __builtin_fmaf(s, (float)((odd >> (8 * i)) & 255u), lo);
  }
  if (__builtin_fmaf(15.f, s, lo) > kFiniteMax<T>) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = f[e] > kFiniteMax<T> ? kFiniteMax<T> : f[e];
  }
  V8 y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = from_f32<T>(f[e]);
  return y;
}

}  // namespace vsp
