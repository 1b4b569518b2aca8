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

// Eight features of a row held by L adjacent lanes (lanes past the row's width are not live): the
// lane's dword of codes, and the row's pair in every lane.
template <typename T, int L>
__device__ __forceinline__ uint32_t quantize_row8(const float (&x)[8], bool live, uint32_t& pair) {
  float lo = kInf, hi = -kInf, bad = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float f = 0.5f * x[e];
    if (live) {
      lo = __builtin_fminf(lo, f);
      hi = __builtin_fmaxf(hi, f);
      if (!(__builtin_fabsf(x[e]) < kInf)) bad = 1.f;
    }
  }
  lo = -group_max<L>(-lo);
  hi = group_max<L>(hi);
  bad = group_max<L>(bad);
  const T s = from_f32<T>(2.f * ((hi - lo) / 15.f));
  const float half = 0.5f * to_f32(s);
  uint32_t codes = 0;
  if (half > 0.f && bad == 0.f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float c = __builtin_rintf((0.5f * x[e] - lo) / half);
      codes |= (uint32_t)__builtin_fminf(__builtin_fmaxf(c, 0.f), 15.f) << (4 * e);
    }
  }
  const T nan = from_f32<T>(__builtin_nanf(""));
  pair = bad == 0.f ? pack_pair<T>(s, from_f32<T>(2.f * lo)) : pack_pair<T>(nan, nan);
  return codes;
}

template <typename T> constexpr float kFiniteMax = 0.f;
template <> constexpr float kFiniteMax<__bf16> = 3.38953139e38f;
template <> constexpr float kFiniteMax<_Float16> = 65504.f;

// A lane's eight features from its dword of codes. The top code may land past T's largest number by
// the rounding of s: it is brought back to it.
template <typename T, typename V8>
__device__ __forceinline__ V8 dequantize_row8(uint32_t codes, uint32_t pair) {
  const float s = pair_scale<T>(pair), lo = pair_low<T>(pair);
  V8 y;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float v = __builtin_fmaf(s, (float)((codes >> (4 * e)) & 15u), lo);
    if (v > kFiniteMax<T>) v = kFiniteMax<T>;
    if (v < -kFiniteMax<T>) v = -kFiniteMax<T>;
    y[e] = from_f32<T>(v);
  }
  return y;
}

}  // namespace vsp
