// Rotary positions: the angle of a pair of columns and the turned values, for the kernels that turn q and k (rotary.cu) and
// the one that turns k on its way into a cache (paged_ops.cu).  And the scale of a row of 8-bit codes, for the latter and for
// attention over such caches (paged_attention.cu).
#pragma once

#include "../../include/attn_b200.h"
#include "sm100.cuh"

namespace b200 {

// (cos, sin) of `position` * `turns` / 2^64 full turns.  The 64-bit product wraps at whole turns, so the range reduction is
// exact for any position and the error of the angle is that of `turns` itself, 2^-64 turns a position, plus 2^-32 turns of
// what is dropped here.  In 32 bits position * frequency is off by 0.03 radians at position 2^20.
// kExact: sincospif (2 ulp), for results in 32 bits.  Otherwise the special-function unit on the reduced angle: off by 2^-21
// at most, a 2^-12th of a 16-bit rounding.
template <bool kExact>
__device__ __forceinline__ float2 rotary_cos_sin(uint64_t turns, long long position, float magnitude, bool inverse) {
  const int part = static_cast<int>((turns * static_cast<uint64_t>(position)) >> 32);   // signed: [-1/2, 1/2) of a turn
  float c, s;
  if constexpr (kExact) {
    sincospif(static_cast<float>(part) * 4.656612873077393e-10f, &s, &c);   // 2^-31: half turns
  } else {
    const float angle = static_cast<float>(part) * 1.4629180792671596e-09f;   // 2 pi / 2^32
    s = __sinf(angle);
    c = __cosf(angle);
  }
  return make_float2(c * magnitude, (inverse ? -s : s) * magnitude);
}

__device__ __forceinline__ void rotary_turn(float& a, float& b, float2 cs) {
  const float x = a, y = b;
  a = fmaf(x, cs.x, -y * cs.y);
  b = fmaf(y, cs.x, x * cs.y);
}

// two 16-bit values of a word as floats
template <bool kBf16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (kBf16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// The least e with a value of these bits (without sign) <= 448 * 2^e = 1.75 * 2^(8 + e); down to -127 - 8 for zero.
__device__ __forceinline__ int code_exponent(uint32_t top) {
  return static_cast<int>(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
}

}  // namespace b200
