// Angles of rotary positions, shared by nvkv_rope and nvkv_rope_append.
//
// The angle of pair i at position p is p * inv_freq[i].  It is formed in 64
// bits and reduced to a fraction of a turn there: at p = 10^5 an f32 product
// is already 2^-8 radians off.  With f = inv_freq / 2 pi, the fraction r = p f
// - rint(p f) lies in [-1/2, 1/2].  Three roundings (1 / 2 pi, the two products)
// put it off by at most 3 x 2^-53 of |p f|, so cos and sin inherit at most 3 x
// 2^-53 |p inv_freq|: 2^-27 at |p| = 2^24 and inv_freq = 1, a quarter of half an
// f32 ulp of 1.  The f32 form rounds r once more, 2^-24 of the reduced angle.
#pragma once

#include "common.cuh"

namespace nvkv {

constexpr double kInv2Pi = 0.15915494309189533577;

__device__ __forceinline__ double rope_turns(int64_t pos, double inv_freq) {
  const double t = (double)pos * (inv_freq * kInv2Pi);
  return t - rint(t);
}

// (a cos, a sin) of the angle in f32
__device__ __forceinline__ float2 rope_cs(int64_t pos, double inv_freq, float a) {
  float s, c;
  sincospif(2.0f * (float)rope_turns(pos, inv_freq), &s, &c);
  return make_float2(a * c, a * s);
}

// the same in f64
__device__ __forceinline__ double2 rope_cs64(int64_t pos, double inv_freq, double a) {
  double s, c;
  sincospi(2.0 * rope_turns(pos, inv_freq), &s, &c);
  return make_double2(a * c, a * s);
}

}  // namespace nvkv
