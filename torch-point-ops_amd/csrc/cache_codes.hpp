// cache_codes.hpp -- from a value in 64 bits to the code of an 8-bit cache: how it is rounded on
// the way, and the exponents of scales.  Arithmetic of one value, the same on the host.
#pragma once

#include "tpo_common.hpp"

namespace tpo {

constexpr int E_LEAST = -40, E_MOST = 40;
constexpr float CODE_MOST = 448.f;

// A double as a float whose last bit says that something was cut off (rounding to odd), so that
// the next rounding, to a code, is that of the double itself.  Keys are turned in 64 bits and
// rounded once in all: their codes are those of the exact products.  Which way the float went off
// is seen from d: the float of a small one is 0, and the least float of d's sign is then the odd
// one.  What is finite but beyond the floats becomes the largest of them (an infinity's bits less
// 1), which is odd; of an infinity nothing is cut off (the rest is NaN).
__host__ __device__ __forceinline__ float to_odd(double d) {
  const float f = (float)d;
  const double rest = d - (double)f;
  int b = __builtin_bit_cast(int, f);
  if (fabs(rest) > 0. && !(b & 1)) b += (rest > 0.) == (d > 0.) ? 1 : -1;
  return __builtin_bit_cast(float, b);
}
__host__ __device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_inff(); }

// The smallest e with top <= 448 2^e (448 = 0.875 2^9).
__host__ __device__ __forceinline__ int exponent_for(float top) {
  int e;
  const float m = frexpf(top, &e);
  e += m > 0.875f ? -8 : -9;
  if (top == 0.f || e < E_LEAST) e = E_LEAST;
  return e > E_MOST ? E_MOST : e;
}
// The smallest e with scale <= 2^e, for a scale from anywhere.
__host__ __device__ __forceinline__ int exponent_of(float scale) {
  if (!(scale > 0.f)) return E_LEAST;
  if (!finite(scale)) return E_MOST;
  int e;
  const float m = frexpf(scale, &e);
  if (m == 0.5f) --e;
  return e < E_LEAST ? E_LEAST : (e > E_MOST ? E_MOST : e);
}

}  // namespace tpo
