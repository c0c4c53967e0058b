// rotary.hpp -- rotary positions: pairs of a head's values turned by angles that grow with a
// token's place.  Shared by the operator itself and by what puts keys into a cache.
//   pair j: y1 = m (x1 cos a - x2 sin a), y2 = m (x2 cos a + x1 sin a), a = place * f_j
#pragma once

#include "nn_common.hpp"

namespace tpo {

// Sine and cosine of an angle in 64 bits: the nearest multiple of pi / 2 taken off (in two
// parts, so that what is left is exact to 2^-53 of the angle), then Taylor's series on
// [-pi / 4, pi / 4], whose next terms are under 5e-17.  Places reach millions, where 32 bits
// would leave angles off by tenths; the sixteen products of the series take no time beside a
// token's heads, which share them.  Angles beyond 2^45, and what is not finite, give NaN.
__device__ __forceinline__ void sine_cosine(double a, double& s, double& c) {
  const double n = rint(a * 0.63661977236758134308);
  double r = __builtin_fma(-n, 1.5707963267948965580, a);
  r = __builtin_fma(-n, 6.1232339957367658861e-17, r);
  const double z = r * r;
  double p = -1. / 1307674368000.;
  p = __builtin_fma(p, z, 1. / 6227020800.);
  p = __builtin_fma(p, z, -1. / 39916800.);
  p = __builtin_fma(p, z, 1. / 362880.);
  p = __builtin_fma(p, z, -1. / 5040.);
  p = __builtin_fma(p, z, 1. / 120.);
  p = __builtin_fma(p, z, -1. / 6.);
  const double sr = __builtin_fma(p * z, r, r);
  double q = 1. / 20922789888000.;
  q = __builtin_fma(q, z, -1. / 87178291200.);
  q = __builtin_fma(q, z, 1. / 479001600.);
  q = __builtin_fma(q, z, -1. / 3628800.);
  q = __builtin_fma(q, z, 1. / 40320.);
  q = __builtin_fma(q, z, -1. / 720.);
  q = __builtin_fma(q, z, 1. / 24.);
  q = __builtin_fma(q, z, -0.5);
  const double cr = __builtin_fma(q, z, 1.);
  const bool far = !(fabs(a) < 35184372088832.);  // 2^45
  const int k = far ? 0 : (int)((int64_t)n & 3);
  s = k & 1 ? cr : sr;
  c = k & 1 ? sr : cr;
  if (k & 2) s = -s;
  if ((k + 1) & 2) c = -c;
  if (far) s = c = __builtin_nan("");
}

constexpr int TURN_DMAX = 512;  // a head's values: its pieces are no more than a workgroup

// Angles of a call.  pairs = 0: nothing is turned.  Places are int64 or float, `axes` of a
// token; the pairs are shared out evenly among the axes.
struct Turn {
  const double* f;
  const void* at;
  int pairs, axes, each, interleaved, floats;  // each: pairs an axis
  double m;

  __device__ __forceinline__ double place(int64_t t, int pair) const {
    const int64_t i = t * axes + (axes > 1 ? pair / each : 0);
    return floats ? (double)((const float*)at)[i] : (double)((const int64_t*)at)[i];
  }
};
// Checks a call's angles and fills in t.
int turn_args(const char* op, const double* f, const void* at, int64_t pairs, int64_t axes,
              int floats, int interleaved, double m, int64_t D, Turn& t);

// How a head's D values are taken in pieces of 16 bytes: the pairs' (halves: two pieces of n
// pairs; interleaved: one of n / 2), then those that are left as they are.
template <typename T>
struct TurnPieces {
  static constexpr int PER = 16 / sizeof(T);
  int turned, all;
  __host__ __device__ __forceinline__ TurnPieces(int pairs, int interleaved, int D) {
    turned = interleaved ? (2 * pairs + PER - 1) / PER : (pairs + PER - 1) / PER;
    all = turned + (D - 2 * pairs + PER - 1) / PER;
  }
};

// n values from p (at any element) and back; `n` of them, PER at once where there are as many.
template <typename T, int PER>
__device__ __forceinline__ Piece<T, PER> some(const T* p, int n) {
  Piece<T, PER> v = {};
  if (n >= PER)
    v = *(const Piece<T, PER>*)p;
  else
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (e < n) v.v[e] = p[e];
  return v;
}
template <typename T, int PER>
__device__ __forceinline__ void put_some(T* p, const Piece<T, PER>& v, int n) {
  if (n >= PER)
    *(Piece<T, PER>*)p = v;
  else
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (e < n) p[e] = v.v[e];
}

// The rows of H heads of `tokens` tokens from t0 on, x strided, y (T, H, D): turned by cs
// (cosine and sine of a token's pairs, m times each, in LDS); a token whose `live` is 0 gives
// zeros.  THREADS of a workgroup go round (head, piece): pieces lie side by side in memory,
// then heads.
template <typename T, int THREADS>
__device__ __forceinline__ void turn_rows(const T* __restrict__ x, int64_t x_row, int64_t x_head,
                                          T* __restrict__ y, int H, int D, int64_t t0, int tokens,
                                          int pairs, int interleaved, const float2* cs,
                                          const int* live) {
  constexpr int PER = 16 / sizeof(T);
  const TurnPieces<T> pieces(pairs, interleaved, D);
  const int I = pieces.all, step = THREADS / I;
  const int i = threadIdx.x % I, r0 = threadIdx.x / I;
  if (r0 >= step) return;
  const int dt = step / H, dh = step % H;
  int t = r0 / H, h = r0 % H;
  const bool turned = i < pieces.turned;
  const int a = !turned ? 2 * pairs + (i - pieces.turned) * PER : i * PER;
  const int left = !turned ? D - a : (interleaved ? 2 * pairs : pairs) - a;
  for (; t < tokens; t += dt, h += dh) {
    if (h >= H) {
      h -= H;
      if (++t >= tokens) break;
    }
    const T* from = x + (t0 + t) * x_row + h * x_head + a;
    T* to = y + ((t0 + t) * H + h) * D + a;
    const bool on = !live || live[t];
    Piece<T, PER> u = on ? some<T, PER>(from, left) : Piece<T, PER>{};
    if (turned) {
      const float2* c = cs + t * pairs;
      if (interleaved) {
#pragma unroll
        for (int e = 0; e < PER; e += 2) {
          const float2 w = c[a / 2 + e / 2 < pairs ? a / 2 + e / 2 : 0];
          const float p = (float)u.v[e], q = (float)u.v[e + 1];
          u.v[e] = (T)__builtin_fmaf(-q, w.y, p * w.x);
          u.v[e + 1] = (T)__builtin_fmaf(p, w.y, q * w.x);
        }
      } else {
        Piece<T, PER> v = on ? some<T, PER>(from + pairs, left) : Piece<T, PER>{};
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const float2 w = c[a + e < pairs ? a + e : 0];
          const float p = (float)u.v[e], q = (float)v.v[e];
          u.v[e] = (T)__builtin_fmaf(-q, w.y, p * w.x);
          v.v[e] = (T)__builtin_fmaf(p, w.y, q * w.x);
        }
        put_some<T, PER>(to + pairs, on ? v : Piece<T, PER>{}, left);
      }
    }
    put_some<T, PER>(to, on ? u : Piece<T, PER>{}, left);
  }
}

}  // namespace tpo
