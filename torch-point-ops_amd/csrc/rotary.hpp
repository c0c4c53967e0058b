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

// PER values as they come from memory.  They stay words until they are used: taken apart into
// values of two bytes where both ways of loading meet, they would be waited for right there.
template <typename T, int PER>
struct Loaded {
  static constexpr int N = PER * sizeof(T) / 4;
  uint32_t w[N];

  __device__ __forceinline__ void fresh() {  // what was worked out of them is not kept
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(w[i]));
  }
  __device__ __forceinline__ Piece<T, PER> values() const {
    Loaded o = *this;
    o.fresh();
    return __builtin_bit_cast(Piece<T, PER>, o);
  }
};
// n values from p (at any element), PER at once where there are as many; and back.
template <typename T, int PER>
__device__ __forceinline__ Loaded<T, PER> some(const T* p, int n) {
  typedef uint32_t words __attribute__((ext_vector_type(4)));
  typedef words anywhere __attribute__((aligned(2)));  // (of every type)
  Loaded<T, PER> v = {};
  if (n >= PER) {
#pragma unroll
    for (int i = 0; i < v.N; i += 4) {
      const words x = ((const anywhere*)p)[i / 4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v.w[i + j] = x[j];
    }
  } else {
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (e < n) {
        if constexpr (sizeof(T) == 4)
          v.w[e] = __builtin_bit_cast(uint32_t, p[e]);
        else
          v.w[e / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[e]) << 16 * (e % 2);
      }
  }
  return v;
}
// STREAM: past the caches.
template <bool STREAM, typename T, int PER>
__device__ __forceinline__ void put_some(T* p, const Piece<T, PER>& v, int n) {
  static_assert(PER * sizeof(T) == 16, "a piece is 16 bytes");
  if (n >= PER && STREAM) {
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    typedef words anywhere __attribute__((aligned(2)));  // (of every type)
    __builtin_nontemporal_store(__builtin_bit_cast(words, v), (anywhere*)p);
  } else if (n >= PER) {
    *(Piece<T, PER>*)p = v;
  } else
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (e < n) p[e] = v.v[e];
}

// Where a token's cosines and sines lie: for the pairs of each piece, two at a time, the pieces
// side by side, so that the lanes of a read (a piece each) touch all banks once.
template <typename T>
struct TurnAngles {
  int per, pieces, pitch;  // pairs of a piece, pieces, places of a token (some not used)
  __host__ __device__ __forceinline__ TurnAngles(int pairs, int interleaved) {
    per = (interleaved ? 8 : 16) / (int)sizeof(T);
    pieces = (pairs + per - 1) / per;
    pitch = pieces * per;
  }
  // the pair at a place
  __device__ __forceinline__ int pair(int place) const {
    const int i = place >> 1;
    return i % pieces * per + i / pieces * 2 + (place & 1);
  }
};

// A float in T, rounded as a float first: to half also in one instruction with the product, which
// rounds once; the compiler takes it in one kernel and not in another, whose results would
// differ.
template <typename T>
__device__ __forceinline__ T result(float v) {
  if constexpr (sizeof(T) == 2) asm("" : "+v"(v));
  return (T)v;
}

// The rows of H heads of `tokens` tokens from t0 on, x strided, y (T, H, D): turned by cs (cosine
// and sine of a token's pairs, m times each, in LDS).  THREADS of a workgroup go round (head,
// piece): pieces lie side by side in memory, then heads.  A thread's next piece is on its way
// while one is turned, the first while the angles are worked out.
// STREAM: the rows go past the caches, for more than these hold (TURN_STREAM): 32768 x 20 x 128
// in bfloat16, 336 MB there and back, 58 us (5.8 TB/s), through the caches 82.
constexpr int64_t TURN_STREAM = 64 << 20;
template <typename T, int THREADS, bool STREAM>
struct TurnRows {
  static constexpr int PER = 16 / sizeof(T);
  typedef Piece<T, PER> P;
  const T* x;
  T* y;
  int64_t x_row, x_head, t0;
  int H, D, tokens, pairs, interleaved;
  int t, h, dt, dh, a, left;  // the piece at hand; the step to the next
  bool turned, on;
  Loaded<T, PER> u, v;

  __device__ __forceinline__ TurnRows(const T* x, int64_t x_row, int64_t x_head, T* y, int H,
                                      int D, int64_t t0, int tokens, int pairs, int interleaved)
      : x(x), y(y), x_row(x_row), x_head(x_head), t0(t0), H(H), D(D), tokens(tokens), pairs(pairs),
        interleaved(interleaved) {
    const TurnPieces<T> pieces(pairs, interleaved, D);
    const int I = pieces.all, step = THREADS / I;
    const int i = threadIdx.x % I, r0 = threadIdx.x / I;
    dt = step / H;
    dh = step % H;
    t = r0 / H;
    h = r0 % H;
    on = r0 < step && t < tokens;
    turned = i < pieces.turned;
    a = !turned ? 2 * pairs + (i - pieces.turned) * PER : i * PER;
    left = !turned ? D - a : (interleaved ? 2 * pairs : pairs) - a;
  }
  __device__ __forceinline__ void load() {
    if (!on) return;
    const T* from = x + (t0 + t) * x_row + h * x_head + a;
    u = some<T, PER>(from, left);
    if (turned && !interleaved) v = some<T, PER>(from + pairs, left);
  }
  __device__ __forceinline__ void next() {
    t += dt;
    h += dh;
    if (h >= H) {
      h -= H;
      ++t;
    }
    on = on && t < tokens;
  }
  // live: of each token, whether its rows are turned or 0; NULL: all
  __device__ __forceinline__ void run(const float2* cs, const int* live) {
    const TurnAngles<T> angles(pairs, interleaved);
    const int piece = a / PER;
    while (on) {
      P p = u.values(), q = v.values();
      const int tp = t, hp = h;
      next();
      load();
      if (turned) {
        const float4* c = (const float4*)(cs + tp * angles.pitch) + piece;
        if (interleaved) {
#pragma unroll
          for (int e = 0; e < PER; e += 2) {
            const float4 z = c[e / 4 * angles.pieces];
            const float2 w = e & 2 ? make_float2(z.z, z.w) : make_float2(z.x, z.y);
            const float x0 = (float)p.v[e], x1 = (float)p.v[e + 1];
            p.v[e] = result<T>(__builtin_fmaf(-x1, w.y, x0 * w.x));
            p.v[e + 1] = result<T>(__builtin_fmaf(x0, w.y, x1 * w.x));
          }
        } else {
#pragma unroll
          for (int e = 0; e < PER; ++e) {
            const float4 z = c[e / 2 * angles.pieces];
            const float2 w = e & 1 ? make_float2(z.z, z.w) : make_float2(z.x, z.y);
            const float x0 = (float)p.v[e], x1 = (float)q.v[e];
            p.v[e] = result<T>(__builtin_fmaf(-x1, w.y, x0 * w.x));
            q.v[e] = result<T>(__builtin_fmaf(x0, w.y, x1 * w.x));
          }
        }
      }
      if (live && !live[tp]) p = q = P{};
      T* to = y + ((t0 + tp) * H + hp) * D + a;
      put_some<STREAM, T, PER>(to, p, left);
      if (turned && !interleaved) put_some<STREAM, T, PER>(to + pairs, q, left);
    }
  }
};

}  // namespace tpo
