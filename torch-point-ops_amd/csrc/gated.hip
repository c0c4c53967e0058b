// gated.hip -- gated projection h = act(x Wg^T) * (x Wu^T) and its gradients.
//   x (M, K), Wg and Wu (F, K), h (M, F)
//   with g = x Wg^T, u = x Wu^T: dg = dh u act'(g), du = dh act(g),
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
#include "gemm_tile.hpp"

namespace tpo {

constexpr float LOG2E = 1.44269504088896341f;
constexpr float INV_SQRT2 = 0.70710678118654752f;
constexpr float INV_SQRT_2PI = 0.39894228040143268f;

// The normal distribution function.  For the half types by Abramowitz and
// Stegun 7.1.26 (1.5e-7 absolute, far below their rounding): erff is several
// times as long, and a tile's outputs are many instructions with no products to
// hide behind.  e2: exp(-g^2 / 2).
template <typename T>
__device__ __forceinline__ float normal_cdf(float g, float e2) {
  if constexpr (sizeof(T) == 4) {
    return 0.5f * (1.f + erff(g * INV_SQRT2));
  } else {
    const float x = fabsf(g) * INV_SQRT2;
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.f));
    float y = __builtin_fmaf(1.061405429f, t, -1.453152027f);
    y = __builtin_fmaf(y, t, 1.421413741f);
    y = __builtin_fmaf(y, t, -0.284496736f);
    y = __builtin_fmaf(y, t, 0.254829592f);
    const float tail = 0.5f * y * t * e2;
    return g > 0.f ? 1.f - tail : tail;
  }
}

// The activation a and its derivative d.
template <typename T>
__device__ __forceinline__ void gated_act(int act, float g, float& a, float& d) {
  if (act == TPO_ACT_SILU || act == TPO_ACT_SIGMOID) {
    // exp2 of a large gate is inf and its reciprocal 0: both ends are exact
    const float e = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * g));
    a = act == TPO_ACT_SILU ? g * e : e;
    d = act == TPO_ACT_SILU ? e + e * (1.f - e) * g : e * (1.f - e);
  } else if (act == TPO_ACT_GELU) {
    const float e2 = __builtin_amdgcn_exp2f(-0.5f * LOG2E * g * g);
    const float c = normal_cdf<T>(g, e2);
    a = g * c;
    d = c + g * (e2 * INV_SQRT_2PI);
  } else {
    a = g > 0.f ? g : (g != g ? g : 0.f);
    d = g > 0.f ? 1.f : 0.f;
  }
}

// f with the activation as a constant: asked for at every value it costs as many
// branches, and no two values' instructions go side by side (16384 x 1024 x 4096,
// training: 1160 us, 1151 with the activation asked for once a tile).
template <typename F>
__device__ __forceinline__ void with_act(int act, const F& f) {
  switch (act) {
    case TPO_ACT_SILU: f(std::integral_constant<int, TPO_ACT_SILU>()); break;
    case TPO_ACT_GELU: f(std::integral_constant<int, TPO_ACT_GELU>()); break;
    case TPO_ACT_RELU: f(std::integral_constant<int, TPO_ACT_RELU>()); break;
    default: f(std::integral_constant<int, TPO_ACT_SIGMOID>());
  }
}

// Slabs: 64 bytes three deep for the large tile (256 x 128), whose waves hold so
// many operands at a time that a slab's loads and reads go between its products;
// 128 bytes two deep for the others.  Two workgroups or more share a CU, so that
// one's products run beside the other's epilogue: a tile of 256 x 256, alone on
// its CU, took 583 us where 256 x 128 takes 559 (8192 x 2048 x 8192, gelu), and
// 489 where it takes 390 in the backward's first product.
template <int BM, int BN>
using GatedLds = TileLds<BM, BN, BM == 256 ? 64 : 128, BM == 256 ? 3 : 2, BM == 256>;
constexpr int UNIT = 128;  // bytes of the summed axis that widths and shares are rounded to

// Tile (m, n) of a grid of tiles_m x tiles_n: an XCD takes consecutive tiles
// (workgroups go round-robin over the eight), which run down groups of eight
// row tiles, so that the tiles that an XCD works on at a time share rows of both
// operands in its L2.  A group begins at a column as far on as it is down, so that the
// XCDs' stores, a row's length apart each, go to different places in the rows.
__device__ __forceinline__ void tile_of(int tiles_m, int tiles_n, int& m, int& n) {
  const int grid = tiles_m * tiles_n, p = blockIdx.x;
  const int q = grid >> 3, r = grid & 7, x = p & 7;
  const int t = x * q + (x < r ? x : r) + (p >> 3);
  const int group = t / (8 * tiles_n), first = group * 8;
  const int rows = tiles_m - first < 8 ? tiles_m - first : 8;
  const int in = t - group * 8 * tiles_n;
  m = first + in % rows;
  n = in / rows + (int)((int64_t)group * tiles_n / ((tiles_m + 7) / 8));
  n -= n >= tiles_n ? tiles_n : 0;
}

// The values from one row of d to the next: dg, du, and 256 bytes more, so that rows of
// a power of two of bytes begin in different channels of the memory (8192 x 512 x 2048
// in bfloat16, training: 203 us without them, 195).
template <typename T>
__host__ __device__ constexpr int64_t d_pitch(int64_t Fp) {
  return 2 * Fp + 256 / (int64_t)sizeof(T);
}

// Both projections of a tile of BM / 2 features and BN tokens.  The products'
// rows are the features: BM / 4 of the gate and the same of the up projection
// for either half of the waves' rows, so that a lane holds both sums of an
// output, and four neighbouring outputs of one token.
// Forward: h, and with keep g and u themselves, a token's 2 F values.  Backward
// (gh): dg and du into d, a token's 2 Fp values, Fp >= F with 0 past F, d_pitch apart.
template <typename T, int BM, int BN, bool BWD>
__global__ __launch_bounds__(256, 2) void gated_pair_kernel(
    Matrix x, Matrix wg, Matrix wu, int act, const T* __restrict__ gh, int64_t F,
    T* __restrict__ out, T* __restrict__ keep, int64_t Fp) {
  __shared__ GatedLds<BM, BN> lds;
  constexpr int SLAB = GatedLds<BM, BN>::SLAB;
  typedef RowLoader<T, BM, SLAB> LA;
  typedef RowLoader<T, BN, SLAB> LB;
  const int64_t M = x.rows;
  int tm, tn;
  tile_of((int)((M + BN - 1) / BN), (int)((F + BM / 2 - 1) / (BM / 2)), tm, tn);
  const int w = wave_id();
  const int64_t t0 = (int64_t)tm * BN, f0 = (int64_t)tn * (BM / 2) + (w >> 1) * (BM / 4);
  const LA la((w & 1) ? wu : wg, f0);
  const LB lb(x, t0 + w * (BN / 4));
  constexpr int TF = BM / 128;  // feature tiles of a wave
  typedef Rows32<T, BM / 4> R;
  f32x16 acc[BM / 64][BN / 64];
  gemm_tile<T, BM, BN>(lds, la, lb, 0, (int)((x.bytes + SLAB - 1) / SLAB), acc);

  const R rg{(char*)&lds + w * 2 * R::BYTES}, ru{rg.lds + R::BYTES};
  const int h = lane_id() >> 5;
#pragma unroll
  for (int j = 0; j < BN / 64; ++j) {
    const int64_t t = t0 + (w & 1) * (BN / 2) + 32 * j;
    if (BWD) rg.load(gh, F, t, M, f0, F);
    with_act(act, [&](auto name) {
#pragma unroll
      for (int i = 0; i < TF; ++i)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int at = 32 * i + 8 * b + 4 * h;
          Four<T> p, q;
          if (BWD) p = *(Four<T>*)rg.four(at);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float g = acc[i][j][4 * b + e], u = acc[i + TF][j][4 * b + e];
            float a, d;
            gated_act<T>(name, g, a, d);
            if (BWD) {
              const float y = (float)p.v[e];
              const bool in = f0 + at + e < F;
              p.v[e] = in ? (T)(y * u * d) : (T)0.f;
              q.v[e] = in ? (T)(y * a) : (T)0.f;
            } else {
              p.v[e] = (T)(a * u);
            }
          }
          *(Four<T>*)rg.four(at) = p;
          if (BWD) *(Four<T>*)ru.four(at) = q;
        }
    });
    if (!BWD && sizeof(T) == 4 && keep) {
      rg.store(out, F, t, M, f0, F);
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int i = 0; i < TF; ++i)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            Four<T> p;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              p.v[e] = (T)(y ? acc[i + TF][j][4 * b + e] : acc[i][j][4 * b + e]);
            *(Four<T>*)rg.four(32 * i + 8 * b + 4 * h) = p;
          }
        rg.store(keep + y * F, 2 * F, t, M, f0, F);
      }
    } else if (BWD) {
      rg.store(out, d_pitch<T>(Fp), t, M, f0, Fp);
      ru.store(out + Fp, d_pitch<T>(Fp), t, M, f0, Fp);
    } else {
      rg.store(out, F, t, M, f0, F);
    }
  }
}

// Few tokens, where the weights' way from memory is all that counts, and few tiles: a
// workgroup takes 32 features and 32 TN tokens; its four waves take every fourth slab
// of the summed axis each, through LDS of their own and without waiting for each
// other, and add up their sums at the end.  Results as gated_pair_kernel's.
template <typename T, int TN>
struct alignas(1024) FewLds {
  static constexpr int SLAB = 128, DEPTH = TN == 1 ? 3 : 2, STAGE = (64 + 32 * TN) * SLAB;
  char b[4][DEPTH][STAGE];
};

// A wave's loads of a slab: 32 rows of the gate's weights, of the up projection's,
// of 32 TN tokens.
template <typename T, int TN>
struct FewLoader {
  typedef RowLoader<T, 128, 128> L;  // 32 rows: a quarter of 128
  static constexpr int LOADS = (2 + TN) * L::N;
  L g, u, x0, x1;  // (x1: the second 32 tokens)
  __device__ __forceinline__ FewLoader(const Matrix& wg, const Matrix& wu, const Matrix& xs,
                                       int64_t f0, int64_t m0)
      : g(wg, f0), u(wu, f0), x0(xs, m0), x1(xs, m0 + 32) {}
  __device__ __forceinline__ void load(char* lds, int slab) const {
    lds -= wave_id() * L::N * 1024;  // (where the loader puts wave 0's rows)
    const auto sg = g.slab(slab), su = u.slab(slab);
#pragma unroll
    for (int j = 0; j < L::N; ++j) sg.load(lds, j);
#pragma unroll
    for (int j = 0; j < L::N; ++j) su.load(lds + 32 * 128, j);
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      const auto sx = (i ? x1 : x0).slab(slab);
#pragma unroll
      for (int j = 0; j < L::N; ++j) sx.load(lds + (64 + 32 * i) * 128, j);
    }
  }
};

template <typename T, int TN>
__device__ __forceinline__ void few_step(const char* __restrict__ cur, char* __restrict__ nxt,
                                         const FewLoader<T, TN>& load, int next,
                                         f32x16 (&acc)[2][TN]) {
  typedef RowLoader<T, 128, 128> L;
  load.load(nxt, next);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const auto g = L::read(cur, 0, s), u = L::read(cur, 32, s);
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      const auto x = L::read(cur, 64 + 32 * i, s);
      mma(acc[0][i], g, x);
      mma(acc[1][i], u, x);
    }
  }
}

template <typename T, int TN, bool BWD>
__global__ __launch_bounds__(256) void gated_few_kernel(Matrix x, Matrix wg, Matrix wu, int act,
                                                        const T* __restrict__ gh, int64_t F,
                                                        T* __restrict__ out, T* __restrict__ keep,
                                                        int64_t Fp) {
  typedef FewLds<T, TN> Lds;
  __shared__ Lds lds;
  const int w = wave_id(), l = lane_id();
  const int64_t f0 = (int64_t)blockIdx.x * 32, m0 = (int64_t)blockIdx.y * 32 * TN;
  const FewLoader<T, TN> load(wg, wu, x, f0, m0);
  const int slabs = (int)((x.bytes + 127) / 128);
  f32x16 acc[2][TN];
#pragma unroll
  for (int i = 0; i < TN; ++i) acc[0][i] = acc[1][i] = f32x16{};
#pragma unroll
  for (int d = 0; d < Lds::DEPTH - 1; ++d) load.load(lds.b[w][d], w + 4 * d);
  int at = 0;
  for (int k = w; k < slabs; k += 4) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    constexpr int n = (Lds::DEPTH - 2) * FewLoader<T, TN>::LOADS;
    __builtin_amdgcn_s_waitcnt((n & 15) | (n >> 4) << 14 | 0x70);  // the slab has landed
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    const int free = at == 0 ? Lds::DEPTH - 1 : at - 1;
    few_step<T, TN>(lds.b[w][at], lds.b[w][free], load, k + 4 * (Lds::DEPTH - 1), acc);
    at = at + 1 == Lds::DEPTH ? 0 : at + 1;
  }
  wait_loads_and_meet<0>();
  f32x4* sums = (f32x4*)&lds;  // [wave][gate, up][tokens][b][lane]
#pragma unroll
  for (int y = 0; y < 2; ++y)
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        sums[(((w * 2 + y) * TN + i) * 4 + b) * 64 + l] =
            f32x4{acc[y][i][4 * b], acc[y][i][4 * b + 1], acc[y][i][4 * b + 2],
                  acc[y][i][4 * b + 3]};
  __syncthreads();
  // wave w finishes values b = w of the lanes' columns
#pragma unroll
  for (int i = 0; i < TN; ++i) {
    f32x4 g = {}, u = {};
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const f32x4 y = sums[(((v * 2 + 0) * TN + i) * 4 + w) * 64 + l];
      const f32x4 z = sums[(((v * 2 + 1) * TN + i) * 4 + w) * 64 + l];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        g[e] += y[e];
        u[e] += z[e];
      }
    }
    const int64_t m = m0 + 32 * i + (l & 31), f = f0 + 8 * w + 4 * (l >> 5);
    if (m >= x.rows) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float a, d;
      gated_act<T>(act, g[e], a, d);
      if (BWD) {
        const bool in = f + e < F;
        const float y = in ? (float)gh[m * F + f + e] : 0.f;
        if (f + e < Fp) {
          out[m * d_pitch<T>(Fp) + f + e] = in ? (T)(y * u[e] * d) : (T)0.f;
          out[m * d_pitch<T>(Fp) + Fp + f + e] = in ? (T)(y * a) : (T)0.f;
        }
      } else if (f + e < F) {
        out[m * F + f + e] = (T)(a * u[e]);
        if (keep) {
          keep[m * 2 * F + f + e] = (T)g[e];
          keep[m * 2 * F + F + f + e] = (T)u[e];
        }
      }
    }
  }
}

// dg and du into d from the g and u that the forward kept.
__global__ __launch_bounds__(256) void gated_kept_kernel(const float* __restrict__ keep,
                                                         const float* __restrict__ gh, int64_t M,
                                                         int64_t F, int64_t Fp, int act,
                                                         float* __restrict__ d) {
  const int64_t f = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (f >= Fp) return;
  for (int64_t m = blockIdx.y; m < M; m += gridDim.y) {
    float dg = 0.f, du = 0.f;
    if (f < F) {
      const float g = keep[m * 2 * F + f], u = keep[m * 2 * F + F + f], y = gh[m * F + f];
      float a, s;
      gated_act<float>(act, g, a, s);
      dg = y * u * s;
      du = y * a;
    }
    d[m * d_pitch<float>(Fp) + f] = dg;
    d[m * d_pitch<float>(Fp) + Fp + f] = du;
  }
}

// A tile of sums to out (M rows of N values) or, as floats, to part.
template <typename T, int BM, int BN, typename Lds>
__device__ __forceinline__ void gated_put(Lds& lds, const f32x16 (&acc)[BM / 64][BN / 64],
                                          int64_t n0, int64_t m0, int64_t N, int64_t M,
                                          T* __restrict__ out, float* __restrict__ part) {
  const int w = wave_id(), h = lane_id() >> 5;
  n0 += (w >> 1) * (BM / 2);
  m0 += (w & 1) * (BN / 2);
  auto put = [&](auto t, auto* to) {
    typedef decltype(t) V;
    typedef Rows32<V, BM / 2> R;
    const R r{(char*)&lds + w * R::BYTES};
#pragma unroll
    for (int j = 0; j < BN / 64; ++j) {
#pragma unroll
      for (int i = 0; i < BM / 64; ++i)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          Four<V> p;
#pragma unroll
          for (int e = 0; e < 4; ++e) p.v[e] = (V)acc[i][j][4 * b + e];
          *(Four<V>*)r.four(32 * i + 8 * b + 4 * h) = p;
        }
      r.store(to, N, m0 + 32 * j, M, n0, N);
    }
  };
  if (part)
    put(float(), part);
  else
    put(T(), out);
}

// dx = [dg du] [Wg; Wu], M tokens of K values; blockIdx.y: a share of the sum.
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256, 2) void gated_dx_kernel(
    Matrix d, Matrix wg, const char* wu, int units, int share, int64_t K, T* __restrict__ out,
    float* __restrict__ part) {
  __shared__ GatedLds<BM, BN> lds;
  constexpr int SLAB = GatedLds<BM, BN>::SLAB;
  const int64_t M = d.rows;
  int tm, tn;
  tile_of((int)((M + BN - 1) / BN), (int)((K + BM - 1) / BM), tm, tn);
  const int64_t m0 = (int64_t)tm * BN, n0 = (int64_t)tn * BM;
  const PairLoader<T, BM, SLAB> la(wg, wu, units * (UNIT / SLAB), n0);
  const RowLoader<T, BN, SLAB> lb(d, m0 + wave_id() * (BN / 4));
  const int u0 = blockIdx.y * share, u1 = u0 + share < 2 * units ? u0 + share : 2 * units;
  f32x16 acc[BM / 64][BN / 64];
  gemm_tile<T, BM, BN>(lds, la, lb, u0 * (UNIT / SLAB), u1 * (UNIT / SLAB), acc);
  if (part) part += blockIdx.y * M * K;
  gated_put<T, BM, BN>(lds, acc, n0, m0, K, M, out, part);
}

// dWg = dg^T x and dWu = du^T x (blockIdx.z), F rows of K values; blockIdx.y: a
// share of the sum over the tokens.
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256, 2) void gated_dw_kernel(
    Matrix x, Matrix d, int64_t F, int units, int share, int64_t K, T* __restrict__ dwg,
    T* __restrict__ dwu, float* __restrict__ part) {
  __shared__ GatedLds<BM, BN> lds;
  constexpr int SLAB = GatedLds<BM, BN>::SLAB;
  int tm, tn;
  tile_of((int)((F + BN - 1) / BN), (int)((K + BM - 1) / BM), tm, tn);
  const int64_t m0 = (int64_t)tm * BN, n0 = (int64_t)tn * BM;
  if (blockIdx.z) d.p += d.bytes;
  const ColLoader<T, BM, SLAB> la(x, n0);
  const ColLoader<T, BN, SLAB> lb(d, m0);
  const int u0 = blockIdx.y * share, u1 = u0 + share < units ? u0 + share : units;
  f32x16 acc[BM / 64][BN / 64];
  gemm_tile<T, BM, BN>(lds, la, lb, u0 * (UNIT / SLAB), u1 * (UNIT / SLAB), acc);
  if (part) part += ((int64_t)blockIdx.y * 2 + blockIdx.z) * F * K;
  gated_put<T, BM, BN>(lds, acc, n0, m0, K, F, blockIdx.z ? dwu : dwg, part);
}

// out, out2 (n values each): the shares of a split product added in order
template <typename T>
__global__ __launch_bounds__(256) void gated_join_kernel(const float* __restrict__ part, int shares,
                                                         int64_t n, T* __restrict__ out,
                                                         T* __restrict__ out2) {
  const int64_t all = n * gridDim.y;
  T* to = blockIdx.y ? out2 : out;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float s = 0.f;
    for (int p = 0; p < shares; ++p) s += part[p * all + blockIdx.y * n + i];
    to[i] = (T)s;
  }
}

// Copies of up to three matrices of C columns with rows padded with 0 to `pitch`
// values (16 bytes).
struct Copies {
  const void* in[3];
  void* out[3];
  int64_t rows[3];
};
template <typename T>
__global__ __launch_bounds__(256) void gated_pad_kernel(Copies m, int C, int pitch) {
  constexpr int PER = 16 / sizeof(T);
  const int y = blockIdx.z;
  const T* in = (const T*)m.in[y];
  T* out = (T*)m.out[y];
  const int c = (blockIdx.x * 64 + threadIdx.x % 64) * PER;
  if (c >= pitch) return;
  for (int64_t r = blockIdx.y * 4 + threadIdx.x / 64; r < m.rows[y]; r += gridDim.y * 4) {
    Piece<T, PER> v = {};
    if (c + PER <= C)
      v = *(const Piece<T, PER>*)(in + r * C + c);
    else
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (c + e < C) v.v[e] = in[r * C + c + e];
    *(f32x4*)(out + r * pitch + c) = __builtin_bit_cast(f32x4, v);
  }
}

// ---------------------------------------------------------------------- host
int gated_check(const char* op, int dtype, int64_t M, int64_t K, int64_t F, int act) {
  if (dtype != TPO_F32 && dtype != TPO_F16 && dtype != TPO_BF16)
    return set_error(TPO_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  // a wave's 64 rows of an operand span less than 2^31 bytes
  if (M < 0 || K < 1 || F < 0 || M > (1 << 22) || K > (1 << 20) || F > (1 << 20))
    return set_error(TPO_ERR_ARG, "%s: bad sizes M=%lld K=%lld F=%lld", op, (long long)M,
                     (long long)K, (long long)F);
  if (act < TPO_ACT_SILU || act > TPO_ACT_SIGMOID)
    return set_error(TPO_ERR_ARG, "%s: unknown activation %d", op, act);
  return TPO_OK;
}

int gated_aligned(const char* op, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p & 15)
      return set_error(TPO_ERR_ARG, "%s: x, the weights and the workspace must be 16-byte aligned",
                       op);
  return TPO_OK;
}

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a product of `rows` x `cols` sums (the rows being what the tile's longer
// side covers) is cut: the tile and the number of shares of the summed axis,
// `units` long (0: not to be shared).  By estimated time: a tile's products at the
// rate that the tile reached with every place on the CUs taken (PFLOP/s of half
// types, of float at about a seventh: 256 x 128 1.05, 128 x 128 0.9, 64 x 64
// 0.56), in as many rounds as there are places; shares' sums at 4 TB/s through
// memory, and a launch that adds them.  dX of 4096 x 1024 x 4096: 117 us in
// 64-tiles, 97 as it is cut; float 1000 x 385 x 1023 training: 115 us with
// 64-tiles, 233 with 128.
enum Tile { LARGE, MIDDLE, SMALL };  // 256 x 128, 128 x 128, 64 x 64 (128 x 64 for the pair)
struct Cut {
  Tile tile;
  int shares;
};
Cut gated_cut(int dtype, int64_t rows, int64_t cols, int64_t products, int64_t units,
              int64_t summed) {
  static const int64_t R[] = {256, 128, 64}, C[] = {128, 128, 64}, PLACES[] = {512, 512, 1024};
  static const double RATE[] = {1.05e15, 0.9e15, 0.56e15};
  static const double FLOAT_RATE[] = {0.13e15, 0.13e15, 0.1e15};
  Cut best{SMALL, 1};
  double least = 1e30;
  for (int t = 0; t < 3; ++t) {
    const double rate = dtype == TPO_F32 ? FLOAT_RATE[t] : RATE[t];
    const int64_t blocks = cdiv(rows, R[t]) * cdiv(cols, C[t]) * products;
    for (int64_t s = 1; s <= 64; s *= 2) {
      if (s > 1 && s > units / 8) break;
      // rounds by halves: places that are half taken work faster, though not twice
      const double filled = (double)(blocks * s) / PLACES[t];
      const double halves = (double)(int64_t)(2 * filled + 0.99);
      const double rounds = filled <= 0.5 ? 0.62 : filled <= 1 ? 1 : 0.5 * halves;
      const double tile = 2.0 * R[t] * C[t] * ((double)summed / s);
      double time = rounds * tile * PLACES[t] / rate;
      if (s > 1) time += 8.0 * s * rows * cols * products / 4e12 + 5e-6;
      if (time < least) {
        least = time;
        best = Cut{(Tile)t, (int)s};
      }
    }
  }
  return best;
}

// What the calls keep in the workspace, in bytes from its start.
struct Plan {
  int64_t Kp, Fp;          // K padded to 16 bytes, F to a unit
  int64_t x, wg, wu;       // padded copies (-1: the inputs do)
  int64_t d, part;
  int64_t funits, munits;  // units of F and of M
  Cut dx, dw;
  int64_t bytes;
};
Plan gated_plan(int dtype, int64_t M, int64_t K, int64_t F, bool bwd) {
  const int64_t z = element_bytes(dtype), per = UNIT / z;
  Plan p = {};
  p.Kp = round_up(K, 16 / z);
  p.Fp = round_up(F, per);
  p.funits = p.Fp / per;
  p.munits = cdiv(M, per);
  auto take = [&](int64_t values, int64_t size) {
    const int64_t at = p.bytes;
    p.bytes += round_up(values * size, 256);
    return at;
  };
  p.x = p.wg = p.wu = -1;
  if (p.Kp != K) {
    p.x = take(M * p.Kp, z);
    p.wg = take(F * p.Kp, z);
    p.wu = take(F * p.Kp, z);
  }
  if (bwd) {
    p.d = take(M * (2 * p.Fp + 256 / z), z);  // d_pitch
    p.dx = gated_cut(dtype, K, M, 1, 2 * p.funits, 2 * p.Fp);
    p.dw = gated_cut(dtype, K, F, 2, p.munits, M);
    const int64_t a = p.dx.shares > 1 ? p.dx.shares * M * K : 0;
    const int64_t b = p.dw.shares > 1 ? p.dw.shares * 2 * F * K : 0;
    p.part = take(a > b ? a : b, 4);
  }
  return p;
}

unsigned gated_blocks(int64_t n) { return (unsigned)(cdiv(n, 256) < 4096 ? cdiv(n, 256) : 4096); }

// The inputs as the products read them, padded copies made where needed.
template <typename T>
void gated_inputs(const Plan& p, const void* x, const void* wg, const void* wu, int64_t M,
                  int64_t K, int64_t F, char* ws, hipStream_t s, Matrix (&r)[3]) {
  const void* in[3] = {x, wg, wu};
  const int64_t at[3] = {p.x, p.wg, p.wu}, rows[3] = {M, F, F}, pitch = p.Kp * sizeof(T);
  Copies c;
  for (int i = 0; i < 3; ++i) {
    c.in[i] = in[i];
    c.out[i] = ws + at[i];
    c.rows[i] = rows[i];
    r[i] = Matrix{p.Kp != K ? ws + at[i] : (const char*)in[i], pitch, rows[i], pitch};
  }
  if (p.Kp != K) {
    const int64_t rows4 = cdiv(M > F ? M : F, 4);
    gated_pad_kernel<T><<<dim3((unsigned)cdiv(p.Kp * sizeof(T), 1024),
                               (unsigned)(rows4 < 2048 ? rows4 : 2048), 3),
                          256, 0, s>>>(c, (int)K, (int)p.Kp);
  }
}

template <typename T, bool BWD>
void gated_pair(const Matrix (&r)[3], int act, const T* gh, int64_t F, T* out, T* keep, int64_t Fp,
                hipStream_t s) {
  const int64_t M = r[0].rows;
  auto run = [&](auto bm, auto bn) {
    constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value;
    const int64_t tiles = cdiv(M, BN) * cdiv(F, BM / 2);
    gated_pair_kernel<T, BM, BN, BWD><<<dim3((unsigned)tiles), 256, 0, s>>>(
        r[0], r[1], r[2], act, gh, F, out, keep, Fp);
  };
  // In one round of a workgroup a CU the shared sums beat the tiles' (float 185 x 384
  // -> 315: 9 us where the smallest tile takes 17; bfloat16 128 x 4096 -> 1024: 11,
  // 26), by 32 tokens if that is one round, by 64 if not (float 200 x 512 -> 2048: 13,
  // by 32 15, tiles 21); in two rounds they do not (500 x 512 -> 2048: 25, 22), but
  // where there are no more tokens and all else waits for the weights (16 x 2048 ->
  // 8192: 13, 22).
  const int64_t fs = cdiv(BWD ? Fp : F, 32);
  auto few = [&](auto n) {
    constexpr int TN = decltype(n)::value;
    gated_few_kernel<T, TN, BWD><<<dim3((unsigned)fs, (unsigned)cdiv(M, 32 * TN)), 256, 0, s>>>(
        r[0], r[1], r[2], act, gh, F, out, keep, Fp);
  };
  if (M <= 32 || fs * cdiv(M, 32) <= 256) return few(std::integral_constant<int, 1>());
  if (M <= 64 || fs * cdiv(M, 64) <= 256) return few(std::integral_constant<int, 2>());
  typedef std::integral_constant<int, 256> I256;
  typedef std::integral_constant<int, 128> I128;
  typedef std::integral_constant<int, 64> I64;
  const int type = sizeof(T) == 4 ? TPO_F32 : TPO_BF16;
  switch (gated_cut(type, 2 * F, M, 1, 0, r[0].bytes / sizeof(T)).tile) {
    case LARGE: run(I256(), I128()); break;
    case MIDDLE: run(I128(), I128()); break;
    case SMALL: run(I128(), I64()); break;
  }
}

template <typename T, int BM, int BN>
void gated_dx(const Plan& p, const Matrix& d, const Matrix& wg, const Matrix& wu, int64_t K, T* out,
              float* part, hipStream_t s) {
  const int64_t M = d.rows;
  const int share = (int)cdiv(2 * p.funits, p.dx.shares), shares = p.dx.shares;
  gated_dx_kernel<T, BM, BN><<<dim3((unsigned)(cdiv(M, BN) * cdiv(K, BM)), shares), 256, 0, s>>>(
      d, wg, wu.p, (int)p.funits, share, K, out, shares > 1 ? part : nullptr);
  if (shares > 1)
    gated_join_kernel<T><<<dim3(gated_blocks(M * K)), 256, 0, s>>>(part, shares, M * K, out, out);
}

template <typename T, int BM, int BN>
void gated_dw(const Plan& p, const Matrix& x, const Matrix& d, int64_t F, int64_t K, T* dwg, T* dwu,
              float* part, hipStream_t s) {
  const int share = (int)cdiv(p.munits, p.dw.shares), shares = p.dw.shares;
  gated_dw_kernel<T, BM, BN><<<dim3((unsigned)(cdiv(F, BN) * cdiv(K, BM)), shares, 2), 256, 0, s>>>(
      x, d, F, (int)p.munits, share, K, dwg, dwu, shares > 1 ? part : nullptr);
  if (shares > 1)
    gated_join_kernel<T><<<dim3(gated_blocks(F * K), 2), 256, 0, s>>>(part, shares, F * K, dwg,
                                                                      dwu);
}

}  // namespace tpo

using namespace tpo;

extern "C" int64_t tpo_gated_fwd_workspace_size(int dtype, int64_t M, int64_t K, int64_t F) {
  if (gated_check("gated_fwd_workspace_size", dtype, M, K, F, TPO_ACT_SILU)) return -1;
  return gated_plan(dtype, M, K, F, false).bytes;
}

extern "C" int tpo_gated_fwd(int dtype, const void* x, const void* w_gate, const void* w_up,
                             int64_t M, int64_t K, int64_t F, int activation, void* h,
                             void* keep, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = gated_check("gated_fwd", dtype, M, K, F, activation)) return rc;
  if (M == 0 || F == 0) return TPO_OK;
  if (int rc = all_there("gated_fwd", {x, w_gate, w_up, h})) return rc;
  if (int rc = gated_aligned("gated_fwd", {x, w_gate, w_up, workspace})) return rc;
  if (keep && dtype != TPO_F32)
    return set_error(TPO_ERR_ARG, "gated_fwd: only float projections are kept");
  const Plan p = gated_plan(dtype, M, K, F, false);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes))
    return set_error(TPO_ERR_WORKSPACE, "gated_fwd: workspace of %lld bytes needed",
                     (long long)p.bytes);
  hipStream_t s = (hipStream_t)stream;
  with_element(dtype, [&](auto t) {
    typedef decltype(t) T;
    Matrix r[3];
    gated_inputs<T>(p, x, w_gate, w_up, M, K, F, (char*)workspace, s, r);
    gated_pair<T, false>(r, activation, nullptr, F, (T*)h, (T*)keep, 0, s);
  });
  return check_launch("gated_fwd");
}

extern "C" int64_t tpo_gated_bwd_workspace_size(int dtype, int64_t M, int64_t K, int64_t F) {
  if (gated_check("gated_bwd_workspace_size", dtype, M, K, F, TPO_ACT_SILU)) return -1;
  return gated_plan(dtype, M, K, F, true).bytes;
}

extern "C" int tpo_gated_bwd(int dtype, const void* grad_h, const void* x, const void* w_gate,
                             const void* w_up, const void* kept, int64_t M, int64_t K, int64_t F,
                             int activation,
                             void* grad_x, void* grad_w_gate, void* grad_w_up, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  if (int rc = gated_check("gated_bwd", dtype, M, K, F, activation)) return rc;
  if ((grad_w_gate == nullptr) != (grad_w_up == nullptr))
    return set_error(TPO_ERR_ARG, "gated_bwd: the weights' gradients go together");
  const Plan p = gated_plan(dtype, M, K, F, true);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes))
    return set_error(TPO_ERR_WORKSPACE, "gated_bwd: workspace of %lld bytes needed",
                     (long long)p.bytes);
  if (int rc = gated_aligned("gated_bwd", {x, w_gate, w_up, workspace})) return rc;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  if (M == 0 && F == 0) return TPO_OK;
  if (M > 0 && F > 0)
    if (int rc = all_there("gated_bwd", {grad_h, x, w_gate, w_up})) return rc;
  if (kept && dtype != TPO_F32)
    return set_error(TPO_ERR_ARG, "gated_bwd: only float projections are kept");
  with_element(dtype, [&](auto t) {
    typedef decltype(t) T;
    Matrix r[3];
    gated_inputs<T>(p, x, w_gate, w_up, M, K, F, ws, s, r);
    const int64_t row = 2 * p.Fp * sizeof(T), pitch = d_pitch<T>(p.Fp) * sizeof(T);
    float* part = (float*)(ws + p.part);
    if (M > 0 && F > 0 && kept)
      gated_kept_kernel<<<dim3((unsigned)cdiv(p.Fp, 256), (unsigned)(M < 16384 ? M : 16384)), 256,
                          0, s>>>((const float*)kept, (const float*)grad_h, M, F, p.Fp, activation,
                               (float*)(ws + p.d));
    else if (M > 0 && F > 0)
      gated_pair<T, true>(r, activation, (const T*)grad_h, F, (T*)(ws + p.d), nullptr, p.Fp, s);
    if (grad_x && M > 0) {
      const Matrix d{ws + p.d, pitch, M, row};
      T* to = (T*)grad_x;
      switch (p.dx.tile) {
        case LARGE: gated_dx<T, 256, 128>(p, d, r[1], r[2], K, to, part, s); break;
        case MIDDLE: gated_dx<T, 128, 128>(p, d, r[1], r[2], K, to, part, s); break;
        case SMALL: gated_dx<T, 64, 64>(p, d, r[1], r[2], K, to, part, s); break;
      }
    }
    if (grad_w_gate && F > 0) {
      const Matrix d{ws + p.d, pitch, M, row / 2};
      T *g = (T*)grad_w_gate, *u = (T*)grad_w_up;
      switch (p.dw.tile) {
        case LARGE: gated_dw<T, 256, 128>(p, r[0], d, F, K, g, u, part, s); break;
        case MIDDLE: gated_dw<T, 128, 128>(p, r[0], d, F, K, g, u, part, s); break;
        case SMALL: gated_dw<T, 64, 64>(p, r[0], d, F, K, g, u, part, s); break;
      }
    }
  });
  return check_launch("gated_bwd");
}
