// gated.hip -- gated projection h = act(x Wg^T) * (x Wu^T) and its gradients.
//   x (M, K), Wg and Wu (F, K), h (M, F)
//   with g = x Wg^T, u = x Wu^T: dg = dh u act'(g), du = dh act(g),
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
#include "gemm_tile.hpp"

namespace tpo {

constexpr float LOG2E = 1.44269504088896341f;
constexpr float INV_SQRT2 = 0.70710678118654752f;
constexpr float INV_SQRT_2PI = 0.39894228040143268f;

// The activation a and its derivative d.
__device__ __forceinline__ void gated_act(int act, float g, float& a, float& d) {
  if (act == TPO_ACT_SILU || act == TPO_ACT_SIGMOID) {
    // exp2 of a large gate is inf and its reciprocal 0: both ends are exact
    const float e = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * g));
    a = act == TPO_ACT_SILU ? g * e : e;
    d = act == TPO_ACT_SILU ? e + e * (1.f - e) * g : e * (1.f - e);
  } else if (act == TPO_ACT_GELU) {
    const float c = 0.5f * (1.f + erff(g * INV_SQRT2));
    a = g * c;
    d = c + g * (__builtin_amdgcn_exp2f(-0.5f * LOG2E * g * g) * INV_SQRT_2PI);
  } else {
    a = g > 0.f ? g : (g != g ? g : 0.f);
    d = g > 0.f ? 1.f : 0.f;
  }
}

// Tile (m, n) of a grid of tiles_m x tiles_n: an XCD takes consecutive tiles
// (workgroups go round-robin over the eight), which run down groups of eight
// row tiles, so that the tiles that an XCD works on at a time share rows of both
// operands in its L2.
__device__ __forceinline__ void tile_of(int tiles_m, int tiles_n, int& m, int& n) {
  const int grid = tiles_m * tiles_n, p = blockIdx.x;
  const int q = grid >> 3, r = grid & 7, x = p & 7;
  const int t = x * q + (x < r ? x : r) + (p >> 3);
  const int group = t / (8 * tiles_n), first = group * 8;
  const int rows = tiles_m - first < 8 ? tiles_m - first : 8;
  const int in = t - group * 8 * tiles_n;
  m = first + in % rows;
  n = in / rows;
}

template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};

// Both projections of a tile of BM rows and BN / 2 features.  The columns of the
// product are BN / 4 gate and BN / 4 up features for either half of the waves'
// columns, so that a lane holds both sums of an output.
// Forward: h.  Backward (gh given): dg and du, which the two products after it
// read by rows (d, gate features and then up features, each padded with 0 to
// Fp) and by columns (dt, rows padded with 0 to Mp).
template <typename T, int BM, int BN, bool BWD>
__global__ __launch_bounds__(256, BM == 256 ? 1 : 2) void gated_pair_kernel(
    Rows x, Rows wg, Rows wu, int bytes, int act, const T* __restrict__ gh, int64_t F,
    T* __restrict__ h, T* __restrict__ d, int64_t Fp, T* __restrict__ dt, int64_t Mp) {
  __shared__ TileLds<BM, BN> lds;
  const int64_t M = x.rows;
  int tm, tn;
  tile_of((int)((M + BM - 1) / BM), (int)((F + BN / 2 - 1) / (BN / 2)), tm, tn);
  const int64_t m0 = (int64_t)tm * BM, f0 = (int64_t)tn * (BN / 2);
  const int w = wave_id(), l = lane_id();
  const Loader<BM> la(x, m0 + w * (BM / 4));
  const Loader<BN> lb((w & 1) ? wu : wg, f0 + (w >> 1) * (BN / 4));
  f32x16 acc[BM / 64][BN / 64];
  gemm_tile<T, BM, BN>(lds, la, lb, 0, bytes, acc);
  constexpr int TF = BN / 128;  // feature tiles of a wave
  const int64_t row = m0 + (w >> 1) * (BM / 2) + 4 * (l >> 5);
  const int64_t col = f0 + (w & 1) * (BN / 4) + (l & 31);
#pragma unroll
  for (int i = 0; i < BM / 64; ++i)
#pragma unroll
    for (int j = 0; j < TF; ++j) {
      const int64_t f = col + 32 * j;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int64_t m = row + 32 * i + 8 * b;
        Four<T> pg, pu;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float g = acc[i][j][4 * b + e], u = acc[i][j + TF][4 * b + e];
          float a, s;
          gated_act(act, g, a, s);
          const bool in = m + e < M && f < F;
          if (!BWD) {
            if (in) h[(m + e) * F + f] = (T)(a * u);
          } else {
            const float t = in ? (float)gh[(m + e) * F + f] : 0.f;
            pg.v[e] = in ? (T)(t * u * s) : (T)0.f;
            pu.v[e] = in ? (T)(t * a) : (T)0.f;
            if (m + e < M && f < Fp) {
              d[(m + e) * 2 * Fp + f] = pg.v[e];
              d[(m + e) * 2 * Fp + Fp + f] = pu.v[e];
            }
          }
        }
        if (BWD && f < F && m < Mp) {
          *(Four<T>*)(dt + f * Mp + m) = pg;
          *(Four<T>*)(dt + (F + f) * Mp + m) = pu;
        }
      }
    }
}

// out = A B^T, or with part the float sums over one of gridDim.z's shares of
// the summed axis.  blockIdx.y chooses one of two products (A and out a fixed
// distance on).
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256, BM == 256 ? 1 : 2) void gated_product_kernel(
    Rows a, Rows b, int bytes, int share, T* __restrict__ out, T* __restrict__ out2,
    float* __restrict__ part) {
  __shared__ TileLds<BM, BN> lds;
  const int64_t M = a.rows, N = b.rows;
  int tm, tn;
  tile_of((int)((M + BM - 1) / BM), (int)((N + BN - 1) / BN), tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int w = wave_id(), l = lane_id();
  if (blockIdx.y) {
    a.p += M * a.pitch;
    out = out2;
  }
  const Loader<BM> la(a, m0 + w * (BM / 4));
  const Loader<BN> lb(b, n0 + w * (BN / 4));
  const int k0 = (int)blockIdx.z * share;
  f32x16 acc[BM / 64][BN / 64];
  gemm_tile<T, BM, BN>(lds, la, lb, k0, bytes - k0 < share ? bytes : k0 + share, acc);
  const int64_t row = m0 + (w >> 1) * (BM / 2) + 4 * (l >> 5);
  const int64_t col = n0 + (w & 1) * (BN / 2) + (l & 31);
  if (part) part += ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * M * N;
#pragma unroll
  for (int i = 0; i < BM / 64; ++i)
#pragma unroll
    for (int j = 0; j < BN / 64; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int64_t m = row + 32 * i + 8 * (v >> 2) + (v & 3), n = col + 32 * j;
        if (m < M && n < N) {
          if (part)
            part[m * N + n] = acc[i][j][v];
          else
            out[m * N + n] = (T)acc[i][j][v];
        }
      }
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

// Copies of a matrix (R, C) that the products can read: rows padded with 0 to
// `pitch` values (plain), or its transpose (C rows of `pitch` values, R of them
// the matrix's, from column `at` on; 0 up to column `at` + pad).
template <typename T>
__global__ __launch_bounds__(256) void gated_pad_kernel(const T* __restrict__ in, int64_t R,
                                                        int64_t C, T* __restrict__ out,
                                                        int64_t pitch) {
  const int64_t n = R * pitch;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / pitch, c = i - r * pitch;
    out[i] = c < C ? in[r * C + c] : (T)0.f;
  }
}
template <typename T>
__global__ __launch_bounds__(256) void gated_turn_kernel(const T* __restrict__ in, int64_t R,
                                                         int64_t C, T* __restrict__ out,
                                                         int64_t pitch, int64_t pad) {
  __shared__ T s[64][65];
  const int64_t r0 = (int64_t)blockIdx.x * 64, c0 = (int64_t)blockIdx.y * 64;
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < 64; i += 4)
    s[y + i][x] = r0 + y + i < R && c0 + x < C ? in[(r0 + y + i) * C + c0 + x] : (T)0.f;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 64; i += 4)
    if (c0 + y + i < C && r0 + x < pad) out[(c0 + y + i) * pitch + r0 + x] = s[x][y + i];
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

// How a product of M x N sums over `bytes` of the summed axis is cut: the tile's
// edge and the number of shares of that axis.
struct Cut {
  int tile, shares;
};
Cut gated_cut(int64_t M, int64_t N, int64_t products, int64_t bytes, bool may_split) {
  const int64_t large = cdiv(M, 256) * cdiv(N, 256) * products;
  const int64_t small = cdiv(M, 128) * cdiv(N, 128) * products;
  Cut c{256, 1};
  if (large < 192) c.tile = 128;
  if (may_split) {
    const int64_t have = c.tile == 256 ? large : cdiv(small, 2);
    int64_t s = 256 / (have < 1 ? 1 : have);
    const int64_t most = bytes / (16 * SLAB);  // a share is worth its sums' way through memory
    if (s > most) s = most;
    c.shares = s < 1 ? 1 : (int)s;
  }
  return c;
}
inline int gated_share(int64_t bytes, int shares) {
  return (int)(cdiv(cdiv(bytes, SLAB), shares) * SLAB);
}

// What the calls keep in the workspace, in bytes from its start.
struct Plan {
  int64_t Kp, Fp, Mp;               // widths padded to 16 bytes
  int64_t x, wg, wu;                // padded copies (-1: the inputs do)
  int64_t d, dt, wt, xt, part;
  Cut dx, dw;
  int64_t bytes;
};
Plan gated_plan(int dtype, int64_t M, int64_t K, int64_t F, bool bwd) {
  const int64_t z = element_bytes(dtype), per = 16 / z;
  Plan p = {};
  p.Kp = round_up(K, per);
  p.Fp = round_up(F, per);
  p.Mp = round_up(M, per);
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
    p.d = take(M * 2 * p.Fp, z);
    p.dt = take(2 * F * p.Mp, z);
    p.wt = take(K * 2 * p.Fp, z);
    p.xt = take(K * p.Mp, z);
    p.dx = gated_cut(M, K, 1, 2 * p.Fp * z, true);
    p.dw = gated_cut(F, K, 2, p.Mp * z, true);
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
                  int64_t K, int64_t F, char* ws, hipStream_t s, Rows (&r)[3]) {
  const void* in[3] = {x, wg, wu};
  const int64_t at[3] = {p.x, p.wg, p.wu}, rows[3] = {M, F, F};
  for (int i = 0; i < 3; ++i) {
    if (at[i] >= 0)
      gated_pad_kernel<T><<<dim3(gated_blocks(rows[i] * p.Kp)), 256, 0, s>>>(
          (const T*)in[i], rows[i], K, (T*)(ws + at[i]), p.Kp);
    r[i] = Rows{at[i] >= 0 ? ws + at[i] : (const char*)in[i], p.Kp * (int64_t)sizeof(T), rows[i]};
  }
}

template <typename T, bool BWD>
void gated_pair(const Rows (&r)[3], int act, const T* gh, int64_t F, T* h, T* d, int64_t Fp, T* dt,
                int64_t Mp, hipStream_t s) {
  const int64_t M = r[0].rows;
  const Cut c = gated_cut(M, 2 * F, 1, r[0].pitch, false);
  const unsigned grid = (unsigned)(cdiv(M, c.tile) * cdiv(F, c.tile / 2));
  if (c.tile == 256)
    gated_pair_kernel<T, 256, 256, BWD><<<dim3(grid), 256, 0, s>>>(
        r[0], r[1], r[2], (int)r[0].pitch, act, gh, F, h, d, Fp, dt, Mp);
  else
    gated_pair_kernel<T, 128, 128, BWD><<<dim3(grid), 256, 0, s>>>(
        r[0], r[1], r[2], (int)r[0].pitch, act, gh, F, h, d, Fp, dt, Mp);
}

// out (and out2, the product with the rows of A after its first ones)
template <typename T>
void gated_product(const Rows& a, const Rows& b, const Cut& c, T* out, T* out2, float* part,
                   hipStream_t s) {
  const int products = out2 ? 2 : 1, share = gated_share(a.pitch, c.shares);
  const int shares = share > 0 ? (int)cdiv(a.pitch, share) : 1;
  const dim3 grid((unsigned)(cdiv(a.rows, c.tile) * cdiv(b.rows, c.tile)), products, shares);
  float* to = shares > 1 ? part : nullptr;
  if (c.tile == 256)
    gated_product_kernel<T, 256, 256><<<grid, 256, 0, s>>>(a, b, (int)a.pitch, share, out, out2, to);
  else
    gated_product_kernel<T, 128, 128><<<grid, 256, 0, s>>>(a, b, (int)a.pitch, share, out, out2, to);
  if (shares > 1)
    gated_join_kernel<T><<<dim3(gated_blocks(a.rows * b.rows), products), 256, 0, s>>>(
        part, shares, a.rows * b.rows, out, out2);
}

}  // namespace tpo

using namespace tpo;

extern "C" int64_t tpo_gated_fwd_workspace_size(int dtype, int64_t M, int64_t K, int64_t F) {
  if (gated_check("gated_fwd_workspace_size", dtype, M, K, F, TPO_ACT_SILU)) return -1;
  return gated_plan(dtype, M, K, F, false).bytes;
}

extern "C" int tpo_gated_fwd(int dtype, const void* x, const void* w_gate, const void* w_up,
                             int64_t M, int64_t K, int64_t F, int activation, void* h,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = gated_check("gated_fwd", dtype, M, K, F, activation)) return rc;
  if (M == 0 || F == 0) return TPO_OK;
  if (int rc = gated_aligned("gated_fwd", {x, w_gate, w_up, workspace})) return rc;
  const Plan p = gated_plan(dtype, M, K, F, false);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes))
    return set_error(TPO_ERR_WORKSPACE, "gated_fwd: workspace of %lld bytes needed",
                     (long long)p.bytes);
  hipStream_t s = (hipStream_t)stream;
  with_element(dtype, [&](auto t) {
    typedef decltype(t) T;
    Rows r[3];
    gated_inputs<T>(p, x, w_gate, w_up, M, K, F, (char*)workspace, s, r);
    gated_pair<T, false>(r, activation, nullptr, F, (T*)h, nullptr, 0, nullptr, 0, s);
  });
  return check_launch("gated_fwd");
}

extern "C" int64_t tpo_gated_bwd_workspace_size(int dtype, int64_t M, int64_t K, int64_t F) {
  if (gated_check("gated_bwd_workspace_size", dtype, M, K, F, TPO_ACT_SILU)) return -1;
  return gated_plan(dtype, M, K, F, true).bytes;
}

extern "C" int tpo_gated_bwd(int dtype, const void* grad_h, const void* x, const void* w_gate,
                             const void* w_up, int64_t M, int64_t K, int64_t F, int activation,
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
  with_element(dtype, [&](auto t) {
    typedef decltype(t) T;
    const int64_t z = sizeof(T);
    T *d = (T*)(ws + p.d), *dt = (T*)(ws + p.dt), *wt = (T*)(ws + p.wt), *xt = (T*)(ws + p.xt);
    float* part = (float*)(ws + p.part);
    if (M > 0 && F > 0) {
      Rows r[3];
      gated_inputs<T>(p, x, w_gate, w_up, M, K, F, ws, s, r);
      gated_pair<T, true>(r, activation, (const T*)grad_h, F, nullptr, d, p.Fp, dt, p.Mp, s);
    }
    if (grad_x && M > 0) {
      if (F > 0) {
        const dim3 grid((unsigned)cdiv(p.Fp, 64), (unsigned)cdiv(K, 64));
        gated_turn_kernel<T><<<grid, 256, 0, s>>>((const T*)w_gate, F, K, wt, 2 * p.Fp, p.Fp);
        gated_turn_kernel<T><<<grid, 256, 0, s>>>((const T*)w_up, F, K, wt + p.Fp, 2 * p.Fp, p.Fp);
      }
      gated_product<T>(Rows{(const char*)d, 2 * p.Fp * z, M}, Rows{(const char*)wt, 2 * p.Fp * z, K},
                       p.dx, (T*)grad_x, nullptr, part, s);
    }
    if (grad_w_gate && F > 0) {
      if (M > 0)
        gated_turn_kernel<T><<<dim3((unsigned)cdiv(p.Mp, 64), (unsigned)cdiv(K, 64)), 256, 0, s>>>(
            (const T*)x, M, K, xt, p.Mp, p.Mp);
      gated_product<T>(Rows{(const char*)dt, p.Mp * z, F}, Rows{(const char*)xt, p.Mp * z, K}, p.dw,
                       (T*)grad_w_gate, (T*)grad_w_up, part, s);
    }
  });
  return check_launch("gated_bwd");
}
