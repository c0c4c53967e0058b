// gated.hip -- gated projection h = act(x Wg^T) * (x Wu^T) and its gradients.
//   x (M, K), Wg and Wu (F, K), h (M, F)
//   with g = x Wg^T, u = x Wu^T: dg = dh u act'(g), du = dh act(g),
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
#include "nn_common.hpp"

namespace tpo {

constexpr float INV_SQRT2 = 0.70710678118654752f;
constexpr float INV_SQRT_2PI = 0.39894228040143268f;

// The activation a and its derivative d.
template <int ACT>
__device__ __forceinline__ void gated_act(float g, float& a, float& d) {
  if (ACT == TPO_ACT_SILU || ACT == TPO_ACT_SIGMOID) {
    const float e = 1.f / (1.f + expf(-g));
    a = ACT == TPO_ACT_SILU ? g * e : e;
    d = ACT == TPO_ACT_SILU ? e * (1.f + g * (1.f - e)) : e * (1.f - e);
  } else if (ACT == TPO_ACT_GELU) {
    const float c = 0.5f * (1.f + erff(g * INV_SQRT2));
    a = g * c;
    d = c + g * expf(-0.5f * g * g) * INV_SQRT_2PI;
  } else {
    a = g > 0.f ? g : (g != g ? g : 0.f);
    d = g > 0.f ? 1.f : 0.f;
  }
}

constexpr int GP_T = 64;  // tile of outputs; 16 x 16 threads, 4 x 4 each
constexpr int GP_K = 16;

// acc += the tile's products A(i, k) B(j, k), A at a[i ai + k ak], B alike.
template <typename T>
__device__ __forceinline__ void gated_tile(const T* a, int64_t ai, int64_t ak, const T* b,
                                           int64_t bj, int64_t bk, int64_t I, int64_t J, int64_t N,
                                           int64_t i0, int64_t j0, float (&acc)[4][4]) {
  __shared__ float sa[GP_K][GP_T + 1], sb[GP_K][GP_T + 1];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int64_t k0 = 0; k0 < N; k0 += GP_K) {
    for (int e = threadIdx.x; e < GP_T * GP_K; e += 256) {
      const int k = e & (GP_K - 1), i = e / GP_K;
      const bool in = k0 + k < N;
      sa[k][i] = in && i0 + i < I ? (float)a[(i0 + i) * ai + (k0 + k) * ak] : 0.f;
      sb[k][i] = in && j0 + i < J ? (float)b[(j0 + i) * bj + (k0 + k) * bk] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < GP_K; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __builtin_fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
}

// h, or with gh its gradients dg and du.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void gated_pair_kernel(
    const T* __restrict__ x, const T* __restrict__ wg, const T* __restrict__ wu,
    const T* __restrict__ gh, int64_t M, int64_t K, int64_t F, T* __restrict__ h,
    T* __restrict__ dg, T* __restrict__ du) {
  const int64_t i0 = (int64_t)blockIdx.y * GP_T, j0 = (int64_t)blockIdx.x * GP_T;
  float g[4][4] = {}, u[4][4] = {};
  gated_tile<T>(x, K, 1, wg, K, 1, M, F, K, i0, j0, g);
  gated_tile<T>(x, K, 1, wu, K, 1, M, F, K, i0, j0, u);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = i0 + ty * 4 + i, c = j0 + tx * 4 + j;
      if (r >= M || c >= F) continue;
      float a, d;
      gated_act<ACT>(g[i][j], a, d);
      if (gh) {
        const float e = (float)gh[r * F + c];
        dg[r * F + c] = (T)(e * u[i][j] * d);
        du[r * F + c] = (T)(e * a);
      } else {
        h[r * F + c] = (T)(a * u[i][j]);
      }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void gated_dx_kernel(const T* __restrict__ dg,
                                                       const T* __restrict__ du,
                                                       const T* __restrict__ wg,
                                                       const T* __restrict__ wu, int64_t M,
                                                       int64_t K, int64_t F, T* __restrict__ dx) {
  const int64_t i0 = (int64_t)blockIdx.y * GP_T, j0 = (int64_t)blockIdx.x * GP_T;
  float acc[4][4] = {};
  gated_tile<T>(dg, F, 1, wg, 1, K, M, K, F, i0, j0, acc);
  gated_tile<T>(du, F, 1, wu, 1, K, M, K, F, i0, j0, acc);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = i0 + ty * 4 + i, c = j0 + tx * 4 + j;
      if (r < M && c < K) dx[r * K + c] = (T)acc[i][j];
    }
}

template <typename T>
__global__ __launch_bounds__(256) void gated_dw_kernel(const T* __restrict__ dg,
                                                       const T* __restrict__ du,
                                                       const T* __restrict__ x, int64_t M,
                                                       int64_t K, int64_t F, T* __restrict__ dwg,
                                                       T* __restrict__ dwu) {
  const int64_t i0 = (int64_t)blockIdx.y * GP_T, j0 = (int64_t)blockIdx.x * GP_T;
  float acc[4][4] = {};
  gated_tile<T>(blockIdx.z ? du : dg, 1, F, x, 1, K, F, K, M, i0, j0, acc);
  T* out = blockIdx.z ? dwu : dwg;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = i0 + ty * 4 + i, c = j0 + tx * 4 + j;
      if (r < F && c < K) out[r * K + c] = (T)acc[i][j];
    }
}

int gated_check(const char* op, int dtype, int64_t M, int64_t K, int64_t F, int act) {
  if (dtype != TPO_F32 && dtype != TPO_F16 && dtype != TPO_BF16)
    return set_error(TPO_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (M < 0 || K < 1 || F < 0 || M > (1 << 22) || K > (1 << 20) || F > (1 << 20))
    return set_error(TPO_ERR_ARG, "%s: bad sizes M=%lld K=%lld F=%lld", op, (long long)M,
                     (long long)K, (long long)F);
  if (act < TPO_ACT_SILU || act > TPO_ACT_SIGMOID)
    return set_error(TPO_ERR_ARG, "%s: unknown activation %d", op, act);
  return TPO_OK;
}

template <typename F>
void with_act(int act, F&& f) {
  switch (act) {
    case TPO_ACT_SILU: f(std::integral_constant<int, TPO_ACT_SILU>()); break;
    case TPO_ACT_GELU: f(std::integral_constant<int, TPO_ACT_GELU>()); break;
    case TPO_ACT_RELU: f(std::integral_constant<int, TPO_ACT_RELU>()); break;
    default: f(std::integral_constant<int, TPO_ACT_SIGMOID>()); break;
  }
}

inline unsigned tiles(int64_t n) { return (unsigned)((n + GP_T - 1) / GP_T); }

}  // namespace tpo

using namespace tpo;

extern "C" int64_t tpo_gated_fwd_workspace_size(int dtype, int64_t M, int64_t K, int64_t F) {
  if (gated_check("gated_fwd_workspace_size", dtype, M, K, F, TPO_ACT_SILU)) return -1;
  return 0;
}

extern "C" int tpo_gated_fwd(int dtype, const void* x, const void* w_gate, const void* w_up,
                             int64_t M, int64_t K, int64_t F, int activation, void* h,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = gated_check("gated_fwd", dtype, M, K, F, activation)) return rc;
  (void)workspace;
  (void)workspace_bytes;
  if (M == 0 || F == 0) return TPO_OK;
  with_element(dtype, [&](auto t) {
    typedef decltype(t) T;
    with_act(activation, [&](auto act) {
      gated_pair_kernel<T, decltype(act)::value>
          <<<dim3(tiles(F), tiles(M)), 256, 0, (hipStream_t)stream>>>(
              (const T*)x, (const T*)w_gate, (const T*)w_up, nullptr, M, K, F, (T*)h, nullptr,
              nullptr);
    });
  });
  return check_launch("gated_fwd");
}

extern "C" int64_t tpo_gated_bwd_workspace_size(int dtype, int64_t M, int64_t K, int64_t F) {
  if (gated_check("gated_bwd_workspace_size", dtype, M, K, F, TPO_ACT_SILU)) return -1;
  return 2 * round_up(M * F * element_bytes(dtype), 256);
}

extern "C" int tpo_gated_bwd(int dtype, const void* grad_h, const void* x, const void* w_gate,
                             const void* w_up, int64_t M, int64_t K, int64_t F, int activation,
                             void* grad_x, void* grad_w_gate, void* grad_w_up, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  if (int rc = gated_check("gated_bwd", dtype, M, K, F, activation)) return rc;
  const int64_t need = tpo_gated_bwd_workspace_size(dtype, M, K, F);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(TPO_ERR_WORKSPACE, "gated_bwd: workspace of %lld bytes needed",
                     (long long)need);
  hipStream_t s = (hipStream_t)stream;
  with_element(dtype, [&](auto t) {
    typedef decltype(t) T;
    T* dg = (T*)workspace;
    T* du = (T*)((char*)workspace + need / 2);
    if (M > 0 && F > 0)
      with_act(activation, [&](auto act) {
        gated_pair_kernel<T, decltype(act)::value><<<dim3(tiles(F), tiles(M)), 256, 0, s>>>(
            (const T*)x, (const T*)w_gate, (const T*)w_up, (const T*)grad_h, M, K, F, nullptr, dg,
            du);
      });
    if (grad_x && M > 0)
      gated_dx_kernel<T><<<dim3(tiles(K), tiles(M)), 256, 0, s>>>(
          dg, du, (const T*)w_gate, (const T*)w_up, M, K, F, (T*)grad_x);
    if (grad_w_gate && F > 0)
      gated_dw_kernel<T><<<dim3(tiles(K), tiles(F), 2), 256, 0, s>>>(
          dg, du, (const T*)x, M, K, F, (T*)grad_w_gate, (T*)grad_w_up);
  });
  return check_launch("gated_bwd");
}
