// layer_norm.hip -- layer norm over the last axis, forward and backward.
//   y = (x - mean) r w + b,  r = 1 / sqrt(var + eps)
//   with g = gy w and h = (x - mean) r:
//   gx = r (g - mean(g) - h mean(g h)),  gw = sum over rows of gy h,
//   gb = sum over rows of gy
#include "nn_common.hpp"

namespace tpo {

template <typename W>
__device__ __forceinline__ float ln_at(const W* w, int64_t c, float none) {
  return w ? (float)w[c] : none;
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void layer_norm_fwd_kernel(
    const T* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b, int64_t rows,
    int64_t width, float eps, T* __restrict__ y, float* __restrict__ mean,
    float* __restrict__ rstd) {
  const int64_t r = (int64_t)blockIdx.x * 4 + wave_id();
  if (r >= rows) return;
  const int lane = lane_id();
  const T* xr = x + r * width;
  float s = 0.f;
  for (int64_t c = lane; c < width; c += 64) s += (float)xr[c];
  const float m = wave_sum(s) / (float)width;
  float v = 0.f;
  for (int64_t c = lane; c < width; c += 64) {
    const float d = (float)xr[c] - m;
    v += d * d;
  }
  const float q = 1.f / sqrtf(wave_sum(v) / (float)width + eps);
  for (int64_t c = lane; c < width; c += 64)
    y[r * width + c] = (T)(((float)xr[c] - m) * q * ln_at(w, c, 1.f) + ln_at(b, c, 0.f));
  if (lane == 0 && mean) {
    mean[r] = m;
    rstd[r] = q;
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void layer_norm_bwd_x_kernel(
    const T* __restrict__ gy, const T* __restrict__ x, const W* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd, int64_t rows, int64_t width,
    T* __restrict__ gx) {
  const int64_t r = (int64_t)blockIdx.x * 4 + wave_id();
  if (r >= rows) return;
  const int lane = lane_id();
  const float m = mean[r], q = rstd[r];
  float s1 = 0.f, s2 = 0.f;
  for (int64_t c = lane; c < width; c += 64) {
    const float g = (float)gy[r * width + c] * ln_at(w, c, 1.f);
    s1 += g;
    s2 += g * (((float)x[r * width + c] - m) * q);
  }
  s1 = wave_sum(s1) / (float)width;
  s2 = wave_sum(s2) / (float)width;
  for (int64_t c = lane; c < width; c += 64) {
    const float g = (float)gy[r * width + c] * ln_at(w, c, 1.f);
    const float h = ((float)x[r * width + c] - m) * q;
    gx[r * width + c] = (T)(q * (g - s1 - h * s2));
  }
}

// Rows of up to LN_NARROW values, a lane a row, in double from x itself: where
// two values are all of a row, h is +-1 but for eps, and the gradient is what
// eps leaves of a difference that float would lose.
constexpr int LN_NARROW = 8;
template <typename T, typename W>
__global__ __launch_bounds__(64) void layer_norm_bwd_narrow_kernel(
    const T* __restrict__ gy, const T* __restrict__ x, const W* __restrict__ w, double eps,
    int64_t rows, int width, T* __restrict__ gx) {
  const int64_t r = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (r >= rows) return;
  double m = 0, v = 0, s1 = 0, s2 = 0;
  for (int c = 0; c < width; ++c) m += (double)(float)x[r * width + c];
  m /= width;
  for (int c = 0; c < width; ++c) {
    const double d = (double)(float)x[r * width + c] - m;
    v += d * d;
  }
  const double q = 1 / sqrt(v / width + eps);
  for (int c = 0; c < width; ++c) {
    const double g = (double)(float)gy[r * width + c] * ln_at(w, c, 1.f);
    s1 += g;
    s2 += g * (((double)(float)x[r * width + c] - m) * q);
  }
  for (int c = 0; c < width; ++c) {
    const double g = (double)(float)gy[r * width + c] * ln_at(w, c, 1.f);
    const double h = ((double)(float)x[r * width + c] - m) * q;
    gx[r * width + c] = (T)(float)(q * (g - s1 / width - h * (s2 / width)));
  }
}

// Sums of the weight's and the bias's gradient: a block sums 64 columns over
// its share of the rows, the second kernel adds the shares in order.
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_bwd_w_kernel(
    const T* __restrict__ gy, const T* __restrict__ x, const float* __restrict__ mean,
    const float* __restrict__ rstd, int64_t rows, int64_t width, float* __restrict__ part) {
  __shared__ float sw[4][64], sb[4][64];
  const int lane = lane_id(), wv = wave_id();
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float a = 0.f, b = 0.f;
  if (c < width)
    for (int64_t r = (int64_t)blockIdx.y * 4 + wv; r < rows; r += (int64_t)gridDim.y * 4) {
      const float g = (float)gy[r * width + c];
      a += g * (((float)x[r * width + c] - mean[r]) * rstd[r]);
      b += g;
    }
  sw[wv][lane] = a;
  sb[wv][lane] = b;
  __syncthreads();
  if (wv == 0 && c < width) {
    float* p = part + (int64_t)blockIdx.y * 2 * width;
    p[c] = sw[0][lane] + sw[1][lane] + sw[2][lane] + sw[3][lane];
    p[width + c] = sb[0][lane] + sb[1][lane] + sb[2][lane] + sb[3][lane];
  }
}

template <typename W>
__global__ __launch_bounds__(256) void layer_norm_bwd_sum_kernel(const float* __restrict__ part,
                                                                 int parts, int64_t width,
                                                                 W* __restrict__ gw,
                                                                 W* __restrict__ gb) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= width) return;
  float a = 0.f, b = 0.f;
  for (int p = 0; p < parts; ++p) {
    a += part[(int64_t)p * 2 * width + c];
    b += part[(int64_t)p * 2 * width + width + c];
  }
  if (gw) gw[c] = (W)a;
  if (gb) gb[c] = (W)b;
}

constexpr int64_t LN_WIDTH_MAX = 1 << 20;
inline int ln_parts(int64_t rows) { return (int)(rows < 256 ? (rows + 3) / 4 : 64); }

// The weights are of the input's type or float.
template <typename F>
int ln_dispatch(const char* op, int dtype, int wdtype, F&& f) {
  if (wdtype != dtype && wdtype != TPO_F32)
    return set_error(TPO_ERR_DTYPE, "%s: weight dtype %d with input dtype %d", op, wdtype, dtype);
  const bool ok = with_element(dtype, [&](auto t) {
    if (wdtype == TPO_F32)
      f(t, float());
    else
      f(t, t);
  });
  return ok ? TPO_OK : set_error(TPO_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
}

int ln_check(const char* op, int64_t rows, int64_t width) {
  if (rows < 0 || rows >= ((int64_t)1 << 31) || width < 1 || width > LN_WIDTH_MAX)
    return set_error(TPO_ERR_ARG, "%s: bad sizes rows=%lld width=%lld", op, (long long)rows,
                     (long long)width);
  return TPO_OK;
}

}  // namespace tpo

using namespace tpo;

extern "C" int tpo_layer_norm_fwd(int dtype, int wdtype, const void* x, const void* weight,
                                  const void* bias, int64_t rows, int64_t width, double eps,
                                  void* y, float* mean, float* rstd, void* stream) {
  if (int rc = ln_check("layer_norm_fwd", rows, width)) return rc;
  if ((mean == nullptr) != (rstd == nullptr))
    return set_error(TPO_ERR_ARG, "layer_norm_fwd: mean and rstd go together");
  hipStream_t s = (hipStream_t)stream;
  bool none = false;
  const int rc = ln_dispatch("layer_norm_fwd", dtype, wdtype, [&](auto t, auto w) {
    typedef decltype(t) T;
    typedef decltype(w) W;
    if (rows == 0) {
      none = true;
      return;
    }
    layer_norm_fwd_kernel<T, W><<<dim3((unsigned)((rows + 3) / 4)), 256, 0, s>>>(
        (const T*)x, (const W*)weight, (const W*)bias, rows, width, (float)eps, (T*)y, mean, rstd);
  });
  return rc || none ? rc : check_launch("layer_norm_fwd");
}

extern "C" int64_t tpo_layer_norm_bwd_workspace_size(int64_t rows, int64_t width) {
  if (ln_check("layer_norm_bwd_workspace_size", rows, width)) return -1;
  return round_up((int64_t)ln_parts(rows) * 2 * width * 4, 256);
}

extern "C" int tpo_layer_norm_bwd(int dtype, int wdtype, const void* grad_y, const void* x,
                                  const void* weight, const float* mean, const float* rstd,
                                  int64_t rows, int64_t width, double eps, void* grad_x,
                                  void* grad_weight, void* grad_bias, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  if (int rc = ln_check("layer_norm_bwd", rows, width)) return rc;
  const bool sums = grad_weight || grad_bias;
  if (sums && (workspace_bytes < tpo_layer_norm_bwd_workspace_size(rows, width) ||
               (!workspace && rows > 0)))
    return set_error(TPO_ERR_WORKSPACE, "layer_norm_bwd: workspace of %lld bytes needed",
                     (long long)tpo_layer_norm_bwd_workspace_size(rows, width));
  hipStream_t s = (hipStream_t)stream;
  const int rc = ln_dispatch("layer_norm_bwd", dtype, wdtype, [&](auto t, auto w) {
    typedef decltype(t) T;
    typedef decltype(w) W;
    if (grad_x && rows > 0 && width <= LN_NARROW)
      layer_norm_bwd_narrow_kernel<T, W><<<dim3((unsigned)((rows + 63) / 64)), 64, 0, s>>>(
          (const T*)grad_y, (const T*)x, (const W*)weight, eps, rows, (int)width, (T*)grad_x);
    else if (grad_x && rows > 0)
      layer_norm_bwd_x_kernel<T, W><<<dim3((unsigned)((rows + 3) / 4)), 256, 0, s>>>(
          (const T*)grad_y, (const T*)x, (const W*)weight, mean, rstd, rows, width, (T*)grad_x);
    if (!sums) return;
    const int parts = ln_parts(rows);
    if (parts > 0)
      layer_norm_bwd_w_kernel<T><<<dim3((unsigned)((width + 63) / 64), parts), 256, 0, s>>>(
          (const T*)grad_y, (const T*)x, mean, rstd, rows, width, (float*)workspace);
    layer_norm_bwd_sum_kernel<W><<<dim3((unsigned)((width + 255) / 256)), 256, 0, s>>>(
        (const float*)workspace, parts, width, (W*)grad_weight, (W*)grad_bias);
  });
  return rc ? rc : check_launch("layer_norm_bwd");
}
