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

// Sums over a team, two at a time.  The waves' sums go to one of two places in
// turn, so that a place is written again only after a barrier that follows its
// reads.
template <int TEAM>
struct TeamSums {
  float2 s[2][TEAM / 64];
};
template <int TEAM>
__device__ __forceinline__ void team_sum(float& a, float& b, TeamSums<TEAM>& lds, int& turn) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (TEAM > 64) {
    float2* s = lds.s[turn];
    turn ^= 1;
    if (lane_id() == 0) s[wave_id()] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < TEAM / 64; ++i) {
      a += s[i].x;
      b += s[i].y;
    }
  }
}
template <int TEAM>
__device__ __forceinline__ float team_sum(float a, TeamSums<TEAM>& lds, int& turn) {
  float none = 0.f;
  team_sum<TEAM>(a, none, lds, turn);
  return a;
}
constexpr int ln_threads(int team) { return team == 64 ? 256 : team; }

// A row held in registers by a team of 64 to 1024 lanes: N loads a lane of PER
// values (16 bytes) each.  Rows of other widths begin anywhere: the memory takes
// 16-byte accesses at any element (at 32768 x 1023 in bfloat16 one value a load
// took 188 us where this takes 77), and only a row's last piece goes value by
// value.  x is read once; the variance is taken about the mean, from the
// registers.  HBM-bound: what is read and written is all that counts, so teams go
// on to other rows with the weights in registers, and there are enough of them to
// keep the memory busy.
template <typename T, int PER, int N, int TEAM>
struct RowHeld {
  float v[N][PER];
  static __device__ __forceinline__ int64_t column(int i) {
    return ((int64_t)i * TEAM + threadIdx.x % TEAM) * PER;
  }
  __device__ __forceinline__ void load(const T* p, int64_t width, float none = 0.f) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t c = column(i);
      Piece<T, PER> x;
      if (c + PER <= width) {
        x = *(const Piece<T, PER>*)(p + c);
      } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) x.v[e] = c + e < width ? p[c + e] : (T)none;
      }
#pragma unroll
      for (int e = 0; e < PER; ++e) v[i][e] = (float)x.v[e];
    }
  }
  __device__ __forceinline__ void fill(float f) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < PER; ++e) v[i][e] = f;
  }
  // f in the places past the row's end
  __device__ __forceinline__ void past(int64_t width, float f) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (column(i) + PER > width) {
#pragma unroll
        for (int e = 0; e < PER; ++e)
          if (column(i) + e >= width) v[i][e] = f;
      }
  }
  __device__ __forceinline__ void store(T* p, int64_t width) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t c = column(i);
      Piece<T, PER> x;
#pragma unroll
      for (int e = 0; e < PER; ++e) x.v[e] = (T)v[i][e];
      if (c + PER <= width) {
        *(Piece<T, PER>*)(p + c) = x;
      } else {
#pragma unroll
        for (int e = 0; e < PER; ++e)
          if (c + e < width) p[c + e] = x.v[e];
      }
    }
  }
};

template <typename T, typename W, int PER, int N, int TEAM>
__global__ __launch_bounds__(ln_threads(TEAM)) void layer_norm_fwd_kernel(
    const T* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b, int64_t rows,
    int64_t width, float eps, T* __restrict__ y, float* __restrict__ mean,
    float* __restrict__ rstd) {
  __shared__ TeamSums<TEAM> s;
  int turn = 0;
  constexpr int TEAMS = ln_threads(TEAM) / TEAM;
  RowHeld<W, PER, N, TEAM> ws, bs;
  RowHeld<T, PER, N, TEAM> xs;
  int64_t r = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
  if (r >= rows) return;  // (with teams of several waves the whole workgroup)
  xs.load(x + r * width, width);
  if (w) ws.load(w, width); else ws.fill(1.f);
  if (b) bs.load(b, width); else bs.fill(0.f);
  const float per = 1.f / (float)width;
  for (;;) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < PER; ++e) t += xs.v[i][e];
    const float m = team_sum<TEAM>(t, s, turn) * per;
    t = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const float d = xs.v[i][e] - m;
        if (xs.column(i) + e < width) t = __builtin_fmaf(d, d, t);
      }
    const float q = 1.f / sqrtf(team_sum<TEAM>(t, s, turn) * per + eps);
    RowHeld<T, PER, N, TEAM> ys;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < PER; ++e)
        ys.v[i][e] = __builtin_fmaf((xs.v[i][e] - m) * q, ws.v[i][e], bs.v[i][e]);
    const int64_t next = r + (int64_t)gridDim.x * TEAMS;
    if (next < rows) xs.load(x + next * width, width);
    ys.store(y + r * width, width);
    if (mean && threadIdx.x % TEAM == 0) {
      mean[r] = m;
      rstd[r] = q;
    }
    if (next >= rows) return;
    r = next;
  }
}

// gx of the team's rows, and the sums over them that the weights' gradients
// need, a workgroup's in part[blockIdx.x] (weight, then bias).  gy and x are read
// once for all three results.
template <typename T, typename W, int PER, int N, int TEAM>
__global__ __launch_bounds__(ln_threads(TEAM)) void layer_norm_bwd_kernel(
    const T* __restrict__ gy, const T* __restrict__ x, const W* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd, int64_t rows, int64_t width,
    T* __restrict__ gx, float* __restrict__ part) {
  __shared__ TeamSums<TEAM> s;
  int turn = 0;
  __shared__ float sums[TEAM == 64 ? 2 * N * PER * 64 : 1];
  constexpr int TEAMS = ln_threads(TEAM) / TEAM;
  typedef RowHeld<T, PER, N, TEAM> Row;
  RowHeld<W, PER, N, TEAM> ws;
  if (w) ws.load(w, width, 1.f); else ws.fill(1.f);
  Row gs, xs;
  RowHeld<float, PER, N, TEAM> sw, sb;
  sw.fill(0.f);
  sb.fill(0.f);
  const float per = 1.f / (float)width;
  for (int64_t r = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM; r < rows;
       r += (int64_t)gridDim.x * TEAMS) {
    gs.load(gy + r * width, width);
    xs.load(x + r * width, width);
    const float m = mean[r], q = rstd[r];
    xs.past(width, m);  // h = 0: (0 - m) q can be infinite, and 0 times it no number
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const float h = (xs.v[i][e] - m) * q, y = gs.v[i][e], g = y * ws.v[i][e];
        xs.v[i][e] = h;  // (past the row's end y and h are 0: nothing is added)
        sw.v[i][e] = __builtin_fmaf(y, h, sw.v[i][e]);
        sb.v[i][e] += y;
        s1 += g;
        s2 = __builtin_fmaf(g, h, s2);
      }
    if (gx) {
      team_sum<TEAM>(s1, s2, s, turn);
      s1 *= per;
      s2 *= per;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < PER; ++e)
          xs.v[i][e] = q * (gs.v[i][e] * ws.v[i][e] - s1 - xs.v[i][e] * s2);
      xs.store(gx + r * width, width);
    }
  }
  if (!part) return;
  float* p = part + (int64_t)blockIdx.x * 2 * width;
  if constexpr (TEAM == 64) {  // the four waves' one after another
    for (int t = 0; t < 4; ++t) {
      __syncthreads();
      if (wave_id() == t)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int e = 0; e < PER; ++e) {
            const int at = (i * PER + e) * 64 + lane_id();
            sums[at] = (t ? sums[at] : 0.f) + sw.v[i][e];
            sums[at + N * PER * 64] = (t ? sums[at + N * PER * 64] : 0.f) + sb.v[i][e];
          }
    }
    __syncthreads();
    for (int64_t c = threadIdx.x; c < width; c += 256) {
      const int64_t i = c / (64 * PER), e = c % PER, l = c / PER % 64;
      const int at = (int)((i * PER + e) * 64 + l);
      p[c] = sums[at];
      p[width + c] = sums[at + N * PER * 64];
    }
  } else {
    sw.store(p, width);
    sb.store(p + width, width);
  }
}

// Rows longer than a team holds: sixteen waves a row, read again for each step (500 x
// 20000 in float, training: 512 us with one wave a row, 76 with sixteen).
constexpr int LN_LONG = 1024;
template <typename T, typename W>
__global__ __launch_bounds__(LN_LONG) void layer_norm_fwd_long_kernel(
    const T* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b, int64_t rows,
    int64_t width, float eps, T* __restrict__ y, float* __restrict__ mean,
    float* __restrict__ rstd) {
  __shared__ TeamSums<LN_LONG> lds;
  int turn = 0;
  const int lane = threadIdx.x;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * width;
    float s = 0.f;
    for (int64_t c = lane; c < width; c += LN_LONG) s += (float)xr[c];
    const float m = team_sum<LN_LONG>(s, lds, turn) / (float)width;
    float v = 0.f;
    for (int64_t c = lane; c < width; c += LN_LONG) {
      const float d = (float)xr[c] - m;
      v += d * d;
    }
    const float q = 1.f / sqrtf(team_sum<LN_LONG>(v, lds, turn) / (float)width + eps);
    for (int64_t c = lane; c < width; c += LN_LONG)
      y[r * width + c] = (T)(((float)xr[c] - m) * q * ln_at(w, c, 1.f) + ln_at(b, c, 0.f));
    if (lane == 0 && mean) {
      mean[r] = m;
      rstd[r] = q;
    }
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(LN_LONG) void layer_norm_bwd_long_kernel(
    const T* __restrict__ gy, const T* __restrict__ x, const W* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd, int64_t rows, int64_t width,
    T* __restrict__ gx) {
  __shared__ TeamSums<LN_LONG> lds;
  int turn = 0;
  const int lane = threadIdx.x;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float m = mean[r], q = rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t c = lane; c < width; c += LN_LONG) {
      const float g = (float)gy[r * width + c] * ln_at(w, c, 1.f);
      s1 += g;
      s2 += g * (((float)x[r * width + c] - m) * q);
    }
    team_sum<LN_LONG>(s1, s2, lds, turn);
    s1 /= (float)width;
    s2 /= (float)width;
    for (int64_t c = lane; c < width; c += LN_LONG) {
      const float g = (float)gy[r * width + c] * ln_at(w, c, 1.f);
      const float h = ((float)x[r * width + c] - m) * q;
      gx[r * width + c] = (T)(q * (g - s1 - h * s2));
    }
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

// Sums of the weight's and the bias's gradient for narrow and for long rows: a
// block sums 64 columns over its share of the rows.
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

// The shares added up, 64 of the 2 width columns a workgroup: sixteen waves take
// every sixteenth share each, in a fixed order.
template <typename W>
__global__ __launch_bounds__(1024) void layer_norm_bwd_sum_kernel(const float* __restrict__ part,
                                                                  int parts, int64_t width,
                                                                  W* __restrict__ gw,
                                                                  W* __restrict__ gb) {
  __shared__ float s[16][64];
  const int lane = lane_id(), wv = wave_id();
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float a = 0.f;
  if (c < 2 * width) {
    int p = wv;
    for (; p + 48 < parts; p += 64) {  // four loads under way
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = part[(int64_t)(p + 16 * i) * 2 * width + c];
      a += (y[0] + y[1]) + (y[2] + y[3]);
    }
    for (; p < parts; p += 16) a += part[(int64_t)p * 2 * width + c];
  }
  s[wv][lane] = a;
  __syncthreads();
  if (wv == 0 && c < 2 * width) {
    a = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) a += s[i][lane];
    W* to = c < width ? gw : gb;
    if (to) to[c < width ? c : c - width] = (W)a;
  }
}

// The kernels' build for a row: loads a lane, lanes a row; held false for rows
// longer than 1024 lanes hold.  A wave a row as long as the backward, which holds
// five arrays, leaves room for other waves; then more waves a row rather than
// more loads a lane (half types, training: 16000 x 2048 98 us with a wave a row, 74
// with four; 4000 x 8192 135 with four, 79 with sixteen), in float with two loads, so
// as many values, a lane (8000 x 3000: 99, with one 109).
struct LnForm {
  int n, team;
  bool held;
};
LnForm ln_form(int64_t width, int64_t size) {
  const int64_t loads = (width * size + 15) / 16;
  const bool single = size == 4;
  if (loads <= 64) return {1, 64, true};
  if (loads <= 128) return {2, 64, true};
  if (loads <= 256) return single ? LnForm{4, 64, true} : LnForm{1, 256, true};
  if (loads <= 512) return single ? LnForm{2, 256, true} : LnForm{1, 512, true};
  if (loads <= 1024) return single ? LnForm{2, 512, true} : LnForm{1, 1024, true};
  if (loads <= 2048) return {2, 1024, true};
  if (loads <= 4096 && single) return {4, 1024, true};  // (32768 half values spill)
  return {0, 0, false};
}
// Calls f with the form as types: values a load, loads, team.
template <typename T, typename F>
void with_form(const LnForm& f, F&& call) {
  constexpr int PER = 16 / sizeof(T);
#define LN_FORM(N, TEAM)                                                              \
  if (f.n == N && f.team == TEAM)                                                     \
  return call(std::integral_constant<int, PER>(), std::integral_constant<int, N>(),   \
              std::integral_constant<int, TEAM>())
  LN_FORM(1, 64);
  LN_FORM(2, 64);
  LN_FORM(2, 1024);
  if constexpr (sizeof(T) == 4) {
    LN_FORM(4, 64);
    LN_FORM(2, 256);
    LN_FORM(2, 512);
    LN_FORM(4, 1024);
  } else {
    LN_FORM(1, 256);
    LN_FORM(1, 512);
    LN_FORM(1, 1024);
  }
#undef LN_FORM
}

constexpr int64_t LN_WIDTH_MAX = 1 << 20;
inline dim3 ln_long_grid(int64_t rows) { return dim3((unsigned)(rows < 65536 ? rows : 65536)); }
// Workgroups where nothing is summed over the rows: up to eight a CU.
inline unsigned ln_blocks(int64_t rows, int64_t teams) {
  const int64_t n = (rows + teams - 1) / teams;
  return (unsigned)(n < 2048 ? n : 2048);
}
// Workgroups of the backward, which are the shares of the rows for the weights'
// gradients: as many as have a row for each of their teams, up to two a CU (one where a
// row takes sixteen waves); where a workgroup is one team, two rows each from half of
// that on; and one for every 8 rows beyond, as the shares' sums go through memory twice.
// (16 x 8192 in bfloat16: 11.6 us by 4 workgroups, 6.8 by 16; 256 x 8192: 16.3 by 256,
// 14.0 by 128; 500 x 16384: 41.5 by 64, 26.8 by 250; 1000 x 1500: 30.3 by 64, 13.8 by
// 500; 1000 x 700, four teams each: 16.0 by 64, 10.3 by 250.)  Loading the next row ahead
// of the sums instead was slower (32768 x 1024: 103 us for 80): it costs the registers
// of other workgroups.
int ln_parts(int64_t rows, int64_t width, int64_t size) {
  const LnForm f = ln_form(width, size);
  const int64_t teams = f.held ? ln_threads(f.team) / f.team : 4;
  int64_t few = (rows + teams - 1) / teams, most = !f.held ? 64 : f.team <= 512 ? 512 : 256;
  if (teams == 1 && few > most / 2) few = rows > most ? rows / 2 : most / 2;
  if (most < rows / 8) most = rows / 8;
  const int64_t top = width > 2048 ? 512 : 1024;
  if (most > top) most = top;
  return (int)(few < most ? few : most);
}
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
  if (rows > 0)
    if (int rc = all_there("layer_norm_fwd", {x, y})) return rc;
  hipStream_t s = (hipStream_t)stream;
  bool none = false;
  const int rc = ln_dispatch("layer_norm_fwd", dtype, wdtype, [&](auto t, auto w) {
    typedef decltype(t) T;
    typedef decltype(w) W;
    if (rows == 0) {
      none = true;
      return;
    }
    const LnForm f = ln_form(width, sizeof(T));
    if (!f.held) {
      layer_norm_fwd_long_kernel<T, W><<<ln_long_grid(rows), LN_LONG, 0, s>>>(
          (const T*)x, (const W*)weight, (const W*)bias, rows, width, (float)eps, (T*)y, mean,
          rstd);
      return;
    }
    with_form<T>(f, [&](auto per, auto n, auto team) {
      constexpr int TEAM = decltype(team)::value, THREADS = ln_threads(TEAM);
      layer_norm_fwd_kernel<T, W, decltype(per)::value, decltype(n)::value, TEAM>
          <<<dim3(ln_blocks(rows, THREADS / TEAM)), THREADS, 0, s>>>(
              (const T*)x, (const W*)weight, (const W*)bias, rows, width, (float)eps, (T*)y, mean,
              rstd);
    });
  });
  return rc || none ? rc : check_launch("layer_norm_fwd");
}

extern "C" int64_t tpo_layer_norm_bwd_workspace_size(int64_t rows, int64_t width) {
  if (ln_check("layer_norm_bwd_workspace_size", rows, width)) return -1;
  const int a = ln_parts(rows, width, 2), b = ln_parts(rows, width, 4);
  return round_up((int64_t)(a > b ? a : b) * 2 * width * 4, 256);
}

extern "C" int tpo_layer_norm_bwd(int dtype, int wdtype, const void* grad_y, const void* x,
                                  const void* weight, const float* mean, const float* rstd,
                                  int64_t rows, int64_t width, double eps, void* grad_x,
                                  void* grad_weight, void* grad_bias, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  if (int rc = ln_check("layer_norm_bwd", rows, width)) return rc;
  const bool sums = grad_weight || grad_bias;
  if (sums && (workspace_bytes < tpo_layer_norm_bwd_workspace_size(rows, width) ||
               (!workspace && rows > 0)))
    return set_error(TPO_ERR_WORKSPACE, "layer_norm_bwd: workspace of %lld bytes needed",
                     (long long)tpo_layer_norm_bwd_workspace_size(rows, width));
  if (rows > 0)
    if (int rc = all_there("layer_norm_bwd", {grad_y, x, mean, rstd})) return rc;
  hipStream_t s = (hipStream_t)stream;
  const int rc = ln_dispatch("layer_norm_bwd", dtype, wdtype, [&](auto t, auto w) {
    typedef decltype(t) T;
    typedef decltype(w) W;
    const LnForm f = ln_form(width, sizeof(T));
    const int parts = ln_parts(rows, width, sizeof(T));
    float* part = sums ? (float*)workspace : nullptr;
    if (rows > 0 && width > LN_NARROW && f.held) {
      with_form<T>(f, [&](auto per, auto n, auto team) {
        constexpr int TEAM = decltype(team)::value, THREADS = ln_threads(TEAM);
        const unsigned blocks = sums ? (unsigned)parts : ln_blocks(rows, THREADS / TEAM);
        layer_norm_bwd_kernel<T, W, decltype(per)::value, decltype(n)::value, TEAM>
            <<<dim3(blocks), THREADS, 0, s>>>(
                (const T*)grad_y, (const T*)x, (const W*)weight, mean, rstd, rows, width,
                (T*)grad_x, part);
      });
    } else if (rows > 0) {
      if (grad_x && width <= LN_NARROW)
        layer_norm_bwd_narrow_kernel<T, W><<<dim3((unsigned)((rows + 63) / 64)), 64, 0, s>>>(
            (const T*)grad_y, (const T*)x, (const W*)weight, eps, rows, (int)width, (T*)grad_x);
      else if (grad_x)
        layer_norm_bwd_long_kernel<T, W><<<ln_long_grid(rows), LN_LONG, 0, s>>>(
            (const T*)grad_y, (const T*)x, (const W*)weight, mean, rstd, rows, width, (T*)grad_x);
      if (sums)
        layer_norm_bwd_w_kernel<T><<<dim3((unsigned)((width + 63) / 64), parts), 256, 0, s>>>(
            (const T*)grad_y, (const T*)x, mean, rstd, rows, width, part);
    }
    if (sums)
      layer_norm_bwd_sum_kernel<W><<<dim3((unsigned)((2 * width + 63) / 64)), 1024, 0, s>>>(
          part, parts, width, (W*)grad_weight, (W*)grad_bias);
  });
  return rc ? rc : check_launch("layer_norm_bwd");
}
