// rotary.hip -- rotary positions of queries and keys, and their gradient (the same with the
// angles' sign turned).
#include "rotary.hpp"

namespace tpo {

constexpr int TURN_THREADS = 256;
constexpr int TURN_ANGLES = 4096;  // cosines and sines in LDS

// A workgroup takes `block` tokens: first their angles, one a thread, then all heads' rows.
template <typename T>
__global__ __launch_bounds__(TURN_THREADS) void rotary_kernel(
    const T* __restrict__ x, int64_t x_row, int64_t x_head, T* __restrict__ y, int64_t tokens,
    int H, int D, Turn turn, int back, int block) {
  extern __shared__ float2 cs[];
  const int64_t t0 = (int64_t)blockIdx.x * block;
  const int n = (int)(tokens - t0 < block ? tokens - t0 : block);
  for (int i = threadIdx.x; i < n * turn.pairs; i += TURN_THREADS) {
    const int t = i / turn.pairs, j = i % turn.pairs;
    double s, c;
    sine_cosine(turn.place(t0 + t, j) * turn.f[j], s, c);
    cs[i] = make_float2((float)(c * turn.m), (float)(back ? -s * turn.m : s * turn.m));
  }
  __syncthreads();
  turn_rows<T, TURN_THREADS>(x, x_row, x_head, y, H, D, t0, n, turn.pairs, turn.interleaved, cs,
                             nullptr);
}

int turn_args(const char* op, const double* f, const void* at, int64_t pairs, int64_t axes,
              int floats, int interleaved, double m, int64_t D, Turn& t) {
  if (pairs < 0 || 2 * pairs > D || axes < 1 || pairs % axes != 0)
    return set_error(TPO_ERR_ARG,
                     "%s: bad sizes pairs=%lld axes=%lld D=%lld (two values a pair, the pairs a "
                     "multiple of the axes)",
                     op, (long long)pairs, (long long)axes, (long long)D);
  t.f = f;
  t.at = at;
  t.pairs = (int)pairs;
  t.axes = (int)axes;
  t.each = pairs > 0 ? (int)(pairs / axes) : 1;
  t.interleaved = interleaved ? 1 : 0;
  t.floats = floats;
  t.m = m;
  return TPO_OK;
}

}  // namespace tpo

using namespace tpo;

extern "C" int tpo_rotary(int dtype, const void* x, int64_t tokens, int64_t heads, int64_t D,
                          int64_t x_row, int64_t x_head, const void* places, int places_dtype,
                          int64_t axes, const double* frequencies, int64_t pairs, int interleaved,
                          double amplitude, int back, void* y, void* stream) {
  if (dtype != TPO_F32 && dtype != TPO_F16 && dtype != TPO_BF16)
    return set_error(TPO_ERR_DTYPE, "rotary: unsupported dtype %d", dtype);
  if (places_dtype != TPO_I64 && places_dtype != TPO_F32)
    return set_error(TPO_ERR_DTYPE, "rotary: places must be I64 or F32, but got %d", places_dtype);
  if (tokens < 0 || tokens >= ((int64_t)1 << 31) || heads < 0 || heads > (1 << 16) || D < 1 ||
      D > TURN_DMAX)
    return set_error(TPO_ERR_ARG, "rotary: bad sizes tokens=%lld heads=%lld D=%lld (at most %d)",
                     (long long)tokens, (long long)heads, (long long)D, TURN_DMAX);
  Turn t;
  if (int rc = turn_args("rotary", frequencies, places, pairs, axes, places_dtype == TPO_F32,
                         interleaved, amplitude, D, t))
    return rc;
  if (tokens == 0 || heads == 0) return TPO_OK;
  if (int rc = all_there("rotary", {x, y})) return rc;
  if (pairs > 0)
    if (int rc = all_there("rotary", {places, frequencies})) return rc;
  // tokens of a workgroup: enough workgroups for every CU's places (8 of 256 threads), then
  // as many as share the launch of one
  int64_t block = tokens / 4096;
  if (block > 16) block = 16;
  if (pairs > 0 && block > TURN_ANGLES / pairs) block = TURN_ANGLES / pairs;
  if (block < 1) block = 1;
  while ((tokens + block - 1) / block >= ((int64_t)1 << 24)) block *= 2;
  if (block * pairs > 2 * TURN_ANGLES)
    return set_error(TPO_ERR_ARG, "rotary: too many tokens");
  with_element(dtype, [&](auto e) {
    typedef decltype(e) T;
    rotary_kernel<T><<<dim3((unsigned)((tokens + block - 1) / block)), TURN_THREADS,
                       (size_t)(block * pairs * sizeof(float2)), (hipStream_t)stream>>>(
        (const T*)x, x_row, x_head, (T*)y, tokens, (int)heads, (int)D, t, back, (int)block);
  });
  return check_launch("rotary");
}
