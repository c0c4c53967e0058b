// rotary.hip -- rotary positions of queries and keys, and their gradient (the same with the
// angles' sign turned).
#include <type_traits>

#include "rotary.hpp"

namespace tpo {

constexpr int TURN_THREADS = 256;
constexpr int TURN_ANGLES = 4096;  // cosines and sines in LDS

// A workgroup takes `block` tokens: first their angles, one a thread, then all heads' rows.
template <typename T, bool STREAM>
__global__ __launch_bounds__(TURN_THREADS) void rotary_kernel(
    const T* __restrict__ x, int64_t x_row, int64_t x_head, T* __restrict__ y, int64_t tokens,
    int H, int D, Turn turn, int back, int block) {
  extern __shared__ float4 lds[];
  float2* cs = (float2*)lds;
  const int64_t t0 = (int64_t)blockIdx.x * block;
  const int n = (int)(tokens - t0 < block ? tokens - t0 : block);
  const TurnAngles<T> angles(turn.pairs, turn.interleaved);
  TurnRows<T, TURN_THREADS, STREAM> rows(x, x_row, x_head, y, H, D, t0, n, turn.pairs,
                                         turn.interleaved);
  rows.load();
  for (int i = threadIdx.x; i < n * angles.pitch; i += TURN_THREADS) {
    const int t = i / angles.pitch, j = angles.pair(i % angles.pitch);
    if (j >= turn.pairs) continue;  // (its products go nowhere)
    double s, c;
    sine_cosine(turn.place(t0 + t, j) * turn.f[j], s, c);
    cs[i] = make_float2((float)(c * turn.m), (float)(back ? -s * turn.m : s * turn.m));
  }
  __syncthreads();
  rows.run(cs, nullptr);
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
  // tokens of a workgroup: about 16 KB of them (32768 x 20 x 128 bfloat16, through the caches: 2
  // to 4 tokens 81 us, 8 tokens 87, 32 91: a workgroup's angles come before its first store), and
  // 2048 workgroups
  const int64_t pitch = dtype == TPO_F32 ? TurnAngles<float>(t.pairs, t.interleaved).pitch
                                         : TurnAngles<half_t>(t.pairs, t.interleaved).pitch;
  int64_t block = 16384 / (heads * D * element_bytes(dtype));
  if (block > tokens / 2048) block = tokens / 2048;
  if (pitch > 0 && block > TURN_ANGLES / pitch) block = TURN_ANGLES / pitch;
  if (block < 1) block = 1;
  while ((tokens + block - 1) / block >= ((int64_t)1 << 24)) block *= 2;
  if (block * pitch > 2 * TURN_ANGLES)
    return set_error(TPO_ERR_ARG, "rotary: too many tokens");
  const bool stream_out = tokens * heads * D * element_bytes(dtype) > TURN_STREAM;
  const unsigned blocks = (unsigned)((tokens + block - 1) / block);
  const size_t lds = (size_t)(block * pitch * sizeof(float2));
  with_element(dtype, [&](auto e) {
    typedef decltype(e) T;
    auto launch = [&](auto streaming) {
      rotary_kernel<T, decltype(streaming)::value>
          <<<dim3(blocks), TURN_THREADS, lds, (hipStream_t)stream>>>(
              (const T*)x, x_row, x_head, (T*)y, tokens, (int)heads, (int)D, t, back, (int)block);
    };
    if (stream_out)
      launch(std::true_type());
    else
      launch(std::false_type());
  });
  return check_launch("rotary");
}
