// cache_append.hip -- new tokens of many sequences into the pages of an 8-bit cache, keys (and
// the queries beside them) turned by their places on the way.
//   token i of the n new ones of a sequence of `length` tokens: place length - n + i
//   code = e4m3(value / 2^e), e of the page and head: the smallest with every value of the page
//   at most 448 2^e, between -40 and 40
// Scales are powers of two: e4m3 loses nothing by it (its own exponent has the rest), a code's
// value is exact in every type, and older codes of a page whose scale grows stay as they are but
// for those that become subnormal.  Values that are not finite become the code for NaN and do
// not count for the scale.
#include "cache.hpp"
#include "rotary.hpp"

namespace tpo {

constexpr int APPEND_THREADS = 256;
constexpr int E_LEAST = -40, E_MOST = 40;
constexpr float CODE_MOST = 448.f;

// A double as a float whose last bit says that something was cut off (rounding to odd), so that
// the next rounding, to a code, is that of the double itself.  Keys are turned in 64 bits and
// rounded once in all: their codes are those of the exact products.
__device__ __forceinline__ float to_odd(double d) {
  const float f = (float)d;
  const double rest = d - (double)f;
  int b = __builtin_bit_cast(int, f);
  if (rest != 0. && !(b & 1) && fabsf(f) < __builtin_inff()) b += (rest > 0.) == (f > 0.f) ? 1 : -1;
  return __builtin_bit_cast(float, b);
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_inff(); }

// The smallest e with top <= 448 2^e (448 = 0.875 2^9).
__device__ __forceinline__ int exponent_for(float top) {
  int e;
  const float m = frexpf(top, &e);
  e += m > 0.875f ? -8 : -9;
  if (top == 0.f || e < E_LEAST) e = E_LEAST;
  return e > E_MOST ? E_MOST : e;
}
// The smallest e with scale <= 2^e, for a scale from anywhere.
__device__ __forceinline__ int exponent_of(float scale) {
  if (!(scale > 0.f)) return E_LEAST;
  if (!finite(scale)) return E_MOST;
  int e;
  const float m = frexpf(scale, &e);
  if (m == 0.5f) --e;
  return e < E_LEAST ? E_LEAST : (e > E_MOST ? E_MOST : e);
}
__device__ __forceinline__ float power(int e) { return __builtin_bit_cast(float, (e + 127) << 23); }

__device__ __forceinline__ float for_code(float v, float f) {
  const float y = __builtin_amdgcn_fmed3f(v * f, -CODE_MOST, CODE_MOST);
  return finite(v) ? y : __builtin_nanf("");
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
__device__ __forceinline__ uint32_t codes4(const float* v, float f) {
  return codes4(for_code(v[0], f), for_code(v[1], f), for_code(v[2], f), for_code(v[3], f));
}
// Four codes brought to another scale.
__device__ __forceinline__ uint32_t codes_times(uint32_t x, float f) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false);
  const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
  return codes4(a[0] * f, a[1] * f, b[0] * f, b[1] * f);
}

// The call's rows: strides in elements.
template <typename T>
struct AppendRows {
  const T *k, *v, *q;
  T* q_out;
  int64_t k_row, k_head, v_row, v_head, q_row, q_head;
  int Hq, D, places;  // places: the turn's places are given, not the tokens' own
};

// Sixteen values from p on, n of them there.
template <typename T>
__device__ __forceinline__ void load16(const T* p, int n, float (&x)[16]) {
  constexpr int PER = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 16; i += PER) {
    const Piece<T, PER> u = n - i > 0 ? some<T, PER>(p + i, n - i) : Piece<T, PER>{};
#pragma unroll
    for (int e = 0; e < PER; ++e) x[i + e] = (float)u.v[e];
  }
}

// Values d0 .. d0 + 15 of a head turned: row, the head's D values; cs, the token's cosines and
// sines.
template <typename T>
__device__ __forceinline__ void turn16(const T* row, int d0, int D, const Turn& t,
                                       const double2* cs, float (&x)[16]) {
  const int n = t.pairs;
  if (d0 >= 2 * n) return;
  if (t.interleaved) {
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const int j = (d0 + e) / 2;
      if (j < n) {
        const double2 w = cs[j];
        const double a = x[e], b = x[e + 1];
        x[e] = to_odd(__builtin_fma(-b, w.y, a * w.x));
        x[e + 1] = to_odd(__builtin_fma(a, w.y, b * w.x));
      }
    }
    return;
  }
  constexpr int PER = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 16; i += PER) {
    const int d = d0 + i;
    if (d >= 2 * n) break;
    Piece<T, PER> u;
    if (d + PER <= n)  // a piece in one half: its partners lie together
      u = *(const Piece<T, PER>*)(row + d + n);
    else if (d >= n && d + PER <= 2 * n)
      u = *(const Piece<T, PER>*)(row + d - n);
    else
#pragma unroll
      for (int e = 0; e < PER; ++e)
        u.v[e] = d + e < n ? row[d + e + n] : (d + e < 2 * n ? row[d + e - n] : (T)0.f);
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int j = d + e < n ? d + e : d + e - n;
      if (j < n) {
        const double2 w = cs[j];
        const double s = d + e < n ? -w.y : w.y;
        x[i + e] = to_odd(__builtin_fma((double)(float)u.v[e], s, (double)x[i + e] * w.x));
      }
    }
  }
}

__device__ __forceinline__ float top16(const float (&x)[16], float top) {
#pragma unroll
  for (int e = 0; e < 16; ++e) top = fmaxf(top, finite(x[e]) ? fabsf(x[e]) : 0.f);
  return top;
}

// The queries' part: `block` tokens of a workgroup turned by their places.
template <typename T>
__device__ __forceinline__ void append_queries(const Cache& c, const Sequences& sq,
                                               const Turn& turn, const AppendRows<T>& r,
                                               int64_t t0, int block, char* lds) {
  const int n = (int)(sq.T - t0 < block ? sq.T - t0 : block);
  float2* cs = (float2*)lds;
  int* at = (int*)(cs + block * turn.pairs);
  int* live = at + block;
  for (int t = wave_id(); t < n; t += APPEND_THREADS / 64) {
    const CacheRows s =
        cache_rows(sq, c, t0 + t, [](int64_t start, int) { return start; });
    const int i = (int)(t0 + t - s.first), p = s.length - s.used + i;
    if (lane_id() == 0) {
      at[t] = p;
      live[t] = s.b >= 0 && i < s.used && p >= 0;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * turn.pairs; i += APPEND_THREADS) {
    const int t = i / turn.pairs, j = i % turn.pairs;
    const double p = r.places ? turn.place(t0 + t, j) : (double)at[t];
    double s, co;
    sine_cosine(p * turn.f[j], s, co);
    cs[i] = make_float2((float)(co * turn.m), (float)(s * turn.m));
  }
  __syncthreads();
  turn_rows<T, APPEND_THREADS>(r.q, r.q_row, r.q_head, r.q_out, r.Hq, r.D, t0, n, turn.pairs,
                               turn.interleaved, cs, live);
}

// Workgroups 0 .. places * groups take a sequence's page and `heads` of its heads each, one team
// of TEAM lanes a head: a wave where a page gets a few tokens, the workgroup where it gets
// many.  A lane has sixteen values of a token's key and of its value at a time (CH times), which
// are what it stores of a key and, a token's part of sixteen rows, of a value; `round` tokens go
// through at a time.  Where a page is one round (any but a large page of wide heads), what was
// loaded stays in registers between the largest value and the codes; else it is loaded again.
// The workgroups behind them turn `block` tokens' queries each.
template <typename T, int TEAM, int CH>
__global__ __launch_bounds__(APPEND_THREADS) void cache_append_kernel(Cache c, Sequences sq,
                                                                      Turn turn, AppendRows<T> r,
                                                                      int groups, int heads,
                                                                      int round, int kv, int block) {
  extern __shared__ double2 lds[];
  if ((int)blockIdx.x >= kv) {
    append_queries<T>(c, sq, turn, r, (int64_t)((int)blockIdx.x - kv) * block, block, (char*)lds);
    return;
  }
  constexpr int TEAMS = APPEND_THREADS / TEAM;
  const int64_t place = blockIdx.x / groups;
  const int page = c.page, NC = c.chunks;
  const CacheRows s = cache_rows(sq, c, place, [page](int64_t start, int i) {
    return start / page + 2 * (int64_t)i;
  });
  if (s.b < 0) return;
  const int before = s.length - s.used;  // the place of the first new token
  const int from = before < 0 ? 0 : before;
  if (from >= s.length) return;
  const int64_t past = place - s.place;
  if (past > (s.length - 1) / page - from / page) return;
  const int pi = from / page + (int)past;
  const int number = __builtin_amdgcn_readfirstlane(c.page_of(s.b, pi));
  if (number < 0) return;
  const int base = pi * page;
  const int a = from > base ? from - base : 0;                          // slots a .. z - 1 are new
  const int z = s.length - base < page ? s.length - base : page;
  const int64_t row0 = s.first + base - before;                         // slot 0's row

  double2* cs = lds;
  char* tile = (char*)(cs + round * turn.pairs);
  const int tile_pitch = round + 4;
  float* tops = (float*)(tile + (TEAMS == 1 ? tile_pitch * 16 * NC : 0));
  const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
  int tok[CH], chunk[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    tok[i] = (lane + i * TEAM) / NC;
    chunk[i] = (lane + i * TEAM) % NC;
  }
  // rounds begin at multiples of their length where the values' tile is turned over, so that a
  // round holds whole blocks
  const int r0 = TEAMS == 1 ? a / round * round : a;
  const int rounds = (z - r0 + round - 1) / round;
  float k[CH][16], v[CH][16];

  auto angles = [&](int t0) {
    const int n = z - t0 < round ? z - t0 : round;
    for (int i = threadIdx.x; i < n * turn.pairs; i += APPEND_THREADS) {
      const int t = t0 + i / turn.pairs, j = i % turn.pairs;
      if (t < a) continue;
      const double p = r.places ? turn.place(row0 + t, j) : (double)(base + t);
      double sn, co;
      sine_cosine(p * turn.f[j], sn, co);
      cs[i] = make_double2(co * turn.m, sn * turn.m);
    }
  };
  auto in = [&](int t0, int i) {
    const int t = t0 + tok[i];
    return tok[i] < round && t >= a && t < z;
  };
  auto load = [&](int t0, int h) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if (!in(t0, i)) continue;
      const int64_t row = row0 + t0 + tok[i];
      const int d0 = 16 * chunk[i];
      const T* kr = r.k + row * r.k_row + h * r.k_head;
      load16<T>(kr + d0, r.D - d0, k[i]);
      load16<T>(r.v + row * r.v_row + h * r.v_head + d0, r.D - d0, v[i]);
      turn16<T>(kr, d0, r.D, turn, cs + tok[i] * turn.pairs, k[i]);
    }
  };

  const int h0 = (blockIdx.x % groups) * heads;
  const int h1 = h0 + heads < c.Hk ? h0 + heads : c.Hk;
  for (int hh = h0; hh < h1; hh += TEAMS) {
    const bool mine = hh + team < h1;
    const int h = mine ? hh + team : h1 - 1;
    const int64_t scale_at = (int64_t)number * c.Hk + h;
    const float old_k = a > 0 ? c.key_scales[scale_at] : 0.f;
    const float old_v = a > 0 ? c.value_scales[scale_at] : 0.f;
    float top_k = 0.f, top_v = 0.f;
    for (int y = 0; y < rounds; ++y) {
      if (rounds > 1 || hh == h0) {
        __syncthreads();
        angles(r0 + y * round);
        __syncthreads();
      }
      load(r0 + y * round, h);
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (in(r0 + y * round, i)) {
          top_k = top16(k[i], top_k);
          top_v = top16(v[i], top_v);
        }
    }
    top_k = wave_max(top_k);
    top_v = wave_max(top_v);
    if (TEAMS == 1) {
      __syncthreads();
      if (lane_id() == 0) {
        tops[wave_id()] = top_k;
        tops[4 + wave_id()] = top_v;
      }
      __syncthreads();
      top_k = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      top_v = fmaxf(fmaxf(tops[4], tops[5]), fmaxf(tops[6], tops[7]));
    }
    int ek = exponent_for(top_k), ev = exponent_for(top_v);
    if (a > 0) {
      const int ok = exponent_of(old_k), ov = exponent_of(old_v);
      ek = ok > ek ? ok : ek;
      ev = ov > ev ? ov : ev;
    }
    const float fk = power(-ek), fv = power(-ev);

    // older codes of the page at a new scale
    if (a > 0 && mine && (old_k != power(ek) || old_v != power(ev))) {
      if (old_k != power(ek))
        for (int i = lane; i < a * NC; i += TEAM) {
          const int t = i / NC;
          uint4* p = (uint4*)(c.keys + c.block(number, h, t / 32) + (i % NC) * 512 + t % 32 * 16);
          uint4 x = *p;
          x.x = codes_times(x.x, old_k * fk);
          x.y = codes_times(x.y, old_k * fk);
          x.z = codes_times(x.z, old_k * fk);
          x.w = codes_times(x.w, old_k * fk);
          *p = x;
        }
      if (old_v != power(ev)) {
        const int rows = 16 * NC;
        // four tokens of a value at a time, those of new tokens and behind left as they are
        for (int i = lane; i < (a + 3) / 4 * rows; i += TEAM) {
          const int t = i / rows * 4, d = i % rows;
          uint32_t* p = (uint32_t*)(c.values + c.block(number, h, t / 32) + d * 32 + t % 32);
          const uint32_t x = *p, keep = a - t >= 4 ? ~0u : (1u << 8 * (a - t)) - 1;
          *p = (codes_times(x, old_v * fv) & keep) | (x & ~keep);
        }
      }
      __threadfence();  // (a new token's codes may share a word with older ones)
    }
    if (TEAMS == 1 && a > 0) __syncthreads();
    if (mine && lane == 0) {
      c.key_scales[scale_at] = power(ek);
      c.value_scales[scale_at] = power(ev);
    }

    for (int y = 0; y < rounds; ++y) {
      const int t0 = r0 + y * round;
      if (rounds > 1) {
        __syncthreads();
        angles(t0);
        __syncthreads();
        load(t0, h);
      }
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        if (!in(t0, i) || !mine) continue;
        const int t = t0 + tok[i];
        const int64_t block_at = c.block(number, h, t / 32);
        uint4 x;
        x.x = codes4(k[i], fk);
        x.y = codes4(k[i] + 4, fk);
        x.z = codes4(k[i] + 8, fk);
        x.w = codes4(k[i] + 12, fk);
        *(uint4*)(c.keys + block_at + chunk[i] * 512 + t % 32 * 16) = x;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = codes4(v[i] + 4 * e, fv);
        if (TEAMS == 1) {
          char* to = tile + chunk[i] * 16 * tile_pitch + tok[i];
#pragma unroll
          for (int e = 0; e < 16; ++e) to[e * tile_pitch] = (char)(w[e / 4] >> 8 * (e % 4));
        } else {
          uint8_t* to = c.values + block_at + chunk[i] * 512 + t % 32;
#pragma unroll
          for (int e = 0; e < 16; ++e) to[e * 32] = (uint8_t)(w[e / 4] >> 8 * (e % 4));
        }
      }
      if (TEAMS == 1) {
        __syncthreads();
        const int rows = 16 * NC;
        for (int i = threadIdx.x; i < round / 16 * rows; i += APPEND_THREADS) {
          const int half = i & 1, d = (i >> 1) % rows, blk = (i >> 1) / rows;
          const int lt = 32 * blk + 16 * half, t = t0 + lt;
          if (t + 16 <= a || t >= z) continue;
          uint8_t* to = c.values + c.block(number, h, t / 32) + d * 32 + t % 32;
          const uint32_t* at = (const uint32_t*)(tile + d * tile_pitch + lt);
          const uint4 x = make_uint4(at[0], at[1], at[2], at[3]);
          if (t >= a && t + 16 <= z)
            *(uint4*)to = x;
          else
            for (int e = 0; e < 16; ++e)
              if (t + e >= a && t + e < z) to[e] = ((const uint8_t*)at)[e];
        }
        __syncthreads();
      }
    }
  }
}

int cache_check(const char* op, int64_t pages, int64_t Hk, int64_t page, int64_t Dr, int64_t B,
                int64_t M, int64_t D) {
  if (pages < 0 || pages >= ((int64_t)1 << 31) || Hk < 1 || Hk > 1024 || page < CACHE_BLOCK ||
      page > CACHE_PAGE || page % CACHE_BLOCK != 0 || D < 1 || D > CACHE_DMAX ||
      Dr != round_up(D, 16) || B < 0 || B > (1 << 24) || M < 0 ||
      M * page >= ((int64_t)1 << 31) || M >= ((int64_t)1 << 31))
    return set_error(TPO_ERR_ARG,
                     "%s: bad sizes pages=%lld Hk=%lld page=%lld Dr=%lld B=%lld M=%lld D=%lld "
                     "(pages of 32 to %d tokens in steps of 32, D at most %d and Dr the next "
                     "multiple of 16, M page below 2^31)",
                     op, (long long)pages, (long long)Hk, (long long)page, (long long)Dr,
                     (long long)B, (long long)M, (long long)D, CACHE_PAGE, CACHE_DMAX);
  return TPO_OK;
}

Cache cache_args(const void* keys, const void* values, const float* key_scales,
                 const float* value_scales, const int32_t* table, const int64_t* lengths,
                 int64_t pages, int64_t Hk, int64_t page, int64_t D, int64_t M) {
  Cache c;
  c.keys = (uint8_t*)keys;
  c.values = (uint8_t*)values;
  c.key_scales = (float*)key_scales;
  c.value_scales = (float*)value_scales;
  c.table = table;
  c.lengths = lengths;
  c.pages = pages;
  c.M = (int)M;
  c.page = (int)page;
  c.Hk = (int)Hk;
  c.chunks = (int)((D + 15) / 16);
  return c;
}

template <typename T, int TEAM, int CH>
void append_launch(const Cache& c, const Sequences& sq, const Turn& t, const AppendRows<T>& r,
                   int64_t places, int groups, int heads, int64_t q_blocks, int block,
                   hipStream_t s) {
  // tokens of a round: what the team's lanes hold, whole blocks for a workgroup
  int round = TEAM * CH / c.chunks;
  if (TEAM == APPEND_THREADS) round = round >= c.page ? c.page : round / 32 * 32;
  const int64_t angles = (int64_t)round * t.pairs * sizeof(double2);
  const int64_t kv_lds =
      angles + (TEAM == APPEND_THREADS ? (int64_t)(round + 4) * 16 * c.chunks : 0) + 64;
  const int64_t q_lds = (int64_t)block * t.pairs * sizeof(float2) + block * 2 * sizeof(int);
  cache_append_kernel<T, TEAM, CH>
      <<<dim3((unsigned)(places * groups + q_blocks)), APPEND_THREADS,
         (size_t)(kv_lds > q_lds ? kv_lds : q_lds), s>>>(c, sq, t, r, groups, heads, round,
                                                         (int)(places * groups), block);
}

}  // namespace tpo

using namespace tpo;

extern "C" int tpo_cache_append(int dtype, const void* k, const void* v, const void* q,
                                const int64_t* offsets, const int64_t* lengths_new, int64_t B,
                                int64_t T, int64_t Hq, int64_t D, int64_t k_row, int64_t k_head,
                                int64_t v_row, int64_t v_head, int64_t q_row, int64_t q_head,
                                const void* places, int places_dtype, int64_t axes,
                                const double* frequencies, int64_t pairs, int interleaved,
                                double amplitude, void* keys, void* values, float* key_scales,
                                float* value_scales, const int32_t* table, const int64_t* lengths,
                                int64_t pages, int64_t Hk, int64_t page, int64_t Dr, int64_t M,
                                void* q_out, void* stream) {
  const char* op = "cache_append";
  if (dtype != TPO_F32 && dtype != TPO_F16 && dtype != TPO_BF16)
    return set_error(TPO_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (places && places_dtype != TPO_I64 && places_dtype != TPO_F32)
    return set_error(TPO_ERR_DTYPE, "%s: places must be I64 or F32, but got %d", op, places_dtype);
  if (int rc = cache_check(op, pages, Hk, page, Dr, B, M, D)) return rc;
  if (T < 0 || T >= ((int64_t)1 << 31) || (q && (Hq < 1 || Hq > 1024)))
    return set_error(TPO_ERR_ARG, "%s: bad sizes T=%lld Hq=%lld", op, (long long)T, (long long)Hq);
  Turn t;
  if (int rc = turn_args(op, frequencies, places, pairs, places ? axes : 1,
                         places_dtype == TPO_F32, interleaved, amplitude, D, t))
    return rc;
  if (T == 0) return TPO_OK;
  if (int rc = all_there(op, {k, v, offsets})) return rc;
  if (B > 0)
    if (int rc = all_there(op, {lengths})) return rc;
  if (pairs > 0)
    if (int rc = all_there(op, {frequencies})) return rc;
  if (q)
    if (int rc = all_there(op, {q_out})) return rc;
  if (pages > 0)
    if (int rc = all_there(op, {keys, values, key_scales, value_scales})) return rc;
  if (B > 0 && M > 0)
    if (int rc = all_there(op, {table})) return rc;
  if (((uintptr_t)keys | (uintptr_t)values) & 15)
    return set_error(TPO_ERR_ARG, "%s: keys and values must be 16-byte aligned", op);
  const Cache c = cache_args(keys, values, key_scales, value_scales, table, lengths, pages, Hk,
                             page, D, M);
  const Sequences sq{offsets, lengths_new, T, (int)B};
  // a place for each page that a sequence's new tokens may lie in, see the kernel
  const int64_t slots = T / page + 2 * (B + 2);
  const bool few = T <= 8 * B;
  int64_t heads = few ? (Hk < 4 ? Hk : 4) : 1;
  if (!few)
    while (heads < Hk && (T / page + B) * ((Hk + heads) / (heads + 1)) >= 1024) ++heads;
  const int64_t groups = (Hk + heads - 1) / heads;
  int64_t block = few ? 1 : T / 4096;
  block = block > 16 ? 16 : (block < 1 ? 1 : block);
  const int64_t q_blocks = q ? (T + block - 1) / block : 0;
  if (slots * groups + q_blocks >= ((int64_t)1 << 24))
    return set_error(TPO_ERR_ARG, "%s: too many tokens", op);
  with_element(dtype, [&](auto e) {
    typedef decltype(e) E;
    const AppendRows<E> r{(const E*)k, (const E*)v, (const E*)q, (E*)q_out, k_row, k_head, v_row,
                          v_head, q_row, q_head, (int)Hq, (int)D, places ? 1 : 0};
    if (few)
      append_launch<E, 64, 1>(c, sq, t, r, slots, (int)groups, (int)heads, q_blocks, (int)block,
                              (hipStream_t)stream);
    else
      append_launch<E, APPEND_THREADS, 2>(c, sq, t, r, slots, (int)groups, (int)heads, q_blocks,
                                          (int)block, (hipStream_t)stream);
  });
  return check_launch(op);
}
