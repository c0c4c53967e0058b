// cache_append.hip -- new tokens of many sequences into the pages of an 8-bit cache, keys (and
// the queries beside them) turned by their places on the way.
//   token i of the n new ones of a sequence of `length` tokens: place length - n + i
//   code = e4m3(value / 2^e), e of the page and head: the smallest with every value of the page
//   at most 448 2^e, between -40 and 40
// Scales are powers of two: e4m3 loses nothing by it (its own exponent has the rest), a code's
// value is exact in every type, and older codes of a page whose scale grows stay as they are but
// for those that become subnormal.  Values that are not finite become the code for NaN and do
// not count for the scale.
#include <type_traits>

#include "cache.hpp"
#include "cache_codes.hpp"
#include "rotary.hpp"

namespace tpo {

__device__ __forceinline__ float power(int e) { return __builtin_bit_cast(float, (e + 127) << 23); }

__device__ __forceinline__ float for_code(float v, float f) {
  const float y = __builtin_amdgcn_fmed3f(v * f, -CODE_MOST, CODE_MOST);
  return finite(v) ? y : __builtin_nanf("");
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
// rare: values that are not finite, or a scale that is as large as it gets
__device__ __forceinline__ uint32_t codes4(const float* v, float f, bool rare) {
  if (rare)
    return codes4(for_code(v[0], f), for_code(v[1], f), for_code(v[2], f), for_code(v[3], f));
  return codes4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
}
// Four codes brought to another scale; f > 1 only where the old scale was above the largest.
__device__ __forceinline__ uint32_t codes_times(uint32_t x, float f) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false);
  const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
  const float v[4] = {a[0], a[1], b[0], b[1]};
  return codes4(v, f, f > 1.f);
}

// The call's rows: strides in elements.
template <typename T>
struct AppendRows {
  const T *k, *v, *q;
  T* q_out;
  int64_t k_row, k_head, v_row, v_head, q_row, q_head;
  int Hq, D, places;  // places: the turn's places are given, not the tokens' own
};

// A lane's part of a token's key or value: two pieces of eight values, from pa and from pb on.
// Keys that are turned: eight pairs (halves: the pieces lie n apart; interleaved: side by side);
// the others sixteen values side by side.  load: how many are there, store: how many the cache
// has (those behind D are 0).
struct Part {
  int pa, pb, load_a, load_b, store_a, store_b, pair;  // pair: the first, -1: not turned

  static __device__ __forceinline__ int upto8(int n) { return n < 0 ? 0 : (n > 8 ? 8 : n); }
  __device__ __forceinline__ void plain(int from, int D, int Dr) {
    pa = from;
    pb = from + 8;
    load_a = upto8(D - pa);
    load_b = upto8(D - pb);
    store_a = upto8(Dr - pa);
    store_b = upto8(Dr - pb);
    pair = -1;
  }
  __device__ __forceinline__ void key(int i, const Turn& t, int D, int Dr) {
    const int turned = (t.pairs + 7) / 8;
    if (i >= turned) {
      plain(2 * t.pairs + 16 * (i - turned), D, Dr);
      return;
    }
    pair = 8 * i;
    pa = t.interleaved ? 16 * i : 8 * i;
    pb = t.interleaved ? 16 * i + 8 : t.pairs + 8 * i;
    const int n = t.pairs - pair;
    load_a = store_a = upto8(t.interleaved ? 2 * n : n);
    load_b = store_b = upto8(t.interleaved ? 2 * n - 8 : n);
  }
  // What follows from these is worked out where it is used: kept for all heads it would take
  // 100 registers more.
  __device__ __forceinline__ void fresh() {
    asm volatile("" : "+v"(pa), "+v"(pb), "+v"(load_a), "+v"(load_b), "+v"(store_a), "+v"(store_b));
  }
  // parts of a token: of its key, and of its value
  static __host__ __device__ __forceinline__ int of_key(int pairs, int Dr) {
    return (pairs + 7) / 8 + (Dr - 2 * pairs + 15) / 16;
  }
};

template <typename T>
struct PartValues {
  Loaded<T, 8> a, b;
  __device__ __forceinline__ void load(const T* row, const Part& p) {
    a = some<T, 8>(row + p.pa, p.load_a);
    b = some<T, 8>(row + p.pb, p.load_b);
  }
  __device__ __forceinline__ void fresh() {
    a.fresh();
    b.fresh();
  }
  // the sixteen as floats
  __device__ __forceinline__ void to(float (&x)[16]) const {
    const Piece<T, 8> p = a.values(), q = b.values();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = (float)p.v[e];
      x[8 + e] = (float)q.v[e];
    }
  }
};

// Eight pairs turned, x[e] and x[8 + e] being pair e; angle(e): its cosine and sine.  ODD: rounded
// to odd; else to the nearest float, which has the same code but where it lies half-way between
// two of them, or is 0 or infinite: its last 19 bits are 0 then (e4m3 keeps 3 of 23): true where
// one may.
template <bool ODD, typename T, typename F>
__device__ __forceinline__ bool turn_pairs(const PartValues<T>& u, bool interleaved,
                                           const F& angle, float (&x)[16]) {
  const Piece<T, 8> p = u.a.values(), q = u.b.values();
  uint32_t least = ~0u;
  auto rounded = [&](double d) {
    const float f = ODD ? to_odd(d) : (float)d;
    const uint32_t low = __builtin_bit_cast(uint32_t, f) & 0x7ffff;
    least = low < least ? low : least;
    return f;
  };
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = 2 * e & 7;
    const T s0 = e < 4 ? p.v[i] : q.v[i], s1 = e < 4 ? p.v[i + 1] : q.v[i + 1];  // side by side
    const double v0 = (float)(interleaved ? s0 : p.v[e]);
    const double v1 = (float)(interleaved ? s1 : q.v[e]);
    const double2 cs = angle(e);
    x[e] = rounded(__builtin_fma(-v1, cs.y, v0 * cs.x));
    x[8 + e] = rounded(__builtin_fma(v0, cs.y, v1 * cs.x));
    if (e % 2) __builtin_amdgcn_sched_barrier(0);
  }
  return least == 0;
}
template <typename T, typename F>
__device__ __forceinline__ void turn_part(const PartValues<T>& u, bool interleaved, const F& angle,
                                          float (&x)[16]) {
  if (turn_pairs<false>(u, interleaved, angle, x)) turn_pairs<true>(u, interleaved, angle, x);
}

// Eight codes to a key's place in a block: values d .. d + n - 1 of a token.
__device__ __forceinline__ void store_part(uint8_t* block, int token, int d, int n, uint32_t lo,
                                           uint32_t hi) {
  uint8_t* to = block + token * 16;
  if (n == 8 && d % 8 == 0) {
    *(uint2*)(to + d / 16 * 512 + d % 16) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n)
        to[(d + e) / 16 * 512 + (d + e) % 16] = (uint8_t)((e < 4 ? lo : hi) >> 8 * (e % 4));
  }
}

// The queries' part: `block` tokens of a workgroup turned by their places.
template <typename T, int THREADS, bool STREAM>
__device__ __forceinline__ void append_queries(const Cache& c, const Sequences& sq,
                                               const Turn& turn, const AppendRows<T>& r,
                                               int64_t t0, int block, char* lds) {
  const int n = (int)(sq.T - t0 < block ? sq.T - t0 : block);
  const TurnAngles<T> angles(turn.pairs, turn.interleaved);
  float2* cs = (float2*)lds;
  int* at = (int*)(cs + block * angles.pitch);
  int* live = at + block;
  TurnRows<T, THREADS, STREAM> rows(r.q, r.q_row, r.q_head, r.q_out, r.Hq, r.D, t0, n, turn.pairs,
                                    turn.interleaved);
  rows.load();
  for (int t = wave_id(); t < n; t += THREADS / 64) {
    const CacheRows s =
        cache_rows(sq, c, t0 + t, [](int64_t start, int) { return start; });
    const int i = (int)(t0 + t - s.first), p = s.length - s.used + i;
    if (lane_id() == 0) {
      at[t] = p;
      live[t] = s.b >= 0 && i < s.used && p >= 0;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * angles.pitch; i += THREADS) {
    const int t = i / angles.pitch, j = angles.pair(i % angles.pitch);
    if (j >= turn.pairs) continue;
    const double p = r.places ? turn.place(t0 + t, j) : (double)at[t];
    double s, co;
    sine_cosine(p * turn.f[j], s, co);
    cs[i] = make_float2((float)(co * turn.m), (float)(s * turn.m));
  }
  __syncthreads();
  rows.run(cs, live);
}

// The same in a launch of its own, 8 waves a SIMD, for more queries than the caches hold: their
// way to and from memory is all that counts (21 thousand tokens, 16 heads of 128 in bfloat16: 33
// us, 5.3 TB/s; behind the pages' workgroups in one launch, 16 waves a CU, both took 83 where the
// pages alone took 47).
template <typename T>
__global__ __launch_bounds__(256) void cache_queries_kernel(Cache c, Sequences sq, Turn turn,
                                                            AppendRows<T> r, int block) {
  extern __shared__ double2 lds[];
  append_queries<T, 256, true>(c, sq, turn, r, (int64_t)blockIdx.x * block, block, (char*)lds);
}

// The page's older codes (slots below a) at a new scale, sixteen bytes at a time (a wave's lanes
// with four of them under way): of keys sixteen values of a token, of values sixteen tokens.  A
// piece that ends with new tokens gets its older bytes one by one, so that no byte is written
// twice and the new ones need not wait.
template <int TEAM>
__device__ __forceinline__ void scale_older(const Cache& c, uint8_t* codes, int64_t number, int h,
                                            bool key, int a, float f, int lane) {
  constexpr int N = TEAM == 64 ? 4 : 1;
  const int rows = 16 * c.chunks, all = key ? a * c.chunks : (a + 15) / 16 * rows;
#pragma unroll 1
  for (int i0 = lane; i0 < all; i0 += N * TEAM) {
    uint4 x[N];
    uint8_t* p[N];
    int left[N];
#pragma unroll
    for (int y = 0; y < N; ++y) {
      const int i = i0 + y * TEAM;
      left[y] = 0;
      if (i >= all) continue;
      const int t = key ? i / c.chunks : i / rows * 16, d = key ? i % c.chunks : i % rows;
      p[y] = codes + c.block(number, h, t / 32) +
             (key ? d * 512 + t % 32 * 16 : d * 32 + t % 32);
      left[y] = key ? 16 : a - t;
      x[y] = *(const uint4*)p[y];
    }
#pragma unroll
    for (int y = 0; y < N; ++y) {
      if (left[y] == 0) continue;
      const uint4 w = make_uint4(codes_times(x[y].x, f), codes_times(x[y].y, f),
                                 codes_times(x[y].z, f), codes_times(x[y].w, f));
      if (left[y] >= 16) {
        *(uint4*)p[y] = w;
      } else {
#pragma unroll 1
        for (int e = 0; e < left[y]; ++e) {
          const uint32_t v = e < 8 ? (e < 4 ? w.x : w.y) : (e < 12 ? w.z : w.w);
          p[y][e] = (uint8_t)(v >> 8 * (e % 4));
        }
      }
    }
  }
}

// A workgroup's page: which tokens of which sequence are new in it.
struct AppendPage {
  int found;      // what the table says of the page
  int number;     // the page, -1: none
  int base;       // the place of its first slot
  int a, z;       // slots a .. z - 1 are new
  int64_t row0;   // slot 0's row

  __device__ __forceinline__ AppendPage(const Cache& c, const Sequences& sq, int64_t place) {
    const int page = c.page;
    const CacheRows s = cache_rows(sq, c, place, [page](int64_t start, int i) {
      return start / page + 2 * (int64_t)i;
    });
    a = z = 0;
    if (s.b < 0) return;
    const int before = s.length - s.used;  // the place of the first new token
    const int from = before < 0 ? 0 : before;
    if (from >= s.length) return;
    const int64_t past = place - s.place;
    if (past > (s.length - 1) / page - from / page) return;
    const int pi = from / page + (int)past;
    found = c.page_of(s.b, pi);
    base = pi * page;
    a = from > base ? from - base : 0;
    z = s.length - base < page ? s.length - base : page;
    row0 = s.first + base - before;
  }
  // no new tokens here
  __device__ __forceinline__ bool none() const { return z == 0; }
  // Whether there is a page; asked for once the rows' loads are on their way.
  __device__ __forceinline__ bool there() {
    number = __builtin_amdgcn_readfirstlane(found);
    return number >= 0;
  }
};

// The angles of a part's pairs, of the token in slot t.
template <typename T>
__device__ __forceinline__ void part_angles(const Part& p, const Turn& turn,
                                            const AppendRows<T>& r, const AppendPage& g, int t,
                                            double2 (&cs)[8]) {
  double f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = turn.f[p.pair + e < turn.pairs ? p.pair + e : p.pair];
  if (r.places) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      cs[e].x = turn.place(g.row0 + t, p.pair + e < turn.pairs ? p.pair + e : p.pair) * f[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e].x = (double)(g.base + t) * f[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    double s, c;
    sine_cosine(cs[e].x, s, c);
    cs[e] = make_double2(c * turn.m, s * turn.m);
    if (e % 2) __builtin_amdgcn_sched_barrier(0);  // (eight at once: 200 registers)
  }
}

// The largest of what is finite among sixteen values, as bits; rare: some are not.
__device__ __forceinline__ uint32_t top16(const float (&x)[16], bool& rare) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffff;
    top = b > top ? b : top;
  }
  rare = top >= 0x7f800000;
  if (rare) {
    top = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const uint32_t b = __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffff;
      top = b > top && b < 0x7f800000 ? b : top;
    }
  }
  return top;
}

// The largest of a wave's numbers, the same in all lanes: within sixteen lanes by moves between
// lanes, then over the four of them.
__device__ __forceinline__ uint32_t wave_top(uint32_t v) {
  auto with = [&](auto move) {
    const uint32_t o =
        (uint32_t)__builtin_amdgcn_mov_dpp((int)v, decltype(move)::value, 15, 15, true);
    v = o > v ? o : v;
  };
  with(std::integral_constant<int, 0xb1>());   // the neighbour
  with(std::integral_constant<int, 0x4e>());   // two on
  with(std::integral_constant<int, 0x141>());  // the other four of eight
  with(std::integral_constant<int, 0x140>());  // the other eight of sixteen
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 64; i += 16) {
    const uint32_t o = __builtin_amdgcn_readlane((int)v, i);
    top = o > top ? o : top;
  }
  return top;
}

// The exponent of a page's scale: of its new values (the largest's bits), and not below the old
// scale's where the page holds older codes.
__device__ __forceinline__ int page_exponent(uint32_t top, bool older, float old) {
  const int e = exponent_for(__builtin_bit_cast(float, top));
  if (!older) return e;
  const int o = exponent_of(old);
  return o > e ? o : e;
}

// Sixteen values' codes, of a key's part or a value's.
__device__ __forceinline__ void codes16(const float (&x)[16], float f, bool rare, bool together,
                                        uint32_t (&w)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = codes4(x + 4 * e, f, rare || f == power(-E_MOST));
  if (together) {  // the first and second of pairs side by side again
    const uint32_t p[4] = {w[0], w[1], w[2], w[3]};
    w[0] = __builtin_amdgcn_perm(p[2], p[0], 0x05010400);
    w[1] = __builtin_amdgcn_perm(p[2], p[0], 0x07030602);
    w[2] = __builtin_amdgcn_perm(p[3], p[1], 0x05010400);
    w[3] = __builtin_amdgcn_perm(p[3], p[1], 0x07030602);
  }
}

// A round's values, turned over in LDS (a value's tokens side by side, `pitch` bytes from one
// value to the next), to a page's blocks: slots t0 .. t0 + round - 1, those of a .. z - 1.
template <int THREADS>
__device__ __forceinline__ void store_tile(const Cache& c, const char* tile, int pitch,
                                           const AppendPage& g, int h, int t0, int round) {
  const int Dr = 16 * c.chunks;
  for (int i = threadIdx.x; i < round / 16 * Dr; i += THREADS) {
    const int half = i & 1, d = (i >> 1) % Dr, blk = (i >> 1) / Dr;
    const int lt = 32 * blk + 16 * half, t = t0 + lt;
    if (t + 16 <= g.a || t >= g.z) continue;
    uint8_t* to = c.values + c.block(g.number, h, t / 32) + d * 32 + t % 32;
    const uint32_t* at = (const uint32_t*)(tile + d * pitch + lt);
    if (t >= g.a && t + 16 <= g.z)
      *(uint4*)to = make_uint4(at[0], at[1], at[2], at[3]);
    else
      for (int e = 0; e < 16; ++e)
        if (t + e >= g.a && t + e < g.z) to[e] = ((const uint8_t*)at)[e];
  }
}

// Many tokens: a workgroup takes a sequence's page and `heads` of its heads, one after the
// other.  A lane has one part of one token's key, whose angles it works out once for all
// heads, and one of its value; both stay in registers between the largest value and the codes,
// and the next head's are on their way meanwhile.  Two meetings a head: for the largest values,
// and where the values have been turned over.
// The angles lie in LDS, each read only by the lane that wrote it (in registers, of which 16 waves
// a CU have 128 each, 17 were spilled: 21 MB more written, 46 us where it then took 40).
// Bound by its steps' latencies in turn (copies without the angles, the turn, the keys' stores or
// the values' each took 30 to 33 of then 33 us; a vector instruction is issued in half of the
// time): 8 x 4096 tokens, 4 heads of 128 in bfloat16: 31.5 us, 66 MB read and written (2.1 TB/s).
// Workgroups from kv on turn `block` tokens' queries each.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void cache_page_kernel(Cache c, Sequences sq, Turn turn,
                                                                AppendRows<T> r, int groups,
                                                                int heads, int kv, int block) {
  extern __shared__ double2 lds[];
  if ((int)blockIdx.x >= kv) {
    append_queries<T, THREADS, false>(c, sq, turn, r, (int64_t)((int)blockIdx.x - kv) * block,
                                      block, (char*)lds);
    return;
  }
  constexpr int WAVES = THREADS / 64;
  __shared__ double2 angles[8][THREADS];
  AppendPage g(c, sq, blockIdx.x / groups);
  if (g.none()) return;
  const int NC = c.chunks, Dr = 16 * NC, pitch = c.page + 4;
  char* tile = (char*)lds;
  uint32_t* tops = (uint32_t*)(tile + pitch * Dr);
  const int key_parts = Part::of_key(turn.pairs, Dr), parts = key_parts > NC ? key_parts : NC;
  const int t = threadIdx.x / parts, part = threadIdx.x % parts;
  const bool in = t >= g.a && t < g.z, has_k = in && part < key_parts, has_v = in && part < NC;
  Part pk, pv;
  pk.key(part < key_parts ? part : 0, turn, r.D, Dr);
  pv.plain(16 * (part < NC ? part : 0), r.D, Dr);
  const int64_t row = g.row0 + t;
  const T *kr = r.k + row * r.k_row, *vr = r.v + row * r.v_row;
  PartValues<T> uk = {}, uv = {};
  const int h0 = (blockIdx.x % groups) * heads;
  const int h1 = h0 + heads < c.Hk ? h0 + heads : c.Hk;
  if (has_k) uk.load(kr + h0 * r.k_head, pk);
  if (has_v) uv.load(vr + h0 * r.v_head, pv);
  if (!g.there()) return;
  if (has_k && pk.pair >= 0) {
    double2 cs[8];
    part_angles(pk, turn, r, g, t, cs);
#pragma unroll
    for (int e = 0; e < 8; ++e) angles[e][threadIdx.x] = cs[e];
  }
#pragma unroll 1
  for (int h = h0; h < h1; ++h) {
    pk.fresh();
    pv.fresh();
    const int64_t scale_at = (int64_t)g.number * c.Hk + h;
    const bool older = g.a > 0;
    float old_k = older ? c.key_scales[scale_at] : 0.f;
    float old_v = older ? c.value_scales[scale_at] : 0.f;
    float x[16];
    bool rare_k = false, rare_v = false;
    uint32_t top_k = 0, top_v = 0;
    PartValues<T> v = uv;
    if (has_v) {
      float y[16];
      v.to(y);
      top_v = top16(y, rare_v);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (has_k) {
      if (pk.pair < 0)
        uk.to(x);
      else
        turn_part<T>(uk, turn.interleaved, [&](int e) { return angles[e][threadIdx.x]; }, x);
      top_k = top16(x, rare_k);
    }
    // Everything that was loaded is waited for here, and nothing that the rest of this head does:
    // a wait further down would be one for the next head's rows as well.
    asm volatile("" : "+v"(old_k), "+v"(old_v));
    v.fresh();
    if (h + 1 < h1) {
      if (has_k) uk.load(kr + (h + 1) * r.k_head, pk);
      if (has_v) uv.load(vr + (h + 1) * r.v_head, pv);
    }
    __builtin_amdgcn_sched_barrier(0);
    top_k = wave_top(top_k);
    top_v = wave_top(top_v);
    if (lane_id() == 0) {
      tops[wave_id()] = top_k;
      tops[WAVES + wave_id()] = top_v;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      top_k = tops[i] > top_k ? tops[i] : top_k;
      top_v = tops[WAVES + i] > top_v ? tops[WAVES + i] : top_v;
    }
    const int ek = page_exponent(top_k, older, old_k), ev = page_exponent(top_v, older, old_v);
    const float fk = power(-ek), fv = power(-ev);
    if (older && old_k != power(ek))
      scale_older<THREADS>(c, c.keys, g.number, h, true, g.a, old_k * fk, threadIdx.x);
    if (older && old_v != power(ev))
      scale_older<THREADS>(c, c.values, g.number, h, false, g.a, old_v * fv, threadIdx.x);
    uint32_t w[4];
    if (has_k) {
      codes16(x, fk, rare_k, pk.pair >= 0 && turn.interleaved, w);
      uint8_t* to = c.keys + c.block(g.number, h, t / 32);
      store_part(to, t % 32, pk.pa, pk.store_a, w[0], w[1]);
      store_part(to, t % 32, pk.pb, pk.store_b, w[2], w[3]);
    }
    if (has_v) {
      v.to(x);
      codes16(x, fv, rare_v, false, w);
      char* at = tile + part * 16 * pitch + t;
#pragma unroll
      for (int e = 0; e < 16; ++e) at[e * pitch] = (char)(w[e / 4] >> 8 * (e % 4));
    }
    __syncthreads();
    store_tile<THREADS>(c, tile, pitch, g, h, 0, c.page);
    if (threadIdx.x == 0) {  // (after both meetings: every wave has read the old ones)
      c.key_scales[scale_at] = power(ek);
      c.value_scales[scale_at] = power(ev);
    }
  }
}

// Few tokens a page, or pages that are more than a workgroup's lanes: workgroups 0 .. kv - 1 take a
// sequence's page and `heads` of its heads each, one team of TEAM lanes (a wave, or the
// workgroup) a head; keys, then values.  `round` tokens go through at a time; where a page is
// more than one round, it is loaded twice: for the largest value, then for the codes.  A wave
// writes a value's sixteen rows of a block itself, a byte each.
// Workgroups behind them turn `block` tokens' queries each.
template <typename T, int THREADS, int TEAM>
__global__ __launch_bounds__(THREADS, 2) void cache_append_kernel(Cache c, Sequences sq, Turn turn,
                                                                  AppendRows<T> r, int groups,
                                                                  int heads, int round, int kv,
                                                                  int block) {
  extern __shared__ double2 lds[];
  if ((int)blockIdx.x >= kv) {
    append_queries<T, THREADS, false>(c, sq, turn, r, (int64_t)((int)blockIdx.x - kv) * block,
                                      block, (char*)lds);
    return;
  }
  constexpr int TEAMS = THREADS / TEAM, WAVES = THREADS / 64;
  AppendPage g(c, sq, blockIdx.x / groups);
  if (g.none()) return;
  const int NC = c.chunks, Dr = 16 * NC, pitch = round + 4;
  char* tile = (char*)lds;
  uint32_t* tops = (uint32_t*)(tile + (TEAMS == 1 ? pitch * Dr : 0));
  const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
  const int key_parts = Part::of_key(turn.pairs, Dr), parts = key_parts > NC ? key_parts : NC;
  const int tok = lane / parts, part = lane % parts;
  // rounds begin at multiples of their length where the values' tile is turned over, so that a
  // round holds whole blocks
  const int r0 = TEAMS == 1 ? g.a / round * round : g.a;
  const int rounds = (g.z - r0 + round - 1) / round;
  auto in = [&](int t0) { return tok < round && t0 + tok >= g.a && t0 + tok < g.z; };
  Part pk, pv;
  pk.key(part < key_parts ? part : 0, turn, r.D, Dr);
  pv.plain(16 * (part < NC ? part : 0), r.D, Dr);
  double2 cs[8];
  // A round's angles.  Teams of a workgroup have the same tokens: each lane works out one angle
  // at a time for all of them, in LDS (a lane's eight one after the other are as much code to
  // fetch and as long a wait for the only tokens there are).
  auto angles = [&](int t0) {
    const bool turned = part < key_parts && pk.pair >= 0 && in(t0);
    if constexpr (TEAMS == 1) {
      if (turned) part_angles(pk, turn, r, g, t0 + tok, cs);
    } else {
      const int n = g.z - t0 < round ? g.z - t0 : round;
      __syncthreads();
#pragma unroll 1
      for (int i = threadIdx.x; i < n * turn.pairs; i += THREADS) {
        const int t = t0 + i / turn.pairs, j = i % turn.pairs;
        const double at = r.places ? turn.place(g.row0 + t, j) : (double)(g.base + t);
        double sn, co;
        sine_cosine(at * turn.f[j], sn, co);
        lds[i] = make_double2(co * turn.m, sn * turn.m);
      }
      __syncthreads();
      if (turned)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          cs[e] = lds[tok * turn.pairs + (pk.pair + e < turn.pairs ? pk.pair + e : pk.pair)];
    }
  };

  const int h0 = (blockIdx.x % groups) * heads;
  const int h1 = h0 + heads < c.Hk ? h0 + heads : c.Hk;
  // job 2 i: keys of the team's head i of these, job 2 i + 1: its values
  const int jobs = 2 * ((h1 - h0 + TEAMS - 1) / TEAMS);
  PartValues<T> u = {};
  auto load = [&](int job, int t0) {
    const int h = h0 + (job >> 1) * TEAMS + team;
    if (!in(t0) || h >= h1) return;
    const int64_t row = g.row0 + t0 + tok;
    if (job & 1) {
      if (part < NC) u.load(r.v + row * r.v_row + h * r.v_head, pv);
    } else if (part < key_parts) {
      u.load(r.k + row * r.k_row + h * r.k_head, pk);
    }
  };
  auto old_scale = [&](int job) {
    const int h = h0 + (job >> 1) * TEAMS + team;
    return g.a > 0 && h < h1
               ? (job & 1 ? c.value_scales : c.key_scales)[(int64_t)g.number * c.Hk + h]
               : 0.f;
  };
  load(0, r0);
  if (!g.there()) return;
  float next_old = old_scale(0);
  if (rounds == 1) angles(r0);
#pragma unroll 1
  for (int job = 0; job < jobs; ++job) {
    pk.fresh();
    pv.fresh();
    const bool key = !(job & 1);
    const int h = h0 + (job >> 1) * TEAMS + team;
    const bool mine = h < h1, has = mine && part < (key ? key_parts : NC);
    uint8_t* codes = key ? c.keys : c.values;
    const float old = next_old;
    if (job + 1 < jobs) next_old = old_scale(job + 1);
    uint32_t top = 0;
    float x[16], f = 0.f;
    bool rare = false;
    auto take = [&](int t0) {  // what was loaded as the cache takes it
      if (!(has && in(t0) && key && pk.pair >= 0))
        u.to(x);
      else
        turn_part<T>(u, turn.interleaved, [&](int e) { return cs[e]; }, x);
    };
    auto measure = [&](int t0) {
      if (!has || !in(t0)) return;
      const uint32_t y = top16(x, rare);
      top = y > top ? y : top;
    };
    auto settle = [&] {  // the page's scale; older codes brought to it
      top = wave_top(top);
      if (TEAMS == 1) {
        __syncthreads();
        if (lane_id() == 0) tops[wave_id()] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) top = tops[i] > top ? tops[i] : top;
      }
      const int e = page_exponent(top, g.a > 0, old);
      f = power(-e);
      if (g.a > 0 && mine && old != power(e))
        scale_older<TEAM>(c, codes, g.number, h, key, g.a, old * f, lane);
      if (mine && lane == 0)
        (key ? c.key_scales : c.value_scales)[(int64_t)g.number * c.Hk + h] = power(e);
    };
    auto store = [&](int t0) {
      if (has && in(t0)) {
        const int t = t0 + tok;
        uint32_t w[4];
        codes16(x, f, rare, key && pk.pair >= 0 && turn.interleaved, w);
        uint8_t* to = codes + c.block(g.number, h, t / 32);
        if (key) {
          store_part(to, t % 32, pk.pa, pk.store_a, w[0], w[1]);
          store_part(to, t % 32, pk.pb, pk.store_b, w[2], w[3]);
        } else if (TEAMS == 1) {
          char* at = tile + part * 16 * pitch + tok;
#pragma unroll
          for (int e = 0; e < 16; ++e) at[e * pitch] = (char)(w[e / 4] >> 8 * (e % 4));
        } else {
          to += part * 512 + t % 32;
#pragma unroll
          for (int e = 0; e < 16; ++e) to[e * 32] = (uint8_t)(w[e / 4] >> 8 * (e % 4));
        }
      }
      if (TEAMS == 1 && !key) {
        __syncthreads();
        store_tile<THREADS>(c, tile, pitch, g, h, t0, round);
        __syncthreads();
      }
    };
    if (rounds == 1) {
      take(r0);
      measure(r0);
      if (job + 1 < jobs) load(job + 1, r0);
      settle();
      store(r0);
    } else {
#pragma unroll 1
      for (int y = 0; y < 2 * rounds; ++y) {
        const int t0 = r0 + (y < rounds ? y : y - rounds) * round;
        load(job, t0);
        if (key) angles(t0);
        take(t0);
        measure(t0);
        if (y == rounds - 1) settle();
        if (y >= rounds) store(t0);
      }
    }
  }
}

int cache_check(const char* op, int64_t pages, int64_t Hk, int64_t page, int64_t Dr, int64_t B,
                int64_t M, int64_t D) {
  if (pages < 0 || pages >= ((int64_t)1 << 31) || Hk < 1 || Hk > 1024 || page < CACHE_BLOCK ||
      page > CACHE_PAGE || page % CACHE_BLOCK != 0 || D < 1 || D > CACHE_DMAX ||
      Dr != round_up(D, 16) || B < 0 || B > (1 << 24) || M < 0 ||
      M * page > ((int64_t)1 << 30) || M > ((int64_t)1 << 30))
    return set_error(TPO_ERR_ARG,
                     "%s: bad sizes pages=%lld Hk=%lld page=%lld Dr=%lld B=%lld M=%lld D=%lld "
                     "(pages of 32 to %d tokens in steps of 32, D at most %d and Dr the next "
                     "multiple of 16, M page at most 2^30)",
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

// Tokens that a team of `lanes` takes at a time; whole blocks for a workgroup's.
int append_round(const Cache& c, const Turn& t, int lanes, bool whole) {
  const int key_parts = Part::of_key(t.pairs, 16 * c.chunks);
  const int round = lanes / (key_parts > c.chunks ? key_parts : c.chunks);
  return round >= c.page ? c.page : (whole ? round / 32 * 32 : round);
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
  // few tokens a sequence: a wave a head, where pages are many (64 sequences, 8 heads of 128 in
  // bfloat16, a new token each 9.3 us, by whole workgroups 18.4; 8 new 10.3, 17.6; 16 new 25.3,
  // 18.1; 8 sequences: 9 and 8; 16 new 19.9, 8.5).  The rule knows the average only: 63 sequences
  // of one token and one of 400 take 66 us, in calls of their own 10 and 9.
  const bool few = T <= 8 * B;
  // else 512 workgroups (5 x 300 tokens, 6 heads of 80, float16: by 52 workgroups 32 us, 156 14,
  // 312 10; 8 x 4096, 4 heads of 128: 343 32, 686 31.5, 1372 38)
  const int64_t about = T / page + B + 1;  // pages
  int64_t groups = few ? (Hk + 3) / 4 : (512 + about - 1) / about;
  if (groups > Hk) groups = Hk;
  const int64_t heads = (Hk + groups - 1) / groups;
  groups = (Hk + heads - 1) / heads;
  // tokens' queries of a workgroup: as tpo_rotary's
  int64_t block = few || !q ? 1 : 16384 / (Hq * D * element_bytes(dtype));
  if (block > T / 2048) block = T / 2048;
  block = block > 16 ? 16 : (block < 1 ? 1 : block);
  const int64_t q_blocks = q ? (T + block - 1) / block : 0;
  if (slots * groups + q_blocks >= ((int64_t)1 << 23))
    return set_error(TPO_ERR_ARG, "%s: too many tokens", op);
  const int64_t q_pitch = dtype == TPO_F32 ? TurnAngles<float>(t.pairs, t.interleaved).pitch
                                           : TurnAngles<half_t>(t.pairs, t.interleaved).pitch;
  const int64_t q_lds = block * (q_pitch * sizeof(float2) + 2 * sizeof(int));
  const int kv = (int)(slots * groups);
  hipStream_t s = (hipStream_t)stream;
  with_element(dtype, [&](auto e) {
    typedef decltype(e) E;
    const AppendRows<E> r{(const E*)k, (const E*)v, (const E*)q, (E*)q_out, k_row, k_head, v_row,
                          v_head, q_row, q_head, (int)Hq, (int)D, places ? 1 : 0};
    const bool apart = !few && T * Hq * D * element_bytes(dtype) > TURN_STREAM;
    const unsigned blocks = (unsigned)(kv + (apart ? 0 : q_blocks));
    auto bytes = [&](int64_t n) { return (size_t)(n > q_lds ? n : q_lds); };
    auto pages_of = [&](auto threads) {
      constexpr int N = decltype(threads)::value;
      cache_page_kernel<E, N><<<blocks, N, bytes((page + 4) * Dr + 64), s>>>(
          c, sq, t, r, (int)groups, (int)heads, kv, (int)block);
    };
    if (few) {
      const int round = append_round(c, t, 64, false);
      cache_append_kernel<E, 256, 64>
          <<<blocks, 256, bytes((int64_t)round * pairs * sizeof(double2)), s>>>(
              c, sq, t, r, (int)groups, (int)heads, round, kv, (int)block);
    } else if (append_round(c, t, 256, true) >= page) {
      pages_of(std::integral_constant<int, 256>());
    } else if (append_round(c, t, 512, true) >= page) {
      pages_of(std::integral_constant<int, 512>());
    } else {
      const int round = append_round(c, t, 512, true);
      cache_append_kernel<E, 512, 512><<<blocks, 512, bytes((round + 4) * Dr + 64), s>>>(
          c, sq, t, r, (int)groups, (int)heads, round, kv, (int)block);
    }
    if (apart && q)
      cache_queries_kernel<E><<<dim3((unsigned)q_blocks), 256, (size_t)q_lds, s>>>(c, sq, t, r,
                                                                                   (int)block);
  });
  return check_launch(op);
}
