// cache_attention.hip -- softmax attention of new tokens over an 8-bit cache in pages.
//   S = scale q k^T (causal: row i of n sees place j where j <= i + length - n)
//   o = softmax(S) v; a row that sees no key is 0
// with k = 2^.. codes: the scales of a page and head never touch its codes.  A key's scale
// multiplies its score; a value's goes into the exponent, so that a key weighs
//   p = 2^(s + log2 vs - m)
// of which the products take the codes, and the row's sum p / vs; m follows the maximum of
// s + log2 vs.  Both cost one number a page and no instruction a value.
// Codes are exact in bfloat16 and float16: the products are those of the queries' type.  Float
// queries and probabilities are taken in three bfloat16 parts of 8 bits each, whose products
// with a code are exact: three products of a sixteenth of the float instruction's time.
#include "attention.hpp"
#include "cache.hpp"

namespace tpo {

typedef uint32_t u32x4 __attribute__((vector_size(16)));

struct CacheAttnArgs {
  Cache c;
  Sequences sq;
  int64_t q_row, q_head;
  int Hq, D, causal;
  float scale;
};

// The type of the products and the parts of a value in it.
template <typename T> struct CodeType { typedef T E; static constexpr int PARTS = 1; };
template <> struct CodeType<float> { typedef bf16_t E; static constexpr int PARTS = 3; };

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Eight codes as the matrix instructions take them.
template <typename E>
__device__ __forceinline__ typename Chunk<E>::V from_codes(uint32_t lo, uint32_t hi) {
  if constexpr (std::is_same_v<E, bf16_t>) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  } else {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
}
// Which of four codes are NaN: 0x80 in their bytes.
__device__ __forceinline__ uint32_t nan_codes(uint32_t x) {
  return ((x & 0x7f7f7f7f) + 0x01010101) & 0x80808080;
}

// A wave's 32 rows of q as the products take them, in PARTS parts: of values 32 s + 16 (l / 32) +
// 8 e .. + 7 (e = 0, 1; codes straight from memory), or ROWS: 16 s + 8 (l / 32) .. + 7 (from LDS).
template <typename T, int DP, bool ROWS = false>
struct CodeRows {
  typedef typename CodeType<T>::E E;
  typedef typename Chunk<E>::V V;
  static constexpr int PARTS = CodeType<T>::PARTS, N = DP / 16;
  V x[PARTS][N];
  __device__ __forceinline__ void load(const T* p, bool in, int D, bool negative) {
    const int h = lane_id() >> 5;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = ROWS ? 16 * i + 8 * h : 32 * (i / 2) + 16 * h + 8 * (i % 2);
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; e += 16 / sizeof(T)) {
        typename Chunk<T>::V u = {};
        if (in && d + e < D) u = *(const typename Chunk<T>::V*)(p + d + e);
#pragma unroll
        for (int j = 0; j < (int)(16 / sizeof(T)); ++j)
          y[e + j] = negative ? -(float)u[j] : (float)u[j];
      }
#pragma unroll
      for (int part = 0; part < PARTS; ++part)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const E z = (E)y[e];
          x[part][i][e] = z;
          y[e] -= (float)z;
        }
    }
  }
};

// 32 keys and values as they come from memory: a lane has 16 values of a key (place
// 16 h' + 4 a + b of the tile in row 8 a + 4 h' + b of the product, so that the scores that a
// lane receives are those of sixteen tokens in a row) and 16 tokens of a value.
template <int DP>
struct CodeTile {
  u32x4 k[DP / 32], v[DP / 32];
  // at: see BlockPlaces; STREAM: past the caches
  template <bool STREAM = false>
  __device__ __forceinline__ void load(const Cache& c, int64_t at) {
    constexpr int HOW = STREAM ? 2 : 0;
    const int l = lane_id(), r = l & 31, h = l >> 5;
    const int bytes = at < 0 ? 0 : 512 * c.chunks;
    const auto kr = buffer(c.keys + (at < 0 ? 0 : at), bytes);
    const auto vr = buffer(c.values + (at < 0 ? 0 : at), bytes);
    const int key = 16 * (r >> 2 & 1) + 4 * (r >> 3) + (r & 3);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
      k[i] = __builtin_amdgcn_raw_buffer_load_b128(kr, (2 * i + h) * 512 + key * 16, 0, HOW);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
      v[i] = __builtin_amdgcn_raw_buffer_load_b128(vr, 1024 * i + 32 * r + 16 * h, 0, HOW);
  }
};

// Where a wave's next 64 blocks are, a lane each: what follows from a block's number is worked
// out once for all of them.
// NARROW: also which blocks are small, see CodeSums::follow: those whose value's scale is less than
// 2^-HALF_LIFT of the largest so far (and no less than 2^-80, the most that cache_append's differ,
// nor than 2^-80 itself, where sums over them would leave float's range).
constexpr float HALF_LIFT = 7.f;
template <bool NARROW>
struct BlockPlaces {
  int lo, hi;    // bytes from the first block; hi < 0: the page is not there
  float ks, lv;  // the key's scale (small ones': less than 0), log2 of the value's
  float high = NEG_INF;  // the largest lv so far
  // (scales are positive numbers)
  static __device__ __forceinline__ float inside(float v) {
    return fminf(fmaxf(v, 0x1p-100f), 0x1p100f);
  }
  // blocks first, first + step, .. below end of sequence b
  __device__ __forceinline__ void load(const Cache& c, int b, int hk, int first, int step,
                                       int end) {
    const int t = first + lane_id() * step, per = c.page / CACHE_BLOCK;
    const int page = t < end ? c.page_of(b, t / per) : -1;
    const int64_t at = page < 0 ? -1 : c.block(page, hk, t % per);
    lo = (int)(uint32_t)at;
    hi = (int)(at >> 32);
    float vs = 0.f;
    ks = 1.f;
    if (page >= 0) {
      const int64_t at = (int64_t)page * c.Hk + hk;
      ks = inside(c.key_scales[at]);
      vs = inside(c.value_scales[at]);
    }
    // (what a page that is not there holds weighs nothing)
    lv = page < 0 ? NEG_INF : __builtin_amdgcn_logf(vs);
    if constexpr (NARROW) {
      high = fmaxf(high, wave_max(lv));
      if (lv < high - HALF_LIFT && lv >= fmaxf(high - 80.f, -80.f)) ks = -ks;
    }
  }
  __device__ __forceinline__ bool small(int i) const {
    return NARROW && __builtin_amdgcn_readlane(__builtin_bit_cast(int, ks), i & 63) < 0;
  }
  // of block i, the same in all lanes
  __device__ __forceinline__ int64_t place(int i) const {
    const uint32_t l = (uint32_t)__builtin_amdgcn_readlane(lo, i & 63);
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, i & 63) << 32 | l);
  }
  static __device__ __forceinline__ float lane(float v, int i) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i & 63));
  }
  // What a score of block i counts in the exponent of 2, count being that of a score of its
  // own; never 0, as a masked score is -inf.
  __device__ __forceinline__ float score(int i, float count) const {
    return fmaxf(count * fabsf(lane(ks, i)), 1e-37f);
  }
  __device__ __forceinline__ float value_log(int i) const { return lane(lv, i); }
};

// A wave's rows under way.
template <typename T, int DP>
struct CodeSums {
  typedef typename CodeType<T>::E E;
  static constexpr int PARTS = CodeType<T>::PARTS;
  static constexpr bool NARROW = std::is_same_v<E, half_t>;
  // Weights are 2^(s + lv - m), m being LIFT under the maximum and up to 8 more.  In half they go
  // up to 2^15 and end at 2^-25, which is 2^-32 of the maximum's; the other type has float's range.
  static constexpr float LIFT = NARROW ? HALF_LIFT : 0.f;
  f32x16 acc[DP / 32];
  float m, l;  // l: of the lane's own keys, half of the row's

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{};
    m = NEG_INF;
    l = 0.f;
  }
  // The keys j0 .. j0 + 31, of which the lane's row sees those below n (masked: not all rows
  // see all), the sequence has those below length; f: what a score counts in the exponent of
  // 2, with the keys' scale; small: see follow.
  __device__ __forceinline__ void add(CodeTile<DP>& t, const CodeRows<T, DP>& q, int j0, int n,
                                      bool masked, int length, float f, float lv, bool small) {
    f32x16 s = {};
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const auto x = from_codes<E>(t.k[i][2 * e], t.k[i][2 * e + 1]);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) mma(s, x, q.x[p][2 * i + e]);
      }
    if (__builtin_expect(masked, 0)) {
      const int first = j0 + 16 * (lane_id() >> 5);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (first + e >= n) s[e] = NEG_INF;
      mask_values(t, first, n, length);
      asm volatile("");  // (a branch: for every tile the masks' 70 instructions were a third)
    }
    float top = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
    top = __builtin_fmaf(top, f, lv);
    top = fmaxf(top, other_half(top));
    follow(top, lv, small);
    weigh(s, f, lv);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      typename Chunk<E>::V p[PARTS];
      parts(s, e, p);
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        const auto x = from_codes<E>(t.v[i][2 * e], t.v[i][2 * e + 1]);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) mma(acc[i], x, p[part]);
      }
    }
  }
  // The maximum follows where it grows by more than 2^8.  And in half it goes down where it has
  // to: the row's largest product of probability and value scale has set m, so that a page of
  // small values could have most of the probability and weights of nothing.  Where the weights'
  // last step, 2^(-25 - lv) in probability, is more than 2^-25 of the row's sum, m is set by the
  // tile's largest weight, unless no key of the tile has 2^-24 of the sum.  So a key's weight is
  // rounded by 2^-11 of itself and 2^-24 of the row's sum, whatever the scales; acc stays under
  // 2^120 by that.  (8 sequences of up to 8192 tokens, 1024 new, 16 heads on 4, D = 128 in float16:
  // 392 us, without it and LIFT 383; each is half of that.)
  // small: whether it may be so.  The key that set m is 2^LIFT in the sum over its scale, so the
  // scales have to be more than 2^LIFT apart, which those of values at common levels are not.
  __device__ __forceinline__ void follow(float top, float lv, bool small) {
    if (__builtin_amdgcn_ballot_w64(top - m > 8.f + LIFT) || small) {
      float m2 = fmaxf(m, top - LIFT);
      if (small) {
        const float own = __builtin_amdgcn_exp2f(-lv), row = l + other_half(l);
        if (own > row && __builtin_amdgcn_exp2f(top - m) * own > row * 0x1p-24f) m2 = top - LIFT;
      }
      const float a = m2 == NEG_INF ? 1.f : __builtin_amdgcn_exp2f(m - m2);
      m = m2;
      l *= a;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] *= a;
    }
  }
  // Scores to weights, and their part of the row's sum.
  __device__ __forceinline__ void weigh(f32x16& s, float f, float lv) {
    // (a row that has seen nothing: its scores are -inf, or of a page that is not there)
    const float b = m == NEG_INF ? NEG_INF : lv - m;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], f, b));
      sum += s[e];
    }
    l = __builtin_fmaf(sum, lv == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(-lv), l);
  }
  // Weights 8 e .. + 7 in the products' type.
  static __device__ __forceinline__ void parts(const f32x16& s, int e,
                                               typename Chunk<E>::V (&p)[PARTS]) {
#pragma unroll
    for (int y = 0; y < 8; ++y) {
      float r = s[8 * e + y];
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        const E z = (E)r;
        p[part][y] = z;
        r -= (float)z;
      }
    }
  }
  // Values of places behind the sequence become 0 (they may hold anything).  A NaN of a value
  // that some rows see and others do not is taken out and given to the rows that see it: 0
  // times it would reach the others.
  __device__ __forceinline__ void mask_values(CodeTile<DP>& t, int first, int n, int length) {
    uint32_t any = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int left = length - first - 4 * w;
      const uint32_t keep = left >= 4 ? ~0u : (left <= 0 ? 0u : (1u << 8 * left) - 1);
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        t.v[i][w] &= keep;
        any |= nan_codes(t.v[i][w]);
      }
    }
    if (!__builtin_amdgcn_ballot_w64(any != 0)) return;
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
      typename Chunk<E>::V sees;
#pragma unroll
      for (int y = 0; y < 8; ++y) sees[y] = (E)(first + 8 * e + y < n ? 1.f : 0.f);
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        typename Chunk<E>::V x;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t v = e ? t.v[i][2 + w] : t.v[i][w], bad = nan_codes(v);
          const uint32_t good = v & ~((bad >> 7) * 255u);
          if (e)
            t.v[i][2 + w] = good;
          else
            t.v[i][w] = good;
#pragma unroll
          for (int y = 0; y < 4; ++y) x[4 * w + y] = (E)((bad >> (8 * y + 7)) & 1 ? 1.f : 0.f);
        }
        f32x16 count = {};
        mma(count, x, sees);
#pragma unroll
        for (int y = 0; y < 16; ++y)
          if (count[y] > 0.f) acc[i][y] = __builtin_nanf("");
      }
    }
  }
};

// The keys that row r (token r / G) of a sequence's n rows sees.
__device__ __forceinline__ int cache_keys(int r, int G, int n, int length, int causal) {
  if (!causal) return length;
  const int k = r / G + length - n + 1;
  return k < 0 ? 0 : (k > length ? length : k);
}

// A wave's sums as another wave takes them, lane by lane: both have the same rows and columns.
template <typename T, int DP>
struct WaveSums {
  float4 acc[DP / 8][64];
  float m[64], l[64];

  __device__ __forceinline__ void put(const CodeSums<T, DP>& s) {
    const int l = lane_id();
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
      acc[i][l] = make_float4(s.acc[i / 4][4 * (i % 4)], s.acc[i / 4][4 * (i % 4) + 1],
                              s.acc[i / 4][4 * (i % 4) + 2], s.acc[i / 4][4 * (i % 4) + 3]);
    m[l] = s.m;
    this->l[l] = s.l;
  }
  // Adds them to s.  Rows that have seen nothing have m = -inf and sums of 0.
  __device__ __forceinline__ void add_to(CodeSums<T, DP>& s) const {
    const int l = lane_id();
    const float mo = m[l], top = fmaxf(s.m, mo);
    const float f = s.m == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(s.m - top);
    const float g = mo == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(mo - top);
    s.m = top;
    s.l = __builtin_fmaf(s.l, f, this->l[l] * g);
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) {
      const float4 o = acc[i][l];
      const float y[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = 4 * (i % 4) + e;
        s.acc[i / 4][at] = __builtin_fmaf(s.acc[i / 4][at], f, y[e] * g);
      }
    }
  }
};

// A workgroup takes 32 rows (tokens times the heads of a group, as the packed attention's) and
// one of gridDim.z shares of their keys, its W waves in turn a tile of 32 keys each.  A tile
// goes from memory to registers, the next ones are on their way while one is multiplied; LDS is
// used at the end only, where the waves' sums come together, two and two.
// part, ml: see attn_join_kernel; m is in the exponent of 2, the values' scales with it.
template <typename T, int DP, int W, bool STREAM>
__global__ __launch_bounds__(64 * W, (DP * sizeof(T) <= 256 ? 2 : 1)) void
cache_step_kernel(CacheAttnArgs a, const T* __restrict__ q, T* __restrict__ out,
                  float* __restrict__ part, float2* __restrict__ ml) {
  constexpr int N = 2;  // tiles in registers (three: no faster)
  __shared__ WaveSums<T, DP> lds[W / 2];
  const int G = a.Hq / a.c.Hk, hk = blockIdx.y, shares = gridDim.z;
  const CacheRows p = cache_rows(a.sq, a.c, blockIdx.x, [G](int64_t start, int s) {
    return start * G / 32 + s;
  });
  const int64_t past = blockIdx.x - p.place;
  if (past * 32 >= (int64_t)p.room * G) return;
  const int w = wave_id(), l = lane_id(), r0 = (int)past * 32, r = r0 + (l & 31);
  const int all = p.room * G, used = p.b < 0 ? 0 : p.used * G, length = p.b < 0 ? 0 : p.length;
  auto keys = [&](int row) {
    return used ? cache_keys(row < used ? row : used - 1, G, p.used, length, a.causal) : 0;
  };
  const int n = keys(r), least = keys(r0), most = r0 < used ? keys(r0 + 31) : 0;
  const int tiles = (most + 31) / 32, per = (tiles + shares - 1) / shares;
  const int t0 = per * blockIdx.z + w;
  const int t1 = per * (blockIdx.z + 1) < tiles ? per * (blockIdx.z + 1) : tiles;
  CodeSums<T, DP> rows;
  rows.clear();
  const float c = attn_count(a.scale);
  CodeRows<T, DP> x;
  const int mine = t0 < t1 ? (t1 - t0 + W - 1) / W : 0;  // the wave's tiles
  // the places of 64 of them at a time: of those that are loaded, and of those multiplied
  BlockPlaces<CodeSums<T, DP>::NARROW> ahead, now;
  if (mine > 0) ahead.load(a.c, p.b, hk, t0, W, t1);
  x.load(q + (p.first + r / G) * a.q_row + (hk * G + r % G) * a.q_head, r < used, a.D,
         a.scale < 0.f);
  CodeTile<DP> tile[N];
  auto load = [&](CodeTile<DP>& to, int i) {
    if (i >= mine) return;
    if (i > 0 && (i & 63) == 0) ahead.load(a.c, p.b, hk, t0 + i * W, W, t1);
    to.template load<STREAM>(a.c, ahead.place(i));
  };
#pragma unroll
  for (int y = 0; y < N - 1; ++y) load(tile[y], y);
  for (int i = 0; i < mine; i += N) {
#pragma unroll
    for (int y = 0; y < N; ++y) {
      const int at = i + y, j0 = (t0 + at * W) * CACHE_BLOCK;
      if (at >= mine) break;
      if ((at & 63) == 0) now = ahead;
      load(tile[(y + N - 1) % N], at + N - 1);
      rows.add(tile[y], x, j0, n, j0 + 32 > least, length, now.score(at, c), now.value_log(at),
               now.small(at));
    }
  }

#pragma unroll
  for (int half = W / 2; half > 0; half /= 2) {
    if (w >= half && w < 2 * half) lds[w - half].put(rows);
    __syncthreads();
    if (w < half) lds[w].add_to(rows);
    if (half > 1) __syncthreads();
  }
  if (w != 0 || r >= all) return;
  float total = rows.l + other_half(rows.l);
  if (r >= used) total = 0.f;
  const int64_t at = (p.first + r / G) * a.Hq + hk * G + r % G;
  const int64_t to = shares > 1 ? at * shares + blockIdx.z : at;
  const float inv = total == 0.f ? 0.f : shares > 1 ? 1.f : 1.f / total;
  if (shares == 1 || total != 0.f)
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) {
      const int d = 32 * (i / 4) + 8 * (i % 4) + 4 * (l >> 5);
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        y[e] = inv == 0.f ? 0.f : rows.acc[i / 4][4 * (i % 4) + e] * inv;
      if (d >= a.D) continue;  // (D is a multiple of four)
      if (shares > 1) {
        *(float4*)(part + to * a.D + d) = make_float4(y[0], y[1], y[2], y[3]);
      } else {
        Four<T> f;
#pragma unroll
        for (int e = 0; e < 4; ++e) f.v[e] = (T)y[e];
        *(Four<T>*)(out + to * a.D + d) = f;
      }
    }
  if (shares > 1 && l < 32) ml[to] = make_float2(rows.m, total);
}

// Prompts over a cache: a workgroup of four waves takes 128 rows, 32 a wave, and their keys in
// tiles of 64, which its waves load (a quarter each, two tiles ahead), turn into the products'
// type and put into LDS for all four: a code is converted once for 128 rows, where the kernel
// above does it for 32 (8 sequences of up to 8192, 1024 new tokens, 16 heads on 4, D = 128 in
// bfloat16: 386 us by itself, the kernel above 425; among other calls 359 to 388, as the clock
// goes).  Keys lie in LDS in the order of the product's rows in
// which a lane receives the scores of sixteen tokens in a row; values by value, 64 tokens each, so
// that sixteen bytes are what a product sums over.  Chunks of 16 bytes change places with the row,
// as in HeadLds, so that a read touches all banks.
template <typename T, int DP>
struct alignas(1024) CodeLds {
  typedef typename CodeType<T>::E E;
  static constexpr int PITCH = HeadLds<E, DP>::PITCH, KEYS_AT = 64 * PITCH;
  static constexpr int TILE = KEYS_AT + DP * 128, OUT = 4 * Rows32<T, DP>::BYTES;
  char b[2 * TILE > OUT ? 2 * TILE : OUT];
};

// A wave's quarter of a tile on its way: every other KB of one of its two blocks.
template <typename T, int DP>
struct CodeLoads {
  typedef typename CodeType<T>::E E;
  typedef CodeLds<T, DP> L;
  static constexpr int ALL = DP / 32, N = (ALL + 1) / 2;
  u32x4 k[N], v[N];
  int u, block;      // of the tile's blocks, every other KB from KB u on
  int kat[N][2];     // where a lane's two chunks of a key go, and of its value
  int vat[2], half;  // (half: which sixteen tokens of the value's)

  __device__ __forceinline__ explicit CodeLoads(int w) : u(w & 1), block(w >> 1) {
    const int l = lane_id(), token = l & 31;
    const int row = 32 * block + 8 * (token >> 2 & 3) + 4 * (token >> 4) + (token & 3);
    const int swap = HeadLds<E, DP>::swap(row), d = 32 * u + (l & 31), turn = d >> 1 & 7;
    half = l >> 5;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        kat[j][e] = row * L::PITCH + (((2 * (2 * (2 * j + u) + (l >> 5)) + e) ^ swap) << 4);
      vat[e] = L::KEYS_AT + d * 128 + (((4 * block + 2 * half + e) ^ turn) << 4);
    }
  }
  __device__ __forceinline__ void load(const Cache& c, int64_t at) {
    const int bytes = at < 0 ? 0 : 512 * c.chunks;
    const auto kr = buffer(c.keys + (at < 0 ? 0 : at), bytes);
    const auto vr = buffer(c.values + (at < 0 ? 0 : at), bytes);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (2 * j + u < ALL) {
        k[j] = __builtin_amdgcn_raw_buffer_load_b128(kr, lane_id() * 16, (2 * j + u) * 1024, 0);
        v[j] = __builtin_amdgcn_raw_buffer_load_b128(
            vr, 32 * (lane_id() & 31) + 16 * (lane_id() >> 5), (2 * j + u) * 1024, 0);
      }
  }
  // To the tile at lds; `left` places from its first are the sequence's.  masked: not all of
  // the workgroup's rows see all of the tile: values that are NaN become 0, and the result says
  // that there were some.
  __device__ __forceinline__ bool put(char* lds, int left, bool masked) {
    typedef typename Chunk<E>::V V;
    bool bad = false;
    if (__builtin_expect(masked, 0)) {
      uint32_t any = 0;
#pragma unroll
      for (int j = 0; j < N; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int n = left - 32 * block - 16 * half - 4 * w;
          const uint32_t x = v[j][w] & (n >= 4 ? ~0u : (n <= 0 ? 0u : (1u << 8 * n) - 1));
          const uint32_t nans = nan_codes(x);
          v[j][w] = x & ~((nans >> 7) * 255u);
          any |= 2 * j + u < ALL ? nans : 0;
        }
      bad = __builtin_amdgcn_ballot_w64(any != 0) != 0;
      asm volatile("");  // (a branch: worked out for every tile it took as long as the codes)
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (2 * j + u >= ALL) continue;
      *(V*)(lds + kat[j][0]) = from_codes<E>(k[j][0], k[j][1]);
      *(V*)(lds + kat[j][1]) = from_codes<E>(k[j][2], k[j][3]);
      *(V*)(lds + vat[0] + j * 64 * 128) = from_codes<E>(v[j][0], v[j][1]);
      *(V*)(lds + vat[1] + j * 64 * 128) = from_codes<E>(v[j][2], v[j][3]);
    }
    return bad;
  }
};

// The tiles' work of a wave.
template <typename T, int DP>
struct CodePrompt {
  typedef typename CodeType<T>::E E;
  typedef typename Chunk<E>::V V;
  typedef CodeLds<T, DP> L;
  static constexpr int PARTS = CodeType<T>::PARTS;
  CodeSums<T, DP> sums;
  HeadLanes<E, DP> lanes;
  int at[4];  // of values l % 32, tokens 8 y + 16 (l / 32) - 8 (y % 2) ..: chunk y of a lane's four

  __device__ __forceinline__ CodePrompt() {
    const int l = lane_id(), r = l & 31;
#pragma unroll
    for (int y = 0; y < 4; ++y)
      at[y] = L::KEYS_AT + r * 128 + (((4 * (y / 2) + 2 * (l >> 5) + y % 2) ^ (r >> 1 & 7)) << 4);
  }
  // values 32 i + l % 32, tokens 32 t + 16 (l / 32) + 8 e .. + 7 of the tile, y = 2 t + e
  __device__ __forceinline__ V value(const char* lds, int y, int i) const {
    return *(const V*)(lds + at[y] + 32 * 128 * i);
  }
  // Weights of the keys j0 .. j0 + 63 at lds, of which the lane's row sees those below n.  f, lv:
  // of the two blocks, see CodeSums.
  // small: see CodeSums::follow.
  __device__ __forceinline__ void weigh(f32x16 (&s)[2], const char* lds,
                                        const CodeRows<T, DP, true>& q, int j0, int n, bool masked,
                                        const float (&f)[2], const float (&lv)[2], bool small) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x16{};
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        const V x = lanes.by_row(lds + 32 * t * L::PITCH, c);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) mma(s[t], x, q.x[p][c]);
      }
    }
    if (__builtin_expect(masked, 0)) {
      const int first = j0 + 16 * (lane_id() >> 5);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (first + 32 * t + e >= n) s[t][e] = NEG_INF;
      asm volatile("");
    }
    float top = NEG_INF;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float y = s[t][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) y = fmaxf(y, s[t][e]);
      top = fmaxf(top, __builtin_fmaf(y, f[t], lv[t]));
    }
    sums.follow(fmaxf(top, other_half(top)), fmaxf(lv[0], lv[1]), small);
#pragma unroll
    for (int t = 0; t < 2; ++t) sums.weigh(s[t], f[t], lv[t]);
  }
  __device__ __forceinline__ void gather(const f32x16 (&s)[2], const char* lds) {
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      V p[PARTS];
      sums.parts(s[y / 2], y % 2, p);
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        const V x = value(lds, y, i);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) mma(sums.acc[i], x, p[part]);
      }
    }
  }
};

// Places in the order of falling lengths (up to 62 sequences: the long ones start first), 128 rows
// each; false: none.
__device__ __forceinline__ bool cache_prompt_rows(const CacheAttnArgs& a, int64_t place, int G,
                                                  CacheRows& p, int64_t& past) {
  const int B = a.sq.B;
  auto first = [G](int64_t start, int s) { return start * G / 128 + s; };
  if (B <= 62) {
    const int l = lane_id();
    const int i = l < 1 ? 0 : (l - 1 < B ? l - 1 : B), j = l < B ? l : B;
    const bool own = l >= 1 && l <= B;
    const int64_t o0 = a.sq.offsets[i], o1 = a.sq.offsets[j];
    const int64_t nn = own ? (a.sq.lengths ? a.sq.lengths[l - 1] : a.sq.T) : 0;
    const int64_t kept = own ? a.c.lengths[l - 1] : 0;
    const int T = (int)a.sq.T;
    auto inside = [](int64_t v, int most) { return v < 0 ? 0 : (v > most ? most : (int)v); };
    const int start = l < 1 ? 0 : (l > B + 1 ? T : inside(o0, T));
    const int next = l > B ? T : inside(o1, T);
    const int room = l < B + 2 && next > start ? next - start : 0;
    const int used = inside(nn, room), length = a.c.length(kept);
    const int c = (int)(((int64_t)room * G + 127) / 128);
    int before = 0;  // places of longer sequences
    for (int k = 0; k < B + 2; ++k) {
      const int n = __builtin_amdgcn_readlane(length, k), ck = __builtin_amdgcn_readlane(c, k);
      before += n > length || (n == length && k < l) ? ck : 0;
    }
    const uint64_t m = __builtin_amdgcn_ballot_w64(c > 0 && before <= place && place < before + c);
    if (!m) return false;
    const int s = __builtin_ctzll(m);
    p.first = __builtin_amdgcn_readlane(start, s);
    p.room = __builtin_amdgcn_readlane(room, s);
    p.used = __builtin_amdgcn_readlane(used, s);
    p.length = __builtin_amdgcn_readlane(length, s);
    p.b = s >= 1 && s <= B ? s - 1 : -1;
    past = place - __builtin_amdgcn_readlane(before, s);
    return true;
  }
  p = cache_rows(a.sq, a.c, place, first);
  past = place - p.place;
  return past * 128 < (int64_t)p.room * G;
}

// The codes of the next tile into a half of LDS, and this one's products from the other.
template <typename T, int DP>
__device__ __forceinline__ bool code_step(const char* __restrict__ cur, char* __restrict__ nxt,
                                          CodeLoads<T, DP>& raw, bool more, int left,
                                          bool next_masked, CodePrompt<T, DP>& rows,
                                          const CodeRows<T, DP, true>& q, bool any, int j0, int n,
                                          bool masked, const float (&f)[2], const float (&lv)[2],
                                          bool small) {
  const bool bad = more && raw.put(nxt, left, next_masked);
  if (any) {
    f32x16 s[2];
    if (__builtin_expect(small, 0)) {  // a block at a time, as if the other's page were not there
      const float one[2] = {lv[0], NEG_INF};
      rows.weigh(s, cur, q, j0, n, masked, f, one, true);
      rows.gather(s, cur);
    }
    const float rest[2] = {small ? NEG_INF : lv[0], lv[1]};
    rows.weigh(s, cur, q, j0, n, masked, f, rest, small);
    rows.gather(s, cur);
  }
  return bad;
}

template <typename T, int DP>
__global__ __launch_bounds__(256, (DP * sizeof(T) <= 256 ? 2 : 1)) void cache_prompt_kernel(
    CacheAttnArgs a, const T* __restrict__ q, T* __restrict__ out) {
  typedef CodeLds<T, DP> L;
  __shared__ L lds;
  __shared__ int taken_out;  // whether a value that some rows do not see was NaN
  if (threadIdx.x == 0) taken_out = 0;
  const int G = a.Hq / a.c.Hk, hk = blockIdx.x % a.c.Hk;
  CacheRows p;
  int64_t past;
  if (!cache_prompt_rows(a, blockIdx.x / a.c.Hk, G, p, past)) return;
  const int w = wave_id(), l = lane_id(), b0 = (int)past * 128, r0 = b0 + 32 * w;
  const int r = r0 + (l & 31);
  const int all = p.room * G, used = p.b < 0 ? 0 : p.used * G, length = p.b < 0 ? 0 : p.length;
  auto keys = [&](int row) {
    return used ? cache_keys(row < used ? row : used - 1, G, p.used, length, a.causal) : 0;
  };
  const int n = keys(r), least = keys(r0), most = r0 < used ? keys(r0 + 31) : 0;
  const int all_see = keys(b0), end = b0 < used ? keys(b0 + 127) : 0, tiles = (end + 63) / 64;
  // (the last tile's second block may be behind the sequence's pages)
  const int blocks = (end + CACHE_BLOCK - 1) / CACHE_BLOCK;
  // 64 blocks' pages at a time: of the tiles that are loaded, and of those that are multiplied
  BlockPlaces<CodeSums<T, DP>::NARROW> ahead, now;
  if (tiles > 0) ahead.load(a.c, p.b, hk, 0, 1, blocks);
  CodeRows<T, DP, true> x;
  x.load(q + (p.first + r / G) * a.q_row + (hk * G + r % G) * a.q_head, r < used, a.D,
         a.scale < 0.f);
  const float c = attn_count(a.scale);
  CodePrompt<T, DP> rows;
  rows.sums.clear();
  CodeLoads<T, DP> raw(w);
  auto load = [&](int t) { raw.load(a.c, ahead.place(2 * t + raw.block)); };
  bool bad = false;
  if (tiles > 0) {
    load(0);
    bad = raw.put(lds.b, length, 64 > all_see);
    if (tiles > 1) load(1);
  }
  auto step = [&](auto half, int t) {  // (the halves by name: LDS addresses are constants)
    constexpr int H = decltype(half)::value;
    __syncthreads();  // tile t is there; the other half of LDS is free
    if ((t & 31) == 0) now = ahead;
    float f[2], lv[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      f[y] = now.score(2 * t + y, c);
      lv[y] = now.value_log(2 * t + y);
    }
    const bool small = now.small(2 * t) || now.small(2 * t + 1);
    bad |= code_step<T, DP>(lds.b + H * L::TILE, lds.b + (1 - H) * L::TILE, raw, t + 1 < tiles,
                            length - 64 * (t + 1), 64 * t + 128 > all_see, rows, x, 64 * t < most,
                            64 * t, n, 64 * t + 64 > least, f, lv, small);
    if (t + 2 < tiles) {
      if (((t + 2) & 31) == 0) ahead.load(a.c, p.b, hk, 2 * (t + 2), 1, blocks);
      load(t + 2);
    }
  };
  for (int t = 0; t < tiles; t += 2) {
    step(std::integral_constant<int, 0>(), t);
    if (t + 1 < tiles) step(std::integral_constant<int, 1>(), t + 1);
  }
  if (bad) taken_out = 1;
  __syncthreads();
  if (r0 >= all) return;
  if (taken_out) {  // rare: the rows that see it get it, see CodeSums
    for (int i = all_see / 64 * 2; i < blocks; ++i) {
      const int per = a.c.page / CACHE_BLOCK;
      const int page = __builtin_amdgcn_readfirstlane(a.c.page_of(p.b, i / per));
      if (page < 0) continue;
      CodeTile<DP> tile;
      tile.load(a.c, uniform(a.c.block(page, hk, i % per)));
      rows.sums.mask_values(tile, 32 * i + 16 * (l >> 5), n, length);
    }
  }
  const float total = rows.sums.l + other_half(rows.sums.l);
  const float inv = r < used && total != 0.f ? 1.f / total : 0.f;
  AttnArgs at;
  at.Hq = a.Hq;
  at.Hk = a.c.Hk;
  at.D = a.D;
  AttnSpan span;
  span.q0 = p.first;
  put_rows<T, DP>(lds.b, rows.sums.acc, inv, out, at, span, hk, r0, all);
}

// Which kernel a call takes, how many workgroups share the keys of 32 rows, and whether the
// codes go past the caches.
// Prompts by 128 rows convert a code once for all of them, which pays where heads are wide and
// two workgroups are there for every CU (half types, D = 128, 8 sequences of up to 8192 tokens:
// 1024 such workgroups 386 us, by 32 rows 425; 512: 212, 236; 256: 55, 47; 256 of 16384 keys: 376,
// 308).  Heads of 64 gain nothing by it (246, 248), float, whose products take three times as
// long, loses (205, 181).
// Shares: for 128 workgroups in all where that leaves a share 256 keys; for long caches up to
// 1024 workgroups, so that sequences of different lengths even out (64 x 16384 tokens, 4 heads:
// one share each 185 us, 2 160, 4 141).
// Past the caches: where a row tile is all that reads them in a call, and the next call finds
// nothing left of a pool that is more than the 256 MB behind the L2s (the same case 141 us, past
// them 129; 3 x 1500 tokens read by seven row tiles each 17.4, past them 19.1).
// Waves: eight where a CU gets no more than one workgroup and each of four would have five tiles
// or more (3 x 1500 tokens, 8 heads of 96, 200 new, float16: 15.6 us, by four waves 16.4; 7
// sequences, 6 heads of 40, 5 new, float, with the join: 4096 tokens 15.4, 15.8; 2048 12.4, 12.1;
// 1 x 300, 8 heads of 64: 8.0, 7.5).
// All this goes by the average of a call's rows and by the table's room, as the lengths are on the
// GPU.  What it costs where they mislead: 63 single tokens over 16384 and a piece of 1024 rows,
// groups of 4 in bfloat16: 189 us on 4 heads (apart 120 and 43), 435 on 8 (232 and 32); 1 x 300 as
// above with room for 320 tokens 8.1, 4096 11.6, 32768 12.8; 16 x 1000, 8 heads of 64 in float16,
// in a pool of 131 MB 10.7, of 2.6 GB 11.3.
struct CacheWay {
  bool prompt, stream;
  int shares, waves;
};
CacheWay cache_way(int dtype, int64_t B, int64_t T, int64_t room, int64_t Hq, int64_t Hk,
                   int64_t D, int64_t bytes) {
  const int64_t G = Hq / Hk, n = B < 1 ? 1 : B;
  const int64_t each = T < 1 ? 1 : (T * G + n - 1) / n;
  if (dtype != TPO_F32 && D > 64 && each > 32 && (each + 127) / 128 * n * Hk >= 512)
    return CacheWay{true, false, 1, 4};
  const int64_t blocks = (each + 31) / 32 * n * Hk;
  int64_t s = (128 + blocks - 1) / blocks, t = 1024 / blocks;
  if (s > room / 256) s = room / 256;
  if (t > room / 1024) t = room / 1024;
  if (s < t) s = t;
  if (room < 1024 || s < 1) s = 1;
  if (s > 64) s = 64;
  const bool eight =
      D * element_bytes(dtype) <= 256 && blocks * s <= 256 && room >= 20 * CACHE_BLOCK * s;
  return CacheWay{false, each <= 32 && bytes > (int64_t)256 << 20, (int)s, eight ? 8 : 4};
}

int cache_attn_check(const char* op, int dtype, int64_t B, int64_t T, int64_t Hq, int64_t Hk,
                     int64_t D, int64_t pages, int64_t page, int64_t Dr, int64_t M) {
  if (dtype != TPO_F32 && dtype != TPO_F16 && dtype != TPO_BF16)
    return set_error(TPO_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (int rc = cache_check(op, pages, Hk, page, Dr, B, M, D)) return rc;
  if (T < 0 || T >= ((int64_t)1 << 31) || Hq < 1 || Hq > 1024 || Hq % Hk != 0 ||
      T * Hq >= ((int64_t)1 << 31))
    return set_error(TPO_ERR_ARG,
                     "%s: bad sizes T=%lld Hq=%lld Hk=%lld (Hq a multiple of Hk, at most 1024)", op,
                     (long long)T, (long long)Hq, (long long)Hk);
  return TPO_OK;
}

}  // namespace tpo

using namespace tpo;

extern "C" int64_t tpo_cache_attention_workspace_size(int dtype, int64_t B, int64_t T, int64_t Hq,
                                                      int64_t Hk, int64_t D, int64_t page,
                                                      int64_t M) {
  const int64_t Dr = round_up(D, 16);
  if (cache_attn_check("cache_attention_workspace_size", dtype, B, T, Hq, Hk, D, 0, page, Dr, M))
    return -1;
  const int64_t s = cache_way(dtype, B, T, M * page, Hq, Hk, D, 0).shares;
  if (s == 1) return 0;
  return round_up(T * Hq * s * D * 4, 256) + round_up(T * Hq * s * 8, 256);
}

extern "C" int tpo_cache_attention_rows(int dtype, int64_t B, int64_t T, int64_t Hq, int64_t Hk,
                                        int64_t D, int64_t page, int64_t M) {
  if (int rc = cache_attn_check("cache_attention_rows", dtype, B, T, Hq, Hk, D, 0, page,
                                round_up(D, 16), M))
    return rc;
  return cache_way(dtype, B, T, M * page, Hq, Hk, D, 0).prompt ? 128 : 32;
}

extern "C" int tpo_cache_attention(int dtype, const void* q, const int64_t* offsets,
                                   const int64_t* lengths_q, int64_t B, int64_t T, int64_t Hq,
                                   int64_t D, int64_t q_row, int64_t q_head, const void* keys,
                                   const void* values, const float* key_scales,
                                   const float* value_scales, const int32_t* table,
                                   const int64_t* lengths, int64_t pages, int64_t Hk, int64_t page,
                                   int64_t Dr, int64_t M, int causal, double scale, void* out,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  const char* op = "cache_attention";
  if (int rc = cache_attn_check(op, dtype, B, T, Hq, Hk, D, pages, page, Dr, M)) return rc;
  if (T == 0) return TPO_OK;
  if (int rc = all_there(op, {q, offsets, out})) return rc;
  if (B > 0)
    if (int rc = all_there(op, {lengths})) return rc;
  if (B > 0 && M > 0)
    if (int rc = all_there(op, {table})) return rc;
  if (pages > 0)
    if (int rc = all_there(op, {keys, values, key_scales, value_scales})) return rc;
  if (int rc = attn_layout(op, dtype, D, {q, keys, values, workspace}, {q_row, q_head}, {q_row}))
    return rc;
  const int64_t need =
      tpo_cache_attention_workspace_size(dtype, B, T, Hq, Hk, D, page, M);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(TPO_ERR_WORKSPACE, "%s: workspace of %lld bytes needed", op, (long long)need);
  CacheAttnArgs a;
  a.c = cache_args(keys, values, key_scales, value_scales, table, lengths, pages, Hk, page, D, M);
  a.sq = Sequences{offsets, lengths_q, T, (int)B};
  a.q_row = q_row;
  a.q_head = q_head;
  a.Hq = (int)Hq;
  a.D = (int)D;
  a.causal = causal ? 1 : 0;
  a.scale = (float)scale;
  const CacheWay way = cache_way(dtype, B, T, M * page, Hq, Hk, D, 2 * pages * Hk * page * Dr);
  const int shares = way.shares;
  const int64_t G = Hq / Hk, places = attn_places(T, G, B, way.prompt ? 128 : 32);
  if ((way.prompt ? places * Hk : places) >= AT_GRID)
    return set_error(TPO_ERR_ARG, "%s: too many rows", op);
  hipStream_t s = (hipStream_t)stream;
  float* part = (float*)workspace;
  float2* ml = (float2*)((char*)workspace + round_up(T * Hq * shares * D * 4, 256));
  with_element(dtype, [&](auto t) {
    typedef decltype(t) E;
    with_head(D, [&](auto dp) {
      constexpr int DP = decltype(dp)::value;
      if constexpr (sizeof(E) == 2 && DP > 64)
        if (way.prompt) {
          cache_prompt_kernel<E, DP>
              <<<dim3((unsigned)(places * Hk)), 256, 0, s>>>(a, (const E*)q, (E*)out);
          return;
        }
      auto step = [&](auto waves, auto stream) {
        constexpr int W = decltype(waves)::value;
        cache_step_kernel<E, DP, W, decltype(stream)::value>
            <<<dim3((unsigned)places, (unsigned)Hk, shares), 64 * W, 0, s>>>(
                a, (const E*)q, (E*)out, part, ml);
      };
      const std::integral_constant<int, 4> four;
      if constexpr (DP * sizeof(E) <= 256)
        if (way.waves == 8) {
          const std::integral_constant<int, 8> eight;
          way.stream ? step(eight, std::true_type()) : step(eight, std::false_type());
          return;
        }
      way.stream ? step(four, std::true_type()) : step(four, std::false_type());
    });
    if (shares > 1)
      attn_join_kernel<E><<<dim3((unsigned)(T * Hq)), 256, 0, s>>>(
          part, ml, shares, (int)Hq, T, (int)D, (E*)out, nullptr, nullptr);
  });
  return check_launch(op);
}
