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

// A wave's 32 rows of q as the products take them: of values 32 s + 16 (l / 32) + 8 e .. + 7
// (e = 0, 1), in PARTS parts.
template <typename T, int DP>
struct CodeRows {
  typedef typename CodeType<T>::E E;
  typedef typename Chunk<E>::V V;
  static constexpr int PARTS = CodeType<T>::PARTS, N = DP / 16;
  V x[PARTS][N];
  __device__ __forceinline__ void load(const T* p, bool in, int D, bool negative) {
    const int h = lane_id() >> 5;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = 32 * (i / 2) + 16 * h + 8 * (i % 2);
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
  __device__ __forceinline__ void load(const Cache& c, int64_t at, bool there) {
    const int l = lane_id(), r = l & 31, h = l >> 5;
    const int bytes = there ? 512 * c.chunks : 0;
    const auto kr = buffer(c.keys + at, bytes), vr = buffer(c.values + at, bytes);
    const int key = 16 * (r >> 2 & 1) + 4 * (r >> 3) + (r & 3);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
      k[i] = __builtin_amdgcn_raw_buffer_load_b128(kr, (2 * i + h) * 512 + key * 16, 0, 0);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
      v[i] = __builtin_amdgcn_raw_buffer_load_b128(vr, 1024 * i + 32 * r + 16 * h, 0, 0);
  }
};

// The pages of a wave's next 64 tiles, a lane each.
struct TilePages {
  int page;      // -1: none
  float ks, lv;  // the key's scale, log2 of the value's
  // tiles first, first + step, .. below end of sequence b
  __device__ __forceinline__ void load(const Cache& c, int b, int hk, int first, int step,
                                       int end) {
    const int t = first + lane_id() * step;
    page = t < end ? c.page_of(b, t * CACHE_BLOCK / c.page) : -1;
    float vs = 0.f;
    ks = 1.f;
    if (page >= 0) {
      const int64_t at = (int64_t)page * c.Hk + hk;
      ks = c.key_scales[at];
      vs = c.value_scales[at];
    }
    // (what a page that is not there holds weighs nothing; scales are positive numbers)
    lv = page < 0 ? NEG_INF : __builtin_amdgcn_logf(fminf(fmaxf(vs, 0x1p-100f), 0x1p100f));
  }
};

// A wave's rows under way.
template <typename T, int DP>
struct CodeSums {
  typedef typename CodeType<T>::E E;
  static constexpr int PARTS = CodeType<T>::PARTS;
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
  // 2, with the keys' scale.
  __device__ __forceinline__ void add(CodeTile<DP>& t, const CodeRows<T, DP>& q, int j0, int n,
                                      bool masked, int length, float f, float lv) {
    f32x16 s = {};
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const auto x = from_codes<E>(t.k[i][2 * e], t.k[i][2 * e + 1]);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) mma(s, x, q.x[p][2 * i + e]);
      }
    const int first = j0 + 16 * (lane_id() >> 5);
    if (masked) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (first + e >= n) s[e] = NEG_INF;
      mask_values(t, first, n, length);
    }
    float top = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
    top = __builtin_fmaf(top, f, lv);
    top = fmaxf(top, other_half(top));
    if (__builtin_amdgcn_ballot_w64(top - m > 8.f)) {
      const float m2 = fmaxf(m, top);
      const float a = m2 == NEG_INF ? 1.f : __builtin_amdgcn_exp2f(m - m2);
      m = m2;
      l *= a;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] *= a;
    }
    const float b = m == NEG_INF ? 0.f : lv - m;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], f, b));
      sum += s[e];
    }
    l = __builtin_fmaf(sum, lv == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(-lv), l);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      typename Chunk<E>::V p[PARTS];
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
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        const auto x = from_codes<E>(t.v[i][2 * e], t.v[i][2 * e + 1]);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) mma(acc[i], x, p[part]);
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

// A workgroup takes 32 rows (tokens times the heads of a group, as the packed attention's) and
// one of gridDim.z shares of their keys, its four waves in turn a tile of 32 keys each.  A tile
// goes from memory to registers, the next one is on its way while one is multiplied; LDS is
// used at the end only, where the waves' sums come together.
// part, ml: see attn_step_kernel; m is in the exponent of 2, the values' scales with it.
constexpr int CODE_WAVES = 4;
template <typename T, int DP>
__global__ __launch_bounds__(64 * CODE_WAVES, (DP * sizeof(T) <= 256 ? 2 : 1)) void
cache_step_kernel(CacheAttnArgs a, const T* __restrict__ q, T* __restrict__ out,
                  float* __restrict__ part, float2* __restrict__ ml) {
  constexpr int W = CODE_WAVES, P = DP + 4;
  __shared__ float sums[W * 32 * P], ms[W][32], ls[W][32];
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
  TilePages pages;
  if (t0 < t1) pages.load(a.c, p.b, hk, t0, W, t1);
  x.load(q + (p.first + r / G) * a.q_row + (hk * G + r % G) * a.q_head, r < used, a.D,
         a.scale < 0.f);
  auto load = [&](CodeTile<DP>& tile, int i) {  // the wave's tile i of those that `pages` has
    const int t = t0 + i * W, page = __builtin_amdgcn_readlane(pages.page, i & 63);
    const int64_t at =
        page < 0 ? 0 : a.c.block(page, hk, t % (a.c.page / CACHE_BLOCK));
    tile.load(a.c, uniform(at), page >= 0);
  };
  auto add = [&](CodeTile<DP>& tile, int i) {
    const int j0 = (t0 + i * W) * CACHE_BLOCK;
    const float ks = __builtin_bit_cast(
        float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, pages.ks), i & 63));
    const float lv = __builtin_bit_cast(
        float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, pages.lv), i & 63));
    rows.add(tile, x, j0, n, j0 + 32 > least, length, c * ks, lv);
  };
  const int mine = t0 < t1 ? (t1 - t0 + W - 1) / W : 0;  // the wave's tiles
  CodeTile<DP> one, two;
  for (int i = 0; i < mine; i += 2) {
    if ((i & 63) == 0) {
      if (i > 0) pages.load(a.c, p.b, hk, t0 + i * W, W, t1);
      load(one, i);
    }
    if (i + 1 < mine) load(two, i + 1);
    add(one, i);
    if (i + 1 < mine) {
      if (i + 2 < mine && ((i + 2) & 63) != 0) load(one, i + 2);
      add(two, i + 1);
    }
  }

  // the waves' sums together
  const float sum = rows.l + other_half(rows.l);
  float* mysums = sums + w * 32 * P;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      Four<float> f;
#pragma unroll
      for (int e = 0; e < 4; ++e) f.v[e] = rows.acc[i][4 * b + e];
      *(Four<float>*)(mysums + (l & 31) * P + 32 * i + 8 * b + 4 * (l >> 5)) = f;
    }
  if (l < 32) {
    ms[w][l] = rows.m;
    ls[w][l] = sum;
  }
  __syncthreads();
  constexpr int PER_ROW = 2 * W, D1 = DP / PER_ROW;  // lanes a row, values a lane
  const int rr = threadIdx.x / PER_ROW, d0 = threadIdx.x % PER_ROW * D1, row = r0 + rr;
  if (row >= all) return;
  float m = NEG_INF, total = 0.f, f[W];
#pragma unroll
  for (int i = 0; i < W; ++i) m = fmaxf(m, ms[i][rr]);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float y = ls[i][rr];
    f[i] = y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ms[i][rr] - m);
    total += f[i] * y;
  }
  if (row >= used) total = 0.f;
  const int64_t at = (p.first + row / G) * a.Hq + hk * G + row % G;
  const float inv = shares > 1 ? 1.f : total != 0.f ? 1.f / total : 0.f;
#pragma unroll
  for (int d = 0; d < D1; ++d) {
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (f[i] != 0.f) y += f[i] * sums[(i * 32 + rr) * P + d0 + d];
    if (d0 + d < a.D) {
      if (shares > 1) {
        if (total != 0.f) part[(at * shares + blockIdx.z) * a.D + d0 + d] = y;
      } else {
        out[at * a.D + d0 + d] = total == 0.f ? (T)0.f : (T)(y * inv);
      }
    }
  }
  if (d0 == 0 && shares > 1) ml[at * shares + blockIdx.z] = make_float2(m, total);
}

// How many workgroups share the keys of 32 rows.
int cache_shares(int64_t B, int64_t T, int64_t room, int64_t Hq, int64_t Hk) {
  const int64_t G = Hq / Hk, n = B < 1 ? 1 : B;
  const int64_t each = T < 1 ? 1 : (T * G + n - 1) / n;
  const int64_t blocks = (each + 31) / 32 * n * Hk;
  int64_t s = (128 + blocks - 1) / blocks, t = 1024 / blocks;
  if (s > room / 256) s = room / 256;
  if (t > room / 1024) t = room / 1024;
  if (s < t) s = t;
  if (room < 1024 || s < 1) s = 1;
  return s > 64 ? 64 : (int)s;
}

int cache_attn_check(const char* op, int dtype, int64_t B, int64_t T, int64_t Hq, int64_t Hk,
                     int64_t D, int64_t pages, int64_t page, int64_t Dr, int64_t M) {
  if (dtype != TPO_F32 && dtype != TPO_F16 && dtype != TPO_BF16)
    return set_error(TPO_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (int rc = cache_check(op, pages, Hk, page, Dr, B, M, D)) return rc;
  if (T < 0 || Hq < 1 || Hq > 1024 || Hq % Hk != 0 || T * Hq >= ((int64_t)1 << 31))
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
  const int64_t s = cache_shares(B, T, M * page, Hq, Hk);
  if (s == 1) return 0;
  return round_up(T * Hq * s * D * 4, 256) + round_up(T * Hq * s * 8, 256);
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
  const int64_t G = Hq / Hk, places = attn_places(T, G, B, 32);
  if (places >= AT_GRID) return set_error(TPO_ERR_ARG, "%s: too many rows", op);
  const int shares = cache_shares(B, T, M * page, Hq, Hk);
  hipStream_t s = (hipStream_t)stream;
  float* part = (float*)workspace;
  float2* ml = (float2*)((char*)workspace + round_up(T * Hq * shares * D * 4, 256));
  with_element(dtype, [&](auto t) {
    typedef decltype(t) E;
    with_head(D, [&](auto dp) {
      constexpr int DP = decltype(dp)::value;
      cache_step_kernel<E, DP>
          <<<dim3((unsigned)places, (unsigned)Hk, shares), 64 * CODE_WAVES, 0, s>>>(
              a, (const E*)q, (E*)out, part, ml);
    });
    if (shares > 1)
      attn_join_kernel<E><<<dim3((unsigned)(T * Hq)), 256, 0, s>>>(
          part, ml, shares, (int)Hq, T, (int)D, (E*)out, nullptr, nullptr);
  });
  return check_launch(op);
}
