// attention_bwd.hip -- backward of softmax attention over packed sequences.
//   dV = P^T dO, dP = dO V^T, dS = P (dP - sum_d dO O),
//   dQ = scale dS K, dK = scale dS^T Q
// P comes from the scores again and the forward's logarithms of the rows' sums.
// Two kernels, so that every sum has one owner and a fixed order: one holds rows
// and passes over their keys (dQ), one holds keys and passes over the rows that
// see them (dK, dV).  The scores and dP are computed in both: 7 products where 5
// with atomic sums for dQ would do, but the results are the same on every run.
// A row that sees a single key has dS = 0 (its probability is 1 whatever the
// score): dP and delta, which are sums in different orders, would leave their
// rounding there, so it is said outright.
// Half types: P and dS are rounded to the type for the products that take them.
// The first kernel also makes, of each row, what is subtracted in the exponent of 2
// (the logarithm of its sum; infinity where the row sees no key, which makes its P
// 0) and delta = sum_d dO O, and leaves them to the second one.
#include "attention.hpp"

namespace tpo {

// Two tiles of 64 rows, twice over; later what waves exchange, and the rows on
// their way out.
constexpr int BWD_ROWS = 64;
template <typename T, int DP>
struct alignas(1024) BwdRowsLds {
  static constexpr int TILE = BWD_ROWS * HeadLds<T, DP>::PITCH;
  static constexpr int OUT = 4 * Rows32<T, DP>::BYTES;
  char b[4 * TILE > OUT ? 4 * TILE : OUT];
};

template <typename T, int DP>
__device__ __forceinline__ void bwd_q_load(char* to, const T* k, const T* v, const AttnArgs& a,
                                           int left) {
  typedef HeadLds<T, DP> L;
  const int w = wave_id();
  L::template load<BWD_ROWS, 4>(to, k, (int)(a.k_row * sizeof(T)), left, a.D, w);
  L::template load<BWD_ROWS, 4>(to + BwdRowsLds<T, DP>::TILE, v, (int)(a.v_row * sizeof(T)), left,
                                a.D, w);
}

// The products of the wave's rows with 32 keys from j0 on, `half` of a tile.
template <typename T, int DP>
__device__ __forceinline__ void bwd_q_step(const char* __restrict__ cur, char* __restrict__ nxt,
                                           const HeadLanes<T, DP>& lanes, const T* k, const T* v,
                                           const AttnArgs& a, int left, const HeadRows<T, DP>& q,
                                           const HeadRows<T, DP>& go, f32x16 (&acc)[DP / 32],
                                           int half, int j0, int n, int least, int most, float c,
                                           float sub, float delta) {
  bwd_q_load<T, DP>(nxt, k, v, a, left);
  __builtin_amdgcn_sched_barrier(0);
  if (j0 >= most) return;
  const char* at = cur + half * 32 * HeadLds<T, DP>::PITCH;
  f32x16 s = scores<T, DP>(lanes, at, q, a.D);
  const f32x16 d = scores<T, DP>(lanes, at + BwdRowsLds<T, DP>::TILE, go, a.D);
  const int first = j0 + 4 * (lane_id() >> 5);
#pragma unroll
  for (int e = 0; e < 16; ++e)
    s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -sub)) * (d[e] - delta);
  if (j0 + 32 > least)  // (a pass of its own: a select for each value would be taken everywhere)
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (first + 8 * (e >> 2) + (e & 3) >= n) s[e] = 0.f;
  multiply_rows<T, DP>(acc, lanes, at, s);
}

// dQ of 64 rows; the rows and their keys as the forward for prompts has them.
// Wave w has rows 32 (w % 2) .. + 31 and half w / 2 of each tile of keys; at the
// end two waves' sums are added.  rest: what rounding took from O.  Without it the
// rounding of O, which is common to all keys of a row, would add to dQ's error about
// half of what the rounding of dS does.  (delta by a kernel of its own, which reads dO
// once more, took 18 us of 234 for 8 x 2048; so they are 226.)  gq null: only what dK
// and dV need of the rows, sub and delta; sub null: only dQ.
template <typename T, int DP>
__global__ __launch_bounds__(256, (DP * sizeof(T) <= 256 ? 2 : 1)) void attn_bwd_q_kernel(
    AttnArgs a, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
    const T* __restrict__ go, const T* __restrict__ o, const T* __restrict__ rest,
    const float* __restrict__ lse, float* __restrict__ sub, float* __restrict__ delta,
    T* __restrict__ gq) {
  constexpr int KT = BWD_ROWS, TILE = BwdRowsLds<T, DP>::TILE;
  __shared__ BwdRowsLds<T, DP> lds;
  const int G = a.Hq / a.Hk, hk = blockIdx.x % a.Hk;
  int local;
  AttnSpan p;
  if (!attn_tile<false>(a, blockIdx.x / a.Hk, gridDim.x / a.Hk, G, 64, p, local)) return;
  const int all = p.room_q * G;
  const int w = wave_id(), l = lane_id(), r0 = local * 64 + 32 * (w & 1), r = r0 + (l & 31);
  const int used = p.Lq * G;
  auto keys = [&](int row) { return used ? attn_keys(a, p, row < used ? row : used - 1, G) : 0; };
  const int least = keys(r0), most = r0 < used ? keys(r0 + 31) : 0;
  const int end = local * 64 < used ? keys(local * 64 + 63) : 0;
  const int n = keys(r);
  const bool in = r < used;
  const int head = hk * G + r % G;
  const int64_t token = p.q0 + r / G;
  const T* kt = k + p.k0 * a.k_row + hk * a.k_head;
  const T* vt = v + p.k0 * a.v_row + hk * a.v_head;
  if (end > 0 && gq) bwd_q_load<T, DP>(lds.b, kt, vt, a, p.Lk);
  HeadRows<T, DP> x, y;
  x.load(q + token * a.q_row + head * a.q_head, in, a.D);
  y.load(go + (token * a.Hq + head) * a.D, in, a.D);
  const int64_t at = head * a.sq.T + token;
  const float m = in ? lse[at] : NEG_INF;
  const float row_sub = m == NEG_INF ? -NEG_INF : m * LOG2E;
  float row_delta = 0.f;
  {
    HeadRows<T, DP> z;
    z.load(o + (token * a.Hq + head) * a.D, in, a.D);
    row_delta += y.dot(z);
    if (rest) {
      z.load(rest + (token * a.Hq + head) * a.D, in, a.D);
      row_delta += y.dot(z);
    }
    row_delta += other_half(row_delta);
    if (m == NEG_INF) row_delta = 0.f;
  }
  if (sub && in && w < 2 && l < 32) {
    sub[at] = row_sub;
    delta[at] = row_delta;
  }
  if (!gq) return;
  const float c = attn_count(a.scale);
  if (a.scale < 0.f) x.negate();
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{};
  const HeadLanes<T, DP> lanes;
  auto step = [&](auto half, int j0) {
    constexpr int H = decltype(half)::value;
    wait_loads_and_meet<0>();
    kt += KT * a.k_row;
    vt += KT * a.v_row;
    bwd_q_step<T, DP>(lds.b + H * 2 * TILE, lds.b + (1 - H) * 2 * TILE, lanes, kt, vt, a,
                      j0 + KT < end ? p.Lk - j0 - KT : 0, x, y, acc, w >> 1, j0 + 32 * (w >> 1), n,
                      least, most, c, row_sub, row_delta);
  };
  for (int j0 = 0; j0 < end; j0 += 2 * KT) {
    step(std::integral_constant<int, 0>(), j0);
    if (j0 + KT < end) step(std::integral_constant<int, 1>(), j0 + KT);
  }
  wait_loads_and_meet<0>();
  f32x4* sums = (f32x4*)(lds.b + (w & 1) * DP * 128) + l;
  if (w >= 2) {
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        sums[(4 * i + b) * 64] =
            f32x4{acc[i][4 * b], acc[i][4 * b + 1], acc[i][4 * b + 2], acc[i][4 * b + 3]};
  }
  __syncthreads();
  if (w < 2) {
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const f32x4 z = sums[(4 * i + b) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][4 * b + e] += z[e];
      }
  }
  __syncthreads();
  if (w >= 2 || r0 >= all) return;
  put_rows<T, DP>(lds.b, acc, in && row_sub != -NEG_INF && n > 1 ? a.scale : 0.f, gq, a, p, hk, r0,
                  all);
}

// A tile of 64 rows of q and of go, and what is theirs of sub and delta; later
// the sums that the waves exchange, and the rows on their way out.
template <typename T, int DP>
struct alignas(1024) BwdKeysLds {
  static constexpr int TILE = BWD_ROWS * HeadLds<T, DP>::PITCH;
  static constexpr int STAGE = 2 * TILE + 1024;
  static constexpr int OUT = 4 * Rows32<T, DP>::BYTES, SUMS = 4 * DP * 128;
  static constexpr int MORE = OUT > SUMS ? OUT : SUMS;
  char b[2 * STAGE > MORE ? 2 * STAGE : MORE];
};

template <typename T, int DP>
__device__ __forceinline__ void bwd_keys_load(char* to, const T* q, const T* go, const float* sub,
                                              const float* delta, const AttnArgs& a, int left) {
  constexpr int KT = BWD_ROWS, TILE = BwdKeysLds<T, DP>::TILE;
  typedef HeadLds<T, DP> L;
  const int w = wave_id();
  L::template load<KT, 4>(to, q, (int)(a.q_row * sizeof(T)), left, a.D, w);
  L::template load<KT, 4>(to + TILE, go, (int)(a.Hq * a.D * sizeof(T)), left, a.D, w);
  if (w < 2) {
    const int n = __builtin_amdgcn_readfirstlane(left < 0 ? 0 : (left > 64 ? 64 : left));
    __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer(w ? delta : sub, n * 4),
                                             (lds_t*)(to + 2 * TILE + 256 * w), 4, lane_id() * 4, 0,
                                             0, 0);
  }
}

template <typename T, int DP>
struct KeySums {
  f32x16 k[DP / 32], v[DP / 32];
};

// The products of half a tile's rows (half t; the tile from row i0 on, `left` of
// its rows in use) with the wave's keys, of which the lane's is seen by rows from
// `lo` on, the wave's by rows between least and most on.  only: the row that sees
// a single key (every row: ALL_ROWS).
constexpr int ALL_ROWS = INT32_MIN;
template <typename T, int DP>
__device__ __forceinline__ void bwd_keys_step(const char* __restrict__ cur, char* __restrict__ nxt,
                                              const HeadLanes<T, DP>& lanes, const T* q,
                                              const T* go, const float* sub,
                                              const float* delta, const AttnArgs& a, int next,
                                              const HeadRows<T, DP>& k, const HeadRows<T, DP>& v,
                                              KeySums<T, DP>& sums, int t, int i0, int left,
                                              int lo, int least, int most, int only, float c) {
  constexpr int TILE = BwdKeysLds<T, DP>::TILE, PITCH = HeadLds<T, DP>::PITCH;
  bwd_keys_load<T, DP>(nxt, q, go, sub, delta, a, next);
  __builtin_amdgcn_sched_barrier(0);
  const int h = lane_id() >> 5;
  const int i = i0 + 32 * t;
  if (i + 32 <= least || 32 * t >= left) return;
  const char* at = cur + 32 * t * PITCH;
  f32x16 s = scores<T, DP>(lanes, at, k, a.D);
  f32x16 d = scores<T, DP>(lanes, at + TILE, v, a.D);
  const bool masked = i < most || 32 * t + 32 > left || only == ALL_ROWS;
  const float* ps = (const float*)(cur + 2 * TILE) + 32 * t + 4 * h;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const f32x4 m = *(const f32x4*)(ps + 8 * b), y = *(const f32x4*)(ps + 64 + 8 * b);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[4 * b + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * b + e], c, -m[e]));
      d[4 * b + e] = s[4 * b + e] * (d[4 * b + e] - y[e]);
    }
  }
  if (masked)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int row = 32 * t + 8 * (e >> 2) + 4 * h + (e & 3);
      if (i0 + row == only || only == ALL_ROWS) d[e] = 0.f;
      if (i0 + row < lo || row >= left) s[e] = d[e] = 0.f;
    }
  multiply_rows<T, DP>(sums.v, lanes, at + TILE, s);
  multiply_rows<T, DP>(sums.k, lanes, at, d);
}

// dK and dV of 64 keys: for each head of the group, the rows that see them in
// tiles that all four waves share.  Wave w has keys 32 (w % 2) .. + 31 and half w /
// 2 of each tile's rows; at the end two waves add what they have, one stores dK,
// one dV.  blockIdx.y: a share of the group's heads, `heads` of them; with more than
// one its sums go to part as floats (dK, then dV).  (128 keys with all rows a wave:
// half as many workgroups of twice the length, 128 us where this takes 123 for 8 x
// 2048.)
template <typename T, int DP>
__global__ __launch_bounds__(256, (DP * sizeof(T) <= 192 ? 2 : 1)) void attn_bwd_keys_kernel(
    AttnArgs a, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
    const T* __restrict__ go, const float* __restrict__ sub, const float* __restrict__ delta,
    T* __restrict__ gk, T* __restrict__ gv, int heads, float* __restrict__ part) {
  constexpr int KT = BWD_ROWS, STAGE = BwdKeysLds<T, DP>::STAGE;
  __shared__ BwdKeysLds<T, DP> lds;
  const int G = a.Hq / a.Hk, hk = blockIdx.x % a.Hk;
  int local;
  AttnSpan p;
  if (!attn_tile<true>(a, blockIdx.x / a.Hk, gridDim.x / a.Hk, 1, 64, p, local)) return;
  const int w = wave_id(), l = lane_id(), b0 = local * 64;
  const int j0 = b0 + 32 * (w & 1), j = j0 + (l & 31);
  const bool in = j < p.Lk;
  HeadRows<T, DP> x, y;
  x.load(k + (p.k0 + j) * a.k_row + hk * a.k_head, in, a.D);
  y.load(v + (p.k0 + j) * a.v_row + hk * a.v_head, in, a.D);
  const float c = attn_count(a.scale);
  if (a.scale < 0.f) x.negate();
  // the first row that sees a key
  auto first = [&](int key) {
    const int i = key - (p.Lk - p.Lq);
    return a.causal && i > 0 ? i : 0;
  };
  const int lo = first(j), least = first(j0), most = first(j0 + 31);
  // (the row that sees key 0 alone is the first that sees it, among the masked)
  const int only = p.Lk == 1 ? ALL_ROWS : a.causal ? p.Lq - p.Lk : -1;
  const int start = first(b0) / KT * KT, end = b0 < p.Lk ? p.Lq : 0;
  KeySums<T, DP> sums;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) sums.k[i] = sums.v[i] = f32x16{};
  const int tiles = start < end ? (end - start + KT - 1) / KT : 0;
  // tiles of rows, head after head; the next one to load is head ng's from row ni on
  const T *qt, *gt;
  const float *st, *dt;
  const int g0 = blockIdx.y * heads, g1 = g0 + heads < G ? g0 + heads : G;
  int ng = g0, ni = start;
  auto head_at = [&]() {
    const int64_t head = hk * G + ng, row = p.q0 + start;
    qt = q + row * a.q_row + head * a.q_head;
    gt = go + (row * a.Hq + head) * a.D;
    st = sub + head * a.sq.T + row;
    dt = delta + head * a.sq.T + row;
  };
  auto advance = [&]() {
    ni += KT;
    qt += KT * a.q_row;
    gt += (int64_t)KT * a.Hq * a.D;
    st += KT;
    dt += KT;
    if (ni >= end) {
      ni = start;
      if (++ng < g1) head_at();
    }
  };
  const HeadLanes<T, DP> lanes;
  auto step = [&](auto half, int i) {
    constexpr int H = decltype(half)::value;
    wait_loads_and_meet<0>();
    bwd_keys_step<T, DP>(lds.b + H * STAGE, lds.b + (1 - H) * STAGE, lanes, qt, gt, st, dt, a,
                         ng < g1 ? end - ni : 0, x, y, sums, w >> 1, i, end - i, lo, least, most,
                         only, c);
    advance();
  };
  if (tiles > 0) {
    head_at();
    bwd_keys_load<T, DP>(lds.b, qt, gt, st, dt, a, end - start);
    advance();
    int i = start;
    const int all = tiles * (g1 - g0);
    for (int n = 0; n < all; n += 2) {
      step(std::integral_constant<int, 0>(), i);
      i = i + KT >= end ? start : i + KT;
      if (n + 1 < all) step(std::integral_constant<int, 1>(), i);
      i = i + KT >= end ? start : i + KT;
    }
  }
  wait_loads_and_meet<0>();
  // waves 0 and 1 take dK from waves 2 and 3 and give them their dV
  f32x16(&own)[DP / 32] = w < 2 ? sums.k : sums.v;
  {
    const f32x16(&give)[DP / 32] = w < 2 ? sums.v : sums.k;
    f32x4* to = (f32x4*)(lds.b + w * DP * 128) + l;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        to[(4 * i + b) * 64] = f32x4{give[i][4 * b], give[i][4 * b + 1], give[i][4 * b + 2],
                                     give[i][4 * b + 3]};
    __syncthreads();
    const f32x4* from = (const f32x4*)(lds.b + (w ^ 2) * DP * 128) + l;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const f32x4 y = from[(4 * i + b) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) own[i][4 * b + e] += y[e];
      }
    __syncthreads();
  }
  if (j0 >= p.room_k) return;
  const float f = w < 2 ? a.scale : 1.f;
  if (part) {  // a lane's values one after another: few bytes beside the products
    if (j < p.room_k) {
      float* to = part + (((int64_t)blockIdx.y * 2 + (w >> 1)) * a.sk.T + p.k0 + j) * a.Hk * a.D +
                  hk * a.D + 4 * (l >> 5);
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (32 * i + 8 * b + 4 * (l >> 5) < a.D) {
            f32x4 z;
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = in ? own[i][4 * b + e] * f : 0.f;
            *(f32x4*)(to + 32 * i + 8 * b) = z;
          }
    }
    return;
  }
  typedef Rows32<T, DP> R;
  const R to{lds.b + w * R::BYTES};
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      Four<T> z;
#pragma unroll
      for (int e = 0; e < 4; ++e) z.v[e] = in ? (T)(own[i][4 * b + e] * f) : (T)0.f;
      *(Four<T>*)to.four(32 * i + 8 * b + 4 * (l >> 5)) = z;
    }
  to.store((w < 2 ? gk : gv) + hk * a.D, (int64_t)a.Hk * a.D, p.k0 + j0, p.k0 + p.room_k, 0, a.D);
}

// The shares of the group's heads added up: n values of dK, then n of dV.
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_join_kernel(const float* __restrict__ part,
                                                            int shares, int64_t n,
                                                            T* __restrict__ gk,
                                                            T* __restrict__ gv) {
  T* to = blockIdx.y ? gv : gk;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n;
       i += (int64_t)gridDim.x * 1024) {
    f32x4 s = {};
    for (int p = 0; p < shares; ++p) {
      const f32x4 x = *(const f32x4*)(part + ((int64_t)p * 2 + blockIdx.y) * n + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += x[e];
    }
    Four<T> z;
#pragma unroll
    for (int e = 0; e < 4; ++e) z.v[e] = (T)s[e];
    *(Four<T>*)(to + i) = z;
  }
}

// How many shares of a group's heads dK and dV take: enough to give every CU four
// workgroups, where keys alone do not (2000 keys of two heads, eight query heads
// each: 270 us for all heads in one, 157 and 11 for the sums by three shares).
int attn_bwd_shares(int64_t B, int64_t Tk, int64_t Hq, int64_t Hk) {
  const int64_t G = Hq / Hk, blocks = (Tk / 64 + B / 2 + 1) * Hk;
  int64_t s = 1024 / blocks;
  if (s > G) s = G;
  return s < 2 ? 1 : (int)s;
}

}  // namespace tpo

using namespace tpo;

extern "C" int64_t tpo_attention_bwd_workspace_size(int dtype, int64_t B, int64_t Tq, int64_t Tk,
                                                    int64_t Hq, int64_t Hk, int64_t D) {
  if (attn_check("attention_bwd_workspace_size", dtype, B, Tq, Tk, Hq, Hk, D)) return -1;
  const int64_t shares = attn_bwd_shares(B, Tk, Hq, Hk);
  return 2 * round_up(Tq * Hq * 4, 256) +
         (shares > 1 ? round_up(shares * 2 * Tk * Hk * D * 4, 256) : 0);
}

extern "C" int tpo_attention_bwd(int dtype, const void* grad_out, const void* q, const void* k,
                                 const void* v, const void* out, const void* rest,
                                 const float* lse,
                                 const int64_t* offsets_q, const int64_t* offsets_k,
                                 const int64_t* lengths_q, const int64_t* lengths_k, int64_t B,
                                 int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D,
                                 int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                                 int64_t v_row, int64_t v_head, int causal, double scale,
                                 void* grad_q, void* grad_k, void* grad_v, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  if (int rc = attn_check("attention_bwd", dtype, B, Tq, Tk, Hq, Hk, D)) return rc;
  if ((grad_k == nullptr) != (grad_v == nullptr))
    return set_error(TPO_ERR_ARG, "attention_bwd: grad_k and grad_v go together");
  // (dQ alone needs nothing beside its rows)
  const int64_t need =
      grad_k ? tpo_attention_bwd_workspace_size(dtype, B, Tq, Tk, Hq, Hk, D) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(TPO_ERR_WORKSPACE, "attention_bwd: workspace of %lld bytes needed",
                     (long long)need);
  if ((Tq == 0 && Tk == 0) || (!grad_q && !grad_k)) return TPO_OK;
  if (int rc = all_there("attention_bwd", {offsets_q, offsets_k})) return rc;
  if (Tq > 0)
    if (int rc = all_there("attention_bwd", {grad_out, q, out, lse})) return rc;
  if (Tk > 0)
    if (int rc = all_there("attention_bwd", {k, v})) return rc;
  if (int rc = attn_layout("attention_bwd", dtype, D,
                           {grad_out, q, k, v, out, rest, grad_q, grad_k, grad_v, workspace},
                           {q_row, q_head, k_row, k_head, v_row, v_head}, {q_row, k_row, v_row}))
    return rc;
  const AttnArgs a = attn_args(offsets_q, offsets_k, lengths_q, lengths_k, B, Tq, Tk, Hq, Hk, D,
                               q_row, q_head, k_row, k_head, v_row, v_head, causal, scale);
  const int64_t G = Hq / Hk;
  const int64_t places_q = attn_places(Tq, G, B, 64), places_k = attn_places(Tk, 1, B, 64);
  if (places_q * Hk >= AT_GRID || (grad_k && places_k * Hk >= AT_GRID))
    return set_error(TPO_ERR_ARG, "attention_bwd: too many rows");
  const int64_t stats = round_up(Tq * Hq * 4, 256);
  float* sub = grad_k ? (float*)workspace : nullptr;
  float* delta = grad_k ? (float*)((char*)workspace + stats) : nullptr;
  const int shares = attn_bwd_shares(B, Tk, Hq, Hk), heads = (int)((G + shares - 1) / shares);
  const int used = (int)((G + heads - 1) / heads);  // shares that have a head
  float* part = grad_k && used > 1 ? (float*)((char*)workspace + 2 * stats) : nullptr;
  hipStream_t s = (hipStream_t)stream;
  with_element(dtype, [&](auto t) {
    typedef decltype(t) T;
    const T *go = (const T*)grad_out, *qt = (const T*)q, *kt = (const T*)k, *vt = (const T*)v;
    with_head(D, [&](auto dp) {
      constexpr int DP = decltype(dp)::value;
      if (Tq > 0)
        attn_bwd_q_kernel<T, DP><<<dim3((unsigned)(places_q * Hk)), 256, 0, s>>>(
            a, qt, kt, vt, go, (const T*)out, (const T*)rest, lse, sub, delta, (T*)grad_q);
      if (Tk > 0 && grad_k)
        attn_bwd_keys_kernel<T, DP><<<dim3((unsigned)(places_k * Hk), used), 256, 0, s>>>(
            a, qt, kt, vt, go, sub, delta, (T*)grad_k, (T*)grad_v, heads, part);
    });
    if (part && Tk > 0) {
      const int64_t n = Tk * Hk * D, blocks = (n + 1023) / 1024;
      attn_bwd_join_kernel<T><<<dim3((unsigned)(blocks < 2048 ? blocks : 2048), 2), 256, 0, s>>>(
          part, used, n, (T*)grad_k, (T*)grad_v);
    }
  });
  return check_launch("attention_bwd");
}
