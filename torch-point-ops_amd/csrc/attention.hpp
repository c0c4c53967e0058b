// attention.hpp -- what the attention kernels share: arguments, the way from a
// workgroup's number to its rows, and the products of one tile of keys.
//
// The rows of a sequence and key head are its queries of all G = Hq / Hk heads of
// the group, row r = token r / G, head r % G, so that the group shares what is
// read of k and v, also where a sequence has a single query.
//
// A wave works on 32 rows.  Scores are computed transposed, S^T = K Q^T: a lane
// then has one row (column l % 32 of the product), and of every 32 keys the
// sixteen 8 (v / 4) + 4 (l / 32) + v % 4.  Its row's maximum and sum need one
// exchange with the lane 32 on, and the probabilities are already what the
// second product O^T = V^T P^T takes, if v is read in the same order of keys.
#pragma once

#include "gemm_tile.hpp"

namespace tpo {

constexpr int AT_DMAX = 128;
constexpr float LOG2E = 1.44269504088896341f;
constexpr float LN2 = 0.69314718055994531f;
#define NEG_INF (-__builtin_inff())

struct AttnArgs {
  Sequences sq, sk;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  int Hq, Hk, D, causal;
  float scale;
};

// Workgroups of 256 along one axis of a launch: it takes fewer than 2^32 threads there.
constexpr int64_t AT_GRID = (int64_t)1 << 24;

// The rows of a packed batch in tiles of `tile`: sequence s begins at tile
// start(s) G / tile + s.  That leaves room for each sequence's tiles (the last
// one of a sequence and the first of the next may meet in one place, hence + s)
// without a sum over the sequences before it; some places stay empty.
inline int64_t attn_places(int64_t T, int64_t G, int64_t B, int tile) {
  return T * G / tile + B + 2;
}
__device__ __forceinline__ int64_t attn_first(const Sequences& s, int i, int G, int tile) {
  return s.start(i) * G / tile + i;
}
// The last sequence that begins at or before a place: 64 guesses a step.
__device__ __forceinline__ int attn_sequence(const Sequences& s, int64_t place, int G, int tile) {
  int lo = 0, n = s.B + 2;  // among lo .. lo + n - 1
  while (n > 1) {
    const int step = (n + 63) >> 6, i = lo + lane_id() * step;
    const bool at = i < lo + n && attn_first(s, i, G, tile) <= place;
    const uint64_t m = __builtin_amdgcn_ballot_w64(at);
    const int top = m ? 63 - __builtin_clzll(m) : 0;
    const int rest = n - top * step;
    lo += top * step;
    n = rest < step ? rest : step;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// 64-bit values that all lanes share
__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// Tile number p in the order of falling size: a sequence of c tiles has one of
// each size 1 .. c (a causal prompt's last tile sees the most keys, its first keys
// are seen by the most rows).  Where workgroups are few, the long ones have to
// start first: in the order of places a training step's dK and dV kept the CUs
// busy for 58 % of its time.  A lane tries one size; the sequences, `seqs` of them, each
// with the c tiles of its lane, are passed round.  Returns the sequence, or -1, and
// the tile's size.
__device__ __forceinline__ int attn_by_size(int c, int seqs, int p, int& size) {
  const int l = lane_id();
  int lo = 0, hi = 0;
  for (int i = 0; i < seqs; ++i) {
    const int y = __builtin_amdgcn_readlane(c, i);
    hi = y > hi ? y : hi;
  }
  // the smallest u of lo .. hi with n(u) <= p, n(u): tiles larger than u
  while (hi > lo) {
    const int step = (hi - lo + 63) >> 6, u = lo + l * step;
    int n = 0;
    for (int i = 0; i < seqs; ++i) {
      const int y = __builtin_amdgcn_readlane(c, i) - u;
      n += y > 0 ? y : 0;
    }
    const uint64_t m = __builtin_amdgcn_ballot_w64(n <= p);
    const int f = m ? __builtin_ctzll(m) : 64;
    const int top = lo + f * step;
    if (top < hi) hi = top;
    if (f > 0) lo += (f - 1) * step + 1;
    if (lo > hi) lo = hi;
  }
  size = lo;
  if (lo == 0) return -1;
  int n = 0;
  for (int i = 0; i < seqs; ++i) {
    const int y = __builtin_amdgcn_readlane(c, i) - lo;
    n += y > 0 ? y : 0;
  }
  const uint64_t m = __builtin_amdgcn_ballot_w64(c >= lo);
  const int rank = __builtin_popcountll(m & ((1ull << l) - 1));
  const uint64_t at = __builtin_amdgcn_ballot_w64(c >= lo && rank == p - n);
  return at ? __builtin_ctzll(at) : -1;
}

// A workgroup's sequence: its queries and keys, and where they begin.
struct AttnSpan {
  int64_t q0, k0;       // first rows in the packed arrays
  int room_q, Lq, Lk;   // query rows (with those not in use), queries and keys in use
  int room_k;
};
__device__ __forceinline__ AttnSpan attn_span(const AttnArgs& a, int s) {
  AttnSpan p;
  p.q0 = uniform(a.sq.start(s));
  p.k0 = uniform(a.sk.start(s));
  p.room_q = (int)uniform(a.sq.room(s));
  p.room_k = (int)uniform(a.sk.room(s));
  p.Lq = (int)uniform(a.sq.used(s));
  p.Lk = (int)uniform(a.sk.used(s));
  return p;
}

// Up to 62 sequences: each lane has one of them (with the rows before the first and
// after the last), so that one trip to memory brings what decides and all that is
// needed of the sequence then.  (In two or three trips a workgroup's beginning took
// 5 us of its 40 for 8 x 2048.)
constexpr int ATTN_LANES = 62;
struct AttnLanes {
  int start[2], room[2], used[2];  // of queries, of keys
  __device__ __forceinline__ explicit AttnLanes(const AttnArgs& a) {
    const int l = lane_id(), B = a.sq.B;
    const int i = l < 1 ? 0 : (l - 1 < B ? l - 1 : B), j = l < B ? l : B;
    int64_t o[2], p[2], n[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const Sequences& s = y ? a.sk : a.sq;
      o[y] = s.offsets[i];
      p[y] = s.offsets[j];
      n[y] = s.T;
      if (s.lengths && l >= 1 && l <= B) n[y] = s.lengths[l - 1];
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int T = (int)(y ? a.sk.T : a.sq.T);
      auto inside = [](int64_t v, int most) { return v < 0 ? 0 : (v > most ? most : (int)v); };
      start[y] = l < 1 ? 0 : (l > B + 1 ? T : inside(o[y], T));
      const int next = l > B ? T : inside(p[y], T);
      room[y] = next > start[y] ? next - start[y] : 0;
      used[y] = l < 1 || l > B ? 0 : inside(n[y], room[y]);
    }
  }
  __device__ __forceinline__ AttnSpan span(int s) const {
    AttnSpan p;
    p.q0 = __builtin_amdgcn_readlane(start[0], s);
    p.k0 = __builtin_amdgcn_readlane(start[1], s);
    p.room_q = __builtin_amdgcn_readlane(room[0], s);
    p.room_k = __builtin_amdgcn_readlane(room[1], s);
    p.Lq = __builtin_amdgcn_readlane(used[0], s);
    p.Lk = __builtin_amdgcn_readlane(used[1], s);
    return p;
  }
};

// The sequence and tile (of queries, or with KEYS_ of keys) of workgroup p of
// `places`, the largest first; false: none.  A sequence's last tile of queries is its
// largest, its first tile of keys.
template <bool KEYS_>
__device__ __forceinline__ bool attn_tile(const AttnArgs& a, int p, int places, int G, int tile,
                                          AttnSpan& span, int& local) {
  if (a.sq.B <= ATTN_LANES) {
    const AttnLanes lanes(a);
    const int c = (int)(((int64_t)lanes.room[KEYS_] * G + tile - 1) / tile);
    int size;
    int i = attn_by_size(c, a.sq.B + 2, p, size);
    if (i < 0) return false;
    i = __builtin_amdgcn_readfirstlane(i);
    local = KEYS_ ? __builtin_amdgcn_readlane(c, i) - size : size - 1;
    span = lanes.span(i);
    return true;
  }
  // many sequences: many workgroups
  const Sequences& s = KEYS_ ? a.sk : a.sq;
  const int64_t place = KEYS_ ? p : places - 1 - p;
  const int i = attn_sequence(s, place, G, tile);
  const int64_t n = uniform(place - attn_first(s, i, G, tile));
  if (n < 0 || n * tile >= uniform(s.room(i)) * G) return false;
  local = (int)n;
  span = attn_span(a, i);
  return true;
}

// As much for the rows at a place, in the order of places.
__device__ __forceinline__ bool attn_place(const AttnArgs& a, int64_t place, int G, int tile,
                                           AttnSpan& span, int& local) {
  int64_t first;
  if (a.sq.B <= ATTN_LANES) {
    const AttnLanes lanes(a);
    const int64_t at = (int64_t)lanes.start[0] * G / tile + lane_id();
    const uint64_t m = __builtin_amdgcn_ballot_w64(lane_id() < a.sq.B + 2 && at <= place);
    const int i = m ? 63 - __builtin_clzll(m) : 0;
    span = lanes.span(i);
    first = span.q0 * G / tile + i;
  } else {
    const int i = attn_sequence(a.sq, place, G, tile);
    span = attn_span(a, i);
    first = span.q0 * G / tile + i;
  }
  const int64_t n = place - first;
  local = (int)n;
  return n >= 0 && n * tile < (int64_t)span.room_q * G;
}

// The value of lane l ^ 32
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// How rows of up to DP values lie in LDS.
template <typename T, int DP>
struct HeadLds {
  static constexpr int Z = sizeof(T);
  static constexpr int PITCH = DP * Z <= 64 ? 64 : DP * Z <= 128 ? 128 : DP * Z <= 256 ? 256 : 512;
  static constexpr int CPR = PITCH / 16, RPL = 1024 / PITCH;
  // Chunk c of a row is at place c ^ swap(row), so that both ways of reading touch
  // different banks: sixteen rows, one chunk (for products that sum over the head),
  // and four rows, 64 bytes (for those that sum over the rows; floats: two rows
  // four apart, 128 bytes, but where a row is no longer than that).
  static __device__ __forceinline__ constexpr int swap(int r) {
    if (PITCH == 64) return r >> 2 & 3;
    if (Z == 4) return PITCH == 128 ? r >> 1 & 7 : (r >> 2 & 1) << 3 | (r >> 3 & 1) << 2 | (r & 3);
    return PITCH == 128 ? (r >> 1 & 1) << 2 | (r >> 2 & 3) : (r & 3) << 2 | (r >> 2 & 3);
  }
  // Loads `R` rows into lds, by NW waves of which this is w: the first n rows
  // from p on, row_bytes apart, D values of each; the rest is 0.
  template <int R, int NW>
  static __device__ __forceinline__ void load(char* lds, const T* p, int row_bytes, int n, int D,
                                              int w) {
    constexpr int N = R / RPL / NW;
    static_assert(N >= 1 && N * RPL * NW == R, "rows of a tile");
    // (clamped by vector instructions: said to be uniform, or each load becomes a loop)
    n = __builtin_amdgcn_readfirstlane(n < 0 ? 0 : (n > R ? R : n));
    const __amdgpu_buffer_rsrc_t rsrc = buffer(p, n * row_bytes);
    const int l = lane_id(), r = l / CPR, bytes = D * Z;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int row = (w * N + j) * RPL;  // a multiple of RPL: its part of swap() is apart
      const int c = ((l % CPR) ^ swap(r) ^ swap(row)) << 4;
      load_lds(rsrc, lds + (w * N + j) * 1024, c < bytes ? r * row_bytes + c : NOWHERE,
               row * row_bytes);
    }
  }
};

// Where a lane reads, from the start of a tile's rows: as numbers that are made
// once, so that a read in the loop is one instruction with a constant offset.
template <typename T, int DP>
struct HeadLanes {
  typedef HeadLds<T, DP> L;
  typedef typename Chunk<T>::V V;
  static constexpr int N = DP * L::Z / 32, M = DP / 32, PITCH = L::PITCH;
  int row[N];        // row l % 32, chunk 2 s + l / 32
  int lo[M], hi[M];  // half types: see by_col; float: lo[0]

  __device__ __forceinline__ HeadLanes() {
    const int l = lane_id(), h = l >> 5, r = l & 31;
#pragma unroll
    for (int s = 0; s < N; ++s) row[s] = r * PITCH + (((2 * s + h) ^ L::swap(r)) << 4);
    if constexpr (L::Z == 4) {
      lo[0] = 4 * h * PITCH + ((((l & 31) >> 2) ^ L::swap(4 * h)) << 4) + (l & 3) * 4;
    } else {
      const int e = l & 15, g = (l >> 4) & 1, q = 4 * h + (e >> 2), c = 2 * g + (e >> 1 & 1);
#pragma unroll
      for (int i = 0; i < M; ++i) {
        lo[i] = q * PITCH + 8 * (e & 1) + (((c ^ L::swap(q)) << 4) ^ (64 * i));
        hi[i] = (q + 8) * PITCH + 8 * (e & 1) + (((c ^ L::swap(q + 8)) << 4) ^ (64 * i));
      }
    }
  }
  // chunk 2 s + l / 32 of row l % 32 of the rows at lds
  __device__ __forceinline__ V by_row(const char* lds, int s) const {
    return *(const V*)(lds + row[s]);
  }
  // half types: value 32 i + l % 32 of the rows 16 s + 4 (l / 32) + 0 .. 3 and + 8 ..
  // 11: sixteen lanes give the addresses of 4 rows x 16 columns and get a column each
  __device__ __forceinline__ V by_col(const char* lds, int s, int i) const {
    static_assert(L::Z == 2, "half types");
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    lds += 16 * s * PITCH;
    const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(lds + lo[i]));
    const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(lds + hi[i]));
    return __builtin_bit_cast(V, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  // float: value 32 i + l % 32 of row 8 (v / 4) + 4 (l / 32) + v % 4
  __device__ __forceinline__ float by_col1(const char* lds, int v, int i) const {
    const int r = 8 * (v >> 2) + (v & 3);
    return *(const float*)(lds + r * PITCH + (lo[0] ^ (L::swap(r) << 4) ^ (128 * i)));
  }
};

// acc[i] += X^T P^T over the 32 rows of X at lds: sums of value
// 32 i + .. of X times the lane's sixteen p.  Half types round p to the type.
template <typename T, int DP>
__device__ __forceinline__ void multiply_rows(f32x16 (&acc)[DP / 32], const HeadLanes<T, DP>& x,
                                              const char* lds, const f32x16& p) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int v = 0; v < 16; ++v)
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
        acc[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.by_col1(lds, v, i), p[v], acc[i], 0, 0, 0);
  } else {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      typename Chunk<T>::V y;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (T)p[8 * s + e];
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) mma(acc[i], x.by_col(lds, s, i), y);
    }
  }
}

// A wave's 32 rows of q (or of another array laid out as it) as the products
// take them, chunk 2 s + l / 32 of row l % 32; 0 where there is no row.
template <typename T, int DP>
struct HeadRows {
  static constexpr int N = DP * sizeof(T) / 32;
  typename Chunk<T>::V x[N];
  __device__ __forceinline__ void load(const T* p, bool in, int D) {
    constexpr int PER = 16 / sizeof(T);
    const int h = lane_id() >> 5;
#pragma unroll
    for (int s = 0; s < N; ++s) {
      x[s] = typename Chunk<T>::V{};
      if (in && (2 * s + h) * PER < D) x[s] = *(const typename Chunk<T>::V*)(p + (2 * s + h) * PER);
    }
  }
  __device__ __forceinline__ void negate() {
#pragma unroll
    for (int s = 0; s < N; ++s) x[s] = -x[s];
  }
  // The lane's part of the sum of products with another array's row.
  __device__ __forceinline__ float dot(const HeadRows& y) const {
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < N; ++s)
#pragma unroll
      for (int e = 0; e < (int)(16 / sizeof(T)); ++e)
        sum = __builtin_fmaf((float)x[s][e], (float)y.x[s][e], sum);
    return sum;
  }
};

// A wave's 32 rows of sums, f times each, to the rows r0 .. of a sequence and key
// head in an array laid out as out (f 0: nothing but zeros), by way of LDS.
// REST: what rounding takes from them instead.
template <typename T, int DP, bool REST = false>
__device__ __forceinline__ void put_rows(char* lds, const f32x16 (&acc)[DP / 32], float f,
                                         T* __restrict__ out, const AttnArgs& a, const AttnSpan& p,
                                         int hk, int r0, int all) {
  typedef Rows32<T, DP> R;
  const R to{lds + wave_id() * R::BYTES};
  const int l = lane_id(), G = a.Hq / a.Hk;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      Four<T> y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float z = f == 0.f ? 0.f : acc[i][4 * b + e] * f;
        y.v[e] = (T)(REST ? z - (float)(T)z : z);
      }
      *(Four<T>*)to.four(32 * i + 8 * b + 4 * (l >> 5)) = y;
    }
  to.wait();
#pragma unroll
  for (int i = 0; i < 32 * R::CHUNKS; i += 64) {
    const int rr = (i + l) / R::CHUNKS, cc = (i + l) % R::CHUNKS * R::PER, row = r0 + rr;
    if (row < all && cc < a.D)
      *(f32x4*)(out + ((p.q0 + row / G) * a.Hq + hk * G + row % G) * a.D + cc) =
          *(const f32x4*)((const T*)(to.lds + rr * R::PITCH) + cc);
  }
  to.wait();
}

// The keys that row r (of the rows of a sequence and key head) sees.
__device__ __forceinline__ int attn_keys(const AttnArgs& a, const AttnSpan& p, int r, int G) {
  const int t = r / G;
  if (!a.causal) return p.Lk;
  const int n = t + p.Lk - p.Lq + 1;
  return n < 0 ? 0 : (n > p.Lk ? p.Lk : n);
}

// What a score counts in the exponent of 2; never 0, as 0 x -inf is not a number.
// A negative scale turns the sign of one operand instead.
__device__ __forceinline__ float attn_count(float scale) {
  return fmaxf(fabsf(scale) * LOG2E, 1e-37f);
}

// Keys (or rows) a tile in LDS: what two operands' tiles leave room for, twice over.
template <typename T> constexpr int KEYS = sizeof(T) == 4 ? 32 : 64;

template <typename T, int DP>
struct alignas(1024) PromptLds {
  static constexpr int TILE = KEYS<T> * HeadLds<T, DP>::PITCH;
  static constexpr int OUT = 4 * Rows32<T, DP>::BYTES;
  char b[4 * TILE > OUT ? 4 * TILE : OUT];
};

// X Y^T of the 32 rows of X at lds and the wave's rows: transposed scores.
// Float chunks past D (of 8 values, four slow matrix instructions) are left out.
template <typename T, int DP>
__device__ __forceinline__ f32x16 scores(const HeadLanes<T, DP>& x, const char* lds,
                                         const HeadRows<T, DP>& y, int D) {
  f32x16 s = {};
#pragma unroll
  for (int c = 0; c < HeadRows<T, DP>::N; ++c)
    if (sizeof(T) == 2 || 8 * c < D) mma(s, x.by_row(lds, c), y.x[c]);
  return s;
}

int attn_check(const char* op, int dtype, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq,
               int64_t Hk, int64_t D);
int attn_layout(const char* op, int dtype, int64_t D, std::initializer_list<const void*> p,
                std::initializer_list<int64_t> strides, std::initializer_list<int64_t> rows);
AttnArgs attn_args(const int64_t* oq, const int64_t* ok, const int64_t* lq, const int64_t* lk,
                   int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D,
                   int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head, int64_t v_row,
                   int64_t v_head, int causal, double scale);

// Calls f with the head size rounded up to one that the kernels are built for.
template <typename F>
void with_head(int64_t D, F&& f) {
  if (D <= 32) f(std::integral_constant<int, 32>());
  else if (D <= 64) f(std::integral_constant<int, 64>());
  else if (D <= 96) f(std::integral_constant<int, 96>());
  else f(std::integral_constant<int, 128>());
}

}  // namespace tpo
