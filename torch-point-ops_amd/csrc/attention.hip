// attention.hip -- softmax attention over packed sequences with grouped heads,
// forward.  Sequence by sequence, head by head:
//   S = scale q k^T (causal: row i sees key j where j <= i + Lk - Lq)
//   P = softmax(S), o = P v; a row that sees no key is 0
//
// One pass over the keys with each row's running maximum m and sum l:
//   m' = max(m, max S), a = exp(m - m'), l' = a l + sum exp(S - m'),
//   o' = a o + exp(S - m') v.
// m follows only when it would grow by more than 2^8 (in the exponentials'
// measure): until then exponentials of up to 2^8 are summed, which costs floats
// nothing, and most tiles need no pass over the sums o.
// Half types: probabilities are rounded to the type for the second product (the
// same relative rounding as the result's); their sum is taken before that.
#include "attention.hpp"

namespace tpo {

// A wave's rows under way.
template <typename T, int DP>
struct RowSums {
  f32x16 acc[DP / 32];
  float m, l;  // l: of the lane's own keys, half of the row's

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{};
    m = NEG_INF;
    l = 0.f;
  }
  // The exponentials of KT keys from j0 on (k at lds), of which the lane's row sees
  // those below n, with the sums brought to their maximum; c: what a score counts in
  // the exponent of 2.
  template <int KT>
  __device__ __forceinline__ void weigh(f32x16 (&s)[KT / 32], const HeadLanes<T, DP>& lanes,
                                        const char* lds, const HeadRows<T, DP>& q, int D, int j0,
                                        int n, bool masked, float c) {
    constexpr int PITCH = HeadLds<T, DP>::PITCH;
#pragma unroll
    for (int t = 0; t < KT / 32; ++t) s[t] = scores<T, DP>(lanes, lds + 32 * t * PITCH, q, D);
    if (masked) {
      const int first = j0 + 4 * (lane_id() >> 5);
#pragma unroll
      for (int t = 0; t < KT / 32; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (first + 32 * t + 8 * (e >> 2) + (e & 3) >= n) s[t][e] = NEG_INF;
    }
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < KT / 32; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[t][e]);
    top = fmaxf(top, other_half(top));
    if (__builtin_amdgcn_ballot_w64((top - m) * c > 8.f)) {
      const float m2 = fmaxf(m, top);
      const float a = m2 == NEG_INF ? 1.f : __builtin_amdgcn_exp2f((m - m2) * c);
      m = m2;
      l *= a;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] *= a;
    }
    const float b = m == NEG_INF ? 0.f : -m * c;
#pragma unroll
    for (int t = 0; t < KT / 32; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[t][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e], c, b));
        l += s[t][e];
      }
  }
  // Their part of the sums (v at lds).
  template <int KT>
  __device__ __forceinline__ void gather(const f32x16 (&s)[KT / 32], const HeadLanes<T, DP>& lanes,
                                         const char* lds) {
#pragma unroll
    for (int t = 0; t < KT / 32; ++t)
      multiply_rows<T, DP>(acc, lanes, lds + 32 * t * HeadLds<T, DP>::PITCH, s[t]);
  }
};

// The loads of a tile of keys and one's products, in parts of LDS that are apart.
template <typename T, int DP>
__device__ __forceinline__ void prompt_step(const char* __restrict__ cur, char* __restrict__ nxt,
                                            const HeadLanes<T, DP>& lanes, const T* k, const T* v,
                                            const AttnArgs& a, int left,
                                            const HeadRows<T, DP>& q, RowSums<T, DP>& rows, int j0,
                                            int n, int least, int most, float c) {
  constexpr int KT = KEYS<T>, TILE = PromptLds<T, DP>::TILE;
  typedef HeadLds<T, DP> L;
  L::template load<KT, 4>(nxt, k, (int)(a.k_row * sizeof(T)), left, a.D, wave_id());
  L::template load<KT, 4>(nxt + TILE, v, (int)(a.v_row * sizeof(T)), left, a.D, wave_id());
  __builtin_amdgcn_sched_barrier(0);
  if (j0 < most) {
    f32x16 s[KT / 32];
    rows.template weigh<KT>(s, lanes, cur, q, a.D, j0, n, j0 + KT > least, c);
    rows.template gather<KT>(s, lanes, cur + TILE);
  }
}

// Prompts: a workgroup of four waves takes 128 rows, 32 a wave, and all their
// keys in tiles that it loads once for all four.
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void attn_prompt_kernel(AttnArgs a, const T* __restrict__ q,
                                                             const T* __restrict__ k,
                                                             const T* __restrict__ v,
                                                             T* __restrict__ out,
                                                             float* __restrict__ lse,
                                                             T* __restrict__ rest) {
  constexpr int KT = KEYS<T>, TILE = PromptLds<T, DP>::TILE;
  __shared__ PromptLds<T, DP> lds;
  const int G = a.Hq / a.Hk, hk = blockIdx.x % a.Hk;
  int local;
  AttnSpan p;
  if (!attn_tile<false>(a, blockIdx.x / a.Hk, gridDim.x / a.Hk, G, 128, p, local)) return;
  const int all = p.room_q * G;
  const int w = wave_id(), l = lane_id(), r0 = local * 128 + 32 * w, r = r0 + (l & 31);
  const int used = p.Lq * G;
  // the wave's rows see between `least` and `most` keys, the workgroup's up to `end`
  auto keys = [&](int row) { return used ? attn_keys(a, p, row < used ? row : used - 1, G) : 0; };
  const int least = keys(r0), most = r0 < used ? keys(r0 + 31) : 0;
  const int end = local * 128 < used ? keys(local * 128 + 127) : 0;
  const int n = keys(r);
  const bool in = r < used;
  const int head = hk * G + r % G;
  const int64_t token = p.q0 + r / G;
  const T* kt = k + p.k0 * a.k_row + hk * a.k_head;
  const T* vt = v + p.k0 * a.v_row + hk * a.v_head;
  typedef HeadLds<T, DP> L;
  if (end > 0) {
    L::template load<KT, 4>(lds.b, kt, (int)(a.k_row * sizeof(T)), p.Lk, a.D, w);
    L::template load<KT, 4>(lds.b + TILE, vt, (int)(a.v_row * sizeof(T)), p.Lk, a.D, w);
  }
  HeadRows<T, DP> x;
  x.load(q + token * a.q_row + head * a.q_head, in, a.D);
  const float c = attn_count(a.scale);
  if (a.scale < 0.f) x.negate();
  RowSums<T, DP> rows;
  rows.clear();
  const HeadLanes<T, DP> lanes;
  auto step = [&](auto half, int j0) {  // (the halves by name: LDS addresses are constants)
    constexpr int H = decltype(half)::value;
    wait_loads_and_meet<0>();
    kt += KT * a.k_row;
    vt += KT * a.v_row;
    prompt_step<T, DP>(lds.b + H * 2 * TILE, lds.b + (1 - H) * 2 * TILE, lanes, kt, vt, a,
                       j0 + KT < end ? p.Lk - j0 - KT : 0, x, rows, j0, n, least, most, c);
  };
  for (int j0 = 0; j0 < end; j0 += 2 * KT) {
    step(std::integral_constant<int, 0>(), j0);
    if (j0 + KT < end) step(std::integral_constant<int, 1>(), j0 + KT);
  }
  wait_loads_and_meet<0>();
  if (r0 >= all) return;

  const float sum = rows.l + other_half(rows.l);
  const float inv = in && sum != 0.f ? 1.f / sum : 0.f;
  put_rows<T, DP>(lds.b, rows.acc, inv, out, a, p, hk, r0, all);
  if (rest) put_rows<T, DP, true>(lds.b, rows.acc, inv, rest, a, p, hk, r0, all);
  if (lse && l < 32 && r < all)
    lse[head * a.sq.T + token] =
        inv == 0.f ? NEG_INF : (rows.m * c + __builtin_amdgcn_logf(sum)) * LN2;
}

// Few rows over many keys: a workgroup takes 32 rows and one of gridDim.z shares
// of their keys, its four waves in turn a tile of 32 keys each from LDS of their
// own, so that no wave waits for another before the end.  A wave has room for one
// tile of k and one of v: v is on its way while the scores are computed, the next
// k while they are multiplied with v.
constexpr int STEP_WAVES = 4;
template <typename T, int DP>
struct alignas(1024) StepLds {
  static constexpr int TILE = 32 * HeadLds<T, DP>::PITCH;
  static constexpr int SUMS = STEP_WAVES * 32 * (DP + 4) * 4;
  static constexpr int TILES = STEP_WAVES * 2 * TILE;
  char b[TILES > SUMS ? TILES : SUMS];
  float m[STEP_WAVES][32], l[STEP_WAVES][32];
};

// 32 rows of k or of v from p on, `left` of them, to a wave's own LDS.
template <typename T, int DP>
__device__ __forceinline__ void step_load(char* to, const T* p, int64_t row, const AttnArgs& a,
                                          int left) {
  HeadLds<T, DP>::template load<32, 1>(to, p, (int)(row * sizeof(T)), left, a.D, 0);
}
// Waits until of a wave's loads only the youngest tile's are under way and its LDS
// reads have ended.
template <int LOADS>
__device__ __forceinline__ void step_wait() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((LOADS & 15) | (LOADS >> 4) << 14 | 0x70);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// What a lane's row sees: n keys, the rows of its 32 between least and most.
struct StepRows {
  int n, least, most;
};

// The two halves of a tile's work; k and v are apart in LDS.
template <typename T, int DP>
__device__ __forceinline__ void step_weigh(const char* __restrict__ kl, char* __restrict__ vl,
                                           const HeadLanes<T, DP>& lanes, const T* v,
                                           const AttnArgs& a, int left,
                                           const HeadRows<T, DP>& q, RowSums<T, DP>& rows,
                                           const StepRows& sees, f32x16 (&s)[1], int j0, float c) {
  step_load<T, DP>(vl, v, a.v_row, a, left);
  step_wait<StepLds<T, DP>::TILE / 1024>();  // k has landed
  if (j0 < sees.most)
    rows.template weigh<32>(s, lanes, kl, q, a.D, j0, sees.n, j0 + 32 > sees.least, c);
}
template <typename T, int DP>
__device__ __forceinline__ void step_gather(char* __restrict__ kl, const char* __restrict__ vl,
                                            const HeadLanes<T, DP>& lanes, const T* k,
                                            const AttnArgs& a, int left,
                                            RowSums<T, DP>& rows, const StepRows& sees,
                                            const f32x16 (&s)[1], int j0) {
  step_load<T, DP>(kl, k, a.k_row, a, left);
  step_wait<StepLds<T, DP>::TILE / 1024>();  // v has landed
  if (j0 < sees.most) rows.template gather<32>(s, lanes, vl);
}

// part: with shares, each row's sums (D floats, not divided), and in ml their
// maximum (in the exponent of 2) and sum
template <typename T, int DP>
__global__ __launch_bounds__(64 * STEP_WAVES,
                             (DP * sizeof(T) <= 256 ? 2 : 1)) void attn_step_kernel(
    AttnArgs a, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
    T* __restrict__ out, float* __restrict__ lse, T* __restrict__ rest,
    float* __restrict__ part, float2* __restrict__ ml) {
  constexpr int W = STEP_WAVES, TILE = StepLds<T, DP>::TILE;
  __shared__ StepLds<T, DP> lds;
  const int G = a.Hq / a.Hk, hk = blockIdx.y, shares = gridDim.z;
  int local;
  AttnSpan p;
  if (!attn_place(a, blockIdx.x, G, 32, p, local)) return;
  const int all = p.room_q * G;
  const int w = wave_id(), l = lane_id(), r0 = local * 32;
  const int used = p.Lq * G;
  auto keys = [&](int row) { return used ? attn_keys(a, p, row < used ? row : used - 1, G) : 0; };
  const int r = r0 + (l & 31), most = r0 < used ? keys(r0 + 31) : 0;
  const StepRows sees{keys(r), keys(r0), most};
  HeadRows<T, DP> x;
  x.load(q + (p.q0 + r / G) * a.q_row + (hk * G + r % G) * a.q_head, r < used, a.D);
  if (a.scale < 0.f) x.negate();
  RowSums<T, DP> rows;
  rows.clear();
  const int tiles = (most + 31) / 32, per = (tiles + shares - 1) / shares;
  const int t0 = per * blockIdx.z, t1 = t0 + per < tiles ? t0 + per : tiles;
  const float c = attn_count(a.scale);
  const T* kt = k + p.k0 * a.k_row + hk * a.k_head;
  const T* vt = v + p.k0 * a.v_row + hk * a.v_head;
  char *kl = lds.b + w * 2 * TILE, *vl = kl + TILE;
  const HeadLanes<T, DP> lanes;
  if (t0 + w < t1)
    step_load<T, DP>(kl, kt + (int64_t)(t0 + w) * 32 * a.k_row, a.k_row, a, most - (t0 + w) * 32);
  for (int t = t0 + w; t < t1; t += W) {
    const int64_t j0 = (int64_t)t * 32, next = j0 + 32 * W;
    f32x16 sc[1];
    step_wait<TILE / 1024>();  // (the reads of v's place have ended)
    step_weigh<T, DP>(kl, vl, lanes, vt + j0 * a.v_row, a, most - (int)j0, x, rows, sees, sc,
                      (int)j0, c);
    step_wait<TILE / 1024>();  // (and those of k's)
    step_gather<T, DP>(kl, vl, lanes, kt + next * a.k_row, a, t + W < t1 ? most - (int)next : 0,
                       rows, sees, sc, (int)j0);
  }
  wait_loads_and_meet<0>();

  // the waves' sums together
  constexpr int P = DP + 4;
  const float sum = rows.l + other_half(rows.l);
  float* mysums = (float*)lds.b + w * 32 * P;
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
    lds.m[w][l] = rows.m;
    lds.l[w][l] = sum;
  }
  __syncthreads();
  constexpr int PER_ROW = 2 * W, D1 = DP / PER_ROW;  // lanes a row, values a lane
  const int rr = threadIdx.x / PER_ROW, d0 = threadIdx.x % PER_ROW * D1, row = r0 + rr;
  if (row >= all) return;
  float m = NEG_INF, total = 0.f, f[W];
#pragma unroll
  for (int i = 0; i < W; ++i) m = fmaxf(m, lds.m[i][rr]);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float y = lds.l[i][rr];
    f[i] = y == 0.f ? 0.f : __builtin_amdgcn_exp2f((lds.m[i][rr] - m) * c);
    total += f[i] * y;
  }
  if (row >= used) total = 0.f;
  const int64_t at = (p.q0 + row / G) * a.Hq + hk * G + row % G;
  const float inv = shares > 1 ? 1.f : total != 0.f ? 1.f / total : 0.f;
#pragma unroll
  for (int d = 0; d < D1; ++d) {
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (f[i] != 0.f) y += f[i] * ((float*)lds.b)[(i * 32 + rr) * P + d0 + d];
    if (d0 + d < a.D) {
      if (shares > 1) {
        if (total != 0.f) part[(at * shares + blockIdx.z) * a.D + d0 + d] = y;
      } else {
        const T z = total == 0.f ? (T)0.f : (T)(y * inv);
        out[at * a.D + d0 + d] = z;
        if (rest) rest[at * a.D + d0 + d] = total == 0.f ? (T)0.f : (T)(y * inv - (float)z);
      }
    }
  }
  if (d0 == 0) {
    if (shares > 1)
      ml[at * shares + blockIdx.z] = make_float2(m * c, total);
    else if (lse)
      lse[(at % a.Hq) * a.sq.T + at / a.Hq] =
          total == 0.f ? NEG_INF : (m * c + __builtin_amdgcn_logf(total)) * LN2;
  }
}

int attn_check(const char* op, int dtype, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq,
               int64_t Hk, int64_t D) {
  if (dtype != TPO_F32 && dtype != TPO_F16 && dtype != TPO_BF16)
    return set_error(TPO_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (B < 0 || B > (1 << 24) || Tq < 0 || Tk < 0 || Tq >= ((int64_t)1 << 31) ||
      Tk >= ((int64_t)1 << 31) || Hq < 1 || Hk < 1 || Hq > 1024 || Hq % Hk != 0 || D < 1 ||
      D > AT_DMAX || Tq * Hq >= ((int64_t)1 << 31) || Tk * Hk >= ((int64_t)1 << 31))
    return set_error(TPO_ERR_ARG,
                     "%s: bad sizes B=%lld Tq=%lld Tk=%lld Hq=%lld Hk=%lld D=%lld (Hq a multiple "
                     "of Hk, D at most %d)",
                     op, (long long)B, (long long)Tq, (long long)Tk, (long long)Hq, (long long)Hk,
                     (long long)D, AT_DMAX);
  return TPO_OK;
}

// Pointers and strides that the kernels can load 16 bytes at a time, 64 rows of
// an operand spanning less than 2^31 bytes.
int attn_layout(const char* op, int dtype, int64_t D, std::initializer_list<const void*> ptrs,
                std::initializer_list<int64_t> strides, std::initializer_list<int64_t> rows) {
  const int64_t z = element_bytes(dtype);
  bool ok = D * z % 16 == 0;
  for (const void* p : ptrs) ok = ok && ((uintptr_t)p & 15) == 0;
  for (int64_t s : strides) ok = ok && s >= 0 && s * z % 16 == 0;
  for (int64_t s : rows) ok = ok && s > 0 && s * z < (1 << 25);
  return ok ? TPO_OK
            : set_error(TPO_ERR_ARG,
                        "%s: pointers, heads and strides must be multiples of 16 bytes, rows apart "
                        "by 16 to 2^25 bytes",
                        op);
}

AttnArgs attn_args(const int64_t* oq, const int64_t* ok, const int64_t* lq, const int64_t* lk,
                   int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D,
                   int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head, int64_t v_row,
                   int64_t v_head, int causal, double scale) {
  AttnArgs a;
  a.sq = Sequences{oq, lq, Tq, (int)B};
  a.sk = Sequences{ok, lk, Tk, (int)B};
  a.q_row = q_row;
  a.q_head = q_head;
  a.k_row = k_row;
  a.k_head = k_head;
  a.v_row = v_row;
  a.v_head = v_head;
  a.Hq = (int)Hq;
  a.Hk = (int)Hk;
  a.D = (int)D;
  a.causal = causal ? 1 : 0;
  a.scale = (float)scale;
  return a;
}


// Which kernel a call takes, and the shares of the keys.
// Prompts' workgroups of 128 rows load each key once for all of them; the others'
// of 32 rows share the keys among their waves, and fill the CUs where there are few
// rows.  So it goes by the number of workgroups of 128 rows, with each sequence and
// key head's last one not full: half types, heads of 64 and less (four such
// workgroups on a CU) from 352 on (384 of 4096 keys, causal: 66 us, by 32 rows 69;
// 256: 62, 50), longer heads from 144 on (128 of 1024: 25, 22; 144 of 1536: 34, 36;
// 192 of 3000: 59, 65), float, whose products take longer, from 448 on (350 of 1000
// keys: 80, 69; 512 of 4096, heads of 128: 735, 911).  Where there are at most 32 rows
// to a sequence, three of four waves only help to load: that pays for 512 and more of
// them with keys few enough to be no more than a wave's share (64 x 8 heads, 512
// keys: 21, 24; 256 x 8, 2048 keys: 256, 237), not in float.
// Shares (by the room for keys: what is in use is not known here): for 128
// workgroups in all where that leaves a share 256 keys (64 in float); starting and
// adding up cost more than the other CUs would give (16384 keys, 8 workgroups: 16
// shares 21.5 us, 32 23.9, 64 26.2).  For long keys up to 1024 workgroups, so that
// sequences of different lengths even out (64 x 16384 keys: one share each 162 us, 4
// 99, 16 76).
struct Way {
  int rows;  // a workgroup's: 32 (few rows) or 128 (prompts)
  int shares;
};
Way attn_way(int dtype, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D) {
  const int64_t G = Hq / Hk, n = B < 1 ? 1 : B, keys = Tk / n;
  const int64_t each = Tq < 1 ? 1 : (Tq * G + n - 1) / n;
  const bool single = dtype == TPO_F32;
  const int64_t prompts = (each + 127) / 128 * n * Hk, blocks = (each + 31) / 32 * n * Hk;
  if (each > 32 ? prompts >= (single ? 448 : D > 64 ? 144 : 352)
                : prompts >= 512 && keys <= 1024 && !single)
    return Way{128, 1};
  const int64_t least = single ? 64 : 256, more = single ? 512 : 1024;
  int64_t s = (128 + blocks - 1) / blocks, t = 1024 / blocks;
  if (s > keys / least) s = keys / least;
  if (t > keys / more) t = keys / more;
  if (s < t) s = t;
  if (keys < 4 * least || s < 1) s = 1;
  return Way{32, s > 64 ? 64 : (int)s};
}

}  // namespace tpo

using namespace tpo;

extern "C" int64_t tpo_attention_fwd_workspace_size(int dtype, int64_t B, int64_t Tq, int64_t Tk,
                                                    int64_t Hq, int64_t Hk, int64_t D) {
  if (attn_check("attention_fwd_workspace_size", dtype, B, Tq, Tk, Hq, Hk, D)) return -1;
  const Way w = attn_way(dtype, B, Tq, Tk, Hq, Hk, D);
  if (w.shares == 1) return 0;
  return round_up(Tq * Hq * w.shares * D * 4, 256) + round_up(Tq * Hq * w.shares * 8, 256);
}

extern "C" int tpo_attention_fwd_rows(int dtype, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq,
                                      int64_t Hk, int64_t D) {
  if (int rc = attn_check("attention_fwd_rows", dtype, B, Tq, Tk, Hq, Hk, D)) return rc;
  return attn_way(dtype, B, Tq, Tk, Hq, Hk, D).rows;
}

extern "C" int tpo_attention_fwd(int dtype, const void* q, const void* k, const void* v,
                                 const int64_t* offsets_q, const int64_t* offsets_k,
                                 const int64_t* lengths_q, const int64_t* lengths_k, int64_t B,
                                 int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D,
                                 int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                                 int64_t v_row, int64_t v_head, int causal, double scale,
                                 void* out, float* lse, void* rest, void* workspace,
                                 int64_t workspace_bytes,
                                 void* stream) {
  if (int rc = attn_check("attention_fwd", dtype, B, Tq, Tk, Hq, Hk, D)) return rc;
  if (Tq == 0) return TPO_OK;
  if (int rc = all_there("attention_fwd", {q, offsets_q, offsets_k, out})) return rc;
  if (Tk > 0)
    if (int rc = all_there("attention_fwd", {k, v})) return rc;
  if (int rc = attn_layout("attention_fwd", dtype, D, {q, k, v, out, rest, workspace},
                           {q_row, q_head, k_row, k_head, v_row, v_head}, {q_row, k_row, v_row}))
    return rc;
  const int64_t need = tpo_attention_fwd_workspace_size(dtype, B, Tq, Tk, Hq, Hk, D);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(TPO_ERR_WORKSPACE, "attention_fwd: workspace of %lld bytes needed",
                     (long long)need);
  const AttnArgs a = attn_args(offsets_q, offsets_k, lengths_q, lengths_k, B, Tq, Tk, Hq, Hk, D,
                               q_row, q_head, k_row, k_head, v_row, v_head, causal, scale);
  const Way w = attn_way(dtype, B, Tq, Tk, Hq, Hk, D);
  const int64_t G = Hq / Hk, places = attn_places(Tq, G, B, w.rows);
  if ((w.rows == 128 ? places * Hk : places) >= AT_GRID)
    return set_error(TPO_ERR_ARG, "attention_fwd: too many rows");
  hipStream_t s = (hipStream_t)stream;
  float* part = (float*)workspace;
  float2* ml = (float2*)((char*)workspace + round_up(Tq * Hq * w.shares * D * 4, 256));
  with_element(dtype, [&](auto t) {
    typedef decltype(t) T;
    with_head(D, [&](auto dp) {
      constexpr int DP = decltype(dp)::value;
      if (w.rows == 128)
        attn_prompt_kernel<T, DP><<<dim3((unsigned)(places * Hk)), 256, 0, s>>>(
            a, (const T*)q, (const T*)k, (const T*)v, (T*)out, lse, (T*)rest);
      else
        attn_step_kernel<T, DP>
            <<<dim3((unsigned)places, (unsigned)Hk, w.shares), 64 * STEP_WAVES, 0, s>>>(
                a, (const T*)q, (const T*)k, (const T*)v, (T*)out, lse, (T*)rest, part, ml);
    });
    if (w.shares > 1)
      attn_join_kernel<T><<<dim3((unsigned)(Tq * Hq)), 256, 0, s>>>(
          part, ml, w.shares, (int)Hq, Tq, (int)D, (T*)out, lse, (T*)rest);
  });
  return check_launch("attention_fwd");
}
