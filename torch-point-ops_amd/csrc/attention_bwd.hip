// attention_bwd.hip -- backward of softmax attention over packed sequences.
//   dV = P^T dO, dP = dO V^T, dS = P (dP - sum_d dO O),
//   dQ = scale dS K, dK = scale dS^T Q
#include "attention.hpp"

namespace tpo {

// The sequence (1 .. B, or 0 and B + 1) that row t belongs to.
__device__ __forceinline__ int attn_row_sequence(const Sequences& s, int64_t t) {
  int lo = 0, hi = s.B + 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s.start(mid) <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ void attn_load(const T* p, int D, float (&x)[2]) {
  const int l = lane_id();
  x[0] = l < D ? (float)p[l] : 0.f;
  x[1] = l + 64 < D ? (float)p[l + 64] : 0.f;
}
template <typename T>
__device__ __forceinline__ void attn_store(T* p, int D, const float (&x)[2]) {
  const int l = lane_id();
  if (l < D) p[l] = (T)x[0];
  if (l + 64 < D) p[l + 64] = (T)x[1];
}
__device__ __forceinline__ float attn_dot(const float (&a)[2], const float (&b)[2]) {
  return wave_sum(a[0] * b[0] + a[1] * b[1]);
}

// dQ: one wave a query row and head.
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_q_kernel(
    AttnArgs a, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
    const T* __restrict__ o, const T* __restrict__ go, const float* __restrict__ lse,
    float* __restrict__ delta, T* __restrict__ gq) {
  const int64_t w = (int64_t)blockIdx.x * 4 + wave_id();
  const int64_t t = w / a.Hq;
  const int h = (int)(w % a.Hq);
  if (t >= a.sq.T) return;
  const int s = attn_row_sequence(a.sq, t);
  const int64_t Lq = a.sq.used(s), Lk = a.sk.used(s), i = t - a.sq.start(s), k0 = a.sk.start(s);
  int64_t n = i < Lq ? Lk : 0;
  if (a.causal && i + Lk - Lq + 1 < n) n = i + Lk - Lq + 1;
  const int hk = h / (a.Hq / a.Hk);
  const float m = lse[h * a.sq.T + t];
  if (m == -__builtin_inff()) n = 0;
  float x[2], y[2], z[2], g[2], acc[2] = {0.f, 0.f};
  attn_load(o + (t * a.Hq + h) * a.D, a.D, x);
  attn_load(go + (t * a.Hq + h) * a.D, a.D, g);
  const float d = n > 0 ? attn_dot(x, g) : 0.f;
  if (lane_id() == 0) delta[h * a.sq.T + t] = d;
  attn_load(q + t * a.q_row + h * a.q_head, a.D, x);
  for (int64_t j = 0; j < n; ++j) {
    attn_load(k + (k0 + j) * a.k_row + hk * a.k_head, a.D, y);
    attn_load(v + (k0 + j) * a.v_row + hk * a.v_head, a.D, z);
    const float p = expf(attn_dot(x, y) * a.scale - m);
    const float e = p * (attn_dot(g, z) - d) * a.scale;
    acc[0] += e * y[0];
    acc[1] += e * y[1];
  }
  attn_store(gq + (t * a.Hq + h) * a.D, a.D, acc);
}

// dK and dV: one wave a key row and key head.
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_kv_kernel(
    AttnArgs a, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
    const T* __restrict__ go, const float* __restrict__ lse, const float* __restrict__ delta,
    T* __restrict__ gk, T* __restrict__ gv) {
  const int64_t w = (int64_t)blockIdx.x * 4 + wave_id();
  const int64_t t = w / a.Hk;
  const int hk = (int)(w % a.Hk);
  if (t >= a.sk.T) return;
  const int s = attn_row_sequence(a.sk, t);
  const int64_t Lq = a.sq.used(s), Lk = a.sk.used(s), j = t - a.sk.start(s), q0 = a.sq.start(s);
  const int64_t n = j < Lk ? Lq : 0;
  const int64_t first = a.causal && j - (Lk - Lq) > 0 ? j - (Lk - Lq) : 0;
  const int G = a.Hq / a.Hk;
  float x[2], y[2], z[2], g[2], ak[2] = {0.f, 0.f}, av[2] = {0.f, 0.f};
  attn_load(k + t * a.k_row + hk * a.k_head, a.D, y);
  attn_load(v + t * a.v_row + hk * a.v_head, a.D, z);
  for (int h = hk * G; h < hk * G + G; ++h)
    for (int64_t i = first; i < n; ++i) {
      const int64_t r = q0 + i;
      const float m = lse[h * a.sq.T + r];
      if (m == -__builtin_inff()) continue;
      attn_load(q + r * a.q_row + h * a.q_head, a.D, x);
      attn_load(go + (r * a.Hq + h) * a.D, a.D, g);
      const float p = expf(attn_dot(x, y) * a.scale - m);
      const float e = p * (attn_dot(g, z) - delta[h * a.sq.T + r]) * a.scale;
      ak[0] += e * x[0];
      ak[1] += e * x[1];
      av[0] += p * g[0];
      av[1] += p * g[1];
    }
  attn_store(gk + (t * a.Hk + hk) * a.D, a.D, ak);
  attn_store(gv + (t * a.Hk + hk) * a.D, a.D, av);
}

}  // namespace tpo

using namespace tpo;

extern "C" int64_t tpo_attention_bwd_workspace_size(int dtype, int64_t B, int64_t Tq, int64_t Tk,
                                                    int64_t Hq, int64_t Hk, int64_t D) {
  if (attn_check("attention_bwd_workspace_size", dtype, B, Tq, Tk, Hq, Hk, D)) return -1;
  return round_up(Tq * Hq * 4, 256);
}

extern "C" int tpo_attention_bwd(int dtype, const void* grad_out, const void* q, const void* k,
                                 const void* v, const void* out, const float* lse,
                                 const int64_t* offsets_q, const int64_t* offsets_k,
                                 const int64_t* lengths_q, const int64_t* lengths_k, int64_t B,
                                 int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D,
                                 int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                                 int64_t v_row, int64_t v_head, int causal, double scale,
                                 void* grad_q, void* grad_k, void* grad_v, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  if (int rc = attn_check("attention_bwd", dtype, B, Tq, Tk, Hq, Hk, D)) return rc;
  const int64_t need = tpo_attention_bwd_workspace_size(dtype, B, Tq, Tk, Hq, Hk, D);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(TPO_ERR_WORKSPACE, "attention_bwd: workspace of %lld bytes needed",
                     (long long)need);
  const AttnArgs a = attn_args(offsets_q, offsets_k, lengths_q, lengths_k, B, Tq, Tk, Hq, Hk, D,
                               q_row, q_head, k_row, k_head, v_row, v_head, causal, scale);
  float* delta = (float*)workspace;
  hipStream_t s = (hipStream_t)stream;
  with_element(dtype, [&](auto t) {
    typedef decltype(t) T;
    if (Tq > 0)
      attn_bwd_q_kernel<T><<<dim3((unsigned)((Tq * Hq + 3) / 4)), 256, 0, s>>>(
          a, (const T*)q, (const T*)k, (const T*)v, (const T*)out, (const T*)grad_out, lse, delta,
          (T*)grad_q);
    if (Tk > 0)
      attn_bwd_kv_kernel<T><<<dim3((unsigned)((Tk * Hk + 3) / 4)), 256, 0, s>>>(
          a, (const T*)q, (const T*)k, (const T*)v, (const T*)grad_out, lse, delta, (T*)grad_k,
          (T*)grad_v);
  });
  return check_launch("attention_bwd");
}
