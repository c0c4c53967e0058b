// nn_common.hpp -- what the transformer operators (layer norm, packed
// attention, gated projection) share: element types, wave sums, the sequences
// of a packed batch.
//
// Elements are float, half or bfloat16; every product is summed in float and
// an output is rounded to its type once.
#pragma once

#include <initializer_list>

#include "tpo_common.hpp"

namespace tpo {

typedef __bf16 bf16_t;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// Values that are loaded and stored at once and begin at any element: the memory
// takes 16-byte accesses there too.
template <typename T, int PER>
struct __attribute__((packed, aligned(sizeof(T)))) Piece {
  T v[PER];
};

// Calls f with a value of the element type of `dtype`; false for another code.
template <typename F>
inline bool with_element(int dtype, F&& f) {
  switch (dtype) {
    case TPO_F32: f(float()); return true;
    case TPO_F16: f(half_t()); return true;
    case TPO_BF16: f(bf16_t()); return true;
    default: return false;
  }
}
// An error where one of the arrays that a call reads or writes is missing.
inline int all_there(const char* op, std::initializer_list<const void*> arrays) {
  for (const void* p : arrays)
    if (!p) return set_error(TPO_ERR_ARG, "%s: an array is NULL", op);
  return TPO_OK;
}
inline int64_t element_bytes(int dtype) { return dtype == TPO_F32 ? 4 : 2; }
inline int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Sequences of a packed batch of T rows.  Sequence b has the rows
// offsets[b] .. offsets[b + 1], of which the first lengths[b] are in use (all
// of them without lengths).  Whatever the arrays hold, the bounds stay inside
// [0, T).  The rows before offsets[0] and from offsets[B] on count as two more
// sequences without rows in use, so that every row of the batch belongs to one:
// sequence 0 of B + 2 is the rows before, 1 .. B the batch's, B + 1 those after.
struct Sequences {
  const int64_t* offsets;
  const int64_t* lengths;
  int64_t T;
  int B;

  __device__ __forceinline__ int64_t start(int s) const {
    if (s <= 0) return 0;
    if (s >= B + 2) return T;
    const int64_t o = offsets[s - 1];
    return o < 0 ? 0 : (o > T ? T : o);
  }
  // rows of sequence s, and how many of them are in use
  __device__ __forceinline__ int64_t room(int s) const {
    const int64_t n = start(s + 1) - start(s);
    return n < 0 ? 0 : n;
  }
  __device__ __forceinline__ int64_t used(int s) const {
    if (s <= 0 || s >= B + 1) return 0;
    const int64_t n = room(s);
    if (!lengths) return n;
    const int64_t l = lengths[s - 1];
    return l < 0 ? 0 : (l > n ? n : l);
  }
};

}  // namespace tpo
