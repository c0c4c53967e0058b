// cache.hpp -- keys and values of many sequences in pages of 8-bit codes, laid out for the
// matrix instructions.
//
// A page holds `page` tokens of every key head, in blocks of 32 tokens.  Dr is the head size
// rounded up to 16.
//   keys    (pages, Hk, page / 32, Dr / 16, 32, 16)  16 values of a token lie together
//   values  (pages, Hk, page / 32, Dr, 32)           32 tokens of a value lie together
//   key_scales, value_scales (pages, Hk) float
// A block has 32 Dr bytes in both, so that a wave that reads one goes straight through them:
// sixteen bytes a lane, 1 KB a load, and what a lane gets is what the products sum over (a
// key's values; a value's tokens).  Codes are e4m3 (448 the largest, no infinities); a value is
// its code times the scale of its page and head.
#pragma once

#include "nn_common.hpp"

namespace tpo {

constexpr int CACHE_BLOCK = 32;   // tokens of a block
constexpr int CACHE_PAGE = 256;   // the largest page
constexpr int CACHE_DMAX = 128;

struct Cache {
  uint8_t *keys, *values;
  float *key_scales, *value_scales;
  const int32_t* table;    // (B, M): the pages of each sequence; outside of [0, pages): none
  const int64_t* lengths;  // (B): tokens of each sequence, those that a call brings included
  int64_t pages;
  int M, page, Hk, chunks;  // chunks: Dr / 16

  __device__ __forceinline__ int64_t block(int64_t p, int head, int i) const {
    return ((p * Hk + head) * (page / CACHE_BLOCK) + i) * (CACHE_BLOCK * 16 * chunks);
  }
  // what the table has room for is all that a length can count
  __device__ __forceinline__ int length(int64_t n) const {
    const int64_t room = (int64_t)M * page;
    return n < 0 ? 0 : (int)(n > room ? room : n);
  }
  // the number of page i of sequence b; -1: none
  __host__ __device__ __forceinline__ int page_of(int b, int i) const {
    if (i < 0 || i >= M) return -1;
    const int p = table[(int64_t)b * M + i];
    return p >= 0 && p < pages ? p : -1;
  }
};

// A sequence of a call's rows, and what the cache holds of it.
struct CacheRows {
  int64_t first;           // its first row
  int room, used, length;  // rows, those in use, and tokens in the cache (with them)
  int b;                   // -1: the rows before the first sequence or behind the last
  int64_t place;           // of its first in the order asked for
};
// The last sequence whose first place is at or before `place`; first(start, s): the first place
// of sequence s (0 and B + 1 being the rows before and behind), not decreasing.  Up to 126
// sequences: each lane has one or two of them, and one trip to memory brings all that is needed
// (64 sequences' new tokens: 11.0 us, by four trips 11.4).
template <typename F>
__device__ __forceinline__ CacheRows cache_rows(const Sequences& sq, const Cache& c, int64_t place,
                                                const F& first) {
  const int l = lane_id(), B = sq.B;
  CacheRows r;
  if (B <= 126) {
    int64_t o[2], p[2], n[2], kept[2];
    auto load = [&](int y) {
      const int k = l + 64 * y;  // sequence k of B + 2
      const int i = k < 1 ? 0 : (k - 1 < B ? k - 1 : B), j = k < B ? k : B;
      const bool own = k >= 1 && k <= B;
      o[y] = sq.offsets[i];
      p[y] = sq.offsets[j];
      n[y] = own ? (sq.lengths ? sq.lengths[k - 1] : sq.T) : 0;
      kept[y] = own ? c.lengths[k - 1] : 0;
    };
    load(0);
    if (B > 62) load(1);
    const int T = (int)sq.T;
    auto inside = [](int64_t v, int most) { return v < 0 ? 0 : (v > most ? most : (int)v); };
    auto pick = [&](int y) {
      const int k = l + 64 * y;
      const int start = k < 1 ? 0 : (k > B + 1 ? T : inside(o[y], T));
      const int next = k > B ? T : inside(p[y], T);
      const int room = next > start ? next - start : 0;
      const int used = inside(n[y], room), length = c.length(kept[y]);
      const uint64_t m = __builtin_amdgcn_ballot_w64(k < B + 2 && first(start, k) <= place);
      if (y > 0 && m == 0) return;
      const int at = m ? 63 - __builtin_clzll(m) : 0, s = at + 64 * y;
      r.first = __builtin_amdgcn_readlane(start, at);
      r.room = __builtin_amdgcn_readlane(room, at);
      r.used = __builtin_amdgcn_readlane(used, at);
      r.length = __builtin_amdgcn_readlane(length, at);
      r.b = s >= 1 && s <= B ? s - 1 : -1;
      r.place = first(r.first, s);
    };
    pick(0);
    if (B > 62) pick(1);
    return r;
  }
  int lo = 0, n = B + 2;  // among lo .. lo + n - 1: 64 guesses a step
  while (n > 1) {
    const int step = (n + 63) >> 6, i = lo + l * step;
    const bool at = i < lo + n && first(sq.start(i), i) <= place;
    const uint64_t m = __builtin_amdgcn_ballot_w64(at);
    const int top = m ? 63 - __builtin_clzll(m) : 0;
    const int rest = n - top * step;
    lo += top * step;
    n = rest < step ? rest : step;
  }
  const int s = __builtin_amdgcn_readfirstlane(lo);
  r.first = __builtin_amdgcn_readfirstlane((int)sq.start(s));
  r.room = __builtin_amdgcn_readfirstlane((int)sq.room(s));
  r.used = __builtin_amdgcn_readfirstlane((int)sq.used(s));
  r.b = s >= 1 && s <= B ? s - 1 : -1;
  r.length = r.b < 0 ? 0 : __builtin_amdgcn_readfirstlane(c.length(c.lengths[r.b]));
  r.place = first(r.first, s);
  return r;
}

// Checks the sizes of a call's cache.
int cache_check(const char* op, int64_t pages, int64_t Hk, int64_t page, int64_t Dr, int64_t B,
                int64_t M, int64_t D);
// The checked arguments of a call as the kernels take them.
Cache cache_args(const void* keys, const void* values, const float* key_scales,
                 const float* value_scales, const int32_t* table, const int64_t* lengths,
                 int64_t pages, int64_t Hk, int64_t page, int64_t D, int64_t M);

}  // namespace tpo
