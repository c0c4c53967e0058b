// gemm_tile.hpp -- the matrix-core product that the gated projection's kernels
// share: a workgroup's tile of A B^T, A (rows, n) and B (cols, n), both with
// the summed axis contiguous.
//
// Four waves hold BM x BN sums in registers, a quarter (BM/2 x BN/2) each, as
// 32 x 32 tiles.  The operands pass through LDS in slabs of 128 bytes of every
// row (64 half or 32 float values), two slabs deep: while a slab is multiplied
// the next is on its way from memory, written into LDS by the loads themselves.
// A slab's row is eight chunks of 16 bytes, chunk c at place c ^ (row % 8), so
// that the eight lanes of a 16-byte LDS read that go together (eight rows, one
// chunk) touch all banks once.
//
// Per slab a wave reads (BM + BN) / 2 rows of LDS for BM BN / 4 sums: at 256 x
// 256 the reads and the slab's own write fill 1536 of the 2048 cycles that its
// matrix instructions take, at 128 x 128 all of them; so the large tile is used
// wherever there are enough tiles.
#pragma once

#include <type_traits>

#include "nn_common.hpp"

namespace tpo {

typedef __attribute__((address_space(3))) void lds_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// 16 bytes of a row, as the matrix instructions take them.
template <typename T> struct Chunk;
template <> struct Chunk<float> { typedef f32x4 V; };
template <> struct Chunk<half_t> { typedef f16x8 V; };
template <> struct Chunk<bf16_t> { typedef bf16x8 V; };

// acc += A B over two chunks of the summed axis: lane l gives row (column) l %
// 32 and chunk l / 32 of both; it receives column l % 32, rows 8 (v / 4) +
// 4 (l / 32) + v % 4.
__device__ __forceinline__ void mma(f32x16& acc, bf16x8 a, bf16x8 b) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& acc, f16x8 a, f16x8 b) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
}
// float: 32x32x2, the k of step j being value j of both chunks
__device__ __forceinline__ void mma(f32x16& acc, f32x4 a, f32x4 b) {
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], acc, 0, 0, 0);
}

constexpr int SLAB = 128;          // bytes of a row in a slab
constexpr int NOWHERE = (int)0x80000000;  // beyond every buffer: such a load gives 0

// Rows of an operand: a pointer, the row's length in bytes, the number of rows.
struct Rows {
  const char* p;
  int64_t pitch;  // bytes from row to row, a multiple of 16
  int64_t rows;
};

// A wave's quarter of the ROWS x SLAB bytes of LDS that hold an operand's slab:
// ROWS / 4 rows from row0 on (its own, not the workgroup's).  Rows past the end
// and bytes past `bytes` (a multiple of 16) become 0.  A load covers 8 rows: a
// lane's place among them is one offset, the rows' and the slab's are scalar;
// the buffer's bound, checked against the sum of both, ends the rows.
template <int ROWS>
struct Loader {
  static constexpr int N = ROWS / 32;  // loads a wave
  int off, chunk, step;
  __amdgpu_buffer_rsrc_t rsrc;

  __device__ __forceinline__ Loader(const Rows& m, int64_t row0) {
    const int l = lane_id();
    int64_t n = m.rows - row0;
    n = n < 0 ? 0 : (n > ROWS / 4 ? ROWS / 4 : n);
    rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(m.p + (n > 0 ? row0 * m.pitch : 0)), 0,
                                             (int)(n * m.pitch), 0x00027000);
    chunk = ((l & 7) ^ (l >> 3)) << 4;
    off = (l >> 3) * (int)m.pitch + chunk;
    step = 8 * (int)m.pitch;
  }
  // bytes k .. k + SLAB of the rows into the operand's place in LDS
  __device__ __forceinline__ void load(char* lds, int k, int bytes) const {
    const int w = wave_id();
    const int at = k + chunk < bytes ? off : NOWHERE;
#pragma unroll
    for (int j = 0; j < N; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_t*)(lds + (w * N + j) * 1024), 16, at,
                                               k + j * step, 0, 0);
  }
};

// A wave's operands of two chunks (of a slab's eight) of the summed axis.
template <typename T, int TM, int TN>
struct Operands {
  typename Chunk<T>::V x[TM], y[TN];

  // chunks 2 s and 2 s + 1; row0, col0: the wave's first row and column
  __device__ __forceinline__ void read(const char* a, const char* b, int row0, int col0, int s) {
    typedef typename Chunk<T>::V V;
    const int l = lane_id(), r = l & 31, h = l >> 5;
    const int at = (((2 * s + h) ^ (r & 7)) << 4) + r * SLAB;
#pragma unroll
    for (int i = 0; i < TM; ++i) x[i] = *(const V*)(a + at + (row0 + 32 * i) * SLAB);
#pragma unroll
    for (int j = 0; j < TN; ++j) y[j] = *(const V*)(b + at + (col0 + 32 * j) * SLAB);
    __builtin_amdgcn_sched_barrier(0);
  }
  __device__ __forceinline__ void multiply(f32x16 (&acc)[TM][TN]) const {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) mma(acc[i][j], x[i], y[j]);
    __builtin_amdgcn_sched_barrier(0);
  }
};

// A slab's products while the next slab (from byte k) loads into the other
// half of LDS.  Operands are read one step ahead of the products that take
// them: u holds the slab before's last ones, and this slab's at the end, so
// that the matrix cores are busy while the first reads of a slab are under way.
// (That the halves are apart is what `restrict` says: a read need not wait for
// the loads into the other one.)
template <typename T, int BM, int BN>
__device__ __forceinline__ void slab_step(const char* __restrict__ cur, char* __restrict__ nxt,
                                          const Loader<BM>& la, const Loader<BN>& lb, int k,
                                          int bytes, int row0, int col0,
                                          Operands<T, BM / 64, BN / 64>& u,
                                          f32x16 (&acc)[BM / 64][BN / 64]) {
  const char* b = cur + BM * SLAB;
  Operands<T, BM / 64, BN / 64> t;
  la.load(nxt, k, bytes);
  lb.load(nxt + BM * SLAB, k, bytes);
  t.read(cur, b, row0, col0, 0);
  u.multiply(acc);
  u.read(cur, b, row0, col0, 1);
  t.multiply(acc);
  t.read(cur, b, row0, col0, 2);
  u.multiply(acc);
  u.read(cur, b, row0, col0, 3);
  t.multiply(acc);
}

template <int BM, int BN>
struct TileLds {
  __attribute__((aligned(1024))) char slab[2][(BM + BN) * SLAB];
};

// The sums over bytes k0 .. k1 of the summed axis; wave w's quarter begins at
// row (w / 2) BM / 2, column (w % 2) BN / 2 of the tile.
template <typename T, int BM, int BN>
__device__ __forceinline__ void gemm_tile(TileLds<BM, BN>& s, const Loader<BM>& la,
                                          const Loader<BN>& lb, int k0, int k1,
                                          f32x16 (&acc)[BM / 64][BN / 64]) {
  const int w = wave_id(), row0 = (w >> 1) * (BM / 2), col0 = (w & 1) * (BN / 2);
#pragma unroll
  for (int i = 0; i < BM / 64; ++i)
#pragma unroll
    for (int j = 0; j < BN / 64; ++j) acc[i][j] = f32x16{};
  if (k0 >= k1) return;
  la.load(s.slab[0], k0, k1);
  lb.load(s.slab[0] + BM * SLAB, k0, k1);
  Operands<T, BM / 64, BN / 64> u = {};  // nothing before the first slab
  int half = 0;
  for (int k = k0; k < k1; k += SLAB) {
    // every wave's loads of the slab have landed, and every wave's reads of the
    // other half have ended
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    slab_step<T, BM, BN>(s.slab[half], s.slab[half ^ 1], la, lb, k + SLAB, k1, row0, col0, u,
                         acc);
    half ^= 1;
  }
  u.multiply(acc);
}

}  // namespace tpo
