// gemm_tile.hpp -- the matrix-core product that the gated projection's kernels
// share: a workgroup's BM x BN tile of A B^T, with float sums in registers.
//
// Four waves hold a quarter (BM/2 x BN/2) of the sums each, as 32 x 32 tiles.
// The operands pass through LDS in slabs of 128 bytes of the summed axis (64
// half or 32 float values), two slabs deep: while a slab is multiplied the next
// is on its way from memory, written into LDS by the loads themselves.  An
// operand comes in either of two layouts, so that no matrix is ever turned
// round in memory:
//   by rows (RowLoader): the summed axis contiguous.  A slab's row is eight
//     chunks of 16 bytes, chunk c at place c ^ (row % 8): the eight lanes of a
//     16-byte LDS read that go together (eight rows, one chunk) touch all banks
//     once.
//   by columns (ColLoader): the other axis contiguous, a slab is 64 (32) rows
//     of BM values.  Half operands are read with the transposing LDS read (four
//     summed values of one column a lane), float ones value by value; chunks
//     change places so that the four (two) rows read together lie in different
//     banks.
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
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// 16 bytes of the summed axis, as the matrix instructions take them.
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

constexpr int SLAB = 128;                 // bytes of the summed axis in a slab
constexpr int NOWHERE = (int)0x80000000;  // beyond every buffer: such a load gives 0

// The loads of `bytes` bytes from p; anything beyond reads as 0.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00027000);
}
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t r, char* lds, int lane_off,
                                         int off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_t*)lds, 16, lane_off, off, 0, 0);
}

// A matrix in memory: rows `pitch` bytes apart (a multiple of 16, as p is), each
// with `bytes` bytes in use (rounded up to 16: what is past the values is 0).
struct Matrix {
  const char* p;
  int64_t pitch, rows, bytes;
};

// An operand by rows: R of the matrix's rows.  Wave w loads R / 4 of them, from
// its own row0 on.  A load covers 8 rows: a lane's place among them is one
// offset, the rows' and the slab's are scalar; the buffer's bound, checked
// against the sum of both, ends the rows.
template <typename T, int R>
struct RowLoader {
  static constexpr int N = R / 32;  // loads a wave
  int off, chunk, step, bytes;
  __amdgpu_buffer_rsrc_t rsrc;

  __device__ __forceinline__ RowLoader(const Matrix& m, int64_t row0) {
    const int l = lane_id();
    int64_t n = m.rows - row0;
    n = n < 0 ? 0 : (n > R / 4 ? R / 4 : n);
    rsrc = buffer(m.p + (n > 0 ? row0 * m.pitch : 0), (int)(n * m.pitch));
    chunk = ((l & 7) ^ (l >> 3)) << 4;
    off = (l >> 3) * (int)m.pitch + chunk;
    step = 8 * (int)m.pitch;
    bytes = (int)m.bytes;
  }
  __device__ __forceinline__ void load(char* lds, int slab) const {
    const int w = wave_id(), k = slab * SLAB;
    const int at = k + chunk < bytes ? off : NOWHERE;
#pragma unroll
    for (int j = 0; j < N; ++j) load_lds(rsrc, lds + (w * N + j) * 1024, at, k + j * step);
  }
  // rows row0 + l % 32, chunk 2 s + l / 32 of a slab
  static __device__ __forceinline__ typename Chunk<T>::V read(const char* lds, int row0, int s) {
    const int l = lane_id(), r = l & 31, h = l >> 5;
    return *(const typename Chunk<T>::V*)(lds + (((2 * s + h) ^ (r & 7)) << 4) +
                                          (row0 + r) * SLAB);
  }
};

// An operand by columns: R columns from col0 (a multiple of R / 2) on, the
// matrix's rows being the summed axis.
template <typename T, int R>
struct ColLoader {
  static constexpr int Z = sizeof(T), PITCH = R * Z, K = SLAB / Z;
  static constexpr int N = R / 32;            // loads a wave, 1 KB each
  static constexpr int RPL = 1024 / PITCH;    // rows a load
  static constexpr int CPR = PITCH / 16;      // chunks a row
  // chunk c of row r is at place c ^ swap(r)
  static __device__ __forceinline__ constexpr int swap(int r) {
    return Z == 4 ? ((r >> 2) & 1) << 3 : PITCH == 128 ? ((r >> 1) & 1) << 2 : (r & 3) << 2;
  }
  const char* p;
  int64_t pitch, rows;
  int off[2], step;

  __device__ __forceinline__ ColLoader(const Matrix& m, int64_t col0) {
    const int l = lane_id(), r = l / CPR, c = (l % CPR) ^ swap(r);
    p = m.p + col0 * Z;
    pitch = m.pitch;
    rows = m.rows;
    step = RPL * (int)m.pitch;
#pragma unroll
    for (int v = 0; v < 2; ++v) {  // loads whose rows' places differ by `other`
      const int at = (c ^ (v ? other() : 0)) << 4;
      off[v] = col0 * Z + at < m.bytes ? r * (int)m.pitch + at : NOWHERE;
    }
  }
  static __device__ __forceinline__ constexpr int other() {
    return Z == 4 ? 8 : RPL == 2 ? 8 : 0;
  }
  __device__ __forceinline__ void load(char* lds, int slab) const {
    load_from(p, (int64_t)slab * K, lds);
  }
  __device__ __forceinline__ void load_from(const char* from, int64_t row, char* lds) const {
    const int w = wave_id();
    int64_t n = rows - row;
    n = n < 0 ? 0 : (n > K ? K : n);
    const __amdgpu_buffer_rsrc_t rsrc = buffer(from + (n > 0 ? row * pitch : 0), (int)(n * pitch));
#pragma unroll
    for (int j = 0; j < N; ++j)
      load_lds(rsrc, lds + (w * N + j) * 1024, off[swap(j * RPL) != 0], (w * N + j) * step);
  }
  static __device__ __forceinline__ typename Chunk<T>::V read(const char* lds, int row0, int s) {
    const int l = lane_id();
    if constexpr (Z == 4) {
      const int h = l >> 5;
      const char* at = lds + (8 * s + 4 * h) * PITCH + ((row0 * 4) ^ (128 * h)) + (l & 31) * 4;
      f32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *(const float*)(at + j * PITCH);
      return v;
    } else {
      // 16 lanes give the addresses of 4 rows x 16 columns and receive a column
      // each: rows 8 h .. 8 h + 3 of the step, then the next four
      const int i = l & 15, g = (l >> 4) & 1, h = l >> 5, q = i >> 2;
      const char* at = lds + ((16 * s + 8 * h + q) * PITCH + (swap(q) << 4) + 32 * g + 8 * (i & 3));
      const int turn = row0 * 2;  // a multiple of 64 below PITCH
      typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
      const int a0 = (int)(uintptr_t)(lds_t*)at ^ turn;
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(uintptr_t)a0);
      const i16x4 hi =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(uintptr_t)(a0 + 4 * PITCH));
      return __builtin_bit_cast(typename Chunk<T>::V,
                                __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// Two matrices by columns, one below the other: slabs from `slabs` on are the
// second's.
template <typename T, int R>
struct PairLoader {
  typedef ColLoader<T, R> L;
  static constexpr int N = L::N;
  L one;
  const char* second;
  int slabs;
  __device__ __forceinline__ PairLoader(const Matrix& m, const char* p2, int slabs, int64_t col0)
      : one(m, col0), second(p2 + col0 * sizeof(T)), slabs(slabs) {}
  __device__ __forceinline__ void load(char* lds, int slab) const {
    const bool up = slab >= slabs;
    one.load_from(up ? second : one.p, (int64_t)(up ? slab - slabs : slab) * L::K, lds);
  }
  static __device__ __forceinline__ typename Chunk<T>::V read(const char* lds, int row0, int s) {
    return L::read(lds, row0, s);
  }
};

// A wave's operands of two chunks (of a slab's eight) of the summed axis.
template <typename T, typename LA, typename LB, int TM, int TN>
struct Operands {
  typename Chunk<T>::V x[TM], y[TN];

  // chunks 2 s and 2 s + 1; row0, col0: the wave's first row and column
  __device__ __forceinline__ void read(const char* a, const char* b, int row0, int col0, int s) {
#pragma unroll
    for (int i = 0; i < TM; ++i) x[i] = LA::read(a, row0 + 32 * i, s);
#pragma unroll
    for (int j = 0; j < TN; ++j) y[j] = LB::read(b, col0 + 32 * j, s);
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

// A slab's products while slab `next` loads into the other half of LDS.
// Operands are read one step ahead of the products that take them: u holds the
// slab before's last ones, and this slab's at the end, so that the matrix cores
// are busy while the first reads of a slab are under way.  (That the halves are
// apart is what `restrict` says: a read need not wait for the loads into the
// other one.)
template <typename T, int BM, typename LA, typename LB, int TM, int TN>
__device__ __forceinline__ void slab_step(const char* __restrict__ cur, char* __restrict__ nxt,
                                          const LA& la, const LB& lb, int next, bool more,
                                          int row0, int col0, Operands<T, LA, LB, TM, TN>& u,
                                          f32x16 (&acc)[TM][TN]) {
  const char* b = cur + BM * SLAB;
  Operands<T, LA, LB, TM, TN> t;
  if (more) {
    la.load(nxt, next);
    lb.load(nxt + BM * SLAB, next);
  }
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
struct alignas(1024) TileLds {
  char slab[2][(BM + BN) * SLAB];
};

// The sums over slabs s0 .. s1 of the summed axis; wave w's quarter begins at
// row (w / 2) BM / 2, column (w % 2) BN / 2 of the tile.  LDS is free for other
// use afterwards.
template <typename T, int BM, int BN, typename LA, typename LB>
__device__ __forceinline__ void gemm_tile(TileLds<BM, BN>& s, const LA& la, const LB& lb, int s0,
                                          int s1, f32x16 (&acc)[BM / 64][BN / 64]) {
  const int w = wave_id(), row0 = (w >> 1) * (BM / 2), col0 = (w & 1) * (BN / 2);
#pragma unroll
  for (int i = 0; i < BM / 64; ++i)
#pragma unroll
    for (int j = 0; j < BN / 64; ++j) acc[i][j] = f32x16{};
  if (s0 >= s1) return;
  la.load(s.slab[0], s0);
  lb.load(s.slab[0] + BM * SLAB, s0);
  Operands<T, LA, LB, BM / 64, BN / 64> u = {};  // nothing before the first slab
  int half = 0;
  for (int k = s0; k < s1; ++k) {
    // every wave's loads of the slab have landed, and every wave's reads of the
    // other half have ended
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    slab_step<T, BM>(s.slab[half], s.slab[half ^ 1], la, lb, k + 1, k + 1 < s1, row0, col0, u, acc);
    half ^= 1;
  }
  u.multiply(acc);
  __syncthreads();
}

// A wave's way from its sums to rows in memory.  A 32-column tile of sums lies
// with a column (a row of the output) in each lane, four consecutive values at a
// time; through LDS it becomes rows of W values that 16-byte stores write
// without gaps.  The wave has the LDS to itself.
template <typename T, int W>
struct Rows32 {
  static constexpr int PITCH = W * sizeof(T) + 16;  // a step over the banks each row
  static constexpr int PER = 16 / sizeof(T), CHUNKS = W / PER;
  static constexpr int BYTES = 32 * PITCH;
  char* lds;

  // the four values from `at` of row l % 32
  __device__ __forceinline__ T* four(int at) const {
    return (T*)(lds + (lane_id() & 31) * PITCH) + at;
  }
  __device__ __forceinline__ void wait() const {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  // rows row0 .. row0 + 31 of a matrix with `rows` rows, columns col0 .. col0 + W of
  // `cols`; whole: rows start on 16 bytes and cols is a multiple of 16 bytes
  __device__ __forceinline__ void store(T* out, int64_t pitch, int64_t row0, int64_t rows,
                                        int64_t col0, int64_t cols, bool whole) const {
    wait();
    if (whole) {
#pragma unroll
      for (int i = 0; i < 32 * CHUNKS; i += 64) {
        const int r = (i + lane_id()) / CHUNKS, c = (i + lane_id()) % CHUNKS * PER;
        if (row0 + r < rows && col0 + c < cols)
          *(f32x4*)(out + (row0 + r) * pitch + col0 + c) = *(const f32x4*)((T*)(lds + r * PITCH) + c);
      }
    } else {
      for (int i = 0; i < 32 * W; i += 64) {
        const int r = (i + lane_id()) / W, c = (i + lane_id()) % W;
        if (row0 + r < rows && col0 + c < cols)
          out[(row0 + r) * pitch + col0 + c] = ((T*)(lds + r * PITCH))[c];
      }
    }
    wait();
  }
  __device__ __forceinline__ void load(const T* in, int64_t pitch, int64_t row0, int64_t rows,
                                       int64_t col0, int64_t cols, bool whole) const {
    if (whole) {
#pragma unroll
      for (int i = 0; i < 32 * CHUNKS; i += 64) {
        const int r = (i + lane_id()) / CHUNKS, c = (i + lane_id()) % CHUNKS * PER;
        f32x4 v = {};
        if (row0 + r < rows && col0 + c < cols)
          v = *(const f32x4*)(in + (row0 + r) * pitch + col0 + c);
        *(f32x4*)((T*)(lds + r * PITCH) + c) = v;
      }
    } else {
      for (int i = 0; i < 32 * W; i += 64) {
        const int r = (i + lane_id()) / W, c = (i + lane_id()) % W;
        ((T*)(lds + r * PITCH))[c] =
            row0 + r < rows && col0 + c < cols ? in[(row0 + r) * pitch + col0 + c] : (T)0.f;
      }
    }
    wait();
  }
};

template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};

}  // namespace tpo
