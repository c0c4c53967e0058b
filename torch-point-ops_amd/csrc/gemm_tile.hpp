// gemm_tile.hpp -- the matrix-core product that the gated projection's kernels
// share: a workgroup's BM x BN tile of A B^T, with float sums in registers.
//
// Four waves hold a quarter (BM/2 x BN/2) of the sums each, as 32 x 32 tiles.
// The operands pass through LDS in slabs of 128 bytes of the summed axis (64
// half or 32 float values), two slabs deep: while a slab is multiplied the next
// is on its way from memory, written into LDS by the loads themselves.  An
// operand comes in either of two layouts, so that no matrix is ever turned
// round in memory:
//   by rows (RowLoader): the summed axis contiguous.  A slab's row is eight (or
//     four) chunks of 16 bytes, which change places with the row so that the
//     sixteen lanes of a 16-byte LDS read that go together (sixteen rows, one
//     chunk) touch all 64 banks once.
//   by columns (ColLoader): the other axis contiguous, a slab is 64 (32) rows
//     of BM values.  Half operands are read with the transposing LDS read (four
//     summed values of one column a lane), float ones value by value; chunks
//     change places so that the four (two) rows read together lie in different
//     banks.
//
// Measured (rocprofv3, 8192 x 2048 x 8192 gelu): LDS 25 % busy, no bank
// conflicts to speak of, the matrix cores 50 - 60 % busy at the 1.8 - 1.9 GHz
// that the card's power leaves at that load.
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

// An operand by rows: R of the matrix's rows, SLAB bytes of each a slab.  Wave w
// loads R / 4 of them, from its own row0 on.  A load covers 1024 / SLAB rows: a
// lane's place among them is one offset, the rows' and the slab's are scalar;
// the buffer's bound, checked against the sum of both, ends the rows.
template <typename T, int R, int SLAB>
struct RowLoader {
  static constexpr int CPR = SLAB / 16, RPL = 64 / CPR, N = R / 4 / RPL;
  // chunk c of row r is at place c ^ swap(r)
  static __device__ __forceinline__ constexpr int swap(int r) {
    return SLAB == 128 ? r >> 1 & 7 : r >> 2 & 3;
  }
  int off, chunk, step, bytes;
  __amdgpu_buffer_rsrc_t rsrc;

  __device__ __forceinline__ RowLoader(const Matrix& m, int64_t row0) {
    const int l = lane_id();
    int64_t n = m.rows - row0;
    n = n < 0 ? 0 : (n > R / 4 ? R / 4 : n);
    rsrc = buffer(m.p + (n > 0 ? row0 * m.pitch : 0), (int)(n * m.pitch));
    chunk = ((l % CPR) ^ swap(l / CPR)) << 4;  // of the loads from rows 0, 16, ..
    off = (l / CPR) * (int)m.pitch;
    step = RPL * (int)m.pitch;
    bytes = (int)m.bytes;
  }
  // a slab's loads, one after another
  struct Slab {
    __amdgpu_buffer_rsrc_t rsrc;
    int at[2], k, step;
    __device__ __forceinline__ void load(char* lds, int j) const {
      load_lds(rsrc, lds + (wave_id() * N + j) * 1024, at[SLAB == 128 ? j & 1 : 0], k + j * step);
    }
  };
  __device__ __forceinline__ Slab slab(int n) const {
    const int k = n * SLAB;
    // (rows 8, 24, ..: with eight rows a load, bit 2 of the places turns)
    return Slab{rsrc,
                {k + chunk < bytes ? off + chunk : NOWHERE,
                 k + (chunk ^ 64) < bytes ? off + (chunk ^ 64) : NOWHERE},
                k,
                step};
  }
  // rows row0 + l % 32, chunk 2 s + l / 32 of a slab
  static __device__ __forceinline__ typename Chunk<T>::V read(const char* lds, int row0, int s) {
    const int l = lane_id(), r = l & 31, h = l >> 5;
    return *(const typename Chunk<T>::V*)(lds + (((2 * s + h) ^ swap(r)) << 4) + (row0 + r) * SLAB);
  }
};

// An operand by columns: R columns from col0 (a multiple of R / 2) on, the
// matrix's rows being the summed axis.
template <typename T, int R, int SLAB>
struct ColLoader {
  static constexpr int Z = sizeof(T), PITCH = R * Z, K = SLAB / Z;
  static constexpr int N = R * SLAB / 4096;   // loads a wave, 1 KB each
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
    const int l = lane_id(), r = l / CPR;
    const int c = (l % CPR) ^ swap(r) ^ swap(wave_id() * (K / 4));
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
  struct Slab {
    __amdgpu_buffer_rsrc_t rsrc;
    int off[2], step;
    __device__ __forceinline__ void load(char* lds, int j) const {
      const int i = wave_id() * N + j;
      load_lds(rsrc, lds + i * 1024, off[swap(j * RPL) != 0], i * step);
    }
  };
  __device__ __forceinline__ Slab slab(int n) const { return slab_of(p, (int64_t)n * K); }
  __device__ __forceinline__ Slab slab_of(const char* from, int64_t row) const {
    const int64_t left = rows - row;
    // (said to be uniform: what a vector instruction clamps would make each load a loop)
    const int n = __builtin_amdgcn_readfirstlane(left < 0 ? 0 : (left > K ? K : (int)left));
    return Slab{buffer(from + (n > 0 ? row * pitch : 0), n * (int)pitch), {off[0], off[1]}, step};
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
template <typename T, int R, int SLAB>
struct PairLoader {
  typedef ColLoader<T, R, SLAB> L;
  static constexpr int N = L::N;
  L one;
  const char* second;
  int slabs;
  __device__ __forceinline__ PairLoader(const Matrix& m, const char* p2, int slabs, int64_t col0)
      : one(m, col0), second(p2 + col0 * sizeof(T)), slabs(slabs) {}
  __device__ __forceinline__ typename L::Slab slab(int n) const {
    const bool up = n >= slabs;
    return one.slab_of(up ? second : one.p, (int64_t)(up ? n - slabs : n) * L::K);
  }
  static __device__ __forceinline__ typename Chunk<T>::V read(const char* lds, int row0, int s) {
    return L::read(lds, row0, s);
  }
};

// A wave's operands of two chunks of the summed axis.
template <typename T, typename LA, typename LB, int TM, int TN>
struct Operands {
  typename Chunk<T>::V x[TM], y[TN];

  // operand i (the columns' first) of chunks 2 s and 2 s + 1; row0, col0: the
  // wave's first row and column
  __device__ __forceinline__ void read(const char* a, const char* b, int row0, int col0, int s,
                                       int i) {
    if (i < TN)
      y[i] = LB::read(b, col0 + 32 * i, s);
    else
      x[i - TN] = LA::read(a, row0 + 32 * (i - TN), s);
  }
};

// A slab's products while another slab loads into a part of LDS that no wave
// reads.  Operands are read one step ahead of the products that take them: u
// holds the slab before's last ones, and this slab's at the end, so that the
// matrix cores are busy while the first reads of a slab are under way.  SPREAD:
// reads and loads go between the matrix instructions; a wave issues in order,
// and a row of loads that waits for its turn at the memory pipe keeps its
// products waiting as well (where other waves' fill in, the row is quicker: 276
// against 318 us for a product of 275 GFLOP in 128 x 128 tiles).  That the two parts of
// LDS are apart is what `restrict` says: a read need not wait for the loads.
template <typename T, int BM, int SLAB, bool SPREAD, typename LA, typename LB, int TM, int TN>
__device__ __forceinline__ void slab_step(const char* __restrict__ cur, char* __restrict__ nxt,
                                          const LA& la, const LB& lb, int next, int row0, int col0,
                                          Operands<T, LA, LB, TM, TN>& u,
                                          f32x16 (&acc)[TM][TN]) {
  constexpr int STEPS = SLAB / 32, Q = TM * TN, READS = TM + TN, LOADS = LA::N + LB::N;
  const char* b = cur + BM * SLAB;
  const auto sa = la.slab(next);
  const auto sb = lb.slab(next);
  Operands<T, LA, LB, TM, TN> t;
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    Operands<T, LA, LB, TM, TN>& now = s % 2 ? t : u;
    Operands<T, LA, LB, TM, TN>& then = s % 2 ? u : t;
    if (!SPREAD) {
      if (s == 0) {
#pragma unroll
        for (int i = 0; i < LA::N; ++i) sa.load(nxt, i);
#pragma unroll
        for (int i = 0; i < LB::N; ++i) sb.load(nxt + BM * SLAB, i);
      }
#pragma unroll
      for (int i = 0; i < READS; ++i) then.read(cur, b, row0, col0, s, i);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (SPREAD) {
#pragma unroll
        for (int i = q * READS / Q; i < (q + 1) * READS / Q; ++i)
          then.read(cur, b, row0, col0, s, i);
#pragma unroll
        for (int i = (s * Q + q) * LOADS / (STEPS * Q); i < (s * Q + q + 1) * LOADS / (STEPS * Q);
             ++i)
          if (i < LA::N)
            sa.load(nxt, i);
          else
            sb.load(nxt + BM * SLAB, i - LA::N);
      }
      mma(acc[q / TN][q % TN], now.x[q / TN], now.y[q % TN]);
      if (SPREAD) __builtin_amdgcn_sched_barrier(0);
    }
    if (!SPREAD) __builtin_amdgcn_sched_barrier(0);
  }
}

// The LDS of a tile: slabs of SLAB bytes of the summed axis, DEPTH of them.
template <int BM, int BN, int SLAB_, int DEPTH_, bool SPREAD_>
struct alignas(1024) TileLds {
  static constexpr int SLAB = SLAB_, DEPTH = DEPTH_;
  static constexpr bool SPREAD = SPREAD_;
  char slab[DEPTH][(BM + BN) * SLAB];
};

// Waits until at most n of the wave's loads are under way and its LDS reads have
// ended, then for the workgroup's other waves.
template <int n>
__device__ __forceinline__ void wait_loads_and_meet() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((n & 15) | (n >> 4) << 14 | 0x70);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// The sums over slabs s0 .. s1 of the summed axis; wave w's quarter begins at
// row (w / 2) BM / 2, column (w % 2) BN / 2 of the tile.  Slabs after the last
// one that are loaded are not used.  LDS is free for other use afterwards.
template <typename T, int BM, int BN, typename Lds, typename LA, typename LB>
__device__ __forceinline__ void gemm_tile(Lds& lds, const LA& la, const LB& lb, int s0, int s1,
                                          f32x16 (&acc)[BM / 64][BN / 64]) {
  constexpr int SLAB = Lds::SLAB, DEPTH = Lds::DEPTH;
  const int w = wave_id(), row0 = (w >> 1) * (BM / 2), col0 = (w & 1) * (BN / 2);
#pragma unroll
  for (int i = 0; i < BM / 64; ++i)
#pragma unroll
    for (int j = 0; j < BN / 64; ++j) acc[i][j] = f32x16{};
  if (s0 >= s1) return;
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) {
    const auto sa = la.slab(s0 + d);
    const auto sb = lb.slab(s0 + d);
#pragma unroll
    for (int j = 0; j < LA::N; ++j) sa.load(lds.slab[d], j);
#pragma unroll
    for (int j = 0; j < LB::N; ++j) sb.load(lds.slab[d] + BM * SLAB, j);
  }
  Operands<T, LA, LB, BM / 64, BN / 64> u = {};  // nothing before the first slab
  int at = 0;
  for (int k = s0; k < s1; ++k) {
    // the slab has landed (DEPTH - 2 younger ones may be on their way), and every
    // wave has read the last of the slab before it, whose place is loaded next
    wait_loads_and_meet<(DEPTH - 2) * (LA::N + LB::N)>();
    const int free = at == 0 ? DEPTH - 1 : at - 1;
    slab_step<T, BM, SLAB, Lds::SPREAD>(lds.slab[at], lds.slab[free], la, lb, k + DEPTH - 1, row0,
                                        col0, u, acc);
    at = at + 1 == DEPTH ? 0 : at + 1;
  }
#pragma unroll
  for (int i = 0; i < BM / 64; ++i)
#pragma unroll
    for (int j = 0; j < BN / 64; ++j) mma(acc[i][j], u.x[i], u.y[j]);
  wait_loads_and_meet<0>();
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
  // `cols`.  Rows may begin at any element: only what is left of a row under 16 bytes
  // goes value by value (2240 x 91 -> 7877 in bfloat16: 33 us with single values, 27).
  __device__ __forceinline__ void store(T* out, int64_t pitch, int64_t row0, int64_t rows,
                                        int64_t col0, int64_t cols) const {
    wait();
#pragma unroll
    for (int i = 0; i < 32 * CHUNKS; i += 64) {
      const int r = (i + lane_id()) / CHUNKS, c = (i + lane_id()) % CHUNKS * PER;
      if (row0 + r >= rows) continue;
      const T* from = (const T*)(lds + r * PITCH) + c;
      T* to = out + (row0 + r) * pitch + col0 + c;
      if (col0 + c + PER <= cols)
        *(Piece<T, PER>*)to = *(const Piece<T, PER>*)__builtin_assume_aligned(from, 16);
      else
        for (int e = 0; col0 + c + e < cols; ++e) to[e] = from[e];
    }
    wait();
  }
  __device__ __forceinline__ void load(const T* in, int64_t pitch, int64_t row0, int64_t rows,
                                       int64_t col0, int64_t cols) const {
#pragma unroll
    for (int i = 0; i < 32 * CHUNKS; i += 64) {
      const int r = (i + lane_id()) / CHUNKS, c = (i + lane_id()) % CHUNKS * PER;
      const T* from = in + (row0 + r) * pitch + col0 + c;
      Piece<T, PER> v = {};
      if (row0 + r < rows) {
        if (col0 + c + PER <= cols)
          v = *(const Piece<T, PER>*)from;
        else
#pragma unroll
          for (int e = 0; e < PER; ++e)
            if (col0 + c + e < cols) v.v[e] = from[e];
      }
      *(f32x4*)((T*)(lds + r * PITCH) + c) = __builtin_bit_cast(f32x4, v);
    }
    wait();
  }
};

template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};

}  // namespace tpo
