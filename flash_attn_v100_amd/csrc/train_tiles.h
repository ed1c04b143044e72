// Tile building blocks of the kernels that keep 32 rows per wave in registers
// and stream 32-row tiles of two tensors past them (training, scored
// attention): operand types and products, LDS tile layouts and readers, the
// two-stage tile ring, and the slots in which split waves hand over partials.
#pragma once

#include <math.h>

#include "capi_internal.h"
#include "common.h"

namespace fa {
namespace train {

typedef float float8_t __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kRows = 32;                   // rows per wave and per streamed tile
constexpr int kBlockRows = kWaves * kRows;  // rows per workgroup
constexpr float kLn2 = 0.69314718055994531f;

template <typename T>
struct Elem;
template <>
struct Elem<half_t> {
  typedef half8_t frag;
};
template <>
struct Elem<float> {
  typedef float8_t frag;
};

__device__ __forceinline__ float16_t mma(const half8_t& a, const half8_t& b, const float16_t& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float16_t mma(const float8_t& a, const float8_t& b, float16_t c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

template <typename T>
using lds_ptr = __attribute__((address_space(3))) T*;

// LDS tile layout for 32 rows of DP elements.  off(r, c) is the element offset
// of logical (row r, column c); columns move in 8-element groups (c % 8 is
// kept), so 16-byte row reads and 8-byte transposing reads stay contiguous.
template <typename T, int DP>
struct Layout;
template <int DP>
struct Layout<half_t, DP> {  // unpadded, 16-byte chunks XOR-swizzled per row
  static constexpr int LD = DP;
  __device__ static __forceinline__ int off(int r, int c) {
    return r * DP + ((((c >> 3) ^ chunk_swizzle<DP>(r)) << 3) | (c & 7));
  }
};
template <int DP>
struct Layout<float, DP> {  // rows padded by 32 bytes (8 banks apart mod 64)
  static constexpr int LD = DP + 8;
  __device__ static __forceinline__ int off(int r, int c) { return r * LD + c; }
};

// Per-lane LDS operand reads from a tile at LDS byte address `tile`:
//   row(tile, kk)     8 elements of row lane % 32, columns 16 kk + 8 (lane / 32) ..
//   tr(tile, r0, db)  element j = M[r0 + 8 (j / 4) + 4 (lane / 32) + j % 4][32 db + lane % 32]
// (r0 in {0, 16}).  The fp16 reader folds the swizzle into per-lane byte
// offsets once; each read then XORs in the compile-time part of its chunk
// index (tile bases are multiples of the row length, so they have no bits in
// the chunk field).
template <typename T, int DP>
struct Reader;
template <int DP>
struct Reader<half_t, DP> {
  unsigned row_lane, tr_lane;
  __device__ explicit Reader(int lane) {
    const int l32 = lane & 31, hi = lane >> 5, s16 = lane & 15;
    row_lane = static_cast<unsigned>((l32 * DP + ((chunk_swizzle<DP>(l32) ^ hi) * 8)) * 2);
    // source lane s16 of each 16-lane group reads row 4 hi + s16 / 4 (+ r0 + 8 jj),
    // columns 32 db + 16 ((lane >> 4) & 1) + 4 (s16 & 3) .. +4
    const int v_sw = (DP <= 64 ? (((s16 >> 3) & 1) << 2) : ((s16 >> 2) << 2)) | hi;
    const int v_row = 4 * hi + (s16 >> 2);
    tr_lane = static_cast<unsigned>(
        (v_row * DP + (((2 * ((lane >> 4) & 1) + ((s16 & 3) >> 1)) ^ v_sw) * 8) + (s16 & 1) * 4) * 2);
  }
  __device__ __forceinline__ half8_t row(unsigned tile, int kk) const {
    return *lds_at<half8_t>((tile + row_lane) ^ (32 * kk));
  }
  __device__ __forceinline__ half8_t tr(unsigned tile, int r0, int db) const {
    half4_t part[2];
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      const unsigned src = ((tile + tr_lane) ^ (16 * (4 * db ^ 2 * jj))) + (r0 + 8 * jj) * DP * 2;
      const short4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          const_cast<__attribute__((address_space(3))) short4_t*>(lds_at<short4_t>(src)));
      part[jj] = __builtin_bit_cast(half4_t, x);
    }
    return __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }
};
template <int DP>
struct Reader<float, DP> {
  int lane;
  __device__ explicit Reader(int lane_) : lane(lane_) {}
  __device__ __forceinline__ float8_t row(unsigned tile, int kk) const {
    const int off = Layout<float, DP>::off(lane & 31, 16 * kk + 8 * (lane >> 5));
    return *lds_at<float8_t>(tile + off * 4);
  }
  __device__ __forceinline__ float8_t tr(unsigned tile, int r0, int db) const {
    const int hi = lane >> 5;
    const int col = 32 * db + (lane & 31);
    const __attribute__((address_space(3))) float* t = lds_at<float>(tile);
    float8_t f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = t[Layout<float, DP>::off(r0 + 8 * (j >> 2) + 4 * hi + (j & 3), col)];
    return f;
  }
};

// Eight elements of global row `row` (length d) from column `col`, zero past d;
// the vector row modes have 16-byte aligned rows of whole 8-element groups, so
// one vector load serves (kRowFull: d is the padded width).
template <typename T>
__device__ __forceinline__ typename Elem<T>::frag zero_frag() {
  typename Elem<T>::frag f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = static_cast<T>(0.0f);
  return f;
}

template <typename T, int ROWS>
__device__ __forceinline__ typename Elem<T>::frag load_frag(const T* row, int col, int d) {
  typedef typename Elem<T>::frag F;
  if constexpr (ROWS == kRowFull) {
    (void)d;
    return *reinterpret_cast<const F*>(row + col);
  } else if constexpr (ROWS == kRowChunks) {
    return col < d ? *reinterpret_cast<const F*>(row + col) : zero_frag<T>();
  } else {
    F f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (col + j < d) ? row[col + j] : static_cast<T>(0.0f);
    return f;
  }
}

// Operand slice `sl` (accumulator registers 8 sl .. 8 sl + 7) converted to T.
template <typename T>
__device__ __forceinline__ typename Elem<T>::frag acc_frag(const float16_t& a, int sl) {
  typename Elem<T>::frag f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = static_cast<T>(a[8 * sl + j]);
  return f;
}

// Streams SR-row tiles of two [N, D] row-major tensors (and, with VECS, two
// per-row float vectors) through an LDS ring.  A stage holds
//   [tensor A tile | tensor B tile | VECS: VSLOT floats of vector 0 | VSLOT of vector 1]
// (only the first SR floats of each vector slot are used).
//  DMA (fp16, rows of whole 16-byte aligned chunks): stages filled by
//    global_load_lds, one tile ahead; rows past `rows` re-read the last row
//    (callers mask them); chunks past d are zeroed once and never copied.
//  otherwise: stages filled through registers; rows past `rows` are 0
//    and vector 0 / vector 1 read +inf / 0 there.
// Vector 0 is stored pre-multiplied by log2(e) on the register path only; DMA
// consumers scale at the read (vec_scale()).
template <typename T, int DP, bool DMA, bool VECS, int SR_, int ROWS>
struct TileRing {
  typedef typename Elem<T>::frag F;
  typedef Layout<T, DP> L;
  static constexpr int SR = SR_;
  static constexpr int NS = 2;  // three DMA stages measured 4.7 % slower (config 7 backward 367 vs 350 us)
  static constexpr int VSLOT = SR < 64 ? 64 : SR;
  static constexpr int VEC_FLOATS = VECS ? 2 * VSLOT : 0;
  static constexpr int TILE_BYTES = SR * L::LD * static_cast<int>(sizeof(T));
  static constexpr int STAGE_BYTES = 2 * TILE_BYTES + VEC_FLOATS * 4;
  static constexpr int BYTES = NS * STAGE_BYTES;
  static constexpr int CPR = DP / 8;            // 8-element groups per row
  static constexpr int CHUNKS = SR * CPR;       // groups per tile
  static constexpr int PER_THREAD = (CHUNKS + kThreads - 1) / kThreads;
  // DMA instructions this wave issues per tile (the first 2 * VSLOT / 64 waves also copy a vector part)
  static constexpr int DMA_PER_TILE = 2 * PER_THREAD;

  unsigned lds_base;  // byte address of stage 0
  int tid, lane, wave;
  // register path staging
  F a[DMA ? 1 : PER_THREAD], b[DMA ? 1 : PER_THREAD];
  float v0 = 0.0f, v1 = 0.0f;
  // DMA path: per copy, the tile row, column and byte offset of this lane's chunk
  int cp_row[PER_THREAD], cp_col[PER_THREAD];
  unsigned cp_off[PER_THREAD];

  __device__ TileRing(void* smem, int tid_, int d)
      : tid(tid_), lane(tid_ & 63), wave(__builtin_amdgcn_readfirstlane(tid_ >> 6)) {
    lds_base = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)smem));
    if constexpr (DMA) {
      static_assert(sizeof(T) == 2 && CHUNKS % kThreads == 0, "DMA tiles are whole fp16 chunks per thread");
#pragma unroll
      for (int i = 0; i < PER_THREAD; ++i) {
        // slot g (16-byte LDS chunk) = i * 256 + tid holds logical chunk
        // (g % CPR) ^ swizzle(row) of row g / CPR
        const int g = i * kThreads + tid;
        cp_row[i] = g / CPR;
        cp_col[i] = ((g % CPR) ^ chunk_swizzle<DP>(g / CPR)) * 8;
        cp_off[i] = static_cast<unsigned>((cp_row[i] * d + cp_col[i]) * 2);
      }
      if constexpr (ROWS == kRowChunks) {
        // chunks past d are products' zeros: they must not hold a NaN
#pragma unroll
        for (int i = 0; i < PER_THREAD; ++i)
          if (cp_col[i] >= d)
#pragma unroll
            for (int s = 0; s < 2 * NS; ++s)
              *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(static_cast<size_t>(
                  lds_base + (s >> 1) * STAGE_BYTES + (s & 1) * TILE_BYTES + (i * kThreads + tid) * 16)) =
                  u32x4{0u, 0u, 0u, 0u};
      }
    }
  }
  __device__ __forceinline__ unsigned addr_a(int stage) const { return lds_base + stage * STAGE_BYTES; }
  __device__ __forceinline__ unsigned addr_b(int stage) const { return addr_a(stage) + TILE_BYTES; }
  __device__ __forceinline__ lds_ptr<T> tile_a(int stage) const {
    return reinterpret_cast<lds_ptr<T>>(static_cast<size_t>(addr_a(stage)));
  }
  __device__ __forceinline__ lds_ptr<T> tile_b(int stage) const {
    return reinterpret_cast<lds_ptr<T>>(static_cast<size_t>(addr_b(stage)));
  }
  __device__ __forceinline__ const __attribute__((address_space(3))) float* vec(int stage, int which) const {
    return reinterpret_cast<const __attribute__((address_space(3))) float*>(
        static_cast<size_t>(addr_a(stage) + 2 * TILE_BYTES + which * VSLOT * 4));
  }

  // DMA path: copy rows [r0, r0 + SR) of pa/pb (row stride d) and, with
  // VECS, va/vb[r0 .. r0 + SR) into `stage`.
  __device__ __forceinline__ void dma(const T* pa, const T* pb, const float* va, const float* vb, int r0, int rows,
                                      int d, int stage) const {
    const T* ba = pa + static_cast<size_t>(r0) * d;
    const T* bb = pb + static_cast<size_t>(r0) * d;
    const unsigned sbase = lds_base + stage * STAGE_BYTES;
    const bool tail = r0 + SR > rows;
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
      unsigned off = cp_off[i];
      if (tail) {
        const int row = min(cp_row[i], rows - 1 - r0);
        off = static_cast<unsigned>(static_cast<int>(off) + (row - cp_row[i]) * d * 2);
      }
      const unsigned slot = sbase + (i * kThreads + wave * 64) * 16;
      // (a copy covers whole rows: it has active lanes whatever d, so vmcnt counts hold)
      if (ROWS == kRowFull || cp_col[i] < d) {
        copy16_to_lds(reinterpret_cast<const half_t*>(ba), off, slot);
        copy16_to_lds(reinterpret_cast<const half_t*>(bb), off, slot + TILE_BYTES);
      }
    }
    if constexpr (VECS) {
      if (wave < 2 * VSLOT / 64) {  // wave w: 64 rows from 64 (w / 2) of vector w % 2
        const float* base = ((wave & 1) ? vb : va) + r0;
        const int row = SR < 64 ? (lane & (SR - 1)) : lane + 64 * (wave >> 1);
        const unsigned off = static_cast<unsigned>(min(row, rows - 1 - r0)) * 4;
        copy4_to_lds(base, off, sbase + 2 * TILE_BYTES + (wave & 1) * (VSLOT * 4) + (wave >> 1) * 256);
      }
    }
  }
  // Waits until this wave's copies of every tile but the newest `pending` ones
  // have landed (DMA path).
  __device__ __forceinline__ void wait_dma(bool one_pending) const {
    const bool extra = VECS && wave < 2 * VSLOT / 64;
    if (one_pending) {
      if (extra) wait_vm_lgkm0<DMA_PER_TILE + 1>();
      else wait_vm_lgkm0<DMA_PER_TILE>();
    } else {
      wait_vm_lgkm0<0>();
    }
  }

  // The thread index; opaque to the compiler in fp32's split blocks at DP = 64, so
  // that the register path's addresses are formed anew for each tile (a few VALU
  // instructions) and not kept in registers: the key-major kernel has none left
  // there (5 went to scratch: causal [1,8,2048,64] backward 371 -> 363 us without).
  // Unsplit blocks have them, and pay ([4,16,2048,64] 1053 -> 1096).
  __device__ __forceinline__ int thread_now() const {
    int t = tid;
    if constexpr (sizeof(T) == 4 && DP == 64 && SR > kRows) asm volatile("" : "+v"(t));
    return t;
  }

  // Register path: load rows [r0, r0 + SR) (zero past `rows`) into registers ...
  __device__ __forceinline__ void load(const T* pa, const T* pb, const float* va, const float* vb, int r0, int rows,
                                       int d) {
    const int tid = thread_now();
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
      const int c = tid + i * kThreads;
      const int row = c / CPR;
      const int col = (c % CPR) * 8;
      if ((CHUNKS % kThreads == 0 || c < CHUNKS) && r0 + row < rows) {
        a[i] = load_frag<T, ROWS>(pa + static_cast<size_t>(r0 + row) * d, col, d);
        b[i] = load_frag<T, ROWS>(pb + static_cast<size_t>(r0 + row) * d, col, d);
      } else {
        a[i] = zero_frag<T>();
        b[i] = zero_frag<T>();
      }
    }
    if constexpr (VECS) {
      if (tid < SR) {
        const int r = r0 + tid;
        v0 = r < rows ? va[r] * kLog2e : INFINITY;  // padding rows: P = 0
        v1 = r < rows ? vb[r] : 0.0f;
      }
    }
  }
  // ... and store them into `stage`.
  __device__ __forceinline__ void store(int stage) const {
    lds_ptr<T> ta = tile_a(stage);
    lds_ptr<T> tb = tile_b(stage);
    const int tid = thread_now();
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
      const int c = tid + i * kThreads;
      if (CHUNKS % kThreads == 0 || c < CHUNKS) {
        const int row = c / CPR;
        const int col = (c % CPR) * 8;
        *reinterpret_cast<__attribute__((address_space(3))) F*>(ta + L::off(row, col)) = a[i];
        *reinterpret_cast<__attribute__((address_space(3))) F*>(tb + L::off(row, col)) = b[i];
      }
    }
    if constexpr (VECS) {
      if (tid < SR) {
        auto* v = const_cast<__attribute__((address_space(3))) float*>(vec(stage, 0));
        v[tid] = v0;
        v[VSLOT + tid] = v1;
      }
    }
  }
};

// Split walks: SPLIT waves of a workgroup share one 32-row block and take the
// 32-row sub-tiles of every streamed SPLIT * 32-row tile in turn (wave w:
// block w % (4 / SPLIT), sub-tile w / (4 / SPLIT)); their partial accumulators
// meet in LDS at the end.  A wave's serial walk is then 1 / SPLIT as long and
// there are SPLIT times as many workgroups, which is what bounds calls whose
// 128-row blocks are few.  All of a row block's waves hold the same element in
// the same lane and register, so partials pass lane to lane: slot
// [wave][register][lane], conflict-free.
template <int REGS>
__device__ __forceinline__ lds_ptr<float> part_slot(char* smem, int wave, int lane) {
  return reinterpret_cast<lds_ptr<float>>(static_cast<size_t>(static_cast<unsigned>(
             reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)smem)))) + wave * REGS * 64 + lane;
}

}  // namespace train
}  // namespace fa
