// Device kernels of attention with modified scores for gfx950: forward (with
// optional log-sum-exp) and backward (dQ, dK, dV), fp16 and fp32, grouped KV
// heads.  Instantiated by scored.hip and scored_backward.hip (fp16) and
// scored_fp32.hip.
//
//   s_ij   = q_i . k_j / sqrt(D)
//   c_ij   = cap tanh(s_ij / cap)            (cap > 0; else s_ij)
//   y_ij   = c_ij - slope_h |i - j|
//   j is visible to i iff (no ids, or id_i = id_j >= 0) and
//                         (not causal, or j <= i, or j < prefix_b)
//   P_ij   = exp(y_ij - lse_i) over the visible j, O_i = sum_j P_ij V_j
//   dY_ij  = P_ij (dO_i . V_j - delta_i), delta_i = sum_d dO_id O_id
//   dS_ij  = dY_ij (1 - (c_ij / cap)^2)
//   dQ = dS K / sqrt(D), dK = dS^T Q / sqrt(D), dV = P^T dO (dK, dV summed over
//   the query heads of the KV head)
// A row that sees nothing has O = 0, lse = -inf and takes no part in the
// gradients.  Rows of negative id are padding: whatever they hold, NaN
// included, reaches no other row (their staged tile rows are zeroed).
//
// Shapes, operand layouts and tile streaming are the training kernels'
// (train_tiles.h): 4 waves of 32 rows, 32-row tiles through a two-stage LDS
// ring, S^T = K Q^T with one query per lane (query-major: forward, dQ), S = Q
// K^T with one key per lane (key-major: dK, dV).  A KV head's query heads are
// streamed in turn past the key-major kernel's keys, so dK and dV add up in
// registers in a fixed order, without atomics.
//
// Document masks: a workgroup walks only the tiles that hold an id in the range of its
// own rows' ids.  Every 64 sub-tiles of 32 rows each lane reads one
// sub-tile's ids (8 16-byte loads) and keeps its range; the live ones
// are a 64-bit ballot that scalar code steps through.  A sub-tile of a single id needs no
// per-element mask where the wave's rows hold that id too; the others compare
// ids element by element.
#pragma once

#include "train_tiles.h"

namespace fa {
namespace scored {

using train::acc_frag;
using train::Elem;
using train::kBlockRows;
using train::kLn2;
using train::kRows;
using train::kThreads;
using train::kWaves;
using train::Layout;
using train::lds_ptr;
using train::load_frag;
using train::mma;
using train::part_slot;
using train::Reader;
using train::TileRing;
using train::zero_frag;

// What a kernel variant applies to the scores; kAnyMods reads it from the
// call's parameters instead (uniform branches).
enum Mods : int { kCap = 1, kBias = 2, kDocs = 4, kAnyMods = 8 };

struct ScoredParams {
  const void* q;
  const void* k;
  const void* v;
  const void* o;          // backward: forward output
  const void* dout;       // backward
  void* out;              // forward: O; backward: dQ
  void* dk;
  void* dv;
  float* lse;             // forward: written if non-null; backward: read
  float* delta;           // backward workspace [B * H_Q * N]: delta, and
  float* row_lse;         // [B * H_Q * N]: log-sum-exp as the key-major passes take it (dQ writes both)
  const float* slopes;    // [H_Q] or null
  const int32_t* ids;     // [B, N] or null
  const int32_t* prefix;  // [B] or null (causal only)
  int mods;
  int B, H_Q, H_KV, N, D, G, causal;
  int nblk;               // row blocks (one workgroup each) per head
  int heads;              // query heads dealt with one unit (query-major)
  int units, group_units; // units of the grid, and how many an XCD interleaves
  int snake;              // every other round of an XCD's blocks lightest first
  float scale;            // 1/sqrt(D)
  float scale_log2;       // scale * log2(e)
  float cap_in;           // scale / cap
  float cap_log2;         // cap * log2(e)
  float cap_slope;        // 1 / cap_log2^2
  float cap_near;         // raw products up to which the tanh's polynomial serves
  float cap_poly[5];      // its coefficients
};

template <int MODS>
__device__ __forceinline__ bool has(const ScoredParams& p, int m) {
  if constexpr ((MODS & kAnyMods) != 0) return (p.mods & m) != 0;
  return (MODS & m) != 0;
}

constexpr int kXcds = 8;
constexpr int kXcdCus = 32;

// Workgroup -> (unit u, head of the unit, row block).  Units are dealt to the
// XCDs round-robin (the dispatcher sends workgroup j to XCD j % 8), an XCD
// interleaves group_units of them, heaviest block first, so the blocks that
// stream the same tiles run together behind one L2.  Heavy first suits grids
// that the dispatcher refills as workgroups end; where the whole grid is
// resident at once, workgroups i and i + 32 of an XCD share a CU, and the snake
// order (every other 32 of them backwards) gives each CU about the same work.  Returns false for the
// padding workgroups of the last round.  group_units 0: block by block, all
// heads' heaviest first.
__device__ __forceinline__ bool map_block(const ScoredParams& p, int heads, bool heavy_last, int& u, int& head, int& blk) {
  const int j = static_cast<int>(blockIdx.x);
  if (p.group_units == 0) {
    const int pair = j % (p.units * heads), b = j / (p.units * heads);
    u = pair / heads;
    head = pair % heads;
    blk = heavy_last ? p.nblk - 1 - b : b;
    return true;
  }
  const int i = j / kXcds;
  const int per_row = p.group_units * heads;
  const int n = per_row * p.nblk;
  const int group = i / n;
  int ii = i % n;
  if (p.snake && ((ii / kXcdCus) & 1)) {
    const int first = ii / kXcdCus * kXcdCus;
    ii = first + min(n, first + kXcdCus) - 1 - ii;
  }
  const int b = ii / per_row;
  const int hg = ii % per_row;
  u = j % kXcds + kXcds * (group * p.group_units + hg / heads);
  head = hg % heads;
  blk = heavy_last ? p.nblk - 1 - b : b;
  return u < p.units;
}

typedef int int4u __attribute__((ext_vector_type(4), aligned(4)));

// Least and largest over the wave: lane permutes within the rows of 16, scalar
// instructions over the four rows.
__device__ __forceinline__ int wave_min_i(int x) {
  x = min(x, dpp_mov_i<kDppQuadXor1>(x));
  x = min(x, dpp_mov_i<kDppQuadXor2>(x));
  x = min(x, dpp_mov_i<kDppRowHalfMirror>(x));
  x = min(x, dpp_mov_i<kDppRowMirror>(x));
  return min(min(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)),
             min(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
}
__device__ __forceinline__ int wave_max_i(int x) { return -wave_min_i(-x); }

// Columns d0 .. d0 + 3 of an output row (d0 a multiple of 4; rows of whole 8-element
// chunks hold all four or none of them).
template <typename T, int ROWS>
__device__ __forceinline__ void store4(T* row, int d0, int d, float a, float b, float c, float e) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  const vec4 x = {static_cast<T>(a), static_cast<T>(b), static_cast<T>(c), static_cast<T>(e)};
  if constexpr (ROWS == kRowElems) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (d0 + j < d) row[d0 + j] = x[j];
  } else {
    if (ROWS == kRowFull || d0 < d) *reinterpret_cast<vec4*>(row + d0) = x;
  }
}

constexpr int kMixedIds = -1;       // a sub-tile of several ids (or a ragged one)
constexpr int kNoId = -2147483646;  // own rows that see nothing; differs from every staged id

// The tiles a workgroup streams: SUBS 32-row sub-tiles each, `count` of them
// from row `first`, last to first with `rev`, else from tile `start` on and
// round to it.  With ids, only those that hold an id of [lo, hi], and the first in
// walk order where `own` says that it holds the workgroup's own rows (its copies
// start before any id has arrived).
template <int SUBS>
struct TileWalk {
  const int32_t* ids;  // of the streamed rows' batch row, or null
  int rows, first, count, lo, hi;
  int start = 0;
  bool rev, own;
  int vt = 0;          // without ids: next tile in walk order
  int base = 0;        // with ids: first sub-tile (in walk order) of the group held
  uint64_t live = 0, pads = 0;
  int uni = 0;         // this lane's sub-tile: its single id, or kMixedIds
  // the tile that next() gave
  int tile = -1, at = 0;
  uint64_t cur_pads = 0;

  __device__ __forceinline__ int phys(int t) const {
    if (rev) return count - 1 - t;
    return t + start < count ? t + start : t + start - count;
  }
  // First row of this lane's sub-tile of the group, past the last row if it has none.
  __device__ __forceinline__ int lane_row() const {
    const int v = base + (threadIdx.x & 63);
    return v / SUBS < count ? first + (phys(v / SUBS) * SUBS + v % SUBS) * kRows : rows;
  }
  typedef int4u Ids[kRows / 4];
  // Issues the reads of the first group's ids ...
  __device__ __forceinline__ void load(Ids& raw) const {
    const int r0 = lane_row();
    if (r0 + kRows <= rows) {
#pragma unroll
      for (int i = 0; i < kRows / 4; ++i) raw[i] = *reinterpret_cast<const int4u*>(ids + r0 + 4 * i);
    }
  }
  // ... and turns them into its masks.
  __device__ __forceinline__ void digest(const Ids& raw) {
    masks([&](auto&& take) {
#pragma unroll
      for (int i = 0; i < kRows / 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) take(raw[i][j]);
    });
    if (own) live |= 1;
  }
  // A later group, in the loop: few registers rather than all reads at once.
  __device__ __forceinline__ void scan() {
    const int r0 = lane_row();
    masks([&](auto&& take) {
#pragma unroll 1
      for (int i = 0; i < kRows / 4; ++i) {
        const int4u x = *reinterpret_cast<const int4u*>(ids + r0 + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) take(x[j]);
      }
    });
  }
  // The group's masks, from a whole sub-tile's ids as `whole` passes them on.
  template <typename Whole>
  __device__ __forceinline__ void masks(Whole&& whole) {
    const int r0 = lane_row();
    int mn = 0x7fffffff, mx = -1, least = 0;
    auto take = [&](int id) {
      least = min(least, id);
      mn = min(mn, id < 0 ? 0x7fffffff : id);
      mx = max(mx, id);
    };
    const bool full = r0 + kRows <= rows;
    if (full) whole(take);
    else for (int r = r0; r < rows; ++r) take(ids[r]);
    uni = full && least >= 0 && mn == mx ? mn : kMixedIds;
    live = __builtin_amdgcn_ballot_w64(mx >= lo && mn <= hi && mn <= mx);
    pads = __builtin_amdgcn_ballot_w64(least < 0);
  }
  // Steps to the next tile; false when there is none.  Every lane of every
  // wave of the workgroup takes the same steps.
  __device__ __forceinline__ bool next() {
    if (ids == nullptr) {
      if (vt >= count) return false;
      tile = phys(vt++);
      return true;
    }
    while (live == 0) {
      base += 64;
      if (base >= count * SUBS) return false;
      scan();
    }
    const int bit = __builtin_ctzll(live) / SUBS * SUBS;
    const uint64_t mask = (SUBS == 1 ? 1ull : (1ull << SUBS) - 1) << bit;
    live &= ~mask;
    cur_pads = pads & mask;
    tile = phys((base + bit) / SUBS);
    at = bit;
    return true;
  }
  // Single id of sub-tile `sub` of the current tile, or kMixedIds.
  __device__ __forceinline__ int sub_id(int sub) const { return __builtin_amdgcn_readlane(uni, at + sub); }
};

// ---- scores ----
// A masked score of the backward: its P is 0, and its square stays finite in the
// derivative of the cap.  Real ones lie far above (fp16 products within 1e12).
constexpr float kDeadScore = -1e15f;

// Raw products s -> capped scores in the log2 domain, cap log2(e) tanh(s scale / cap).
// Where every score of the wave's tile is at most half the cap, tanh is the odd
// polynomial of common.h with the scales folded into its coefficients, y = s (c0 +
// c1 s^2 + ...): 6 full-rate operations a score, where the exponential form takes two
// quarter-rate ones and 9 others.  (These kernels are bound by their vector
// instructions: with the coefficients unfolded, 9 a score, prefill
// [1,32:8,8192,128] takes 689 us for 658.)
__device__ __forceinline__ float cap_factor(float s, const ScoredParams& p) {
  const float w = s * s;
  return fmaf(fmaf(fmaf(fmaf(p.cap_poly[4], w, p.cap_poly[3]), w, p.cap_poly[2]), w, p.cap_poly[1]), w, p.cap_poly[0]);
}
__device__ __forceinline__ bool cap_is_near(const float16_t& s, const ScoredParams& p) {
  float big = 0.0f;
#pragma unroll
  for (int r = 0; r < 16; r += 2) big = fmaxf(fmaxf(fabsf(s[r]), fabsf(s[r + 1])), big);
  return __builtin_amdgcn_ballot_w64(!(big <= p.cap_near)) == 0;
}
__device__ __forceinline__ void cap_scores(float16_t& s, bool near, const ScoredParams& p) {
  if (near) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] *= cap_factor(s[r], p);
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = tanh_f32(s[r] * p.cap_in) * p.cap_log2;
  }
}

// Distances of a tile's elements: element r lies `rel` + 8 (r / 4) + r % 4 from the lane's row.
__device__ __forceinline__ void add_bias(float16_t& y, float slope2, float rel) {
#pragma unroll
  for (int r = 0; r < 16; ++r) y[r] = fmaf(-slope2, fabsf(rel + static_cast<float>(8 * (r >> 2) + (r & 3))), y[r]);
}

// Ids of the staged tiles' rows, beside the ring: they travel with the tile, so
// that a tile of several documents waits for nothing of its own.  (Read from global
// memory where a tile needs them, they drain the copies in flight; measured the same,
// 116 to 120 us either way for the forward of documents [4,32:8,2048,128].)
constexpr int kStagedIds = kWaves * kRows;  // rows of a stage, at most

// Fetches the ids of rows [r0, r0 + SR) (past `rows`: the last row's) into a stage's slots.
template <int SR, bool DMA>
__device__ __forceinline__ void fetch_ids(const int32_t* ids, int r0, int rows, int (&slots)[kStagedIds]) {
  const int row = min(static_cast<int>(threadIdx.x) & (SR - 1), rows - 1 - r0);
  if constexpr (DMA) {
    // 64 slots a wave; of 32-row tiles half of them are used
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (64 * wave < SR)
      copy4_to_lds(reinterpret_cast<const float*>(ids + r0), static_cast<unsigned>(row) * 4,
                   static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) int*)slots)) + wave * 256);
  } else {
    if (threadIdx.x < SR) slots[threadIdx.x] = ids[r0 + row];
  }
}

// Calls use(r, same) for the 16 tile rows 8 (r / 4) + r % 4 from `at`: whether the row's id is `mine`
// (an id >= 0, or one that no row has).
template <typename Use>
__device__ __forceinline__ void compare_ids(const int* at, int mine, Use&& use) {
#pragma unroll
  for (int rr = 0; rr < 4; ++rr) {
    typedef int int4a __attribute__((ext_vector_type(4)));
    const int4a x = *reinterpret_cast<const int4a*>(at + 8 * rr);
#pragma unroll
    for (int j = 0; j < 4; ++j) use(4 * rr + j, max(x[j], -1) == mine);
    // four ids at a time: the registers are full here, and such tiles are few
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Zeroes the rows of negative id in the staged tile pair (rows past the last may
// hold it again, with its id).
template <typename T, typename Ring>
__device__ __forceinline__ void zero_pad_rows(const Ring& ring, int stage, const int* ids) {
  lds_ptr<T> ta = ring.tile_a(stage);
  lds_ptr<T> tb = ring.tile_b(stage);
  typedef typename Elem<T>::frag F;
  for (int c = threadIdx.x; c < Ring::CHUNKS; c += kThreads) {
    const int row = c / Ring::CPR, col = c % Ring::CPR * 8;
    if (ids[row] < 0) {
      *reinterpret_cast<__attribute__((address_space(3))) F*>(ta + Ring::L::off(row, col)) = zero_frag<T>();
      *reinterpret_cast<__attribute__((address_space(3))) F*>(tb + Ring::L::off(row, col)) = zero_frag<T>();
    }
  }
}

// Streams the walk's tiles through the ring, HEADS rounds a tile (key-major:
// the query heads in turn), and calls compute(stage, tile, round, sub id) for
// each; fetch(tile, round, stage) copies (DMA) or loads (registers) one.  The
// caller has fetched the first tile of a walk that starts at its own rows.
template <typename T, typename Ring, bool DMA, int SUBS, typename Fetch, typename Compute>
__device__ __forceinline__ void stream_tiles(Ring& ring, TileWalk<SUBS>& walk, int heads, int sub,
                                             const int (&ids)[2][kStagedIds], Fetch&& fetch, Compute&& compute) {
  bool more = walk.next();
  if (!more) return;
  int tile = walk.tile, id = walk.ids ? walk.sub_id(sub) : 0, head = 0, stage = 0;
  uint64_t pads = walk.cur_pads;
  if (!walk.own) fetch(tile, 0, 0);
  if constexpr (!DMA) ring.store(0);
  for (;;) {
    // the (tile, head) after this one
    int ntile = tile, nid = id, nhead = head + 1;
    uint64_t npads = pads;
    if (nhead == heads) {
      nhead = 0;
      more = walk.next();
      ntile = walk.tile;
      npads = walk.cur_pads;
      if (walk.ids && more) nid = walk.sub_id(sub);
    }
    if constexpr (DMA) {
      ring.wait_dma(false);  // this wave's copies of the tile have landed
      tile_barrier();        // everyone's have; the other stage is free
    } else {
      __syncthreads();
    }
    if (pads != 0) {
      zero_pad_rows<T>(ring, stage, ids[stage]);
      __syncthreads();
    }
    if (more) fetch(ntile, nhead, stage ^ 1);
    compute(stage, tile, head, id);
    if (!more) break;
    if constexpr (!DMA) ring.store(stage ^ 1);
    tile = ntile;
    id = nid;
    head = nhead;
    pads = npads;
    stage ^= 1;
  }
}

// ---------------------------------------------------------------------------
// Query-major kernel: MODE 0 = forward (O, optional LSE), MODE 1 = dQ + delta.
// Registers: the fp16 forward asks for three waves per SIMD up to D = 128, four up to
// 96 (LDS allows them in whole blocks), fp32 at D <= 64 for two.
template <typename T, int DC, int MODE, int SPLIT, int MODS>
constexpr int query_waves() {
  if (sizeof(T) == 4) return DC <= 64 && SPLIT <= 2 ? 2 : 1;
  if (MODE != 0 || DC > 128 || SPLIT > 1 || (MODS & kAnyMods) != 0) return 1;
  return DC <= 96 && (MODS & kDocs) == 0 ? 4 : 3;
}
template <typename T, int DP, int DC, int ROWS, int MODE, int SPLIT, int MODS>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(query_waves<T, DC, MODE, SPLIT, MODS>()))) void scored_query_kernel(
    ScoredParams p) {
  typedef typename Elem<T>::frag F;
  constexpr int KK = DC / 16;
  constexpr int DB = (DC + 31) / 32;
  constexpr bool DMA = ROWS != kRowElems && sizeof(T) == 2;
  constexpr int RW = kWaves / SPLIT;  // 32-row blocks per workgroup
  typedef TileRing<T, DP, DMA, false, kRows * SPLIT, ROWS> Ring;
  __shared__ __attribute__((aligned(1024))) char smem[Ring::BYTES];
  __shared__ __attribute__((aligned(16))) int s_ids[2][kStagedIds];

  const int N = p.N, D = p.D;
  int u, hg, blk;
  if (!map_block(p, p.heads, p.causal != 0, u, hg, blk)) return;
  const int units_per_b = p.H_Q / p.heads;
  const int b = u / units_per_b;
  const int h = u % units_per_b * p.heads + hg;
  const int hk = h / p.G;
  const int q0 = blk * (RW * kRows);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31;
  const int hi = lane >> 5;
  const int sub = wave / RW;
  const int wq0 = q0 + (wave % RW) * kRows;
  const int qrow = wq0 + l32;
  const size_t qhead = static_cast<size_t>(b) * p.H_Q + h;
  const size_t qbase = qhead * N * D;
  const size_t kbase = (static_cast<size_t>(b) * p.H_KV + hk) * N * D;
  const T* __restrict__ kp = static_cast<const T*>(p.k) + kbase;
  const T* __restrict__ vp = static_cast<const T*>(p.v) + kbase;
  const bool cap = has<MODS>(p, kCap), bias = has<MODS>(p, kBias), docs = has<MODS>(p, kDocs);

  // keys every row sees, and the last key of this lane's row
  const int pre = p.prefix != nullptr ? max(0, min(p.prefix[b], N)) : 0;
  const int last = p.causal ? max(min(qrow, N - 1), pre - 1) : N - 1;
  const int kend = p.causal ? max(min(N, q0 + RW * kRows), pre) : N;
  const int kend_w = wq0 >= N ? 0 : (p.causal ? max(min(N, wq0 + kRows), pre) : N);
  constexpr int SR = Ring::SR;
  TileWalk<SPLIT> walk;
  walk.ids = docs ? p.ids + static_cast<size_t>(b) * N : nullptr;
  walk.rows = N;
  walk.first = 0;
  walk.count = (kend + SR - 1) / SR;
  // With a bias the nearest keys weigh most: a walk that starts at the diagonal
  // finds the running maximum at once (full [8,16,577,80] 43.6 -> 38.4 us).  With ids, the
  // diagonal tile is sure to be needed.
  walk.rev = p.causal && (bias || docs);
  walk.start = !p.causal && (bias || docs) ? q0 / SR : 0;
  walk.own = docs && pre == 0;

  Ring ring(smem, tid, D);
  auto fetch = [&](int tile, int, int stage) {
    if constexpr (DMA) ring.dma(kp, vp, nullptr, nullptr, tile * SR, N, D, stage);
    else ring.load(kp, vp, nullptr, nullptr, tile * SR, N, D);
    if (docs) fetch_ids<SR, DMA>(walk.ids, tile * SR, N, s_ids[stage]);
  };
  // Every read that the walk waits for is issued here, before the first wait:
  // ids, this lane's rows, the first tile.
  int my_id = 0, wlo = 0, whi = 0, block_id[(RW * kRows + 63) / 64];
  typename TileWalk<SPLIT>::Ids group_ids;
  if (docs) {
    walk.load(group_ids);
    my_id = qrow < N ? walk.ids[qrow] : -1;
#pragma unroll
    for (int i = 0; i < (RW * kRows + 63) / 64; ++i) {
      const int r = q0 + (lane + 64 * i) % (RW * kRows);
      block_id[i] = r < N ? walk.ids[r] : -1;
    }
  }
  // resident B operands: lane's query row, d = 16 kk + 8 hi .. +8
  F qf[KK], df[KK], of[KK];
  float lse2 = 0.0f, delta = 0.0f;
  {
    const size_t row = qbase + static_cast<size_t>(min(qrow, N - 1)) * D;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      qf[kk] = load_frag<T, ROWS>(static_cast<const T*>(p.q) + row, 16 * kk + 8 * hi, D);
      if constexpr (MODE == 1) {
        df[kk] = load_frag<T, ROWS>(static_cast<const T*>(p.dout) + row, 16 * kk + 8 * hi, D);
        of[kk] = load_frag<T, ROWS>(static_cast<const T*>(p.o) + row, 16 * kk + 8 * hi, D);
      }
    }
    if constexpr (MODE == 1) lse2 = p.lse[qhead * N + min(qrow, N - 1)] * kLog2e;
  }
  const float slope2 = bias ? p.slopes[h] * kLog2e : 0.0f;
  if (walk.own) fetch(walk.phys(0), 0, 0);
  if (docs) {
    my_id = my_id < 0 ? kNoId : my_id;
    wlo = wave_min_i(my_id < 0 ? 0x7fffffff : my_id);
    whi = wave_max_i(my_id);
    int lo = 0x7fffffff, top = -1;
#pragma unroll
    for (int i = 0; i < (RW * kRows + 63) / 64; ++i) {
      lo = min(lo, block_id[i] < 0 ? 0x7fffffff : block_id[i]);
      top = max(top, block_id[i]);
    }
    walk.lo = wave_min_i(lo);
    walk.hi = wave_max_i(top);
    walk.digest(group_ids);
  }
  const bool live = qrow < N && my_id >= 0;  // this lane's row sees something
  // single id of the wave's rows, or none
  const int wid = docs && wlo == whi && __builtin_amdgcn_ballot_w64(my_id != whi) == 0 ? whi : kNoId;
  if (!live) {
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      qf[kk] = zero_frag<T>();
      if constexpr (MODE == 1) df[kk] = of[kk] = zero_frag<T>();
    }
  }
  if constexpr (MODE == 1) {
    float part = 0.0f;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int j = 0; j < 8; ++j) part = fmaf(static_cast<float>(df[kk][j]), static_cast<float>(of[kk][j]), part);
    delta = part + __shfl_xor(part, 32, 64);
    const bool empty = !live || lse2 == -INFINITY;  // rows that see nothing: P = 0
    if (qrow < N && hi == 0 && sub == 0) {
      p.delta[qhead * N + qrow] = delta;
      // the key-major passes mask scores to kDead, and so need a finite value (the
      // register-staged ring scales by log2(e) itself)
      p.row_lse[qhead * N + qrow] = empty ? 0.0f : (DMA ? lse2 : p.lse[qhead * N + qrow]);
    }
    if (empty) lse2 = INFINITY;
  }

  float16_t acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = 0.0f;
  float m_run = kNegBig, l_run = 0.0f;  // forward only (log2 domain)
  const float c = cap || bias ? 1.0f : p.scale_log2;
  const Reader<T, DP> rd(lane);
  constexpr unsigned kSubBytes = kRows * Layout<T, DP>::LD * sizeof(T);
  stream_tiles<T, Ring, DMA, SPLIT>(ring, walk, 1, sub, s_ids, fetch, [&](int stage, int tile, int, int id) {
    const int kt = tile * SR + sub * kRows;
    if (kt >= kend_w) return;                               // past this wave's rows
    if (docs && id >= 0 && (id < wlo || id > whi)) return;  // a document of other waves' rows
    const unsigned ks = ring.addr_a(stage) + sub * kSubBytes;
    const unsigned vs = ring.addr_b(stage) + sub * kSubBytes;
    // S^T = K Q^T: lane <-> query, register r <-> key kt + 8 (r/4) + 4 hi + r%4
    float16_t s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) s = mma(rd.row(ks, kk), qf[kk], s);
    const bool edge = kt + kRows > N || (p.causal && kt + kRows - 1 > max(wq0, pre - 1));
    const bool mixed = docs && (id < 0 || id != wid);
    const bool near = cap && cap_is_near(s, p);
    // The forward's unmasked tiles take the cap's last product into the exponent, p =
    // exp2(s f(s) - m), one operation a score less (prefill [1,32:8,8192,128] 658 -> 649 us).
    const bool fused = MODE == 0 && cap && !bias && near && !edge && !mixed;
    if (cap && !fused) {
      cap_scores(s, near, p);
    } else if (bias && !cap) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] *= p.scale_log2;
    }
    // dQ: derivative of the cap, from the capped score where that stays at hand
    constexpr bool kKeepDt = MODE == 1 && (MODS & kAnyMods) != 0;
    float16_t dt;
    if constexpr (kKeepDt) {
#pragma unroll
      for (int r = 0; r < 16; ++r) dt[r] = cap ? fmaf(s[r] * s[r], -p.cap_slope, 1.0f) : 1.0f;
    }
    if (bias) add_bias(s, slope2, static_cast<float>(kt + 4 * hi - qrow));
    constexpr float kDead = MODE == 1 ? kDeadScore : -INFINITY;
    if (edge) {
      const int bound = last - kt - 4 * hi;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 8 * (r >> 2) + (r & 3) > bound ? kDead : s[r];
    }
    if (mixed) {
      if (id >= 0) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = my_id == id ? s[r] : kDead;
      } else {
        compare_ids(s_ids[stage] + sub * kRows + 4 * hi, my_id, [&](int r, bool same) { s[r] = same ? s[r] : kDead; });
      }
    }
    float16_t pm;  // P^T (forward) or dS^T (dQ)
    if constexpr (MODE == 0) {
      // p = exp2(s c - m) against the running max m, which is only refreshed
      // (and O, l rescaled) when a lane's partial sum passes 2^8, i.e. some
      // score outgrew m by more than the slack (always so from m = -1e30).
      constexpr float kRescaleLimit = 256.0f;
      float ls = 0.0f;
      if (fused) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          pm[r] = fast_exp2(fmaf(s[r], cap_factor(s[r], p), -m_run));
          ls += pm[r];
        }
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          pm[r] = fast_exp2(fmaf(s[r], c, -m_run));
          ls += pm[r];
        }
      }
      if (__builtin_amdgcn_ballot_w64(!(ls <= kRescaleLimit)) != 0) {
        if (fused) cap_scores(s, true, p);
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * c;
        const float mn = fmaxf(m_run, mx);
        const float alpha = fast_exp2(m_run - mn);
        m_run = mn;
        l_run *= alpha;
        ls = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          pm[r] = fast_exp2(fmaf(s[r], c, -mn));
          ls += pm[r];
        }
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[db][r] *= alpha;
      }
      l_run += ls;
    } else {
      // dP^T = V dO^T
      float16_t dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) dp = mma(rd.row(vs, kk), df[kk], dp);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        pm[r] = fast_exp2(fmaf(s[r], c, -lse2)) * (dp[r] - delta);
        if constexpr (kKeepDt) pm[r] *= dt[r];
        else if (cap) pm[r] *= fmaf(s[r] * s[r], -p.cap_slope, 1.0f);
      }
    }
    const F pf0 = acc_frag<T>(pm, 0), pf1 = acc_frag<T>(pm, 1);
    // forward: O^T += V^T P^T;  dQ: dQ^T += K^T dS^T
    const unsigned src = (MODE == 0) ? vs : ks;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      acc[db] = mma(rd.tr(src, 0, db), pf0, acc[db]);
      acc[db] = mma(rd.tr(src, 16, db), pf1, acc[db]);
    }
  });

  // ---- join the row block's waves: wave `sub` 0 takes the others' partials ----
  if constexpr (SPLIT > 1) {
    constexpr int REGS = 16 * DB + (MODE == 0 ? 2 : 0);
    static_assert((SPLIT - 1) * RW * REGS * 256 <= Ring::BYTES, "partials fit the ring");
    __syncthreads();  // every wave is done reading the ring
    if (sub > 0) {
      lds_ptr<float> out = part_slot<REGS>(smem, wave - RW, lane);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) out[(16 * db + r) * 64] = acc[db][r];
      if constexpr (MODE == 0) {
        out[16 * DB * 64] = m_run;
        out[(16 * DB + 1) * 64] = l_run;
      }
    }
    __syncthreads();
    if (sub > 0) return;
    // a wave that saw no key has m = -1e30, l = 0 and weighs nothing
#pragma unroll
    for (int w = 0; w < SPLIT - 1; ++w) {
      lds_ptr<float> in = part_slot<REGS>(smem, w * RW + wave, lane);
      float a0 = 1.0f, a1 = 1.0f;
      if constexpr (MODE == 0) {
        const float m1 = in[16 * DB * 64];
        const float mn = fmaxf(m_run, m1);
        a0 = fast_exp2(m_run - mn);
        a1 = fast_exp2(m1 - mn);
        m_run = mn;
        l_run = l_run * a0 + in[(16 * DB + 1) * 64] * a1;
      }
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          acc[db][r] = MODE == 0 ? acc[db][r] * a0 + in[(16 * db + r) * 64] * a1 : acc[db][r] + in[(16 * db + r) * 64];
    }
  }

  // ---- store: lane's row, d = 32 db + 8 (r/4) + 4 hi + r%4 ----
  float mul;
  if constexpr (MODE == 0) {
    const float lt = l_run + __shfl_xor(l_run, 32, 64);
    mul = !live || lt == 0.0f ? 0.0f : 1.0f / lt;
    if (p.lse != nullptr && qrow < N && hi == 0)
      p.lse[qhead * N + qrow] = !live || lt == 0.0f ? -INFINITY : (m_run + log2f(lt)) * kLn2;
  } else {
    mul = p.scale;
  }
  if (qrow >= N) return;
  T* op = static_cast<T*>(p.out) + qbase + static_cast<size_t>(qrow) * D;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
      auto x = [&](int j) { return live ? acc[db][4 * rr + j] * mul : 0.0f; };
      store4<T, ROWS>(op, 32 * db + 8 * rr + 4 * hi, D, x(0), x(1), x(2), x(3));
    }
}

// ---------------------------------------------------------------------------
// Waves per SIMD that the key kernel's registers leave room for: two where LDS holds two
// workgroups and the variant is compiled in.  At D = 128 that spills up to 41 registers
// and still wins: documents [4,32:8,2048,128] 248 us, with one wave 346.
template <typename T, int DP, int SPLIT, int MODS>
constexpr int key_waves() {
  if (SPLIT > 2) return 1;
  return (sizeof(T) == 4 ? DP <= 64 : DP == 128 && (MODS & kAnyMods) == 0) ? 2 : 1;
}

// Key-major kernel for 32 keys per wave: dV += P^T dO and dK += dS^T Q.
template <typename T, int DP, int DC, int ROWS, int SPLIT, int MODS>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(key_waves<T, DP, SPLIT, MODS>()))) void scored_key_kernel(
    ScoredParams p) {
  typedef typename Elem<T>::frag F;
  constexpr int KK = DC / 16;
  constexpr int DB = (DC + 31) / 32;
  constexpr bool DMA = ROWS != kRowElems && sizeof(T) == 2;
  constexpr int RW = kWaves / SPLIT;  // 32-key blocks per workgroup
  typedef TileRing<T, DP, DMA, true, kRows * SPLIT, ROWS> Ring;
  __shared__ __attribute__((aligned(1024))) char smem[Ring::BYTES];
  __shared__ __attribute__((aligned(16))) int s_ids[2][kStagedIds];

  const int N = p.N, D = p.D;
  int u, hg, blk;
  if (!map_block(p, 1, false, u, hg, blk)) return;
  const int b = u / p.H_KV, hk = u % p.H_KV;
  const int k0 = blk * (RW * kRows);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31;
  const int hi = lane >> 5;
  const int sub = wave / RW;
  const int wk0 = k0 + (wave % RW) * kRows;
  const int krow = wk0 + l32;
  const size_t kbase = (static_cast<size_t>(b) * p.H_KV + hk) * N * D;
  const size_t qhead0 = static_cast<size_t>(b) * p.H_Q + static_cast<size_t>(hk) * p.G;  // first query head of the group
  const bool cap = has<MODS>(p, kCap), bias = has<MODS>(p, kBias), docs = has<MODS>(p, kDocs);

  const int pre = p.prefix != nullptr ? max(0, min(p.prefix[b], N)) : 0;
  // causal: rows before the first key see it only inside the prefix
  const int qstart = p.causal && k0 >= pre ? k0 : 0;
  constexpr int SR = Ring::SR;
  TileWalk<SPLIT> walk;
  walk.ids = docs ? p.ids + static_cast<size_t>(b) * N : nullptr;
  walk.rows = N;
  walk.first = qstart;
  walk.count = (N - qstart + SR - 1) / SR;
  // causal blocks of a head all end at the last query tile: walking backwards
  // they read each tile at about the same time and share it through L2.  With
  // ids, the first tile is the diagonal one, sure to be needed.
  walk.rev = p.causal != 0 && !docs;
  walk.own = docs && p.causal && qstart == k0;

  Ring ring(smem, tid, D);
  auto fetch = [&](int tile, int g, int stage) {
    const size_t head = qhead0 + g;
    const T* qp = static_cast<const T*>(p.q) + head * N * D;
    const T* dp = static_cast<const T*>(p.dout) + head * N * D;
    const float* lse = p.row_lse + head * N;
    const float* delta = p.delta + head * N;
    if constexpr (DMA) ring.dma(qp, dp, lse, delta, qstart + tile * SR, N, D, stage);
    else ring.load(qp, dp, lse, delta, qstart + tile * SR, N, D);
    if (docs) fetch_ids<SR, DMA>(walk.ids, qstart + tile * SR, N, s_ids[stage]);
  };
  // every read that the walk waits for, before the first wait
  int my_id = 0, wlo = 0, whi = 0, block_id[(RW * kRows + 63) / 64];
  typename TileWalk<SPLIT>::Ids group_ids;
  if (docs) {
    walk.load(group_ids);
    my_id = krow < N ? walk.ids[krow] : -1;
#pragma unroll
    for (int i = 0; i < (RW * kRows + 63) / 64; ++i) {
      const int r = k0 + (lane + 64 * i) % (RW * kRows);
      block_id[i] = r < N ? walk.ids[r] : -1;
    }
  }
  F kf[KK], vf[KK];
  {
    const size_t row = kbase + static_cast<size_t>(min(krow, N - 1)) * D;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      kf[kk] = load_frag<T, ROWS>(static_cast<const T*>(p.k) + row, 16 * kk + 8 * hi, D);
      vf[kk] = load_frag<T, ROWS>(static_cast<const T*>(p.v) + row, 16 * kk + 8 * hi, D);
    }
  }
  if (walk.own) fetch(0, 0, 0);
  if (docs) {
    my_id = my_id < 0 ? kNoId : my_id;
    wlo = wave_min_i(my_id < 0 ? 0x7fffffff : my_id);
    whi = wave_max_i(my_id);
    int lo = 0x7fffffff, top = -1;
#pragma unroll
    for (int i = 0; i < (RW * kRows + 63) / 64; ++i) {
      lo = min(lo, block_id[i] < 0 ? 0x7fffffff : block_id[i]);
      top = max(top, block_id[i]);
    }
    walk.lo = wave_min_i(lo);
    walk.hi = wave_max_i(top);
    walk.digest(group_ids);
  }
  const bool live = krow < N && my_id >= 0;
  const int wid = docs && wlo == whi && __builtin_amdgcn_ballot_w64(my_id != whi) == 0 ? whi : kNoId;
  if (!live) {
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      kf[kk] = zero_frag<T>();
      vf[kk] = zero_frag<T>();
    }
  }
  float16_t dk[DB], dv[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      dk[db][r] = 0.0f;
      dv[db][r] = 0.0f;
    }
  const float c = cap || bias ? 1.0f : p.scale_log2;
  const bool every = !p.causal || wk0 + kRows <= pre;  // every query sees the wave's keys
  const int key_from = p.causal && krow >= pre ? krow : 0;

  const Reader<T, DP> rd(lane);
  constexpr unsigned kSubBytes = kRows * Layout<T, DP>::LD * sizeof(T);
  stream_tiles<T, Ring, DMA, SPLIT>(ring, walk, p.G, sub, s_ids, fetch, [&](int stage, int tile, int g, int id) {
    const int qt = qstart + tile * SR + sub * kRows;
    if (qt >= N || wk0 >= N) return;
    if (!every && wk0 >= pre && qt + kRows <= wk0) return;  // rows before every key of the wave
    if (docs && id >= 0 && (id < wlo || id > whi)) return;
    const unsigned qs = ring.addr_a(stage) + sub * kSubBytes;
    const unsigned ds = ring.addr_b(stage) + sub * kSubBytes;
    // S = Q K^T and dP = dO V^T: lane <-> key, register r <-> query qt + 8 (r/4) + 4 hi + r%4
    float16_t s, dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = 0.0f;
      dp[r] = 0.0f;
    }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      s = mma(rd.row(qs, kk), kf[kk], s);
      dp = mma(rd.row(ds, kk), vf[kk], dp);
    }
    if (cap) {
      cap_scores(s, cap_is_near(s, p), p);
    } else if (bias) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] *= p.scale_log2;
    }
    // derivative of the cap: from the capped score where that is still at hand
    constexpr bool kKeepDt = (MODS & kAnyMods) != 0;
    float16_t dt;
    if constexpr (kKeepDt) {
#pragma unroll
      for (int r = 0; r < 16; ++r) dt[r] = cap ? fmaf(s[r] * s[r], -p.cap_slope, 1.0f) : 1.0f;
    }
    if (bias) add_bias(s, p.slopes[hk * p.G + g] * kLog2e, static_cast<float>(qt + 4 * hi - krow));
    if (qt + kRows > N || (!every && qt < wk0 + kRows - 1)) {
      const int from = key_from - qt - 4 * hi, lim = N - qt - 4 * hi;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int rel = 8 * (r >> 2) + (r & 3);
        s[r] = rel >= from && rel < lim ? s[r] : kDeadScore;
      }
    }
    if (docs && (id < 0 || id != wid)) {
      if (id >= 0) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = my_id == id ? s[r] : kDeadScore;
      } else {
        compare_ids(s_ids[stage] + sub * kRows + 4 * hi, my_id, [&](int r, bool same) { s[r] = same ? s[r] : kDeadScore; });
      }
    }
    const __attribute__((address_space(3))) float* lv = ring.vec(stage, 0) + sub * kRows;
    const __attribute__((address_space(3))) float* dvv = ring.vec(stage, 1) + sub * kRows;
    float16_t pm, dsm;
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
      const float4_t l4 = *reinterpret_cast<const __attribute__((address_space(3))) float4_t*>(lv + 8 * rr + 4 * hi);
      const float4_t d4 = *reinterpret_cast<const __attribute__((address_space(3))) float4_t*>(dvv + 8 * rr + 4 * hi);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * rr + j;
        pm[r] = fast_exp2(fmaf(s[r], c, -l4[j]));
        dsm[r] = (dp[r] - d4[j]) * pm[r];
        if constexpr (kKeepDt) dsm[r] *= dt[r];
        else if (cap) dsm[r] *= fmaf(s[r] * s[r], -p.cap_slope, 1.0f);
      }
    }
    const F pf0 = acc_frag<T>(pm, 0), pf1 = acc_frag<T>(pm, 1);
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      dv[db] = mma(rd.tr(ds, 0, db), pf0, dv[db]);
      dv[db] = mma(rd.tr(ds, 16, db), pf1, dv[db]);
    }
    const F sf0 = acc_frag<T>(dsm, 0), sf1 = acc_frag<T>(dsm, 1);
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      dk[db] = mma(rd.tr(qs, 0, db), sf0, dk[db]);
      dk[db] = mma(rd.tr(qs, 16, db), sf1, dk[db]);
    }
  });

  // ---- join the key block's waves: wave `sub` 0 takes the others' partials ----
  if constexpr (SPLIT > 1) {
    constexpr int REGS = 16 * DB;
    static_assert((SPLIT - 1) * RW * REGS * 256 <= Ring::BYTES, "partials fit the ring");
    auto join = [&](float16_t (&x)[DB]) {
      __syncthreads();  // every wave is done reading the ring (or the previous partials)
      if (sub > 0) {
        lds_ptr<float> out = part_slot<REGS>(smem, wave - RW, lane);
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) out[(16 * db + r) * 64] = x[db][r];
      }
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int w = 0; w < SPLIT - 1; ++w) {
          lds_ptr<float> in = part_slot<REGS>(smem, w * RW + wave, lane);
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) x[db][r] += in[(16 * db + r) * 64];
        }
      }
    };
    join(dv);
    join(dk);
    if (sub > 0) return;
  }

  if (krow >= N) return;
  T* dkp = static_cast<T*>(p.dk) + kbase + static_cast<size_t>(krow) * D;
  T* dvp = static_cast<T*>(p.dv) + kbase + static_cast<size_t>(krow) * D;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
      const int d0 = 32 * db + 8 * rr + 4 * hi;
      auto x = [&](int j) { return dk[db][4 * rr + j] * p.scale; };
      auto y = [&](int j) { return dv[db][4 * rr + j]; };
      store4<T, ROWS>(dkp, d0, D, x(0), x(1), x(2), x(3));
      store4<T, ROWS>(dvp, d0, D, y(0), y(1), y(2), y(3));
    }
}

}  // namespace scored
}  // namespace fa
