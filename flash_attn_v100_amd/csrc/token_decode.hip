// Single-token attention with modified scores for gfx950: over a ragged
// contiguous fp16 cache (optionally adding up each token's softmax weight) and
// over a paged cache held in 8 bits with a scale for each page and head.
//
//   y_t = cap tanh(q.k_t scale / cap) - slope (L - 1 - t)  (either part optional)
//   o = sum_t softmax(y)_t v_t,  weight_out[t] = weight[t] + sum over the KV
//   head's query heads of softmax(y)_t
// with k_t, v_t = code * scale[page of t] in the 8-bit cache.
//
// One workgroup of 4 waves serves up to 16 query heads of one KV head over a
// range of keys; each wave walks 32-key tiles.  Both products run on
// v_mfma_f32_16x16x32_f16, whatever the group's size (decode is bound by the
// cache's bytes, and the products of one 32-key tile at D = 128 are 16 MFMAs of
// 16 cycles against 8 or 16 KB read):
//   S^T = K Q^T     lane <-> head l % 16, 4 keys of each 16-key sub-tile in its
//                   registers: keys 4 (l / 16) .. +3
//   O^T = V^T P^T   P straight from those registers as the B operand; the A
//                   operand's 8 reduction slots of lane group l / 16 are the
//                   same 4 + 4 keys, gathered by the transposing LDS reads
//                   (ds_read_b64_tr_b16: 4 keys x 16 columns a lane group;
//                   ds_read_b64_tr_b8: 8 keys x 16 columns)
// so neither product needs a lane exchange and the softmax statistics are
// per-lane scalars, joined over the 4 lane groups only where the running maximum
// moves, and at the end.
//
// K and V tiles come HBM -> LDS by 16-byte-per-lane copies of whole rows into
// buffers of the wave's own (no barriers in the walk), 16-byte chunks
// XOR-swizzled by row so that both kinds of operand reads hit distinct banks.
// A tile's operands are read into registers as soon as it has landed, and the
// next tile's copies travel while this one is computed.
//
// 8-bit codes become fp16 exactly (both formats fit): a page's K scale
// multiplies its scores and its V scale its probabilities, in fp32.  The
// running reference m follows max(y + log2 v_scale), so what is rounded to fp16,
// p v_scale / 2^m, is at most about 2^8 and anything that flushes there is
// negligible beside the reference term.
//
// Splits and their merge follow decode.hip: plans from the lengths on the
// device (ragged_plan.h), partials and arrival counters in a workspace that is
// zero before and after each call, the last split to arrive merges.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "capi_internal.h"
#include "common.h"
#include "ragged_plan.h"

namespace fa {
namespace token {

enum Cache : int { kF16 = 0, kPagedI8 = 1, kPagedF8 = 2 };

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kTile = 32;   // keys per wave per step
constexpr int kHeads = 16;  // query heads per workgroup
constexpr int kMinPage = 16;
constexpr int kRoundKeys = 4096;  // keys whose page ids and scales are in LDS at a time
constexpr unsigned kCounterSlots = 65536;  // arrival counters at the start of the workspace, as decode.hip's
constexpr int kMaxSplits = 128;
constexpr int kPlanMaxSeqs = 512;
constexpr int kStaticMaxBlocks = 600;
// Ragged plans (ragged_plan.h): chunks past which one round leaves the CUs unevenly
// loaded; enough sequences on the 8-bit cache run unsplit ([128] to 4096 of 32:8 heads
// 103 us, split in 1280 106).
constexpr int kLongChunk = 768;

struct TokenParams {
  const half_t* q;
  const void* k;               // fp16 [B, H_KV, N, D] or codes [pages, H_KV, page, D]
  const void* v;
  const float* k_scale;        // [pages, H_KV]
  const float* v_scale;
  half_t* o;
  const int32_t* lens;
  int len_plus;                // keys of sequence b: lens[b] + len_plus
  const int32_t* block_table;  // [B, max_blocks]
  int max_blocks, num_pages, page_shift;
  const float* slopes;         // [H_Q] or null
  float cap_in, cap_log2;      // scale / cap, cap log2(e); 0 without a cap
  float scale_log2;
  float* scores;               // [B, H_Q, N] log2-domain scores, written if non-null
  float* lse;                  // [B, H_Q] log2-sum-exp, written with them
  float* ws_o;                 // [B*H_Q, S, DP] normalised partial outputs
  float* ws_lse;               // [B*H_Q, S] log2-sum-exp of each
  unsigned* counters;
  int unit_base;
  int B, H_Q, H_KV, N, D, G;   // N: rows of the cache (paged: of a table row)
  int num_hg, chunk, num_splits, ragged;
};

__device__ __forceinline__ int len_of(const TokenParams& p, int b) {
  const long long n = static_cast<long long>(p.lens[b]) + p.len_plus;
  return static_cast<int>(n < 0 ? 0 : (n > p.N ? p.N : n));
}

// Counters of consecutive slots lie in different 128-byte lines.
__device__ __forceinline__ int counter_index(int slot) {
  constexpr int kLines = static_cast<int>(kCounterSlots / 32);
  return (slot % kLines) * 32 + slot / kLines;
}

// Physical 16-byte chunk of logical chunk c in tile row r is c ^ swizzle(r).
// K reads: 16 lanes read rows 0..15 at one chunk.  V reads: 32 lanes read, in
// fp16, rows 8j..8j+7 at two neighbouring chunks, in 8 bits rows 8j..8j+7 and
// 16+8j.. (4 each) at one.  RB: row bytes; rows of less than 256 share a bank window.
template <int RB, int ES>
__device__ __forceinline__ int swizzle_k(int r) {
  return ES == 2 ? (RB >= 256 ? (2 * (r & 7)) ^ ((r >> 3) & 1) : (2 * ((r >> 1) & 3)) ^ ((r >> 3) & 1))
                 : (RB >= 256 ? (r & 15) : (RB == 128 ? (r >> 1) & 7 : (r >> 2) & 3));
}
template <int RB, int ES>
__device__ __forceinline__ int swizzle_v(int r) {
  return ES == 2 ? swizzle_k<RB, 2>(r)
                 : (RB >= 256 ? (r & 7) | ((r >> 4) & 1) << 3
                              : (RB == 128 ? ((r >> 1) & 3) | ((r >> 4) & 1) << 2 : ((r >> 2) & 1) | ((r >> 4) & 1) << 1));
}

// Eight codes as fp16.
template <int CACHE>
__device__ __forceinline__ half8_t codes8(u32x2 raw) {
  half2_t h[4];
  if constexpr (CACHE == kPagedI8) {
    // u = code + 128 under 0x64 is the fp16 value 1024 + u; minus 1152 exact
    const u32x2 x = raw ^ u32x2{0x80808080u, 0x80808080u};
    const half2_t bias = {static_cast<half_t>(-1152.0f), static_cast<half_t>(-1152.0f)};
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      h[2 * w] = as_h2(__builtin_amdgcn_perm(0x64646464u, x[w], 0x05010400u)) + bias;
      h[2 * w + 1] = as_h2(__builtin_amdgcn_perm(0x64646464u, x[w], 0x05030402u)) + bias;
    }
  } else {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      h[2 * w] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[w], 1.0f, false);
      h[2 * w + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[w], 1.0f, true);
    }
  }
  return half8_t{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}

// Every argument at once: left to itself the compiler fetches them in dependent
// rounds behind the early exits, a memory round trip each.
template <int CACHE>
__device__ __forceinline__ void preload_args(const TokenParams& p) {
  asm volatile("" ::"s"(p.q), "s"(p.k), "s"(p.v), "s"(p.o), "s"(p.lens), "s"(p.slopes), "s"(p.scores), "s"(p.lse));
  asm volatile("" ::"s"(p.ws_o), "s"(p.ws_lse), "s"(p.counters), "s"(p.unit_base), "s"(p.len_plus), "s"(p.cap_in), "s"(p.cap_log2));
  asm volatile("" ::"s"(p.B), "s"(p.H_Q), "s"(p.H_KV), "s"(p.N), "s"(p.D), "s"(p.G), "s"(p.num_hg), "s"(p.chunk));
  asm volatile("" ::"s"(p.num_splits), "s"(p.ragged), "s"(p.scale_log2));
  if constexpr (CACHE != kF16)
    asm volatile("" ::"s"(p.k_scale), "s"(p.v_scale), "s"(p.block_table), "s"(p.max_blocks), "s"(p.num_pages), "s"(p.page_shift));
}

// Registers: 8-bit rows of up to 128 leave room for four waves per SIMD, three where D
// is less than the padded width (their tiles are half as large: LDS holds four
// workgroups).
template <int DP, int ROWS, int CACHE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(CACHE != kF16 && DP <= 128 ? (ROWS == kRowFull ? 4 : (ROWS == kRowChunks ? 3 : 1)) : 1))) void token_kernel(
    TokenParams p) {
  constexpr bool C8 = CACHE != kF16;
  constexpr int ES = C8 ? 1 : 2;
  constexpr int RB = DP * ES;               // LDS row bytes
  constexpr int CPR = RB / 16;              // 16-byte chunks per row
  constexpr int COPIES = kTile * CPR / 64;  // copies per lane per tensor per tile
  constexpr int RPC = 64 / CPR;             // rows per copy instruction
  constexpr int NC = DP / 32;               // 32-column slices of Q K^T
  constexpr int NB = DP / 16;               // 16-column blocks of P V
  constexpr int TILE_BYTES = kTile * RB;
  static_assert(COPIES * 64 == kTile * CPR && RPC <= 16, "copy shape");
  __shared__ __attribute__((aligned(1024))) char smem[kWaves * 2 * TILE_BYTES];
  constexpr int kSlots = C8 ? kRoundKeys / kMinPage : 1;
  __shared__ int s_page[kSlots];
  __shared__ float s_ks[kSlots], s_vs[kSlots];
  __shared__ float s_m[kWaves][kHeads], s_l[kWaves][kHeads];
  __shared__ int s_bad, s_last;

  preload_args<CACHE>(p);
  const int S = p.num_splits, D = p.D, G = p.G;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, q4 = lane >> 4;
  int split = static_cast<int>(blockIdx.x) % S;
  int slot = static_cast<int>(blockIdx.x) / S;
  int chunk = p.chunk, L, sb;
  if (p.ragged) {
    auto len = [&](int b) { return len_of(p, b); };
    const int per_seq = p.H_KV * p.num_hg;
    // A page's scales lie side by side for all its heads, one line for the units of a
    // sequence: workgroups go to XCD j % 8, and within every whole 64 of them an XCD takes
    // eight neighbours, so that eight heads share a line in one L2 (step of [128] to 4096 keys
    // 103.4 -> 100.9 us).
    int item = static_cast<int>(blockIdx.x);
    if (C8 && (item | 63) < static_cast<int>(gridDim.x)) item = (item & ~63) | (item & 7) << 3 | (item >> 3 & 7);
    const RaggedItem it = p.B <= 64    ? ragged_item<1>(len, item, p.B, per_seq, p.N, S, kLongChunk, C8)
                          : p.B <= 128 ? ragged_item<2>(len, item, p.B, per_seq, p.N, S, kLongChunk, C8)
                          : p.B <= 256 ? ragged_item<4>(len, item, p.B, per_seq, p.N, S, kLongChunk, C8)
                                       : ragged_item<kPlanMaxSeqs / 64>(len, item, p.B, per_seq, p.N, S, kLongChunk, C8);
    if (it.b < 0) return;
    chunk = it.chunk;
    split = it.split;
    L = it.len;
    sb = it.splits;
    slot = it.b * per_seq + it.unit;
  }
  const int unit = p.unit_base + slot;
  const int hg = unit % p.num_hg;
  const int pair = unit / p.num_hg;
  const int hkv = pair % p.H_KV;
  const int b = pair / p.H_KV;
  if (!p.ragged) {
    L = len_of(p, b);
    sb = (L + chunk - 1) / chunk;
  }
  const int g_base = hg * kHeads;
  const int g_valid = min(kHeads, G - g_base);
  const size_t unit_bh = static_cast<size_t>(b) * p.H_Q + hkv * G + g_base;  // first head of the unit
  // a length past the table row would read another sequence's pages
  const bool too_long = C8 && p.lens[b] > p.N;

  const int k0 = split * chunk;
  const int k1 = min(L, k0 + chunk);
  if (k0 >= k1 || (C8 && p.num_pages == 0)) {
    // nothing to attend: zeros (NaN where there are no pages to attend)
    if (split == 0 && (L <= 0 || C8))
      for (int i = tid; i < g_valid * D; i += kThreads)
        p.o[unit_bh * D + i] = static_cast<half_t>(too_long || L > 0 ? __builtin_nanf("") : 0.0f);
    return;
  }

  // Page ids and scales of the keys [from, to) being walked, at most
  // kRoundKeys of them.  An id outside [0, num_pages) makes the sequence NaN.
  int round = k0;
  auto stage_pages = [&](int from, int to) {
    const int first = from >> p.page_shift;
    const int np = ((to - 1) >> p.page_shift) - first + 1;
    for (int i = tid; i < np; i += kThreads) {
      int id = p.block_table[static_cast<size_t>(b) * p.max_blocks + first + i];
      if (id < 0 || id >= p.num_pages) {
        s_bad = 1;
        id = 0;
      }
      s_page[i] = id;
    }
    round = from;
  };
  // Their scales, read while the first tiles travel.
  auto stage_scales = [&](int from, int to) {
    const int np = ((to - 1) >> p.page_shift) - (from >> p.page_shift) + 1;
    for (int i = tid; i < np; i += kThreads) {
      const size_t at = static_cast<size_t>(s_page[i]) * p.H_KV + hkv;
      s_ks[i] = p.k_scale[at];
      s_vs[i] = p.v_scale[at];
    }
  };
  if constexpr (C8) {
    if (tid == 0) s_bad = too_long ? 1 : 0;
    __syncthreads();
    stage_pages(k0, min(k1, k0 + kRoundKeys));
    __syncthreads();
  }
  auto slot_of = [&](int t) { return (t >> p.page_shift) - (round >> p.page_shift); };

  // ---- Q as the B operand of S^T: head l16, columns k_col(c) .. +8 of slice c ----
  // The score sums over every column whatever the order, so 8-bit rows pair
  // slices (c, c + 1) at 16 contiguous columns 16 q4 + 64 (c / 2) (+8 for c + 1): one
  // 16-byte read of codes per pair.
  auto k_col = [&](int c) {
    if constexpr (C8) return 16 * q4 + 64 * (c / 2) + 8 * (c % 2);
    else return 32 * c + 8 * q4;
  };
  half8_t qf[NC];
  {
    const half_t* row = p.q + (unit_bh + (l16 < g_valid ? l16 : 0)) * D;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      u32x4 x = u32x4{0u, 0u, 0u, 0u};
      if (l16 < g_valid && (ROWS == kRowFull || k_col(c) < D)) x = load_row8<ROWS != kRowElems>(row, k_col(c), D);
      qf[c] = __builtin_bit_cast(half8_t, x);
    }
  }
  const float slope2 = p.slopes != nullptr && l16 < g_valid ? p.slopes[hkv * G + g_base + l16] * kLog2e : 0.0f;
  const bool cap = p.cap_log2 != 0.0f, bias = p.slopes != nullptr;

  // ---- tile copies ----
  const unsigned lds_k = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)smem)) +
                         wave * 2 * TILE_BYTES;
  const unsigned lds_v = lds_k + TILE_BYTES;
  const size_t kv_head = (static_cast<size_t>(b) * p.H_KV + hkv) * static_cast<size_t>(p.N) * D;
  const int klast = k1 - 1;
  typedef __attribute__((address_space(3))) u32x4* lds_u4;
  if constexpr (ROWS == kRowChunks) {
    // chunks past D are never copied; K's meet Q's zeros and must not hold a NaN
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int s = i * 64 + lane, r = s / CPR;
      if (((s % CPR) ^ swizzle_k<RB, ES>(r)) * 16 >= D * ES)
        *reinterpret_cast<lds_u4>(static_cast<size_t>(lds_k + s * 16)) = u32x4{0u, 0u, 0u, 0u};
    }
  }
  // Rows past the last key read that key again (its scores are masked).
  auto issue = [&](int t0) __attribute__((always_inline)) {
#pragma unroll ROWS == kRowElems ? 1 : COPIES
    for (int i = 0; i < COPIES; ++i) {
      const int s = i * 64 + lane;
      const int r = s / CPR;  // tile row
      const int ck = (s % CPR) ^ swizzle_k<RB, ES>(r), cv = (s % CPR) ^ swizzle_v<RB, ES>(r);
      // the copy's rows lie in one group of 16 keys, and so in one page
      const int g0 = C8 ? min(t0 + i * RPC / 16 * 16, klast & ~15) : t0;
      const unsigned row = static_cast<unsigned>(min(t0 + r, klast) - g0);
      const char *kb, *vb;
      if constexpr (C8) {
        const int pg = __builtin_amdgcn_readfirstlane(s_page[slot_of(g0)]);
        const size_t at = (((static_cast<size_t>(pg) * p.H_KV + hkv) << p.page_shift) + (g0 & ((1 << p.page_shift) - 1))) * D;
        kb = static_cast<const char*>(p.k) + at;
        vb = static_cast<const char*>(p.v) + at;
      } else {
        const size_t at = (kv_head + static_cast<size_t>(g0) * D) * 2;
        kb = static_cast<const char*>(p.k) + at;
        vb = static_cast<const char*>(p.v) + at;
      }
      const unsigned dst = i * 1024;
      if constexpr (ROWS == kRowElems) {
        auto elems = [&](const char* base, int c) __attribute__((always_inline)) {
          if constexpr (C8) {
            uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (16 * c + j < D) w[j >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(base[static_cast<size_t>(row) * D + 16 * c + j])) << (8 * (j & 3));
            return u32x4{w[0], w[1], w[2], w[3]};
          } else {
            return load_row8<false>(reinterpret_cast<const half_t*>(base) + static_cast<size_t>(row) * D, 8 * c, D);
          }
        };
        const u32x4 kx = elems(kb, ck), vx = elems(vb, cv);
        *reinterpret_cast<lds_u4>(static_cast<size_t>(lds_k + dst + lane * 16)) = kx;
        *reinterpret_cast<lds_u4>(static_cast<size_t>(lds_v + dst + lane * 16)) = vx;
      } else {
        // (a copy covers whole rows: it has active lanes whatever D)
        if (ROWS == kRowFull || ck * 16 < D * ES)
          copy16_to_lds_nt(reinterpret_cast<const half_t*>(kb), row * D * ES + ck * 16, lds_k + dst);
        if (ROWS == kRowFull || cv * 16 < D * ES)
          copy16_to_lds_nt(reinterpret_cast<const half_t*>(vb), row * D * ES + cv * 16, lds_v + dst);
      }
    }
  };

  float4_t acc[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) acc[nb] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float m = kNegBig, l = 0.0f;  // reference (log2) and this lane's share of the sum
  const int step = kWaves * kTile;
  auto walk = [&](int from, int to) __attribute__((always_inline)) {
    int t0 = from + wave * kTile;
    if (t0 < to) issue(t0);
    if constexpr (C8) {
      stage_scales(from, to);
      __syncthreads();
    }
    while (t0 < to) {
      wait_vm_lgkm0<0>();  // the tile has landed (the copies are this wave's own)
      __builtin_amdgcn_wave_barrier();
      u32x4 kraw[2][C8 ? NC / 2 : NC];
  #pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const int r = 16 * tt + l16;
  #pragma unroll
        for (int c = 0; c < (C8 ? NC / 2 : NC); ++c)
          kraw[tt][c] = *lds_at<u32x4>(lds_k + r * RB + ((4 * c + q4) ^ swizzle_k<RB, ES>(r)) * 16);
      }
      u32x4 vraw[C8 ? 1 : NB];
      u32x2 vraw8[C8 ? NB : 1];
      if constexpr (C8) {
        const int half = l16 >> 1;
        const int r = (half & 3) + 4 * q4 + 16 * (half >> 2);
  #pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          typedef int v2i __attribute__((ext_vector_type(2)));
          const unsigned src = lds_v + r * RB + (nb ^ swizzle_v<RB, 1>(r)) * 16 + (l16 & 1) * 8;
          vraw8[nb] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
              const_cast<__attribute__((address_space(3))) v2i*>(lds_at<v2i>(src))));
        }
      } else {
  #pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          u32x2 part[2];
  #pragma unroll
          for (int tt = 0; tt < 2; ++tt) {
            const int r = 16 * tt + 4 * q4 + (l16 >> 2);
            const unsigned src = lds_v + r * RB + ((2 * nb + ((l16 & 3) >> 1)) ^ swizzle_v<RB, 2>(r)) * 16 + (l16 & 1) * 8;
            part[tt] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                const_cast<__attribute__((address_space(3))) short4_t*>(lds_at<short4_t>(src))));
          }
          vraw[nb] = u32x4{part[0][0], part[0][1], part[1][0], part[1][1]};
        }
      }
      float ks[2] = {1.0f, 1.0f}, vs[2] = {1.0f, 1.0f};
      if constexpr (C8) {
  #pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const int at = slot_of(min(t0 + 16 * tt, klast));
          ks[tt] = s_ks[at];
          vs[tt] = s_vs[at];
        }
      }
      const int tn = t0 + step;
      // the reads have returned before the buffers are overwritten
      __builtin_amdgcn_sched_barrier(0);
      wait_vm_lgkm0<63>();
      __builtin_amdgcn_wave_barrier();
      if (tn < to) issue(tn);
      __builtin_amdgcn_sched_barrier(0);

      // ---- scores, log2 domain ----
      float y[8];
  #pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        float4_t s = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  #pragma unroll
        for (int c = 0; c < NC; ++c) {
          half8_t a;
          if constexpr (C8) a = codes8<CACHE>(c % 2 ? u32x2{kraw[tt][c / 2][2], kraw[tt][c / 2][3]} : u32x2{kraw[tt][c / 2][0], kraw[tt][c / 2][1]});
          else a = __builtin_bit_cast(half8_t, kraw[tt][c]);
          s = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[c], s, 0, 0, 0);
        }
  #pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = s[r] * ks[tt];
          if (cap) {
            // cap log2(e) tanh(z): below |z| = 1/2 by series (common.h), else exponentials
            const float z = x * p.cap_in;
            x = tanh_f32(z) * p.cap_log2;
          } else {
            x *= p.scale_log2;
          }
          if (bias) x = fmaf(-slope2, static_cast<float>(L - 1 - (t0 + 16 * tt + 4 * q4 + r)), x);
          y[4 * tt + r] = x;
        }
      }
      if (p.scores != nullptr && l16 < g_valid) {
        float* row = p.scores + (unit_bh + l16) * p.N;
  #pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int t = t0 + 16 * (j >> 2) + 4 * q4 + (j & 3);
          if (t < k1) row[t] = y[j];
        }
      }
      if (t0 + kTile > k1) {
  #pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = t0 + 16 * (j >> 2) + 4 * q4 + (j & 3) < k1 ? y[j] : -INFINITY;
      }
      // ---- probabilities against the reference, raised only when one outgrows it by 2^8 ----
      float e[8], w[8];
      auto exponentiate = [&]() __attribute__((always_inline)) {
        float sum = 0.0f;
  #pragma unroll
        for (int j = 0; j < 8; ++j) {
          e[j] = fast_exp2(y[j] - m);
          w[j] = C8 ? e[j] * vs[j >> 2] : e[j];
          sum += w[j];
        }
        return sum;
      };
      float sum = exponentiate();
      if (__builtin_amdgcn_ballot_w64(!(sum <= 256.0f)) != 0) {
        float mx = -INFINITY;
  #pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const float lv = C8 ? __log2f(fmaxf(vs[tt], 0x1p-60f)) : 0.0f;
  #pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, y[4 * tt + r] + lv);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mn = fmaxf(m, mx);
        const float alpha = fast_exp2(m - mn);
        m = mn;
        l *= alpha;
  #pragma unroll
        for (int nb = 0; nb < NB; ++nb) acc[nb] *= alpha;
        exponentiate();
      }
      half8_t pf;
  #pragma unroll
      for (int j = 0; j < 8; ++j) {
        l += e[j];
        pf[j] = static_cast<half_t>(w[j]);
      }
      // ---- O^T += V^T P^T ----
  #pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const half8_t a = C8 ? codes8<C8 ? CACHE : kPagedI8>(vraw8[C8 ? nb : 0]) : __builtin_bit_cast(half8_t, vraw[C8 ? 0 : nb]);
        acc[nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pf, acc[nb], 0, 0, 0);
      }
      t0 = tn;
    }
  };
  if constexpr (C8) {
    static_assert(kRoundKeys % (kWaves * kTile) == 0 && kRoundKeys % 256 == 0, "rounds hold whole steps and pages");
    for (int rb = k0; rb < k1; rb += kRoundKeys) {
      const int re = min(k1, rb + kRoundKeys);
      if (rb != k0) {
        __syncthreads();  // every wave is done with the previous round's ids
        stage_pages(rb, re);
        __syncthreads();
      }
      walk(rb, re);
    }
  } else {
    walk(k0, k1);
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // ---- merge the waves through LDS (the tile buffers, done with) ----
  __syncthreads();
  static_assert(kHeads * DP * 4 <= 2 * TILE_BYTES, "a wave's partial fits its tile buffers");
  float* part = reinterpret_cast<float*>(smem);  // [wave][head][DP], 16-byte chunks XORed by head
  if (q4 == 0) {
    s_m[wave][l16] = m;
    s_l[wave][l16] = l;
  }
  if (l16 < g_valid) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      *reinterpret_cast<float4_t*>(part + (wave * kHeads + l16) * DP + ((4 * nb + q4) ^ l16) * 4) = acc[nb];
  }
  __syncthreads();
  const bool bad = C8 && s_bad != 0;
  constexpr int NC4 = DP / 4;
  for (int i = tid; i < g_valid * NC4; i += kThreads) {
    const int g = i / NC4, d4 = (i % NC4) * 4;
    if (d4 >= D) continue;
    float mx = s_m[0][g];
#pragma unroll
    for (int wv = 1; wv < kWaves; ++wv) mx = fmaxf(mx, s_m[wv][g]);
    float lsum = 0.0f;
    float4_t a = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int wv = 0; wv < kWaves; ++wv) {
      const float al = fast_exp2(s_m[wv][g] - mx);
      lsum += s_l[wv][g] * al;
      a += *reinterpret_cast<const float4_t*>(part + (wv * kHeads + g) * DP + ((d4 / 4) ^ g) * 4) * al;
    }
    float4_t out = a / lsum;
    float lse = mx + __log2f(lsum);
    if (bad) {
      lse = __builtin_nanf("");
      out = float4_t{lse, lse, lse, lse};
    }
    if (sb == 1) {
      half_t* op = p.o + (unit_bh + g) * D + d4;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (d4 + j < D) op[j] = static_cast<half_t>(out[j]);
      if (p.lse != nullptr && d4 == 0) p.lse[unit_bh + g] = lse;
    } else {
      const size_t at = (unit_bh + g) * S + split;
      store_coherent4(&p.ws_o[at * DP + d4], out);
      if (d4 == 0) store_coherent(&p.ws_lse[at], lse);
    }
  }
  if (sb == 1) return;

  // ---- publish; the last split to arrive merges (as decode.hip) ----
  wait_vmem_stores();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(&p.counters[counter_index(slot)], 1u) == static_cast<unsigned>(sb - 1);
  __syncthreads();
  if (!s_last) return;
  if (tid == 0) __hip_atomic_store(&p.counters[counter_index(slot)], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const __amdgpu_buffer_rsrc_t o_rsrc = __builtin_amdgcn_make_buffer_rsrc(p.ws_o + unit_bh * S * DP, 0, 0x7fffffff, 0x00020000);
  const __amdgpu_buffer_rsrc_t lse_rsrc = __builtin_amdgcn_make_buffer_rsrc(p.ws_lse + unit_bh * S, 0, 0x7fffffff, 0x00020000);
  // columns of 4 outputs over the threads, spare threads taking splits in phases
  const int ncol = g_valid * NC4;
  const int phases = ncol >= kThreads ? 1 : kThreads / ncol;
  constexpr int BATCH = C8 ? 8 : 20;  // loads in flight: a phase of a 33-split merge waits once
  float4_t* s_num = reinterpret_cast<float4_t*>(smem);                       // [kThreads]
  float* s_den = reinterpret_cast<float*>(smem) + 4 * kThreads;              // [kThreads]
  float* s_max = s_den + kThreads;                                           // [kThreads]
  for (int c0 = 0; c0 < ncol; c0 += kThreads) {
    const int c = phases > 1 ? tid % ncol : c0 + tid;
    const int ph = phases > 1 ? tid / ncol : 0;
    const int g = c / NC4, d4 = (c % NC4) * 4;
    float4_t num = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float den = 0.0f, mx = -INFINITY;
    if (c < ncol && ph < phases && d4 < D) {
      for (int s0 = ph; s0 < sb; s0 += BATCH * phases) {
        float4_t v[BATCH];
        float lv[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const int sp = s0 + j * phases;
          v[j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
          lv[j] = -INFINITY;
          if (sp < sb) {
            v[j] = __builtin_bit_cast(float4_t, __builtin_amdgcn_raw_buffer_load_b128(o_rsrc, ((g * S + sp) * DP + d4) * 4, 0, 16));
            lv[j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(lse_rsrc, (g * S + sp) * 4, 0, 16));
          }
        }
        // (a NaN partial stays NaN through its own term)
        float mn = mx;
#pragma unroll
        for (int j = 0; j < BATCH; ++j) mn = fmaxf(mn, lv[j]);
        const float al = fast_exp2(mx - mn);
        num *= al;
        den *= al;
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const float wj = s0 + j * phases < sb ? fast_exp2(lv[j] - mn) : 0.0f;
          den += wj;
          num += wj * v[j];
        }
        mx = mn;
      }
    }
    if (phases > 1) {
      __syncthreads();
      s_num[tid] = num;
      s_den[tid] = den;
      s_max[tid] = mx;
      __syncthreads();
      if (tid >= ncol) continue;
      float mn = mx;
      for (int q = 1; q < phases; ++q) mn = fmaxf(mn, s_max[q * ncol + tid]);
      const float al = fast_exp2(mx - mn);
      num *= al;
      den *= al;
      for (int q = 1; q < phases; ++q) {
        const float mq = s_max[q * ncol + tid];
        const float wq = mq == -INFINITY ? 0.0f : fast_exp2(mq - mn);
        num += wq * s_num[q * ncol + tid];
        den += wq * s_den[q * ncol + tid];
      }
      mx = mn;
    }
    if (c >= ncol || d4 >= D) continue;
    half_t* op = p.o + (unit_bh + g) * D + d4;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (d4 + j < D) op[j] = static_cast<half_t>(num[j] / den);
    if (p.lse != nullptr && d4 == 0) p.lse[unit_bh + g] = mx + __log2f(den);
  }
}

// weight_out[b, h_kv, t] = weight[b, h_kv, t] + sum over the KV head's query
// heads of exp2(score - lse), for the keys of each sequence; other entries are
// left as they are.  VEC: four keys a thread (N % 4 == 0, aligned arrays).
template <bool VEC>
__global__ __launch_bounds__(kThreads) void add_weights_kernel(TokenParams p, const float* weight, float* weight_out) {
  constexpr int K = VEC ? 4 : 1;
  typedef float vec __attribute__((ext_vector_type(K)));
  const int pair = blockIdx.y;
  const int b = pair / p.H_KV, hkv = pair % p.H_KV;
  const int L = len_of(p, b);
  const int t = (static_cast<int>(blockIdx.x) * kThreads + threadIdx.x) * K;
  if (t >= L) return;
  const size_t bh = static_cast<size_t>(b) * p.H_Q + hkv * p.G;
  const size_t at = static_cast<size_t>(pair) * p.N + t;
  vec sum = *reinterpret_cast<const vec*>(weight + at);
  for (int g = 0; g < p.G; ++g) {
    // (scores past the last key were never written: what comes of them is not stored)
    const vec s = *reinterpret_cast<const vec*>(p.scores + (bh + g) * p.N + t);
    const float lse = p.lse[bh + g];
#pragma unroll
    for (int j = 0; j < K; ++j) sum[j] += fast_exp2(s[j] - lse);
  }
  if (t + K <= L) {
    *reinterpret_cast<vec*>(weight_out + at) = sum;
  } else {
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (t + j < L) weight_out[at + j] = sum[j];
  }
}

// ---------------------------------------------------------------------------
// Host side

static size_t align256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

template <int CACHE>
static void dispatch(int dp, int rows, const TokenParams& p, int blocks, hipStream_t st) {
  constexpr std::integral_constant<int, 64> w64;
  constexpr std::integral_constant<int, 128> w128;
  constexpr std::integral_constant<int, 256> w256;
  auto by_rows = [&](auto w) {
    const dim3 grid(blocks), block(kThreads);
    if (rows == kRowFull) hipLaunchKernelGGL((token_kernel<w(), kRowFull, CACHE>), grid, block, 0, st, p);
    else if (rows == kRowChunks) hipLaunchKernelGGL((token_kernel<w(), kRowChunks, CACHE>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((token_kernel<w(), kRowElems, CACHE>), grid, block, 0, st, p);
  };
  if (dp == 64) by_rows(w64);
  else if (dp == 128) by_rows(w128);
  else by_rows(w256);
}

// Splits of equal chunks for about `target` workgroups: chunks of a multiple of 128
// keys (one tile a wave), at most kMaxChunk keys and kMaxSplits of them.
// fa_decode_workspace_size covers it: its bound takes the same quantum and a
// target of kRaggedTarget.
constexpr int kStaticTarget = 1024;
constexpr int kRaggedTarget = 4096;
constexpr int kQuantum = kWaves * kTile;

struct Splits {
  long long chunk, count;
};
static Splits plan_splits(long long len, long long units, int target) {
  long long chunk = std::max((len * units + target - 1) / target, (len + kMaxSplits - 1) / kMaxSplits);
  chunk = std::min<long long>((chunk + kQuantum - 1) / kQuantum * kQuantum, kMaxChunk);
  return {chunk, (len + chunk - 1) / chunk};
}

template <int CACHE>
static int run(const char* fn, TokenParams p, float softcap, void* ws, size_t ws_bytes, hipStream_t st) {
  if (softcap != 0.0f && !(softcap >= 1e-2f && softcap <= 1e3f))
    return set_error(FA_ERR_INVALID_ARG, "%s: softcap must be 0 (none) or lie in [0.01, 1000]", fn);
  p.G = p.H_Q / p.H_KV;
  p.num_hg = ceil_div(p.G, kHeads);
  const float scale = 1.0f / sqrtf(static_cast<float>(p.D));
  p.scale_log2 = scale * kLog2e;
  p.cap_in = softcap != 0.0f ? scale / softcap : 0.0f;
  p.cap_log2 = softcap * kLog2e;
  const int dp = p.D <= 64 ? 64 : (p.D <= 128 ? 128 : 256);
  const long long units = static_cast<long long>(p.B) * p.H_KV * p.num_hg;
  const long long len = std::max(p.N, 1);
  Splits plan = plan_splits(len, units, kStaticTarget);
  // more work than is resident at once: planned from the lengths on the device,
  // with room for shorter splits
  const bool many = units * plan.count > kStaticMaxBlocks && p.B <= kPlanMaxSeqs && units <= static_cast<long long>(kCounterSlots);
  if (many) plan = plan_splits(len, units, kRaggedTarget);
  const long long splits = plan.count;
  if (splits > kMaxSplits)
    return set_error(FA_ERR_UNSUPPORTED, "%s: %d keys per sequence exceed %d", fn, p.N, kMaxSplits * kMaxChunk);
  p.chunk = static_cast<int>(plan.chunk);
  p.num_splits = static_cast<int>(splits);
  if (splits > 1) {
    const size_t entries = static_cast<size_t>(p.B) * p.H_Q * splits;
    const size_t lse_at = align256(kCounterSlots * sizeof(unsigned));
    const size_t o_at = lse_at + align256(entries * sizeof(float));
    const size_t need = o_at + entries * dp * sizeof(float);
    if (ws == nullptr || ws_bytes < need)
      return set_error(FA_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", fn, need, ws_bytes);
    char* base = static_cast<char*>(ws);
    p.counters = reinterpret_cast<unsigned*>(base);
    p.ws_lse = reinterpret_cast<float*>(base + lse_at);
    p.ws_o = reinterpret_cast<float*>(base + o_at);
  }
  if (p.B == 0) return FA_OK;
  // Vector paths: every row starts 16-byte aligned and is whole 16-byte chunks.
  const int per_chunk = CACHE == kF16 ? 8 : 16;
  const bool vec = aligned16(p.q) && aligned16(p.k) && aligned16(p.v) && p.D % per_chunk == 0;
  const int rows = !vec ? kRowElems : (p.D == dp ? kRowFull : kRowChunks);
  if (many && splits > 1) {
    const long long full = std::max<long long>(kRoundBlocks, std::min<long long>(kManyBlocks, units * len / kLongChunk));
    p.ragged = 1;
    dispatch<CACHE>(dp, rows, p, static_cast<int>(full + units), st);
    return check_launch(fn);
  }
  for (long long u0 = 0; u0 < units; u0 += kCounterSlots) {
    p.unit_base = static_cast<int>(u0);
    dispatch<CACHE>(dp, rows, p, static_cast<int>(std::min<long long>(units - u0, kCounterSlots) * splits), st);
    if (const int rc = check_launch(fn)) return rc;
  }
  return FA_OK;
}

static int check_sizes(const char* fn, int B, int H_Q, int H_KV, int D) {
  if (B < 0 || H_Q <= 0 || H_KV <= 0 || D <= 0)
    return set_error(FA_ERR_INVALID_ARG, "%s: sizes must be positive (B=%d H_Q=%d H_KV=%d D=%d)", fn, B, H_Q, H_KV, D);
  if (H_Q < H_KV || H_Q % H_KV != 0)
    return set_error(FA_ERR_INVALID_ARG, "%s: H_Q (%d) must be a multiple of H_KV (%d)", fn, H_Q, H_KV);
  if (D > 256) return set_error(FA_ERR_UNSUPPORTED, "%s: D=%d exceeds 256", fn, D);
  if (static_cast<long long>(B) * H_Q > 0x3fffffffLL)
    return set_error(FA_ERR_UNSUPPORTED, "%s: too many heads (B=%d H_Q=%d)", fn, B, H_Q);
  return FA_OK;
}

static int contiguous(const char* fn, const void* q, const void* k, const void* v, void* o, const int32_t* cache_lens,
                      const float* weight, float* weight_out, bool weighted, int B, int H_Q, int H_KV, int N, int D,
                      float softcap, const float* slopes, float* scores, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = check_sizes(fn, B, H_Q, H_KV, D)) return rc;
  if (N <= 0) return set_error(FA_ERR_INVALID_ARG, "%s: N must be positive", fn);
  if (B > 0 && (!q || !k || !v || !o || !cache_lens)) return set_error(FA_ERR_INVALID_ARG, "%s: null pointer", fn);
  if (weighted && (reinterpret_cast<uintptr_t>(scores) & 15) != 0)
    return set_error(FA_ERR_INVALID_ARG, "%s: scratch must be 16-byte aligned", fn);
  if (B > 0 && weighted && (!weight || !weight_out || !scores)) return set_error(FA_ERR_INVALID_ARG, "%s: null pointer", fn);
  // one array, or two apart: in between, a sum would be read as another key's weight
  const size_t weight_bytes = static_cast<size_t>(B) * H_KV * N * sizeof(float);
  const uintptr_t w0 = reinterpret_cast<uintptr_t>(weight), w1 = reinterpret_cast<uintptr_t>(weight_out);
  if (weighted && w0 != w1 && w0 < w1 + weight_bytes && w1 < w0 + weight_bytes)
    return set_error(FA_ERR_INVALID_ARG, "%s: weight and weight_out overlap in part", fn);
  if (weighted && static_cast<long long>(B) * H_KV > 65535)
    return set_error(FA_ERR_UNSUPPORTED, "%s: more than 65535 (sequence, KV head) pairs", fn);
  TokenParams p = {};
  p.q = static_cast<const half_t*>(q);
  p.k = k;
  p.v = v;
  p.o = static_cast<half_t*>(o);
  p.lens = cache_lens;
  p.len_plus = 1;
  p.slopes = slopes;
  p.B = B; p.H_Q = H_Q; p.H_KV = H_KV; p.N = N; p.D = D;
  if (weighted) {
    p.scores = scores;
    p.lse = scores + static_cast<size_t>(B) * H_Q * N;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int rc = run<kF16>(fn, p, softcap, ws, ws_bytes, st);
  if (rc != FA_OK || !weighted || B == 0) return rc;
  p.G = H_Q / H_KV;
  const bool vec = N % 4 == 0 && aligned16(weight) && aligned16(weight_out) && aligned16(scores);
  const dim3 grid(ceil_div(N, kThreads * (vec ? 4 : 1)), B * H_KV);
  if (vec) hipLaunchKernelGGL(add_weights_kernel<true>, grid, dim3(kThreads), 0, st, p, weight, weight_out);
  else hipLaunchKernelGGL(add_weights_kernel<false>, grid, dim3(kThreads), 0, st, p, weight, weight_out);
  return check_launch(fn);
}

}  // namespace token
}  // namespace fa

using namespace fa;

extern "C" int fa_decode_scored_fp16(const void* q, const void* k, const void* v, void* o, const int32_t* cache_lens, int B,
                                     int H_Q, int H_KV, int N, int D, float softcap, const float* slopes, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  return token::contiguous("fa_decode_scored_fp16", q, k, v, o, cache_lens, nullptr, nullptr, false, B, H_Q, H_KV, N, D, softcap,
                           slopes, nullptr, workspace, workspace_bytes, stream);
}

extern "C" size_t fa_decode_weighted_scratch_size(int B, int H_Q, int N) {
  if (B <= 0 || H_Q <= 0 || N <= 0) return 0;
  return static_cast<size_t>(B) * H_Q * (static_cast<size_t>(N) + 1) * sizeof(float);
}

extern "C" int fa_decode_weighted_fp16(const void* q, const void* k, const void* v, void* o, const int32_t* cache_lens,
                                       const float* weight, float* weight_out, int B, int H_Q, int H_KV, int N, int D,
                                       float softcap, const float* slopes, void* scratch, size_t scratch_bytes, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  const char* fn = "fa_decode_weighted_fp16";
  const size_t need = fa_decode_weighted_scratch_size(B, H_Q, N);
  if (need > 0 && (!scratch || scratch_bytes < need))
    return set_error(FA_ERR_WORKSPACE, "%s: scratch of %zu bytes needed, %zu given", fn, need,
                     scratch ? scratch_bytes : static_cast<size_t>(0));
  return token::contiguous(fn, q, k, v, o, cache_lens, weight, weight_out, true, B, H_Q, H_KV, N, D, softcap, slopes,
                           static_cast<float*>(scratch), workspace, workspace_bytes, stream);
}

extern "C" int fa_paged_decode_kv8(const void* q, const void* k_cache, const void* v_cache, const float* k_scale,
                                   const float* v_scale, void* o, const int32_t* block_table, const int32_t* seq_lens, int fp8,
                                   int B, int H_Q, int H_KV, int D, int num_pages, int page, int max_blocks, float softcap,
                                   const float* slopes, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "fa_paged_decode_kv8";
  if (const int rc = token::check_sizes(fn, B, H_Q, H_KV, D)) return rc;
  if (page < token::kMinPage || page > 256 || (page & (page - 1)) != 0)
    return set_error(FA_ERR_UNSUPPORTED, "%s: page of %d tokens is not 16, 32, 64, 128 or 256", fn, page);
  if (num_pages < 0 || max_blocks < 0)
    return set_error(FA_ERR_INVALID_ARG, "%s: negative page count / table size", fn);
  if (B > 0 && (!q || !o || !seq_lens || ((!k_cache || !v_cache || !k_scale || !v_scale || !block_table) && num_pages > 0 && max_blocks > 0)))
    return set_error(FA_ERR_INVALID_ARG, "%s: null pointer", fn);
  const long long keys = static_cast<long long>(max_blocks) * page;
  if (keys > 0x3fffffffLL) return set_error(FA_ERR_UNSUPPORTED, "%s: max_blocks too large", fn);
  token::TokenParams p = {};
  p.q = static_cast<const half_t*>(q);
  p.k = k_cache;
  p.v = v_cache;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.o = static_cast<half_t*>(o);
  p.lens = seq_lens;
  p.block_table = block_table;
  p.max_blocks = max_blocks;
  p.num_pages = num_pages;
  p.page_shift = __builtin_ctz(static_cast<unsigned>(page));
  p.slopes = slopes;
  p.B = B; p.H_Q = H_Q; p.H_KV = H_KV; p.N = static_cast<int>(keys); p.D = D;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return fp8 ? token::run<token::kPagedF8>(fn, p, softcap, workspace, workspace_bytes, st)
             : token::run<token::kPagedI8>(fn, p, softcap, workspace, workspace_bytes, st);
}
