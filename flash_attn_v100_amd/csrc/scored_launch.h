// Launches of the scored-attention kernels, shared by the fp16 and the fp32
// translation unit.
#pragma once

#include <algorithm>
#include <type_traits>

#include "capi_internal.h"
#include "scored_kernels.h"

namespace fa {
namespace scored {

// Deals `units` of `heads` heads over the XCDs (map_block).  Units that do not
// fill the XCDs evenly leave some of them idle, so fewer than 32 that are no
// multiple of eight are dealt block by block instead (group_units 0).
inline long long deal(ScoredParams& p, long long units, int heads) {
  p.units = static_cast<int>(units);
  p.heads = heads;
  if (units % kXcds != 0 && units < 4 * kXcds) {
    p.group_units = 0;
    return units * heads * p.nblk;
  }
  const long long per_xcd = (units + kXcds - 1) / kXcds;
  const long long per_unit = static_cast<long long>(heads) * p.nblk;
  constexpr long long kGroupWorkgroups = 128;  // an XCD's blocks in flight, about
  p.group_units = static_cast<int>(std::max<long long>(1, std::min(per_xcd, (kGroupWorkgroups + per_unit - 1) / per_unit)));
  return (per_xcd + p.group_units - 1) / p.group_units * p.group_units * kXcds * per_unit;
}

// A query-major grid: the heads of a KV head share a unit where the units then
// still fill the XCDs.
inline long long deal_query(ScoredParams& p) {
  const long long units = static_cast<long long>(p.B) * p.H_KV;
  if (units % kXcds == 0 || units >= 4 * kXcds) return deal(p, units, p.G);
  return deal(p, static_cast<long long>(p.B) * p.H_Q, 1);
}

// Calls run(SPLIT) with the waves that share a row block as a compile-time number:
// 1, 2, or 4 where four waves' tiles fit LDS (fp16 rows of at most 128, fp32 of 64).
template <typename T, int DP, int ROWS, typename Run>
void by_split(int split, Run&& run) {
  if constexpr (ROWS != kRowElems) {
    if constexpr (DP * sizeof(T) <= 256) {
      if (split == 4) return run(std::integral_constant<int, 4>());
    }
    if (split >= 2) return run(std::integral_constant<int, 2>());
  }
  run(std::integral_constant<int, 1>());
}

// Whether a causal call's blocks are dealt as a snake (map_block), by the
// workgroups of its grid (us, heavy first -> snake): fp32 forward [2,16,1000,64], 512 of
// them, 72 -> 60, backward 218 -> 174; fp16 backward [4,16,2048,128], 1024, 321 -> 310; but
// forward [4,16,2048,128], 1024, 97 -> 105, fp32 [4,16,2048,64] 315 -> 340, backward
// [8,32:8,2048,64], 4096, 695 -> 734.  With documents walks do not grow down the rows.
inline int snake_order(const ScoredParams& p, long long workgroups, bool backward) {
  return p.causal && !p.ids && workgroups <= (backward ? 1024 : 512);
}

template <typename T, int DP, int DC, int ROWS, int MODE, int MODS>
void launch_query(ScoredParams p, int split, hipStream_t st) {
  by_split<T, DP, ROWS>(split, [&](auto s) {
    p.nblk = ceil_div(p.N, kBlockRows / s());
    const long long blocks = deal_query(p);
    p.snake = snake_order(p, blocks, MODE == 1);
    hipLaunchKernelGGL((scored_query_kernel<T, DP, DC, ROWS, MODE, s(), MODS>), dim3(static_cast<unsigned>(blocks)),
                       dim3(kThreads), 0, st, p);
  });
}

template <typename T, int DP, int DC, int ROWS, int MODS>
void launch_key(ScoredParams p, int split, hipStream_t st) {
  by_split<T, DP, ROWS>(split, [&](auto s) {
    p.nblk = ceil_div(p.N, kBlockRows / s());
    const long long blocks = deal(p, static_cast<long long>(p.B) * p.H_KV, 1);
    p.snake = snake_order(p, blocks, true);
    hipLaunchKernelGGL((scored_key_kernel<T, DP, DC, ROWS, s(), MODS>), dim3(static_cast<unsigned>(blocks)),
                       dim3(kThreads), 0, st, p);
  });
}

// Waves that share a row block (each walks 1 / split of its tiles), by the 128-row
// blocks of the call: few blocks leave CUs idle or with little to switch to, and are
// bound by the longest walk.  Four against one, 16 blocks, [1,8,256,64]: forward 6.7 us
// for 10.4, dQ 7.7 for 13.0, key kernel 7.8 for 13.3; the fp32 step [2,16,1000,64], 256
// blocks, 242 for 392.  With enough blocks the split only adds its join: prefill
// [8,16,577,80], 640 blocks, 38.5 unsplit, 53.3 in two.  The key kernel at 512 blocks
// (documents [4,32:8,2048,128]): in two 248, unsplit 314.
inline int split_query(const ScoredParams& p, bool backward) {
  const long long blocks = static_cast<long long>(p.B) * p.H_Q * ceil_div(p.N, kBlockRows);
  if (blocks <= 64) return 4;
  if (blocks <= 256) return 2;
  return blocks <= 512 && (backward || (p.causal && p.N > 1024)) ? 2 : 1;
}
inline int split_key(const ScoredParams& p) {
  const long long blocks = static_cast<long long>(p.B) * p.H_KV * ceil_div(p.N, kBlockRows);
  return blocks <= 64 ? 4 : (blocks <= 512 ? 2 : 1);
}

template <typename T, int DP, int DC, int ROWS, int MODS>
void launch_backward_shape(const ScoredParams& p, hipStream_t st) {
  launch_query<T, DP, DC, ROWS, 1, MODS>(p, split_query(p, true), st);
  launch_key<T, DP, DC, ROWS, MODS>(p, split_key(p), st);
}

// Calls run with the variant of the call's modifications: those met in practice
// have one of their own, what is left reads them from the parameters.
// Compiled in, prefill [1,32:8,8192,128] with a cap takes 658 us for 690, a training
// layer of documents [4,32:8,2048,128] 495 for 633.
template <typename Run>
void by_mods(int mods, Run&& run) {
  switch (mods) {
    case 0: run(std::integral_constant<int, 0>()); break;
    case kCap: run(std::integral_constant<int, kCap>()); break;
    case kBias: run(std::integral_constant<int, kBias>()); break;
    case kDocs: run(std::integral_constant<int, kDocs>()); break;
    case kCap | kDocs: run(std::integral_constant<int, kCap | kDocs>()); break;
    case kBias | kDocs: run(std::integral_constant<int, kBias | kDocs>()); break;
    default: run(std::integral_constant<int, kAnyMods>());
  }
}

// fp16 shapes: padded width DP, computed columns DC, row mode (elems: no vector
// rows, and every modification read from the parameters).  WIDE: D up to 256.
template <bool WIDE, typename Run>
void by_shape_fp16(int D, bool vec, int mods, Run&& run) {
  constexpr std::integral_constant<int, 64> w64;
  constexpr std::integral_constant<int, 96> w96;
  constexpr std::integral_constant<int, 128> w128;
  constexpr std::integral_constant<int, 192> w192;
  constexpr std::integral_constant<int, 256> w256;
  constexpr std::integral_constant<int, kRowElems> elems;
  constexpr std::integral_constant<int, kRowFull> full;
  constexpr std::integral_constant<int, kRowChunks> chunks;
  constexpr std::integral_constant<int, kAnyMods> any;
  if (!vec || D % 8 != 0) {
    if (D <= 64) run(w64, w64, elems, any);
    else if (D <= 128) run(w128, w128, elems, any);
    else if constexpr (WIDE) run(w256, w256, elems, any);
    return;
  }
  by_mods(mods, [&](auto m) {
    if (D == 64) run(w64, w64, full, m);
    else if (D < 64) run(w64, w64, chunks, m);
    else if (D <= 96) run(w128, w96, chunks, m);
    else if (D == 128) run(w128, w128, full, m);
    else if (D < 128) run(w128, w128, chunks, m);
    else if constexpr (WIDE) {
      if (D == 256) run(w256, w256, full, m);
      else if (D <= 192) run(w256, w192, chunks, m);
      else run(w256, w256, chunks, m);
    }
  });
}

// Entry points of the other translation units.
void backward_fp16(const ScoredParams& p, bool vec, hipStream_t st);
void forward_fp32(const ScoredParams& p, bool vec, hipStream_t st);
void backward_fp32(const ScoredParams& p, bool vec, hipStream_t st);

}  // namespace scored
}  // namespace fa
