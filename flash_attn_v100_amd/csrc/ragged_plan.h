// Splitting a ragged batch of decode calls over workgroups, from the lengths on the device.
#pragma once

#include "common.h"

namespace fa {

#ifndef FA_DEC_CHUNK_QUANTUM
#define FA_DEC_CHUNK_QUANTUM 256
#endif
constexpr int kMaxChunk = 8192;                        // keys per split, upper bound
constexpr int kChunkQuantum = FA_DEC_CHUNK_QUANTUM;    // split boundaries are multiples of this

// A workgroup's share of a continuous-batching or paged call, planned from the
// lengths (each wave for itself: no barrier, one read of the lengths, which
// the static plan waits for as well).  A plan from the longest possible
// sequence alone leaves half of its workgroups empty or short where lengths
// are uniform, and each costs its slot a launch and a read of its length.
// The chunk is the keys of all sequences over kRoundBlocks workgroups (one
// resident round of two per CU); past long_chunk keys, where one round leaves
// the CUs unevenly loaded at its end, over kManyBlocks; and at least what the
// workspace's S splits ask of the longest sequence; paged calls of at least
// kUnsplitUnits units, a resident round by themselves, run unsplit where no
// sequence is long against the batch.  Workgroups first take the full chunks of
// all sequences, which are equal work, then the remainders, in classes of
// length, longest first.
// Uniform lengths, D = 128, 32:8 heads (us, static -> planned): continuous
// batching [64] to 8192 keys 171.7 -> 164.0, [128] to 4096 256 -> 191, [32] to 2048
// 32.3 -> 28.9, [128] to 257 28.6 -> 19.5; paged [128] to 4096 186.6 -> 184.8
// (split in 2048 192), [64] to 8192 212 -> 189, [16] to 2048 26.1 -> 14.1, [64] to
// 1024 34 -> 26.7.  One round against 2048 workgroups: paged [32] to 2048 28.9,
// 31.1; continuous batching [100,32:4] to 1500 26.0, 31.3, but [64] to 8192 209,
// 183.  Equal lengths gain from the round size: continuous batching [16] of 2047
// keys 28.8 -> 25.7, [64] of 4095 178 -> 167; paged [40,64:8] of 2999 pays 87.5 -> 90.9.
// The planning itself is felt where sequences are short or many (R lengths a
// lane), so the class of the remainder sought is found from counts that one
// scan adds up over the wave, and only its members are looked through; with
// every class counted by a ballot a length, in code unrolled 8 R times, one
// long sequence among short ones lost to the static plan (static, ballots,
// scan): continuous batching [400,32:4] to 1500 33.6, 53.1, 32.4, [200] to 1500
// 27.7, 34.7, 24.9, [128] to 2000 35.4, 19.1, 16.3; uniform [256] to 1024 122.1,
// 100.8, 93.0, paged [256] to 2048 183.0, 173.8, 170.8.  Left: sequences of a few
// keys beside one of 600, [400,32:4], 22.2, 40.9, 27.1.
constexpr int kRoundBlocks = 512;
constexpr int kManyBlocks = 2048;
constexpr int kUnsplitUnits = 768;  // a resident round of paged workgroups, three per CU
constexpr int kSplitCost = 256;     // keys that a workgroup walks in the time that splitting costs it
struct RaggedItem {
  int b;  // sequence (-1: none, the workgroup leaves)
  int unit, split, splits, len, chunk;
};

// a / c for 0 <= a < 2^24 and c > 0 with inv = 1 / c
__device__ __forceinline__ int div_by(int a, int c, float inv) {
  int q = static_cast<int>(static_cast<float>(a) * inv);
  const int r = a - q * c;
  return q + (r >= c ? 1 : 0) - (r < 0 ? 1 : 0);
}

// item: which share (the workgroup's number); R: lengths a lane holds (B <= 64 R); len_of(q): keys of sequence q; per_seq:
// units per sequence; plan_len: longest plannable sequence; S: splits a
// sequence has room for; long_chunk: keys past which one round leaves the CUs
// unevenly loaded; unsplit: enough sequences run unsplit.
template <int R, typename LenOf>
__device__ __forceinline__ RaggedItem ragged_item(LenOf&& len_of, int item, int B, int per_seq, int plan_len, int S, int long_chunk,
                                                  bool unsplit) {
  const int lane = threadIdx.x & 63;
  int len[R], plan[R], full[R], upto[R];
  int sum = 0, mx = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int q = lane + 64 * i;
    len[i] = q < B ? len_of(q) : 0;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    plan[i] = max(0, min(len[i], plan_len));
    sum += plan[i];
    mx = max(mx, plan[i]);
  }
  const int total = __builtin_amdgcn_readlane(wave_scan_add(sum), 63);
  const int longest = __builtin_amdgcn_readlane(wave_scan_max(mx), 63);
  const long long keys = static_cast<long long>(total) * per_seq;
  const int round = static_cast<int>((keys + kRoundBlocks - 1) / kRoundBlocks);
  const int many = static_cast<int>((keys + kManyBlocks - 1) / kManyBlocks);
  int want = max(min(round, max(long_chunk, many)), (longest + S - 1) / S);
  // paged: enough sequences to fill the CUs run unsplit (no partials, no second
  // staging of page ids), the length classes below keeping the tail short, if
  // the longest walk ends within the call: a workgroup alone walks 64 keys a us
  // and a full chip takes 12400 keys a us, so a walk is as long as the call at
  // 2.6 shares of a round; beyond two, and what a split costs, it would trail
  // it.  (us, split at kMaxChunk, all unsplit, this rule; 32:8 heads, D = 128)
  // [128] one of 4096 keys, mean 66: 67.7, 64.5, 22.5; a tenth of 4096, mean 703:
  // 85.3, 80.2, 63.2; one of 32768, mean 529: 150, 499, 137; uniform to 32768 1597,
  // 1238, 1225; uniform to 4096 174.9, 171.3, 171.3 (split 175.9).  Equal lengths
  // of 12000, [96], pay: 766, 697, 705.
  if (unsplit && B * per_seq >= kUnsplitUnits && longest <= min(kMaxChunk, 2 * round + kSplitCost))
    want = longest;
  RaggedItem it;
  it.chunk = max(1, (want + kChunkQuantum - 1) / kChunkQuantum) * kChunkQuantum;
  const float inv = 1.0f / static_cast<float>(it.chunk);
  int all = 0;  // full chunks of every sequence
#pragma unroll
  for (int i = 0; i < R; ++i) {
    // (a sequence past its plannable length leaves at least one key to its
    // last split, which takes the rest)
    full[i] = div_by(len[i] > plan_len ? max(0, plan[i] - 1) : plan[i], it.chunk, inv);
    upto[i] = all + wave_scan_add(full[i]);
    all = __builtin_amdgcn_readlane(upto[i], 63);
  }
  it.b = -1;
  it.unit = it.split = it.splits = it.len = 0;
  uint64_t in = 0;      // the lanes that may hold the item's sequence, in block `base` / 64,
  int base = 0;         // and these lanes' values there
  int its_len = 0, its_full = 0, its_before = 0;
  if (item < all * per_seq) {
    const int c = item / per_seq;
    it.unit = item % per_seq;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int before = upto[i] - full[i];
      const uint64_t owner = __builtin_amdgcn_ballot_w64(c >= before && c < upto[i]);
      if (owner != 0) {
        in = owner;
        base = 64 * i;
        its_len = len[i];
        its_full = full[i];
        its_before = before;
      }
    }
    const int l = __builtin_ctzll(in);
    it.b = base + l;
    it.split = c - __builtin_amdgcn_readlane(its_before, l);
    it.len = __builtin_amdgcn_readlane(its_len, l);
    it.splits = __builtin_amdgcn_readlane(its_full, l);
    it.splits += it.len > it.splits * it.chunk ? 1 : 0;
    return it;
  }
  // remainders: the sequences' in eight classes of length, longest first, so
  // that the short ones fill the end of the grid
  int c = (item - all * per_seq) / per_seq;  // c-th remainder of that order
  it.unit = (item - all * per_seq) % per_seq;
  int cls[R];            // class of the lane's sequences (-1: no remainder)
  uint64_t mine = 0;     // how many it has of each: 8 bits a class
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int rest = len[i] - full[i] * it.chunk;  // keys past the full chunks
    const bool has = lane + 64 * i < B && (rest > 0 || len[i] <= 0);
    const int eighth = max(0, min(7, static_cast<int>(static_cast<float>(rest) * (8.0f * inv))));
    cls[i] = has ? eighth : -1;
    mine += has ? 1ull << (8 * eighth) : 0ull;
  }
  // the wave's: 16 bits a class, classes 0 2 | 1 3 | 4 6 | 5 7
  uint32_t counts[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    counts[j] = static_cast<uint32_t>(__builtin_amdgcn_readlane(
        wave_scan_add(static_cast<int>(static_cast<uint32_t>(mine >> (8 * (j & 1) + 32 * (j >> 1))) & 0x00ff00ffu)), 63));
  int its_cls = -1;
#pragma unroll
  for (int k = 7; k >= 0; --k) {
    const int count = static_cast<int>(counts[2 * (k >> 2) + (k & 1)] >> (16 * (k >> 1 & 1)) & 0xffffu);
    if (its_cls < 0) {
      if (c < count) its_cls = k;
      else c -= count;
    }
  }
  if (its_cls < 0) return it;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const uint64_t of_cls = __builtin_amdgcn_ballot_w64(cls[i] == its_cls);
    const int count = __builtin_popcountll(of_cls);
    if (in == 0) {
      if (c < count) {
        in = of_cls;
        base = 64 * i;
        its_len = len[i];
        its_full = full[i];
      } else {
        c -= count;
      }
    }
  }
  const int rank = static_cast<int>(__builtin_amdgcn_mbcnt_hi(
      static_cast<uint32_t>(in >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(in), 0u)));
  const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64((in >> lane & 1) && rank == c));
  it.b = base + l;
  it.len = __builtin_amdgcn_readlane(its_len, l);
  it.split = __builtin_amdgcn_readlane(its_full, l);
  it.splits = it.split + (it.len > 0 ? 1 : 0);
  return it;
}

}  // namespace fa
