// KV-cache maintenance for gfx950: the append that writes a paged cache held in
// 8 bits, and the eviction of a cache's lightest tokens.
//
// ---- append (fa_paged_append_kv8) ----
// A page of one head has one scale for its keys and one for its values:
//   scale = max |x| (1 / top) over the page's tokens (top: 127 int8, 448 e4m3)
//   code  = x / scale rounded to nearest even
// A page that already holds tokens keeps the larger of its scale and the new
// tokens' one; where it grows, the old codes are rounded again, code * old /
// new.  All of it is IEEE fp32 arithmetic as written (1 / top rounded, one
// product; the quotients correctly rounded), so codes are reproducible.
// One wave per (page, head, K or V) does all of it: it alone reads and writes
// that page's codes and scale, so no barrier and no atomics.  Bound by bytes
// (2 read and 1 written a value): up to four 16-value chunks a lane stay in
// registers between the maximum and the rounding (16 tokens at D = 256, 32 at
// D = 128); longer pages are read again, from L2.
//
// ---- eviction (fa_evict_by_weight) ----
// Per (sequence, KV head), of L tokens the last `recent` are kept and, of the
// others, the budget - recent heaviest (ties: lower index first; NaN lightest),
// in their order.  A workgroup a head finds the threshold weight by a radix
// select (digits of 11, 11 and 10 bits over LDS histograms), turns it into the map
// row -> source token with one ballot scan, and a second kernel, with a
// workgroup per 32 rows, copies the K and V rows of that map: the
// part that is bound by bytes needs more workgroups than there are heads.
#include <type_traits>

#include "capi_internal.h"
#include "common.h"

namespace fa {
namespace kvops {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

struct AppendParams {
  const half_t* k;  // new tokens [total, H_KV, D]
  const half_t* v;
  const int32_t* cu;          // [B + 1]
  const int32_t* cache_lens;  // [B] tokens already there
  uint8_t* k_cache;           // codes [pages, H_KV, page, D]
  uint8_t* v_cache;
  float* k_scale;  // [pages, H_KV]
  float* v_scale;
  const int32_t* block_table;  // [B, max_blocks]
  int B, H_KV, D, total, max_new, num_pages, page_shift, max_blocks;
  int pages_per_seq;  // pages a sequence's new tokens can touch
};

// x / scale as a code's value before rounding, for one scale and many x: with r the
// correctly rounded reciprocal, two residual corrections of x r give the correctly
// rounded quotient (Markstein) in five operations where a division each takes twice as
// many.  Nothing in between leaves fp32's normal numbers: fp16 x, and scales of their
// maxima.  Scale 0 (a page of zeros) gives 0.  SIGNED: a zero keeps its sign, as a
// quotient does (the corrections lose it; whole numbers have none).
template <bool SIGNED>
struct Divisor {
  float scale, r;
  uint32_t sign;
  __device__ __forceinline__ explicit Divisor(float s)
      : scale(s), r(s > 0.0f ? 1.0f / s : 0.0f), sign(s > 0.0f ? 0x80000000u : 0u) {}
  __device__ __forceinline__ float operator()(float x) const {
    float q = x * r;
    q = fmaf(fmaf(-q, scale, x), r, q);
    q = fmaf(fmaf(-q, scale, x), r, q);
    if constexpr (!SIGNED) return q;
    return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, q) | (__builtin_bit_cast(uint32_t, x) & sign));
  }
  // of a code that may be anything: clamped (a NaN stays one)
  __device__ __forceinline__ float clamped(float x, float top) const {
    const float y = (*this)(x);
    return y > top ? top : (y < -top ? -top : y);
  }
};
// Four quotients as codes.  Of values within the page's maximum none exceeds the
// largest code by more than a rounding, which the rounding to a code takes back.
template <bool FP8>
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  if constexpr (FP8) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
  } else {
    // adding 1.5 2^23 rounds to nearest even and leaves the whole number in the low bits
    auto bits = [](float x) { return __builtin_bit_cast(uint32_t, x + 12582912.0f); };
    const uint32_t lo = __builtin_amdgcn_perm(bits(b), bits(a), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(bits(d), bits(c), 0x04000c0cu);
    return lo | hi;
  }
}
// The values of 4 codes.
template <bool FP8>
__device__ __forceinline__ void unpack4(uint32_t w, float (&x)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (FP8) {
      typedef float float2v __attribute__((ext_vector_type(2)));
      const float2v f = j < 2 ? __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false)
                              : __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
      x[j] = f[j & 1];
    } else {
      x[j] = static_cast<float>(static_cast<int8_t>(w >> (8 * j)));
    }
  }
}

// VEC: D % 16 == 0, aligned rows: 16-value chunks, HOLD of them a lane kept in
// registers; else single values.
template <bool FP8, bool VEC, int HOLD = 1>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendParams p) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  long long w = static_cast<long long>(blockIdx.x) * kWaves + wave;
  const bool is_v = w & 1;
  w >>= 1;
  const int hkv = static_cast<int>(w % p.H_KV);
  w /= p.H_KV;
  const int j = static_cast<int>(w % p.pages_per_seq);
  const long long b = w / p.pages_per_seq;
  if (b >= p.B) return;
  const int from = max(0, min(p.cu[b], p.total)), to = max(0, min(p.cu[b + 1], p.total));
  const long long old = p.cache_lens[b];
  const long long n = min(to - from, p.max_new);
  if (n <= 0 || old < 0) return;
  const int page = 1 << p.page_shift;
  const long long pi = (old >> p.page_shift) + j;  // page of the sequence
  const long long start = max(old, pi << p.page_shift), end = min(old + n, (pi + 1) << p.page_shift);
  if (start >= end || pi >= p.max_blocks) return;
  const int id = p.block_table[b * p.max_blocks + pi];

  constexpr float kTop = FP8 ? 448.0f : 127.0f, kInvTop = 1.0f / kTop;
  const int D = p.D;
  const int first = static_cast<int>(start & (page - 1));  // rows [first, first + rows) of the page are new
  const int rows = static_cast<int>(end - start);
  const size_t stride = static_cast<size_t>(p.H_KV) * D;
  const half_t* src = (is_v ? p.v : p.k) + (from + static_cast<size_t>(start - old)) * stride + static_cast<size_t>(hkv) * D;
  if constexpr (VEC) {
    const int cpr = D / 16;
    const int chunks = rows * cpr;
    u32x4 held[HOLD][2];
    auto load = [&](int c, u32x4 (&x)[2]) {
      const half_t* at = src + static_cast<size_t>(c / cpr) * stride + c % cpr * 16;
      x[0] = *reinterpret_cast<const u32x4*>(at);
      x[1] = *reinterpret_cast<const u32x4*>(at + 8);
    };
    half2_t top2 = {static_cast<half_t>(0.0f), static_cast<half_t>(0.0f)};
    auto raise = [&](const u32x4 (&x)[2]) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) top2 = __builtin_elementwise_max(top2, as_h2(x[i][q] & 0x7fff7fffu));
    };
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      held[i][0] = held[i][1] = u32x4{0u, 0u, 0u, 0u};
      if (lane + 64 * i < chunks) load(lane + 64 * i, held[i]);
    }
    // the new rows are on their way while the page's id arrives; then its scale and
    // old codes, which are needed only where the scale grows, together
    if (id < 0 || id >= p.num_pages) return;
    uint8_t* dst = (is_v ? p.v_cache : p.k_cache) + ((static_cast<size_t>(id) * p.H_KV + hkv) << p.page_shift) * D;
    float* scale_at = (is_v ? p.v_scale : p.k_scale) + static_cast<size_t>(id) * p.H_KV + hkv;
    const float before = first > 0 ? *scale_at : 0.0f;
    const int old_chunks = first * cpr;
    u32x4 old_codes[HOLD];
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      old_codes[i] = u32x4{0u, 0u, 0u, 0u};
      if (lane + 64 * i < old_chunks) old_codes[i] = *reinterpret_cast<const u32x4*>(dst + static_cast<size_t>(lane + 64 * i) * 16);
    }
#pragma unroll
    for (int i = 0; i < HOLD; ++i) raise(held[i]);
    for (int c = lane + 64 * HOLD; c < chunks; c += 64) {
      u32x4 x[2];
      load(c, x);
      raise(x);
    }
    const float amax = wave_max(fmaxf(static_cast<float>(top2[0]), static_cast<float>(top2[1])));
    const float scale = fmaxf(amax * kInvTop, before);
    const Divisor<FP8> by(scale);
    auto store = [&](int c, const u32x4 (&x)[2]) {
      u32x4 codes;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const half2_t h = as_h2(x[q >> 1][2 * (q & 1) + (e >> 1)]);
          y[e] = by(static_cast<float>(h[e & 1]));
        }
        codes[q] = pack4<FP8>(y[0], y[1], y[2], y[3]);
      }
      *reinterpret_cast<u32x4*>(dst + static_cast<size_t>(first + c / cpr) * D + c % cpr * 16) = codes;
    };
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
      if (lane + 64 * i < chunks) store(lane + 64 * i, held[i]);
    for (int c = lane + 64 * HOLD; c < chunks; c += 64) {
      u32x4 x[2];
      load(c, x);
      store(c, x);
    }
    if (first > 0 && scale > before) {
      auto again = [&](int c, u32x4 codes) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float y[4];
          unpack4<FP8>(codes[q], y);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = by.clamped(y[e] * before, kTop);
          codes[q] = pack4<FP8>(y[0], y[1], y[2], y[3]);
        }
        *reinterpret_cast<u32x4*>(dst + static_cast<size_t>(c) * 16) = codes;
      };
#pragma unroll
      for (int i = 0; i < HOLD; ++i)
        if (lane + 64 * i < old_chunks) again(lane + 64 * i, old_codes[i]);
      for (int c = lane + 64 * HOLD; c < old_chunks; c += 64) again(c, *reinterpret_cast<const u32x4*>(dst + static_cast<size_t>(c) * 16));
    }
    if (lane == 0) *scale_at = scale;
  } else {
    if (id < 0 || id >= p.num_pages) return;
    uint8_t* dst = (is_v ? p.v_cache : p.k_cache) + ((static_cast<size_t>(id) * p.H_KV + hkv) << p.page_shift) * D;
    float* scale_at = (is_v ? p.v_scale : p.k_scale) + static_cast<size_t>(id) * p.H_KV + hkv;
    const float before = first > 0 ? *scale_at : 0.0f;
    const int values = rows * D;
    float amax = 0.0f;
    for (int e = lane; e < values; e += 64) amax = fmaxf(amax, fabsf(static_cast<float>(src[static_cast<size_t>(e / D) * stride + e % D])));
    amax = wave_max(amax);
    const float scale = fmaxf(amax * kInvTop, before);
    const Divisor<FP8> by(scale);
    for (int e = lane; e < values; e += 64) {
      const float y = by(static_cast<float>(src[static_cast<size_t>(e / D) * stride + e % D]));
      dst[static_cast<size_t>(first) * D + e] = static_cast<uint8_t>(pack4<FP8>(y, 0.0f, 0.0f, 0.0f));
    }
    if (first > 0 && scale > before) {
      for (int e = lane; e < first * D; e += 64) {
        float y[4];
        unpack4<FP8>(dst[e], y);
        dst[e] = static_cast<uint8_t>(pack4<FP8>(by.clamped(y[0] * before, kTop), 0.0f, 0.0f, 0.0f));
      }
    }
    if (lane == 0) *scale_at = scale;
  }
}

// ---------------------------------------------------------------------------

struct EvictParams {
  const half_t* k;  // [B, H_KV, N, D]
  const half_t* v;
  const float* weight;      // [B, H_KV, N]
  const int32_t* seq_lens;  // [B]
  half_t* k_out;            // [B, H_KV, capacity, D]
  half_t* v_out;
  float* weight_out;   // [B, H_KV, capacity]
  int32_t* index;      // [B, H_KV, capacity] source token, -1 past the kept
  int32_t* new_lens;   // [B]
  int B, H_KV, N, D, budget, recent, capacity;
};

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048;

// Order-preserving key; +-0 share one, NaN lies below everything.
__device__ __forceinline__ uint32_t weight_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __builtin_bit_cast(uint32_t, x == 0.0f ? 0.0f : x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ __launch_bounds__(kSelThreads) void select_kernel(EvictParams p) {
  __shared__ int hist[kBins];
  __shared__ int s_wave[1][kSelWaves];
  __shared__ int s_pick[2];
  const int bh = blockIdx.x;
  const int b = bh / p.H_KV;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = max(0, min(p.seq_lens[b], p.N));
  const int kept = min(n, p.budget);
  const float* weight = p.weight + static_cast<size_t>(bh) * p.N;
  int32_t* index = p.index + static_cast<size_t>(bh) * p.capacity;
  float* wout = p.weight_out + static_cast<size_t>(bh) * p.capacity;
  if (bh % p.H_KV == 0 && tid == 0) p.new_lens[b] = kept;
  for (int r = kept + tid; r < p.capacity; r += kSelThreads) {
    index[r] = -1;
    wout[r] = 0.0f;
  }
  auto emit = [&](int r, int t, float x) {
    index[r] = t;
    wout[r] = x;
  };
  if (n <= p.budget) {
    for (int t = tid; t < n; t += kSelThreads) emit(t, t, weight[t]);
    return;
  }
  const int head = n - p.recent;         // the tokens that compete
  const int need = p.budget - p.recent;  // how many of them stay
  for (int t = head + tid; t < n; t += kSelThreads) emit(need + t - head, t, weight[t]);
  if (need == 0) return;

  // ---- the need-th largest key: digit by digit from the top ----
  // Up to 8192 competing tokens' keys stay in registers, eight a thread; of longer
  // caches they are read again for each digit.
  constexpr int HELD = 8;
  const bool held = head <= HELD * kSelThreads;
  uint32_t keys[HELD];
  if (held) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const int t = tid + i * kSelThreads;
      keys[i] = t < head ? weight_key(weight[t]) : 0u;
    }
  }
  uint32_t prefix = 0u, mask = 0u;
  int want = need;  // rank still sought among the keys that share the prefix
  constexpr int kShift[3] = {21, 10, 0}, kBits[3] = {11, 11, 10};
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const uint32_t digits = (1u << kBits[pass]) - 1u;
    hist[tid] = hist[tid + kSelThreads] = 0;
    __syncthreads();
    auto count = [&](int t, uint32_t key) {
      if (t < head && (key & mask) == prefix) atomicAdd(&hist[(key >> kShift[pass]) & digits], 1);
    };
    if (held) {
#pragma unroll
      for (int i = 0; i < HELD; ++i) count(tid + i * kSelThreads, keys[i]);
    } else {
      for (int t = tid; t < head; t += kSelThreads) count(t, weight_key(weight[t]));
    }
    __syncthreads();
    // thread t owns the bins 2t', 2t'+1 from the top
    const int hi = kBins - 1 - 2 * tid;
    const int c0 = hist[hi], c1 = hist[hi - 1];
    const int incl = wave_scan_add(c0 + c1);
    if (lane == 63) s_wave[0][wave] = incl;
    __syncthreads();
    int above = incl - c0 - c1;
#pragma unroll
    for (int q = 0; q < kSelWaves; ++q) above += q < wave ? s_wave[0][q] : 0;
    if (above < want && above + c0 + c1 >= want) {  // exactly one thread
      const bool first = above + c0 >= want;
      s_pick[0] = first ? hi : hi - 1;
      s_pick[1] = first ? above : above + c0;
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(s_pick[0]) << kShift[pass];
    mask |= digits << kShift[pass];
    want -= s_pick[1];
  }

  // ---- keys above the threshold stay, and the first `want` that equal it ----
  int gt_before = 0, eq_before = 0;
  int parity = 0;  // counts of alternate rounds lie apart: one barrier a round
  __shared__ int s_count[2][2][kSelWaves];
  float next = tid < head ? weight[tid] : 0.0f;
  for (int base = 0; base < head; base += kSelThreads, parity ^= 1) {
    const int t = base + tid;
    const float x = next;
    if (t + kSelThreads < head) next = weight[t + kSelThreads];
    const uint32_t key = weight_key(x);
    const bool gt = t < head && key > prefix, eq = t < head && key == prefix;
    const uint64_t gts = __builtin_amdgcn_ballot_w64(gt), eqs = __builtin_amdgcn_ballot_w64(eq);
    if (lane == 0) {
      s_count[parity][0][wave] = __builtin_popcountll(gts);
      s_count[parity][1][wave] = __builtin_popcountll(eqs);
    }
    __syncthreads();
    int g0 = gt_before, e0 = eq_before;
#pragma unroll
    for (int q = 0; q < kSelWaves; ++q) {
      const int g = s_count[parity][0][q], e = s_count[parity][1][q];
      g0 += q < wave ? g : 0;
      e0 += q < wave ? e : 0;
      gt_before += g;
      eq_before += e;
    }
    const uint64_t below = (1ull << lane) - 1;
    g0 += __builtin_popcountll(gts & below);
    e0 += __builtin_popcountll(eqs & below);
    if (gt || (eq && e0 < want)) emit(g0 + min(e0, want), t, x);
  }
}

constexpr int kCopyRows = 32;  // output rows per workgroup

template <bool VEC>
__global__ __launch_bounds__(kThreads) void gather_rows_kernel(EvictParams p) {
  const size_t bh = blockIdx.y;
  const int r0 = static_cast<int>(blockIdx.x) * kCopyRows;
  const int rows = min(kCopyRows, p.capacity - r0);
  const int32_t* index = p.index + bh * p.capacity + r0;
  const half_t* k = p.k + bh * p.N * p.D;
  const half_t* v = p.v + bh * p.N * p.D;
  half_t* ko = p.k_out + (bh * p.capacity + r0) * p.D;
  half_t* vo = p.v_out + (bh * p.capacity + r0) * p.D;
  if constexpr (VEC) {
    const int cpr = p.D / 8, total = rows * cpr;
    constexpr int U = 2;  // chunks of each tensor in flight per thread
    for (int c0 = threadIdx.x; c0 < total; c0 += U * kThreads) {
      u32x4 kx[U], vx[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        kx[u] = vx[u] = u32x4{0u, 0u, 0u, 0u};
        const int c = c0 + u * kThreads;
        const int t = c < total ? index[c / cpr] : -1;
        if (t >= 0) {
          const size_t at = static_cast<size_t>(t) * p.D + c % cpr * 8;
          kx[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(k + at));
          vx[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(v + at));
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * kThreads;
        if (c < total) {
          *reinterpret_cast<u32x4*>(ko + static_cast<size_t>(c) * 8) = kx[u];
          *reinterpret_cast<u32x4*>(vo + static_cast<size_t>(c) * 8) = vx[u];
        }
      }
    }
  } else {
    const int total = rows * p.D;
    for (int e = threadIdx.x; e < total; e += kThreads) {
      const int t = index[e / p.D];
      const size_t at = static_cast<size_t>(max(t, 0)) * p.D + e % p.D;
      ko[e] = t >= 0 ? k[at] : static_cast<half_t>(0.0f);
      vo[e] = t >= 0 ? v[at] : static_cast<half_t>(0.0f);
    }
  }
}

}  // namespace kvops
}  // namespace fa

using namespace fa;

extern "C" int fa_paged_append_kv8(const void* k, const void* v, const int32_t* cu_seqlens, const int32_t* cache_lens,
                                   void* k_cache, void* v_cache, float* k_scale, float* v_scale, const int32_t* block_table,
                                   int fp8, int B, int total, int max_new, int H_KV, int D, int num_pages, int page,
                                   int max_blocks, void* stream) {
  const char* fn = "fa_paged_append_kv8";
  if (B < 0 || total < 0 || max_new < 0 || H_KV <= 0 || D <= 0 || num_pages < 0 || max_blocks < 0)
    return set_error(FA_ERR_INVALID_ARG, "%s: bad sizes (B=%d total=%d max_new=%d H_KV=%d D=%d pages=%d table=%d)", fn, B, total,
                     max_new, H_KV, D, num_pages, max_blocks);
  if (D > 256) return set_error(FA_ERR_UNSUPPORTED, "%s: D=%d exceeds 256", fn, D);
  if (page < 16 || page > 256 || (page & (page - 1)) != 0)
    return set_error(FA_ERR_UNSUPPORTED, "%s: page of %d tokens is not 16, 32, 64, 128 or 256", fn, page);
  if (B == 0 || total == 0 || max_new == 0 || num_pages == 0 || max_blocks == 0) return FA_OK;
  if (!k || !v || !cu_seqlens || !cache_lens || !k_cache || !v_cache || !k_scale || !v_scale || !block_table)
    return set_error(FA_ERR_INVALID_ARG, "%s: null pointer", fn);
  kvops::AppendParams p = {};
  p.k = static_cast<const half_t*>(k);
  p.v = static_cast<const half_t*>(v);
  p.cu = cu_seqlens;
  p.cache_lens = cache_lens;
  p.k_cache = static_cast<uint8_t*>(k_cache);
  p.v_cache = static_cast<uint8_t*>(v_cache);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_table = block_table;
  p.B = B; p.H_KV = H_KV; p.D = D; p.total = total; p.num_pages = num_pages; p.max_blocks = max_blocks;
  p.max_new = max_new < total ? max_new : total;
  p.page_shift = __builtin_ctz(static_cast<unsigned>(page));
  // n tokens from any offset of a page touch at most this many
  p.pages_per_seq = static_cast<int>((static_cast<long long>(p.max_new) + 2 * page - 2) / page);
  const long long waves = 2LL * B * p.pages_per_seq * H_KV;
  const long long blocks = (waves + kvops::kWaves - 1) / kvops::kWaves;
  if (blocks > 0x7fffffffLL) return set_error(FA_ERR_UNSUPPORTED, "%s: problem too large for one launch", fn);
  const bool vec = D % 16 == 0 && aligned16(k) && aligned16(v) && aligned16(k_cache) && aligned16(v_cache);
  const dim3 grid(static_cast<unsigned>(blocks)), block(kvops::kThreads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  // a page's chunks in registers: two a lane (16 tokens at D = 128) or four, past that
  // the rest is read again
  const bool two = page * D <= 2 * 64 * 16;
  auto launch = [&](auto f8) {
    constexpr bool F = decltype(f8)::value;
    if (!vec) hipLaunchKernelGGL((kvops::append_kernel<F, false>), grid, block, 0, st, p);
    else if (two) hipLaunchKernelGGL((kvops::append_kernel<F, true, 2>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((kvops::append_kernel<F, true, 4>), grid, block, 0, st, p);
  };
  if (fp8) launch(std::true_type());
  else launch(std::false_type());
  return check_launch(fn);
}

extern "C" int fa_evict_by_weight(const void* k, const void* v, const float* weight, const int32_t* seq_lens, void* k_out,
                                  void* v_out, float* weight_out, int32_t* index, int32_t* new_lens, int B, int H_KV, int N,
                                  int D, int budget, int recent, int capacity, void* stream) {
  const char* fn = "fa_evict_by_weight";
  if (B < 0 || H_KV <= 0 || N < 0 || D <= 0 || budget < 0 || recent < 0 || capacity < 0)
    return set_error(FA_ERR_INVALID_ARG, "%s: bad sizes (B=%d H_KV=%d N=%d D=%d budget=%d recent=%d capacity=%d)", fn, B, H_KV, N,
                     D, budget, recent, capacity);
  if (recent > budget) return set_error(FA_ERR_INVALID_ARG, "%s: recent (%d) exceeds budget (%d)", fn, recent, budget);
  if (budget > capacity) return set_error(FA_ERR_INVALID_ARG, "%s: budget (%d) exceeds capacity (%d)", fn, budget, capacity);
  if (static_cast<long long>(B) * H_KV > 65535)
    return set_error(FA_ERR_UNSUPPORTED, "%s: more than 65535 (sequence, KV head) pairs", fn);
  if (N > 0x3fffffff || capacity > 0x3fffffff) return set_error(FA_ERR_UNSUPPORTED, "%s: cache too long", fn);
  if (B == 0) return FA_OK;
  if (!seq_lens || !new_lens || (N > 0 && (!k || !v || !weight)) || (capacity > 0 && (!k_out || !v_out || !weight_out || !index)))
    return set_error(FA_ERR_INVALID_ARG, "%s: null pointer", fn);
  kvops::EvictParams p = {};
  p.k = static_cast<const half_t*>(k);
  p.v = static_cast<const half_t*>(v);
  p.weight = weight;
  p.seq_lens = seq_lens;
  p.k_out = static_cast<half_t*>(k_out);
  p.v_out = static_cast<half_t*>(v_out);
  p.weight_out = weight_out;
  p.index = index;
  p.new_lens = new_lens;
  p.B = B; p.H_KV = H_KV; p.N = N; p.D = D; p.budget = budget; p.recent = recent; p.capacity = capacity;
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(kvops::select_kernel, dim3(B * H_KV), dim3(kvops::kSelThreads), 0, st, p);
  if (const int rc = check_launch(fn)) return rc;
  if (capacity == 0) return FA_OK;
  const dim3 grid(ceil_div(capacity, kvops::kCopyRows), B * H_KV);
  const bool vec = D % 8 == 0 && aligned16(k) && aligned16(v) && aligned16(k_out) && aligned16(v_out);
  if (vec) hipLaunchKernelGGL((kvops::gather_rows_kernel<true>), grid, dim3(kvops::kThreads), 0, st, p);
  else hipLaunchKernelGGL((kvops::gather_rows_kernel<false>), grid, dim3(kvops::kThreads), 0, st, p);
  return check_launch(fn);
}
