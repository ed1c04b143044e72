// fp32 instantiations of the scored-attention kernels.  An fp32 product is
// eight MFMAs to fp16's one, so what is applied to the scores is read from the
// call (kAnyMods) and not compiled into variants of its own.
#include "scored_launch.h"

namespace fa {
namespace scored {

template <int DP, int DC, int ROWS>
static void forward_shape(const ScoredParams& p, hipStream_t st) {
  launch_query<float, DP, DC, ROWS, 0, kAnyMods>(p, split_query(p, false), st);
}

template <typename Run>
static void by_shape(int D, bool vec, Run&& run) {
  constexpr std::integral_constant<int, 32> w32;
  constexpr std::integral_constant<int, 64> w64;
  constexpr std::integral_constant<int, 96> w96;
  constexpr std::integral_constant<int, 128> w128;
  constexpr std::integral_constant<int, kRowElems> elems;
  constexpr std::integral_constant<int, kRowFull> full;
  constexpr std::integral_constant<int, kRowChunks> chunks;
  if (!vec || D % 8 != 0) {
    if (D <= 64) run(w64, elems);
    else run(w128, elems);
  } else if (D == 64) run(w64, full);
  else if (D <= 32) run(w32, chunks);
  else if (D < 64) run(w64, chunks);
  else if (D <= 96) run(w96, chunks);
  else if (D == 128) run(w128, full);
  else run(w128, chunks);
}

void forward_fp32(const ScoredParams& p, bool vec, hipStream_t st) {
  by_shape(p.D, vec, [&](auto dp, auto rows) { forward_shape<dp(), dp(), rows()>(p, st); });
}

void backward_fp32(const ScoredParams& p, bool vec, hipStream_t st) {
  by_shape(p.D, vec, [&](auto dp, auto rows) { launch_backward_shape<float, dp(), dp(), rows(), kAnyMods>(p, st); });
}

}  // namespace scored
}  // namespace fa
