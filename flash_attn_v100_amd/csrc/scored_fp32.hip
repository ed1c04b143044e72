// fp32 instantiations of the scored-attention kernels.  A product is eight MFMAs to
// fp16's one, and still a step with a bias and a prefix, [2,16,1000,64], takes 229 us
// with the modifications compiled in for 242 with all read from the call.
#include "scored_launch.h"

namespace fa {
namespace scored {

// Calls run with the variant of the call's modifications (by_mods); rows read by
// elements are left to kAnyMods.
template <int ROWS, typename Run>
static void by_row_mods(int mods, Run&& run) {
  if constexpr (ROWS == kRowElems) run(std::integral_constant<int, kAnyMods>());
  else by_mods(mods, run);
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
  by_shape(p.D, vec, [&](auto dp, auto rows) {
    by_row_mods<rows()>(p.mods, [&](auto m) { launch_query<float, dp(), dp(), rows(), 0, m()>(p, split_query(p, false), st); });
  });
}

void backward_fp32(const ScoredParams& p, bool vec, hipStream_t st) {
  by_shape(p.D, vec, [&](auto dp, auto rows) {
    by_row_mods<rows()>(p.mods, [&](auto m) { launch_backward_shape<float, dp(), dp(), rows(), m()>(p, st); });
  });
}

}  // namespace scored
}  // namespace fa
