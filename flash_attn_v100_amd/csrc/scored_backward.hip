// fp16 instantiations of the scored-attention backward kernels.
#include "scored_launch.h"

namespace fa {
namespace scored {

void backward_fp16(const ScoredParams& p, bool vec, hipStream_t st) {
  by_shape_fp16<false>(p.D, vec, p.mods, [&](auto dp, auto dc, auto rows, auto mods) {
    launch_backward_shape<half_t, dp(), dc(), rows(), mods()>(p, st);
  });
}

}  // namespace scored
}  // namespace fa
