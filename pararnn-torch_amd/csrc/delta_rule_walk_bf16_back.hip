// Gated delta rule, the walks backwards on bf16 matrix instructions.
#include "delta_rule_walk.h"

namespace prnn {

int dr_walk_bf16_back(const DrWalk& a, DrKind kind, int cols, hipStream_t stream) {
  return kind == kDrBackward ? dr_launch_bf16<kDrBackward>(a, cols, stream)
                             : dr_launch_bf16<kDrAdjoint>(a, cols, stream);
}

}  // namespace prnn
