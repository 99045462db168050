// Gated delta rule, the walks of training's forward pass on bf16 matrix instructions.
#include "delta_rule_walk.h"

namespace prnn {

int dr_walk_bf16_kept(const DrWalk& a, int cols, hipStream_t stream) {
  return dr_launch_bf16<kDrKept>(a, cols, stream);
}

}  // namespace prnn
