// Gated delta rule, the walks forwards on bf16 matrix instructions (their scheduler's option: _build.py).
#include "delta_rule_walk.h"

namespace prnn {

int dr_walk_bf16_out(const DrWalk& a, bool kept, int cols, hipStream_t stream) {
  return kept ? dr_launch_bf16<kDrKept>(a, cols, stream) : dr_launch_bf16<kDrForward>(a, cols, stream);
}

}  // namespace prnn
