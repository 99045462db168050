// Gated delta rule, the walks forwards on bf16 matrix instructions.
#include "delta_rule_walk.h"

namespace prnn {

int dr_walk_bf16(const DrWalk& a, DrKind kind, int cols, hipStream_t stream) {
  switch (kind) {
    case kDrForward: return dr_launch_bf16<kDrForward>(a, cols, stream);
    case kDrKept: return dr_walk_bf16_kept(a, cols, stream);
    case kDrState: return dr_launch_bf16<kDrState>(a, cols, stream);
    default: return dr_walk_bf16_back(a, kind, cols, stream);
  }
}

}  // namespace prnn
