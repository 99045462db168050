// Gated delta rule, the walks on bf16 matrix instructions: which, and pieces' own states forwards.
#include "delta_rule_walk.h"

namespace prnn {

int dr_walk_bf16(const DrWalk& a, DrKind kind, int cols, hipStream_t stream) {
  switch (kind) {
    case kDrForward:
    case kDrKept: return dr_walk_bf16_out(a, kind == kDrKept, cols, stream);
    case kDrState: return dr_launch_bf16<kDrState>(a, cols, stream);
    default: return dr_walk_bf16_back(a, kind, cols, stream);
  }
}

}  // namespace prnn
