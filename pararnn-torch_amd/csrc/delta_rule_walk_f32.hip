// Gated delta rule, the walks in fp32 arithmetic: 16 columns a wave.
#include "delta_rule_walk.h"

namespace prnn {
namespace {

template <int KIND>
int launch_kd(const DrWalk& a, hipStream_t stream) {
  // waves that only load as on bf16 instructions (two chunks in LDS up to widths of 64)
  constexpr int kLoad = KIND != kDrState && KIND != kDrAdjoint ? 4 : 0;
  if (a.Dk <= 32) return dr_launch_walk<InF32, 16, 32, 4, kLoad, KIND>(a, stream);
  if (a.Dk <= 64) return dr_launch_walk<InF32, 16, 64, 4, kLoad, KIND>(a, stream);
  if (a.Dk <= 128) return dr_launch_walk<InF32, 16, 128, 4, 0, KIND>(a, stream);
  return dr_launch_walk<InF32, 16, 256, 2, 0, KIND>(a, stream);
}

}  // namespace

int dr_walk_f32(const DrWalk& a, DrKind kind, hipStream_t stream) {
  switch (kind) {
    case kDrForward: return launch_kd<kDrForward>(a, stream);
    case kDrKept: return launch_kd<kDrKept>(a, stream);
    case kDrState: return launch_kd<kDrState>(a, stream);
    case kDrBackward: return launch_kd<kDrBackward>(a, stream);
    default: return launch_kd<kDrAdjoint>(a, stream);
  }
}

}  // namespace prnn
