// Gated delta rule, the walks forwards on bf16 matrix instructions.
#include "delta_rule_walk.h"

namespace prnn {
namespace {

template <int KIND, int KD>
int launch_cols(const DrWalk& a, int cols, hipStream_t stream) {
  // Waves that only load: not for pieces' own states, of which two workgroups a CU run without (D = 128,
  // 512 of them: 74 us, 87 with), nor where two chunks do not fit LDS.
  constexpr int kLoad = KD <= 128 && KIND != kDrState && KIND != kDrAdjoint ? 4 : 0;
  if (cols == 16 && a.group == 4) return dr_launch_walk<InBf16, 16, KD, 4, kLoad, KIND>(a, stream);
  if constexpr (KD <= 128) {
    if (cols == 16) return dr_launch_walk<InBf16, 16, KD, 2, kLoad, KIND>(a, stream);
    if (a.group == 4) return dr_launch_walk<InBf16, 32, KD, 4, 0, KIND>(a, stream);
    if constexpr (KD <= 64) return dr_launch_walk<InBf16, 32, KD, 2, 0, KIND>(a, stream);
  }
  return fail(PRNN_ERR_RUNTIME, "no walk of %d columns a wave for keys of %d", cols, a.Dk);
}
template <int KIND>
int launch_kd(const DrWalk& a, int cols, hipStream_t stream) {
  if (a.Dk <= 32) return launch_cols<KIND, 32>(a, cols, stream);
  if (a.Dk <= 64) return launch_cols<KIND, 64>(a, cols, stream);
  if (a.Dk <= 128) return launch_cols<KIND, 128>(a, cols, stream);
  return launch_cols<KIND, 256>(a, cols, stream);
}

}  // namespace

int dr_walk_bf16(const DrWalk& a, DrKind kind, int cols, hipStream_t stream) {
  switch (kind) {
    case kDrForward: return launch_kd<kDrForward>(a, cols, stream);
    case kDrState: return launch_kd<kDrState>(a, cols, stream);
    default: return dr_walk_bf16_back(a, kind, cols, stream);
  }
}

}  // namespace prnn
