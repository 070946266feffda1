// Few rows, bf16: symmetric int4 and MXFP4 (w4a16_few.h).
#include "w4a16_few.h"

namespace mi355q {

int launch_w4_few_bf16(const W4Args& g, int kind, const FewPlan& p, float* parts, hipStream_t st) {
  if (kind == kMxfp4) return launch_kind<Bf16, kMxfp4, 4, E8m0>(g, p, parts, st);
  return launch_groups<Bf16, kInt4>(g, p, parts, st);
}

}  // namespace mi355q
