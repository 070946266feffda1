// Few rows, bf16: int4 with zero points (w4a16_few.h).
#include "w4a16_few.h"

namespace mi355q {

int launch_w4_few_zero_bf16(const W4Args& g, const FewPlan& p, float* parts, hipStream_t st) {
  return launch_groups<Bf16, kInt4Zero>(g, p, parts, st);
}

}  // namespace mi355q
