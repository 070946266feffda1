// Tiles of 4-bit products, f16 (w4a16_tiles.h).
#include "w4a16_tiles.h"

namespace mi355q {

int launch_w4_tiles_f16(const W4Args& g, int kind, void* workspace, hipStream_t st) {
  return launch_type<F16>(g, kind, workspace, st);
}

}  // namespace mi355q
