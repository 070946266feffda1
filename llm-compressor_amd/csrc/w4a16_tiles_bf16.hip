// Tiles of 4-bit products, bf16 (w4a16_tiles.h).
#include "w4a16_tiles.h"

namespace mi355q {

int launch_w4_tiles_bf16(const W4Args& g, int kind, void* workspace, hipStream_t st) {
  return launch_type<Bf16>(g, kind, workspace, st);
}

}  // namespace mi355q
