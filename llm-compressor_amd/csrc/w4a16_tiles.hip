// Which tiles a 4-bit product of many rows takes, and the workspace that it asks for (w4a16_tiles.h).
#include "w4a16_tiles.h"

namespace mi355q {

bool w4_tiles_fit(const W4Args& g, int kind) {
  const int64_t row_bytes = kind == kMxfp4 ? g.cols / 2 : (g.cols + 7) / 8 * 4;
  // 32-bit offsets: of a tile's rows (all of x's where they are gathered), of a weight's rows and scales
  const int64_t span = g.rows ? g.n_x : 128;
  const int64_t limit = (int64_t)1 << 32;
  const int64_t steps = (g.cols + kStep - 1) / kStep * kStep;
  const int64_t pitch = g.ldx > steps ? g.ldx : steps;
  return span < limit / (2 * pitch) && g.out < limit / (g.ldw + 16) && (w_in_place(g) || row_bytes % 16) &&
         g.out < limit / (4 * (int64_t)((g.groups + 15) / 16 * 16));
}

// Small tiles while there are few of them, then larger ones, which convert a weight's codes for more rows; and a sum
// over several workgroups where even the smallest leave CUs idle.  4096 x 4096, tiles as rows x columns: 128 rows 25 us
// (32 x 128 in two parts; 27 whole), 512 rows 35 (32 x 128; 64 x 256 58), 1024 rows 51 (64 x 128; 56 in 32 x 128), 2048
// rows 80 (64 x 256; 84 in 64 x 128, 100 in 128 x 256); 1024 x 14336 x 4096 133 (128 x 256; 139 in 64 x 128).  128 x
// 4096 x 14336 40 us in four parts, 45 in two.  128 experts of 1536 x 2048, 32, 64 and 128 x 256: 64 rows each 127, 140
// and 165 us, 128 rows 209, 200 and 238, 256 rows 372, 341 and 343; 8 experts of 8192 x 4096, 250 rows each 242, 201 and
// 220, 750 rows 575, 513 and 486.  Rows told apart by experts or an index (`listed`) keep their sums whole.
TilePlan tile_plan(int64_t rows, int64_t experts, int64_t out, int64_t cols, bool gated, bool listed) {
  const int64_t steps = (cols + kStep - 1) / kStep, mean = rows / experts;
  if (experts > 1 || listed) {
    const int mt = mean < 128 ? 1 : mean < 512 ? 2 : 4;
    return {mt, gated || mean >= 48 ? 2 : 1, 1};
  }
  auto tiles = [&](int mt, int nt) { return ((rows + 32 * mt - 1) / (32 * mt)) * ((out + 128 * nt - 1) / (128 * nt)); };
  if (tiles(4, 2) >= 448) return {4, 2, 1};
  if (tiles(2, 2) >= 400) return {2, 2, 1};
  TilePlan p = {tiles(2, 1) >= 256 ? 2 : 1, 1, 1};
  const int64_t n = tiles(p.mt, 1);
  while (n * 2 * p.splits <= (steps > 64 ? 800 : 400) && steps >= 16 * (int64_t)p.splits) p.splits *= 2;
  if (gated && p.splits == 1) p.nt = 2;      // gate and up of a column meet in one wave, or where the parts are added
  return p;
}

size_t w4_tiles_workspace(int64_t n_x, int64_t rows, int64_t experts, int64_t rows_w, int64_t cols, uint32_t groups,
                          bool mx, bool x_copy) {
  // operands that the DMA cannot read (rows off 16 bytes or not of whole chunks) are copied
  const int64_t w_bytes = mx ? cols / 2 : (cols + 7) / 8 * 4;
  return (mx ? 0 : sums_bytes(n_x, groups) + sums_bytes(rows_w, groups)) + scales_bytes(rows_w, groups) +
         parts_bytes(tile_plan(rows, experts, rows_w / experts, cols, false, false), rows, rows_w / experts) +
         (x_copy ? x_copy_bytes(n_x, cols) : 0) + (w_bytes % 16 ? (size_t)rows_w * ((w_bytes + 15) / 16 * 16) : 0);
}

int launch_w4_tiles(const W4Args& g, mi355q_dtype x_dtype, int kind, void* workspace, hipStream_t st) {
  return x_dtype == MI355Q_BF16 ? launch_w4_tiles_bf16(g, kind, workspace, st)
                                : launch_w4_tiles_f16(g, kind, workspace, st);
}

}  // namespace mi355q
