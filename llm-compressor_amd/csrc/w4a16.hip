// Products of 16-bit activations with 4-bit weights (w4a16.h): which kernel a call takes.
#include "w4a16.h"

namespace mi355q {

// y from the parts of the sums, added in the order of the splits.  A thread takes a column of a row.
__global__ __launch_bounds__(256) void w4_join_kernel(W4Args g, uint32_t splits, const float* parts) {
  const int64_t half = g.out / 2, width = g.gated ? half : g.out;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = (int64_t)(i / (uint64_t)width), n = (int64_t)(i % (uint64_t)width);
  if (row >= g.n_rows) return;
  auto total = [&](int64_t c) __attribute__((always_inline)) {
    const float* p = parts + row * g.out + c;
    float v = 0.f;
#pragma unroll 4
    for (uint32_t s = 0; s < splits; ++s) v += p[(size_t)s * g.n_rows * g.out];
    return g.bias ? v + load_any(g.bias, g.bias_type, c) : v;
  };
  float v = total(n);
  if (g.gated) v = silu(v) * total(half + n);
  const int64_t at = row * g.ldy + n;
  if (g.y_type == MI355Q_F32) static_cast<float*>(g.y)[at] = v;
  else static_cast<uint16_t*>(g.y)[at] = g.y_type == MI355Q_BF16 ? Bf16::store(v) : F16::store(v);
}

// y of an x without rows: zeros.
__global__ __launch_bounds__(256) void w4_zero_kernel(W4Args g) {
  const int64_t width = g.gated ? g.out / 2 : g.out, n = g.n_rows * width;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t at = i / width * g.ldy + i % width;
    if (g.y_type == MI355Q_F32) static_cast<float*>(g.y)[at] = 0.f;
    else static_cast<uint16_t*>(g.y)[at] = 0;
  }
}

int join_parts(const W4Args& g, uint32_t splits, const float* parts, hipStream_t st) {
  const int64_t width = g.gated ? g.out / 2 : g.out;
  hipLaunchKernelGGL(w4_join_kernel, dim3((unsigned)((g.n_rows * width + 255) / 256)), dim3(256), 0, st, g, splits,
                     parts);
  MQ_LAUNCH_CHECK();
  return MI355Q_OK;
}

// Up to this many rows the weight's bytes decide, and the kernel for few rows is the faster one.  One weight (twelve of
// them in turn): 48 rows of 4096 x 4096 13.6 us, in tiles 14.9 (14336 x 4096 27 and 30, 4096 x 14336 28 and 28); 64 rows
// 14.7 and 15.3 (30 and 29, 31 and 30); 96 rows 21 and 18 (51 and 32, 48 and 38).  The tiles have the scales
// laid out first, which costs some 10 us and what the scales weigh: 128 experts of 1536 x 2048 in groups of 128, 2 rows
// each 34 and 44 us, 3 rows 43 and 43, 4 rows 51 and 45; 8 experts of 8192 x 4096 6 rows each 40 and 48, 8 rows 50 and
// 48.  The 128 experts in groups of 64: 8 rows 68 and 72, 10 rows 77 and 73; of 32: 12 rows 114 and 135, 16 rows 134 and
// 149, 24 rows 241 and 155; MXFP4 8 rows 65 and 82, 12 rows 86 and 86, 16 rows 103 and 97.
static bool few_rows(int64_t rows, int64_t experts, int64_t group, bool mx) {
  if (experts == 1) return rows <= 64;
  return rows <= 40 + experts * (group >= 128 ? 3 : group >= 64 ? 9 : mx ? 12 : 16);
}

// Rows per tile (4 or 16 mt), columns, waves and splits of a call of few rows.
//
// A wave's loads are x's and the weight's, and it takes many waves to keep the memory busy.  Up
// to 4 rows (of experts: where a quarter of them have a row, as more rows of one would read its weight again: 128
// experts of 1536 x 2048, 32 rows 20 us in both, 64 rows 29 in tiles of 4 and 20 in tiles of 16): one column tile a
// wave, and fewer waves on one tile's sum the more tiles there are (one token with two, four and eight, twelve weights
// in turn: 28672 x 4096, 1792 tiles, 17.8, 17.0 and 16.5 us; 14336 x 4096, 896, 10.0, 11.2 and 10.8; 4096 x 4096, 256,
// 6.1, 5.3 and 4.9; 4096 x 14336 17.7, 11.7 and 10.3; so the choice is within 12 % of the best of the three.  Gated ones
// have two column tiles, 8 experts of 1536 x 2048 7.8 us).  More rows: x is what is loaded most, so a wave takes up to four
// column tiles (16 x 14336 x 4096 14.7 us, with two 16.9, with one 22.5), and where that leaves CUs idle the sum is split
// over workgroups (23 x 4096 x 14336 34 us whole, 21 in four).  Tiles of experts are many: one or two waves each
// (61 tokens to 8 of 128 experts of 1536 x 2048 54 us, with four waves 85).
static FewPlan few_plan(int64_t rows, int64_t experts, int64_t out, int64_t cols, bool gated) {
  const int64_t mean = (rows + experts - 1) / experts, steps = (cols + kStep - 1) / kStep;
  FewPlan p = {(experts > 1 ? 4 * rows <= experts : rows <= 4) ? 0 : mean <= 16 ? 1 : mean <= 32 ? 2 : 4, 1, 8, 1};
  const int64_t row_tiles = experts > 1 ? (rows < experts ? rows : experts) : (rows + 63) / 64;
  if (p.mt == 0) {
    p.nt = gated ? 2 : 1;
    const int64_t tiles = row_tiles * ((out + 16 * p.nt - 1) / (16 * p.nt));
    p.w = tiles >= 1024 ? 2 : tiles >= 384 ? 4 : 8;
  } else if (p.mt == 1) {
    const int64_t tiles = row_tiles * ((out + 15) / 16);
    p.nt = tiles >= 768 ? 4 : tiles >= 512 || gated ? 2 : 1;
    p.w = experts > 1 ? (tiles >= 4096 ? 1 : 4) : p.nt == 1 ? 8 : 4;
    if (p.w == 1) p.nt = 2;
  } else {
    p.nt = 4;
    const int64_t tiles = row_tiles * ((out + 63) / 64);
    while (tiles * p.splits < 192 && steps >= 16 * (int64_t)p.splits && p.splits < 16) p.splits *= 2;
  }
  return p;
}

}  // namespace mi355q

using namespace mi355q;

// The parts of split sums (`gated` does not split them otherwise).
static size_t few_bytes(int64_t rows, int64_t experts, int64_t out, int64_t cols) {
  const uint32_t splits = few_plan(rows, experts, out, cols, false).splits;
  return splits > 1 ? (size_t)splits * rows * out * sizeof(float) : 0;
}

static size_t workspace_size(int64_t n_x, int64_t rows, int64_t experts, int64_t out, int64_t cols,
                             mi355q_w4_format format, int64_t group_size, bool x_copy) {
  if (n_x <= 0 || rows <= 0 || experts <= 0 || out <= 0 || cols <= 0 || group_size <= 0) return 0;
  const bool mx = format == MI355Q_W4_MXFP4;
  if (group_size > cols) group_size = cols;
  if (few_rows(rows, experts, group_size, mx)) return few_bytes(rows, experts, out, cols);
  return w4_tiles_workspace(n_x, rows, experts, experts * out, cols,
                            (uint32_t)((cols + group_size - 1) / group_size), mx, x_copy);
}

extern "C" size_t mi355q_w4a16_matmul_workspace_size(int64_t n_x, int64_t rows, int64_t experts, int64_t out,
                                                     int64_t cols, mi355q_w4_format format, int64_t group_size) {
  return workspace_size(n_x, rows, experts, out, cols, format, group_size, true);
}

extern "C" size_t mi355q_w4a16_matmul_workspace_size_in_place(int64_t n_x, int64_t rows, int64_t experts, int64_t out,
                                                              int64_t cols, mi355q_w4_format format,
                                                              int64_t group_size) {
  return workspace_size(n_x, rows, experts, out, cols, format, group_size, cols % 8 != 0);
}

extern "C" int mi355q_w4a16_matmul(const void* x_dev, mi355q_dtype x_dtype, int64_t n_x, int64_t ldx,
                                   const int32_t* rows_dev, const int64_t* offsets_dev, int64_t experts,
                                   const void* w_dev, mi355q_w4_format format, int64_t ldw, int64_t stride_w,
                                   const void* scales_dev, mi355q_dtype scales_dtype, int64_t ld_scales,
                                   int64_t stride_scales, const uint32_t* zeros_dev, int64_t ld_zeros,
                                   int64_t stride_zeros, int64_t group_size, const void* bias_dev,
                                   mi355q_dtype bias_dtype, int gated, void* y_dev, mi355q_dtype y_dtype, int64_t ldy,
                                   int64_t rows, int64_t out, int64_t cols, void* workspace_dev,
                                   size_t workspace_bytes, void* stream) {
  const bool mx = format == MI355Q_W4_MXFP4;
  MQ_CHECK_ARG(mx || format == MI355Q_W4_INT4, "w4a16_matmul: unknown weight format %d", (int)format);
  MQ_CHECK_ARG(x_dtype == MI355Q_BF16 || x_dtype == MI355Q_F16, "w4a16_matmul: x must be bf16 or fp16");
  MQ_CHECK_ARG(known_dtype(y_dtype) && (!bias_dev || known_dtype(bias_dtype)) && (mx || known_dtype(scales_dtype)),
               "w4a16_matmul: unknown dtype");
  MQ_CHECK_ARG(rows >= 0 && n_x >= 0 && out > 0 && cols > 0 && experts > 0,
               "w4a16_matmul: sizes must be positive, got rows %lld of %lld, out %lld, cols %lld, experts %lld",
               (long long)rows, (long long)n_x, (long long)out, (long long)cols, (long long)experts);
  MQ_CHECK_ARG(cols >= 8, "w4a16_matmul: x must have 8 columns at the least, got %lld", (long long)cols);
  MQ_CHECK_ARG(!gated || out % 2 == 0, "w4a16_matmul: a gated weight has two halves, got %lld rows", (long long)out);
  MQ_CHECK_ARG(offsets_dev || experts == 1, "w4a16_matmul: several experts take offsets");
  MQ_CHECK_ARG(!offsets_dev || (rows < INT32_MAX && experts < INT32_MAX - 128),
               "w4a16_matmul: %lld rows of %lld experts are too many", (long long)rows, (long long)experts);
  MQ_CHECK_ARG(rows_dev || n_x >= rows, "w4a16_matmul: x has fewer rows than y (%lld of %lld)", (long long)n_x,
               (long long)rows);
  MQ_CHECK_ARG(!mx || (cols % 32 == 0 && group_size == 32 && !zeros_dev),
               "w4a16_matmul: MXFP4 has groups of 32 columns, whole ones, and no zero points");
  MQ_CHECK_ARG(group_size == 32 || group_size == 64 || (group_size > 0 && group_size % 128 == 0) || group_size >= cols,
               "w4a16_matmul: groups must have 32, 64, a multiple of 128 or all columns, got %lld",
               (long long)group_size);
  if (group_size > cols) group_size = cols;
  MQ_CHECK_ARG(ldx >= 0, "w4a16_matmul: x has a pitch of %lld", (long long)ldx);
  if (rows == 0) return MI355Q_OK;
  MQ_CHECK_ARG((x_dev || n_x == 0) && w_dev && scales_dev && y_dev, "w4a16_matmul: a null operand");
  const int64_t row_bytes = mx ? cols / 2 : (cols + 7) / 8 * 4;
  MQ_CHECK_ARG(ldw >= row_bytes && ldw % 4 == 0 && stride_w % 4 == 0 && aligned_to(w_dev, 4),
               "w4a16_matmul: the weight's rows must not overlap and lie on 4-byte boundaries");
  MQ_CHECK_ARG(ldy >= (gated ? out / 2 : out), "w4a16_matmul: the output's rows overlap");
  MQ_CHECK_ARG(cols < INT32_MAX, "w4a16_matmul: %lld columns are too many", (long long)cols);
  W4Args g = {static_cast<const uint16_t*>(x_dev), ldx, n_x, rows_dev, offsets_dev, (int)experts, rows,
              static_cast<const uint8_t*>(w_dev), ldw, stride_w, scales_dev, (int)scales_dtype, ld_scales,
              stride_scales, zeros_dev, ld_zeros, stride_zeros, bias_dev, (int)bias_dtype, y_dev, (int)y_dtype, ldy,
              out, cols, (int)group_size, (uint32_t)((cols + group_size - 1) / group_size),
              fast_div((uint32_t)((group_size + kStep - 1) / kStep)), gated != 0};
  const int kind = mx ? kMxfp4 : zeros_dev ? kInt4Zero : kInt4;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (n_x == 0) {                  // (the kernels read row 0 of x in the place of rows that are not there)
    const int64_t blocks = (rows * (gated ? out / 2 : out) + 255) / 256;
    hipLaunchKernelGGL(w4_zero_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, g);
    MQ_LAUNCH_CHECK();
    return MI355Q_OK;
  }
  if (!few_rows(rows, experts, group_size, mx) && w4_tiles_fit(g, kind) && workspace_dev && aligned16(workspace_dev) &&
      workspace_bytes >= w4_tiles_workspace(n_x, rows, experts, experts * out, cols, g.groups, mx, !in_place(g)))
    return launch_w4_tiles(g, x_dtype, kind, workspace_dev, st);
  FewPlan p = few_plan(rows, experts, out, cols, gated);
  // (rows behind the last expert's and rows that x does not have become zeros where the sum is whole)
  if (rows_dev || offsets_dev || !few_rows(rows, experts, group_size, mx) || !workspace_dev || !aligned16(workspace_dev) ||
      workspace_bytes < few_bytes(rows, experts, out, cols))
    p.splits = 1;
  float* const parts = static_cast<float*>(workspace_dev);
  if (kind == kInt4Zero)
    return x_dtype == MI355Q_BF16 ? launch_w4_few_zero_bf16(g, p, parts, st) : launch_w4_few_zero_f16(g, p, parts, st);
  return x_dtype == MI355Q_BF16 ? launch_w4_few_bf16(g, kind, p, parts, st) : launch_w4_few_f16(g, kind, p, parts, st);
}
