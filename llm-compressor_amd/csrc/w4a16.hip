// Products of 16-bit activations with 4-bit weights (w4a16.h).
#include "w4a16.h"

namespace mi355q {

template <class T>
__device__ __forceinline__ f32x4_t mfma(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) {
  if constexpr (T::code == MI355Q_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
}
// A lane holds 16 bytes of a weight's row, the 32 columns from 32 (lane / 16) on;
// an instruction wants 32 neighbouring columns over the four lanes of a row.  So the
// words are transposed over registers and quarters of the wave: word i then holds
// columns 32 i + 8 (lane / 16) and on.
__device__ __forceinline__ u32x4_t transpose_words(u32x4_t w) {
  auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
  auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
  auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return u32x4_t{(uint32_t)c[0], (uint32_t)c[1], (uint32_t)d[0], (uint32_t)d[1]};
}

// The eight elements at p of which `left` are inside a row of eight or more, zeros
// for the others: the row's last eight, shifted down.
__device__ __forceinline__ u32x4_t last_chunk(const uint16_t* p, int64_t left) {
  uint64_t v[2] = {0, 0};
  if (left <= 0) return u32x4_t{0u, 0u, 0u, 0u};
  const int n = left < 8 ? 8 - (int)left : 0;
  __builtin_memcpy(v, p - n, 16);
  if (n >= 4) v[0] = v[1], v[1] = 0;
  const int bits = 16 * (n & 3);
  v[0] = (v[0] >> bits) | (v[1] << 1 << (63 - bits));
  v[1] >>= bits;
  return u32x4_t{(uint32_t)v[0], (uint32_t)(v[0] >> 32), (uint32_t)v[1], (uint32_t)(v[1] >> 32)};
}

// ---------------------------------------------------------------- few rows
// 16 MT rows of y times 16 NT columns per workgroup; its W waves take every W-th
// step of 128 columns, straight from memory into the MFMAs' registers (x: rows,
// w: columns; a lane's sums are one column's), and join their sums in LDS.
template <class T, int KIND, int GPS, int MT, int NT, int W, int D>
__global__ __launch_bounds__(64 * W) void w4_few_kernel(W4Args g, uint32_t nt) {
  constexpr bool FOLD = KIND == kMxfp4 && T::code == MI355Q_BF16;     // the scale is in the operand
  __shared__ f32x4_t sums[W][NT][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quarter = lane >> 4;
  const RowTile tile = row_tile<16 * MT>(g, blockIdx.x / nt);
  if (tile.count <= 0) return;
  const int64_t half = g.gated ? g.out / 2 : 0, width = g.gated ? half : g.out;   // of y
  const int64_t n0 = (int64_t)(blockIdx.x % nt) * 16 * (g.gated ? NT / 2 : NT);
  // column of tile a on this lane: the second half of a gated weight's tiles holds its second half
  auto column = [&](int a) __attribute__((always_inline)) {
    return g.gated && a >= NT / 2 ? half + n0 + 16 * (a - NT / 2) : n0 + 16 * a;
  };
  const int steps = tile.expert < 0 ? 0 : (int)((g.cols + kStep - 1) / kStep);
  const uint8_t* wp[NT];
  int64_t sp[NT], zp[NT];
  int zs[NT];
#pragma unroll
  for (int a = 0; a < NT; ++a) {
    const int64_t limit = g.gated && a < NT / 2 ? half : g.out;
    int64_t n = column(a) + col;
    n = n < limit ? n : limit - 1;                                   // the columns past the end are not stored
    const int64_t e = tile.expert < 0 ? 0 : tile.expert;
    wp[a] = g.w + e * g.stride_w + n * g.ldw + 16 * quarter;
    sp[a] = e * g.stride_s + n * g.lds;
    zp[a] = e * g.stride_z + n / 8 * g.ldz;
    zs[a] = 4 * (int)(n % 8);
  }
  const uint16_t* xp[MT];
  bool live[MT];
#pragma unroll
  for (int b = 0; b < MT; ++b) {
    const int r = 16 * b + col;
    int64_t row = tile.first + (r < tile.count ? r : 0);
    if (g.rows) row = g.rows[row];
    live[b] = r < tile.count && row >= 0 && row < g.n_x;             // a row that x does not have counts as zeros
    xp[b] = g.x + (live[b] ? row : 0) * g.ldx + 8 * quarter;
  }
  f32x4_t acc[NT][MT];
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int b = 0; b < MT; ++b) acc[a][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  struct Step {
    u32x4_t w[NT], x[MT][4];
    float s[NT][GPS];
    uint32_t z[NT][GPS];
  };
  const int64_t bytes = (g.cols + 1) / 2, words = KIND == kMxfp4 ? bytes / 4 : (g.cols + 7) / 8;
  auto load = [&](Step& o, int s) __attribute__((always_inline)) {
    const int64_t k0 = (int64_t)s * kStep;
    const bool whole = k0 + kStep <= g.cols;
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      if (whole) {
        __builtin_memcpy(&o.w[a], wp[a] + k0 / 2, 16);
      } else {
        const int64_t left = words - k0 / 8 - 4 * quarter;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          o.w[a][i] = i < left ? *reinterpret_cast<const uint32_t*>(wp[a] + k0 / 2 + 4 * i) : 0u;
      }
#pragma unroll
      for (int i = 0; i < GPS; ++i) {
        const uint32_t gs = GPS == 1 ? div((uint32_t)s, g.per) : (uint32_t)s * GPS + i;
        const uint32_t gi = gs < g.groups ? gs : g.groups - 1;        // (groups behind the last column)
        if constexpr (KIND == kMxfp4) {
          const uint32_t e = static_cast<const uint8_t*>(g.s)[sp[a] + gi];
          o.s[a][i] = FOLD ? __uint_as_float((e << 23) | 0x00400000u) : e8m0_to_f32(e);
        } else {
          o.s[a][i] = load_any(g.s, g.s_type, sp[a] + gi);
        }
        if constexpr (KIND == kInt4Zero) o.z[a][i] = g.z[zp[a] + gi];
      }
    }
#pragma unroll
    for (int b = 0; b < MT; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t k = k0 + 32 * i;
        if (whole) {
          o.x[b][i] = u32x4_t{0u, 0u, 0u, 0u};
          if (live[b]) __builtin_memcpy(&o.x[b][i], xp[b] + k, 16);
        } else {
          o.x[b][i] = last_chunk(xp[b] + k, live[b] ? g.cols - k - 8 * quarter : 0);
        }
      }
  };
  constexpr uint32_t one = T::code == MI355Q_BF16 ? 0x3f803f80u : 0x3c003c00u;
  constexpr uint32_t minus8 = T::code == MI355Q_BF16 ? 0xc100c100u : 0xc800c800u;
  constexpr uint32_t unit = KIND == kInt4 ? minus8 : one;
  const u32x4_t units = {unit, unit, unit, unit};
  auto use = [&](const Step& o) __attribute__((always_inline)) {
    constexpr int PER = 4 / GPS;                                   // instructions per group
    u32x4_t q[NT][4];
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      const u32x4_t w = transpose_words(o.w[a]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (KIND == kMxfp4) q[a][i] = e2m1s<T>(w[i], FOLD ? o.s[a][i * GPS / 4] : 1.f);
        else q[a][i] = nibbles<T>(w[i]);
      }
    }
#pragma unroll
    for (int b = 0; b < MT; ++b)
#pragma unroll
      for (int i = 0; i < GPS; ++i) {
        f32x4_t base = {0.f, 0.f, 0.f, 0.f};
        if constexpr (KIND != kMxfp4) {
#pragma unroll
          for (int j = 0; j < PER; ++j) base = mfma<T>(o.x[b][i * PER + j], units, base);
        }
#pragma unroll
        for (int a = 0; a < NT; ++a) {
          if constexpr (FOLD) {
#pragma unroll
            for (int j = 0; j < PER; ++j) acc[a][b] = mfma<T>(o.x[b][i * PER + j], q[a][i * PER + j], acc[a][b]);
          } else {
            f32x4_t t = base;
            if constexpr (KIND == kInt4Zero) {
              const float z = -(float)((o.z[a][i] >> zs[a]) & 15u);
#pragma unroll
              for (int r = 0; r < 4; ++r) t[r] = base[r] * z;
            }
#pragma unroll
            for (int j = 0; j < PER; ++j) t = mfma<T>(o.x[b][i * PER + j], q[a][i * PER + j], t);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[a][b][r] = fmaf(t[r], o.s[a][i], acc[a][b][r]);
          }
        }
      }
  };
  for (int s0 = wave; s0 < steps; s0 += W * D) {
    Step o[D];
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (s0 + d * W < steps) load(o[d], s0 + d * W);
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (s0 + d * W < steps) use(o[d]);
  }
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int b = 0; b < MT; ++b) sums[wave][a][b][lane] = acc[a][b];
  __syncthreads();
  auto total = [&](int a, int b) __attribute__((always_inline)) {
    f32x4_t v = sums[0][a][b][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += sums[w][a][b][lane];
    const int64_t n = column(a) + col;
    if (g.bias && n < g.out) {
      const float bias = load_any(g.bias, g.bias_type, n);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += bias;
    }
    return v;
  };
  for (int i = wave; i < (g.gated ? NT / 2 : NT) * MT; i += W) {
    const int a = i / MT, b = i % MT;
    f32x4_t v = total(a, b);
    if (g.gated) {
      const f32x4_t up = total(a + NT / 2, b);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = v[r] / (1.f + expf(-v[r])) * up[r];
    }
    const int64_t n = n0 + 16 * a + col;
    if (n >= width) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * b + 4 * quarter + r;
      if (row >= tile.count) continue;
      const int64_t at = (tile.first + row) * g.ldy + n;
      if (g.y_type == MI355Q_F32) static_cast<float*>(g.y)[at] = v[r];
      else static_cast<uint16_t*>(g.y)[at] = g.y_type == MI355Q_BF16 ? Bf16::store(v[r]) : F16::store(v[r]);
    }
  }
}

template <class T, int KIND, int GPS, int MT, int NT, int W, int D>
static int launch_few(const W4Args& g, hipStream_t st) {
  const int64_t width = g.gated ? g.out / 2 : g.out, per = 16 * (g.gated ? NT / 2 : NT);
  const int64_t nt = (width + per - 1) / per;
  // an expert's last tile may be short: no more tiles than rows, and at most one short one per expert
  // (and one behind them)
  int64_t mt = (g.n_rows + 16 * MT - 1) / (16 * MT);
  if (g.offsets) mt = g.n_rows / (16 * MT) + g.experts + 1 < g.n_rows ? g.n_rows / (16 * MT) + g.experts + 1 : g.n_rows;
  MQ_CHECK_ARG(nt * mt <= (int64_t)(UINT32_MAX / (64 * W)), "w4a16: %lld rows by %lld columns are too many",
               (long long)g.n_rows, (long long)width);
  hipLaunchKernelGGL((w4_few_kernel<T, KIND, GPS, MT, NT, W, D>), dim3((unsigned)(nt * mt)), dim3(64 * W), 0, st, g,
                     (uint32_t)nt);
  MQ_LAUNCH_CHECK();
  return MI355Q_OK;
}

// Up to this many rows (per expert, in the mean) the weight's bytes decide.
static bool few_rows(int64_t rows, int64_t experts) { return rows <= 64 * experts; }

template <class T, int KIND, int GPS>
static int launch_kind(const W4Args& g, hipStream_t st) {
  const int64_t rows = g.offsets ? (g.n_rows + g.experts - 1) / g.experts : g.n_rows;     // per expert, in the mean
  if (rows <= 16) return launch_few<T, KIND, GPS, 1, 2, 8, 2>(g, st);
  if (rows <= 32) return launch_few<T, KIND, GPS, 2, 2, 4, 2>(g, st);
  return launch_few<T, KIND, GPS, 4, 2, 4, 1>(g, st);
}

template <class T>
static int launch_type(const W4Args& g, int kind, hipStream_t st) {
  if (kind == kMxfp4) return launch_kind<T, kMxfp4, 4>(g, st);
  if (kind == kInt4) {
    if (g.groups > 1 && g.group == 32) return launch_kind<T, kInt4, 4>(g, st);
    if (g.groups > 1 && g.group == 64) return launch_kind<T, kInt4, 2>(g, st);
    return launch_kind<T, kInt4, 1>(g, st);
  }
  if (g.groups > 1 && g.group == 32) return launch_kind<T, kInt4Zero, 4>(g, st);
  if (g.groups > 1 && g.group == 64) return launch_kind<T, kInt4Zero, 2>(g, st);
  return launch_kind<T, kInt4Zero, 1>(g, st);
}

}  // namespace mi355q

using namespace mi355q;

extern "C" size_t mi355q_w4a16_matmul_workspace_size(int64_t n_x, int64_t rows, int64_t experts, int64_t out,
                                                     int64_t cols, mi355q_w4_format format, int64_t group_size) {
  if (n_x <= 0 || rows <= 0 || experts <= 0 || out <= 0 || cols <= 0 || group_size <= 0 || few_rows(rows, experts))
    return 0;
  return w4_tiles_workspace(n_x, experts * out, cols, (uint32_t)((cols + group_size - 1) / group_size), format == MI355Q_W4_MXFP4);
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
  MQ_CHECK_ARG(rows_dev || n_x >= rows, "w4a16_matmul: x has fewer rows than y (%lld of %lld)", (long long)n_x,
               (long long)rows);
  MQ_CHECK_ARG(!mx || (cols % 32 == 0 && group_size == 32 && !zeros_dev),
               "w4a16_matmul: MXFP4 has groups of 32 columns, whole ones, and no zero points");
  MQ_CHECK_ARG(group_size == 32 || group_size == 64 || (group_size > 0 && group_size % 128 == 0) || group_size >= cols,
               "w4a16_matmul: groups must have 32, 64, a multiple of 128 or all columns, got %lld",
               (long long)group_size);
  if (rows == 0) return MI355Q_OK;
  MQ_CHECK_ARG(x_dev && w_dev && scales_dev && y_dev, "w4a16_matmul: a null operand");
  const int64_t row_bytes = mx ? cols / 2 : (cols + 7) / 8 * 4;
  MQ_CHECK_ARG(ldw >= row_bytes && ldw % 4 == 0 && stride_w % 4 == 0 && aligned_to(w_dev, 4),
               "w4a16_matmul: the weight's rows must not overlap and lie on 4-byte boundaries");
  MQ_CHECK_ARG(ldy >= (gated ? out / 2 : out), "w4a16_matmul: the output's rows overlap");
  MQ_CHECK_ARG(cols < INT32_MAX, "w4a16_matmul: %lld columns are too many", (long long)cols);
  W4Args g = {static_cast<const uint16_t*>(x_dev), ldx, n_x, rows_dev, offsets_dev, (int)experts, rows,
              static_cast<const uint8_t*>(w_dev), ldw, stride_w, scales_dev, (int)scales_dtype, ld_scales,
              stride_scales, zeros_dev, ld_zeros, stride_zeros, bias_dev, (int)bias_dtype, y_dev, (int)y_dtype, ldy,
              out, cols, (int)(group_size < cols ? group_size : cols), (uint32_t)((cols + group_size - 1) / group_size),
              fast_div((uint32_t)(group_size < cols ? (group_size + 127) / 128 : (cols + 127) / 128)), gated != 0};
  const int kind = mx ? kMxfp4 : zeros_dev ? kInt4Zero : kInt4;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!few_rows(rows, experts) && w4_tiles_fit(g, kind) && workspace_dev && aligned16(workspace_dev) &&
      workspace_bytes >= w4_tiles_workspace(n_x, experts * out, cols, g.groups, mx))
    return launch_w4_tiles(g, x_dtype, kind, workspace_dev, st);
  return x_dtype == MI355Q_BF16 ? launch_type<Bf16>(g, kind, st) : launch_type<F16>(g, kind, st);
}
