// Products of block-scaled fp8 matrices (fp8.h) and their gradients.
//
//   forward      Y[m][n]  = b[n] + sum_kb xs[m][kb] ws[n / 128][kb] sum_{k in kb} x[m][k] w[n][k]
//   grad input   dX[m][k] = sum_nb ws[nb][k / 128] sum_{n in nb} dY[m][n] w[n][k]
//   grad weight  dW[n][k] = sum_m dY[m][n] x[m][k] 2^e[m][k / 128]
//
// x and w are e4m3 codes, dY is bf16.  Codes, and codes times a power of two,
// are exact in bf16, and products of bf16 values are exact in fp32; so the only
// roundings are those of the fp32 sums, the scales' products and the output.
#include "fp8.h"

namespace mi355q {

enum Product { kForward = 0, kGradInput = 1, kGradWeight = 2 };

// C[p][q] = sum_r A(p, r) B(q, r).  forward: p = m, q = n, r = k; grad input:
// p = m, q = k, r = n; grad weight: p = n, q = k, r = m.
struct ProductArgs {
  const void* a;         // forward: x codes [p][r]; grad input: dY [p][r]; grad weight: dY [r][p]
  int64_t lda;
  const uint8_t* b;      // forward: w codes [q][r]; grad input: w codes [r][q]; grad weight: x codes [r][q]
  int64_t ldb;
  const void* as;        // forward: x scales
  int as_type;
  int64_t ldas;
  const float* bs;       // forward, grad input: w scales; grad weight: unused
  const uint8_t* be;     // grad weight: x scales (e8m0)
  int64_t ldbs;
  const void* bias;      // forward, or null
  int bias_type;
  void* c;
  int64_t ldc;
  int64_t P, Q, R;
  uint32_t q_tiles;
};

__device__ __forceinline__ float load_typed(const void* p, int type, int64_t i) {
  if (type == MI355Q_F32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return type == MI355Q_BF16 ? Bf16::load(v) : F16::load(v);
}

// ---------------------------------------------------------------- any layout
// 64 x 64 tiles over steps of 128, both operands as bf16 in LDS with r
// contiguous, element loads with bounds: right for every size, stride and
// alignment.
constexpr int GT = 64, GPITCH = kGroup + 8;

template <int KIND, class T>
__global__ __launch_bounds__(256) void product_any_kernel(ProductArgs g) {
  __shared__ __attribute__((aligned(16))) uint16_t la[GT * GPITCH];
  __shared__ __attribute__((aligned(16))) uint16_t lb[GT * GPITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t tp = blockIdx.x / g.q_tiles, tq = blockIdx.x - tp * g.q_tiles;
  const int64_t p0 = (int64_t)tp * GT, q0 = (int64_t)tq * GT;
  const int wp = (wave >> 1) * 32, wq = (wave & 1) * 32;
  f32x4_t acc[2][2];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y) acc[x][y] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  // codes and codes times a power of two are exact in bf16
  auto bf16_of = [](uint8_t code, float s) __attribute__((always_inline)) {
    return f32_to_bf16_bits(__builtin_amdgcn_cvt_f32_fp8((int)code, 0) * s);
  };
  for (int64_t r0 = 0; r0 < g.R; r0 += kGroup) {
    __syncthreads();
    // operands with r contiguous: four threads a row; with r as the row: two
    // threads a row of the matrix
    for (int j = 0; j < 32; ++j) {
      const int pi = tid >> 2, ri = (tid & 3) * 32 + j;
      const int64_t p = p0 + pi, r = r0 + ri;
      if constexpr (KIND == kForward)
        la[pi * GPITCH + ri] = p < g.P && r < g.R ? bf16_of(static_cast<const uint8_t*>(g.a)[p * g.lda + r], 1.f) : 0;
      if constexpr (KIND == kGradInput)
        la[pi * GPITCH + ri] = p < g.P && r < g.R ? static_cast<const uint16_t*>(g.a)[p * g.lda + r] : 0;
      if constexpr (KIND == kForward) {
        const int64_t q = q0 + pi;
        lb[pi * GPITCH + ri] = q < g.Q && r < g.R ? bf16_of(g.b[q * g.ldb + r], 1.f) : 0;
      }
      const int rt = tid >> 1, ct = (tid & 1) * 32 + j;
      const int64_t rr = r0 + rt, p2 = p0 + ct, q2 = q0 + ct;
      if constexpr (KIND == kGradWeight)
        la[ct * GPITCH + rt] = p2 < g.P && rr < g.R ? static_cast<const uint16_t*>(g.a)[rr * g.lda + p2] : 0;
      if constexpr (KIND != kForward) {
        float s = 1.f;
        if constexpr (KIND == kGradWeight)
          if (q2 < g.Q && rr < g.R) s = e8m0_to_f32(g.be[rr * g.ldbs + q0 / kGroup]);
        lb[ct * GPITCH + rt] = q2 < g.Q && rr < g.R ? bf16_of(g.b[rr * g.ldb + q2], s) : 0;
      }
    }
    __syncthreads();
    f32x4_t part[2][2];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y) part[x][y] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kGroup / 32; ++s) {
      bf16x8_t fa[2], fb[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int off = (16 * x + (lane & 15)) * GPITCH + 32 * s + 8 * (lane >> 4);
        fa[x] = *reinterpret_cast<const bf16x8_t*>(la + wp * GPITCH + off);
        fb[x] = *reinterpret_cast<const bf16x8_t*>(lb + wq * GPITCH + off);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y)
          part[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[x], fb[y], part[x][y], 0, 0, 0);
    }
    const int64_t rb = r0 / kGroup;
    float sb = 1.f;
    if constexpr (KIND == kForward) sb = g.bs[q0 / kGroup * g.ldbs + rb];
    if constexpr (KIND == kGradInput) sb = g.bs[rb * g.ldbs + q0 / kGroup];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float s = sb;
        if constexpr (KIND == kForward) {
          const int64_t p = p0 + wp + 16 * x + 4 * (lane >> 4) + i;
          s *= load_scale(g.as, g.as_type, (p < g.P ? p : g.P - 1) * g.ldas + rb);
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) acc[x][y][i] = fmaf(part[x][y][i], s, acc[x][y][i]);
      }
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const int64_t q = q0 + wq + 16 * y + (lane & 15);
    const float bias = KIND == kForward && g.bias && q < g.Q ? load_typed(g.bias, g.bias_type, q) : 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t p = p0 + wp + 16 * x + 4 * (lane >> 4) + i;
        if (p < g.P && q < g.Q)
          static_cast<typename T::raw*>(g.c)[p * g.ldc + q] = T::store(acc[x][y][i] + bias);
      }
  }
}

template <int KIND>
static int launch_any(ProductArgs g, mi355q_dtype out, hipStream_t st, const char* who) {
  const int64_t tp = (g.P + GT - 1) / GT, tq = (g.Q + GT - 1) / GT;
  MQ_CHECK_ARG(tp * tq < (int64_t(1) << 31), "%s: output too large", who);
  g.q_tiles = (uint32_t)tq;
  const dim3 grid((unsigned)(tp * tq));
  with_dtype(out, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((product_any_kernel<KIND, T>), grid, dim3(256), 0, st, g);
  });
  MQ_LAUNCH_CHECK();
  return MI355Q_OK;
}

}  // namespace mi355q

using namespace mi355q;

extern "C" size_t mi355q_fp8_block_matmul_workspace_size(int64_t, int64_t, int64_t) { return 0; }

extern "C" int mi355q_fp8_block_matmul(const uint8_t* x_dev, int64_t ldx, const void* x_scales_dev,
                                       mi355q_scale_type x_scale_type, int64_t ld_x_scales, const uint8_t* w_dev,
                                       int64_t ldw, const float* w_scales_dev, int64_t ld_w_scales,
                                       const void* bias_dev, mi355q_dtype bias_dtype, void* y_dev,
                                       mi355q_dtype y_dtype, int64_t ldy, int64_t rows, int64_t out, int64_t cols,
                                       void* workspace_dev, size_t workspace_bytes, void* stream) {
  MQ_CHECK_ARG(rows >= 0 && out > 0 && cols > 0 && ldx >= cols && ldw >= cols && ldy >= out &&
                   ld_x_scales >= group_count(cols) && ld_w_scales >= group_count(cols),
               "fp8_block_matmul: bad shape");
  if (rows == 0) return MI355Q_OK;
  MQ_CHECK_ARG(x_dev && x_scales_dev && w_dev && w_scales_dev && y_dev, "fp8_block_matmul: null pointer");
  MQ_CHECK_ARG(x_scale_type == MI355Q_SCALE_F32 || x_scale_type == MI355Q_SCALE_E8M0,
               "fp8_block_matmul: unknown scale type");
  MQ_CHECK_ARG(known_dtype(y_dtype) && (!bias_dev || known_dtype(bias_dtype)),
               "fp8_block_matmul: output and bias are bf16, fp16 or fp32");
  ProductArgs g{};
  g.a = x_dev;
  g.lda = ldx;
  g.as = x_scales_dev;
  g.as_type = x_scale_type;
  g.ldas = ld_x_scales;
  g.b = w_dev;
  g.ldb = ldw;
  g.bs = w_scales_dev;
  g.ldbs = ld_w_scales;
  g.bias = bias_dev;
  g.bias_type = bias_dtype;
  g.c = y_dev;
  g.ldc = ldy;
  g.P = rows;
  g.Q = out;
  g.R = cols;
  return launch_any<kForward>(g, y_dtype, reinterpret_cast<hipStream_t>(stream), "fp8_block_matmul");
}

extern "C" size_t mi355q_fp8_block_grad_input_workspace_size(int64_t, int64_t, int64_t) { return 0; }

extern "C" int mi355q_fp8_block_grad_input(const uint16_t* dy_dev, int64_t lddy, const uint8_t* w_dev, int64_t ldw,
                                           const float* w_scales_dev, int64_t ld_w_scales, uint16_t* dx_dev,
                                           int64_t lddx, int64_t rows, int64_t out, int64_t cols, void* workspace_dev,
                                           size_t workspace_bytes, void* stream) {
  MQ_CHECK_ARG(rows >= 0 && out > 0 && cols > 0 && lddy >= out && ldw >= cols && lddx >= cols &&
                   ld_w_scales >= group_count(cols),
               "fp8_block_grad_input: bad shape");
  if (rows == 0) return MI355Q_OK;
  MQ_CHECK_ARG(dy_dev && w_dev && w_scales_dev && dx_dev, "fp8_block_grad_input: null pointer");
  ProductArgs g{};
  g.a = dy_dev;
  g.lda = lddy;
  g.b = w_dev;
  g.ldb = ldw;
  g.bs = w_scales_dev;
  g.ldbs = ld_w_scales;
  g.c = dx_dev;
  g.ldc = lddx;
  g.P = rows;
  g.Q = cols;
  g.R = out;
  return launch_any<kGradInput>(g, MI355Q_BF16, reinterpret_cast<hipStream_t>(stream), "fp8_block_grad_input");
}

extern "C" size_t mi355q_fp8_block_grad_weight_workspace_size(int64_t, int64_t, int64_t) { return 0; }

extern "C" int mi355q_fp8_block_grad_weight(const uint16_t* dy_dev, int64_t lddy, const uint8_t* x_dev, int64_t ldx,
                                            const uint8_t* x_scales_dev, int64_t ld_x_scales, void* dw_dev,
                                            mi355q_dtype dw_dtype, int64_t lddw, int64_t rows, int64_t out,
                                            int64_t cols, void* workspace_dev, size_t workspace_bytes, void* stream) {
  MQ_CHECK_ARG(rows >= 0 && out > 0 && cols > 0 && lddy >= out && ldx >= cols && lddw >= cols &&
                   ld_x_scales >= group_count(cols),
               "fp8_block_grad_weight: bad shape");
  MQ_CHECK_ARG(dw_dev && (rows == 0 || (dy_dev && x_dev && x_scales_dev)), "fp8_block_grad_weight: null pointer");
  MQ_CHECK_ARG(known_dtype(dw_dtype), "fp8_block_grad_weight: output is bf16, fp16 or fp32");
  ProductArgs g{};
  g.a = dy_dev;
  g.lda = lddy;
  g.b = x_dev;
  g.ldb = ldx;
  g.be = x_scales_dev;
  g.ldbs = ld_x_scales;
  g.c = dw_dev;
  g.ldc = lddw;
  g.P = out;
  g.Q = cols;
  g.R = rows;
  return launch_any<kGradWeight>(g, dw_dtype, reinterpret_cast<hipStream_t>(stream), "fp8_block_grad_weight");
}
