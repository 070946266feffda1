// Products of 16-bit activations with 4-bit weights as checkpoints hold them.
//
//   y[m][n] = b[n] + sum_g s[n][g] sum_{k in g} x[m][k] (q[n][k] - z[n][g])
//
// int4: q is a nibble 0 .. 15, eight to a 32-bit word, z = 8 or the stored zero
// point of the row and group; groups of 32, 64, a multiple of 128 or all columns.
// MXFP4: q is an e2m1 code, z = 0, s = 2^(byte - 127), groups of 32.
//
// Numerics.  A nibble in a byte is the e4m3 number q 2^-9 (subnormals and the first
// binade have one step), so the conversion with scale 2^9 gives q in bf16 or fp16,
// exactly; e2m1 codes convert exactly too.  Products are exact in fp32.  The
// zero point enters as the first addend of a group's sum, -z sum_k x[m][k], which one
// more product per group forms (with a constant operand).  Group sums are scaled and
// added in fp32, and the result is rounded once.  MXFP4 with bf16 activations has its
// scale in the conversion, exact down to byte 0 and up to 252, so it needs no group sums;
// of bytes 253 and 254 the weights of 2^128 and more are infinite there, as in bf16.
// fp16's range would not hold the weights, and its groups have their sums scaled.
#pragma once

#include "fp8.h"

namespace mi355q {

enum W4Kind { kInt4 = 0, kInt4Zero = 1, kMxfp4 = 2 };

struct W4Args {
  const uint16_t* x;       // [.][cols]
  int64_t ldx, n_x;
  const int32_t* rows;     // row of x behind each row of y, or null: the same
  const int64_t* offsets;  // first row of every expert, or null: one expert has all rows
  int experts;
  int64_t n_rows;          // of y
  const uint8_t* w;        // [experts][out][bytes]
  int64_t ldw, stride_w;   // bytes
  const void* s;           // [experts][out][groups]
  int s_type;              // dtype of int4's scales
  int64_t lds, stride_s;   // elements
  const uint32_t* z;       // [experts][ceil(out / 8)][groups]
  int64_t ldz, stride_z;
  const void* bias;
  int bias_type;
  void* y;
  int y_type;
  int64_t ldy;
  int64_t out, cols;       // out: rows of w
  int group;               // columns per scale
  uint32_t groups;         // scales per row
  FastDiv per;             // steps of 128 columns per scale, where a scale has them whole
  int gated;               // y = silu(first half) * second half
};

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr int kStep = 128;      // columns per step

__device__ __forceinline__ float load_any(const void* p, int type, int64_t i) {
  if (type == MI355Q_F32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return type == MI355Q_BF16 ? Bf16::load(v) : F16::load(v);
}

// ---------------------------------------------------------------- operands
// eight nibbles of a word, lowest first, as 0 .. 15
template <class T>
__device__ __forceinline__ u32x4_t nibbles(uint32_t w) {
  const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
  const uint32_t lo = __builtin_amdgcn_perm(odd, even, 0x05010400u), hi = __builtin_amdgcn_perm(odd, even, 0x07030602u);
  if constexpr (T::code == MI355Q_BF16)
    return u32x4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, true))};
  else
    return u32x4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.f, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.f, true))};
}
// eight e2m1 codes of a word, lowest first, times a power of two
template <class T>
__device__ __forceinline__ u32x4_t e2m1s(uint32_t w, float e) {
  if constexpr (T::code == MI355Q_BF16)
    return u32x4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, e, 0)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, e, 1)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, e, 2)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, e, 3))};
  else
    return u32x4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, e, 0)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, e, 1)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, e, 2)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, e, 3))};
}
// v / (1 + e^-v) for every v: v itself far above zero, 0 far below, NaN for NaN and -infinity.
__device__ __forceinline__ float silu(float v) {
  // e^-v = 2^(-v log2 e), with what the product's rounding leaves put back as a factor: below 2^-16 where the
  // exponential is neither 0 nor infinite, and held there where v log2 e passes fp32, so that it cannot become one
  const float k = -1.44269504f, t = v * k, r = fmaf(v, k, -t) + v * -1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(t);
  return v * __builtin_amdgcn_rcpf(1.f + e * fmaf(__builtin_amdgcn_fmed3f(r, -0x1p-10f, 0x1p-10f), 0.693147181f, 1.f));
}

// ---------------------------------------------------------------- tiles of rows
// The rows [first, first + count) of y that a tile of ROWS rows holds, and their
// expert (-1: rows before the first expert's and behind the last one's, which are written as zeros).
struct RowTile {
  int64_t first;
  int count, expert;
};
// Tile `id` in the order of experts, each expert's last one shorter; count = 0: there is no such
// tile.  A wave looks at 64 experts at a time, a lane at one: its tiles, their prefix sums, and the lane
// whose range holds the tile.  (Whatever the offsets hold, a tile lies within y.)
template <int ROWS>
__device__ __forceinline__ RowTile find_row_tile(const W4Args& g, uint32_t id) {
  if (!g.offsets) {
    const int64_t first = (int64_t)id * ROWS, left = g.n_rows - first;
    return {first, (int)(left < ROWS ? left : ROWS), 0};
  }
  const int lane = threadIdx.x & 63, n_rows = (int)g.n_rows;
  // (the rows before the experts count as one, number -1, and so do those behind them)
  auto begin = [&](int e) __attribute__((always_inline)) {
    const int64_t o = e < 0 ? 0 : e <= g.experts ? g.offsets[e] : (int64_t)n_rows;
    return o < 0 ? 0 : o < n_rows ? (int)o : n_rows;
  };
  uint32_t left = id;
  int a = begin(lane - 1), b = begin(lane);
  for (int e0 = -1; e0 <= g.experts; e0 += 64) {
    const int na = begin(e0 + 64 + lane), nb = begin(e0 + 65 + lane);
    const uint32_t tiles = b > a ? (uint32_t)(b - a + ROWS - 1) / ROWS : 0u;
    uint32_t sum = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    const uint64_t past = __ballot(sum > left);
    if (past) {
      const int src = __builtin_ctzll(past);
      const int first = __shfl(a, src), end = __shfl(b, src);
      const int in = (int)(left - __shfl(sum - tiles, src)) * ROWS, rest = end - first - in;
      return {first + in, rest < ROWS ? rest : ROWS, e0 + src < g.experts ? e0 + src : -1};    // (e0 + src: -1 and up)
    }
    left -= __shfl(sum, 63);
    a = na;
    b = nb;
  }
  return {0, 0, 0};
}
// the same in scalar registers
template <int ROWS>
__device__ __forceinline__ RowTile row_tile(const W4Args& g, uint32_t id) {
  const RowTile t = find_row_tile<ROWS>(g, id);
  const int64_t first = (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)t.first) |
                        (int64_t)__builtin_amdgcn_readfirstlane((int)(t.first >> 32)) << 32;
  return {first, __builtin_amdgcn_readfirstlane(t.count), __builtin_amdgcn_readfirstlane(t.expert)};
}

// How many tiles a call with offsets may have, whatever they hold: no more than rows, and at most one short one per
// expert, before them and behind them.
inline int64_t most_row_tiles(const W4Args& g, int64_t tile_rows) {
  const int64_t n = g.n_rows / tile_rows + g.experts + 2;
  return n < g.n_rows ? n : g.n_rows;
}

// How a call of few rows is cut (w4a16_few.h): rows per tile (16 mt, or 4), column tiles and waves per
// workgroup, and workgroups that share a sum.
struct FewPlan {
  int mt, nt, w;
  uint32_t splits;
};
int launch_w4_few_bf16(const W4Args& g, int kind, const FewPlan& p, float* parts, hipStream_t st);
int launch_w4_few_f16(const W4Args& g, int kind, const FewPlan& p, float* parts, hipStream_t st);
int launch_w4_few_zero_bf16(const W4Args& g, const FewPlan& p, float* parts, hipStream_t st);
int launch_w4_few_zero_f16(const W4Args& g, const FewPlan& p, float* parts, hipStream_t st);
// y from the parts of the sums
int join_parts(const W4Args& g, uint32_t splits, const float* parts, hipStream_t st);

// The tile kernels (w4a16_tiles.hip): whether they take a call, whether they read x where
// it is, the workspace that they ask for, and the launch.
bool w4_tiles_fit(const W4Args& g, int kind);
inline bool in_place(const W4Args& g) { return aligned16(g.x) && g.ldx % 8 == 0 && g.cols % 8 == 0; }
size_t w4_tiles_workspace(int64_t n_x, int64_t rows, int64_t experts, int64_t rows_w, int64_t cols, uint32_t groups,
                          bool mx, bool x_copy);
int launch_w4_tiles(const W4Args& g, mi355q_dtype x_dtype, int kind, void* workspace, hipStream_t st);
int launch_w4_tiles_bf16(const W4Args& g, int kind, void* workspace, hipStream_t st);
int launch_w4_tiles_f16(const W4Args& g, int kind, void* workspace, hipStream_t st);

}  // namespace mi355q
