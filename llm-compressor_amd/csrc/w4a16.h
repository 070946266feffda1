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
// scale in the conversion, exact from 2^-117 up, so it needs no group sums; fp16's
// range would not hold it.
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

}  // namespace mi355q
