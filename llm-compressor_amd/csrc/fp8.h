// Shared pieces of the block-scaled fp8 kernels (fp8_quant.hip, fp8_matmul.hip).
//
// An fp8 matrix is e4m3 codes with one scale per row and kGroup columns
// (activations, gradients' checkpoints) or per kGroup x kGroup block (weights):
// value = code * scale.  Scales are fp32, or for activations e8m0 bytes
// (2^(byte - 127), 255 = NaN).
#pragma once

#include "common.h"

namespace mi355q {

constexpr int kGroup = 128;

inline int64_t group_count(int64_t n) { return (n + kGroup - 1) / kGroup; }

// fp32 value of an e8m0 byte (0 is 2^-127, a subnormal; 255 NaN): the code of 1
// times the scale as the conversions read it, by its exponent bits, in two
// instructions without the special cases
__device__ __forceinline__ float e8m0_to_f32(uint32_t b) {
  return __builtin_amdgcn_cvt_scalef32_f32_fp8(0x38, __uint_as_float((b << 23) | 0x00400000u), 0);
}

__device__ __forceinline__ float load_scale(const void* s, int type, int64_t i) {
  return type == MI355Q_SCALE_E8M0 ? e8m0_to_f32(static_cast<const uint8_t*>(s)[i]) : static_cast<const float*>(s)[i];
}

// 16-bit and fp32 element types of the activations, outputs and biases
struct Bf16 {
  typedef uint16_t raw;
  static constexpr mi355q_dtype code = MI355Q_BF16;
  static __device__ __forceinline__ float load(uint16_t v) { return bf16_bits_to_f32(v); }
  static __device__ __forceinline__ uint16_t store(float f) { return f32_to_bf16_bits(f); }
};
struct F16 {
  typedef uint16_t raw;
  static constexpr mi355q_dtype code = MI355Q_F16;
  static __device__ __forceinline__ float load(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ uint16_t store(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
};
struct F32 {
  typedef float raw;
  static constexpr mi355q_dtype code = MI355Q_F32;
  static __device__ __forceinline__ float load(float v) { return v; }
  static __device__ __forceinline__ float store(float f) { return f; }
};

// calls f(Bf16{} / F16{} / F32{}) for a dtype that the caller has checked
template <class Fn>
inline void with_dtype(mi355q_dtype dt, Fn&& f) {
  if (dt == MI355Q_BF16) f(Bf16{});
  else if (dt == MI355Q_F16) f(F16{});
  else f(F32{});
}

inline bool known_dtype(int dt) { return dt == MI355Q_BF16 || dt == MI355Q_F16 || dt == MI355Q_F32; }
inline int dtype_size(int dt) { return dt == MI355Q_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, unsigned n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// n / d for n < 2^31 without a division: (mulhi(n, mul) + n) >> shift, the division by
// an invariant divisor of Granlund and Montgomery (1994)
struct FastDiv {
  uint32_t d, mul, shift;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t l = 0;
  while ((uint64_t(1) << l) < d) ++l;
  return {d, (uint32_t)((((uint64_t(1) << l) - d) << 32) / d + 1), l};
}
__device__ __forceinline__ uint32_t div(uint32_t n, const FastDiv& f) { return (__umulhi(n, f.mul) + n) >> f.shift; }


// Workgroup id of n, so that the workgroups of one XCD (every eighth) take
// neighbouring items.
__device__ __forceinline__ uint32_t xcd_order(uint32_t id, uint32_t n) {
  const uint32_t q = n / 8, r = n % 8, x = id % 8;
  return x * q + (x < r ? x : r) + id / 8;
}
}  // namespace mi355q
