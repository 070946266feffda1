// Block-scaled fp8: quantizers of activations and weights, and the gated
// activation whose inputs are kept in 8 bits for its backward pass.
//
//   a = max |x| over a group (1 x 128 of an activation, 128 x 128 of a weight)
//   s = a / 448 (fp32, correctly rounded; a = 0: fp32 epsilon), or
//       2^ceil(log2(a / 448)) as an e8m0 byte (a = 0: 1; never below 2^-126)
//   c = e4m3(x / s), round to nearest even, clamped to +-448, e4m3's largest value.
//       Quotients pass it only where an fp32 scale is a few of fp32's smallest steps
//       (a below 9e-42: a / 448 is rounded to whole steps there)
// A group that holds an infinity or a NaN becomes NaN as a whole, scale and
// codes: its largest magnitude is no number to scale by, and a silent zero
// would hide the overflow.
//
// All kernels pass over the data once (a group never leaves the registers
// between its maximum and its codes) and are bound by HBM.  What is read is read
// once, so the 16-byte loads of elements are nontemporal (those of kept codes and of
// unaligned chunks are plain); the stores are where a call moves more than the
// last-level cache holds, and its results could not stay there for their reader
// anyway.  Against plain accesses: gated activation of 8192 x 14336 142 -> 138 us with
// the loads, 131 with the stores too (6.3 TB/s), its backward pass 164 -> 157 -> 149 us
// (146 by itself, 6.4 TB/s); 14336 x 4096 in blocks 37 -> 33 us (31 with the blocks ordered by XCD,
// 5.7 TB/s); 16384 x 4096 in groups 37 -> 36 us (5.6 TB/s).
// Rows of odd widths are moved in whole chunks too, unaligned, and by elements only
// at their ends: 8192 x 4099 in groups 48 -> 21 us, 7392 x 10364 in blocks 135 -> 57.
#include <type_traits>

#include "fp8.h"

namespace mi355q {

constexpr int NT = 256;
constexpr int kChunk = 8;                        // elements per thread and chunk
constexpr int kLanes = kGroup / kChunk;          // 16 lanes per group: one DPP row

typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));

// The largest magnitude is found on the bit patterns with the sign taken off,
// which order as the magnitudes do and put infinities and NaN on top.
template <class T> __device__ __forceinline__ uint32_t magnitude(typename T::raw v);
template <> __device__ __forceinline__ uint32_t magnitude<Bf16>(uint16_t v) { return (uint32_t)(v & 0x7fffu) << 16; }
template <> __device__ __forceinline__ uint32_t magnitude<F16>(uint16_t v) {
  return __float_as_uint(fabsf(F16::load(v)));
}
template <> __device__ __forceinline__ uint32_t magnitude<F32>(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
  return v > o ? v : o;
}
// maximum over the 16 lanes of a DPP row, in every lane (row rotations)
__device__ __forceinline__ uint32_t max_row16(uint32_t v) {
  return max_dpp<0x121>(max_dpp<0x122>(max_dpp<0x124>(max_dpp<0x128>(v))));
}

// A chunk in registers: 8 elements as loaded.
template <class T> struct Chunk { typename T::raw v[kChunk]; };

template <class T, bool VEC>
__device__ __forceinline__ void load_chunk(Chunk<T>& c, const typename T::raw* p, int64_t left) {
  if constexpr (VEC) {
    // 16-byte loads: the row is 16-byte aligned and a multiple of 8 wide, so
    // a chunk is inside it or past its end as a whole
    constexpr int W = kChunk * sizeof(typename T::raw) / 16;
    u32x4_t q[W];
#pragma unroll
    for (int i = 0; i < W; ++i)
      q[i] = left > 0 ? __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p) + i) : u32x4_t{0u, 0u, 0u, 0u};
    __builtin_memcpy(c.v, q, sizeof(c.v));
  } else if (left >= kChunk) {
    __builtin_memcpy(c.v, p, sizeof(c.v));   // unaligned
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) c.v[i] = i < left ? p[i] : typename T::raw(0);
  }
}

template <bool STREAM, class V>
__device__ __forceinline__ void put(V* p, V v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, p);
  else *p = v;
}
template <bool VEC, bool STREAM>
__device__ __forceinline__ void store_codes(uint8_t* p, const uint32_t w[2], int64_t left) {
  if constexpr (VEC) {
    if (left > 0) put<STREAM>(reinterpret_cast<u32x2_t*>(p), u32x2_t{w[0], w[1]});
  } else if (left >= kChunk) {
    __builtin_memcpy(p, w, kChunk);
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (i < left) p[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
  }
}

// The e8m0 byte of a group from its largest magnitude's bits: 448 = 1.75 2^8,
// so the exponent is floor(log2 a) - 8, plus one where a's significand is above
// 1.75.  Subnormal maxima fall under the 2^-126 floor.
__device__ __forceinline__ uint32_t e8m0_of(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  if (top == 0u) return 127u;
  const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(e < 1 ? 1 : e);
}

__device__ __forceinline__ float f32_scale_of(uint32_t top) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const float s = __uint_as_float(top) / 448.f;
  return s == 0.f ? 1.1920929e-07f : s;
}

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Codes of 8 values over an fp32 scale: the correctly rounded quotient x / s
// from the correctly rounded reciprocal r and one residual step (q0 = x r,
// q = q0 + (x - q0 s) r, both steps fused), a third of a division's
// instructions.  Scales outside [2^-100, 2^100] could lose the residual to
// underflow and take the division, and a clamp that only subnormal scales need: past
// 464 the conversion would give NaN (NaN quotients of non-finite groups pass it).
__device__ __forceinline__ void codes_f32(const float x[kChunk], float s, float r, uint32_t w[2]) {
  float q[kChunk];
  if (s >= 0x1p-100f && s <= 0x1p100f) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      const float q0 = x[i] * r;
      q[i] = fmaf(fmaf(-q0, s, x[i]), r, q0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      const float t = x[i] / s;
      q[i] = t > 448.f ? 448.f : t < -448.f ? -448.f : t;
    }
  }
  w[0] = pack4(q[0], q[1], q[2], q[3]);
  w[1] = pack4(q[4], q[5], q[6], q[7]);
}

// ... over a power of two: the product with 2^(127 - byte) is exact (down to
// the fp32 subnormals, far below e4m3's smallest value); bytes are e8m0_of's, 1 .. 247 or 255
__device__ __forceinline__ void codes_e8m0(const float x[kChunk], uint32_t byte, uint32_t w[2]) {
  const float r = __uint_as_float(byte == 255 ? 0x7fc00000u : (254u - byte) << 23);
  w[0] = pack4(x[0] * r, x[1] * r, x[2] * r, x[3] * r);
  w[1] = pack4(x[4] * r, x[5] * r, x[6] * r, x[7] * r);
}

// NaN codes carry no payload: the hardware keeps the input's sign, which the
// format does not mind.

// ---------------------------------------------------------------- groups
struct GroupsArgs {
  const void* x;
  int64_t ldx, cols;
  uint8_t* codes;
  int64_t ldc;
  void* scales;
  int64_t lds;
  uint32_t chunks;    // of this launch: rows * groups * 16
  FastDiv per_row;    // groups * 16
};

// One thread per chunk of 8 columns, 16 lanes per group; consecutive lanes
// take consecutive chunks, so a wave moves 1 KB of 16-bit input per load.
template <class T, bool E8M0, bool VEC, bool STREAM>
__global__ __launch_bounds__(NT) void fp8_groups_kernel(GroupsArgs a) {
  const uint32_t i = blockIdx.x * NT + threadIdx.x;
  const uint32_t j = i < a.chunks ? i : a.chunks - 1;    // whole rows of lanes (chunks is a multiple of 16)
  const uint32_t row = div(j, a.per_row);
  const uint32_t ch = j - row * a.per_row.d;
  const int64_t col = (int64_t)ch * kChunk, left = a.cols - col;
  Chunk<T> c;
  load_chunk<T, VEC>(c, static_cast<const typename T::raw*>(a.x) + row * a.ldx + (left > 0 ? col : 0), left);
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < kChunk; ++e) {
    const uint32_t v = magnitude<T>(c.v[e]);
    m = v > m ? v : m;
  }
  const uint32_t top = max_row16(m);
  float x[kChunk];
#pragma unroll
  for (int e = 0; e < kChunk; ++e) x[e] = T::load(c.v[e]);
  uint32_t w[2];
  const bool first = (ch & (kLanes - 1)) == 0 && i < a.chunks;
  const int64_t si = row * a.lds + ch / kLanes;
  if constexpr (E8M0) {
    const uint32_t b = e8m0_of(top);
    codes_e8m0(x, b, w);
    if (first) static_cast<uint8_t*>(a.scales)[si] = (uint8_t)b;
  } else {
    const float s = f32_scale_of(top);
    codes_f32(x, s, 1.f / s, w);
    if (first) static_cast<float*>(a.scales)[si] = s;
  }
  if (i < a.chunks) store_codes<VEC, STREAM>(a.codes + row * a.ldc + col, w, left);
}

// ---------------------------------------------------------------- blocks
// One workgroup per 128 x 128 block: 16 lanes per row, 16 rows a pass, eight
// passes held in registers between the maximum and the codes.
template <class T, bool VEC, bool STREAM>
__global__ __launch_bounds__(NT) void fp8_blocks_kernel(const void* w, int64_t rows, int64_t cols, int64_t ldw,
                                                        uint8_t* codes, int64_t ldc, float* scales, int64_t lds,
                                                        uint32_t col_blocks) {
  __shared__ uint32_t tops[NT / 64];
  constexpr int P = kGroup / (NT / kLanes);
  // neighbouring blocks on one XCD
  const uint32_t id = xcd_order(blockIdx.x, gridDim.x), br = id / col_blocks, bc = id - br * col_blocks;
  const int64_t r0 = (int64_t)br * kGroup + threadIdx.x / kLanes;
  const int64_t col = (int64_t)bc * kGroup + (threadIdx.x % kLanes) * kChunk;
  Chunk<T> c[P];
  uint32_t m = 0;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int64_t r = r0 + p * (NT / kLanes), left = r < rows ? cols - col : 0;
    load_chunk<T, VEC>(c[p], static_cast<const typename T::raw*>(w) + (left > 0 ? r * ldw + col : 0), left);
  }
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int e = 0; e < kChunk; ++e) {
      const uint32_t v = magnitude<T>(c[p].v[e]);
      m = v > m ? v : m;
    }
  m = max_row16(m);
  m = max(m, (uint32_t)__shfl_xor((int)m, 16));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) m = max(m, tops[i]);
  const float s = f32_scale_of(m), rs = 1.f / s;
  if (threadIdx.x == 0) scales[br * lds + bc] = s;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int64_t r = r0 + p * (NT / kLanes), left = r < rows ? cols - col : 0;
    float x[kChunk];
#pragma unroll
    for (int e = 0; e < kChunk; ++e) x[e] = T::load(c[p].v[e]);
    uint32_t o[2];
    codes_f32(x, s, rs, o);
    store_codes<VEC, STREAM>(codes + (left > 0 ? r * ldc + col : 0), o, left);
  }
}

// ---------------------------------------------------------------- gated activation
// s = 1 / (1 + e^-g) from the hardware's exp2 and reciprocal (each within a unit in the
// last place).  What rounding the argument -log2(e) g costs grows with |g|: 4e-7 of s
// below 8, 3e-6 at 72.  Enough for the forward pass, which ends in the 2^-4 of e4m3 codes
// and is bound by vector instructions where its data are in the caches (2048 x 4099 13
// us, 14 with the correction below).  e^-g = inf gives 0, as it should.
__device__ __forceinline__ float sigmoid_to_8_bits(float g) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * g));
}
// The same with that rounding added back, for gradients that may be written in fp32: with
// e^-g as 2^p, p the rounded argument, a factor e^d is left out, d = -g - p ln 2 (two fused
// steps), so that s' = s (1 - (1 - s) d), in which nothing overflows where 2^p does.  Past
// |g| = 200 s is 0 or 1.  Within 6 2^-24 of s, down to s = 2^-126; smaller ones may become 0.
// The kernel stays bound by HBM (8192 x 14336 132.6 -> 133.5 us).
__device__ __forceinline__ float sigmoid(float g) {
  const float c = __builtin_amdgcn_fmed3f(g, -200.f, 200.f), p = -1.44269504f * c;
  const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(p));
  const float d = fmaf(-p, -1.90465432e-9f, fmaf(-p, 0.693147182f, -c));
  return fmaf(s * (s - 1.f), d, s);
}

struct GluArgs {
  const void* x;       // [rows, 2 cols]: gate, then up
  int64_t ldx, cols;
  uint8_t* h;          // codes of silu(gate) * up
  int64_t ldh;
  uint8_t* hs;         // their e8m0 bytes
  uint8_t* kept;       // codes of gate and up [rows, 2 cols], or null
  int64_t ldk;
  uint8_t* ks;         // [rows, 2 groups]
  uint32_t chunks;
  FastDiv per_row;
};

template <class T, bool KEEP, bool VEC, bool STREAM>
__global__ __launch_bounds__(NT) void fp8_silu_mul_kernel(GluArgs a) {
  const uint32_t i = blockIdx.x * NT + threadIdx.x;
  const uint32_t j = i < a.chunks ? i : a.chunks - 1;
  const uint32_t row = div(j, a.per_row);
  const uint32_t ch = j - row * a.per_row.d;
  const int64_t col = (int64_t)ch * kChunk, left = a.cols - col;
  const typename T::raw* xr = static_cast<const typename T::raw*>(a.x) + row * a.ldx + (left > 0 ? col : 0);
  Chunk<T> cg, cu;
  load_chunk<T, VEC>(cg, xr, left);
  load_chunk<T, VEC>(cu, xr + a.cols, left);
  float g[kChunk], u[kChunk], h[kChunk];
  uint32_t mh = 0, mg = 0, mu = 0;
#pragma unroll
  for (int e = 0; e < kChunk; ++e) {
    g[e] = T::load(cg.v[e]);
    u[e] = T::load(cu.v[e]);
    h[e] = g[e] * sigmoid_to_8_bits(g[e]) * u[e];
    mh = max(mh, __float_as_uint(h[e]) & 0x7fffffffu);
    if constexpr (KEEP) {
      mg = max(mg, magnitude<T>(cg.v[e]));
      mu = max(mu, magnitude<T>(cu.v[e]));
    }
  }
  const uint32_t groups = a.per_row.d / kLanes, gi = ch / kLanes;
  const bool mine = i < a.chunks, first = mine && (ch & (kLanes - 1)) == 0;
  auto quantize = [&](const float* v, uint32_t m, uint8_t* codes, uint8_t* scale) __attribute__((always_inline)) {
    const uint32_t b = e8m0_of(max_row16(m));
    uint32_t w[2];
    codes_e8m0(v, b, w);
    if (first) *scale = (uint8_t)b;
    if (mine) store_codes<VEC, STREAM>(codes, w, left);
  };
  quantize(h, mh, a.h + row * a.ldh + col, a.hs + (int64_t)row * groups + gi);
  if constexpr (KEEP) {
    uint8_t* k = a.kept + row * a.ldk + col;
    uint8_t* s = a.ks + (int64_t)row * 2 * groups + gi;
    quantize(g, mg, k, s);
    quantize(u, mu, k + a.cols, s + groups);
  }
}

struct GluBackArgs {
  const void* dh;
  int64_t lddh, cols;
  const uint8_t* kept;
  int64_t ldk;
  const uint8_t* ks;
  int64_t ldks;
  void* dx;            // [rows, 2 cols]: d gate, then d up
  int64_t lddx;
  uint32_t chunks;
  FastDiv per_row;
};

template <bool VEC>
__device__ __forceinline__ void load_codes(float v[kChunk], const uint8_t* p, float scale, int64_t left) {
  uint32_t w[2] = {0u, 0u};
  if constexpr (VEC) {
    if (left > 0) {
      const u32x2_t q = *reinterpret_cast<const u32x2_t*>(p);
      w[0] = q[0];
      w[1] = q[1];
    }
  } else if (left >= kChunk) {
    __builtin_memcpy(w, p, kChunk);
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (i < left) w[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
    v[4 * i] = lo[0] * scale;
    v[4 * i + 1] = lo[1] * scale;
    v[4 * i + 2] = hi[0] * scale;
    v[4 * i + 3] = hi[1] * scale;
  }
}

template <class T, bool VEC, bool STREAM>
__device__ __forceinline__ void store_chunk(typename T::raw* p, const float v[kChunk], int64_t left) {
  Chunk<T> c;
#pragma unroll
  for (int e = 0; e < kChunk; ++e) c.v[e] = T::store(v[e]);
  if constexpr (VEC) {
    constexpr int W = kChunk * sizeof(typename T::raw) / 16;
    u32x4_t q[W];
    __builtin_memcpy(q, c.v, sizeof(c.v));
    if (left > 0) {
#pragma unroll
      for (int i = 0; i < W; ++i) put<STREAM>(reinterpret_cast<u32x4_t*>(p) + i, q[i]);
    }
  } else if (left >= kChunk) {
    __builtin_memcpy(p, c.v, sizeof(c.v));
  } else {
#pragma unroll
    for (int e = 0; e < kChunk; ++e)
      if (e < left) p[e] = c.v[e];
  }
}

// d gate = dh up s (1 + gate (1 - s)), d up = dh gate s, s = sigmoid(gate)
template <class T, bool VEC, bool STREAM>
__global__ __launch_bounds__(NT) void fp8_silu_mul_backward_kernel(GluBackArgs a) {
  const uint32_t i = blockIdx.x * NT + threadIdx.x;
  if (i >= a.chunks) return;
  const uint32_t row = div(i, a.per_row);
  const uint32_t ch = i - row * a.per_row.d;
  const int64_t col = (int64_t)ch * kChunk, left = a.cols - col;
  if (left <= 0) return;
  Chunk<T> cd;
  load_chunk<T, VEC>(cd, static_cast<const typename T::raw*>(a.dh) + row * a.lddh + col, left);
  const uint8_t* k = a.kept + row * a.ldk + col;
  const uint8_t* s = a.ks + row * a.ldks + ch / kLanes;
  float g[kChunk], u[kChunk], dg[kChunk], du[kChunk];
  load_codes<VEC>(g, k, e8m0_to_f32(s[0]), left);
  load_codes<VEC>(u, k + a.cols, e8m0_to_f32(s[a.per_row.d / kLanes]), left);
#pragma unroll
  for (int e = 0; e < kChunk; ++e) {
    const float d = T::load(cd.v[e]), sg = sigmoid(g[e]);
    dg[e] = d * u[e] * (sg * (1.f + g[e] * (1.f - sg)));
    du[e] = d * (g[e] * sg);
  }
  typename T::raw* o = static_cast<typename T::raw*>(a.dx) + row * a.lddx + col;
  store_chunk<T, VEC, STREAM>(o, dg, left);
  store_chunk<T, VEC, STREAM>(o + a.cols, du, left);
}

// Launches `f(first row, rows)` over row ranges whose chunks fit 31 bits.
template <class Fn>
static void over_rows(int64_t rows, int64_t per_row, Fn&& f) {
  const int64_t most = ((int64_t(1) << 31) - NT) / per_row;
  for (int64_t r = 0; r < rows; r += most) f(r, rows - r < most ? rows - r : most);
}

// Calls f(VEC, STREAM) with the template arguments of a call: whole 16-byte
// chunks, and nontemporal stores where its bytes outgrow the 256 MB last-level
// cache.
template <class Fn>
static void with_access(bool vec, int64_t bytes, Fn&& f) {
  const bool stream = bytes > (int64_t(256) << 20);
  if (vec && stream) f(std::true_type{}, std::true_type{});
  else if (vec) f(std::true_type{}, std::false_type{});
  else f(std::false_type{}, std::false_type{});
}

static unsigned blocks_of(uint32_t chunks) { return (chunks + NT - 1) / NT; }

}  // namespace mi355q

using namespace mi355q;

extern "C" int mi355q_fp8_quantize_groups(const void* x_dev, mi355q_dtype dtype, int64_t rows, int64_t cols,
                                          int64_t ldx, uint8_t* codes_dev, int64_t ld_codes, void* scales_dev,
                                          mi355q_scale_type scale_type, int64_t ld_scales, void* stream) {
  MQ_CHECK_ARG(rows >= 0 && cols > 0 && cols < (int64_t(1) << 30) && ldx >= cols && ld_codes >= cols &&
                   ld_scales >= group_count(cols),
               "fp8_quantize_groups: bad shape");
  if (rows == 0) return MI355Q_OK;
  MQ_CHECK_ARG(x_dev && codes_dev && scales_dev, "fp8_quantize_groups: null pointer");
  MQ_CHECK_ARG(known_dtype(dtype), "fp8_quantize_groups: dtype must be bf16, fp16 or fp32");
  MQ_CHECK_ARG(scale_type == MI355Q_SCALE_F32 || scale_type == MI355Q_SCALE_E8M0,
               "fp8_quantize_groups: unknown scale type");
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int es = dtype_size(dtype);
  const bool vec = cols % kChunk == 0 && (ldx * es) % 16 == 0 && aligned16(x_dev) && ld_codes % kChunk == 0 &&
                   aligned_to(codes_dev, kChunk);
  const int64_t per_row = group_count(cols) * kLanes;
  over_rows(rows, per_row, [&](int64_t r, int64_t n) {
    GroupsArgs a{static_cast<const char*>(x_dev) + r * ldx * es, ldx, cols, codes_dev + r * ld_codes, ld_codes,
                 static_cast<char*>(scales_dev) + r * ld_scales * (scale_type == MI355Q_SCALE_F32 ? 4 : 1), ld_scales,
                 (uint32_t)(n * per_row), fast_div((uint32_t)per_row)};
    with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      const dim3 grid(blocks_of(a.chunks));
      with_access(vec, rows * cols * (es + 1), [&](auto v, auto nt) {
        constexpr bool V = decltype(v)::value, S = decltype(nt)::value;
        if (scale_type == MI355Q_SCALE_E8M0)
          hipLaunchKernelGGL((fp8_groups_kernel<T, true, V, S>), grid, dim3(NT), 0, st, a);
        else
          hipLaunchKernelGGL((fp8_groups_kernel<T, false, V, S>), grid, dim3(NT), 0, st, a);
      });
    });
  });
  MQ_LAUNCH_CHECK();
  return MI355Q_OK;
}

extern "C" int mi355q_fp8_quantize_blocks(const void* w_dev, mi355q_dtype dtype, int64_t rows, int64_t cols,
                                          int64_t ldw, uint8_t* codes_dev, int64_t ld_codes, float* scales_dev,
                                          int64_t ld_scales, void* stream) {
  MQ_CHECK_ARG(rows >= 0 && cols > 0 && ldw >= cols && ld_codes >= cols && ld_scales >= group_count(cols),
               "fp8_quantize_blocks: bad shape");
  if (rows == 0) return MI355Q_OK;
  MQ_CHECK_ARG(w_dev && codes_dev && scales_dev, "fp8_quantize_blocks: null pointer");
  MQ_CHECK_ARG(known_dtype(dtype), "fp8_quantize_blocks: dtype must be bf16, fp16 or fp32");
  const int64_t cb = group_count(cols), n = group_count(rows) * cb;
  MQ_CHECK_ARG(n < (int64_t(1) << 31), "fp8_quantize_blocks: too many blocks");
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool vec = cols % kChunk == 0 && (ldw * dtype_size(dtype)) % 16 == 0 && aligned16(w_dev) &&
                   ld_codes % kChunk == 0 && aligned_to(codes_dev, kChunk);
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const dim3 grid((unsigned)n);
    with_access(vec, rows * cols * (dtype_size(dtype) + 1), [&](auto v, auto nt) {
      hipLaunchKernelGGL((fp8_blocks_kernel<T, decltype(v)::value, decltype(nt)::value>), grid, dim3(NT), 0, st, w_dev,
                         rows, cols, ldw, codes_dev, ld_codes, scales_dev, ld_scales, (uint32_t)cb);
    });
  });
  MQ_LAUNCH_CHECK();
  return MI355Q_OK;
}

extern "C" int mi355q_fp8_silu_mul(const void* x_dev, mi355q_dtype dtype, int64_t rows, int64_t cols, int64_t ldx,
                                   uint8_t* h_codes_dev, int64_t ld_h, uint8_t* h_scales_dev, uint8_t* kept_codes_dev,
                                   int64_t ld_kept, uint8_t* kept_scales_dev, void* stream) {
  MQ_CHECK_ARG(rows >= 0 && cols > 0 && cols < (int64_t(1) << 29) && ldx >= 2 * cols && ld_h >= cols,
               "fp8_silu_mul: bad shape");
  MQ_CHECK_ARG((kept_codes_dev == nullptr) == (kept_scales_dev == nullptr) && (!kept_codes_dev || ld_kept >= 2 * cols),
               "fp8_silu_mul: kept codes and scales come together, 2 cols wide");
  if (rows == 0) return MI355Q_OK;
  MQ_CHECK_ARG(x_dev && h_codes_dev && h_scales_dev, "fp8_silu_mul: null pointer");
  MQ_CHECK_ARG(known_dtype(dtype), "fp8_silu_mul: dtype must be bf16, fp16 or fp32");
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int es = dtype_size(dtype);
  const bool keep = kept_codes_dev != nullptr;
  const bool vec = cols % kChunk == 0 && (ldx * es) % 16 == 0 && aligned16(x_dev) && ld_h % kChunk == 0 &&
                   aligned_to(h_codes_dev, kChunk) &&
                   (!keep || (ld_kept % kChunk == 0 && aligned_to(kept_codes_dev, kChunk)));
  const int64_t groups = group_count(cols), per_row = groups * kLanes;
  over_rows(rows, per_row, [&](int64_t r, int64_t n) {
    GluArgs a{static_cast<const char*>(x_dev) + r * ldx * es, ldx, cols, h_codes_dev + r * ld_h, ld_h,
              h_scales_dev + r * groups, keep ? kept_codes_dev + r * ld_kept : nullptr, ld_kept,
              keep ? kept_scales_dev + r * 2 * groups : nullptr, (uint32_t)(n * per_row),
              fast_div((uint32_t)per_row)};
    with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      const dim3 grid(blocks_of(a.chunks));
      with_access(vec, rows * cols * (2 * es + (keep ? 3 : 1)), [&](auto v, auto nt) {
        constexpr bool V = decltype(v)::value, S = decltype(nt)::value;
        if (keep) hipLaunchKernelGGL((fp8_silu_mul_kernel<T, true, V, S>), grid, dim3(NT), 0, st, a);
        else      hipLaunchKernelGGL((fp8_silu_mul_kernel<T, false, V, S>), grid, dim3(NT), 0, st, a);
      });
    });
  });
  MQ_LAUNCH_CHECK();
  return MI355Q_OK;
}

extern "C" int mi355q_fp8_silu_mul_backward(const void* dh_dev, mi355q_dtype dtype, int64_t rows, int64_t cols,
                                            int64_t ld_dh, const uint8_t* kept_codes_dev, int64_t ld_kept,
                                            const uint8_t* kept_scales_dev, int64_t ld_scales, void* dx_dev,
                                            int64_t ld_dx, void* stream) {
  MQ_CHECK_ARG(rows >= 0 && cols > 0 && cols < (int64_t(1) << 29) && ld_dh >= cols && ld_kept >= 2 * cols &&
                   ld_scales >= 2 * group_count(cols) && ld_dx >= 2 * cols,
               "fp8_silu_mul_backward: bad shape");
  if (rows == 0) return MI355Q_OK;
  MQ_CHECK_ARG(dh_dev && kept_codes_dev && kept_scales_dev && dx_dev, "fp8_silu_mul_backward: null pointer");
  MQ_CHECK_ARG(known_dtype(dtype), "fp8_silu_mul_backward: dtype must be bf16, fp16 or fp32");
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int es = dtype_size(dtype);
  const bool vec = cols % kChunk == 0 && (ld_dh * es) % 16 == 0 && aligned16(dh_dev) && (ld_dx * es) % 16 == 0 &&
                   aligned16(dx_dev) && ld_kept % kChunk == 0 && aligned_to(kept_codes_dev, kChunk);
  const int64_t per_row = group_count(cols) * kLanes;
  over_rows(rows, per_row, [&](int64_t r, int64_t n) {
    GluBackArgs a{static_cast<const char*>(dh_dev) + r * ld_dh * es, ld_dh, cols, kept_codes_dev + r * ld_kept,
                  ld_kept, kept_scales_dev + r * ld_scales, ld_scales, static_cast<char*>(dx_dev) + r * ld_dx * es,
                  ld_dx, (uint32_t)(n * per_row), fast_div((uint32_t)per_row)};
    with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      const dim3 grid(blocks_of(a.chunks));
      with_access(vec, rows * cols * (3 * es + 2), [&](auto v, auto nt) {
        hipLaunchKernelGGL((fp8_silu_mul_backward_kernel<T, decltype(v)::value, decltype(nt)::value>), grid, dim3(NT), 0,
                           st, a);
      });
    });
  });
  MQ_LAUNCH_CHECK();
  return MI355Q_OK;
}
