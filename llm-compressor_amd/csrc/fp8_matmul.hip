// Products of block-scaled fp8 matrices (fp8.h) and their gradients.
//
//   forward      Y[m][n]  = b[n] + sum_kb xs[m][kb] ws[n / 128][kb] sum_{k in kb} x[m][k] w[n][k]
//   grad input   dX[m][k] = sum_nb ws[nb][k / 128] sum_{n in nb} dY[m][n] w[n][k]
//   grad weight  dW[n][k] = sum_m dY[m][n] x[m][k] 2^e[m][k / 128]
//
// x and w are e4m3 codes, dY is bf16.  Codes, and codes times a power of two from
// 2^-117 up (below it a code's last bits fall out of bf16's range), are exact in
// bf16, and products of bf16 values are exact in fp32; so the only roundings are
// those of the fp32 sums, the scales' products and the output.
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
  int c_type;
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
// alignment.  It runs where the tile kernels cannot (operands off 16 bytes without
// a workspace for their copies, pitches past 32-bit offsets), where odd widths
// have a sum of one step, and for a weight gradient of no tokens.  Bound by its
// element loads: input gradient of 8192 x 4096 x 14336 29 ms against the tiles' 0.9.
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

// ---------------------------------------------------------------- forward, tiles
// Rows of 128 codes (one K step) go global -> LDS by the gfx950 LDS-DMA load
// with their 16-byte chunks XOR-swizzled by (row >> 1) & 7: 16 rows of one
// chunk then lie in 16 different 16-byte columns of the banks (two rows a
// 256-byte line of them), which is what a 16-byte read takes at a time.
//
// The fp8 matrix instructions would take the codes as they are at twice the
// rate, but they add with few bits: on heavy-tailed codes 2.9e-4 of the terms'
// magnitudes at the most over 128 terms (16x16x128, 32x32x64, 16x16x32 and 32x32x16
// alike), 2e-5 on normal ones, where the bf16 instructions are within 3.2e-7 and 5e-8
// (512 random tiles each).  So the codes are converted to bf16 in registers (exact,
// two an instruction) and the sums are fp32 sums of exact products.
//
// A step is, per 32 x 32 tile, eight 32x32x16 MFMAs from zero and
// acc += tile * (token scale * block scale) in fp32: the features are the
// MFMA's rows, so a lane holds one token per tile (its scale is one register)
// and the block scale is wave-uniform.
//
// Four waves with 2 x 2 tiles each, two workgroups on a CU: one's scaling and
// conversions run beside the other's MFMAs (one workgroup of eight waves with
// 256 x 128 tiles 2.06 ms against 1.81, where this kernel now takes 1.64 on the same card).
// 8192 x 28672 x 4096 1.64 .. 1.71 ms by the card, 1.13 .. 1.17 PFLOP/s.  Per MFMA it issues 6.3 vector
// instructions (4 conversions, 2 scaling FMAs); MFMAs and vector instructions are
// busy 0.63 and 0.61 of the cycles at 1.68 GHz, down from 2.4: what bounds it is
// power, which the conversions and the traffic from LDS share with the MFMAs.
// (The same loads from one tile's addresses, always in L2: 3 % less.)
typedef __attribute__((address_space(3))) void lds_void_t;

__device__ __forceinline__ uint32_t lds_u32(const void* p) {
  return (uint32_t) reinterpret_cast<uintptr_t>((lds_void_t*)p);
}
// 64 lanes x 16 bytes to LDS at m0, from a scalar base and lane offsets.
// Completion is waited for explicitly (vmcnt).
__device__ __forceinline__ void dma_s(uint32_t off, const void* base, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(m0) : "memory", "m0");
}

// 64 lanes x 1 byte, each as a dword
__device__ __forceinline__ void dma_bytes(uint32_t off, const void* base, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_ubyte %0, %1" ::"v"(off), "s"(base), "s"(m0) : "memory", "m0");
}

typedef int i32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2_t lds_i32x2_t;
typedef short v4s16_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s16_t lds_v4s16_t;

// eight codes times a power of two (its exponent is what counts), as bf16
__device__ __forceinline__ u32x4_t scaled_bf16(uint32_t lo, uint32_t hi, float e) {
  return u32x4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, e, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, e, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, e, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, e, true))};
}
// four tokens of one column each from rows r and r + 4 of PITCH bytes
template <int PITCH>
__device__ __forceinline__ bf16x8_t tr_pair(const char* p) {
  const v4s16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s16_t*)p);
  const v4s16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s16_t*)(p + 4 * PITCH));
  return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
// eight codes as bf16
__device__ __forceinline__ bf16x8_t codes_bf16(uint32_t lo, uint32_t hi) {
  return __builtin_bit_cast(bf16x8_t, scaled_bf16(lo, hi, 1.f));
}

// Work items: the first `full` tiles run whole, the others (what is left over
// when every CU has had its whole tiles) in `splits` parts of the sum each, whose
// fp32 tiles go to partial slots.  The workgroups of one XCD (every eighth) take
// neighbouring tiles, in groups of 8 row tiles, so that they share operands in its L2.
struct TileOrder {
  uint32_t row_tiles, col_tiles, full, splits;
};
struct TileItem {
  uint32_t row, col;   // of the tile
  uint32_t split;
  int64_t slot;        // partial slot, or -1: the output itself
};
__device__ __forceinline__ TileItem tile_of(const TileOrder& o, uint32_t id) {
  const uint32_t rest = o.row_tiles * o.col_tiles - o.full;
  TileItem it;
  uint32_t t;
  if (id < o.full) {
    t = xcd_order(id, o.full);
    it.split = 0;
    it.slot = -1;
  } else {
    const uint32_t lin = xcd_order(id - o.full, rest * o.splits);
    it.split = lin / rest;
    t = o.full + lin - it.split * rest;
    it.slot = o.splits > 1 ? (int64_t)lin : -1;
  }
  const uint32_t g = t / (8 * o.col_tiles), left = o.row_tiles - 8 * g;
  const uint32_t rows = left < 8 ? left : 8, in = t - g * 8 * o.col_tiles;
  it.col = in / rows;
  it.row = 8 * g + in - it.col * rows;
  return it;
}
// the steps [begin, end) of an item: all, or one of `splits` ranges of `per`
__device__ __forceinline__ void item_steps(const TileItem& it, int steps, int per, int& begin, int& end) {
  begin = it.slot < 0 ? 0 : (int)it.split * per;
  end = it.slot < 0 || begin + per > steps ? steps : begin + per;
}

// T x A tiles of 32 tokens x 32 features per wave, WT x WF waves.
template <int T, int A, int WT, int WF>
struct FwdShape {
  static constexpr int W = WT * WF, NTH = 64 * W;
  static constexpr int TT = 32 * T * WT, FT = 32 * A * WF;   // tokens, features per workgroup
  static constexpr int A_SLOT = FT * kGroup, B_SLOT = TT * kGroup;
  // three slots of features, two of tokens: a step's token operands are in
  // registers before the step begins
  static constexpr int RING = 3 * A_SLOT + 2 * B_SLOT;
  static constexpr int PITCH = A * 64 + 16;                  // bytes per token row of the staged output
  static constexpr int BIAS = W * 32 * T * PITCH;            // fp32 biases behind it
  static constexpr int LDS = RING > BIAS + FT * 4 ? RING : BIAS + FT * 4;
};

// One 32 x 32 tile of a split's sums to its partial slot, in fp32 without the
// bias.  Lane l holds row l & 31 and, in registers 4 j .. 4 j + 3, columns
// 8 j + 4 (l / 32) and on; slots hold the tiles in that order (tile, j, lane), so that a
// store moves a whole KB (row by row it moved pieces of 32 bytes: 333 x 4096 x 14336 in 480
// parts 53.3 us, so 50.8).  Rows and tiles past the output's edges are left out.
__device__ __forceinline__ void store_part(float* slot, int tile, const f32x16_t& v, int lane) {
  f32x4_t* const out = reinterpret_cast<f32x4_t*>(slot) + tile * 256 + lane;
#pragma unroll
  for (int j = 0; j < 4; ++j) out[64 * j] = f32x4_t{v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]};
}

// Four neighbouring columns of a row to LDS in the output's type, and 16-byte pieces of
// rows from there to the output, `left` columns before the rows' ends (unaligned in
// rows of odd widths).
template <class O>
__device__ __forceinline__ void stage_columns(char* o, const f32x4_t& v) {
  typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
  typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
  if constexpr (O::code == MI355Q_F32) *reinterpret_cast<f32x4_t*>(o) = v;
  else if constexpr (O::code == MI355Q_BF16) *reinterpret_cast<bf16x4_t*>(o) = __builtin_convertvector(v, bf16x4_t);
  else *reinterpret_cast<f16x4_t*>(o) = __builtin_convertvector(v, f16x4_t);
}
// N pieces of rows `step` bytes apart, the first of row `row`.
template <class O, int RPI, int N>
__device__ __forceinline__ void store_pieces(char* o, int64_t step, const u32x4_t (&v)[N], int64_t row, int64_t rows,
                                             int64_t left, bool whole) {
  constexpr int PER = 16 / sizeof(typename O::raw);
  if (whole) {
#pragma unroll
    for (int i = 0; i < N; ++i) __builtin_memcpy(o + i * step, &v[i], 16);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (row + i * RPI >= rows) break;
    if (left >= PER) {
      __builtin_memcpy(o + i * step, &v[i], 16);
    } else {
      typename O::raw e[PER];
      __builtin_memcpy(e, &v[i], 16);
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (k < left) reinterpret_cast<typename O::raw*>(o + i * step)[k] = e[k];
    }
  }
}
// f(Bf16{} / F16{} / F32{}): the type is told apart once, not at every column
template <class Fn>
__device__ __forceinline__ void by_output_type(int type, Fn&& f) {
  if (type == MI355Q_BF16) f(Bf16{});
  else if (type == MI355Q_F16) f(F16{});
  else f(F32{});
}

// Stores a workgroup's tiles acc[A][T] of C [P][Q] (P on the lanes), laid out as
// above.
template <class S, int T, int A>
__device__ __forceinline__ void store_tiles(const ProductArgs& g, f32x16_t (&acc)[A][T], char* ring, int64_t t0, int64_t f0,
                                            int wt, int wf, int wave, int lane, int64_t slot, float* parts) {
  if (slot >= 0) {
#pragma unroll
    for (int a = 0; a < A; ++a)
#pragma unroll
      for (int b = 0; b < T; ++b) {
        const int r = wt * T + b, q = wf * A + a;
        if (t0 + 32 * r + (lane & 31) < g.P && f0 + 32 * q < g.Q)
          store_part(parts + slot * (S::TT * S::FT), r * (S::FT / 32) + q, acc[a][b], lane);
      }
    return;
  }
  const int64_t tw = t0 + wt * T * 32, fw = f0 + wf * A * 32;   // the wave's first row and column
  __syncthreads();   // the ring is no longer read
  float* const biases = reinterpret_cast<float*>(ring + S::BIAS);
  for (int i = threadIdx.x; i < S::FT; i += S::NTH)
    biases[i] = g.bias && f0 + i < g.Q ? load_typed(g.bias, g.bias_type, f0 + i) : 0.f;
  __syncthreads();
  const float* const bw = biases + wf * A * 32 + 4 * (lane >> 5);
  // Outputs go through LDS (the wave's own part of it), so that a token's features
  // leave as 16-byte stores of whole lines; straight from the tiles they are pieces of
  // 16 or 32 bytes.  A pass of 128 bytes a row: 16-bit types two columns of tiles,
  // fp32 one.  With the type told apart here, rows read before they are stored and whole
  // tiles stored without conditions a 128 x 128 tile takes 1.5 us, with a choice at each
  // column and row 2.4.
  char* const stage = ring + wave * 32 * T * S::PITCH;
  by_output_type(g.c_type, [&](auto type) __attribute__((always_inline)) {
    using O = decltype(type);
    constexpr int ES = sizeof(typename O::raw), GROUP = ES == 4 ? 1 : A, PER = 16 / ES;
    constexpr int LPR = 32 * GROUP / PER, RPI = 64 / LPR, N = 32 * T / RPI;   // lanes per row, rows per pass, passes
    static_assert(A % GROUP == 0 && S::PITCH >= 32 * GROUP * ES + 16, "rows and a shift of the banks");
#pragma unroll
    for (int a0 = 0; a0 < A; a0 += GROUP) {
#pragma unroll
      for (int a = a0; a < a0 + GROUP; ++a)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4_t bias = *reinterpret_cast<const f32x4_t*>(bw + 32 * a + 8 * j);
#pragma unroll
          for (int b = 0; b < T; ++b)
            stage_columns<O>(stage + (32 * b + (lane & 31)) * S::PITCH + (32 * (a - a0) + 8 * j + 4 * (lane >> 5)) * ES,
                             f32x4_t{acc[a][b][4 * j], acc[a][b][4 * j + 1], acc[a][b][4 * j + 2],
                                     acc[a][b][4 * j + 3]} + bias);
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      u32x4_t v[N];
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = *reinterpret_cast<const u32x4_t*>(stage + (i * RPI + lane / LPR) * S::PITCH + 16 * (lane % LPR));
      const int64_t f = fw + 32 * a0 + PER * (lane % LPR), t = tw + lane / LPR;
      store_pieces<O, RPI>(static_cast<char*>(g.c) + (t * g.ldc + f) * ES, RPI * ES * g.ldc, v, t, g.P, g.Q - f,
                           tw + 32 * T <= g.P && fw + 32 * A <= g.Q);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  });
}

template <int T, int A, int WT, int WF, bool E8M0>
__global__ __launch_bounds__(64 * WT * WF) __attribute__((amdgpu_waves_per_eu(2)))
void fp8_forward_kernel(ProductArgs g, TileOrder order, int steps_per_split, float* parts) {
  using S = FwdShape<T, A, WT, WF>;
  __shared__ __attribute__((aligned(16))) char ring[S::LDS];
  char* const ringb = ring + 3 * S::A_SLOT;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wt = wave % WT, wf = wave / WT;
  const TileItem item = tile_of(order, blockIdx.x);
  const int64_t t0 = (int64_t)item.row * S::TT, f0 = (int64_t)item.col * S::FT;
  const int nkb = (int)((g.R + kGroup - 1) / kGroup);
  int s_begin, s_end;
  item_steps(item, nkb, steps_per_split, s_begin, s_end);

  // DMA: instruction j of wave w fills 8 rows; lane l the chunk position l & 7
  // of row l / 8, with the row's chunk (l & 7) ^ ((row >> 1) & 7), the same for
  // every second j.  Rows past the end read the last row again (their results
  // are not stored).
  constexpr int NA = S::FT / 8 / S::W, NB = S::TT / 8 / S::W;
  static_assert(NA * 8 * S::W == S::FT && NB * 8 * S::W == S::TT, "rows per wave");
  static_assert(NA % 2 == 0 && NB % 2 == 0, "a wave's rows begin at a multiple of 16");
  const int chunk[2] = {(lane & 7) ^ (lane >> 4), (lane & 7) ^ (4 + (lane >> 4))};
  uint32_t oa[NA], ob[NB];
#pragma unroll
  for (int j = 0; j < NA; ++j) {
    const int64_t r = f0 + (wave * NA + j) * 8 + (lane >> 3);
    oa[j] = (uint32_t)((r < g.Q ? r : g.Q - 1) - f0) * (uint32_t)g.ldb + 16 * chunk[j & 1];
  }
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int64_t r = t0 + (wave * NB + j) * 8 + (lane >> 3);
    ob[j] = (uint32_t)((r < g.P ? r : g.P - 1) - t0) * (uint32_t)g.lda + 16 * chunk[j & 1];
  }
  const char* const wbase = reinterpret_cast<const char*>(g.b) + f0 * g.ldb;
  const char* const xbase = static_cast<const char*>(g.a) + t0 * g.lda;
  const uint32_t la0 = lds_u32(ring) + wave * NA * 1024, lb0 = lds_u32(ringb) + wave * NB * 1024;
  // A last step of fewer than 128 columns: a chunk past the end is read as its
  // row's first chunk of the step, and the token rows' such chunks are cleared
  // in LDS, so that it adds nothing (a NaN in the first chunk is in the row's
  // sum anyway).
  const int tail = (int)(g.R % kGroup) / 16;                    // whole chunks of a short last step
  auto turn_to_tail = [&](int s) __attribute__((always_inline)) {   // once, before the last step's DMA
    if (tail && s == nkb - 1) {
#pragma unroll
      for (int j = 0; j < NA; ++j) oa[j] -= chunk[j & 1] >= tail ? 16 * chunk[j & 1] : 0;
#pragma unroll
      for (int j = 0; j < NB; ++j) ob[j] -= chunk[j & 1] >= tail ? 16 * chunk[j & 1] : 0;
    }
  };
  auto load_a = [&](int s, int slot, int j) __attribute__((always_inline)) {
    dma_s(oa[j], wbase + (int64_t)s * kGroup, la0 + (uint32_t)(slot % 3) * S::A_SLOT + 1024 * j);
  };
  auto load_b = [&](int s, int slot, int j) __attribute__((always_inline)) {
    dma_s(ob[j], xbase + (int64_t)s * kGroup, lb0 + (uint32_t)(slot & 1) * S::B_SLOT + 1024 * j);
  };
  auto clear_tail = [&](int s, int slot) __attribute__((always_inline)) {
    if (!tail || s != nkb - 1) return;
#pragma unroll
    for (int i = 0; i < S::TT * 8 / S::NTH; ++i) {
      const int at = i * S::NTH + (int)threadIdx.x, row = at >> 3;
      if (((at & 7) ^ ((row >> 1) & 7)) >= tail)
        *reinterpret_cast<u32x4_t*>(ringb + (slot & 1) * S::B_SLOT + at * 16) = u32x4_t{0u, 0u, 0u, 0u};
    }
    __syncthreads();
  };

  // operand reads: lane l holds row l & 31, codes 64 (l / 32) and on: two
  // slices of eight per 16-byte chunk (which codes a slice pairs is free, as
  // long as both operands agree)
  int p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p[i] = (lane & 31) * kGroup + 16 * ((4 * (lane >> 5) + i) ^ ((lane >> 1) & 7));
    asm volatile("" : "+v"(p[i]));
  }
  auto read_a = [&](int slot, int a, int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const u32x4_t*>(ring + (slot % 3) * S::A_SLOT + (wf * A + a) * 32 * kGroup + p[i]);
  };
  auto read_b = [&](int slot, int b, int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const u32x4_t*>(ringb + (slot & 1) * S::B_SLOT + (wt * T + b) * 32 * kGroup + p[i]);
  };

  // scales: this lane's tokens, and the block scale of the wave's features
  uint32_t xsi[T];   // from the tile's first token
#pragma unroll
  for (int b = 0; b < T; ++b) {
    const int64_t t = t0 + (wt * T + b) * 32 + (lane & 31);
    xsi[b] = (uint32_t)((t < g.P ? t : g.P - 1) - t0) * (uint32_t)g.ldas;
    asm volatile("" : "+v"(xsi[b]));
  }
  const char* const xsc = static_cast<const char*>(g.as) + t0 * g.ldas * (E8M0 ? 1 : 4);
  int64_t fb = (f0 + wf * A * 32) / kGroup;
  if (fb > (g.Q - 1) / kGroup) fb = (g.Q - 1) / kGroup;
  const float* const wsc = g.bs + fb * g.ldbs;
  uint32_t sx_load[T];
  float sw_load;
  auto load_scales = [&](int s) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < T; ++b) {
      if constexpr (E8M0) sx_load[b] = reinterpret_cast<const uint8_t*>(xsc + s)[xsi[b]];
      else sx_load[b] = reinterpret_cast<const uint32_t*>(xsc + 4 * (int64_t)s)[xsi[b]];
    }
    sw_load = wsc[s];
  };
  float sc[T], sc_next[T];
  auto take_scales = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < T; ++b) {
      asm volatile("" : "+v"(sx_load[b]));   // (not converted where it is loaded, which would wait for it there)
      sc_next[b] = (E8M0 ? e8m0_to_f32(sx_load[b]) : __uint_as_float(sx_load[b])) * sw_load;
      asm volatile("" : "+v"(sc_next[b]));
    }
  };

  f32x16_t acc[A][T];
#pragma unroll
  for (int a = 0; a < A; ++a)
#pragma unroll
    for (int b = 0; b < T; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;
  bf16x8_t xb[T][8];   // the step's token operands
  u32x4_t ra;          // the next two slices of the features, as codes
  auto convert_b = [&](const u32x4_t* raw, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < T; ++b) {
      xb[b][2 * i] = codes_bf16(raw[b][0], raw[b][1]);
      xb[b][2 * i + 1] = codes_bf16(raw[b][2], raw[b][3]);
    }
  };

  // Step s.  Its token operands and first feature codes are in registers; the
  // barrier before its last row of tiles publishes step s + 1 and frees the
  // feature slot of step s - 1 and the token slot of step s for step s + 2,
  // whose DMA then has a step's time.  In the last row of tiles each token
  // operand is replaced by its successor's as soon as its last MFMA is issued.
  // Slots count from the item's first step.  Steps that are far enough from the
  // end (INNER) leave out its conditions and have their slot numbers `c` as
  // constants.
  auto step = [&](int s, int c, auto inner) __attribute__((always_inline)) {
    constexpr bool INNER = decltype(inner)::value;
    // past the last step the loads repeat it, into slots that nothing reads:
    // without a branch in the step the compiler keeps the sums between the MFMAs
    const int s1 = INNER || s + 1 < s_end ? s + 1 : s, s2 = INNER || s + 2 < s_end ? s + 2 : s_end - 1;
    u32x4_t rb[T];
#pragma unroll
    for (int b = 0; b < T; ++b) sc[b] = sc_next[b];
#pragma unroll
    for (int a = 0; a < A; ++a) {
      constexpr int LAST = A - 1;
      if (a == LAST) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        if constexpr (!INNER) {
          if (s1 != s) clear_tail(s1, c + 1);
          if (s2 > s1) turn_to_tail(s2);
        }
        // (the scales of step s + 1 were requested a step ago, with the DMA
        // that the wait above is for: a use anywhere else would wait for the
        // DMA issued since)
        take_scales();
        load_scales(s2);
#pragma unroll
        for (int b = 0; b < T; ++b) rb[b] = read_b(c + 1, b, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      f32x16_t t[T];
#pragma unroll
      for (int b = 0; b < T; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) t[b][e] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bf16x8_t f0r = codes_bf16(ra[0], ra[1]), f1r = codes_bf16(ra[2], ra[3]);
        ra = i < 3 ? read_a(c, a, i + 1) : a < LAST ? read_a(c, a + 1, 0) : read_a(c + 1, 0, 0);
#pragma unroll
        for (int b = 0; b < T; ++b) t[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f0r, xb[b][2 * i], t[b], 0, 0, 0);
#pragma unroll
        for (int b = 0; b < T; ++b)
          t[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f1r, xb[b][2 * i + 1], t[b], 0, 0, 0);
        if (a == LAST) {
          convert_b(rb, i);
          if (i < 3) {
#pragma unroll
            for (int b = 0; b < T; ++b) rb[b] = read_b(c + 1, b, i + 1);
          }
#pragma unroll
          for (int j = 0; j < NA; ++j)
            if (j * 4 / NA == i) load_a(s2, c + 2, j);
#pragma unroll
          for (int j = 0; j < NB; ++j)
            if (j * 4 / NB == i) load_b(s2, c + 2, j);
        }
      }
#pragma unroll
      for (int b = 0; b < T; ++b) {
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[a][b][e] = fmaf(t[b][e], sc[b], acc[a][b][e]);
        asm volatile("" : "+v"(acc[a][b]));
      }
    }
  };

  {   // every split has a step
    const int s1 = s_begin + 1 < s_end ? s_begin + 1 : s_begin;
    turn_to_tail(s_begin);
#pragma unroll
    for (int j = 0; j < NA; ++j) load_a(s_begin, 0, j);
#pragma unroll
    for (int j = 0; j < NB; ++j) load_b(s_begin, 0, j);
    load_scales(s_begin);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    clear_tail(s_begin, 0);
    take_scales();
    load_scales(s1);
    if (s1 > s_begin) turn_to_tail(s1);
#pragma unroll
    for (int j = 0; j < NA; ++j) load_a(s1, 1, j);
#pragma unroll
    for (int j = 0; j < NB; ++j) load_b(s1, 1, j);
    ra = read_a(0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4_t rb[T];
#pragma unroll
      for (int b = 0; b < T; ++b) rb[b] = read_b(0, b, i);
      convert_b(rb, i);
    }
    int s = s_begin;
    for (; s + 8 < s_end; s += 6) {   // s + 5 + 2, the last one loaded for, is before the item's last step
      step(s, 0, std::true_type{});
      step(s + 1, 1, std::true_type{});
      step(s + 2, 2, std::true_type{});
      step(s + 3, 3, std::true_type{});
      step(s + 4, 4, std::true_type{});
      step(s + 5, 5, std::true_type{});
    }
    for (int c = 0; s < s_end; ++s, ++c) step(s, c, std::false_type{});
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // before the ring is used again
  }

  store_tiles<S, T, A>(g, acc, ring, t0, f0, wt, wf, wave, lane, item.slot, parts);
}

// ---------------------------------------------------------------- input gradient
// As the forward product, with dY's rows (bf16, n contiguous) as the tokens and
// the weight's 32 x 16 operands taken from its rows as they lie: the transposing
// LDS load ds_read_b64_tr_b8 gives lane l of a group of 16 column l of the eight
// rows whose 16-byte pieces the lane pairs point to, that is eight n of one k,
// which are converted to bf16 in registers.  A step is 64 n; the tiles' sums
// run over the two steps of a 128 x 128 block before they take its scale.
//
// 128 x 128 tiles on four waves, two workgroups on a CU (256 x 128 on eight waves
// 1.03 .. 1.05 ms against 1.00 .. 1.02, before the steps lost their conditions).
// 8192 x 4096 x 14336 0.89 .. 0.91 ms by the card, 1.05 .. 1.08 PFLOP/s: MFMAs busy 0.60 of the cycles, vector
// instructions 0.40, at 1.62 GHz: power again, and the LDS, which carries dY in
// 16 bits.  Few tiles are bound by a wave's instructions, not by what they wait
// for: rings of five and seven steps took as long as this one of three.
template <int T, int WT>
struct GradInputShape {
  static constexpr int A = 2, WF = 2;                        // 128 columns: one block scale per workgroup
  static constexpr int W = WT * WF, NTH = 64 * W;
  static constexpr int TT = 32 * T * WT, FT = 32 * A * WF, SN = 64;
  static constexpr int A_SLOT = SN * FT, B_SLOT = TT * SN * 2, NAS = 4, NBS = 3;
  static constexpr int RING = NAS * A_SLOT + NBS * B_SLOT;
  static constexpr int PITCH = A * 64 + 16;
  static constexpr int BIAS = W * 32 * T * PITCH;
  static constexpr int LDS = RING > BIAS + FT * 4 ? RING : BIAS + FT * 4;
};

template <int T, int WT>
__global__ __launch_bounds__(128 * WT) __attribute__((amdgpu_waves_per_eu(2)))
void fp8_grad_input_kernel(ProductArgs g, TileOrder order, int blocks_per_split, float* parts) {
  using S = GradInputShape<T, WT>;
  constexpr int A = S::A;
  __shared__ __attribute__((aligned(16))) char ring[S::LDS];
  char* const ringb = ring + S::NAS * S::A_SLOT;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wt = wave % WT, wf = wave / WT;
  const TileItem item = tile_of(order, blockIdx.x);
  const int64_t t0 = (int64_t)item.row * S::TT, f0 = (int64_t)item.col * S::FT;
  const int nst = (int)((g.R + S::SN - 1) / S::SN);
  int s_begin, s_end;
  item_steps(item, nst, 2 * blocks_per_split, s_begin, s_end);

  // DMA: 8 rows of 128 bytes an instruction; n rows of the weight with chunk
  // (l & 7) ^ (row & 7) at position l & 7 (the eight rows of a transposed read), token
  // rows of dY with (l & 7) ^ ((row >> 1) & 7), as in the forward product.  Columns and tokens past the
  // end repeat the last ones (not stored); n past the end repeat the last weight
  // row and meet zeros of dY (cleared in LDS; codes hold no infinity, and a
  // NaN of the last row is in the sum anyway).
  constexpr int NA = S::SN / 8 / S::W, NB = S::TT / 8 / S::W;
  static_assert(NA * 8 * S::W == S::SN && NB * 8 * S::W == S::TT, "rows per wave");
  static_assert(NB % 2 == 0, "a wave's token rows begin at a multiple of 16");
  const int chunk = (lane & 7) ^ (lane >> 3), ychunk[2] = {(lane & 7) ^ (lane >> 4), (lane & 7) ^ (4 + (lane >> 4))};
  const int last_rows = (int)(g.R - (int64_t)(nst - 1) * S::SN);
  const int64_t wide = (g.Q + 15) & ~int64_t(15);   // (a padded copy's width)
  const int64_t wcol = f0 + 16 * chunk < wide ? f0 + 16 * chunk : wide - 16;
  uint32_t oa[NA], ob[NB];
#pragma unroll
  for (int j = 0; j < NA; ++j)
    oa[j] = (uint32_t)((wave * NA + j) * 8 + (lane >> 3)) * (uint32_t)g.ldb + (uint32_t)(wcol - f0);
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int64_t r = t0 + (wave * NB + j) * 8 + (lane >> 3);
    ob[j] = (uint32_t)((r < g.P ? r : g.P - 1) - t0) * (uint32_t)(2 * g.lda) + 16 * ychunk[j & 1];
  }
  const char* const wbase = reinterpret_cast<const char*>(g.b) + f0;
  const char* const ybase = static_cast<const char*>(g.a) + 2 * t0 * g.lda;
  const uint32_t la0 = lds_u32(ring) + wave * NA * 1024, lb0 = lds_u32(ringb) + wave * NB * 1024;
  const int tail = (int)((g.R + 7) / 8 % (S::SN / 8));   // whole chunks of dY (the last one may be padded)
  auto turn_to_tail = [&](int s) __attribute__((always_inline)) {   // once, before the last step's DMA
    if (last_rows < S::SN && s == nst - 1) {
#pragma unroll
      for (int j = 0; j < NA; ++j) {
        const int r = (wave * NA + j) * 8 + (lane >> 3);
        oa[j] -= r >= last_rows ? (uint32_t)(r - (last_rows - 1)) * (uint32_t)g.ldb : 0u;
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) ob[j] -= tail && ychunk[j & 1] >= tail ? 16 * ychunk[j & 1] : 0;
    }
  };
  auto load_a = [&](int s, int slot, int j) __attribute__((always_inline)) {
    dma_s(oa[j], wbase + (int64_t)s * S::SN * g.ldb, la0 + (uint32_t)(slot % S::NAS) * S::A_SLOT + 1024 * j);
  };
  auto load_b = [&](int s, int slot, int j) __attribute__((always_inline)) {
    dma_s(ob[j], ybase + (int64_t)s * S::SN * 2, lb0 + (uint32_t)(slot % S::NBS) * S::B_SLOT + 1024 * j);
  };
  auto load = [&](int s, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NA; ++j) load_a(s, slot, j);
#pragma unroll
    for (int j = 0; j < NB; ++j) load_b(s, slot, j);
  };
  auto clear_tail = [&](int s, int slot) __attribute__((always_inline)) {
    if (!tail || s != nst - 1) return;
#pragma unroll
    for (int i = 0; i < S::TT * 8 / S::NTH; ++i) {
      const int at = i * S::NTH + (int)threadIdx.x, row = at >> 3;
      if (((at & 7) ^ ((row >> 1) & 7)) >= tail)
        *reinterpret_cast<u32x4_t*>(ringb + (slot % S::NBS) * S::B_SLOT + at * 16) = u32x4_t{0u, 0u, 0u, 0u};
    }
    __syncthreads();
  };

  // operand reads: slice j of a step is n = 16 j .. 16 j + 15, eight per half wave
  const int gq = lane >> 4, gi = lane & 15;
  int pa[A], pb[4];
#pragma unroll
  for (int a = 0; a < A; ++a) {
    pa[a] = (8 * (gq >> 1) + (gi >> 1)) * S::FT + 16 * ((wf * 4 + 2 * a + (gq & 1)) ^ (gi >> 1)) + 8 * (gi & 1);
    asm volatile("" : "+v"(pa[a]));
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    pb[j] = (wt * T * 32 + (lane & 31)) * 2 * S::SN + 16 * ((2 * j + (lane >> 5)) ^ ((lane >> 1) & 7));
    asm volatile("" : "+v"(pb[j]));
  }
  auto read_a = [&](int slot, int a, int j) __attribute__((always_inline)) {
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32(
        (lds_i32x2_t*)(ring + (slot % S::NAS) * S::A_SLOT + j * 16 * S::FT + pa[a]));
  };
  auto read_b = [&](int slot, int b, int j) __attribute__((always_inline)) {
    return *reinterpret_cast<const bf16x8_t*>(ringb + (slot % S::NBS) * S::B_SLOT + b * 32 * 2 * S::SN + pb[j]);
  };

  // the block scales of this column of blocks, 64 at a time, one per lane
  const float* const wsc = g.bs + f0 / kGroup;
  const int nb = (int)((g.R + kGroup - 1) / kGroup);
  float scales = 0.f;

  f32x16_t acc[A][T], t[A][T];
#pragma unroll
  for (int a = 0; a < A; ++a)
#pragma unroll
    for (int b = 0; b < T; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;
  bf16x8_t xb[T][4];
  i32x2_t ra;

  // Step s: as in the forward product, the barrier before the last row of tiles
  // publishes step s + 1 (its DMA, two steps old, is waited for; the youngest
  // step's stays in flight) and frees the slots that step s + 3 takes.
  auto step = [&](int s, int c, bool first, bool last, float sw, auto inner) __attribute__((always_inline)) {
    constexpr bool INNER = decltype(inner)::value;
    const int s1 = INNER || s + 1 < s_end ? s + 1 : s, s3 = INNER || s + 3 < s_end ? s + 3 : s_end - 1;
#pragma unroll
    for (int a = 0; a < A; ++a) {
      if (a == A - 1) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(NA + NB) : "memory");
        if constexpr (!INNER) {
          if (s1 != s) clear_tail(s1, c + 1);
          if (s + 3 < s_end) turn_to_tail(s + 3);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (first)
#pragma unroll
        for (int b = 0; b < T; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e) t[a][b][e] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bf16x8_t f = codes_bf16(ra[0], ra[1]);
        ra = j < 3 ? read_a(c, a, j + 1) : a < A - 1 ? read_a(c, a + 1, 0) : read_a(c + 1, 0, 0);
#pragma unroll
        for (int b = 0; b < T; ++b) t[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, xb[b][j], t[a][b], 0, 0, 0);
        if (a == A - 1) {
#pragma unroll
          for (int b = 0; b < T; ++b) xb[b][j] = read_b(c + 1, b, j);
#pragma unroll
          for (int i = 0; i < NA; ++i)
            if (i * 4 / NA == j) load_a(s3, c + 3, i);
#pragma unroll
          for (int i = 0; i < NB; ++i)
            if (i * 4 / NB == j) load_b(s3, c + 3, i);
        }
      }
      if (last)
#pragma unroll
        for (int b = 0; b < T; ++b) {
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[a][b][e] = fmaf(t[a][b][e], sw, acc[a][b][e]);
          asm volatile("" : "+v"(acc[a][b]));
        }
    }
  };

  const int s_last = s_end - 1;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    if (s_begin + i < s_end) turn_to_tail(s_begin + i);
    load(s_begin + i < s_end ? s_begin + i : s_last, i);
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * (NA + NB)) : "memory");
  clear_tail(s_begin, 0);
  ra = read_a(0, 0, 0);
#pragma unroll
  for (int b = 0; b < T; ++b)
#pragma unroll
    for (int j = 0; j < 4; ++j) xb[b][j] = read_b(0, b, j);
  auto scale_of = [&](int blk) __attribute__((always_inline)) {
    const int rel = blk - (s_begin >> 1);
    if ((rel & 63) == 0) {
      const int i = blk + lane < nb ? blk + lane : nb - 1;
      scales = wsc[(int64_t)i * g.ldbs];
    }
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(scales), rel & 63));
  };
  int s = s_begin;
  for (; s + 15 < s_end; s += 12) {   // s + 11 + 3, the last one loaded for, is before the item's last step
#pragma unroll
    for (int c = 0; c < 12; c += 2) {
      const float sw = scale_of((s + c) >> 1);
      step(s + c, c, true, false, sw, std::true_type{});
      step(s + c + 1, c + 1, false, true, sw, std::true_type{});
    }
  }
  int c = 0;
  for (; s + 1 < s_end; s += 2, c += 2) {
    const float sw = scale_of(s >> 1);
    step(s, c, true, false, sw, std::false_type{});
    step(s + 1, c + 1, false, true, sw, std::false_type{});
  }
  if (s < s_end) step(s, c, true, true, scale_of(s >> 1), std::false_type{});   // a last block of 64 n or fewer
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // before the ring is used again
  store_tiles<S, T, A>(g, acc, ring, t0, f0, wt, wf, wave, lane, item.slot, parts);
}

// ---------------------------------------------------------------- weight gradient
// C[n][k] over tokens m: both operands are needed with m contiguous and lie with m
// as the row, so both come from LDS through the transposing load
// ds_read_b64_tr_b16: lane l = 16 g + 4 q + r receives element r of the 8-byte rows
// that lanes 16 g + 4 e + q, e = 0..3 point to; two of them are eight tokens of
// one column.  Rows are stored with their 16-byte chunks XORed by 4 (row & 3),
// which keeps reads and writes free of bank conflicts.  dY goes to LDS as it is
// (DMA); the checkpoint's scale changes with the token, along the sum, so it has
// to be in the operand: each wave's DMA brings codes and scale bytes of its own
// rows, and the wave writes them to LDS as bf16, scaled by the conversion (exact).
// The MFMAs then add straight into the accumulators: vector instructions are few
// (busy 0.14 of the cycles), so a large tile on eight waves, 256 x 256, saves
// LDS reads (one wave's operands serve 4 x 2 tiles).  8192 x 4096 x 14336 0.78 .. 0.81 ms
// by the card, 1.19 .. 1.24 PFLOP/s, 17 us of it the sum of the split tiles; MFMAs busy 0.65 of the cycles
// at 1.76 GHz.  Bound by power, and by the LDS, which a stage's rows pass twice.
template <int MB, int NB2, int WK, int WN>
struct GradWeightShape {
  static constexpr int W = WK * WN, NTH = 64 * W;
  static constexpr int FK = 32 * MB * WK, FN = 32 * NB2 * WN, SM = 32;   // k, n per workgroup, tokens per stage
  static constexpr int NS = 4, NRS = 2;                       // slots of bf16 rows, of a wave's raw rows
  static constexpr int X_SLOT = SM * FK * 2, Y_SLOT = SM * FN * 2;
  static constexpr int RAW = 1024 + 256;                      // a wave's codes and scale bytes (as dwords)
  static constexpr int RING = NS * (X_SLOT + Y_SLOT) + W * NRS * RAW;
  static constexpr int PITCH = 32 * MB * 4 + 16;              // bytes per staged output row (fp32)
  static constexpr int STAGED = W * 32 * PITCH;
  static constexpr int LDS = RING > STAGED ? RING : STAGED;
  static_assert(SM * FK == NTH * 16, "one 16-byte chunk of codes per thread and stage");
};

// A wave's tiles through LDS, one row of them at a time: lane l holds column n l & 31
// and four consecutive k a register quad; rows of 32 MB k leave as whole lines.
template <class O, int MB, int NB2, int PITCH>
__device__ __forceinline__ void store_weight_rows(const ProductArgs& g, f32x16_t (&acc)[MB][NB2], char* stage, int64_t nw,
                                                  int64_t kw, int lane) {
  constexpr int ES = sizeof(typename O::raw), PER = 16 / ES;
  constexpr int LPR = 32 * MB / PER, RPI = 64 / LPR, N = 32 / RPI;   // lanes per row, rows per pass, passes
  const int64_t k = kw + PER * (lane % LPR);
#pragma unroll
  for (int y = 0; y < NB2; ++y) {
#pragma unroll
    for (int x = 0; x < MB; ++x)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        stage_columns<O>(stage + (lane & 31) * PITCH + (32 * x + 8 * j + 4 * (lane >> 5)) * ES,
                         f32x4_t{acc[x][y][4 * j], acc[x][y][4 * j + 1], acc[x][y][4 * j + 2], acc[x][y][4 * j + 3]});
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave's own region
    u32x4_t v[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = *reinterpret_cast<const u32x4_t*>(stage + (i * RPI + lane / LPR) * PITCH + 16 * (lane % LPR));
    const int64_t n = nw + y * 32 + lane / LPR;
    store_pieces<O, RPI>(static_cast<char*>(g.c) + (n * g.ldc + k) * ES, RPI * ES * g.ldc, v, n, g.P, g.Q - k,
                         nw + 32 * NB2 <= g.P && kw + 32 * MB <= g.Q);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

template <int MB, int NB2, int WK, int WN>
__global__ __launch_bounds__(64 * WK * WN) __attribute__((amdgpu_waves_per_eu(2)))
void fp8_grad_weight_kernel(ProductArgs g, TileOrder order, int stages_per_split, float* parts) {
  using S = GradWeightShape<MB, NB2, WK, WN>;
  __shared__ __attribute__((aligned(16))) char ring[S::LDS];
  char* const ringy = ring + S::NS * S::X_SLOT;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char* const raw = ringy + S::NS * S::Y_SLOT + wave * S::NRS * S::RAW;
  const int wn = wave % WN, wk = wave / WN;
  const TileItem item = tile_of(order, blockIdx.x);
  const int64_t n0 = (int64_t)item.row * S::FN, k0 = (int64_t)item.col * S::FK;
  const int nst = (int)((g.R + S::SM - 1) / S::SM);
  int s_begin, s_end;
  item_steps(item, nst, stages_per_split, s_begin, s_end);
  const int last_rows = (int)(g.R - (int64_t)(nst - 1) * S::SM);   // tokens of the last stage

  // DMA of dY: 1 KB an instruction, RPI rows; n past the end repeat the last ones
  // (not stored), tokens past the end the last one (cleared in LDS, as are
  // their checkpoint rows: an infinity there must not meet a zero).
  constexpr int YC = S::FN / 8, RPI = 64 / YC, NY = S::SM / RPI / S::W;
  const int64_t ywide = (g.P + 7) & ~int64_t(7), xwide = (g.Q + 15) & ~int64_t(15);   // (padded copies' widths)
  uint32_t oy[NY];
#pragma unroll
  for (int j = 0; j < NY; ++j) {
    const int row = (wave * NY + j) * RPI + lane / YC;
    const int64_t col = n0 + 8 * ((lane % YC) ^ (4 * (row & 3))), c = col < ywide ? col : ywide - 8;
    oy[j] = (uint32_t)row * (uint32_t)(2 * g.lda) + (uint32_t)(2 * (c - n0));
  }
  // ... of the checkpoint: lane l takes 16 codes of row XR l / XC of the wave's
  constexpr int XC = S::FK / 16, XR = 64 / XC;
  const int xrow = wave * XR + lane / XC, xch = lane % XC;
  const int64_t xcol = k0 + 16 * xch < xwide ? k0 + 16 * xch : xwide - 16;
  uint32_t ox = (uint32_t)xrow * (uint32_t)g.ldb + (uint32_t)(xcol - k0);
  uint32_t oe = (uint32_t)xrow * (uint32_t)g.ldbs + (uint32_t)(xcol / kGroup - k0 / kGroup);
  // before the last stage's DMA, once (dY's turn comes a stage after the checkpoint's)
  auto turn_x = [&](int s) __attribute__((always_inline)) {
    if (last_rows < S::SM && s == nst - 1 && xrow >= last_rows) {
      ox -= (uint32_t)(xrow - (last_rows - 1)) * (uint32_t)g.ldb;
      oe -= (uint32_t)(xrow - (last_rows - 1)) * (uint32_t)g.ldbs;
    }
  };
  auto turn_y = [&](int s) __attribute__((always_inline)) {
    if (last_rows < S::SM && s == nst - 1)
#pragma unroll
      for (int j = 0; j < NY; ++j) {
        const int row = (wave * NY + j) * RPI + lane / YC;
        oy[j] -= row >= last_rows ? (uint32_t)(row - (last_rows - 1)) * (uint32_t)(2 * g.lda) : 0u;
      }
  };
  // running stage bases; they stop at the item's last stage
  const int64_t ystep = (int64_t)S::SM * 2 * g.lda, xstep = (int64_t)S::SM * g.ldb, estep = (int64_t)S::SM * g.ldbs;
  const char* yp = static_cast<const char*>(g.a) + 2 * n0 + s_begin * ystep;
  const char* xp = reinterpret_cast<const char*>(g.b) + k0 + s_begin * xstep;
  const char* ep = reinterpret_cast<const char*>(g.be) + k0 / kGroup + s_begin * estep;
  const uint32_t ly0 = lds_u32(ringy) + wave * NY * 1024, lr0 = lds_u32(raw);
  auto load_y = [&](int slot, int j) __attribute__((always_inline)) {
    dma_s(oy[j], yp, ly0 + (uint32_t)(slot % S::NS) * S::Y_SLOT + 1024 * j);
  };
  auto load_x = [&](int slot) __attribute__((always_inline)) {
    const uint32_t m0 = lr0 + (uint32_t)(slot % S::NRS) * S::RAW;
    dma_s(ox, xp, m0);
    dma_bytes(oe, ep, m0 + 1024);
  };
  auto next_y = [&](int s) __attribute__((always_inline)) { yp += s < s_end ? ystep : 0; };   // to stage s
  auto next_x = [&](int s) __attribute__((always_inline)) {
    xp += s < s_end ? xstep : 0;
    ep += s < s_end ? estep : 0;
  };
  constexpr int NDMA = NY + 2;
  // the wave's rows of a stage as bf16: (byte << 23) | 2^22 is the scale as the
  // conversion reads it, by its exponent alone (0: the subnormal 2^-127, 255:
  // NaN).  Half of the lanes take the second half of their 16 codes first, so that
  // 8 or 16 neighbouring lanes write to as many different 16-byte columns of the
  // banks.
  const int xswap = ((lane >> 2) ^ (lane >> 3)) & 1;
  const int xw = xrow * S::FK * 2 + 16 * ((2 * xch) ^ (4 * (xrow & 3))) + 16 * xswap, xw2 = xw + 16 - 32 * xswap;
  const int rr = 16 * lane + 8 * xswap, rr2 = rr + 8 - 16 * xswap;
  i32x2_t raw0, raw1;
  uint32_t raw_byte;
  auto fetch = [&](int slot) __attribute__((always_inline)) {
    const char* r = raw + (slot % S::NRS) * S::RAW;
    raw0 = *reinterpret_cast<const i32x2_t*>(r + rr);
    raw1 = *reinterpret_cast<const i32x2_t*>(r + rr2);
    raw_byte = *reinterpret_cast<const uint32_t*>(r + 1024 + 4 * lane);
  };
  auto convert = [&](int slot) __attribute__((always_inline)) {
    const float e = __uint_as_float((raw_byte << 23) | 0x00400000u);
    char* w = ring + (slot % S::NS) * S::X_SLOT;
    *reinterpret_cast<u32x4_t*>(w + xw) = scaled_bf16((uint32_t)raw0[0], (uint32_t)raw0[1], e);
    *reinterpret_cast<u32x4_t*>(w + xw2) = scaled_bf16((uint32_t)raw1[0], (uint32_t)raw1[1], e);
  };
  auto clear_tail = [&](int s, int slot) __attribute__((always_inline)) {
    if (last_rows == S::SM || s != nst - 1) return;
    char* y = ringy + (slot % S::NS) * S::Y_SLOT;
    for (int i = last_rows * YC + (int)threadIdx.x; i < S::SM * YC; i += S::NTH)
      *reinterpret_cast<u32x4_t*>(y + 16 * i) = u32x4_t{0u, 0u, 0u, 0u};
    char* x = ring + (slot % S::NS) * S::X_SLOT;
    for (int i = last_rows * (S::FK / 8) + (int)threadIdx.x; i < S::SM * (S::FK / 8); i += S::NTH)
      *reinterpret_cast<u32x4_t*>(x + 16 * i) = u32x4_t{0u, 0u, 0u, 0u};
    __syncthreads();
  };

  // operand reads: lane 16 g + 4 e + q points to row 8 (g / 2) + e (and + 4) of a
  // 16-token slice, columns 16 (g & 1) + 4 q of the 32-column block
  const int gg = lane >> 4, ee = (lane >> 2) & 3, qq = lane & 3;
  int px[MB], py[NB2];
#pragma unroll
  for (int b = 0; b < MB; ++b)
    px[b] = (8 * (gg >> 1) + ee) * S::FK * 2 + 8 * (qq & 1) +
            16 * ((4 * ((MB * wk + b) ^ ee)) + 2 * (gg & 1) + (qq >> 1));
#pragma unroll
  for (int b = 0; b < NB2; ++b)
    py[b] = (8 * (gg >> 1) + ee) * S::FN * 2 + 8 * (qq & 1) +
            16 * ((4 * ((NB2 * wn + b) ^ ee)) + 2 * (gg & 1) + (qq >> 1));
  auto read_x = [&](int slot, int kk, int b) __attribute__((always_inline)) {
    return tr_pair<S::FK * 2>(ring + (slot % S::NS) * S::X_SLOT + kk * 16 * S::FK * 2 + px[b]);
  };
  auto read_y = [&](int slot, int kk, int b) __attribute__((always_inline)) {
    return tr_pair<S::FN * 2>(ringy + (slot % S::NS) * S::Y_SLOT + kk * 16 * S::FN * 2 + py[b]);
  };

  f32x16_t acc[MB][NB2];
#pragma unroll
  for (int x = 0; x < MB; ++x)
#pragma unroll
    for (int y = 0; y < NB2; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[x][y][e] = 0.f;
  bf16x8_t fx0[MB], fy0[NB2], fx1[MB], fy1[NB2];

  // Stage s, in two slices of 16 tokens; while one is multiplied the other's
  // operands are read.  The barrier between them publishes stage s + 1 (dY's DMA
  // and the converted rows; the checkpoint rows of stage s + 2 have arrived as well)
  // and frees the slots of stage s - 1.  Scalar instructions are a third of what a
  // wave issues, so stages that are far enough from the end (INNER) leave out its
  // conditions, and their slot `c` is a constant in four copies of them.
  auto stage = [&](int s, int c, auto inner) __attribute__((always_inline)) {
    constexpr bool INNER = decltype(inner)::value;
    static_assert(MB * NB2 >= MB + NB2, "an MFMA for each operand read");
#pragma unroll
    for (int i = 0; i < MB * NB2; ++i) {
      const int x = i / NB2, y = i % NB2;
      acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fx0[x], fy0[y], acc[x][y], 0, 0, 0);
      if (i < NB2) fy1[i] = read_y(c, 1, i);
      else if (i < NB2 + MB) fx1[i - NB2] = read_x(c, 1, i - NB2);
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(NDMA) : "memory");
    if constexpr (INNER) {
      yp += ystep;
      xp += xstep;
      ep += estep;
    } else {
      if (s + 1 < s_end) clear_tail(s + 1, c + 1);
      next_y(s + 3);
      next_x(s + 4);
      if (s + 3 < s_end) turn_y(s + 3);
      if (s + 4 < s_end) turn_x(s + 4);
    }
    __builtin_amdgcn_sched_barrier(0);
    fetch(c + 2);
#pragma unroll
    for (int i = 0; i < MB * NB2; ++i) {
      const int x = i / NB2, y = i % NB2;
      acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fx1[x], fy1[y], acc[x][y], 0, 0, 0);
      if (i < NB2) fy0[i] = read_y(c + 1, 0, i);
      else if (i < NB2 + MB) fx0[i - NB2] = read_x(c + 1, 0, i - NB2);
      if (i < NY) load_y(c + 3, i);
      if (i == MB * NB2 - 2) convert(c + 2);
      if (i == MB * NB2 - 1) load_x(c + 4);   // into the slot that `convert` has emptied
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  {   // every item has a stage; slots count from its first one
    auto start_x = [&](int i) __attribute__((always_inline)) {
      if (i > 0) next_x(s_begin + i);
      if (s_begin + i < s_end) turn_x(s_begin + i);
      load_x(i);
    };
    auto start_y = [&](int i) __attribute__((always_inline)) {
      if (i > 0) next_y(s_begin + i);
      if (s_begin + i < s_end) turn_y(s_begin + i);
#pragma unroll
      for (int j = 0; j < NY; ++j) load_y(i, j);
    };
    start_x(0);
    start_x(1);
    start_y(0);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NY) : "memory");
    fetch(0);
    convert(0);
    fetch(1);
    convert(1);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the raw slots are read
    start_y(1);
    start_x(2);
    start_y(2);
    start_x(3);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * NDMA) : "memory");
    clear_tail(s_begin, 0);
#pragma unroll
    for (int b = 0; b < NB2; ++b) fy0[b] = read_y(0, 0, b);
#pragma unroll
    for (int b = 0; b < MB; ++b) fx0[b] = read_x(0, 0, b);
    int s = s_begin;
    for (; s + 8 < s_end; s += 4) {   // s + 3 + 4, the last one loaded for, is before the item's last stage
      stage(s, 0, std::true_type{});
      stage(s + 1, 1, std::true_type{});
      stage(s + 2, 2, std::true_type{});
      stage(s + 3, 3, std::true_type{});
    }
    for (int c = 0; s < s_end; ++s, ++c) stage(s, c, std::false_type{});
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // before the ring is used again
  }

  const int64_t kw = k0 + wk * MB * 32;
  if (item.slot >= 0) {
#pragma unroll
    for (int y = 0; y < NB2; ++y)
#pragma unroll
      for (int x = 0; x < MB; ++x) {
        const int r = wn * NB2 + y, q = wk * MB + x;
        if (n0 + 32 * r + (lane & 31) < g.P && k0 + 32 * q < g.Q)
          store_part(parts + item.slot * (S::FN * S::FK), r * (S::FK / 32) + q, acc[x][y], lane);
      }
    return;
  }
  __syncthreads();
  char* const stage_out = ring + wave * 32 * S::PITCH;
  const int64_t nw = n0 + wn * NB2 * 32;
  if (g.c_type == MI355Q_F32) store_weight_rows<F32, MB, NB2, S::PITCH>(g, acc, stage_out, nw, kw, lane);
  else if (g.c_type == MI355Q_BF16) store_weight_rows<Bf16, MB, NB2, S::PITCH>(g, acc, stage_out, nw, kw, lane);
  else store_weight_rows<F16, MB, NB2, S::PITCH>(g, acc, stage_out, nw, kw, lane);
}

// Sums the partial slots of the split tiles in the splits' order, adds the bias and
// rounds once.  A workgroup takes a 32 x 32 tile, a thread four columns with four
// splits' loads in flight (eight: no faster), and turns it through LDS to store it row by row.
// 333 x 4096 in 5 parts 7.5 us.
template <int TR, int TC>
__global__ __launch_bounds__(256) void sum_splits_kernel(ProductArgs g, TileOrder o, const float* parts) {
  constexpr uint32_t PER = TR * TC / 1024, PITCH = 36;
  __shared__ __attribute__((aligned(16))) float turn[32 * PITCH];
  const uint32_t rest = o.row_tiles * o.col_tiles - o.full, tile = blockIdx.x / PER, in_tile = blockIdx.x - tile * PER;
  const uint32_t t = o.full + tile, gr = t / (8 * o.col_tiles), left = o.row_tiles - 8 * gr;
  const uint32_t rows = left < 8 ? left : 8, in = t - gr * 8 * o.col_tiles, tc = in / rows;
  const int64_t r0 = (int64_t)(8 * gr + in - tc * rows) * TR + in_tile / (TC / 32) * 32;
  const int64_t q0 = (int64_t)tc * TC + in_tile % (TC / 32) * 32;
  if (r0 >= g.P || q0 >= g.Q) return;   // (the whole workgroup)
  const float* p = parts + (int64_t)tile * (TR * TC) + in_tile * 1024 + 4 * threadIdx.x;
  const int64_t step = (int64_t)rest * (TR * TC);
  const int lane = threadIdx.x & 63;
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  if (r0 + (lane & 31) < g.P) {
    uint32_t s = 0;
    for (; s + 4 <= o.splits; s += 4) {
      f32x4_t x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = *reinterpret_cast<const f32x4_t*>(p + (s + u) * step);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += x[u][e];
    }
    for (; s < o.splits; ++s) {
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(p + s * step);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += x[e];
    }
  }
  *reinterpret_cast<f32x4_t*>(turn + (lane & 31) * PITCH + 8 * (threadIdx.x >> 6) + 4 * (lane >> 5)) = v;
  __syncthreads();
  v = *reinterpret_cast<const f32x4_t*>(turn + (threadIdx.x >> 3) * PITCH + 4 * (threadIdx.x & 7));
  const int64_t r = r0 + (threadIdx.x >> 3), q = q0 + 4 * (threadIdx.x & 7);
  if (r >= g.P || q >= g.Q) return;
  const bool whole = q + 4 <= g.Q;
  if (g.bias)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (q + e < g.Q) v[e] += load_typed(g.bias, g.bias_type, q + e);
  const int64_t c = r * g.ldc + q;
  if (g.c_type == MI355Q_F32) {
    float* d = static_cast<float*>(g.c) + c;
    if (whole) {
      __builtin_memcpy(d, &v, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (q + e < g.Q) d[e] = v[e];
    }
    return;
  }
  uint16_t h[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = g.c_type == MI355Q_BF16 ? Bf16::store(v[e]) : F16::store(v[e]);
  uint16_t* d = static_cast<uint16_t*>(g.c) + c;
  if (whole) {
    __builtin_memcpy(d, h, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (q + e < g.Q) d[e] = h[e];
  }
}

// ---------------------------------------------------------------- forward, few tokens
// Up to 16 TF tokens: the weight is read once, straight into the MFMA's
// registers (lane l: row l & 15, 16 bytes each at 16 (l / 16) of
// both halves of the step's 128, so that a load takes 64 bytes of 16 rows), the
// tokens come from L2, and the W waves of a workgroup take every W-th step of 16 AF
// features; their sums are joined in LDS.  What it has to move is the weight, so what
// counts is loads in flight: U steps are requested before the first is used.  It is not
// at HBM's rate: 1 x 14336 x 4096 takes 18 us (58.7 MB, 3.2 of 6.6 TB/s; 16 where the last-level
// cache holds the weight).  A wave requests as many chunks of the tokens as of the
// weight, and none while a batch of U steps is used.  (Eight steps or nontemporal loads: no faster.)
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

template <int TF, int AF, int W, int U, bool E8M0, bool ALIGNED>
__global__ __launch_bounds__(64 * W) void fp8_few_kernel(ProductArgs g) {
  __shared__ f32x4_t sums[W][AF][TF][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t f0 = (int64_t)blockIdx.x * 16 * AF;
  const int nkb = (int)((g.R + kGroup - 1) / kGroup);
  const int koff = 16 * (lane >> 4);
  const uint8_t* wp[AF];
  const uint8_t* xp[TF];
  int64_t xsi[TF];
#pragma unroll
  for (int a = 0; a < AF; ++a) {
    const int64_t f = f0 + 16 * a + (lane & 15);
    wp[a] = g.b + (f < g.Q ? f : g.Q - 1) * g.ldb + koff;
  }
#pragma unroll
  for (int b = 0; b < TF; ++b) {
    const int64_t t = 16 * b + (lane & 15), tt = t < g.P ? t : g.P - 1;
    xp[b] = static_cast<const uint8_t*>(g.a) + tt * g.lda + koff;
    xsi[b] = tt * g.ldas;
  }
  const float* const wsc = g.bs + f0 / kGroup * g.ldbs;   // 16 AF divides 128
  f32x4_t acc[AF][TF];
#pragma unroll
  for (int a = 0; a < AF; ++a)
#pragma unroll
    for (int b = 0; b < TF; ++b) acc[a][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  // 16 codes from column k, zeros past the last one: rows that are a multiple of 16
  // wide and aligned have a chunk inside or outside as a whole
  auto load16 = [&](const uint8_t* p, int64_t k) __attribute__((always_inline)) {
    i32x4_t v = {0, 0, 0, 0};
    const int64_t left = g.R - k - koff;
    if constexpr (ALIGNED) {
      if (left > 0) v = *reinterpret_cast<const i32x4_t*>(p + k);
    } else if (left >= 16) {
      __builtin_memcpy(&v, p + k, 16);
    } else {
      uint8_t b[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) b[e] = e < left ? p[k + e] : 0;
      __builtin_memcpy(&v, b, 16);
    }
    return v;
  };
  auto load32 = [&](const uint8_t* p, int64_t k) __attribute__((always_inline)) {
    return __builtin_shufflevector(load16(p, k), load16(p, k + 64), 0, 1, 2, 3, 4, 5, 6, 7);
  };
  for (int s0 = wave; s0 < nkb; s0 += W * U) {
    i32x8_t wa[U][AF], xb[U][TF];
    float sx[U][TF], sw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * W, sc = s < nkb ? s : nkb - 1;
      const int64_t k = (int64_t)s * kGroup;     // steps past the end load zeros
#pragma unroll
      for (int a = 0; a < AF; ++a) wa[u][a] = load32(wp[a], k);
#pragma unroll
      for (int b = 0; b < TF; ++b) {
        xb[u][b] = load32(xp[b], k);
        sx[u][b] = load_scale(g.as, E8M0 ? MI355Q_SCALE_E8M0 : MI355Q_SCALE_F32, xsi[b] + sc);
      }
      sw[u] = wsc[sc];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * W >= nkb) break;
#pragma unroll
      for (int b = 0; b < TF; ++b) {
        const float s = sx[u][b] * sw[u];
#pragma unroll
        for (int a = 0; a < AF; ++a) {
          f32x4_t t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                codes_bf16(wa[u][a][2 * i], wa[u][a][2 * i + 1]), codes_bf16(xb[u][b][2 * i], xb[u][b][2 * i + 1]), t,
                0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[a][b][e] = fmaf(t[e], s, acc[a][b][e]);
        }
      }
    }
  }
#pragma unroll
  for (int a = 0; a < AF; ++a)
#pragma unroll
    for (int b = 0; b < TF; ++b) sums[wave][a][b][lane] = acc[a][b];
  __syncthreads();
  // wave w finishes tiles w, w + W, ...
  for (int i = wave; i < AF * TF; i += W) {
    const int a = i / TF, b = i % TF;
    f32x4_t v = sums[0][a][b][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += sums[w][a][b][lane];
    const int64_t t = 16 * b + (lane & 15), f = f0 + 16 * a + 4 * (lane >> 4);
    if (t < g.P) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (f + e >= g.Q) continue;
        const float r = v[e] + (g.bias ? load_typed(g.bias, g.bias_type, f + e) : 0.f);
        const int64_t o = t * g.ldc + f + e;
        if (g.c_type == MI355Q_F32) static_cast<float*>(g.c)[o] = r;
        else static_cast<uint16_t*>(g.c)[o] = g.c_type == MI355Q_BF16 ? Bf16::store(r) : F16::store(r);
      }
    }
  }
}

// How a product is cut: a tile shape, the tiles that run whole, and parts of the
// sum for the others.
struct Plan {
  int shape;
  uint32_t tile_rows, tile_cols;
  uint32_t row_tiles, col_tiles, full, splits;
  int steps;          // of the sum, per split
};
// What a shape costs, in us: a step of one workgroup that has its CU to itself,
// a step of two that share one (0: only one fits), and what begins and ends a
// workgroup.
struct ShapeCost {
  int tile_rows, tile_cols;
  double one, two, ends;
};
// The cheapest cut by these costs: every shape, whole tiles for as many rounds of
// the 256 CUs as come out even (or none, for fewer), and 1 .. 16 parts of at least
// `least` steps for the rest.  Parts cost a second launch and a workspace (4 us on
// the device, 5 on the host, which is what small calls wait for) and their partial
// sums' way to it (written and read: 5 TB/s).
static Plan make_plan(const ShapeCost* shapes, int n, int64_t rows, int64_t cols, int64_t steps, int64_t least) {
  Plan best{};
  double best_cost = 0;
  for (int i = 0; i < n; ++i) {
    const ShapeCost& c = shapes[i];
    const int64_t tr = (rows + c.tile_rows - 1) / c.tile_rows, tc = (cols + c.tile_cols - 1) / c.tile_cols;
    const int64_t tiles = tr * tc, even = tiles - tiles % 256;
    for (int f = 0; f < (even > 0 ? 2 : 1); ++f) {
      const int64_t full = f ? even : 0, rest = tiles - full;
      if (full == 0 && tiles > 1024) continue;           // (partial sums of all tiles: never the cheapest)
      for (int64_t want = 1; want <= 16; ++want) {
        if (want > 1 && (rest == 0 || steps / want < least)) break;
        const int64_t per = (steps + want - 1) / want, k = (steps + per - 1) / per;
        const int64_t wgs = rest * k, whole = full / 256, parts = (wgs + 255) / 256;
        double t = (whole + parts) * c.ends;
        if (c.two > 0) {
          // rounds run in pairs; a whole one left over shares its CU with the
          // parts while they last, a part left over has it to itself
          t -= (whole + parts) / 2 * c.ends;
          t += whole / 2 * steps * c.two;
          int64_t left = parts * per, alone = parts % 2 * per;
          if (whole % 2) {
            const int64_t both = left < steps ? left : steps;
            t += both * c.two + (steps - both) * c.one;
            left -= both;
            alone = 0;
          }
          t += (left - alone) * c.two / 2 + alone * c.one;
        } else {
          t += (whole * steps + parts * per) * c.one;
        }
        if (k > 1) t += 7 + (double)wgs * c.tile_rows * c.tile_cols * 8 / 5e6;
        if (best.tile_rows == 0 || t < best_cost) {
          best_cost = t;
          best = Plan{i, (uint32_t)c.tile_rows, (uint32_t)c.tile_cols, (uint32_t)tr, (uint32_t)tc,
                      (uint32_t)(k > 1 ? full : tiles), (uint32_t)(k > 1 ? k : 1), (int)per};
        }
      }
    }
  }
  return best;
}
// Forward and input gradient: `rows` tokens by `cols` columns, `sum` terms in
// blocks of 128.  Measured, forward: 1024 x 4096 x 4096 in 256 tiles of 128 x 128 39 us,
// in 512 of 64 x 128 41; 100 x 4096 x 4096 in 32 tiles of 128 x 128 34 us, 64 of 64 x 128 27,
// these in 2 / 4 / 8 parts 19 / 20 / 20; 333 x 4096 x 14336 in 96 tiles of 128 x 128 116 us,
// in 2 / 5 / 8 parts 69 / 58 / 63, in 192 of 64 x 128 in 1 / 4 parts 101 / 71.
static Plan plan_forward(int64_t rows, int64_t cols, int64_t sum) {
  static const ShapeCost shapes[] = {{64, 128, 0.75, 1.1, 4}, {128, 128, 1.0, 1.75, 4}};
  return make_plan(shapes, 2, rows, cols, group_count(sum), 4);
}
// Input gradient: 1024 x 4096 x 4096 45 us in 256 tiles of 128 x 128, 41 in 512 of 64 x 128;
// 16 x 4096 x 4096 39 us and 31, these in 2 / 4 / 8 / 16 parts 20 / 14 / 14 / 14;
// 450 x 12544 x 7936 139 us in 248 tiles of 128 x 128, 114 in two parts each.
static Plan plan_grad_input(int64_t rows, int64_t cols, int64_t sum) {
  static const ShapeCost shapes[] = {{64, 128, 1.0, 1.25, 4}, {128, 128, 1.3, 2.0, 4}};
  return make_plan(shapes, 2, rows, cols, group_count(sum), 2);
}
// Weight gradient, in stages of 32 tokens: 8192 x 1024 x 4096 in 256 tiles of 128 x 128 98 us, in
// 64 of 256 x 256 in 1 / 2 / 4 / 8 parts 162 / 98 / 77 / 98; 517 x 768 x 2048 in 96 of 128 x 128
// 12 us, in 24 of 256 x 256 20; 1024 x 4096 x 4096 in 256 of 256 x 256 37 us, 1024 of 128 x 128 49.
static Plan plan_weight(int64_t rows, int64_t out, int64_t cols) {
  static const ShapeCost shapes[] = {{128, 128, 0.37, 0.65, 5}, {256, 256, 0.88, 0, 8}};
  return make_plan(shapes, 2, out, cols, (rows + 31) / 32, 4);
}
static size_t plan_bytes(const Plan& p) {
  if (p.splits <= 1) return 0;
  return sizeof(float) * p.tile_rows * p.tile_cols * ((size_t)p.row_tiles * p.col_tiles - p.full) * p.splits;
}
// the splits' partial slots, or null and an unsplit plan without room for them
static float* plan_workspace(Plan& p, void* ws, size_t bytes) {
  if (p.splits <= 1) return nullptr;
  if (ws && bytes >= plan_bytes(p) && aligned16(ws)) return static_cast<float*>(ws);
  p.splits = 1;
  p.full = p.row_tiles * p.col_tiles;
  return nullptr;
}

template <int KIND>
static int launch_any(ProductArgs g, mi355q_dtype out, hipStream_t st, const char* who) {
  const int64_t tp = (g.P + GT - 1) / GT, tq = (g.Q + GT - 1) / GT;
  MQ_CHECK_ARG(tp * tq < (int64_t(1) << 31), "%s: output too large", who);
  g.q_tiles = (uint32_t)tq;
  const dim3 grid((unsigned)(tp * tq));
  if constexpr (KIND == kGradInput) {   // (bf16 outputs only)
    hipLaunchKernelGGL((product_any_kernel<KIND, Bf16>), grid, dim3(256), 0, st, g);
  } else {
    with_dtype(out, [&](auto t) {
      using T = decltype(t);
      hipLaunchKernelGGL((product_any_kernel<KIND, T>), grid, dim3(256), 0, st, g);
    });
  }
  MQ_LAUNCH_CHECK();
  return MI355Q_OK;
}

// Up to here the weight's bytes decide (24 x 4096 x 4096 12 us against 13 in split tiles, which are two launches,
// 24 x 14336 x 4096 23 against 21); beyond, 48 tokens took 15 .. 17 us against 14, and 35 .. 47 against 23.
constexpr int64_t kFewTokens = 32;

template <int TF, int AF, int W, int U>
static void launch_few_shape(const ProductArgs& g, bool e8, bool aligned, hipStream_t st) {
  const dim3 grid((unsigned)((g.Q + 16 * AF - 1) / (16 * AF))), block(64 * W);
  if (aligned) {
    if (e8) hipLaunchKernelGGL((fp8_few_kernel<TF, AF, W, U, true, true>), grid, block, 0, st, g);
    else    hipLaunchKernelGGL((fp8_few_kernel<TF, AF, W, U, false, true>), grid, block, 0, st, g);
  } else {
    if (e8) hipLaunchKernelGGL((fp8_few_kernel<TF, AF, W, U, true, false>), grid, block, 0, st, g);
    else    hipLaunchKernelGGL((fp8_few_kernel<TF, AF, W, U, false, false>), grid, block, 0, st, g);
  }
}
static void launch_few(const ProductArgs& g, bool e8, bool aligned, hipStream_t st) {
  // Four waves / eight, weights from HBM: one token, 4096 x 14336 16.8 / 14.0 us, 4096 x 8192 12.6 / 9.6, 14336 x 4096
  // 18.2 / 16.1; 16 tokens 21.0 / 20.8, 14.4 / 13.9, 23.5 / 23.5, 28672 x 4096 38.2 / 42.9.  (One token would gain from
  // eight on narrower rows too.)
  if (g.P <= 16 && g.R > 8192) launch_few_shape<1, 1, 8, 4>(g, e8, aligned, st);
  else if (g.P <= 16) launch_few_shape<1, 1, 4, 4>(g, e8, aligned, st);
  else launch_few_shape<2, 2, 8, 1>(g, e8, aligned, st);
}

// Runs `kernel(grid, order)` over the plan's items and adds up its splits.
template <int TR, int TC, class Kernel>
static int launch_tiles(const ProductArgs& g, const Plan& p, float* parts, hipStream_t st, const char* who,
                        Kernel&& kernel) {
  const int64_t tiles = (int64_t)p.row_tiles * p.col_tiles, rest = tiles - p.full, items = p.full + rest * p.splits;
  MQ_CHECK_ARG(tiles < (int64_t(1) << 28) && items < (int64_t(1) << 31), "%s: output too large", who);
  const TileOrder o{p.row_tiles, p.col_tiles, p.full, p.splits};
  kernel(dim3((unsigned)items), o);
  MQ_LAUNCH_CHECK();
  if (parts) {
    hipLaunchKernelGGL((sum_splits_kernel<TR, TC>), dim3((unsigned)(rest * (TR * TC / 1024))), dim3(256), 0, st, g, o,
                       parts);
    MQ_LAUNCH_CHECK();
  }
  return MI355Q_OK;
}

template <int T, int A, int WT, int WF>
static int launch_forward(const ProductArgs& g, bool e8, const Plan& p, float* parts, hipStream_t st) {
  using S = FwdShape<T, A, WT, WF>;
  return launch_tiles<S::TT, S::FT>(g, p, parts, st, "fp8_block_matmul", [&](dim3 grid, TileOrder o) {
    if (e8) hipLaunchKernelGGL((fp8_forward_kernel<T, A, WT, WF, true>), grid, dim3(S::NTH), 0, st, g, o, p.steps, parts);
    else    hipLaunchKernelGGL((fp8_forward_kernel<T, A, WT, WF, false>), grid, dim3(S::NTH), 0, st, g, o, p.steps, parts);
  });
}
template <int T, int WT>
static int launch_grad_input(const ProductArgs& g, const Plan& p, float* parts, hipStream_t st) {
  using S = GradInputShape<T, WT>;
  return launch_tiles<S::TT, S::FT>(g, p, parts, st, "fp8_block_grad_input", [&](dim3 grid, TileOrder o) {
    hipLaunchKernelGGL((fp8_grad_input_kernel<T, WT>), grid, dim3(S::NTH), 0, st, g, o, p.steps, parts);
  });
}
template <int MB, int NB2, int WK, int WN>
static int launch_grad_weight(const ProductArgs& g, const Plan& p, float* parts, hipStream_t st) {
  using S = GradWeightShape<MB, NB2, WK, WN>;
  return launch_tiles<S::FN, S::FK>(g, p, parts, st, "fp8_block_grad_weight", [&](dim3 grid, TileOrder o) {
    hipLaunchKernelGGL((fp8_grad_weight_kernel<MB, NB2, WK, WN>), grid, dim3(S::NTH), 0, st, g, o, p.steps, parts);
  });
}

// ---------------------------------------------------------------- rows of odd widths
// The tile kernels take operands in 16-byte chunks.  Rows whose width is no whole
// number of them are first copied to rows that are, ending in zeros: a read and a
// write of both operands, of which the product reads each many times.
// One launch for both operands: the first `blocks` workgroups take the first.
struct PadJob {
  const uint8_t* src;
  int64_t pitch, row_bytes;
  uint8_t* dst;
  uint32_t chunks;
  FastDiv per_row;
};
__global__ __launch_bounds__(256) void pad_rows_kernel(PadJob first, PadJob second, uint32_t blocks) {
  const PadJob& job = blockIdx.x < blocks ? first : second;
  const uint32_t i = (blockIdx.x < blocks ? blockIdx.x : blockIdx.x - blocks) * 256 + threadIdx.x;
  if (i >= job.chunks) return;
  const uint32_t r = div(i, job.per_row);
  const int64_t at = (int64_t)(i - r * job.per_row.d) * 16, left = job.row_bytes - at;
  const uint8_t* p = job.src + r * job.pitch + at;
  u32x4_t v;
  if (left >= 16) {
    __builtin_memcpy(&v, p, 16);
  } else {
    uint8_t b[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) b[e] = e < left ? p[e] : 0;
    __builtin_memcpy(&v, b, 16);
  }
  *reinterpret_cast<u32x4_t*>(job.dst + (int64_t)i * 16) = v;
}
static int64_t padded(int64_t row_bytes) { return (row_bytes + 15) / 16 * 16; }
static size_t padded_bytes(int64_t rows, int64_t row_bytes) { return (size_t)rows * padded(row_bytes); }

// Copies to be made before a product: two of them, of 2^30 chunks at the most, in one launch.
struct Padding {
  PadJob jobs[2] = {};
  int n = 0;
  const hipStream_t st;
  explicit Padding(hipStream_t stream) : st(stream) {}
  static uint32_t blocks(const PadJob& j) { return (j.chunks + 255) / 256; }
  int flush() {
    if (n == 0) return MI355Q_OK;
    hipLaunchKernelGGL(pad_rows_kernel, dim3(blocks(jobs[0]) + (n > 1 ? blocks(jobs[1]) : 0)), dim3(256), 0, st, jobs[0],
                       jobs[1], blocks(jobs[0]));
    n = 0;
    MQ_LAUNCH_CHECK();
    return MI355Q_OK;
  }
  int add(const void* src, int64_t pitch, int64_t rows, int64_t row_bytes, void* dst) {
    const int64_t per = padded(row_bytes) / 16, most = (int64_t(1) << 30) / per;
    for (int64_t r = 0; r < rows; r += most) {
      if (n == 2)
        if (const int rc = flush()) return rc;
      const int64_t m = rows - r < most ? rows - r : most;
      jobs[n++] = PadJob{static_cast<const uint8_t*>(src) + r * pitch, pitch, row_bytes,
                         static_cast<uint8_t*>(dst) + r * per * 16, (uint32_t)(m * per), fast_div((uint32_t)per)};
    }
    return MI355Q_OK;
  }
};

// Odd widths and a sum of one step: the element loads of one launch cost less than a
// launch for copies of both operands while every workgroup has a CU to itself
// (2102 x 80 x 69 9 us against 12, 1000 x 1000 x 69 in 256 workgroups 9 against 12; input
// gradient of 2000 x 99 x 1000 in 512 16 against 10; with three steps 300 x 513 x 515 44 against 14).
static bool short_sum(int64_t rows, int64_t cols, int64_t sum) {
  return sum <= kGroup && ((rows + GT - 1) / GT) * ((cols + GT - 1) / GT) <= 256;
}
// row offsets within a tile and a stage in 32 bits
static bool small_pitch(int64_t ld) { return ld < (int64_t(1) << 22); }

}  // namespace mi355q

using namespace mi355q;

extern "C" size_t mi355q_fp8_block_matmul_workspace_size(int64_t rows, int64_t out, int64_t cols) {
  if (rows <= kFewTokens || out <= 0 || cols <= 0) return 0;
  return plan_bytes(plan_forward(rows, out, cols)) +
         (cols % 16 ? padded_bytes(rows, cols) + padded_bytes(out, cols) : 0);
}

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
  g.c_type = y_dtype;
  g.ldc = ldy;
  g.P = rows;
  g.Q = out;
  g.R = cols;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool e8 = x_scale_type == MI355Q_SCALE_E8M0;
  const bool aligned = cols % 16 == 0 && ldx % 16 == 0 && ldw % 16 == 0 && aligned16(x_dev) && aligned16(w_dev);
  if (rows <= kFewTokens) {
    launch_few(g, e8, aligned, st);
    MQ_LAUNCH_CHECK();
    return MI355Q_OK;
  }
  Plan p = plan_forward(rows, out, cols);
  float* const parts = plan_workspace(p, workspace_dev, workspace_bytes);
  if (!small_pitch(ld_x_scales)) return launch_any<kForward>(g, y_dtype, st, "fp8_block_matmul");
  if (!aligned || !small_pitch(ldx) || !small_pitch(ldw)) {
    const size_t base = plan_bytes(p), need = base + padded_bytes(rows, cols) + padded_bytes(out, cols);
    if (!workspace_dev || !aligned16(workspace_dev) || workspace_bytes < need || !small_pitch(cols) ||
        short_sum(rows, out, cols))
      return launch_any<kForward>(g, y_dtype, st, "fp8_block_matmul");
    char* const xc = static_cast<char*>(workspace_dev) + base;
    char* const wc = xc + padded_bytes(rows, cols);
    Padding pad(st);
    if (const int rc = pad.add(x_dev, ldx, rows, cols, xc)) return rc;
    if (const int rc = pad.add(w_dev, ldw, out, cols, wc)) return rc;
    if (const int rc = pad.flush()) return rc;
    g.a = xc;
    g.b = reinterpret_cast<const uint8_t*>(wc);
    g.lda = g.ldb = g.R = padded(cols);
  }
  return p.shape ? launch_forward<2, 2, 2, 2>(g, e8, p, parts, st) : launch_forward<1, 2, 2, 2>(g, e8, p, parts, st);
}

extern "C" size_t mi355q_fp8_block_grad_input_workspace_size(int64_t rows, int64_t out, int64_t cols) {
  if (rows <= 0 || out <= 0 || cols <= 0) return 0;
  return plan_bytes(plan_grad_input(rows, cols, out)) + (out % 8 ? padded_bytes(rows, 2 * out) : 0) +
         (cols % 16 ? padded_bytes(out, cols) : 0);
}

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
  g.c_type = MI355Q_BF16;
  g.ldc = lddx;
  g.P = rows;
  g.Q = cols;
  g.R = out;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool y_ok = out % 8 == 0 && lddy % 8 == 0 && aligned16(dy_dev) && small_pitch(lddy);
  const bool w_ok = cols % 16 == 0 && ldw % 16 == 0 && aligned16(w_dev) && small_pitch(ldw);
  Plan p = plan_grad_input(rows, cols, out);
  float* const parts = plan_workspace(p, workspace_dev, workspace_bytes);
  if (!y_ok || !w_ok) {
    const size_t base = plan_bytes(p), y_bytes = y_ok ? 0 : padded_bytes(rows, 2 * out);
    const size_t need = base + y_bytes + (w_ok ? 0 : padded_bytes(out, cols));
    if (!workspace_dev || !aligned16(workspace_dev) || workspace_bytes < need || !small_pitch(cols) ||
        !small_pitch(out) || short_sum(rows, cols, out))
      return launch_any<kGradInput>(g, MI355Q_BF16, st, "fp8_block_grad_input");
    char* const yc = static_cast<char*>(workspace_dev) + base;
    Padding pad(st);
    if (!y_ok) {
      if (const int rc = pad.add(dy_dev, 2 * lddy, rows, 2 * out, yc)) return rc;
      g.a = yc;
      g.lda = padded(2 * out) / 2;
    }
    if (!w_ok) {
      if (const int rc = pad.add(w_dev, ldw, out, cols, yc + y_bytes)) return rc;
      g.b = reinterpret_cast<const uint8_t*>(yc + y_bytes);
      g.ldb = padded(cols);
    }
    if (const int rc = pad.flush()) return rc;
  }
  return p.shape ? launch_grad_input<2, 2>(g, p, parts, st) : launch_grad_input<1, 2>(g, p, parts, st);
}

extern "C" size_t mi355q_fp8_block_grad_weight_workspace_size(int64_t rows, int64_t out, int64_t cols) {
  if (rows <= 0 || out <= 0 || cols <= 0) return 0;
  return plan_bytes(plan_weight(rows, out, cols)) + (out % 8 ? padded_bytes(rows, 2 * out) : 0) +
         (cols % 16 ? padded_bytes(rows, cols) : 0);
}

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
  g.c_type = dw_dtype;
  g.ldc = lddw;
  g.P = out;
  g.Q = cols;
  g.R = rows;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (rows == 0) return launch_any<kGradWeight>(g, dw_dtype, st, "fp8_block_grad_weight");   // zeros
  const bool y_ok = out % 8 == 0 && lddy % 8 == 0 && aligned16(dy_dev) && small_pitch(lddy);
  const bool x_ok = cols % 16 == 0 && ldx % 16 == 0 && aligned16(x_dev) && small_pitch(ldx);
  Plan p = plan_weight(rows, out, cols);
  float* const parts = plan_workspace(p, workspace_dev, workspace_bytes);
  if (!small_pitch(ld_x_scales)) return launch_any<kGradWeight>(g, dw_dtype, st, "fp8_block_grad_weight");
  if (!y_ok || !x_ok) {
    const size_t base = plan_bytes(p), y_bytes = y_ok ? 0 : padded_bytes(rows, 2 * out);
    const size_t need = base + y_bytes + (x_ok ? 0 : padded_bytes(rows, cols));
    if (!workspace_dev || !aligned16(workspace_dev) || workspace_bytes < need || !small_pitch(cols) ||
        !small_pitch(out) || short_sum(out, cols, rows))
      return launch_any<kGradWeight>(g, dw_dtype, st, "fp8_block_grad_weight");
    char* const yc = static_cast<char*>(workspace_dev) + base;
    Padding pad(st);
    if (!y_ok) {
      if (const int rc = pad.add(dy_dev, 2 * lddy, rows, 2 * out, yc)) return rc;
      g.a = yc;
      g.lda = padded(2 * out) / 2;
    }
    if (!x_ok) {
      if (const int rc = pad.add(x_dev, ldx, rows, cols, yc + y_bytes)) return rc;
      g.b = reinterpret_cast<const uint8_t*>(yc + y_bytes);
      g.ldb = padded(cols);
    }
    if (const int rc = pad.flush()) return rc;
  }
  return p.shape ? launch_grad_weight<4, 2, 2, 4>(g, p, parts, st) : launch_grad_weight<2, 2, 2, 2>(g, p, parts, st);
}
