// Products of 16-bit activations with 4-bit weights (w4a16.h) for many rows: tiles on
// the matrix instructions.
//
// A workgroup of four waves makes 32 MTW rows by 128 NTW columns of w, each wave all of
// the rows and 32 NTW of the columns, in steps of 128 of the sum.  A step's rows of x go
// global -> LDS by the LDS-DMA load, in 16-byte chunks placed so that an operand read
// takes 16 different bank groups, and are read by all four waves; a weight's codes belong to one
// wave, go through its part of LDS the same way (a load into registers would have the compiler wait for the DMA
// requested before it), and are converted once per step.  Both are requested a step ahead.
//
// Per 32 x 32 tile and group the MFMAs start from zero and acc += s * tile follows in fp32; in tiles of up to 64
// rows two sets of sums take turns, one scaled while the other is made.  The conversions give codes 0 .. 15 (a
// signed one would cost more than it saves), and the zero points' part of the sum,
//   - sum_g s[n][g] z[n][g] sum_{k in g} x[m][k],
// is a product of its own with one column per group: a first pass (w4_prepare_kernel)
// leaves the groups' sums of x as three bf16 numbers each (24 bits) and the factors -s z as one, two or three, as many
// as s z has bits for, and the accumulators begin with the products that count down to 2^-24: three of 1/128
// of the sum's length where one piece holds a factor.  The same pass lays the scales out in fp32 by group, so that
// a tile's 32 are neighbours, and costs 10 to 20 us.
//
// What bounds it (bf16, groups of 128): 8192 x 28672 x 4096, gated, takes 1.67 to 1.76 ms, 1.13 PFLOP/s, the MFMAs 56 %
// and the vector unit 45 % busy at 1.9 GHz.  The two take turns more than they overlap: in the tiles of 128 rows most
// operands of x are read right before their MFMAs, and nothing is multiplied while a tile's sums are scaled.  Those of
// int4, and of MXFP4 with fp16, do not fit the registers either (7 of the 40 kernels, 40 to 108 bytes a lane in
// scratch); in groups of 32 and for fp16 the loop reads offsets back between the requests of a step and waits for what
// is under way: groups of 128, 64 and 32 take 1.75, 1.96 and 2.45 ms, MXFP4 1.55 with bf16 and 2.14 with fp16.  4096
// tokens to 8 of 128 experts of 1536 x 2048 take 0.28 to 0.32 ms: the tiles are 64 rows, so codes are converted twice
// as often (MFMAs 40 % busy), and an eighth of their rows is empty.
#pragma once

#include <type_traits>

#include "w4a16.h"

namespace mi355q {

constexpr int kSlices = kStep / 16;   // MFMAs per step and tile
constexpr int kWaves = 4;

typedef __attribute__((address_space(3))) void lds_void_t;
__device__ __forceinline__ uint32_t lds_u32(const void* p) {
  return (uint32_t) reinterpret_cast<uintptr_t>((lds_void_t*)p);
}
// 64 lanes x 16 bytes to LDS at m0, from a scalar base and lane offsets; waited for explicitly (vmcnt).  The load reads
// m0 one state after it is written, at the earliest.
__device__ __forceinline__ void dma16(uint32_t off, const void* base, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(m0) : "memory", "m0");
}

template <class T>
__device__ __forceinline__ f32x16_t mfma32(const u32x4_t& a, const u32x4_t& b, const f32x16_t& c) {
  if constexpr (T::code == MI355Q_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
}

// v as three bf16 numbers: v - (p0 + p1 + p2) is below 2^-26 of it
__device__ __forceinline__ void split3(float v, uint16_t (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    p[i] = f32_to_bf16_bits(v);
    v -= bf16_bits_to_f32(p[i]);
  }
}

// ---------------------------------------------------------------- sums of x
// sums[m][piece][g]: the sum of x[m] over group g as three bf16 numbers, zeros behind
// the last group; copy: x with rows of whole steps, zeros behind the last column.
// 2^lanes lanes share a group, and a wave holds 64 >> lanes of them.
template <class T>
__device__ __forceinline__ void w4_sums(const W4Args& g, uint32_t padded, int lanes, uint32_t block, uint16_t* sums,
                                        uint16_t* copy, int64_t ld_copy) {
  const int64_t cols = g.cols;
  const int lane = threadIdx.x & 63, sub = lane & ((1 << lanes) - 1);
  const uint32_t per = 64u >> lanes, parts = (padded + per - 1) / per;
  const uint64_t item = (uint64_t)block * 4 + (threadIdx.x >> 6);
  const int64_t m = (int64_t)(item / parts);
  if (m >= g.n_x) return;
  const uint32_t gi = (uint32_t)(item % parts) * per + (lane >> lanes);
  const uint16_t* const row = g.x + m * g.ldx;
  const int64_t k0 = (int64_t)gi * g.group, k1 = gi < g.groups ? (k0 + g.group < cols ? k0 + g.group : cols) : k0;
  float sum = 0.f;
  for (int64_t k = k0 + 8 * sub; k < k1; k += 8 << lanes) {
    uint16_t v[8];
    const int64_t left = cols - k;
    if (left >= 8) {
      __builtin_memcpy(v, row + k, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < left ? row[k + e] : 0;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < k1) sum += T::load(v[e]);
    if (copy) __builtin_memcpy(copy + m * ld_copy + k, v, 16);       // groups are whole chunks but for the last
  }
  for (int d = 1; d < 1 << lanes; d <<= 1) sum += __shfl_xor(sum, d);
  if (sums && sub == 0 && gi < padded) {
    uint16_t p[3];
    split3(sum, p);
#pragma unroll
    for (int i = 0; i < 3; ++i) sums[((size_t)m * 3 + i) * padded + gi] = p[i];
  }
  if (copy && gi == g.groups - 1)
    for (int64_t k = (cols + 7) / 8 * 8 + 8 * sub; k < ld_copy; k += 8 << lanes)
      *reinterpret_cast<u32x4_t*>(copy + m * ld_copy + k) = u32x4_t{0u, 0u, 0u, 0u};
}

// Of every expert's column n: factors[n][piece][g], -s z over group g as `pieces` bf16
// numbers, zeros behind the last group; and scales[expert][g][column], what the tiles
// multiply with (the operand of the conversion where the scale goes there), so that neighbouring
// lanes read neighbouring scales.  A thread takes one, 32 neighbouring columns to 8 groups.
template <int KIND, bool FOLD>
__device__ __forceinline__ void w4_factors(const W4Args& g, uint32_t padded, int pieces, uint32_t block, uint16_t* factors,
                                           uint32_t* scales) {
  const uint32_t cols = (uint32_t)((g.out + 31) / 32), in = block % (cols * (padded / 8));
  const int64_t e = block / (cols * (padded / 8));
  const int64_t c = (int64_t)(in % cols) * 32 + (threadIdx.x >> 3);
  const uint32_t gi = in / cols * 8 + (threadIdx.x & 7);
  __shared__ uint32_t turn[8][33];
  if (c < g.out) {
    float s = 0.f, v = 0.f;
    if (gi < g.groups) {
      if constexpr (KIND == kMxfp4) {
        const uint32_t b = static_cast<const uint8_t*>(g.s)[e * g.stride_s + c * g.lds + gi];
        s = FOLD ? __uint_as_float((b << 23) | 0x00400000u) : e8m0_to_f32(b);
      } else {
        s = load_any(g.s, g.s_type, e * g.stride_s + c * g.lds + gi);
        float z = 8.f;
        if constexpr (KIND == kInt4Zero)
          z = (float)((g.z[e * g.stride_z + c / 8 * g.ldz + gi] >> (4 * (int)(c % 8))) & 15u);
        v = -z * s;
      }
    }
    turn[threadIdx.x & 7][threadIdx.x >> 3] = __float_as_uint(s);
    if constexpr (KIND != kMxfp4) {
      uint16_t p[3];
      split3(v, p);
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (k < pieces) factors[((e * g.out + c) * pieces + k) * padded + gi] = p[k];
    }
  }
  __syncthreads();
  const int64_t n = (int64_t)(in % cols) * 32 + (threadIdx.x & 31);
  if (n < g.out)
    scales[(e * padded + in / cols * 8 + (threadIdx.x >> 5)) * g.out + n] = turn[threadIdx.x >> 5][threadIdx.x & 31];
}

// The weight with rows of whole 16-byte chunks, which the DMA can read.  A thread takes one.
__device__ __forceinline__ void w4_copy(const W4Args& g, uint64_t i, int64_t bytes, uint8_t* copy) {
  const uint64_t chunks = (uint64_t)(bytes + 15) / 16, n = i / chunks;
  const int64_t at = (int64_t)(i - n * chunks) * 16, e = (int64_t)(n / (uint64_t)g.out);
  if (e >= g.experts) return;
  const uint8_t* const p = g.w + e * g.stride_w + (int64_t)(n % (uint64_t)g.out) * g.ldw + at;
  u32x4_t v;
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = at + 4 * k < bytes ? reinterpret_cast<const uint32_t*>(p)[k] : 0u;
  *reinterpret_cast<u32x4_t*>(copy + i * 16) = v;
}

// What the tiles read beside x and the weight, in one launch: the first workgroups take x,
// the next the weight's factors, the others (if there are) its codes.
struct W4Prepare {
  uint32_t padded;         // groups, a multiple of 16
  int lanes;               // log2 of the lanes per group of x
  int pieces;              // of the factors
  uint32_t x_blocks, f_blocks;
  uint16_t *sums, *factors;
  uint32_t* scales;
  uint16_t* x_copy;        // or null
  int64_t ld_copy;
  uint8_t* w_copy;
  int64_t w_bytes;         // of a row
};
template <class T, int KIND>
__global__ __launch_bounds__(256) void w4_prepare_kernel(W4Args g, W4Prepare p) {
  if (blockIdx.x < p.x_blocks)
    w4_sums<T>(g, p.padded, p.lanes, blockIdx.x, p.sums, p.x_copy, p.ld_copy);
  else if (blockIdx.x - p.x_blocks < p.f_blocks)
    w4_factors<KIND, KIND == kMxfp4 && T::code == MI355Q_BF16>(g, p.padded, p.pieces, blockIdx.x - p.x_blocks, p.factors,
                                                                 p.scales);
  else
    w4_copy(g, (uint64_t)(blockIdx.x - p.x_blocks - p.f_blocks) * 256 + threadIdx.x, p.w_bytes, p.w_copy);
}

// ---------------------------------------------------------------- tiles
struct W4Tiles {
  const uint16_t* sums;      // [n_x][3][padded]; MXFP4: unused
  const uint16_t* factors;   // [experts][out][pieces][padded]
  const float* scales;       // [experts][padded][out]
  uint32_t padded;           // groups, a multiple of 16
  int pieces;                // of the factors s z that are not zero: 1, 2 or 3
  uint32_t row_tiles, col_tiles, splits;
  uint32_t band;             // row tiles, of experts
  float* parts;              // with splits: [splits][rows][out], the sums of each range of steps
};

template <int MTW>
struct TileShape {
  static constexpr int R = 32 * MTW;                 // rows of x
  static constexpr int SLOT = R * kStep * 2;         // bytes of a step
  static constexpr int NI = R / 16;                  // DMA instructions per wave and step
  static constexpr int W = 2 * SLOT;                 // where the waves' codes begin
};

template <class T, int KIND, int GPS, int MTW, int NTW>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2)))
void w4_tiles_kernel(W4Args g, W4Tiles o) {
  using S = TileShape<MTW>;
  constexpr int R = S::R;
  constexpr bool FOLD = KIND == kMxfp4 && T::code == MI355Q_BF16;
  constexpr int PER = kSlices / GPS;                 // MFMAs per group
  constexpr int WSTEP = NTW * 2048;                  // bytes of a wave's codes of a step
  __shared__ __attribute__((aligned(16))) char ring[S::W + kWaves * WSTEP];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 31, h = lane >> 5;

  // Workgroups of an XCD (every eighth) that follow each other share rows of x, and in bands of row tiles the
  // weight.  One weight: an XCD takes a run of tiles, in bands of 8.  Experts: the bands go round the XCDs, as the
  // last ones may be empty (how many row tiles there are is known on the device alone).
  // (divisions run on the vector unit: what follows from them is brought back to scalar registers by hand)
  uint32_t split = 0, tc, tr;
  if (g.offsets) {
    const uint32_t xcd = blockIdx.x % 8, l = blockIdx.x / 8, size = o.band * o.col_tiles;
    const uint32_t turn = __builtin_amdgcn_readfirstlane((int)(l / size)), in = l - turn * size;
    tc = __builtin_amdgcn_readfirstlane((int)(in / o.band));
    tr = (turn * 8 + xcd) * o.band + in - tc * o.band;
  } else {
    const uint32_t id = xcd_order(blockIdx.x, gridDim.x);
    split = __builtin_amdgcn_readfirstlane((int)(id / (o.row_tiles * o.col_tiles)));
    const uint32_t t = id - split * (o.row_tiles * o.col_tiles);
    const uint32_t band = __builtin_amdgcn_readfirstlane((int)(t / (8 * o.col_tiles)));
    const uint32_t left = o.row_tiles - 8 * band, in = t - band * 8 * o.col_tiles, high = left < 8 ? left : 8;
    tc = __builtin_amdgcn_readfirstlane((int)(in / high));
    tr = 8 * band + in - tc * high;
  }
  const RowTile tile = row_tile<R>(g, tr);
  if (tile.count <= 0) return;
  const int64_t half = g.gated ? g.out / 2 : 0, width = g.gated ? half : g.out;
  const int per_wave = g.gated ? 16 * NTW : 32 * NTW;                 // columns of y
  const int64_t n0 = ((int64_t)tc * kWaves + wave) * per_wave;
  // first column of tile a of the wave
  auto column = [&](int a) __attribute__((always_inline)) {
    return g.gated ? (a >= NTW / 2 ? half : 0) + n0 + 32 * (a % (NTW / 2 ? NTW / 2 : 1)) : n0 + 32 * a;
  };
  void* const y_dev = o.splits > 1 ? o.parts + (int64_t)split * g.n_rows * g.ldy : g.y;
  if (tile.expert < 0) {                                              // rows of no expert
    const int es = dtype_size((mi355q_dtype)g.y_type);
    for (int r = 0; r < tile.count; ++r) {
      char* const at = static_cast<char*>(y_dev) + ((tile.first + r) * g.ldy + n0) * es;
      for (int c = lane; c < per_wave && n0 + c < width; c += 64) {
        if (es == 4) reinterpret_cast<uint32_t*>(at)[c] = 0;
        else reinterpret_cast<uint16_t*>(at)[c] = 0;
      }
    }
    return;
  }
  // row of x behind row r of the tile, -1: a row that is not there
  auto x_row = [&](int r) __attribute__((always_inline)) {
    int64_t row = tile.first + r;
    if (g.rows && r < tile.count) row = g.rows[row];
    return r < tile.count && row >= 0 && row < g.n_x ? row : (int64_t)-1;
  };

  // DMA: instruction q of a step fills 16 rows' 64 bytes; lane l the place l & 3 of row l / 4, with the
  // row's chunk (l & 3) ^ (row / 4 & 3).  Rows that are not there read another row (their results are
  // not stored).
  const uint32_t all = (uint32_t)((g.cols + kStep - 1) / kStep);
  const int s_begin = __builtin_amdgcn_readfirstlane((int)(all * split / o.splits));
  const int steps = __builtin_amdgcn_readfirstlane((int)(all * (split + 1) / o.splits));
  const int64_t x0 = g.rows ? 0 : tile.first;
  constexpr int NR = S::NI > 4 ? S::NI / 4 : 1;       // rows per lane
  uint32_t xo[NR];
  const int chunk = (lane & 3) ^ ((lane >> 4) & 3);
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int64_t row = x_row(((wave * S::NI + 4 * i) >> 2) * 16 + (lane >> 2));
    xo[i] = (uint32_t)((row < 0 ? x0 : row) - x0) * (uint32_t)(2 * g.ldx) + 16 * chunk;
  }
  const char* const xb = reinterpret_cast<const char*>(g.x + x0 * g.ldx);
  const uint32_t l0 = lds_u32(ring);
  const int whole = (int)(g.cols / kStep) < steps ? (int)(g.cols / kStep) : steps;   // end of the steps of 128 columns
  const int tail = (int)(g.cols % kStep + 7) / 8;     // chunks of a shorter last one (rows that end inside one are copies)
  auto dma = [&](int s, int slot, auto full) __attribute__((always_inline)) {
    const char* const base = xb + (int64_t)s * (2 * kStep);
    const uint32_t m0 = l0 + slot * S::SLOT;
    auto place = [&](int i) __attribute__((always_inline)) {
      const int q = wave * S::NI + i;
      return m0 + (q & 3) * (R * 64) + (q >> 2) * 1024;
    };
    if (decltype(full)::value || s < whole) {
#pragma unroll
      for (int i = 0; i < S::NI; ++i) dma16(xo[i / 4], base + 64 * ((wave * S::NI + i) & 3), place(i));
    } else {
      // chunks past the last column: the row's first one of the step, which meets zeros (offsets are
      // unsigned: the 64 columns of a chunk's quarter are added to them, so that taking the chunk off stays
      // above the base)
#pragma unroll
      for (int i = 0; i < S::NI; ++i) {
        const int hi = (wave * S::NI + i) & 3;
        dma16(xo[i / 4] + (4 * hi + chunk < tail ? 64 * hi : -16 * chunk), base, place(i));
      }
    }
  };
  // operand reads: lane l has row l & 31, columns 16 j + 8 (l / 32) and on of slice j
  int ra[2] = {ln * 64 + 16 * (h ^ ((ln >> 2) & 3)), ln * 64 + 16 * ((2 + h) ^ ((ln >> 2) & 3))};
  static_assert((S::SLOT & (S::SLOT - 1)) == 0 && S::SLOT >= 2048, "the slots differ in one bit of the address");
  auto read_x = [&](int b, int j) __attribute__((always_inline)) {
    return *reinterpret_cast<const u32x4_t*>(ring + (j >> 1) * (R * 64) + b * 2048 + ra[j & 1]);
  };

  // weights: each wave's 32 NTW columns, 64 bytes a step, go through its own part of LDS the same way: an
  // instruction fills 16 columns, and a lane reads its column's 16 bytes at 16 (l / 32) of both halves of the
  // step.  (32-bit offsets everywhere: 64-bit addresses would not fit into the registers.)
  const uint8_t* const wb = g.w + tile.expert * g.stride_w;
  const uint32_t lw = l0 + S::W + wave * WSTEP;
  const char* const w_slot = ring + S::W + wave * WSTEP;
  auto clamped = [&](int64_t n, int a) __attribute__((always_inline)) {
    const int64_t limit = g.gated && column(a) < half ? half : g.out;
    return (uint32_t)(n < limit ? n : limit - 1);                     // columns past the end are not stored
  };
  uint32_t wo[NTW][2], wn[NTW];
#pragma unroll
  for (int a = 0; a < NTW; ++a) {
    wn[a] = clamped(column(a) + ln, a);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      wo[a][i] = clamped(column(a) + 16 * i + (lane >> 2), a) * (uint32_t)g.ldw + 16 * chunk;
  }
  auto dma_w = [&](int s) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < NTW; ++a)
#pragma unroll
      for (int i = 0; i < 2; ++i) dma16(wo[a][i], wb + (int64_t)s * (kStep / 2), lw + a * 2048 + i * 1024);
  };
  const auto s_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<float*>(o.scales) + (size_t)tile.expert * o.padded * g.out, 0, 0xffffffffu, 0x00020000);
  const int words = KIND == kMxfp4 ? (int)(g.cols / 8) : (int)((g.cols + 7) / 8);
  // the codes of a step that is shorter than the others, zeros past the last column
  auto last_w = [&](int s, int a, int b) __attribute__((always_inline)) {
    u32x4_t v;
    const uint8_t* const p = wb + (size_t)wn[a] * g.ldw + (int64_t)s * (kStep / 2) + 32 * b + 16 * h;
    const int last = words - s * (kStep / 8) - 8 * b - 4 * h;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < last ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
    return v;
  };
  auto load_s = [&](float (&v)[NTW][GPS], int s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < GPS; ++i)
#pragma unroll
      for (int a = 0; a < NTW; ++a)
        v[a][i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
            s_rsrc, 4 * wn[a], (GPS == 1 ? div((uint32_t)s, g.per) : (uint32_t)s * GPS + i) * (uint32_t)(4 * g.out), 0));
  };

  // (floats, not the MFMAs' tuples of 16, unless an MFMA adds to them)
  struct Floats {
    float v[16];
    __device__ float& operator[](int i) { return v[i]; }
  };
  typename std::conditional<FOLD, f32x16_t, Floats>::type acc[MTW][NTW];
#pragma unroll
  for (int b = 0; b < MTW; ++b)
#pragma unroll
    for (int a = 0; a < NTW; ++a)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[b][a][e] = 0.f;

  // (what is requested is waited for: a workgroup that ends with DMA under way would leave it to write into the LDS
  // of the next one)
  if (s_begin < steps) dma(s_begin, 0, std::false_type{});
  if (s_begin < whole) dma_w(s_begin);
  if (KIND != kMxfp4 && split == 0) {
    // the zero points' part: sums of x [m][g] times -s z [n][g], 16 groups at a time
    const uint16_t *fp[NTW], *sp[MTW];
#pragma unroll
    for (int a = 0; a < NTW; ++a)
      fp[a] = o.factors + ((size_t)tile.expert * g.out + wn[a]) * o.pieces * o.padded + 8 * h;
#pragma unroll
    for (int b = 0; b < MTW; ++b) {
      const int64_t row = x_row(32 * b + ln);
      sp[b] = o.sums + (size_t)(row < 0 ? 0 : row) * 3 * o.padded + 8 * h;
    }
    f32x16_t p[MTW][NTW];
#pragma unroll
    for (int b = 0; b < MTW; ++b)
#pragma unroll
      for (int a = 0; a < NTW; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) p[b][a][e] = 0.f;
    for (uint32_t g0 = 0; g0 < o.padded; g0 += 16) {
      u32x4_t f[NTW][3], v[MTW][3];
#pragma unroll
      for (int b = 0; b < MTW; ++b)
#pragma unroll
        for (int i = 0; i < 3; ++i) v[b][i] = *reinterpret_cast<const u32x4_t*>(sp[b] + g0 + (size_t)i * o.padded);
#pragma unroll
      for (int a = 0; a < NTW; ++a) f[a][0] = *reinterpret_cast<const u32x4_t*>(fp[a] + g0);
      if (o.pieces > 1) {
#pragma unroll
        for (int a = 0; a < NTW; ++a) {
          f[a][1] = *reinterpret_cast<const u32x4_t*>(fp[a] + g0 + o.padded);
          f[a][2] = o.pieces > 2 ? *reinterpret_cast<const u32x4_t*>(fp[a] + g0 + 2 * (size_t)o.padded)
                                 : u32x4_t{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int b = 0; b < MTW; ++b)
#pragma unroll
          for (int a = 0; a < NTW; ++a) {
            p[b][a] = mfma32<Bf16>(v[b][0], f[a][1], p[b][a]);
            p[b][a] = mfma32<Bf16>(v[b][1], f[a][1], p[b][a]);
            p[b][a] = mfma32<Bf16>(v[b][0], f[a][2], p[b][a]);
          }
      }
#pragma unroll
      for (int b = 0; b < MTW; ++b)
#pragma unroll
        for (int a = 0; a < NTW; ++a)
#pragma unroll
          for (int i = 0; i < 3; ++i) p[b][a] = mfma32<Bf16>(v[b][i], f[a][0], p[b][a]);
    }
#pragma unroll
    for (int b = 0; b < MTW; ++b)
#pragma unroll
      for (int a = 0; a < NTW; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b][a][e] = p[b][a][e];
  }
  float next[NTW][GPS];
  if (s_begin < steps) load_s(next, s_begin);
  // Step s; `full`: the next one is a whole step (no branches then: the order of the loop's
  // instructions is kept).
  auto step = [&](int s, auto full) __attribute__((always_inline)) {
    constexpr bool FULL = decltype(full)::value;
    const int slot = (s - s_begin) & 1;
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");   // the step is here, the other slot read
    float sc[NTW][GPS];
    u32x4_t raw[NTW][2];
#pragma unroll
    for (int a = 0; a < NTW; ++a) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
        raw[a][b] = FULL || s < whole ? *reinterpret_cast<const u32x4_t*>(w_slot + a * 2048 + (ra[b] & (S::SLOT - 1)))
                                      : last_w(s, a, b);
#pragma unroll
      for (int i = 0; i < GPS; ++i) {
        sc[a][i] = next[a][i];
        asm volatile("" : "+v"(sc[a][i]));   // waited for before the DMA, which the compiler does not count
      }
    }
    uint32_t w[NTW][kSlices];
#pragma unroll
    for (int a = 0; a < NTW; ++a)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        // words 0 and 1 of both halves of the wave are slices 0 and 2, words 2 and 3 slices 1 and 3
        const auto u = __builtin_amdgcn_permlane32_swap(raw[a][b][0], raw[a][b][1], false, false);
        const auto v = __builtin_amdgcn_permlane32_swap(raw[a][b][2], raw[a][b][3], false, false);
        w[a][4 * b] = u[0], w[a][4 * b + 1] = v[0], w[a][4 * b + 2] = u[1], w[a][4 * b + 3] = v[1];
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                      // the codes are read
    __builtin_amdgcn_sched_barrier(0);
    if (FULL || s + 1 < steps) {
      dma(s + 1, slot ^ 1, full);
      if (FULL || s + 1 < whole) dma_w(s + 1);
      load_s(next, s + 1);
    }
    u32x4_t q[NTW][kSlices];
    auto convert = [&](int a, int j) __attribute__((always_inline)) {
      if constexpr (KIND == kMxfp4) q[a][j] = e2m1s<T>(w[a][j], FOLD ? sc[a][j * GPS / kSlices] : 1.f);
      else q[a][j] = nibbles<T>(w[a][j]);
    };
    if constexpr (!FOLD && MTW < 4) {
      // Units of PER MFMAs, one tile's group each, take turns with two sets of sums: while one is made the other is
      // scaled and added, and during the first the other tiles' codes are converted.
#pragma unroll
      for (int j = 0; j < kSlices; ++j) convert(0, j);
      u32x4_t v[kSlices];
#pragma unroll
      for (int j = 0; j < kSlices; ++j) v[j] = read_x(0, j);
      f32x16_t p[2];
      constexpr int UNITS = MTW * NTW * GPS;
      auto finish = [&](int u) __attribute__((always_inline)) {
        const int b = u / (NTW * GPS), a = u / GPS % NTW, i = u % GPS;
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b][a][e] = fmaf(p[u & 1][e], sc[a][i], acc[b][a][e]);
      };
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int b = u / (NTW * GPS), a = u / GPS % NTW, i = u % GPS;
        const bool ahead = a == NTW - 1 && b + 1 < MTW, first = b == 0 && a == 0 && NTW > 1;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int j = i * PER + k;
          p[u & 1] = mfma32<T>(v[j], q[a][j], k ? p[u & 1] : f32x16_t{});
          if (ahead) v[j] = read_x(b + 1, j);
          if (first) {
#pragma unroll
            for (int c = 1; c < NTW; ++c) convert(c, j);
          }
        }
        if (u) finish(u - 1);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          if (ahead) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          // (the other unit's last sums are not there at once)
          if (first) __builtin_amdgcn_sched_group_barrier(0x002, 9, 0);
          else if (k >= PER / 4) __builtin_amdgcn_sched_group_barrier(0x002, PER == 8 ? 3 : PER == 4 ? 6 : 8, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      finish(UNITS - 1);
    } else {
      // (256 columns by 128 rows: the registers hold no second set of sums)
#pragma unroll
      for (int a = 0; a < NTW; ++a)
#pragma unroll
        for (int j = 0; j < kSlices; ++j) convert(a, j);
#pragma unroll
      for (int b = 0; b < MTW; ++b) {
        __builtin_amdgcn_sched_barrier(0);
        f32x16_t p[NTW];
#pragma unroll
        for (int j = 0; j < kSlices; ++j) {
          const u32x4_t v = read_x(b, j);
#pragma unroll
          for (int a = 0; a < NTW; ++a) {
            if constexpr (FOLD) {
              acc[b][a] = mfma32<T>(v, q[a][j], acc[b][a]);
            } else {
              p[a] = mfma32<T>(v, q[a][j], j % PER ? p[a] : f32x16_t{});
              if (j % PER == PER - 1) {
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[b][a][e] = fmaf(p[a][e], sc[a][j / PER], acc[b][a][e]);
              }
            }
          }
        }
        // asks for two operand reads ahead of their MFMAs (the compiled loop waits for 18 of 32 right behind the read)
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
        for (int j = 0; j < kSlices - 2; ++j) {
          __builtin_amdgcn_sched_group_barrier(0x008, NTW, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    ra[0] ^= S::SLOT;
    ra[1] ^= S::SLOT;
  };
  int s = s_begin;
  for (; s + 1 < whole; ++s) step(s, std::true_type{});
  for (; s < steps; ++s) step(s, std::false_type{});
  // The arguments are read anew: kept over the loop they would not fit into the scalar registers.
  typedef const __attribute__((address_space(4))) W4Args* args_t;
  args_t again = (args_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(again));
  const auto& z = *again;
  auto missing = [&](int r) __attribute__((always_inline)) {
    const int64_t row = z.rows[tile.first + r];
    return row < 0 || row >= z.n_x;
  };
  // a lane has column l & 31 and rows 8 (e / 4) + 4 (l / 32) + e % 4
  if (z.bias) {
#pragma unroll
    for (int a = 0; a < NTW; ++a) {
      const int64_t n = column(a) + ln;
      const float bias = n < z.out ? load_any(z.bias, z.bias_type, n) : 0.f;
#pragma unroll
      for (int b = 0; b < MTW; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b][a][e] += bias;
    }
  }
  constexpr int UP = NTW / 2;
  if constexpr (UP > 0) {
    if (z.gated) {
#pragma unroll
      for (int b = 0; b < MTW; ++b)
#pragma unroll
        for (int a = 0; a < UP; ++a)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[b][a][e] = silu(acc[b][a][e]) * acc[b][a + UP][e];
    }
  }
  const int tiles = z.gated ? UP : NTW;
  // rows that x does not have (bit r of the tile's rows) are written as zeros
  uint64_t dead[2] = {0, 0};
  if (z.rows) {
    dead[0] = __ballot(lane < tile.count && missing(lane));
    if constexpr (R > 64) dead[1] = __ballot(64 + lane < tile.count && missing(64 + lane));
  }
  char* const y0 = static_cast<char*>(y_dev) + (tile.first * z.ldy + n0) * dtype_size((mi355q_dtype)z.y_type);
  if (n0 + 32 * tiles <= width && !(dead[0] | dead[1]) && z.ldy < (1 << 27)) {
    // all of the wave's columns are stored
    auto store_tiles = [&](auto type) __attribute__((always_inline)) {
      using O = decltype(type);
      constexpr int ES = sizeof(typename O::raw);
      const uint32_t pitch = (uint32_t)z.ldy * ES;
      // 16-bit types in pairs of columns: the even lanes take the even rows of both, the odd lanes the odd ones
      constexpr int STEP = ES == 2 ? 2 : 1;
      const bool odd = ES == 2 && (lane & 1);
      const int above = 4 * h + odd;
      const uint32_t off = (uint32_t)above * pitch + (uint32_t)(ln & -STEP) * ES;
#pragma unroll
      for (int b = 0; b < MTW; ++b)
#pragma unroll
        for (int e = 0; e < 16; e += STEP) {
          const int r = 32 * b + 8 * (e >> 2) + (e & 3);
          uint32_t v[NTW];
#pragma unroll
          for (int a = 0; a < NTW; ++a) {
            if constexpr (ES == 4) {
              v[a] = __float_as_uint(acc[b][a][e]);
            } else {
              const float mine = acc[b][a][e], below = acc[b][a][e + 1];
              const float got = __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp(
                  (int)__float_as_uint(odd ? mine : below), 0xb1, 0xf, 0xf, true));   // the neighbour's
              v[a] = O::store(odd ? got : mine) | (uint32_t)O::store(odd ? below : got) << 16;
            }
          }
          if (r + above < tile.count) {
#pragma unroll
            for (int a = 0; a < NTW; ++a)
              if (a < tiles) __builtin_memcpy(y0 + (int64_t)r * pitch + 32 * a * ES + off, &v[a], 4);
          }
        }
    };
    if (z.y_type == MI355Q_BF16) store_tiles(Bf16{});
    else if (z.y_type == MI355Q_F16) store_tiles(F16{});
    else store_tiles(F32{});
    return;
  }
#pragma unroll
  for (int b = 0; b < MTW; ++b)
#pragma unroll
    for (int a = 0; a < NTW; ++a) {
      if (a >= tiles || n0 + 32 * a + ln >= width) continue;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int r = 32 * b + 8 * (e >> 2) + 4 * h + (e & 3);
        if (r >= tile.count) continue;
        const float v = dead[b / 2] >> (r & 63) & 1 ? 0.f : acc[b][a][e];
        const int64_t at = (int64_t)r * z.ldy + 32 * a + ln;
        if (z.y_type == MI355Q_F32) reinterpret_cast<float*>(y0)[at] = v;
        else reinterpret_cast<uint16_t*>(y0)[at] = z.y_type == MI355Q_BF16 ? Bf16::store(v) : F16::store(v);
      }
    }
}

// ---------------------------------------------------------------- launches
// The tile of a call, 32 mt rows by 128 nt columns of w, and how many workgroups share a sum.
struct TilePlan {
  int mt, nt;
  uint32_t splits;
};
TilePlan tile_plan(int64_t rows, int64_t experts, int64_t out, int64_t cols, bool gated, bool listed);

inline bool w_in_place(const W4Args& g) { return aligned16(g.w) && g.ldw % 16 == 0 && g.stride_w % 16 == 0; }
inline size_t sums_bytes(int64_t n_x, uint32_t groups) {
  return ((size_t)n_x * 3 * ((groups + 15) / 16 * 16) * sizeof(uint16_t) + 255) / 256 * 256;
}
inline size_t scales_bytes(int64_t rows_w, uint32_t groups) {
  return ((size_t)rows_w * ((groups + 15) / 16 * 16) * sizeof(float) + 255) / 256 * 256;
}
inline size_t x_copy_bytes(int64_t n_x, int64_t cols) {
  return (size_t)n_x * ((cols + kStep - 1) / kStep * kStep) * sizeof(uint16_t);
}
inline size_t parts_bytes(const TilePlan& p, int64_t rows, int64_t out) {
  return p.splits > 1 ? ((size_t)p.splits * rows * out * sizeof(float) + 255) / 256 * 256 : 0;
}

template <class T, int KIND, int GPS, int MTW, int NTW>
static int launch_shape(W4Args g, W4Tiles o, hipStream_t st) {
  constexpr int R = TileShape<MTW>::R;
  const W4Args whole = g;
  if (o.splits > 1) {              // the parts are of w's columns, without what follows the sum
    g.gated = 0;
    g.bias = nullptr;
    g.y_type = MI355Q_F32;
    g.ldy = g.out;
  }
  const int64_t width = g.gated ? g.out / 2 : g.out, per = kWaves * (g.gated ? 16 * NTW : 32 * NTW);
  const int64_t ct = (width + per - 1) / per;
  const int64_t rt = g.offsets ? most_row_tiles(g, R) : (g.n_rows + R - 1) / R;
  int64_t rounded = rt;
  if (g.offsets) {                 // whole rounds of bands, a band for each XCD
    o.band = (uint32_t)(rt >= 512 ? 8 : rt >= 64 ? rt / 64 : 1);
    rounded = (rt + 8 * o.band - 1) / (8 * o.band) * (8 * o.band);
  }
  MQ_CHECK_ARG(ct * rounded * o.splits <= (int64_t)(UINT32_MAX / 256),
               "w4a16_matmul: %lld rows by %lld columns are too many", (long long)g.n_rows, (long long)width);
  o.row_tiles = (uint32_t)rt;
  o.col_tiles = (uint32_t)ct;
  hipLaunchKernelGGL((w4_tiles_kernel<T, KIND, GPS, MTW, NTW>), dim3((unsigned)(ct * rounded * o.splits)),
                     dim3(64 * kWaves), 0, st, g, o);
  MQ_LAUNCH_CHECK();
  return o.splits > 1 ? join_parts(whole, o.splits, o.parts, st) : MI355Q_OK;
}

template <class T, int KIND, int GPS>
static int launch_kind(const W4Args& g, W4Tiles o, const TilePlan& p, hipStream_t st) {
  o.splits = p.splits;
  if (p.mt == 4) return launch_shape<T, KIND, GPS, 4, 2>(g, o, st);
  if (p.mt == 2 && p.nt == 2) return launch_shape<T, KIND, GPS, 2, 2>(g, o, st);
  if (p.mt == 2) return launch_shape<T, KIND, GPS, 2, 1>(g, o, st);
  if (p.nt == 2) return launch_shape<T, KIND, GPS, 1, 2>(g, o, st);
  return launch_shape<T, KIND, GPS, 1, 1>(g, o, st);
}

template <class T>
static int launch_type(W4Args g, int kind, void* workspace, hipStream_t st) {
  const TilePlan plan = tile_plan(g.n_rows, g.experts, g.out, g.cols, g.gated, g.offsets || g.rows);
  const bool copy = !in_place(g), sums = kind != kMxfp4;
  const uint32_t padded = (g.groups + 15) / 16 * 16;
  char* at = static_cast<char*>(workspace);
  // -s z: bf16's 8 bits times 8 are bf16 numbers, times 4 bits, or fp16's 11 bits times 4, two of them
  const int pieces = g.s_type == MI355Q_F32 ? 3 : g.s_type == MI355Q_BF16 && kind == kInt4 ? 1 : 2;
  uint16_t *to_sums = nullptr, *to_factors = nullptr, *to = nullptr;
  if (sums) {
    to_sums = reinterpret_cast<uint16_t*>(at);
    at += sums_bytes(g.n_x, g.groups);
    to_factors = reinterpret_cast<uint16_t*>(at);
    at += sums_bytes(g.experts * g.out, g.groups);
  }
  float* const to_scales = reinterpret_cast<float*>(at);
  at += scales_bytes(g.experts * g.out, g.groups);
  float* const parts = reinterpret_cast<float*>(at);
  at += parts_bytes(plan, g.n_rows, g.out);
  const int64_t ld_copy = (g.cols + kStep - 1) / kStep * kStep;
  if (copy) to = reinterpret_cast<uint16_t*>(at);
  uint8_t* to_w = nullptr;
  const int64_t w_bytes = kind == kMxfp4 ? g.cols / 2 : (g.cols + 7) / 8 * 4, w_pitch = (w_bytes + 15) / 16 * 16;
  if (w_bytes % 16) {
    if (copy) at += x_copy_bytes(g.n_x, g.cols);
    to_w = reinterpret_cast<uint8_t*>(at);
  }
  const W4Tiles o = {to_sums, to_factors, to_scales, padded, pieces, 0, 0, 1, 1, parts};
  int lanes = 0;
  while (lanes < 6 && (8 << lanes) < g.group) ++lanes;
  const uint64_t waves = (padded + (64u >> lanes) - 1) / (64u >> lanes);
  const uint64_t x_blocks = copy || sums ? (waves * (uint64_t)g.n_x + 3) / 4 : 0;
  const uint64_t f_blocks = (uint64_t)g.experts * ((g.out + 31) / 32) * (padded / 8);
  const uint64_t c_blocks = to_w ? ((uint64_t)g.experts * g.out * (w_pitch / 16) + 255) / 256 : 0;
  MQ_CHECK_ARG(x_blocks + f_blocks + c_blocks <= UINT32_MAX / 256,
               "w4a16_matmul: %lld rows of x and %lld of weights are too many", (long long)g.n_x,
               (long long)(g.experts * g.out));
  const W4Prepare p = {padded, lanes, o.pieces, (uint32_t)x_blocks, (uint32_t)f_blocks, to_sums, to_factors,
                       reinterpret_cast<uint32_t*>(to_scales), to, ld_copy, to_w, w_bytes};
  const dim3 grid((unsigned)(x_blocks + f_blocks + c_blocks)), block(256);
  if (kind == kInt4Zero) hipLaunchKernelGGL((w4_prepare_kernel<T, kInt4Zero>), grid, block, 0, st, g, p);
  else if (kind == kInt4) hipLaunchKernelGGL((w4_prepare_kernel<T, kInt4>), grid, block, 0, st, g, p);
  else hipLaunchKernelGGL((w4_prepare_kernel<T, kMxfp4>), grid, block, 0, st, g, p);
  MQ_LAUNCH_CHECK();
  if (to_w) {
    g.w = to_w;
    g.ldw = w_pitch;
    g.stride_w = g.out * w_pitch;
  }
  if (copy) {
    g.x = to;
    g.ldx = ld_copy;
  }
  const int gps = g.groups > 1 && g.group == 32 ? 4 : g.groups > 1 && g.group == 64 ? 2 : 1;
  // (zero points enter before the sum: the tiles do not tell them apart)
  if (kind == kMxfp4) return launch_kind<T, kMxfp4, 4>(g, o, plan, st);
  if (gps == 4) return launch_kind<T, kInt4, 4>(g, o, plan, st);
  if (gps == 2) return launch_kind<T, kInt4, 2>(g, o, plan, st);
  return launch_kind<T, kInt4, 1>(g, o, plan, st);
}

}  // namespace mi355q
