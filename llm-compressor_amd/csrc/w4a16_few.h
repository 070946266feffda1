// The kernel of 4-bit products for few rows (w4a16.h) and its launch; instantiated in files
// of their own per type and weight, so that they compile in parallel.
#pragma once

#include <type_traits>

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

// The scales' type is a parameter of the kernel (Bf16, F16, F32, and this for MXFP4's bytes).  Told apart by a branch
// between a step's matrix instructions and its sums, the compiler counted the wait for their results along the longer of
// the branch's two paths alone, and the other one read the last registers before they were written.
struct E8m0 {
  typedef uint8_t raw;
};

// ---------------------------------------------------------------- few rows
// The operands, scales and zero points of steps_ neighbouring steps as loaded.
template <int steps_, int NT, int MB, int XL, int GPS, int ES>
struct W4Batch {
  static constexpr int N = steps_;
  u32x4_t w[N][NT], x[N][MB][XL];
  uint32_t s[NT][GPS ? (N * GPS * ES + 3) / 4 : N], z[NT][N * (GPS ? GPS : 1)];
};

// A workgroup makes a tile of rows by 16 NT columns of y; its W waves take a range
// of the steps of 128 columns each, straight from memory into the MFMAs' registers (x: rows,
// w: columns; a lane's sums are one column's), and join their sums in LDS.  With
// `splits` each of so many workgroups takes a range of the steps and leaves its
// sums in fp32, parts[split][row][column of w], for w4_join_kernel.
//
// MT > 0: tiles of 16 MT rows.  MT = 0: tiles of 4 rows.  The MFMA's 16 rows are then the four rows'
// four quarters of a step, 32 columns each, so that one load holds a step's x; instruction i multiplies
// all of them with quarter i of the weight, and of its result row 4 r + i counts, which is
// register i of the lanes 16 r and on.
//
// What counts is loads, their number and how many are in flight: D steps of a wave are requested before
// the first is used, the scales of all D in one load, the next ones as the registers come free, and
// nothing in the loop over whole steps branches (a wait belongs to a branch, so one around a load
// ends the overlap: one token's 14336 x 4096 took 13.2 us with branches around dead rows).  A batch's scales are its
// last request and the first thing that its use needs, so a wave waits for nearly the whole batch at its head, and
// batches hardly overlap.
// Rows past a tile's end read its first row, columns past w's end its last;
// neither is stored.  GPS: scales per step, 0: one for several steps.
//
// One token, 14336 x 4096 in groups of 128: 10.4 us, 2.9 TB/s (9.0 to 9.3 with the same weight again and again, 11.2 with
// twelve in turn; reading the same 30 MB alone 6.0, a launch of nothing 1.8).  23 rows, 4096 x 14336 MXFP4: 19.7 us
// with the join; the MFMAs are 6 % busy: one step is in flight, and every 64 columns read x anew (two column
// tiles a wave 25 us; two steps in flight instead of one 21).  61 tokens to 8 of 128 experts, 1536 x 2048 in groups of 32
// with zero points: 56 us, 4.1 TB/s.  Tiles of 64 rows do not fit the registers for int4: 32 to 52 bytes a lane go to
// scratch with 16-bit scales, up to 520 with zero points (48 rows of 4096 x 4096 in groups of 128 16.3 us, with zero
// points in groups of 32 30).
template <class T, int KIND, int GPS, class S, int MT, int NT, int W, int D>
__global__ __launch_bounds__(64 * W) void w4_few_kernel(W4Args g, uint32_t nt, uint32_t splits, float* parts) {
  constexpr int ES = sizeof(typename S::raw);
  constexpr bool FOLD = KIND == kMxfp4 && T::code == MI355Q_BF16;     // the scale is in the operand
  using Sum = typename std::conditional<MT == 0, float, f32x4_t>::type;
  constexpr int MB = MT ? MT : 1;
  __shared__ Sum sums[W][NT][MB][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quarter = lane >> 4;
  const uint32_t split = splits > 1 ? blockIdx.x % splits : 0, id = splits > 1 ? blockIdx.x / splits : blockIdx.x;
  constexpr int ROWS = MT ? 16 * MT : 4;
  const RowTile tile = row_tile<ROWS>(g, id / nt);
  if (tile.count <= 0) return;
  const int64_t half = g.gated ? g.out / 2 : 0, width = g.gated ? half : g.out;   // of y
  const int64_t n0 = (int64_t)(id % nt) * 16 * (g.gated ? NT / 2 : NT);
  // column of tile a on this lane: the second half of a gated weight's tiles holds its second half
  auto column = [&](int a) __attribute__((always_inline)) {
    return g.gated && a >= NT / 2 ? half + n0 + 16 * (a - NT / 2) : n0 + 16 * a;
  };
  const uint8_t* wp[NT];
  const char* sp[NT];
  const uint32_t* zp[NT];
  int zs[NT];
  const int64_t expert = tile.expert < 0 ? 0 : tile.expert;
#pragma unroll
  for (int a = 0; a < NT; ++a) {
    const int64_t limit = g.gated && a < NT / 2 ? half : g.out;
    int64_t n = column(a) + col;
    n = n < limit ? n : limit - 1;
    wp[a] = g.w + expert * g.stride_w + n * g.ldw + 16 * quarter;
    sp[a] = static_cast<const char*>(g.s) + (expert * g.stride_s + n * g.lds) * ES;
    zp[a] = g.z + expert * g.stride_z + n / 8 * g.ldz;
    zs[a] = 4 * (int)(n % 8);
  }
  const uint16_t* xp[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    const int r = MT ? 16 * b + col : col >> 2;
    int64_t row = tile.first + (r < tile.count ? r : 0);
    if (g.rows) row = g.rows[row];
    xp[b] = g.x + (row >= 0 && row < g.n_x ? row : 0) * g.ldx + 8 * quarter + (MT ? 0 : 32 * (col & 3));
  }
  Sum acc[NT][MB];
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int b = 0; b < MB; ++b) acc[a][b] = Sum{};

  constexpr int XL = MT ? 4 : 1;                                     // loads of x per step and 16 rows
  constexpr int G1 = GPS ? GPS : 1;
  // the operands of N neighbouring steps
  auto load_operands = [&](u32x4_t (&w)[NT], u32x4_t (&x)[MB][XL], int s) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < NT; ++a) __builtin_memcpy(&w[a], wp[a] + (int64_t)s * (kStep / 2), 16);
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int i = 0; i < XL; ++i) __builtin_memcpy(&x[b][i], xp[b] + (int64_t)s * kStep + 32 * i, 16);
  };
  auto load_scales = [&](auto& o, int s) __attribute__((always_inline)) {
    constexpr int N = std::remove_reference_t<decltype(o)>::N;
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      if constexpr (GPS == 0) {
#pragma unroll
        for (int d = 0; d < N; ++d) {
          const uint32_t gi = div((uint32_t)(s + d), g.per);
          if constexpr (ES == 4) o.s[a][d] = reinterpret_cast<const uint32_t*>(sp[a])[gi];
          else o.s[a][d] = reinterpret_cast<const uint16_t*>(sp[a])[gi];
          if constexpr (KIND == kInt4Zero) o.z[a][d] = zp[a][gi];
        }
      } else {
        if constexpr (N * GPS * ES == 2) o.s[a][0] = *reinterpret_cast<const uint16_t*>(sp[a] + (int64_t)s * GPS * ES);
        else __builtin_memcpy(o.s[a], sp[a] + (int64_t)s * GPS * ES, N * GPS * ES);
        if constexpr (KIND == kInt4Zero) __builtin_memcpy(o.z[a], zp[a] + (int64_t)s * GPS, 4 * N * GPS);
      }
    }
  };
  // a step of fewer than 128 columns: zeros past the last one, the last scale for groups past the last
  const int words = KIND == kMxfp4 ? (int)(g.cols / 8) : (int)((g.cols + 7) / 8);
  auto load_last = [&](auto& o, int s) __attribute__((always_inline)) {
    const int left = words - s * (kStep / 8) - 4 * quarter;
#pragma unroll
    for (int a = 0; a < NT; ++a) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o.w[0][a][i] = i < left ? reinterpret_cast<const uint32_t*>(wp[a] + (int64_t)s * (kStep / 2))[i] : 0u;
#pragma unroll
      for (int i = 0; i < (G1 * ES + 3) / 4; ++i) o.s[a][i] = 0;
#pragma unroll
      for (int i = 0; i < G1; ++i) {
        const uint32_t gs = GPS == 0 ? div((uint32_t)s, g.per) : (uint32_t)s * GPS + i;
        const uint32_t gi = gs < g.groups ? gs : g.groups - 1;
        if constexpr (ES == 4) o.s[a][i] = reinterpret_cast<const uint32_t*>(sp[a])[gi];
        else if constexpr (ES == 2)
          o.s[a][i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(sp[a])[gi] << 16 * (i & 1);
        else o.s[a][0] |= (uint32_t)reinterpret_cast<const uint8_t*>(sp[a])[gi] << 8 * i;
        if constexpr (KIND == kInt4Zero) o.z[a][i] = zp[a][gi];
      }
    }
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int i = 0; i < XL; ++i)
        o.x[0][b][i] = last_chunk(xp[b] + (int64_t)s * kStep + 32 * i,
                                  g.cols - (int64_t)s * kStep - 32 * (MT ? i : col & 3) - 8 * quarter);
  };
  // the scales of step d of a batch
  auto scales = [&](const auto& o, int d, float (&sc)[NT][G1]) __attribute__((always_inline)) {
    if constexpr (KIND == kMxfp4) {
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int i = 0; i < G1; ++i) {
          const uint32_t e = (o.s[a][d] >> 8 * i) & 255u;
          sc[a][i] = FOLD ? __uint_as_float((e << 23) | 0x00400000u) : e8m0_to_f32(e);
        }
    } else if constexpr (ES == 4) {
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int i = 0; i < G1; ++i) sc[a][i] = __uint_as_float(o.s[a][d * G1 + i]);
    } else {
      auto half = [&](int a, int i) __attribute__((always_inline)) {
        const int at = GPS ? d * GPS + i : 2 * d;
        return at & 1 ? o.s[a][at / 2] >> 16 : o.s[a][at / 2] & 0xffffu;
      };
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int i = 0; i < G1; ++i) sc[a][i] = S::load((uint16_t)half(a, i));
    }
  };
  constexpr uint32_t one = T::code == MI355Q_BF16 ? 0x3f803f80u : 0x3c003c00u;
  constexpr uint32_t minus8 = T::code == MI355Q_BF16 ? 0xc100c100u : 0xc800c800u;
  constexpr uint32_t unit = KIND == kInt4 ? minus8 : one;
  const u32x4_t units = {unit, unit, unit, unit};
  auto use = [&](const auto& o, int d) __attribute__((always_inline)) {
    constexpr int PER = 4 / G1;                                    // instructions per group
    u32x4_t q[NT][4];
    float sc[NT][G1], z[NT][G1];
    scales(o, d, sc);
#pragma unroll
    for (int a = 0; a < NT; ++a) {
#pragma unroll
      for (int i = 0; i < G1; ++i) {
        if constexpr (KIND == kInt4Zero) z[a][i] = -(float)((o.z[a][d * G1 + i] >> zs[a]) & 15u);
      }
      const u32x4_t w = transpose_words(o.w[d][a]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (KIND == kMxfp4) q[a][i] = e2m1s<T>(w[i], FOLD ? sc[a][i * G1 / 4] : 1.f);
        else q[a][i] = nibbles<T>(w[i]);
      }
    }
    if constexpr (MT == 0) {
      const u32x4_t x = o.x[d][0][0];
      f32x4_t base = {0.f, 0.f, 0.f, 0.f};
      if constexpr (KIND != kMxfp4) base = mfma<T>(x, units, base);
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x4_t t = base;
          if constexpr (KIND == kInt4Zero) t[i] *= z[a][i / PER];
          t = mfma<T>(x, q[a][i], t);
          acc[a][0] = FOLD ? acc[a][0] + t[i] : fmaf(t[i], sc[a][i / PER], acc[a][0]);
        }
    } else {
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int i = 0; i < G1; ++i) {
          f32x4_t base = {0.f, 0.f, 0.f, 0.f};
          if constexpr (KIND != kMxfp4) {
#pragma unroll
            for (int j = 0; j < PER; ++j) base = mfma<T>(o.x[d][b][i * PER + j], units, base);
          }
#pragma unroll
          for (int a = 0; a < NT; ++a) {
            if constexpr (FOLD) {
#pragma unroll
              for (int j = 0; j < PER; ++j) acc[a][b] = mfma<T>(o.x[d][b][i * PER + j], q[a][i * PER + j], acc[a][b]);
            } else {
              f32x4_t t = base;
              if constexpr (KIND == kInt4Zero) {
#pragma unroll
                for (int r = 0; r < 4; ++r) t[r] = base[r] * z[a][i];
              }
#pragma unroll
              for (int j = 0; j < PER; ++j) t = mfma<T>(o.x[d][b][i * PER + j], q[a][i * PER + j], t);
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[a][b][r] = fmaf(t[r], sc[a][i], acc[a][b][r]);
            }
          }
        }
    }
  };
  // this wave's whole steps are first + i, i < n
  const uint32_t all = (uint32_t)((g.cols + kStep - 1) / kStep);
  const int begin = (int)(all * split / splits), end = (int)(all * (split + 1) / splits);
  const int whole = (int)(g.cols / kStep) < end ? (int)(g.cols / kStep) : end;
  const int mine = whole > begin ? whole - begin : 0;
  const int first = begin + mine * wave / W, n = tile.expert < 0 ? 0 : begin + mine * (wave + 1) / W - first;
  using Many = W4Batch<D, NT, MB, XL, GPS, ES>;
  using One = W4Batch<1, NT, MB, XL, GPS, ES>;
  {
    Many o;
    One rest[D > 1 ? D - 1 : 1];
    int i = 0;
    if (n >= D) {
#pragma unroll
      for (int d = 0; d < D; ++d) load_operands(o.w[d], o.x[d], first + d);
      load_scales(o, first);
      for (; i + 2 * D <= n; i += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
          use(o, d);
          load_operands(o.w[d], o.x[d], first + i + D + d);
        }
        load_scales(o, first + i + D);
      }
    }
    const int more = n >= D ? i + D : 0;
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
      if (more + d < n) {
        load_operands(rest[d].w[0], rest[d].x[0], first + more + d);
        load_scales(rest[d], first + more + d);
      }
    if (n >= D) {
#pragma unroll
      for (int d = 0; d < D; ++d) use(o, d);
    }
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
      if (more + d < n) use(rest[d], 0);
  }
  if (tile.expert >= 0 && whole < end && wave == W - 1) {
    One o;
    load_last(o, whole);
    use(o, 0);
  }
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int b = 0; b < MB; ++b) sums[wave][a][b][lane] = acc[a][b];
  __syncthreads();
  // register r of tile b on this lane is row row_of(b, r)
  constexpr int REGS = MT ? 4 : 1;
  auto row_of = [&](int b, int r) __attribute__((always_inline)) { return MT ? 16 * b + 4 * quarter + r : quarter; };
  auto total = [&](int a, int b, float (&v)[REGS]) __attribute__((always_inline)) {
    Sum t = sums[0][a][b][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) t += sums[w][a][b][lane];
    __builtin_memcpy(v, &t, sizeof(t));
    const int64_t n = column(a) + col;
    if (g.bias && n < g.out && splits == 1 && tile.expert >= 0) {      // (rows of no expert are zeros)
      const float bias = load_any(g.bias, g.bias_type, n);
#pragma unroll
      for (int r = 0; r < REGS; ++r) v[r] += bias;
    }
  };
  if (splits > 1) {
    for (int i = wave; i < NT * MB; i += W) {
      const int a = i / MB, b = i % MB;
      float v[REGS];
      total(a, b, v);
      const int64_t n = column(a) + col, limit = g.gated && a < NT / 2 ? half : g.out;
#pragma unroll
      for (int r = 0; r < REGS; ++r)
        if (row_of(b, r) < tile.count && n < limit)
          parts[(split * g.n_rows + tile.first + row_of(b, r)) * g.out + n] = v[r];
    }
    return;
  }
  for (int i = wave; i < (g.gated ? NT / 2 : NT) * MB; i += W) {
    const int a = i / MB, b = i % MB;
    float v[REGS];
    total(a, b, v);
    if (g.gated) {
      float up[REGS];
      total(a + NT / 2, b, up);
#pragma unroll
      for (int r = 0; r < REGS; ++r) v[r] = silu(v[r]) * up[r];
    }
    const int64_t n = n0 + 16 * a + col;
    if (n >= width) continue;
#pragma unroll
    for (int r = 0; r < REGS; ++r) {
      const int row = row_of(b, r);
      if (row >= tile.count) continue;
      if (g.rows) {                                                  // a row that x does not have counts as zeros
        const int64_t from = g.rows[tile.first + row];
        if (from < 0 || from >= g.n_x) v[r] = 0.f;
      }
      const int64_t at = (tile.first + row) * g.ldy + n;
      if (g.y_type == MI355Q_F32) static_cast<float*>(g.y)[at] = v[r];
      else static_cast<uint16_t*>(g.y)[at] = g.y_type == MI355Q_BF16 ? Bf16::store(v[r]) : F16::store(v[r]);
    }
  }
}

template <class T, int KIND, int GPS, class S, int MT, int NT, int W, int D>
static int launch_few(const W4Args& g, uint32_t splits, float* parts, hipStream_t st) {
  const int64_t width = g.gated ? g.out / 2 : g.out, per = 16 * (g.gated ? NT / 2 : NT);
  const int64_t nt = (width + per - 1) / per;
  constexpr int ROWS = MT ? 16 * MT : 4;
  const int64_t mt = g.offsets ? most_row_tiles(g, ROWS) : (g.n_rows + ROWS - 1) / ROWS;
  MQ_CHECK_ARG(nt * mt * splits <= (int64_t)(UINT32_MAX / (64 * W)),
               "w4a16_matmul: %lld rows by %lld columns are too many", (long long)g.n_rows, (long long)width);
  hipLaunchKernelGGL((w4_few_kernel<T, KIND, GPS, S, MT, NT, W, D>), dim3((unsigned)(nt * mt * splits)), dim3(64 * W), 0,
                     st, g, (uint32_t)nt, splits, parts);
  MQ_LAUNCH_CHECK();
  return splits > 1 ? join_parts(g, splits, parts, st) : MI355Q_OK;
}

template <class T, int KIND, int GPS, class S>
static int launch_kind(const W4Args& g, const FewPlan& p, float* parts, hipStream_t st) {
  const uint32_t splits = p.splits;
  if (p.mt == 4) return launch_few<T, KIND, GPS, S, 4, 4, 8, 1>(g, splits, parts, st);
  if (p.mt == 2) return launch_few<T, KIND, GPS, S, 2, 4, 8, 1>(g, splits, parts, st);
  if (p.mt == 1) {
    if (p.w == 1) return launch_few<T, KIND, GPS, S, 1, 2, 1, 2>(g, 1, parts, st);
    if (p.nt == 4) return launch_few<T, KIND, GPS, S, 1, 4, 4, 2>(g, 1, parts, st);
    if (p.nt == 2) return launch_few<T, KIND, GPS, S, 1, 2, 4, 2>(g, 1, parts, st);
    return launch_few<T, KIND, GPS, S, 1, 1, 8, 2>(g, 1, parts, st);
  }
  if (p.nt == 2) {
    if (p.w == 2) return launch_few<T, KIND, GPS, S, 0, 2, 2, 4>(g, 1, parts, st);
    if (p.w == 4) return launch_few<T, KIND, GPS, S, 0, 2, 4, 2>(g, 1, parts, st);
    return launch_few<T, KIND, GPS, S, 0, 2, 8, 2>(g, 1, parts, st);
  }
  if (p.w == 2) return launch_few<T, KIND, GPS, S, 0, 1, 2, 4>(g, 1, parts, st);
  if (p.w == 4) return launch_few<T, KIND, GPS, S, 0, 1, 4, 4>(g, 1, parts, st);
  return launch_few<T, KIND, GPS, S, 0, 1, 8, 2>(g, 1, parts, st);
}

template <class T, int KIND, class S>
static int launch_scales(const W4Args& g, const FewPlan& p, float* parts, hipStream_t st) {
  if (g.groups > 1 && g.group == 32) return launch_kind<T, KIND, 4, S>(g, p, parts, st);
  if (g.groups > 1 && g.group == 64) return launch_kind<T, KIND, 2, S>(g, p, parts, st);
  if (g.per.d == 1) return launch_kind<T, KIND, 1, S>(g, p, parts, st);
  return launch_kind<T, KIND, 0, S>(g, p, parts, st);
}

template <class T, int KIND>
static int launch_groups(const W4Args& g, const FewPlan& p, float* parts, hipStream_t st) {
  if (g.s_type == MI355Q_F32) return launch_scales<T, KIND, F32>(g, p, parts, st);
  if (g.s_type == MI355Q_BF16) return launch_scales<T, KIND, Bf16>(g, p, parts, st);
  return launch_scales<T, KIND, F16>(g, p, parts, st);
}

}  // namespace mi355q
