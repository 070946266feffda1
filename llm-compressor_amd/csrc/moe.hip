// Tokens into the order of the experts that they are routed to and back.
//
// A pair (t, k) is token t's k-th choice, expert ids[t][k].  The plan is a stable
// counting sort of the pairs by expert, the pairs taken position by position
// (f = k T + t), which is the order in which a loop over experts meets them; pairs
// whose id is no expert go behind the last one:
//
//   slots[t][k] = pairs of smaller ids + earlier pairs of the same id
//   rows[slots[t][k]] = t,  offsets[e] = pairs of ids below e
//
//   sort              s[slots[t][k]] = x[t]             (zeros from offsets[E] on)
//   its gradient      dx[t] = sum_k ds[slots[t][k]]
//   combine           y[t] = sum_k w[t][k] o[slots[t][k]]
//   its gradients     do[slots[t][k]] = w[t][k] dy[t],  dw[t][k] = <o[slots[t][k]], dy[t]>
//
// Sums are fp32, in the order of k, rounded once; rows from offsets[E] on take no part
// (their gradients are zeros).  Nothing is added with atomics that are not integer
// counts, so results do not change from run to run.
#include "fp8.h"

namespace mi355q {

// ---------------------------------------------------------------- plan
// Workgroups of 8 waves take `chunk` consecutive pairs each, a wave an eighth of
// them.  With one workgroup the plan is one launch; else a first launch leaves each
// chunk's counts per expert, and the second adds up those before its own.
constexpr int kPlanWaves = 8, kPlanThreads = 64 * kPlanWaves;
constexpr int kMaxExperts = 2040;                   // 8 waves' counts of E + 1 ids in 64 KB of LDS
constexpr int kPlanChunk = 2048;                    // pairs per workgroup, at the least
constexpr int kPlanGroups = 512;                    // workgroups, at the most

struct PlanArgs {
  const void* ids;
  int wide;            // ids are int64
  int64_t ld;
  uint32_t tokens, top, pairs, experts, chunk;
  int32_t* rows;
  int32_t* slots;
  int64_t* offsets;
  uint32_t* counts;    // [workgroups][experts + 1]
};

__device__ __forceinline__ uint32_t id_of(const PlanArgs& g, uint32_t f, uint32_t& t, uint32_t& k) {
  k = f / g.tokens;
  t = f - k * g.tokens;
  const int64_t at = (int64_t)t * g.ld + k;
  const int64_t id = g.wide ? static_cast<const int64_t*>(g.ids)[at] : static_cast<const int32_t*>(g.ids)[at];
  return id >= 0 && id < (int64_t)g.experts ? (uint32_t)id : g.experts;
}

__global__ __launch_bounds__(kPlanThreads) void moe_count_kernel(PlanArgs g) {
  extern __shared__ uint32_t hist[];
  for (uint32_t e = threadIdx.x; e <= g.experts; e += kPlanThreads) hist[e] = 0;
  __syncthreads();
  const uint32_t begin = blockIdx.x * g.chunk, end = begin + g.chunk < g.pairs ? begin + g.chunk : g.pairs;
  for (uint32_t f = begin + threadIdx.x; f < end; f += kPlanThreads) {
    uint32_t t, k;
    atomicAdd(&hist[id_of(g, f, t, k)], 1u);
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e <= g.experts; e += kPlanThreads)
    g.counts[(size_t)blockIdx.x * (g.experts + 1) + e] = hist[e];
}

// exclusive prefix sums of v over the workgroup's threads, and their total
__device__ __forceinline__ uint32_t scan_threads(uint32_t v, uint32_t* part, uint32_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(s, d);
    if (lane >= d) s += o;
  }
  if (lane == 63) part[wave] = s;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    before += w < wave ? part[w] : 0u;
    total += part[w];
  }
  __syncthreads();
  return before + s - v;
}

// LDS: [8][E + 1] counts of the waves, then the ranks at which their pairs begin
template <bool ONE>
__global__ __launch_bounds__(kPlanThreads) void moe_place_kernel(PlanArgs g) {
  extern __shared__ uint32_t at[];
  __shared__ uint32_t part[kPlanWaves];
  const uint32_t ids = g.experts + 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (uint32_t i = threadIdx.x; i < kPlanWaves * ids; i += kPlanThreads) at[i] = 0;
  __syncthreads();
  const uint32_t per = g.chunk / kPlanWaves;                   // a multiple of 64
  const uint32_t begin = blockIdx.x * g.chunk + wave * per;
  const uint32_t end = begin + per < g.pairs ? begin + per : g.pairs;
  uint32_t* const mine = at + wave * ids;
  for (uint32_t f = begin + lane; f < end; f += 64) {
    uint32_t t, k;
    atomicAdd(&mine[id_of(g, f, t, k)], 1u);
  }
  __syncthreads();
  uint32_t run = 0;                                            // pairs of the ids before this round's
  for (uint32_t e0 = 0; e0 < ids; e0 += kPlanThreads) {
    const uint32_t e = e0 + threadIdx.x;
    uint32_t all = 0, before = 0;
    if (e < ids) {
      if constexpr (ONE) {
#pragma unroll
        for (int w = 0; w < kPlanWaves; ++w) all += at[w * ids + e];
      } else {
        const uint32_t n = gridDim.x;
#pragma unroll 8
        for (uint32_t b = 0; b < n; ++b) {
          const uint32_t c = g.counts[(size_t)b * ids + e];
          all += c;
          before += b < blockIdx.x ? c : 0u;
        }
      }
    }
    uint32_t total;
    const uint32_t first = run + scan_threads(all, part, total);
    run += total;
    if (e < ids) {
      if (blockIdx.x == 0) g.offsets[e] = first;               // offsets[E]: where the dropped pairs begin
      uint32_t r = first + before;
#pragma unroll
      for (int w = 0; w < kPlanWaves; ++w) {
        const uint32_t c = at[w * ids + e];
        at[w * ids + e] = r;
        r += c;
      }
    }
  }
  __syncthreads();
  // 64 pairs at a time: a pair's rank is its wave's running rank plus the equal ids in lower lanes
  int bits = 0;
  while ((1u << bits) < ids) ++bits;
  for (uint32_t f0 = begin; f0 < end; f0 += 64) {
    const uint32_t f = f0 + lane;
    uint32_t t = 0, k = 0, id = 0;
    const bool in = f < end;
    if (in) id = id_of(g, f, t, k);
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((id >> b) & 1u);
      same &= (id >> b) & 1u ? set : ~set;
    }
    const uint64_t below = same & ((1ull << lane) - 1);
    if (in) {
      const uint32_t slot = mine[id] + (uint32_t)__popcll(below);
      g.slots[(size_t)t * g.top + k] = (int32_t)slot;
      g.rows[slot] = (int32_t)t;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (!below) mine[id] += (uint32_t)__popcll(same);        // its lowest lane, after every lane's read
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// ---------------------------------------------------------------- rows
struct RowsArgs {
  const void* x;          // sort: x; combine: o
  int64_t ldx;
  const void* dy;         // combine's backward pass
  int64_t lddy;
  const void* w;          // [tokens][top] contiguous, or null: ones
  int w_type;
  const int32_t* slots;
  const int64_t* end;     // offsets[E]
  int64_t pairs;
  void* y;                // sort: s; combine: y; backward: do or null
  int64_t ldy;
  void* dw;               // backward, or null
  uint32_t tokens, top;
  int64_t cols;
  FastDiv chunks;         // 16-byte chunks per row
};

template <class T> struct Piece {
  static constexpr int N = 16 / sizeof(typename T::raw);
  typename T::raw v[N];
};
// 16 bytes of a row with `left` elements from p on, zeros past its end
template <class T>
__device__ __forceinline__ Piece<T> load_piece(const typename T::raw* p, int64_t left) {
  Piece<T> c;
  if (left >= Piece<T>::N) {
    __builtin_memcpy(&c, p, 16);
  } else {
#pragma unroll
    for (int e = 0; e < Piece<T>::N; ++e) c.v[e] = e < left ? p[e] : typename T::raw(0);
  }
  return c;
}
template <class T>
__device__ __forceinline__ void store_piece(typename T::raw* p, const Piece<T>& c, int64_t left) {
  if (left >= Piece<T>::N) {
    __builtin_memcpy(p, &c, 16);
  } else {
#pragma unroll
    for (int e = 0; e < Piece<T>::N; ++e)
      if (e < left) p[e] = c.v[e];
  }
}
__device__ __forceinline__ float weight_of(const RowsArgs& g, int64_t i) {
  if (!g.w) return 1.f;
  if (g.w_type == MI355Q_F32) return static_cast<const float*>(g.w)[i];
  const uint16_t v = static_cast<const uint16_t*>(g.w)[i];
  return g.w_type == MI355Q_BF16 ? Bf16::load(v) : F16::load(v);
}

// A thread takes 16 bytes of one token: loaded once, stored `top` times.
template <class T>
__global__ __launch_bounds__(256) void moe_sort_kernel(RowsArgs g) {
  using raw = typename T::raw;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint64_t t = i / g.chunks.d;
  if (t >= g.tokens) return;
  const int64_t c = (int64_t)(i - t * g.chunks.d) * Piece<T>::N, left = g.cols - c;
  const int64_t end = *g.end;
  const Piece<T> v = load_piece<T>(static_cast<const raw*>(g.x) + t * g.ldx + c, left);
  for (uint32_t k = 0; k < g.top; ++k) {
    const int64_t s = g.slots[t * g.top + k];
    if ((uint64_t)s >= (uint64_t)g.pairs) continue;
    store_piece<T>(static_cast<raw*>(g.y) + s * g.ldy + c, s < end ? v : Piece<T>{}, left);
  }
}

// A thread takes 16 bytes of one token's sum.
template <class T>
__global__ __launch_bounds__(256) void moe_combine_kernel(RowsArgs g) {
  using raw = typename T::raw;
  constexpr int N = Piece<T>::N;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint64_t t = i / g.chunks.d;
  if (t >= g.tokens) return;
  const int64_t c = (int64_t)(i - t * g.chunks.d) * N, left = g.cols - c;
  const int64_t end = *g.end;
  float acc[N] = {};
  for (uint32_t k = 0; k < g.top; ++k) {
    const int64_t s = g.slots[t * g.top + k];
    if (s >= end || (uint64_t)s >= (uint64_t)g.pairs) continue;
    const float w = weight_of(g, t * g.top + k);
    const Piece<T> v = load_piece<T>(static_cast<const raw*>(g.x) + s * g.ldx + c, left);
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = fmaf(w, T::load(v.v[e]), acc[e]);
  }
  Piece<T> o;
#pragma unroll
  for (int e = 0; e < N; ++e) o.v[e] = T::store(acc[e]);
  store_piece<T>(static_cast<raw*>(g.y) + t * g.ldy + c, o, left);
}

// A workgroup takes one token.
template <class T>
__global__ __launch_bounds__(256) void moe_combine_backward_kernel(RowsArgs g) {
  using raw = typename T::raw;
  constexpr int N = Piece<T>::N;
  __shared__ float sums[4];
  const int64_t t = blockIdx.x;
  const int64_t end = *g.end;
  for (uint32_t k = 0; k < g.top; ++k) {
    const int64_t s = g.slots[t * g.top + k];
    const bool in = (uint64_t)s < (uint64_t)g.pairs, kept = in && s < end;
    const float w = kept ? weight_of(g, t * g.top + k) : 0.f;
    float dot = 0.f;
    for (int64_t c = threadIdx.x * N; c < g.cols; c += 256 * N) {
      const int64_t left = g.cols - c;
      const Piece<T> d = load_piece<T>(static_cast<const raw*>(g.dy) + t * g.lddy + c, left);
      if (g.dw && kept) {
        const Piece<T> v = load_piece<T>(static_cast<const raw*>(g.x) + s * g.ldx + c, left);
#pragma unroll
        for (int e = 0; e < N; ++e) dot = fmaf(T::load(v.v[e]), T::load(d.v[e]), dot);
      }
      if (g.y && in) {
        Piece<T> o;
#pragma unroll
        for (int e = 0; e < N; ++e) o.v[e] = kept ? T::store(w * T::load(d.v[e])) : typename T::raw(0);
        store_piece<T>(static_cast<raw*>(g.y) + s * g.ldy + c, o, left);
      }
    }
    if (g.dw) {
#pragma unroll
      for (int m = 32; m; m >>= 1) dot += __shfl_xor(dot, m);
      if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = dot;
      __syncthreads();
      if (threadIdx.x == 0) {
        const float v = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        const int64_t o = t * g.top + k;
        if (g.w_type == MI355Q_F32) static_cast<float*>(g.dw)[o] = v;
        else static_cast<uint16_t*>(g.dw)[o] = g.w_type == MI355Q_BF16 ? Bf16::store(v) : F16::store(v);
      }
      __syncthreads();
    }
  }
}

static uint32_t plan_chunk(uint64_t pairs) {
  const uint64_t step = 64 * kPlanWaves, fair = (pairs + kPlanGroups - 1) / kPlanGroups;
  const uint64_t chunk = (fair + step - 1) / step * step;
  return (uint32_t)(chunk > kPlanChunk ? chunk : kPlanChunk);
}

static int check_rows(const RowsArgs& g, int64_t tokens, int64_t top, int64_t cols, int dtype) {
  MQ_CHECK_ARG(tokens >= 0 && top > 0 && cols > 0 && tokens <= INT32_MAX / top,
               "moe: need tokens >= 0, top > 0, cols > 0 and fewer than 2^31 pairs, got %lld, %lld and %lld",
               (long long)tokens, (long long)top, (long long)cols);
  MQ_CHECK_ARG(known_dtype(dtype), "moe: unknown dtype %d", dtype);
  MQ_CHECK_ARG(!g.w || known_dtype(g.w_type), "moe: unknown dtype %d of the weights", g.w_type);
  if (tokens == 0) return MI355Q_OK;
  MQ_CHECK_ARG(g.slots && g.end, "moe: slots and offsets must not be null");
  return MI355Q_OK;
}

// launches `kernel`, a thread per 16 bytes of a token's row
template <class Fn>
static int launch_rows(RowsArgs& g, int64_t tokens, int64_t cols, mi355q_dtype dt, Fn&& kernel) {
  const int64_t chunks = (cols * dtype_size(dt) + 15) / 16;
  MQ_CHECK_ARG(chunks <= INT32_MAX, "moe: rows of %lld columns are too wide", (long long)cols);
  const int64_t blocks = (tokens * chunks + 255) / 256;
  MQ_CHECK_ARG(blocks <= INT32_MAX, "moe: %lld rows of %lld columns are too many", (long long)tokens, (long long)cols);
  g.chunks = {(uint32_t)chunks, 0, 0};
  with_dtype(dt, [&](auto type) { kernel(type, dim3((unsigned)blocks)); });
  MQ_LAUNCH_CHECK();
  return MI355Q_OK;
}

}  // namespace mi355q

using namespace mi355q;

extern "C" {

size_t mi355q_moe_plan_workspace_size(int64_t tokens, int64_t top, int64_t experts) {
  if (tokens <= 0 || top <= 0 || experts <= 0 || experts > kMaxExperts || tokens > INT32_MAX / top) return 0;
  const uint64_t pairs = (uint64_t)tokens * top, chunk = plan_chunk(pairs), n = (pairs + chunk - 1) / chunk;
  return n > 1 ? n * (experts + 1) * sizeof(uint32_t) : 0;
}

int mi355q_moe_plan(const void* ids_dev, int id_bits, int64_t tokens, int64_t top, int64_t ld_ids, int64_t experts,
                    int32_t* rows_dev, int32_t* slots_dev, int64_t* offsets_dev, void* workspace_dev,
                    size_t workspace_bytes, void* stream) {
  MQ_CHECK_ARG(id_bits == 32 || id_bits == 64, "moe_plan: ids must have 32 or 64 bits, got %d", id_bits);
  MQ_CHECK_ARG(tokens >= 0 && top > 0 && tokens <= INT32_MAX / top,
               "moe_plan: need tokens >= 0, top > 0 and fewer than 2^31 pairs, got %lld and %lld", (long long)tokens,
               (long long)top);
  MQ_CHECK_ARG(experts > 0, "moe_plan: experts must be positive, got %lld", (long long)experts);
  if (experts > kMaxExperts) {
    set_error("moe_plan: at most %d experts, got %lld", kMaxExperts, (long long)experts);
    return MI355Q_UNSUPPORTED;
  }
  MQ_CHECK_ARG(offsets_dev, "moe_plan: offsets must not be null");
  MQ_CHECK_ARG(tokens == 0 || (ids_dev && rows_dev && slots_dev), "moe_plan: a null operand");
  MQ_CHECK_ARG(tokens <= 1 || ld_ids >= top, "moe_plan: ids' rows overlap (pitch %lld)", (long long)ld_ids);
  const size_t need = mi355q_moe_plan_workspace_size(tokens, top, experts);
  MQ_CHECK_ARG(workspace_bytes >= need && (need == 0 || workspace_dev), "moe_plan: workspace too small (%zu of %zu)",
               workspace_bytes, need);
  const uint32_t pairs = (uint32_t)(tokens * top);
  PlanArgs g = {ids_dev, id_bits == 64, ld_ids, tokens ? (uint32_t)tokens : 1u, (uint32_t)top, pairs,
                (uint32_t)experts, plan_chunk(pairs), rows_dev, slots_dev, offsets_dev,
                static_cast<uint32_t*>(workspace_dev)};
  const size_t lds = (size_t)(experts + 1) * sizeof(uint32_t);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned groups = need ? (pairs + g.chunk - 1) / g.chunk : 1;
  if (groups == 1) {
    hipLaunchKernelGGL((moe_place_kernel<true>), dim3(1), dim3(kPlanThreads), kPlanWaves * lds, st, g);
  } else {
    hipLaunchKernelGGL(moe_count_kernel, dim3(groups), dim3(kPlanThreads), lds, st, g);
    hipLaunchKernelGGL((moe_place_kernel<false>), dim3(groups), dim3(kPlanThreads), kPlanWaves * lds, st, g);
  }
  MQ_LAUNCH_CHECK();
  return MI355Q_OK;
}

int mi355q_moe_sort(const void* x_dev, mi355q_dtype dtype, int64_t tokens, int64_t top, int64_t cols, int64_t ldx,
                    const int32_t* slots_dev, const int64_t* end_dev, void* y_dev, int64_t ldy, void* stream) {
  RowsArgs g = {x_dev, ldx, nullptr, 0, nullptr, 0, slots_dev, end_dev, tokens * top, y_dev, ldy, nullptr, (uint32_t)tokens,
                (uint32_t)top, cols, {}};
  const int rc = check_rows(g, tokens, top, cols, dtype);
  if (rc != MI355Q_OK || tokens == 0) return rc;
  MQ_CHECK_ARG(x_dev && y_dev, "moe_sort: a null operand");
  MQ_CHECK_ARG((tokens <= 1 || ldx >= 0) && (tokens * top <= 1 || ldy >= cols), "moe_sort: rows overlap");
  return launch_rows(g, tokens, cols, dtype, [&](auto type, dim3 grid) {
    hipLaunchKernelGGL((moe_sort_kernel<decltype(type)>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), g);
  });
}

int mi355q_moe_combine(const void* x_dev, mi355q_dtype dtype, int64_t tokens, int64_t top, int64_t cols, int64_t ldx,
                       const void* weights_dev, mi355q_dtype weights_dtype, const int32_t* slots_dev,
                       const int64_t* end_dev, void* y_dev, int64_t ldy, void* stream) {
  RowsArgs g = {x_dev, ldx, nullptr, 0, weights_dev, weights_dtype, slots_dev, end_dev, tokens * top, y_dev, ldy, nullptr,
                (uint32_t)tokens, (uint32_t)top, cols, {}};
  const int rc = check_rows(g, tokens, top, cols, dtype);
  if (rc != MI355Q_OK || tokens == 0) return rc;
  MQ_CHECK_ARG(x_dev && y_dev, "moe_combine: a null operand");
  MQ_CHECK_ARG(ldx >= 0 && (tokens <= 1 || ldy >= cols), "moe_combine: rows overlap");
  return launch_rows(g, tokens, cols, dtype, [&](auto type, dim3 grid) {
    hipLaunchKernelGGL((moe_combine_kernel<decltype(type)>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), g);
  });
}

int mi355q_moe_combine_backward(const void* dy_dev, mi355q_dtype dtype, int64_t tokens, int64_t top, int64_t cols,
                                int64_t lddy, const void* x_dev, int64_t ldx, const void* weights_dev,
                                mi355q_dtype weights_dtype, const int32_t* slots_dev, const int64_t* end_dev,
                                void* dx_dev, int64_t lddx, void* dw_dev, void* stream) {
  RowsArgs g = {x_dev, ldx, dy_dev, lddy, weights_dev, weights_dtype, slots_dev, end_dev, tokens * top, dx_dev, lddx, dw_dev,
                (uint32_t)tokens, (uint32_t)top, cols, {}};
  const int rc = check_rows(g, tokens, top, cols, dtype);
  if (rc != MI355Q_OK || tokens == 0) return rc;
  MQ_CHECK_ARG(dy_dev && weights_dev && (x_dev || !dw_dev), "moe_combine_backward: a null operand");
  MQ_CHECK_ARG(ldx >= 0 && lddy >= 0 && (!dx_dev || tokens * top <= 1 || lddx >= cols),
               "moe_combine_backward: rows overlap");
  if (!dx_dev && !dw_dev) return MI355Q_OK;
  with_dtype(dtype, [&](auto type) {
    hipLaunchKernelGGL((moe_combine_backward_kernel<decltype(type)>), dim3((unsigned)tokens), dim3(256), 0,
                       static_cast<hipStream_t>(stream), g);
  });
  MQ_LAUNCH_CHECK();
  return MI355Q_OK;
}

}  // extern "C"
