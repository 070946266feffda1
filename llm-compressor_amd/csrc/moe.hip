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
#include <type_traits>

#include "fp8.h"

namespace mi355q {

// ---------------------------------------------------------------- plan
// Workgroups of 8 waves take `chunk` consecutive pairs each, a wave an eighth of
// them.  With one workgroup the plan is one launch; else a first launch leaves each
// chunk's counts per expert, and the second adds up those before its own.  Latency bounds it: one token's 8 pairs
// 3.2 us, 8192 tokens to 8 of 128 experts (32 chunks) 2.5 and 8.9 us.
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
  uint32_t run = 0;                                            // pairs of the ids before these
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
// 16 bytes of a row with `left` elements from p on, zeros past its end.  FULL: there are 16 (a branch around loads
// has them waited for one by one, so the kernels tell rows' ends apart around all of a thread's).
typedef uint32_t __attribute__((ext_vector_type(4), aligned(2))) chunk_t;
template <class T, bool FULL, bool NT>
__device__ __forceinline__ Piece<T> load_piece(const typename T::raw* p, int64_t left) {
  Piece<T> c;
  if constexpr (FULL) {
    const chunk_t* const q = reinterpret_cast<const chunk_t*>(p);
    const chunk_t v = NT ? __builtin_nontemporal_load(q) : *q;
    __builtin_memcpy(&c, &v, 16);
  } else {
#pragma unroll
    for (int e = 0; e < Piece<T>::N; ++e) c.v[e] = e < left ? p[e] : typename T::raw(0);
  }
  return c;
}
template <class T, bool FULL, bool NT>
__device__ __forceinline__ void store_piece(typename T::raw* p, const Piece<T>& c, int64_t left) {
  if constexpr (FULL) {
    chunk_t v;
    __builtin_memcpy(&v, &c, 16);
    if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<chunk_t*>(p));
    else *reinterpret_cast<chunk_t*>(p) = v;
  } else {
#pragma unroll
    for (int e = 0; e < Piece<T>::N; ++e)
      if (e < left) p[e] = c.v[e];
  }
}

// the weights of K pairs from pair i on, of which `n` are there
template <int K>
__device__ __forceinline__ void load_weights(const RowsArgs& g, int64_t i, uint32_t n, float (&w)[K]) {
  if (!g.w) {
#pragma unroll
    for (int k = 0; k < K; ++k) w[k] = 1.f;
  } else if (g.w_type == MI355Q_F32) {
#pragma unroll
    for (int k = 0; k < K; ++k) w[k] = static_cast<const float*>(g.w)[i + (k < (int)n ? k : 0)];
  } else {
    uint16_t v[K];
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = static_cast<const uint16_t*>(g.w)[i + (k < (int)n ? k : 0)];
#pragma unroll
    for (int k = 0; k < K; ++k) w[k] = g.w_type == MI355Q_BF16 ? Bf16::load(v[k]) : F16::load(v[k]);
  }
}
// the places of K pairs from pair i on, -1 for those that are not there
template <int K>
__device__ __forceinline__ void load_places(const RowsArgs& g, int64_t i, uint32_t n, int64_t (&s)[K]) {
#pragma unroll
  for (int k = 0; k < K; ++k) s[k] = g.slots[i + (k < (int)n ? k : 0)];
#pragma unroll
  for (int k = 0; k < K; ++k) s[k] = k < (int)n && (uint64_t)s[k] < (uint64_t)g.pairs ? s[k] : -1;
}
// f(std::true_type) where 16 bytes are left, else f(std::false_type)
template <class Fn>
__device__ __forceinline__ void by_fullness(bool full, Fn&& f) {
  if (full) f(std::true_type{});
  else f(std::false_type{});
}

// The kernels below take K of a token's pairs at a time, whose rows are in flight together.
//
// A thread takes 16 bytes of one token: loaded once, stored `top` times.
// NT: what moves once bypasses the caches.  8192 tokens of 2048 bf16 to 8 experts, 302 MB: 54 to 60 us, 5.0 to 5.6 TB/s.
template <class T, int K, bool NT>
__global__ __launch_bounds__(256) void moe_sort_kernel(RowsArgs g) {
  using raw = typename T::raw;
  const uint32_t i = blockIdx.x * 256u + threadIdx.x, t = div(i, g.chunks);
  if (t >= g.tokens) return;
  const int64_t c = (int64_t)(i - t * g.chunks.d) * Piece<T>::N, left = g.cols - c;
  const int64_t end = *g.end;
  by_fullness(left >= Piece<T>::N, [&](auto full) __attribute__((always_inline)) {
    constexpr bool FULL = decltype(full)::value;
    const Piece<T> v = load_piece<T, FULL, NT>(static_cast<const raw*>(g.x) + t * g.ldx + c, left);
    for (uint32_t k0 = 0; k0 < g.top; k0 += K) {
      int64_t s[K];
      load_places(g, (int64_t)t * g.top + k0, g.top - k0, s);
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (s[k] >= 0)
          store_piece<T, FULL, NT>(static_cast<raw*>(g.y) + s[k] * g.ldy + c, s[k] < end ? v : Piece<T>{}, left);
    }
  });
}

// A thread takes 16 bytes of one token's sum; the K rows' loads are what keeps the memory busy.  8192 tokens of 2048
// bf16 from 8 experts: 52 to 54 us, 5.6 to 5.8 TB/s.  (Row after row and without going around the caches sort and
// combine took 179 and 292 us there with their gradients, now 124 and 160.)
template <class T, int K, bool NT>
__global__ __launch_bounds__(256) void moe_combine_kernel(RowsArgs g) {
  using raw = typename T::raw;
  constexpr int N = Piece<T>::N;
  const uint32_t i = blockIdx.x * 256u + threadIdx.x, t = div(i, g.chunks);
  if (t >= g.tokens) return;
  const int64_t c = (int64_t)(i - t * g.chunks.d) * N, left = g.cols - c;
  const int64_t end = *g.end;
  by_fullness(left >= N, [&](auto full) __attribute__((always_inline)) {
    constexpr bool FULL = decltype(full)::value;
    float acc[N] = {};
    for (uint32_t k0 = 0; k0 < g.top; k0 += K) {
      int64_t s[K];
      float w[K];
      Piece<T> v[K];
      load_places(g, (int64_t)t * g.top + k0, g.top - k0, s);
      load_weights(g, (int64_t)t * g.top + k0, g.top - k0, w);
      // rows that take no part: the first one is read, and counts as zeros
#pragma unroll
      for (int k = 0; k < K; ++k) {
        s[k] = s[k] < end ? s[k] : -1;
        v[k] = load_piece<T, FULL, NT>(static_cast<const raw*>(g.x) + (s[k] < 0 ? 0 : s[k]) * g.ldx + c, left);
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float f = s[k] < 0 ? 0.f : w[k];
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = fmaf(f, s[k] < 0 ? 0.f : T::load(v[k].v[e]), acc[e]);
      }
    }
    Piece<T> o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.v[e] = T::store(acc[e]);
    store_piece<T, FULL, false>(static_cast<raw*>(g.y) + t * g.ldy + c, o, left);
  });
}

// Sums of K (2, 4 or 8) values over the wave, value k in the lanes with l % K = k: at each of log2 K steps a lane
// hands half of its values to its partner and adds the partner's other half; the last steps add what is left.
template <int K>
__device__ __forceinline__ float sum_values(float (&v)[K], int lane) {
#pragma unroll
  for (int n = K / 2, d = 1; n; n >>= 1, d <<= 1) {
    const bool up = lane & d;
#pragma unroll
    for (int k = 0; k < n; ++k) {
      // value bits go to lane bits from the lowest on: of the pair (2 k, 2 k + 1) the lane keeps the one of its bit
      const float keep = up ? v[2 * k + 1] : v[2 * k], give = up ? v[2 * k] : v[2 * k + 1];
      v[k] = keep + __shfl_xor(give, d);
    }
  }
  float s = v[0];
#pragma unroll
  for (int d = K; d < 64; d <<= 1) s += __shfl_xor(s, d);
  return s;
}

// W waves take one token: they read its gradient and its experts' rows, write the rows' gradients and add up the
// weights' over the row.  8192 tokens of 2048 bf16, 8 experts, 570 MB: 106 to 113 us, 5.0 to 5.4 TB/s.  Rows of up to
// 1 KB have a wave per token, longer ones a workgroup, so that few tokens fill the CUs too.
template <class T, int K, int W, bool NT>
__global__ __launch_bounds__(256) void moe_combine_backward_kernel(RowsArgs g) {
  using raw = typename T::raw;
  constexpr int N = Piece<T>::N, PER = 4 / W;            // tokens per workgroup
  __shared__ float sums[4][K];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * PER + wave / W;
  const bool in = t < g.tokens;
  const int64_t end = *g.end;
  for (uint32_t k0 = 0; k0 < g.top; k0 += K) {
    int64_t s[K], from[K];
    float w[K], dot[K] = {};
    load_places(g, (in ? t : 0) * g.top + k0, g.top - k0, s);
    load_weights(g, (in ? t : 0) * g.top + k0, g.top - k0, w);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      from[k] = s[k] < end ? s[k] : -1;
      w[k] = from[k] < 0 ? 0.f : w[k];
    }
    if (in)
      for (int64_t c = ((wave % W) * 64 + lane) * N; c < g.cols; c += 64 * W * N) {
        const int64_t left = g.cols - c;
        by_fullness(left >= N, [&](auto full) __attribute__((always_inline)) {
          constexpr bool FULL = decltype(full)::value;
          const Piece<T> d = load_piece<T, FULL, false>(static_cast<const raw*>(g.dy) + t * g.lddy + c, left);
          Piece<T> v[K];
          if (g.dw) {                                     // rows that take no part: the first one, as zeros
#pragma unroll
            for (int k = 0; k < K; ++k)
              v[k] = load_piece<T, FULL, NT>(static_cast<const raw*>(g.x) + (from[k] < 0 ? 0 : from[k]) * g.ldx + c, left);
          }
          if (g.y) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
              if (s[k] < 0) continue;
              Piece<T> o;
#pragma unroll
              for (int e = 0; e < N; ++e) o.v[e] = from[k] < 0 ? typename T::raw(0) : T::store(w[k] * T::load(d.v[e]));
              store_piece<T, FULL, NT>(static_cast<raw*>(g.y) + s[k] * g.ldy + c, o, left);
            }
          }
          if (g.dw) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
              for (int e = 0; e < N; ++e)
                dot[k] = fmaf(from[k] < 0 ? 0.f : T::load(v[k].v[e]), from[k] < 0 ? 0.f : T::load(d.v[e]), dot[k]);
          }
        });
      }
    if (!g.dw) continue;
    float v = sum_values<K>(dot, lane);
    if constexpr (W > 1) {
      if (lane < K) sums[wave][lane] = v;
      __syncthreads();
      v = sums[0][lane & (K - 1)];
#pragma unroll
      for (int i = 1; i < W; ++i) v += sums[i][lane & (K - 1)];
      __syncthreads();
      if (wave) continue;
    }
    if (in && lane < K && k0 + lane < g.top) {
      const int64_t o = t * g.top + k0 + lane;
      if (g.w_type == MI355Q_F32) static_cast<float*>(g.dw)[o] = v;
      else static_cast<uint16_t*>(g.dw)[o] = g.w_type == MI355Q_BF16 ? Bf16::store(v) : F16::store(v);
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

// f(std::integral_constant) of the pairs that are taken at a time
template <class Fn>
static void by_top(int64_t top, Fn&& f) {
  if (top <= 2) f(std::integral_constant<int, 2>{});
  else if (top <= 4) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 8>{});
}

// Experts' rows of more bytes than this, half of the last-level cache, go around the caches: 8192 tokens to 8 experts
// of 2048 bf16 (256 MB) combine 60 -> 54 us, their gradients 120 -> 113, sort 59 -> 54.
constexpr int64_t kCached = 128ll << 20;

// launches `kernel(type, grid, g)`, a thread per 16 bytes of a token's row, over as many tokens at a time as
// the kernels' 31 bits count
template <class Fn>
static int launch_rows(RowsArgs g, int64_t tokens, int64_t cols, mi355q_dtype dt, int64_t row_x, int64_t row_y,
                       Fn&& kernel) {
  const int64_t chunks = (cols * dtype_size(dt) + 15) / 16, most = INT32_MAX / 2;
  MQ_CHECK_ARG(chunks <= most, "moe: rows of %lld columns are too wide", (long long)cols);
  g.chunks = fast_div((uint32_t)chunks);
  const int64_t step = most / chunks;
  for (int64_t t = 0; t < tokens; t += step) {
    RowsArgs part = g;
    part.tokens = (uint32_t)(tokens - t < step ? tokens - t : step);
    part.x = static_cast<const char*>(g.x) + t * row_x * dtype_size(dt);
    part.y = static_cast<char*>(g.y) + t * row_y * dtype_size(dt);
    part.slots = g.slots + t * g.top;
    if (g.w) part.w = static_cast<const char*>(g.w) + t * g.top * dtype_size((mi355q_dtype)g.w_type);
    with_dtype(dt, [&](auto type) { kernel(type, dim3((unsigned)((part.tokens * chunks + 255) / 256)), part); });
    MQ_LAUNCH_CHECK();
  }
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
  RowsArgs g = {x_dev, ldx, nullptr, 0, nullptr, 0, slots_dev, end_dev, tokens * top, y_dev, ldy, nullptr,
                (uint32_t)tokens, (uint32_t)top, cols, {}};
  const int rc = check_rows(g, tokens, top, cols, dtype);
  if (rc != MI355Q_OK || tokens == 0) return rc;
  MQ_CHECK_ARG(x_dev && y_dev, "moe_sort: a null operand");
  MQ_CHECK_ARG((tokens <= 1 || ldx >= 0) && (tokens * top <= 1 || ldy >= cols), "moe_sort: rows overlap");
  const bool past = tokens * top * cols * dtype_size(dtype) > kCached;
  return launch_rows(g, tokens, cols, dtype, ldx, 0, [&](auto type, dim3 grid, const RowsArgs& part) {
    using T = decltype(type);
    hipStream_t st = static_cast<hipStream_t>(stream);
    by_top(top, [&](auto k) {
      constexpr int K = decltype(k)::value;
      if (past) hipLaunchKernelGGL((moe_sort_kernel<T, K, true>), grid, dim3(256), 0, st, part);
      else hipLaunchKernelGGL((moe_sort_kernel<T, K, false>), grid, dim3(256), 0, st, part);
    });
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
  const bool past = tokens * top * cols * dtype_size(dtype) > kCached;
  return launch_rows(g, tokens, cols, dtype, 0, ldy, [&](auto type, dim3 grid, const RowsArgs& part) {
    by_top(top, [&](auto k) {
      using T = decltype(type);
      constexpr int K = decltype(k)::value;
      hipStream_t st = static_cast<hipStream_t>(stream);
      if (past) hipLaunchKernelGGL((moe_combine_kernel<T, K, true>), grid, dim3(256), 0, st, part);
      else hipLaunchKernelGGL((moe_combine_kernel<T, K, false>), grid, dim3(256), 0, st, part);
    });
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
  const bool past = dx_dev && tokens * top * cols * dtype_size(dtype) > kCached;
  const bool wide = cols * dtype_size(dtype) > 64 * 16;
  // a launch has fewer than 2^32 threads: 2^22 tokens, a workgroup of 256 each where rows are wide
  constexpr int64_t step = 1 << 22;
  for (int64_t t = 0; t < tokens; t += step) {
    RowsArgs part = g;
    part.tokens = (uint32_t)(tokens - t < step ? tokens - t : step);
    part.dy = static_cast<const char*>(dy_dev) + t * lddy * dtype_size(dtype);
    part.w = static_cast<const char*>(weights_dev) + t * top * dtype_size(weights_dtype);
    part.slots = slots_dev + t * top;
    if (dw_dev) part.dw = static_cast<char*>(dw_dev) + t * top * dtype_size(weights_dtype);
    const dim3 grid(wide ? part.tokens : (part.tokens + 3) / 4), block(256);
    with_dtype(dtype, [&](auto type) {
      using T = decltype(type);
      hipStream_t st = static_cast<hipStream_t>(stream);
      by_top(top, [&](auto k) {
        constexpr int K = decltype(k)::value;
        if (wide && past) hipLaunchKernelGGL((moe_combine_backward_kernel<T, K, 4, true>), grid, block, 0, st, part);
        else if (wide) hipLaunchKernelGGL((moe_combine_backward_kernel<T, K, 4, false>), grid, block, 0, st, part);
        else hipLaunchKernelGGL((moe_combine_backward_kernel<T, K, 1, false>), grid, block, 0, st, part);
      });
    });
    MQ_LAUNCH_CHECK();
  }
  return MI355Q_OK;
}

}  // extern "C"
