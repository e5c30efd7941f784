// Routing of tokens to experts, the row order of the routed choices, the
// weighted sum of the experts' rows back to tokens, and the 8-bit rounding of
// token rows. The products between routing and sum are in grouped_tc.cu.
//
// T tokens choose k of E experts each; choice a = t * k + j. Row r of the
// grouped order holds choice order[r]; expert e owns rows offsets[e] to
// offsets[e + 1]; position[a] is the row of choice a. A choice of no expert
// (-1) has no row, and the rows from offsets[E] on are empty.
#include <cuda_fp16.h>

#include <cfloat>

#include "common.cuh"
#include "experts.cuh"

namespace es {
namespace {

constexpr unsigned kFull = 0xffffffffu;

// ------------------------------------------------------------------ routing
//
// One warp per token, the token's logits in registers (lane l holds experts
// l, l + 32, ...). The k largest are found one after the other: each lane's
// largest, one warp reduction of the order-preserving bits, one of the lowest
// index among equals. With m the largest logit, w_j = exp(l_j - m) / sum,
// where the sum runs over the chosen (renorm) or over all experts. -inf is a
// masked expert and is never chosen. NaN is never chosen either, and makes
// every weight of its token NaN. Bound by launch latency for decode steps (3 us)
// and by the selection's instructions for long prompts: 32768 tokens, 128
// experts, k 8 take 18 us, the 17 MB of logits alone 2.6 us.

// Bits whose unsigned order is the order of the floats; 0 for -inf and NaN.
// x + 0 makes -0 equal to +0, so that ties go by index alone.
__device__ __forceinline__ uint32_t order_bits(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float from_order_bits(uint32_t u) {
  return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}

template <typename T, int PER>
__device__ __forceinline__ void load_logits(const T* row, int E, float (&v)[PER]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    v[i] = e < E ? to_f32(row[e]) : -INFINITY;
  }
}

template <int PER>
__device__ __forceinline__ float row_max(const float (&v)[PER]) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < PER; ++i) m = fmaxf(m, v[i]);
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
  return m;
}

__device__ __forceinline__ float warp_sum(float s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
  return s;
}

template <typename T, int PER>
__global__ void __launch_bounds__(128) route_kernel(const T* logits, int64_t ntok, int E, int64_t stride, int k,
                                                    int renorm, float* weights, int32_t* experts) {
  const int lane = threadIdx.x & 31;
  const int64_t t = blockIdx.x * 4LL + (threadIdx.x >> 5);
  if (t >= ntok) return;
  float v[PER];
  load_logits<T, PER>(logits + t * stride, E, v);
  uint32_t key[PER];
  bool nan = false;
  float all = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    key[i] = order_bits(v[i]);
    nan |= v[i] != v[i];
  }
  const float m = row_max<PER>(v);
  if (!renorm) {
#pragma unroll
    for (int i = 0; i < PER; ++i) all += key[i] ? expf(v[i] - m) : 0.0f;
    all = warp_sum(all);
  }
  const bool poison = __any_sync(kFull, nan);
  // each lane offers its largest; the lane whose offer is taken looks again.
  // Choice j ends in lane j (k <= 32).
  uint32_t best = 0, mine_bits = 0;
  int slot = 0, chosen = -1;
  auto look = [&] {
    best = key[0];
    slot = 0;
#pragma unroll
    for (int i = 1; i < PER; ++i)
      if (key[i] > best) {
        best = key[i];
        slot = i;
      }
  };
  look();
  for (int j = 0; j < k; ++j) {
    const uint32_t top = __reduce_max_sync(kFull, best);
    if (top == 0) break;  // nothing left but masked experts
    const int at = lane + 32 * slot;
    const int e = __reduce_min_sync(kFull, best == top ? at : 0x7fffffff);
    if (lane == j) {
      chosen = e;
      mine_bits = top;
    }
    if (at == e) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i == slot) key[i] = 0;
      look();
    }
  }
  const float mine = chosen >= 0 ? expf(from_order_bits(mine_bits) - m) : 0.0f;
  const float total = renorm ? warp_sum(mine) : all;
  if (lane < k) {
    const float w = chosen >= 0 ? mine / total : 0.0f;
    weights[t * k + lane] = poison ? NAN : w;
    experts[t * k + lane] = chosen;
  }
}

// dl_i = w_i (g_i - d), d = sum_j w_j g_j, for the chosen experts (whose w_i
// is p_i); for the others 0 (renorm), or -p_i d with p recomputed from the
// logits. Every dlogit is written as if not chosen, in whole rows, and then
// the chosen ones over it.
template <typename T, int PER>
__global__ void __launch_bounds__(128) route_grad_kernel(const T* logits, int64_t ntok, int E, int64_t stride, int k,
                                                         int renorm, const float* weights, const int32_t* experts,
                                                         const float* dweights, T* dlogits) {
  const int lane = threadIdx.x & 31;
  const int64_t t = blockIdx.x * 4LL + (threadIdx.x >> 5);
  if (t >= ntok) return;
  float w = 0.0f, g = 0.0f;
  int e = -1;
  if (lane < k) {
    w = weights[t * k + lane];
    e = experts[t * k + lane];
    g = e >= 0 ? dweights[t * k + lane] : 0.0f;
  }
  const float d = warp_sum(w * g);
  T* out = dlogits + t * static_cast<int64_t>(E);
  if (renorm) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 32 * i < E) out[lane + 32 * i] = from_f32<T>(0.0f);
  } else {
    float v[PER];
    load_logits<T, PER>(logits + t * stride, E, v);
    const float m = row_max<PER>(v);
    float all = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      // NaN logits keep their NaN here, masked ones add nothing
      v[i] = v[i] == -INFINITY ? 0.0f : expf(v[i] - m);
      all += v[i];
    }
    all = warp_sum(all);
    const float f = all > 0.0f || all != all ? -d / all : 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 32 * i < E) out[lane + 32 * i] = from_f32<T>(v[i] * f);
  }
  __syncwarp();
  if (e >= 0) out[e] = from_f32<T>(w * (g - d));
}

template <typename T>
int route_typed(const void* logits, int64_t T_, int E, int64_t stride, int k, int renorm, float* weights,
                int32_t* experts, const float* dweights, void* dlogits, cudaStream_t s) {
  const T* x = static_cast<const T*>(logits);
  const int64_t blocks = (T_ + 3) / 4;
#define ES_ROUTE(PER)                                                                                            \
  if (E <= 32 * PER) {                                                                                           \
    if (dlogits)                                                                                                 \
      ES_LAUNCH((route_grad_kernel<T, PER>), static_cast<unsigned>(blocks), 128, 0, s, x, T_, E, stride, k,       \
                renorm, weights, experts, dweights, static_cast<T*>(dlogits));                                   \
    else                                                                                                         \
      ES_LAUNCH((route_kernel<T, PER>), static_cast<unsigned>(blocks), 128, 0, s, x, T_, E, stride, k, renorm,    \
                weights, experts);                                                                               \
    return ES_OK;                                                                                                \
  }
  ES_ROUTE(1)
  ES_ROUTE(2)
  ES_ROUTE(4)
  ES_ROUTE(8)
  ES_ROUTE(16)
  ES_ROUTE(32)
#undef ES_ROUTE
  return ES_ERR_UNSUPPORTED;
}

// ----------------------------------------------------------------- row order
//
// A stable counting sort of the choices by expert ("no expert" sorts last, as
// expert E). Up to 2048 choices: one CTA, one launch. Else the choices are cut
// into chunks: one launch counts each chunk's experts, a second places them.
// Every chunk adds up the counts of the chunks before it, while there are few
// (kPlanDirect); else a launch in between does that for all. Within a CTA each
// warp owns a consecutive run of choices, 32 at a time; a choice's rank is the
// warp's earlier choices of the same expert (match + popcount), so the order
// never depends on the schedule. Bound by latency: each choice is read once, and
// 262144 choices of 128 experts take three launches of 4, 3 and 8 us.

constexpr int kPlanThreads = 512;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanChunk = 2048;  // choices of one CTA
constexpr int kPlanItems = kPlanChunk / kPlanThreads;
constexpr int kPlanDirect = 64;   // chunks whose counts a CTA adds up by itself

__device__ __forceinline__ int expert_of(const int32_t* experts, int64_t a, int E, bool& bad) {
  const int e = experts[a];
  if (e < -1 || e >= E) bad = true;
  return e >= 0 && e < E ? e : E;
}

__global__ void __launch_bounds__(kPlanThreads) plan_count_kernel(const int32_t* experts, int64_t n, int E,
                                                                  int32_t* counts) {
  extern __shared__ int32_t hist[];
  for (int i = threadIdx.x; i <= E; i += kPlanThreads) hist[i] = 0;
  __syncthreads();
  const int64_t c0 = blockIdx.x * static_cast<int64_t>(kPlanChunk);
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kPlanItems; ++i) {
    const int64_t a = c0 + i * kPlanThreads + threadIdx.x;
    if (a < n) atomicAdd(&hist[expert_of(experts, a, E, bad)], 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i <= E; i += kPlanThreads) counts[blockIdx.x * static_cast<int64_t>(E + 1) + i] = hist[i];
}

// Replaces every chunk's count of expert blockIdx.x by the count of the chunks
// before it, and writes the total behind the last chunk's.
__global__ void __launch_bounds__(kPlanThreads) plan_scan_kernel(int32_t* counts, int64_t chunks, int E) {
  __shared__ int32_t sums[kPlanWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e = blockIdx.x;
  int run = 0;
  for (int64_t c0 = 0; c0 < chunks; c0 += kPlanThreads) {
    const int64_t c = c0 + threadIdx.x;
    const int v = c < chunks ? counts[c * (E + 1) + e] : 0;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(kFull, s, o);
      if (lane >= o) s += u;
    }
    if (lane == 31) sums[warp] = s;
    __syncthreads();
    int before = run;
    for (int w = 0; w < kPlanWarps; ++w) {
      if (w < warp) before += sums[w];
      run += sums[w];
    }
    if (c < chunks) counts[c * (E + 1) + e] = before + s - v;
    __syncthreads();
  }
  if (threadIdx.x == 0) counts[chunks * (E + 1) + e] = run;
}

// counts: of every chunk; nullptr: this CTA is the only chunk; scanned: as
// plan_scan_kernel leaves them.
__global__ void __launch_bounds__(kPlanThreads) plan_place_kernel(const int32_t* experts, int64_t n, int E,
                                                                  const int32_t* counts, int scanned,
                                                                  int32_t* offsets, int32_t* order,
                                                                  int32_t* position, int32_t* err) {
  extern __shared__ int32_t sm[];
  const int E1 = E + 1;
  int32_t* cnt = sm;                       // [kPlanWarps][E1]: counts, then first row of (warp, expert)
  int32_t* before = sm + kPlanWarps * E1;  // [E1] rows of this expert in the chunks before
  int32_t* total = before + E1;            // [E1] rows of this expert in all, then its first row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c0 = blockIdx.x * static_cast<int64_t>(kPlanChunk);
  const int m = static_cast<int>(min(n - c0, static_cast<int64_t>(kPlanChunk)));
  const int per = m <= kPlanThreads ? 32 : kPlanItems * 32;  // a warp's run of choices
  int e[kPlanItems], rank[kPlanItems];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kPlanItems; ++i) {
    const int a = warp * per + i * 32 + lane;
    e[i] = i * 32 < per && a < m ? expert_of(experts, c0 + a, E, bad) : E1;
  }
  for (int i = threadIdx.x; i < (kPlanWarps + 2) * E1; i += kPlanThreads) sm[i] = 0;
  __syncthreads();
  if (bad && err) *static_cast<volatile int32_t*>(err) = ES_ERR_INDEX;
#pragma unroll
  for (int i = 0; i < kPlanItems; ++i) {
    if (warp * per + i * 32 >= m || i * 32 >= per) break;  // the whole warp
    const unsigned same = __match_any_sync(kFull, e[i]);
    const int had = e[i] < E1 ? cnt[warp * E1 + e[i]] : 0;
    rank[i] = had + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (e[i] < E1 && lane == __ffs(same) - 1) cnt[warp * E1 + e[i]] = had + __popc(same);
    __syncwarp();
  }
  if (counts && scanned) {
    for (int x = threadIdx.x; x < E1; x += kPlanThreads) {
      before[x] = counts[blockIdx.x * static_cast<int64_t>(E1) + x];
      total[x] = counts[gridDim.x * static_cast<int64_t>(E1) + x];
    }
  } else if (counts) {
    for (int i = threadIdx.x; i < static_cast<int>(gridDim.x) * E1; i += kPlanThreads) {
      const int v = counts[i];
      if (v) {
        atomicAdd(&total[i % E1], v);
        if (i < static_cast<int>(blockIdx.x) * E1) atomicAdd(&before[i % E1], v);
      }
    }
  }
  __syncthreads();
  if (!counts) {
    for (int x = threadIdx.x; x < E1; x += kPlanThreads) {
      int all = 0;
#pragma unroll
      for (int w = 0; w < kPlanWarps; ++w) all += cnt[w * E1 + x];
      total[x] = all;
    }
    __syncthreads();
  }
  if (warp == 0) {  // exclusive sum of the totals: each expert's first row
    int run = 0;
    for (int e0 = 0; e0 < E1; e0 += 32) {
      const int x = e0 + lane;
      const int v = x < E1 ? total[x] : 0;
      int s = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(kFull, s, o);
        if (lane >= o) s += u;
      }
      if (x < E1) {
        total[x] = run + s - v;
        if (blockIdx.x == 0) offsets[x] = run + s - v;
      }
      run += __shfl_sync(kFull, s, 31);
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < E1; x += kPlanThreads) {
    int at = total[x] + before[x];
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) {
      const int v = cnt[w * E1 + x];
      cnt[w * E1 + x] = at;
      at += v;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPlanItems; ++i) {
    const int a = warp * per + i * 32 + lane;
    if (i * 32 >= per || a >= m) break;
    const int row = cnt[warp * E1 + e[i]] + rank[i];
    order[row] = e[i] < E ? static_cast<int32_t>(c0 + a) : -1;
    position[c0 + a] = e[i] < E ? row : -1;
  }
}

size_t plan_smem(int E) { return static_cast<size_t>(kPlanWarps + 2) * (E + 1) * sizeof(int32_t); }

// --------------------------------------------------- weighted sum to tokens
//
// out_t = sum_j w_tj y_pos(t,j), in fp32, rounded once. Backward in one pass:
// dy_pos(t,j) = w_tj dout_t and dw_tj = <dout_t, y_pos(t,j)>. Both are bound
// by memory: every row is read (and written) once, in 16-byte pieces, by tp
// threads a token (16384 x 4 rows of 4096 bf16: 105 us and 182 us, 6.4 and 6.6
// TB/s of their bytes).

template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Piece {
  T v[VEC];
};

constexpr int kCombineThreads = 256;

__device__ __forceinline__ int row_of(const int32_t* position, int64_t a, int64_t rows) {
  const int p = position[a];
  return p >= 0 && p < rows ? p : -1;
}

// The rows and weights of choices j0 .. of token t; none past the last token.
template <int AHEAD>
__device__ __forceinline__ void load_choices(const float* weights, const int32_t* position, int64_t t, int64_t ntok,
                                             int j0, int k, int64_t rows, int (&row)[AHEAD], float (&w)[AHEAD]) {
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    row[j] = t < ntok && j0 + j < k ? row_of(position, t * k + j0 + j, rows) : -1;
    w[j] = row[j] >= 0 ? (weights ? weights[t * k + j0 + j] : 1.0f) : 0.0f;
  }
}

// One token for tp threads. Each thread has AHEAD choices of TWO pieces in
// flight; more choices go round again. Measured on 8192 x 8, 16384 x 4 and
// 16384 x 2 rows of 4096 bf16: 6.0, 6.25 and 5.25 TB/s (more CTAs or more in
// flight a thread were slower).
template <typename T, typename U, int VEC, int AHEAD, int TWO>
__global__ void __launch_bounds__(kCombineThreads, AHEAD == 4 ? 6 : 4)
    combine_kernel(const T* y, int64_t rows, int64_t stride, const float* weights, const int32_t* position,
                   int64_t ntok, int k, int64_t D, U* out, int tp) {
  const int64_t t = blockIdx.x * static_cast<int64_t>(kCombineThreads / tp) + threadIdx.x / tp;
  if (t >= ntok) return;
  const int64_t pieces = D / VEC;
  int row[AHEAD];
  float w[AHEAD];
  load_choices<AHEAD>(weights, position, t, ntok, 0, k, rows, row, w);
  for (int64_t c0 = threadIdx.x % tp; c0 < pieces; c0 += TWO * tp) {
    float acc[TWO][VEC];
#pragma unroll
    for (int u = 0; u < TWO; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[u][i] = 0.0f;
    for (int j0 = 0; j0 < k; j0 += AHEAD) {
      if (k > AHEAD) load_choices<AHEAD>(weights, position, t, ntok, j0, k, rows, row, w);
      Piece<T, VEC> p[TWO][AHEAD];
#pragma unroll
      for (int u = 0; u < TWO; ++u)
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          const int64_t c = c0 + u * tp;
          p[u][j] = row[j] >= 0 && c < pieces ? reinterpret_cast<const Piece<T, VEC>*>(y + row[j] * stride)[c]
                                              : Piece<T, VEC>{};
        }
#pragma unroll
      for (int u = 0; u < TWO; ++u)
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[u][i] = fmaf(w[j], to_f32(p[u][j].v[i]), acc[u][i]);
    }
#pragma unroll
    for (int u = 0; u < TWO; ++u) {
      const int64_t c = c0 + u * tp;
      Piece<U, VEC> o;
#pragma unroll
      for (int i = 0; i < VEC; ++i) o.v[i] = from_f32<U>(acc[u][i]);
      if (c < pieces) reinterpret_cast<Piece<U, VEC>*>(out + t * D)[c] = o;
    }
  }
}

template <typename T, int VEC, int AHEAD>
__global__ void __launch_bounds__(kCombineThreads, AHEAD == 2 ? 6 : 4) combine_grad_kernel(
    const T* y, int64_t rows, int64_t stride, const float* weights, const int32_t* position, const int32_t* kept,
    int64_t ntok, int k, int64_t D, const T* dout, int64_t dstride, T* dy, float* dweights, int tp) {
  __shared__ float part[2][kCombineThreads / 32][AHEAD];
  const int group = threadIdx.x / tp, lane = threadIdx.x & 31;
  const int64_t step = gridDim.x * static_cast<int64_t>(kCombineThreads / tp);
  const int64_t pieces = D / VEC;
  int round = 0;
  // a CTA's groups go together: they share the barrier
  for (int64_t t0 = blockIdx.x * static_cast<int64_t>(kCombineThreads / tp); t0 < ntok; t0 += step) {
    const int64_t t = t0 + group;
    for (int j0 = 0; j0 < k; j0 += AHEAD, round ^= 1) {
      float dot[AHEAD];
      int row[AHEAD];
      float w[AHEAD];
      load_choices<AHEAD>(weights, position, t, ntok, j0, k, rows, row, w);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) dot[j] = 0.0f;
      if (t < ntok) {
        for (int64_t c = threadIdx.x % tp; c < pieces; c += tp) {
          const Piece<T, VEC> g = reinterpret_cast<const Piece<T, VEC>*>(dout + t * dstride)[c];
          Piece<T, VEC> p[AHEAD];
#pragma unroll
          for (int j = 0; j < AHEAD; ++j)
            if (row[j] >= 0) p[j] = reinterpret_cast<const Piece<T, VEC>*>(y + row[j] * stride)[c];
#pragma unroll
          for (int j = 0; j < AHEAD; ++j)
            if (row[j] >= 0) {
              Piece<T, VEC> o;
#pragma unroll
              for (int i = 0; i < VEC; ++i) {
                const float gi = to_f32(g.v[i]);
                dot[j] = fmaf(gi, to_f32(p[j].v[i]), dot[j]);
                o.v[i] = from_f32<T>(w[j] * gi);
              }
              reinterpret_cast<Piece<T, VEC>*>(dy + row[j] * D)[c] = o;
            }
        }
      }
      // the group's threads are whole warps (tp is a multiple of 32); two
      // rounds' worth of parts, so that one barrier is enough
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) dot[j] = warp_sum(dot[j]);
      if (lane == 0) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) part[round][threadIdx.x >> 5][j] = dot[j];
      }
      __syncthreads();
      const int j = threadIdx.x % tp;
      if (t < ntok && j < AHEAD && j0 + j < k) {
        float s = 0.0f;
        for (int i = 0; i < tp / 32; ++i) s += part[round][group * (tp / 32) + i][j];
        dweights[t * k + j0 + j] = row_of(position, t * k + j0 + j, rows) >= 0 ? s : 0.0f;
      }
    }
  }
  // rows of no choice
  const int64_t first = min(max(static_cast<int64_t>(*kept), int64_t{0}), rows);
  for (int64_t r = first + blockIdx.x; r < rows; r += gridDim.x)
    for (int64_t c = threadIdx.x; c < pieces; c += kCombineThreads)
      reinterpret_cast<Piece<T, VEC>*>(dy + r * D)[c] = Piece<T, VEC>{};
}

// Threads per token: enough that each takes one or two pieces, in whole warps.
int token_threads(int64_t pieces) {
  int tp = 32;
  while (tp < kCombineThreads && tp < pieces) tp *= 2;
  return tp;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// CTAs: all that are resident at once, no more than the tokens fill.
unsigned token_blocks(int64_t ntok, int tp, int resident) {
  const int64_t per = kCombineThreads / tp;
  return static_cast<unsigned>(min((ntok + per - 1) / per, static_cast<int64_t>(kSMs) * resident));
}

template <typename T, typename U, int VEC>
int combine_vec(const void* y, int64_t rows, int64_t stride, const float* weights, const int32_t* position, int64_t T_,
                int k, int64_t D, void* out, cudaStream_t s) {
  const int tp = token_threads(D / VEC / (k <= 2 ? 2 : 1));
  const int64_t per = kCombineThreads / tp;
#define ES_COMBINE(AHEAD, TWO)                                                                                    \
  ES_LAUNCH((combine_kernel<T, U, VEC, AHEAD, TWO>), static_cast<unsigned>((T_ + per - 1) / per), kCombineThreads, \
            0, s, static_cast<const T*>(y), rows, stride, weights, position, T_, k, D, static_cast<U*>(out), tp)
  if (k <= 2)
    ES_COMBINE(2, 2);
  else if (k <= 4)
    ES_COMBINE(4, 1);
  else
    ES_COMBINE(8, 1);
#undef ES_COMBINE
  return ES_OK;
}

template <typename T, typename U>
int combine_typed(const void* y, int64_t rows, int64_t stride, const float* weights, const int32_t* position,
                  int64_t T_, int k, int64_t D, void* out, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  if (D % VEC == 0 && stride % VEC == 0 && aligned16(y) && aligned16(out))
    return combine_vec<T, U, VEC>(y, rows, stride, weights, position, T_, k, D, out, s);
  return combine_vec<T, U, 1>(y, rows, stride, weights, position, T_, k, D, out, s);
}

template <typename T, int VEC>
int combine_grad_vec(const void* y, int64_t rows, int64_t stride, const float* weights, const int32_t* position,
                     const int32_t* kept, int64_t T_, int k, int64_t D, const void* dout, int64_t dstride, void* dy,
                     float* dweights, cudaStream_t s) {
  const int tp = token_threads(D / VEC);
#define ES_COMBINE(AHEAD, RESIDENT)                                                                               \
  ES_LAUNCH((combine_grad_kernel<T, VEC, AHEAD>), token_blocks(T_, tp, RESIDENT), kCombineThreads, 0, s,          \
            static_cast<const T*>(y), rows, stride, weights, position, kept, T_, k, D, static_cast<const T*>(dout), \
            dstride, static_cast<T*>(dy), dweights, tp)
  if (k <= 2)
    ES_COMBINE(2, 6);
  else
    ES_COMBINE(4, 4);
#undef ES_COMBINE
  return ES_OK;
}

template <typename T>
int combine_grad_typed(const void* y, int64_t rows, int64_t stride, const float* weights, const int32_t* position,
                       const int32_t* kept, int64_t T_, int k, int64_t D, const void* dout, int64_t dstride, void* dy,
                       float* dweights, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  if (D % VEC == 0 && stride % VEC == 0 && dstride % VEC == 0 && aligned16(y) && aligned16(dout) && aligned16(dy))
    return combine_grad_vec<T, VEC>(y, rows, stride, weights, position, kept, T_, k, D, dout, dstride, dy, dweights, s);
  return combine_grad_vec<T, 1>(y, rows, stride, weights, position, kept, T_, k, D, dout, dstride, dy, dweights, s);
}

// ------------------------------------------------------------ 8-bit rounding
//
// scale_t = max_i |x_ti| / 127 (one division rounded to nearest), q_ti =
// rint(x_ti / scale_t), kept within +-127. A row of zeros has scale 0 and q 0;
// a row with an infinity or NaN has scale NaN, so that its products are NaN
// and not a finite guess. A row is read once and its 8-bit copy written once:
// 8191 x 4096 bf16 take 25 us, 4.0 TB/s, between memory and the conversions.

constexpr int kQuantThreads = 256;

// The larger of two magnitudes; NaN where one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <int VEC>
__device__ __forceinline__ float piece_peak(const Piece<float, VEC>& p) {
  float m = fabsf(p.v[0]);
#pragma unroll
  for (int i = 1; i < VEC; ++i) m = max_nan(m, fabsf(p.v[i]));
  return m;
}
template <int VEC>
__device__ __forceinline__ float piece_peak(const Piece<__nv_bfloat16, VEC>& p) {
  if constexpr (VEC == 1) {
    return fabsf(to_f32(p.v[0]));
  } else {
    const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(p.v);
    __nv_bfloat162 m = __habs2(v[0]);
#pragma unroll
    for (int i = 1; i < VEC / 2; ++i) m = __hmax2_nan(m, __habs2(v[i]));
    return max_nan(__low2float(m), __high2float(m));
  }
}
template <int VEC>
__device__ __forceinline__ float piece_peak(const Piece<__half, VEC>& p) {
  if constexpr (VEC == 1) {
    return fabsf(to_f32(p.v[0]));
  } else {
    const __half2* v = reinterpret_cast<const __half2*>(p.v);
    __half2 m = __habs2(v[0]);
#pragma unroll
    for (int i = 1; i < VEC / 2; ++i) m = __hmax2_nan(m, __habs2(v[i]));
    return max_nan(__low2float(m), __high2float(m));
  }
}

// rint(x / s) as a division rounded to nearest gives it; inv = 1 / s, rounded.
// Adding 1.5 * 2^23 rounds to the nearest integer and leaves it in the low bits.
//
// 16 bits: x * inv is corrected by its remainder x - q s, which an FMA gives
// exactly (Markstein, IBM J. Res. Dev. 34, 1990): q + (x - q s) * inv is the
// quotient rounded to nearest for all pairs of values and largest values of both
// types. Scales are kept clear of underflow. Ties are common in 16 bits (half the
// pieces of a warp have one), so no form that treats them apart is as fast.
//
// fp32: x * inv is within 2e-5 of the quotient (at most 127), so a piece is divided
// where one of its values is as close to a tie, or the reciprocal overflows.
template <typename T, int VEC>
__device__ __forceinline__ Piece<int8_t, VEC> quantize_piece(const Piece<T, VEC>& p, float s, float inv) {
  constexpr float kRound = 12582912.0f, kClear = 18446744073709551616.0f;  // 2^64
  Piece<int8_t, VEC> o;
  bool divide;
  if constexpr (sizeof(T) == 2) {
    divide = !(s > 1.0f / kClear && s < kClear);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float v = to_f32(p.v[i]), q = v * inv;
      o.v[i] = static_cast<int8_t>(__float_as_int(fmaf(fmaf(-q, s, v), inv, q) + kRound));
    }
  } else {
    float off = 0.0f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float q = to_f32(p.v[i]) * inv;
      const float r = q + kRound;
      off = max_nan(off, fabsf(q - (r - kRound)));
      o.v[i] = static_cast<int8_t>(__float_as_int(r));
    }
    divide = !(off < 0.4999f);
  }
  if (divide) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float r = s > 0.0f ? rintf(__fdiv_rn(to_f32(p.v[i]), s)) : 0.0f;
      o.v[i] = static_cast<int8_t>(fminf(fmaxf(r, -127.0f), 127.0f));
    }
  }
  return o;
}

// A row for tp threads, its first NP pieces a thread held in registers between
// the search for the largest and the rounding (what is beyond is read again).
template <typename T, int VEC, int NP>
__global__ void __launch_bounds__(kQuantThreads) quantize_kernel(const T* x, int64_t rows, int64_t K, int64_t stride,
                                                                 int8_t* q, float* scale, int tp) {
  let_next_grid_start();
  __shared__ float part[kQuantThreads / 32];
  const int group = threadIdx.x / tp;
  const int64_t t = blockIdx.x * static_cast<int64_t>(kQuantThreads / tp) + group;
  const bool live = t < rows;
  const int64_t pieces = K / VEC;
  const Piece<T, VEC>* row = reinterpret_cast<const Piece<T, VEC>*>(x + t * stride);
  Piece<T, VEC> held[NP];
  float peak = 0.0f;
  const int64_t c0 = threadIdx.x % tp;
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    const int64_t c = c0 + n * tp;
    held[n] = live && c < pieces ? row[c] : Piece<T, VEC>{};
  }
#pragma unroll
  for (int n = 0; n < NP; ++n) peak = max_nan(peak, piece_peak<VEC>(held[n]));
  if (live)
    for (int64_t c = c0 + NP * tp; c < pieces; c += tp) peak = max_nan(peak, piece_peak<VEC>(row[c]));
#pragma unroll
  for (int o = 16; o; o >>= 1) peak = max_nan(peak, __shfl_xor_sync(kFull, peak, o));
  if (tp > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = peak;
    __syncthreads();
    for (int w = 0; w < tp / 32; ++w) peak = max_nan(peak, part[group * (tp / 32) + w]);
  }
  if (!live) return;
  const bool finite = peak <= FLT_MAX;
  const float s = finite ? __fdiv_rn(peak, 127.0f) : NAN;
  const float inv = __fdiv_rn(1.0f, s);
  if (c0 == 0) scale[t] = s;
  Piece<int8_t, VEC>* out = reinterpret_cast<Piece<int8_t, VEC>*>(q + t * K);
#pragma unroll
  for (int n = 0; n < NP; ++n)
    if (c0 + n * tp < pieces) out[c0 + n * tp] = quantize_piece<T, VEC>(held[n], s, inv);
  for (int64_t c = c0 + NP * tp; c < pieces; c += tp) out[c] = quantize_piece<T, VEC>(row[c], s, inv);
}

template <typename T, int VEC>
int quantize_vec(const void* x, int64_t rows, int64_t K, int64_t stride, int8_t* q, float* scale, cudaStream_t s) {
  // few rows: a CTA a row; else as few threads a row as hold it in registers
  const int64_t pieces = K / VEC;
  int tp = rows >= 4 * kSMs ? 32 : kQuantThreads;
  while (tp < kQuantThreads && tp * 4 < pieces) tp *= 2;
  const int64_t per = kQuantThreads / tp, np = (pieces + tp - 1) / tp;
  const unsigned blocks = static_cast<unsigned>((rows + per - 1) / per);
#define ES_QUANT(NP)                                                                                             \
  ES_LAUNCH((quantize_kernel<T, VEC, NP>), blocks, kQuantThreads, 0, s, static_cast<const T*>(x), rows, K, stride, \
            q, scale, tp)
  if (np <= 2)
    ES_QUANT(2);
  else
    ES_QUANT(4);
#undef ES_QUANT
  return ES_OK;
}

template <typename T>
int quantize_typed(const void* x, int64_t rows, int64_t K, int64_t stride, int8_t* q, float* scale, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  if (K % VEC == 0 && stride % VEC == 0 && aligned16(x) && aligned16(q))
    return quantize_vec<T, VEC>(x, rows, K, stride, q, scale, s);
  return quantize_vec<T, 1>(x, rows, K, stride, q, scale, s);
}

// Largest sizes: a row index fits 31 bits, a grid dimension too.
bool rows_ok(int64_t n) { return n >= 0 && n <= 0x7fffff00LL; }

}  // namespace
}  // namespace es

using namespace es;

extern "C" int es_route_experts(const void* logits, int dtype, int64_t num_tokens, int num_experts,
                                int64_t row_stride, int top_k, int renormalize, float* weights, int32_t* experts,
                                void* stream) {
  if (num_experts < 1 || top_k < 1 || top_k > num_experts || num_tokens < 0) return ES_ERR_INVALID;
  if (num_experts > kMaxExperts || top_k > kMaxTopK || !rows_ok(num_tokens * top_k)) return ES_ERR_UNSUPPORTED;
  if (num_tokens == 0) return ES_OK;
  if (!logits || !weights || !experts) return ES_ERR_INVALID;
  ES_BY_TYPE(dtype, return route_typed<T>(logits, num_tokens, num_experts, row_stride, top_k, renormalize, weights,
                                          experts, nullptr, nullptr, as_stream(stream)));
  return ES_ERR_UNSUPPORTED;
}

extern "C" int es_route_experts_grad(const void* logits, int dtype, int64_t num_tokens, int num_experts,
                                     int64_t row_stride, int top_k, int renormalize, const float* weights,
                                     const int32_t* experts, const float* dweights, void* dlogits, void* stream) {
  if (num_experts < 1 || top_k < 1 || top_k > num_experts || num_tokens < 0) return ES_ERR_INVALID;
  if (num_experts > kMaxExperts || top_k > kMaxTopK || !rows_ok(num_tokens * top_k)) return ES_ERR_UNSUPPORTED;
  if (num_tokens == 0) return ES_OK;
  if (!logits || !weights || !experts || !dweights || !dlogits) return ES_ERR_INVALID;
  ES_BY_TYPE(dtype, return route_typed<T>(logits, num_tokens, num_experts, row_stride, top_k, renormalize,
                                          const_cast<float*>(weights), const_cast<int32_t*>(experts), dweights,
                                          dlogits, as_stream(stream)));
  return ES_ERR_UNSUPPORTED;
}

extern "C" size_t es_expert_plan_workspace_size(int64_t num_choices, int num_experts) {
  if (num_choices <= kPlanChunk || num_experts < 1) return 0;
  const int64_t chunks = (num_choices + kPlanChunk - 1) / kPlanChunk;
  return static_cast<size_t>(chunks + 1) * (num_experts + 1) * sizeof(int32_t);
}

extern "C" int es_expert_plan(const int32_t* experts, int64_t num_choices, int num_experts, void* workspace,
                              size_t workspace_bytes, int32_t* offsets, int32_t* order, int32_t* position,
                              int32_t* status, void* stream) {
  if (num_choices < 0 || num_experts < 1 || !offsets) return ES_ERR_INVALID;
  if (num_experts > kMaxExperts || !rows_ok(num_choices)) return ES_ERR_UNSUPPORTED;
  if (num_choices > 0 && (!experts || !order || !position)) return ES_ERR_INVALID;
  if (workspace_bytes < es_expert_plan_workspace_size(num_choices, num_experts)) return ES_ERR_WORKSPACE;
  cudaStream_t s = as_stream(stream);
  const size_t smem = plan_smem(num_experts);
  if (smem > 48 * 1024) {
    // to the largest, once a device: a limit of this call's own size could be
    // lowered by another thread's call before the launch
    static std::atomic<bool> raised[kMaxAttrDevices];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return ES_ERR_CUDA;
    const bool tracked = dev >= 0 && dev < kMaxAttrDevices;
    if (!tracked || !raised[dev].load(std::memory_order_relaxed)) {
      if (cudaFuncSetAttribute(plan_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(plan_smem(kMaxExperts))) != cudaSuccess)
        return ES_ERR_CUDA;
      if (tracked) raised[dev].store(true, std::memory_order_relaxed);
    }
  }
  const int64_t chunks = num_choices > kPlanChunk ? (num_choices + kPlanChunk - 1) / kPlanChunk : 1;
  int32_t* counts = nullptr;
  if (chunks > 1) {
    counts = static_cast<int32_t*>(workspace);
    ES_LAUNCH(plan_count_kernel, static_cast<unsigned>(chunks), kPlanThreads, (num_experts + 1) * sizeof(int32_t), s,
              experts, num_choices, num_experts, counts);
  }
  const int scanned = chunks > kPlanDirect;
  if (scanned)
    ES_LAUNCH(plan_scan_kernel, static_cast<unsigned>(num_experts + 1), kPlanThreads, 0, s, counts, chunks,
              num_experts);
  ES_LAUNCH(plan_place_kernel, static_cast<unsigned>(chunks), kPlanThreads, smem, s, experts, num_choices,
            num_experts, static_cast<const int32_t*>(counts), scanned, offsets, order, position, status);
  return ES_OK;
}

extern "C" int es_combine_experts(const void* y, int dtype, int64_t num_rows, int64_t row_stride,
                                  const float* weights, const int32_t* position, int64_t num_tokens, int top_k,
                                  int64_t width, void* out, int out_dtype, void* stream) {
  if (num_rows < 0 || num_tokens < 0 || top_k < 1 || width < 0) return ES_ERR_INVALID;
  if (!rows_ok(num_rows) || !rows_ok(num_tokens * top_k)) return ES_ERR_UNSUPPORTED;
  if (num_tokens == 0 || width == 0) return ES_OK;
  if ((!y && num_rows) || !position || !out) return ES_ERR_INVALID;
  cudaStream_t s = as_stream(stream);
  if (dtype == out_dtype)
    ES_BY_TYPE(dtype, return (combine_typed<T, T>(y, num_rows, row_stride, weights, position, num_tokens, top_k,
                                                  width, out, s)));
  if (dtype == ES_F32)  // the sum of fp32 rows in the operands' type
    ES_BY_TYPE(out_dtype, return (combine_typed<float, T>(y, num_rows, row_stride, weights, position, num_tokens,
                                                          top_k, width, out, s)));
  return ES_ERR_UNSUPPORTED;
}

extern "C" int es_combine_experts_grad(const void* y, int dtype, int64_t num_rows, int64_t row_stride,
                                       const float* weights, const int32_t* position, const int32_t* kept_rows,
                                       int64_t num_tokens, int top_k, int64_t width, const void* dout,
                                       int64_t dout_stride, void* dy, float* dweights, void* stream) {
  if (num_rows < 0 || num_tokens < 0 || top_k < 1 || width < 0) return ES_ERR_INVALID;
  if (!rows_ok(num_rows) || !rows_ok(num_tokens * top_k)) return ES_ERR_UNSUPPORTED;
  if (num_tokens == 0) return ES_OK;
  if (!weights || !position || !kept_rows || !dweights || (width && (!dout || (num_rows && (!y || !dy)))))
    return ES_ERR_INVALID;
  ES_BY_TYPE(dtype, return combine_grad_typed<T>(y, num_rows, row_stride, weights, position, kept_rows, num_tokens,
                                                 top_k, width, dout, dout_stride, dy, dweights, as_stream(stream)));
  return ES_ERR_UNSUPPORTED;
}

extern "C" int es_quantize_rows(const void* x, int dtype, int64_t num_rows, int64_t width, int64_t row_stride,
                                int8_t* q, float* scale, void* stream) {
  if (num_rows < 0 || width < 0) return ES_ERR_INVALID;
  if (!rows_ok(num_rows)) return ES_ERR_UNSUPPORTED;
  if (num_rows == 0) return ES_OK;
  if ((width && (!x || !q)) || !scale) return ES_ERR_INVALID;
  ES_BY_TYPE(dtype, return quantize_typed<T>(x, num_rows, width, row_stride, q, scale, as_stream(stream)));
  return ES_ERR_UNSUPPORTED;
}
