// The rows' product grouped by expert for groups of a few rows (a decode step,
// or a short prompt over many experts), on the CUDA cores: each weight is read
// once from HBM, as it lies, and multiplied with up to RT rows in fp32. Bound by
// the weights' bytes: at HBM's rate an SM gets 6 fp32 weights a clock, 8 rows of
// which are 47 of its 128 multiply-adds.
//
// A CTA makes a tile of columns for up to RT (4 or 8) rows of one expert, in
// chunks of kChunk of the depth, whose part of x is staged in shared memory. Every
// lane has eight 16-byte loads of weights in flight. A longer group is several
// CTAs' that meet in L2, so a step whose rows all chose one expert fills the SMs.
//
// Columns contiguous (forward): a lane owns four columns, the half warps share
// the depth and their sums are added in the end. Depth contiguous (the gradient
// of the rows): the lanes share the depth of four columns a warp (so that each
// value of x that is read serves four weights) and add up by shuffles. Both
// orders of addition are fixed.
//
// fp32 only: in 16 bits the tensor cores read the weights as fast.
#include "grouped.cuh"

namespace es {
namespace {

constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kChunk = 1024;
constexpr int kWarpCols = 4;  // columns of a warp, depth contiguous
constexpr int kTileCols = 64;  // columns of a CTA, columns contiguous
constexpr int kFewRows = 8;
// Rows of a group (the mean) up to which this is taken. 36 experts of 2520 x 1456,
// rows spread by chance, us here and on the tensor cores (which read the weights'
// planes after writing them): columns contiguous 70 and 241 at 1 row, 125 and 339
// at 4, 196 and 340 at 8, 242 and 343 at 12, 292 and 345 at 16, 406 and 349 at 24;
// depth contiguous 83 and 243, 153 and 345, 248 and 346, 327 and 350, 409 and 353
// (121 experts of 1136 x 728: 245 and 280 at 9 rows, 306 and 286 at 12). The
// weights alone take 52 us at 1 row (23 experts in use) and 81 from 4. Where all
// rows chose one expert: 129 and 188 us at a mean of 8, 241 at 16 (tensor cores 147).
constexpr int64_t kColumnsMean = 16, kDepthMean = 10;

// The n-th tile of up to kFewRows rows of one expert; false: there is none.
__device__ __forceinline__ bool nth_tile(const GroupedArgs& g, int n, int& expert, int64_t& r0, int64_t& hi) {
  __shared__ int64_t found[3];
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int64_t at = -1, a = 0, b = 0, seen = 0;
    for (int e0 = 0; e0 < g.groups() && at < 0; e0 += 32) {
      int64_t l = 0, h = 0;
      if (e0 + lane < g.groups()) g.bounds(e0 + lane, l, h);
      const int64_t tiles = h > l ? (h - l + kFewRows - 1) / kFewRows : 0;
      int64_t past = tiles;  // tiles of the lanes up to this one
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t before = __shfl_up_sync(0xffffffffu, past, o);
        if (lane >= o) past += before;
      }
      past += seen;
      const unsigned mine = __ballot_sync(0xffffffffu, n < past && n >= past - tiles);
      if (mine) {
        const int src = __ffs(mine) - 1;
        at = e0 + src;
        a = __shfl_sync(0xffffffffu, l + (n - (past - tiles)) * kFewRows, src);
        b = __shfl_sync(0xffffffffu, h, src);
      }
      seen = __shfl_sync(0xffffffffu, past, 31);
    }
    if (lane == 0) {
      found[0] = at;
      found[1] = a;
      found[2] = min(b, a + kFewRows);
    }
  }
  __syncthreads();
  expert = static_cast<int>(found[0]);
  r0 = found[1];
  hi = found[2];
  return expert >= 0;
}

// The tokens of rows r0 .. r0 + RT, -1 past the last.
template <int RT>
__device__ __forceinline__ void load_sources(const GroupedArgs& g, int64_t r0, int64_t hi, int64_t* src) {
  __syncthreads();
  if (threadIdx.x < RT) src[threadIdx.x] = r0 + threadIdx.x < hi ? g.source(r0 + threadIdx.x) : -1;
  __syncthreads();
}

__device__ __forceinline__ void clear_columns(const GroupedArgs& g, float* y, int64_t n0, int64_t n1) {
  for (int64_t r = g.kept() + blockIdx.y; r < g.rows; r += gridDim.y)
    for (int64_t n = n0 + threadIdx.x; n < n1; n += kFewThreads) y[r * g.N + n] = 0.0f;
}

template <int RT>
__device__ __forceinline__ void columns_tile(const GroupedArgs& g, const float* x, const float* we, float* y,
                                             int64_t n0, int64_t r0, int64_t hi, float* buffer, int64_t* src) {
  constexpr int AHEAD = 8, SHARES = 2 * kFewWarps;
  static_assert(kChunk % (AHEAD * SHARES) == 0, "reads of x past the depth stay in the chunk");
  const int share = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const bool live = n0 + lane * 4 < g.N;
  load_sources<RT>(g, r0, hi, src);
  float4 acc[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int64_t k0 = 0; k0 < g.K; k0 += kChunk) {
    const int depth = static_cast<int>(min(g.K - k0, static_cast<int64_t>(kChunk)));
    __syncthreads();
    for (int i = threadIdx.x; i < RT * kChunk; i += kFewThreads) {  // x[depth][row]
      const int r = i / kChunk, k = i % kChunk;
      buffer[k * RT + r] = k < depth && src[r] >= 0 ? x[src[r] * g.x_stride + k0 + k] : 0.0f;
    }
    __syncthreads();
    const int per = ((depth + SHARES - 1) / SHARES + AHEAD - 1) / AHEAD * AHEAD;
    const int k1 = min(depth, (share + 1) * per);
    if (!live) continue;
    for (int k = share * per; k < k1; k += AHEAD) {
      float4 p[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        p[u] = k + u < k1 ? __ldcs(reinterpret_cast<const float4*>(we + (k0 + k + u) * g.w_k + lane * 4))
                          : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const float* xr = buffer + (k + u) * RT;  // past the depth both factors are zeros
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          acc[r].x = fmaf(xr[r], p[u].x, acc[r].x);
          acc[r].y = fmaf(xr[r], p[u].y, acc[r].y);
          acc[r].z = fmaf(xr[r], p[u].z, acc[r].z);
          acc[r].w = fmaf(xr[r], p[u].w, acc[r].w);
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < RT; ++r)  // [share][row][column]
    *reinterpret_cast<float4*>(buffer + (share * RT + r) * kTileCols + lane * 4) = acc[r];
  __syncthreads();
  for (int i = threadIdx.x; i < RT * kTileCols; i += kFewThreads) {
    const int r = i / kTileCols, c = i % kTileCols;
    if (r0 + r >= hi || n0 + c >= g.N) continue;
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < SHARES; ++v) s += buffer[(v * RT + r) * kTileCols + c];
    y[(r0 + r) * g.N + n0 + c] = s;
  }
}

__global__ void __launch_bounds__(kFewThreads, 2) few_columns_kernel(const __grid_constant__ GroupedArgs g,
                                                                     const float* x, const float* w, float* y) {
  __shared__ alignas(16) float buffer[kFewRows * kChunk];
  static_assert(2 * kFewWarps * kFewRows * kTileCols <= kFewRows * kChunk, "the shares' sums");
  __shared__ int64_t src[kFewRows];
  const int64_t n0 = blockIdx.x * static_cast<int64_t>(kTileCols);
  clear_columns(g, y, n0, min(n0 + kTileCols, g.N));
  int e;
  int64_t r0, hi;
  if (!nth_tile(g, blockIdx.y, e, r0, hi)) return;
  const float* we = w + e * g.w_e + n0;
  if (hi - r0 > 4)
    columns_tile<kFewRows>(g, x, we, y, n0, r0, hi, buffer, src);
  else
    columns_tile<4>(g, x, we, y, n0, r0, hi, buffer, src);
}

template <int RT>
__device__ __forceinline__ void depth_tile(const GroupedArgs& g, const float* x, const float* we, float* y, int64_t n,
                                           int64_t r0, int64_t hi, float* buffer, int64_t* src) {
  constexpr int AHEAD = 2;
  static_assert(kChunk % (128 * AHEAD) == 0, "reads of x past the depth stay in the chunk");
  const int lane = threadIdx.x & 31;
  load_sources<RT>(g, r0, hi, src);
  float acc[RT][kWarpCols];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < kWarpCols; ++c) acc[r][c] = 0.0f;
  for (int64_t k0 = 0; k0 < g.K; k0 += kChunk) {
    const int depth = static_cast<int>(min(g.K - k0, static_cast<int64_t>(kChunk)));
    __syncthreads();
    for (int i = threadIdx.x; i < RT * kChunk; i += kFewThreads) {  // x[row][depth]
      const int r = i / kChunk, k = i % kChunk;
      buffer[i] = k < depth && src[r] >= 0 ? x[src[r] * g.x_stride + k0 + k] : 0.0f;
    }
    __syncthreads();
    for (int k = lane * 4; k < depth; k += 128 * AHEAD) {
      float4 p[AHEAD][kWarpCols];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int c = 0; c < kWarpCols; ++c)
          p[u][c] = n + c < g.N && k + u * 128 < depth
                        ? __ldcs(reinterpret_cast<const float4*>(we + c * g.w_n + k0 + k + u * 128))
                        : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          // past the depth both factors are zeros
          const float4 xv = *reinterpret_cast<const float4*>(buffer + r * kChunk + k + u * 128);
#pragma unroll
          for (int c = 0; c < kWarpCols; ++c) {
            acc[r][c] = fmaf(xv.x, p[u][c].x, acc[r][c]);
            acc[r][c] = fmaf(xv.y, p[u][c].y, acc[r][c]);
            acc[r][c] = fmaf(xv.z, p[u][c].z, acc[r][c]);
            acc[r][c] = fmaf(xv.w, p[u][c].w, acc[r][c]);
          }
        }
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < kWarpCols; ++c) {
      float s = acc[r][c];
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0 && r0 + r < hi && n + c < g.N) y[(r0 + r) * g.N + n + c] = s;
    }
}

__global__ void __launch_bounds__(kFewThreads, 2) few_depth_kernel(const __grid_constant__ GroupedArgs g,
                                                                   const float* x, const float* w, float* y) {
  constexpr int COLS = kFewWarps * kWarpCols;
  __shared__ alignas(16) float buffer[kFewRows * kChunk];
  __shared__ int64_t src[kFewRows];
  const int64_t n0 = blockIdx.x * static_cast<int64_t>(COLS), n = n0 + (threadIdx.x >> 5) * kWarpCols;
  clear_columns(g, y, n0, min(n0 + COLS, g.N));
  int e;
  int64_t r0, hi;
  if (!nth_tile(g, blockIdx.y, e, r0, hi)) return;
  const float* we = w + e * g.w_e + n * g.w_n;
  if (hi - r0 > 4)
    depth_tile<kFewRows>(g, x, we, y, n, r0, hi, buffer, src);
  else
    depth_tile<4>(g, x, we, y, n, r0, hi, buffer, src);
}

bool by_columns(const GroupedArgs& g) { return g.w_n == 1 && g.N > 1; }

}  // namespace

bool grouped_rows_few_ok(const GroupedArgs& g, int dtype, const void* w) {
  if (g.num_experts < 1 || dtype != ES_F32 || g.rows < 1) return false;
  const int64_t live = min(static_cast<int64_t>(g.num_experts), g.rows);
  // 16-byte loads of the weights as they lie
  const bool columns = by_columns(g);
  const int64_t inner = columns ? g.N : g.K, row = columns ? g.w_k : g.w_n, rows = columns ? g.K : g.N;
  if (!columns && g.w_k != 1 && g.K > 1) return false;
  if ((reinterpret_cast<uintptr_t>(w) & 15) != 0 || inner % 4 != 0 || (rows > 1 && row % 4 != 0) ||
      (g.num_experts > 1 && g.w_e % 4 != 0))
    return false;
  return g.rows <= live * (columns ? kColumnsMean : kDepthMean);
}

int grouped_rows_few(const GroupedArgs& g, const void* x, const void* w, void* y, cudaStream_t s) {
  const bool columns = by_columns(g);
  const int64_t cols = columns ? kTileCols : kFewWarps * kWarpCols;
  // groups of n rows have at most this many tiles: one begun by each live group, the others full
  const int64_t live = min(static_cast<int64_t>(g.num_experts), g.rows);
  const int64_t tiles = live + (g.rows - live) / kFewRows;
  const dim3 grid(static_cast<unsigned>((g.N + cols - 1) / cols), static_cast<unsigned>(tiles));
  const float *xf = static_cast<const float*>(x), *wf = static_cast<const float*>(w);
  if (columns)
    ES_LAUNCH(few_columns_kernel, grid, kFewThreads, 0, s, g, xf, wf, static_cast<float*>(y));
  else
    ES_LAUNCH(few_depth_kernel, grid, kFewThreads, 0, s, g, xf, wf, static_cast<float*>(y));
  return ES_OK;
}

}  // namespace es
