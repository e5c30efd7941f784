// The rows' product grouped by expert in fp32 for groups of a few rows (a decode
// step, or a short prompt over many experts): each weight is read once from HBM,
// as it lies, cut into three bf16 planes in the registers that it was loaded to and
// multiplied there. The planes that the tcgen05 kernels read from memory cost 16
// bytes of traffic a weight for its 4.
//
// x w = sum of xi wj over the planes with i + j <= 2 (the others are below the last
// bit of an fp32 product). The planes are rounded to nearest, so three hold all 24
// bits. x0 w0 and the five smaller products have sums of their own; the first is
// added in fp32 after each chunk of the depth, since the tensor cores' own
// addition truncates. Error at 8 rows, 2520 deep: 1.4e-7 of the output.
//
// A CTA makes kTileCols channels for up to 16 rows of one expert. Its 8 warps are 2
// groups of 32 channels x 4 shares of the depth; the shares' sums are added in the
// end, in their order. (4 groups x 2 shares: half the staging of x for a weight,
// but 121 us for 71 where all rows chose one of 8 experts of 4096 x 4096, and
// 133 for 120 at 36 of 2520 x 1456, 8 rows.) The channels are the rows of the MMA
// and the expert's rows its columns. Depth and channels are permuted within a step
// so that every lane's part of it is four 16-byte loads, whichever of the two is
// contiguous: (columns) depths 4t .. 4t+3 of channels 4g .. 4g+3; (depth) the same
// depths of channels g, g+8, g+16, g+24. A longer group is several CTAs' that meet
// in L2, so a step whose rows all chose one expert fills the SMs.
//
// Bound by HBM up to 4 rows (36 experts of 2520 x 1456, 4 rows each: 105 us, 4.8
// TB/s with the 2.8 rounds of CTAs taking 3; the weights alone 78), then by the
// dependent chain load, cut, multiply of the 16 warps that an SM holds (16 rows: 130
// us, 42% of the issue slots, 36% of the tensor pipe). A ring of asynchronous copies,
// 48 KB ahead, did not help (107 us at 4 rows, 171 for 167 at 16).
//
// fp32 only: in 16 bits the grouped_tc kernels read the weights as fast.
#include "grouped.cuh"

namespace es {
namespace {

constexpr int kFewThreads = 256;
constexpr int kFewRows = 16;
constexpr int kTileCols = 64;  // channels of a CTA
constexpr int kGroups = kTileCols / 32;  // of its channels, 32 a warp
constexpr int kShares = kFewThreads / 32 / kGroups;  // of the depth
constexpr int kStep = 16;      // depth of an MMA
constexpr int kPlanes = 3;
constexpr int kPlaneBytes = 12288;  // of x in shared memory: chunk x rows
// Rows of a group (the mean) up to which this is taken. 36 experts of 2520 x 1456,
// rows spread by chance, us here and on the tcgen05 kernels: 71 and 241 at 1 row,
// 105 and 339 at 4, 120 and 340 at 8, 178 and 345 at 16, 222 and 349 at 24, 267 and
// 373 at 32, 375 and 372 at 48 (121 of 1136 x 728: 188 and 294 at 24, 317 and 301 at
// 48). Both orders of the weights are within 6%. Where all rows chose one of the
// 36: 118 and 147 at a mean of 16, 227 and 145 at 32; 24 is between the two.
constexpr int64_t kFewMean = 24;
constexpr int64_t kMaxDepth = 1 << 30;  // counted in 32 bits

// The n-th tile of up to kFewRows rows of one expert, left in shared memory too (expert,
// first row, end); false: there is none.
__device__ __forceinline__ bool nth_tile(const GroupedArgs& g, int n, int& expert, int64_t& r0, int64_t& hi,
                                         int64_t* found) {
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

struct Planes {
  uint32_t p[kPlanes];  // two values each
};

__device__ __forceinline__ Planes split(float a, float b) {
  Planes s;
#pragma unroll
  for (int i = 0; i < kPlanes; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    s.p[i] = *reinterpret_cast<const uint32_t*>(&h);
    a -= __uint_as_float(s.p[i] << 16);
    b -= __uint_as_float(s.p[i] & 0xffff0000u);
  }
  return s;
}

__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint2 b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}

// Planes of a chunk of x, [plane][step][8 rows][row][t] of depths 4t .. 4t+3 (so a
// warp's operand is 256 bytes in a row); zeros past the depth and the rows. A
// thread has the same row and t of every step it fills; `from` is there, `left`
// the depth from there on (none: no row).
template <int NT>
__device__ __forceinline__ void stage_rows(const float* from, int left, bool wide, uint2* planes) {
  constexpr int QUADS = kPlaneBytes / 8, EACH = QUADS / kFewThreads, DEPTH = kFewThreads / (32 * NT) * kStep;
  static_assert(kFewThreads % (32 * NT) == 0 && QUADS % kFewThreads == 0);
  planes += threadIdx.x;
  float4 v[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const float* p = from + i * DEPTH;
    const int n = left - i * DEPTH;
    v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (wide && n >= 4) {
      v[i] = *reinterpret_cast<const float4*>(p);
    } else if (n > 0) {
      v[i].x = p[0];
      if (n > 1) v[i].y = p[1];
      if (n > 2) v[i].z = p[2];
      if (n > 3) v[i].w = p[3];
    }
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const Planes a = split(v[i].x, v[i].y), b = split(v[i].z, v[i].w);
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) planes[p * QUADS + i * kFewThreads] = make_uint2(a.p[p], b.p[p]);
  }
}

// A lane's part of a step, 4 depths x 4 channels. COLUMNS: depth j (of the `left`
// ones) of four channels; else depths 0 .. 3 of channel 8 j.
template <bool COLUMNS>
__device__ __forceinline__ void load_step(float4* v, const float* from, int64_t stride, int left, int live) {
#pragma unroll
  for (int j = 0; j < 4; ++j, from += stride) {
    const bool in = COLUMNS ? j < left : left > 0 && (live >> j & 1);
    v[j] = in ? __ldcs(reinterpret_cast<const float4*>(from)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
}

__device__ __forceinline__ float lane_of(const float4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// The step's products: MMA tile i has channels (i, 0) in its rows 0 .. 7 and (i, 1) in 8 .. 15.
template <bool COLUMNS, int NT>
__device__ __forceinline__ void multiply(float (*main)[NT][4], float (*small)[NT][4], const float4* v,
                                         const uint2* planes) {
  constexpr int QUADS = kPlaneBytes / 8;
  uint2 b[NT][kPlanes];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) b[n][p] = planes[p * QUADS + n * 32];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t a[kPlanes][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        const int c = 2 * i + h;
        const Planes s = COLUMNS ? split(lane_of(v[2 * d], c), lane_of(v[2 * d + 1], c))
                                 : split(lane_of(v[c], 2 * d), lane_of(v[c], 2 * d + 1));
#pragma unroll
        for (int p = 0; p < kPlanes; ++p) a[p][2 * d + h] = s.p[p];
      }
#pragma unroll
    for (int m = 2; m > 0; --m)  // planes i + j = m, smallest first
#pragma unroll
      for (int j = 0; j <= m; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) mma(small[i][n], a[m - j], b[n][j]);
#pragma unroll
    for (int n = 0; n < NT; ++n) mma(main[i][n], a[0], b[n][0]);
  }
}

template <bool COLUMNS, int NT>
__device__ __forceinline__ void few_tile(const GroupedArgs& g, const float* x, const float* we, float* y, bool wide,
                                         int64_t n0, int64_t r0, int64_t hi, uint2* planes, int64_t* src, int* again) {
  constexpr int CHUNK = kPlaneBytes / 2 / (8 * NT), STEPS = CHUNK / kStep / kShares;
  static_assert(STEPS % 2 == 0 && kShares * 8 * NT * kTileCols * 4 <= kPlanes * kPlaneBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, share = warp / kGroups, t = lane & 3, q = lane >> 2;
  const int64_t c0 = n0 + warp % kGroups * 32 + (COLUMNS ? 4 * q : q);  // the lane's first channel
  int live = 0;  // COLUMNS: all four or none
#pragma unroll
  for (int j = 0; j < 4; ++j) live |= (COLUMNS ? c0 : c0 + 8 * j) < g.N ? 1 << j : 0;
  if (threadIdx.x < 8 * NT) src[threadIdx.x] = r0 + threadIdx.x < hi ? g.source(r0 + threadIdx.x) : -1;
  __syncthreads();
  const int depth = static_cast<int>(g.K);
  // this thread's part of x to stage, this lane's weights and what is left of their depth
  const int x_row = (threadIdx.x >> 2) % (8 * NT), x_k = threadIdx.x / (32 * NT) * kStep + (threadIdx.x & 3) * 4;
  const float* x_from = x + src[x_row] * g.x_stride + x_k;
  const bool x_live = src[x_row] >= 0;
  int k = share * kStep + 4 * t;
  const int64_t stride = COLUMNS ? g.w_k : 8 * g.w_n;
  const int64_t ahead = kStep * kShares * (COLUMNS ? g.w_k : 1);
  const float* from = we + c0 * g.w_n + k * g.w_k;
  const int end = COLUMNS && !live ? 0 : depth;

  float main[2][NT][4] = {}, small[2][NT][4] = {}, total[2][NT][4] = {};
  float4 v[2][4];
  const auto load = [&](float4* to) {
    load_step<COLUMNS>(to, from, stride, end - k, live);
    k += kStep * kShares;
    from += ahead;
  };
  load(v[0]);
  for (int k0 = 0; k0 < depth; k0 += CHUNK, x_from += CHUNK) {
    if (k0) __syncthreads();
    stage_rows<NT>(x_from, x_live ? depth - k0 - x_k : 0, wide, planes);
    __syncthreads();
    const uint2* mine = planes + share * 32 * NT + lane;
    const int steps = min(STEPS, (depth - k0 - share * kStep + kStep * kShares - 1) / (kStep * kShares));
#pragma unroll 1
    for (int i = 0; i < steps; i += 2, mine += 2 * kShares * 32 * NT) {
      load(v[1]);
      multiply<COLUMNS, NT>(main, small, v[0], mine);
      load(v[0]);
      multiply<COLUMNS, NT>(main, small, v[1], mine + kShares * 32 * NT);
    }
#pragma unroll
    for (int i = 0; i < 2 * NT * 4; ++i) {
      (&total[0][0][0])[i] += (&main[0][0][0])[i];
      (&main[0][0][0])[i] = 0.0f;
    }
  }

  __syncthreads();
  float* sums = reinterpret_cast<float*>(planes);  // [share][row][channel]
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = n * 8 + 2 * t + (j & 1), c = 2 * i + (j >> 1);
        const int channel = warp % kGroups * 32 + (COLUMNS ? 4 * q + c : 8 * c + q);
        sums[(share * 8 * NT + row) * kTileCols + channel] = total[i][n][j] + small[i][n][j];
      }
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * NT * kTileCols; i += kFewThreads) {
    const int row = i / kTileCols, c = i % kTileCols;
    if (r0 + row >= hi || n0 + c >= g.N) continue;
    float s = 0.0f;
#pragma unroll
    for (int h = 0; h < kShares; ++h) s += sums[(h * 8 * NT + row) * kTileCols + c];
    if (!isfinite(s) && src[row] >= 0) atomicOr(again, 1 << row);
    y[(r0 + row) * g.N + n0 + c] = s;
  }
}

// Sums of the CTA's channels that are not finite, in the rows of `left`: made again from the
// values, in fp32, since infinities have no planes, nor has a value that rounds to one. A NaN
// in a row of x (a poisoned token) has made all its sums NaN already. Four threads share
// a channel's depth; four rows are made from one reading of the weights. 36 experts of 2520
// x 1456, 8 rows each, 104 us: 130 with an infinity in one row, 683 with one in every row,
// 124 with a NaN in every row.
__device__ __forceinline__ void sums_again(const GroupedArgs& g, const float* x, const int64_t* src, const float* we,
                                           float* y, int64_t n0, int left, float* part) {
  constexpr int kParts = kFewThreads / kTileCols, kAtOnce = 4;
  static_assert(kAtOnce == kParts, "one thread for each row and channel in the end");
  for (int rows = left; rows; rows &= rows - 1) {
    const int row = __ffs(rows) - 1;
    const float* xr = x + src[row] * g.x_stride;
    bool nan = false;
    for (int64_t k = threadIdx.x; k < g.K; k += kFewThreads) nan |= isnan(xr[k]);
    if (__syncthreads_or(nan)) left &= ~(1 << row);
  }
  const int c = threadIdx.x % kTileCols, p = threadIdx.x / kTileCols;
  while (left) {
    int row[kAtOnce];  // the last of them again where there are fewer
    bool any = false;
    float s[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      row[i] = left ? __ffs(left) - 1 : row[i > 0 ? i - 1 : 0];
      left &= left - 1;
      any |= n0 + c < g.N && !isfinite(y[row[i] * g.N + n0 + c]);
      s[i] = 0.0f;
    }
    if (any) {
      const float* w = we + (n0 + c) * g.w_n;
#pragma unroll 4
      for (int64_t k = p; k < g.K; k += kParts) {
        const float v = w[k * g.w_k];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) s[i] = fmaf(x[src[row[i]] * g.x_stride + k], v, s[i]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) part[i * kFewThreads + threadIdx.x] = s[i];
    __syncthreads();
    // thread (p, c) has the p-th of the rows
    int mine = row[0];
    bool there = n0 + c < g.N;
#pragma unroll
    for (int i = 1; i < kAtOnce; ++i)
      if (p == i) {
        mine = row[i];
        there &= row[i] != row[i - 1];
      }
    float* to = y + mine * g.N + n0 + c;
    if (there && !isfinite(*to)) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kParts; ++i) sum += part[p * kFewThreads + i * kTileCols + c];
      *to = sum;
    }
    __syncthreads();
  }
}

template <bool COLUMNS>
__global__ void __launch_bounds__(kFewThreads, 2) few_kernel(const __grid_constant__ GroupedArgs g, const float* x,
                                                             const float* w, float* y, bool wide) {
  __shared__ alignas(16) uint2 planes[kPlanes * kPlaneBytes / 8];
  __shared__ int64_t src[kFewRows];
  __shared__ int64_t found[3];
  __shared__ int again;  // rows with a sum that is not finite
  if (threadIdx.x == 0) again = 0;
  const int64_t n0 = blockIdx.x * static_cast<int64_t>(kTileCols), n1 = min(n0 + kTileCols, g.N);
  for (int64_t r = g.kept() + blockIdx.y; r < g.rows; r += gridDim.y)
    for (int64_t n = n0 + threadIdx.x; n < n1; n += kFewThreads) y[r * g.N + n] = 0.0f;
  int e;
  int64_t r0, hi;
  if (!nth_tile(g, blockIdx.y, e, r0, hi, found)) return;
  const float* we = w + e * g.w_e;
  if (hi - r0 > 8)
    few_tile<COLUMNS, 2>(g, x, we, y, wide, n0, r0, hi, planes, src, &again);
  else
    few_tile<COLUMNS, 1>(g, x, we, y, wide, n0, r0, hi, planes, src, &again);
  __syncthreads();
  // from shared memory: nothing of this is held in registers through the product
  if (again)
    sums_again(g, x, src, w + found[0] * g.w_e, y + found[1] * g.N, blockIdx.x * static_cast<int64_t>(kTileCols), again,
               reinterpret_cast<float*>(planes));
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
  return g.K <= kMaxDepth && g.rows <= live * kFewMean;
}

int grouped_rows_few(const GroupedArgs& g, const void* x, const void* w, void* y, cudaStream_t s) {
  const bool columns = by_columns(g);
  // groups of n rows have at most this many tiles: one begun by each live group, the others full
  const int64_t live = min(static_cast<int64_t>(g.num_experts), g.rows);
  const int64_t tiles = live + (g.rows - live) / kFewRows;
  const dim3 grid(static_cast<unsigned>((g.N + kTileCols - 1) / kTileCols), static_cast<unsigned>(tiles));
  const float *xf = static_cast<const float*>(x), *wf = static_cast<const float*>(w);
  const bool wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && g.x_stride % 4 == 0;
  const auto kernel = columns ? few_kernel<true> : few_kernel<false>;
  ES_LAUNCH(kernel, grid, kFewThreads, 0, s, g, xf, wf, static_cast<float*>(y), wide);
  return ES_OK;
}

}  // namespace es
