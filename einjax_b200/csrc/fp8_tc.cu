// Products of 8-bit floating point (e4m3) with a scale for each 128 values of a row
// of X and each 128 x 128 block of W, dense or grouped by expert, on the tensor cores:
//
//   y[r, n] = sum_b x_scale[r, b] w_scale[n / 128, b] sum_{k in block b} x[r, k] w[n, k]
//
// The inner sum of a block of depth is made by four MMAs in TMEM; the epilogue warps
// read it, multiply by the two scales and add it to fp32 totals in their registers,
// while the next block's MMAs fill another accumulator. So no sum of the tensor cores
// is longer than 128 products, at any depth, and the scales are any fp32 numbers.
//
// Orientation. The 128 lanes of an accumulator (256 for a pair of CTAs) are rows, the
// columns channels: a thread has one row, so both scales of its columns are one number
// a block, held in a register. (With channels in the lanes, as in grouped_tc.cu, each
// column would need its own, read from shared memory, whose bandwidth the MMAs need.)
// The price is that a group's last tile multiplies empty lanes, which costs nothing where
// few rows leave the product bound by reading W. Results go through shared memory, a
// warp's own 4 KB, so that 128 bytes of a row are stored together.
//
// Roles and waits as in grouped_tc.cu: warp 0 issues the TMA loads, warp 1 the MMAs,
// warps 2-3 clear the rows of no expert, warps 4-11 read the accumulators. Every wait is
// bounded.
#include <cfloat>

#include "experts.cuh"
#include "fp8.cuh"
#include "tc_operands.cuh"
#include "tc_pipe.cuh"

namespace es {
namespace {

constexpr int kEpiWarps = 8;
constexpr int kTcThreads = 128 + 32 * kEpiWarps;
constexpr int kABytes = 16384;  // 128 rows x 128 bytes of depth
constexpr int kBoxRows = 32;    // rows of one TMA box
constexpr int kBoxBytes = kBoxRows * 128;
constexpr int kTileBlock = 8;   // row tiles that share a channel tile's weights in L2
constexpr int kMaxStages = 8;
constexpr int kMaxBufs = 4;

struct Fp8Args {
  GroupedArgs g;
  void* out;
  int out_dtype;
  int col_tiles;
  int expert_step;         // 0: every expert has the same matrix
  int k_blocks, n_blocks;  // scales of a row, rows of scales of a matrix
  int wide;                // 16-byte stores
  int32_t* status;
};

struct Fp8Maps {
  CUtensorMap x, w;
};

struct Fp8Ctl {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t acc_full[kMaxBufs];
  uint64_t acc_empty[kMaxBufs];
  uint64_t red_full, red_empty;
  uint64_t drain;
  uint32_t tmem;
  int abort;
  uint32_t progress;
};

template <int CG_, int NT_, bool SPLIT_>
struct Fp8Shape {
  static constexpr int CG = CG_;  // CTAs of one MMA
  static constexpr int NT = NT_;  // channels of a tile
  static constexpr bool SPLIT = SPLIT_;  // the cluster's CTAs share one tile's depth
  static constexpr int kRows = 128 * CG;
  static constexpr int kCols = NT / 2;  // of an epilogue warp
  static constexpr int kBufs = 512 / NT < kMaxBufs ? 512 / NT : kMaxBufs;
  static constexpr int kColumns = kBufs * NT;
  static constexpr int kStageBytes = kABytes + NT / CG * 128;
  static constexpr int kPitch = NT + 4;  // floats of a row of a split tile's part: no bank is met twice
  static constexpr int kOutBytes = SPLIT ? 128 * kPitch * 4 : kEpiWarps * 4096;
  static constexpr int kFit = (200 * 1024 - kOutBytes) / kStageBytes;
  static constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
  static constexpr bool kSplitRegs = kCols == 128;  // the epilogue takes registers of the other roles
  static_assert(!SPLIT || CG == 1, "a cluster shares the depth or the rows");
};

// One output tile, and which blocks of its depth this CTA multiplies.
struct Fp8Tile {
  int expert;
  int row0, rows;
  int col0, width;  // width: channels of the MMA, from the tile's own rounded up
  int kb0, kb1;
};

template <typename S>
struct Fp8Tiles {
  const Fp8Args& p;
  const int* pre;  // [groups + 1] tiles before each group
  const int* lo;   // [groups]
  const int* cnt;  // [groups]

  __device__ __forceinline__ Fp8Tile at(int t, uint32_t rank, uint32_t split) const {
    int a = 0, b = p.g.groups();
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (pre[m] <= t) a = m;
      else b = m;
    }
    const int idx = t - pre[a], row_tiles = (cnt[a] + S::kRows - 1) / S::kRows;
    // blocks of kTileBlock row tiles walk the channel tiles together
    const int block = idx / (kTileBlock * p.col_tiles);
    const int in = idx - block * kTileBlock * p.col_tiles;
    const int w = min(kTileBlock, row_tiles - block * kTileBlock);
    const int col_tile = in / w, row_tile = block * kTileBlock + in % w;
    Fp8Tile r;
    r.expert = a;
    r.row0 = lo[a] + row_tile * S::kRows;
    r.rows = min(cnt[a] - row_tile * S::kRows, S::kRows);
    r.col0 = col_tile * S::NT;
    r.width = static_cast<int>(min(p.g.N - r.col0, static_cast<int64_t>(S::NT)));
    r.width = (r.width + 16 * S::CG - 1) / (16 * S::CG) * (16 * S::CG);
    r.kb0 = 0;
    r.kb1 = p.k_blocks;
    if constexpr (S::SPLIT) {
      r.kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * rank / split);
      r.kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (rank + 1) / split);
    }
    return r;
  }
};

// Clears the output rows [from, to) with the threads `t` of `nt`.
__device__ __forceinline__ void clear_rows(const Fp8Args& p, int64_t from, int64_t to, int64_t t, int64_t nt) {
  const int64_t words = p.out_dtype == ES_F32 ? 2 : 1, n = (to - from) * p.g.N * words;
  uint16_t* a = static_cast<uint16_t*>(p.out) + from * p.g.N * words;
  const int64_t head = min(n, static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(a) & 15)) & 15) / 2);
  const int64_t body = (n - head) / 8;
  for (int64_t i = t; i < head; i += nt) a[i] = 0;
  uint4* mid = reinterpret_cast<uint4*>(a + head);
  for (int64_t i = t; i < body; i += nt) mid[i] = make_uint4(0, 0, 0, 0);
  for (int64_t i = head + body * 8 + t; i < n; i += nt) a[i] = 0;
}

// A block's sums times the scales of its row and channels, added to the totals: by the
// scales' product, or where that is past the type's ends by one after the other, the
// smaller first where it is infinite, the larger first where it is subnormal, so that a
// result that fp32 holds is met.
__device__ __forceinline__ void add_block(float* total, const uint32_t (&v)[32], float xs, float ws) {
  const float s = xs * ws;
  const bool ends = (fabsf(s) < FLT_MIN && xs != 0.0f && ws != 0.0f) || fabsf(s) == INFINITY;
  if (!ends) {
#pragma unroll
    for (int i = 0; i < 32; ++i) total[i] = fmaf(__uint_as_float(v[i]), s, total[i]);
  } else {
    const bool swap = (fabsf(xs) < fabsf(ws)) != (fabsf(s) == INFINITY);
    const float first = swap ? ws : xs, last = swap ? xs : ws;
#pragma unroll
    for (int i = 0; i < 32; ++i) total[i] = fmaf(__uint_as_float(v[i]) * first, last, total[i]);
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack16(const float* v) {
  alignas(16) T o[16 / sizeof(T)];
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) o[i] = from_f32<T>(v[i]);
  return *reinterpret_cast<uint4*>(o);
}

// Rounds and stores a warp's 32 rows (a lane's each) of COLS channels, 128 bytes of a
// row at a time through the warp's 4 KB: 16-byte pieces, swapped by the row so that
// neither side meets a bank twice.
template <typename T, int COLS>
__device__ __forceinline__ void store_rows(const Fp8Args& p, uint8_t* stage, const float (&total)[COLS], int row0,
                                           int rows, int64_t col0) {
  constexpr int VEC = 16 / sizeof(T), PASS = 8 * VEC;
  const int lane = threadIdx.x & 31, j = lane & 7;
#pragma unroll
  for (int c = 0; c < COLS; c += PASS) {
    uint4* mine = reinterpret_cast<uint4*>(stage + lane * 128);
#pragma unroll
    for (int i = 0; i < 8; ++i) mine[i ^ j] = pack16<T>(total + c + i * VEC);
    __syncwarp();
    const int64_t col = col0 + c + j * VEC;
    T* out = static_cast<T*>(p.out) + (row0 + (lane >> 3)) * p.g.N + col;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = i * 4 + (lane >> 3);
      const uint4 v = reinterpret_cast<const uint4*>(stage + row * 128)[j ^ (row & 7)];
      if (row < rows) {
        if (p.wide && col + VEC <= p.g.N) {
          *reinterpret_cast<uint4*>(out) = v;
        } else {
          const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
          for (int q = 0; q < VEC; ++q)
            if (col + q < p.g.N) out[q] = e[q];
        }
      }
      out += 4 * p.g.N;
    }
    __syncwarp();
  }
}

__device__ __forceinline__ float4 load4_at(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ void store4(const Fp8Args& p, int64_t row, int64_t col, const float4& v) {
  T* out = static_cast<T*>(p.out) + row * p.g.N + col;
  const float f[4] = {v.x, v.y, v.z, v.w};
  if (p.wide && col + 4 <= p.g.N) {
    struct alignas(4 * sizeof(T)) Four {
      T v[4];
    } o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = from_f32<T>(f[i]);
    *reinterpret_cast<Four*>(out) = o;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < p.g.N) out[i] = from_f32<T>(f[i]);
  }
}

// Registers, as in grouped_tc.cu: 128 * kRoleRegs + 256 * kEpiRegs = 384 * kLaunchRegs.
constexpr int kRoleRegs = 72, kEpiRegs = 216, kLaunchRegs = 168;
static_assert(128 * kRoleRegs + 256 * kEpiRegs == kTcThreads * kLaunchRegs, "register split");

template <typename S>
__global__ void __launch_bounds__(kTcThreads, 1)
    fp8_tc_kernel(const __grid_constant__ Fp8Args p, const __grid_constant__ Fp8Maps m) {
  constexpr int CG = S::CG, NT = S::NT, STAGES = S::kStages, BUFS = S::kBufs, COLS = S::kCols;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Fp8Ctl ctl;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* out_smem = smem_raw + (base - smem_u32(smem_raw)) + STAGES * S::kStageBytes;
  int* pre = reinterpret_cast<int*>(out_smem + S::kOutBytes);
  const int groups = p.g.groups();
  int* lo = pre + groups + 1;
  int* cnt = lo + groups;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank(), csize = cluster_size();
  const uint32_t pair_rank = CG == 2 ? rank : 0;
  const bool leader = pair_rank == 0;

  if (threadIdx.x == 0) {
    prefetch_map(&m.x);
    prefetch_map(&m.w);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&ctl.full[s], 1);
      mbar_init(&ctl.empty[s], 1);
    }
    for (int b = 0; b < BUFS; ++b) {
      mbar_init(&ctl.acc_full[b], 1);
      mbar_init(&ctl.acc_empty[b], CG * kEpiWarps);
    }
    mbar_init(&ctl.red_full, csize * kEpiWarps);
    mbar_init(&ctl.red_empty, csize * kEpiWarps);
    mbar_init(&ctl.drain, 1);
    ctl.abort = 0;
    ctl.progress = 0;
    fence_mbar_init();
  }
  if (warp == 1) tc_alloc<CG>(&ctl.tmem, S::kColumns);
  wait_for_earlier_grids();
  if (warp == 2) {  // tiles of each group
    int run = 0;
    for (int e0 = 0; e0 < groups; e0 += 32) {
      const int e = e0 + lane;
      int64_t a = 0, b = 0;
      if (e < groups) p.g.bounds(e, a, b);
      const int n = static_cast<int>(b - a);
      const int tiles = (n + S::kRows - 1) / S::kRows * p.col_tiles;
      int s = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
      }
      if (e < groups) {
        pre[e] = run + s - tiles;
        lo[e] = static_cast<int>(a);
        cnt[e] = n;
      }
      run += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) pre[groups] = run;
  }
  tc_fence_before();
  __syncthreads();
  if (csize > 1) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = ctl.tmem;
  const Fp8Tiles<S> tiles{p, pre, lo, cnt};
  const int total_tiles = pre[groups];
  const int step = static_cast<int>(gridDim.x / csize), t0 = static_cast<int>(blockIdx.x / csize);

  if (warp < 4) {
    if constexpr (S::kSplitRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRoleRegs));
    if (warp == 0) {
      // ------------------------------------------------------------ TMA loads
      int stage = 0, used = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = t0; t < total_tiles && ok; t += step) {
        const Fp8Tile at = tiles.at(t, rank, csize);
        const int half = at.width / CG;
        // boxes of 32 rows: those of X that hold rows, lanes past them are not stored
        auto x_boxes = [&](int r) { return (min(max(at.rows - r * 128, 0), 128) + kBoxRows - 1) / kBoxRows; };
        const int xb = x_boxes(static_cast<int>(pair_rank)), wb = (half + kBoxRows - 1) / kBoxRows;
        const uint32_t bytes = (CG * wb + x_boxes(0) + (CG == 2 ? x_boxes(1) : 0)) * kBoxBytes;
        const int x_row = at.row0 + static_cast<int>(pair_rank) * 128 + lane * kBoxRows;
        const int w_row = at.col0 + static_cast<int>(pair_rank) * half + (lane - 4) * kBoxRows;
        const int z = at.expert * p.expert_step;
        for (int kb = at.kb0; kb < at.kb1; ++kb) {
          int go = 0;
          if (lane == 0) {
            go = tc_wait(&ctl.empty[stage], phase ^ 1, &ctl, p.status) ? 1 : 0;
            if (go && leader) mbar_arrive_expect_tx(&ctl.full[stage], bytes);
            if (go) *reinterpret_cast<volatile uint32_t*>(&ctl.progress) = ++used;
          }
          go = __shfl_sync(0xffffffffu, go, 0);
          if (!go) {
            ok = false;
            break;
          }
          const uint32_t sa = base + stage * S::kStageBytes, sb = sa + kABytes;
          const uint32_t bar = CG == 2 ? at_rank(smem_u32(&ctl.full[stage]), 0) : smem_u32(&ctl.full[stage]);
          if (lane < xb) load_2d<CG>(sa + lane * kBoxBytes, &m.x, kb * 128, x_row, bar);
          if (lane >= 4 && lane - 4 < wb) load_3d<CG>(sb + (lane - 4) * kBoxBytes, &m.w, kb * 128, w_row, z, bar);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (lane == 0) {
        // the stages still held: their MMAs have arrived here before this CTA may end
        for (int s = 0; s < STAGES && ok; ++s) {
          if (s < used) {
            const int last = (stage + STAGES - 1 - s) % STAGES;
            const uint32_t ph = last < stage ? phase : phase ^ 1;
            ok = tc_wait(&ctl.empty[last], ph, &ctl, p.status);
          }
        }
        if (!ok && leader)
          for (int s = 0; s < STAGES && s < used; ++s) {
            const int last = (stage + STAGES - 1 - s) % STAGES;
            tc_drain(&ctl.full[last], last < stage ? phase : phase ^ 1);
          }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMAs
      if (leader) {
        int stage = 0, buf = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int t = t0; t < total_tiles && ok; t += step) {
          const Fp8Tile at = tiles.at(t, rank, csize);
          // D f32, A and B e4m3 (0) and K-major
          const uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(at.width >> 3) << 17) | ((8u * CG) << 24);
          for (int kb = at.kb0; kb < at.kb1; ++kb) {
            ok = tc_wait_warp(&ctl.acc_empty[buf], acc_phase ^ 1, &ctl, p.status) &&
                 tc_wait_warp(&ctl.full[stage], phase, &ctl, p.status);
            if (!ok) break;
            tc_fence_after();
            const uint64_t da = operand(base + stage * S::kStageBytes, false);
            const uint64_t db = operand(base + stage * S::kStageBytes + kABytes, false);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              mma<CG, kKindF8>(tmem + buf * NT, da + i * 2, db + i * 2, idesc, static_cast<uint32_t>(i));
            commit<CG>(&ctl.empty[stage]);
            commit<CG>(&ctl.acc_full[buf]);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1;
            }
            if (++buf == BUFS) {
              buf = 0;
              acc_phase ^= 1;
            }
          }
        }
        if (!ok) {
          commit<CG>(&ctl.drain);
          if (lane == 0) tc_drain(&ctl.drain, 0);
        }
      }
      __syncwarp();
    } else {
      // rows of no expert
      clear_rows(p, p.g.kept(), p.g.rows, blockIdx.x * 64LL + (threadIdx.x - 64), gridDim.x * 64LL);
    }
  } else {
    if constexpr (S::kSplitRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
    // ------------------------------------------------------------- epilogue
    const int quad = warp & 3, set = (warp - 4) >> 2;
    int buf = 0;
    uint32_t acc_phase = 0, red_phase = 0;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      int go = 1;
      if (lane == 0) go = tc_wait(bar, parity, &ctl, p.status, true) ? 1 : 0;
      return __shfl_sync(0xffffffffu, go, 0) != 0;
    };
    bool ok = true;
    for (int t = t0; t < total_tiles && ok; t += step) {
      const Fp8Tile at = tiles.at(t, rank, csize);
      const int first = static_cast<int>(pair_rank) * 128 + quad * 32;  // this warp's rows of the tile
      const int rows = at.rows - first, col0 = at.col0 + set * COLS;
      const bool any = rows > 0 && col0 < p.g.N;
      const int64_t source = lane < rows ? p.g.source(at.row0 + first + lane) : -1;
      const float* xs = p.g.x_scale + source * p.k_blocks;
      const float* ws = p.g.w_scale +
                        (static_cast<int64_t>(at.expert) * p.n_blocks + min(col0 >> 7, p.n_blocks - 1)) * p.k_blocks;
      float total[COLS];
#pragma unroll
      for (int i = 0; i < COLS; ++i) total[i] = 0.0f;
      float next_x = 0.0f, next_w = 0.0f;
      auto fetch = [&](int kb) {
        next_x = source >= 0 ? xs[kb] : 0.0f;
        next_w = ws[kb];
      };
      fetch(at.kb0);
      for (int kb = at.kb0; kb < at.kb1; ++kb) {
        const float x = next_x, w = next_w;
        if (kb + 1 < at.kb1) fetch(kb + 1);
        ok = wait(&ctl.acc_full[buf], acc_phase);
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc = tmem + buf * NT + (static_cast<uint32_t>(quad * 32) << 16) + set * COLS;
        auto release = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_at(at_rank(smem_u32(&ctl.acc_empty[buf]), CG == 2 ? 0 : rank));
        };
        if (any) {
          uint32_t v[2][32];
          tmem_ld32_async(acc, v[0]);
#pragma unroll
          for (int c = 0; c < COLS / 32; ++c) {
            tmem_wait32(v[c & 1]);
            if (c + 1 < COLS / 32) tmem_ld32_async(acc + (c + 1) * 32, v[(c + 1) & 1]);
            else release();
            add_block(total + c * 32, v[c & 1], x, w);
          }
        } else {
          release();
        }
        if (++buf == BUFS) {
          buf = 0;
          acc_phase ^= 1;
        }
      }
      if (!ok) break;
      if constexpr (S::SPLIT) {
        // every CTA puts its part into shared memory, [row][channel], and adds up every
        // csize-th piece of four channels, the parts in the CTAs' order
        ok = wait(&ctl.red_empty, red_phase ^ 1);  // the last tile's parts have been read by the whole cluster
        if (!ok) break;
        float* part = reinterpret_cast<float*>(out_smem);
        if (lane < rows) {
          float4* mine = reinterpret_cast<float4*>(part + (first + lane) * S::kPitch + set * COLS);
#pragma unroll
          for (int i = 0; i < COLS / 4; ++i)
            mine[i] = make_float4(total[4 * i], total[4 * i + 1], total[4 * i + 2], total[4 * i + 3]);
        }
        __syncwarp();
        if (lane < static_cast<int>(csize)) arrive_at(at_rank(smem_u32(&ctl.red_full), lane));
        ok = wait(&ctl.red_full, red_phase);
        if (!ok) break;
        const int pieces = at.rows * (NT / 4), each = 256 * static_cast<int>(csize);
        for (int i = static_cast<int>(rank) * 256 + static_cast<int>(threadIdx.x) - 128; i < pieces; i += each) {
          const int row = i / (NT / 4), c = i % (NT / 4) * 4;
          if (at.col0 + c >= p.g.N) continue;
          const uint32_t from = smem_u32(part + row * S::kPitch + c);
          float4 f[8];
#pragma unroll
          for (int r = 0; r < 8; ++r)
            f[r] = r < static_cast<int>(csize) ? load4_at(at_rank(from, r)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          float4 v = f[0];
#pragma unroll
          for (int r = 1; r < 8; ++r) {
            v.x += f[r].x;
            v.y += f[r].y;
            v.z += f[r].z;
            v.w += f[r].w;
          }
          const int64_t to = at.row0 + row;
          if (p.out_dtype == ES_BF16) store4<__nv_bfloat16>(p, to, at.col0 + c, v);
          else if (p.out_dtype == ES_F16) store4<__half>(p, to, at.col0 + c, v);
          else store4<float>(p, to, at.col0 + c, v);
        }
        __syncwarp();
        if (lane < static_cast<int>(csize)) arrive_at(at_rank(smem_u32(&ctl.red_empty), lane));
        red_phase ^= 1;
      } else if (any) {
        uint8_t* stage = out_smem + (warp - 4) * 4096;
        const int row0 = at.row0 + first;
        if (p.out_dtype == ES_BF16) store_rows<__nv_bfloat16, COLS>(p, stage, total, row0, rows, col0);
        else if (p.out_dtype == ES_F16) store_rows<__half, COLS>(p, stage, total, row0, rows, col0);
        else store_rows<float, COLS>(p, stage, total, row0, rows, col0);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (csize > 1) cluster_sync();
  tc_fence_after();
  if (warp == 1) tc_dealloc<CG>(tmem, S::kColumns);
}

template <typename S>
int launch(const Fp8Args& p, const Fp8Maps& m, int64_t max_tiles, int csize, cudaStream_t stream) {
  constexpr size_t fixed = 1024 + static_cast<size_t>(S::kStages) * S::kStageBytes + S::kOutBytes;
  constexpr size_t most = fixed + (3 * kMaxExperts + 1) * sizeof(int);
  static_assert(most <= 227 * 1024 - sizeof(Fp8Ctl) - 1024, "shared memory of an SM");
  static std::atomic<bool> raised[kMaxAttrDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return ES_ERR_CUDA;
  const bool tracked = dev >= 0 && dev < kMaxAttrDevices;
  if (!tracked || !raised[dev].load(std::memory_order_relaxed)) {
    cudaFuncAttributes attrs;
    if (cudaFuncGetAttributes(&attrs, fp8_tc_kernel<S>) != cudaSuccess) return ES_ERR_CUDA;
    if (S::kSplitRegs && attrs.numRegs < kLaunchRegs) return ES_ERR_UNSUPPORTED;
    if (cudaFuncSetAttribute(fp8_tc_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)) !=
        cudaSuccess)
      return ES_ERR_CUDA;
    if (tracked) raised[dev].store(true, std::memory_order_relaxed);
  }
  int64_t clusters = kSMs / csize;
  if (clusters > max_tiles) clusters = max_tiles;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * csize));
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = fixed + (3 * p.g.groups() + 1) * sizeof(int);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = csize;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, fp8_tc_kernel<S>, p, m) != cudaSuccess) {
    cudaGetLastError();
    return ES_ERR_CUDA;
  }
  count_launch();
  return ES_OK;
}

struct Fp8Form {
  int path;
  int rows, cols;
  int split;  // CTAs that share a tile's depth
  int64_t tiles;
};

Fp8Form form_of(const GroupedArgs& g) {
  const int64_t R = g.rows, groups = g.groups();
  const int64_t live = groups < R ? groups : R;  // groups that can have rows
  const int64_t mean = R / live;
  auto form = [&](int path, int rows, int cols) {
    return Fp8Form{path, rows, cols, 1, (R / rows + live) * ((g.N + cols - 1) / cols)};
  };
  const Fp8Form wide = form(ES_GROUPED_WIDE, 256, 256);
  if (mean > 128 && wide.tiles >= kSMs / 2) return wide;
  Fp8Form narrow = form(ES_GROUPED_NARROW, 128, 128);
  const int64_t nkb = (g.K + 127) / 128;
  while (narrow.split < 8 && narrow.tiles * narrow.split * 2 <= kSMs && nkb >= narrow.split * 4) narrow.split *= 2;
  if (narrow.split > 1) narrow.path = ES_GROUPED_SPLIT;
  return narrow;
}

struct Fp8Operands {
  Operand x, w;
};

Fp8Operands operands(const GroupedArgs& g, const void* x, const void* w) {
  const int64_t depth = g.groups() == 1 || g.w_e == 0 ? 1 : g.num_experts;
  return Fp8Operands{
      operand_of(x, kInt8, 1, g.order ? g.rows : g.x_rows, g.K, 0, g.x_stride, 1, g.order != nullptr),
      operand_of(w, kInt8, depth, g.N, g.K, g.w_e, g.w_n, 1, false)};
}

}  // namespace

bool fp8_tc_ok(const GroupedArgs& g) {
  return g.K > 0 && g.N > 0 && g.rows > 0 && g.x_rows > 0 &&
         (g.rows / 128 + g.groups()) * ((g.N + 127) / 128) < 0x7fffffffLL;
}

int fp8_tc_path(const GroupedArgs& g) { return form_of(g).path; }

size_t fp8_tc_workspace(const GroupedArgs& g, const void* x, const void* w) {
  const Fp8Operands o = operands(g, x, w);
  return o.x.bytes + o.w.bytes;
}

int fp8_tc(const GroupedArgs& g, const void* x, const void* w, void* y, int out_dtype, void* workspace,
           int32_t* status, cudaStream_t stream) {
  Fp8Operands o = operands(g, x, w);
  ES_TRY(lay_out(g, o.x, kInt8, true, false, workspace, stream));
  ES_TRY(lay_out(g, o.w, kInt8, false, o.w.depth > 1, static_cast<char*>(workspace) + o.x.bytes, stream));
  const Fp8Form f = form_of(g);
  Fp8Args p{};
  p.g = g;
  p.out = y;
  p.out_dtype = out_dtype;
  p.col_tiles = static_cast<int>((g.N + f.cols - 1) / f.cols);
  p.expert_step = o.w.depth > 1 ? 1 : 0;
  p.k_blocks = static_cast<int>((g.K + 127) / 128);
  p.n_blocks = static_cast<int>((g.N + 127) / 128);
  const int64_t esz = out_dtype == ES_F32 ? 4 : 2;
  p.wide = g.N * esz % 16 == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
  p.status = status;
  Fp8Maps m{};
  if (!bind_context() || !encode_operand(o.x, kInt8, 128, kBoxRows, 2, &m.x) ||
      !encode_operand(o.w, kInt8, 128, kBoxRows, 3, &m.w))
    return ES_ERR_CUDA;
  if (f.path == ES_GROUPED_WIDE) return launch<Fp8Shape<2, 256, false>>(p, m, f.tiles, 2, stream);
  if (f.path == ES_GROUPED_NARROW) return launch<Fp8Shape<1, 128, false>>(p, m, f.tiles, 1, stream);
  return launch<Fp8Shape<1, 128, true>>(p, m, f.tiles, f.split, stream);
}

}  // namespace es
