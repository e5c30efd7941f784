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
// a block. (With channels in the lanes, as in grouped_tc.cu, each column would need its
// own, read from shared memory, whose bandwidth the MMAs need.)
// The price is that a group's last tile multiplies empty lanes, which costs nothing where
// few rows leave the product bound by reading W. Results go through shared memory, a
// warp's part of a tile as one or two TMA stores.
//
// Roles and waits as in grouped_tc.cu: warp 0 issues the TMA loads, warp 1 the MMAs,
// warps 2-3 make the products of the scales, eight blocks ahead (loaded by the epilogue's
// threads they cost a quarter of the time), and clear the rows of no expert, warps 4-11
// read the accumulators. Every wait is bounded.
//
// Bounds (B200, measured): 8191 x 4096 x 8192 in 224 to 249 us (2.2 to 2.45 PFLOP/s; the
// 8-bit integers' product, whose sums need no scale, 166 to 184). The tensor pipe is busy
// for about half of it: a block of 256 x 256 x 128 takes the MMAs 512 cycles, the epilogue
// about 900, most of them a chain of waits (for the sums, for TMEM's reads, for the
// other CTA) that two accumulators of 256 columns, all that TMEM holds, cannot cover; its
// 64 packed multiply-adds a thread are 130 of them. 16400 rows of 64 experts, 2048 x 2816,
// 134 us (2.8 TB/s of HBM; tiles of 256 rows are two thirds full), 16 rows x 4096 x 4096
// 13 us, where clusters, TMEM and tensor maps take longer than reading W (2.6).
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
constexpr int kFewRows = 32;    // rows of the smaller TMA box
constexpr int kScalesAhead = 8; // blocks of depth whose scales are made together
constexpr int kScaleSlots = 2;  // of so many blocks
constexpr int kScalePitch = 132;  // scales of 128 rows, and no bank met twice
constexpr int kTileBlock = 8;   // row tiles that share a channel tile's weights in L2
constexpr int kWarpOut = 8192;  // an epilogue warp's staging of the output
constexpr int kMaxStages = 8;
constexpr int kMaxBufs = 4;     // accumulators

struct Fp8Args {
  GroupedArgs g;
  void* out;
  int out_dtype;
  int col_tiles;
  int expert_step;         // 0: every expert has the same matrix
  int k_blocks, n_blocks;  // scales of a row, rows of scales of a matrix
  int wide;                // 16-byte stores, and TMA's
  int32_t* status;
};

// Boxes of 128 rows of X and W: a box costs the TMA unit some 130 cycles, so boxes of
// 32 rows fed the MMAs at two thirds of the rate. Tiles of up to 32 rows read one of 32.
struct Fp8Maps {
  CUtensorMap x, x_few, w, out;
};

struct Fp8Ctl {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t acc_full[kMaxBufs];
  uint64_t acc_empty[kMaxBufs];
  uint64_t scale_full[kScaleSlots];
  uint64_t scale_empty[kScaleSlots];
  uint64_t red_full, red_empty;
  uint64_t drain;
  int any_coarse[kScaleSlots][4];  // of 32 rows, whether one of them is coarse from this slot on
  int8_t coarse[kScaleSlots][2][128];
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
  static constexpr int kBlocks = NT / 128;  // blocks of channels
  static constexpr int kBufs = 512 / NT;    // accumulators
  static constexpr int kStageBytes = kABytes + NT / CG * 128;
  static constexpr int kPitch = NT + 4;  // floats of a row of a split tile's part: no bank is met twice
  static constexpr int kOutBytes = SPLIT ? 128 * kPitch * 4 : kEpiWarps * kWarpOut;
  static constexpr int kScaleBytes = kScaleSlots * kScalesAhead * kBlocks * kScalePitch * 4;
  static constexpr int kFit = (213 * 1024 - kOutBytes - kScaleBytes) / kStageBytes;
  static constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
  static constexpr bool kSplitRegs = kCols == 128;  // 128 totals and 64 sums a thread
  static_assert(!SPLIT || CG == 1, "a cluster shares the depth or the rows");
  static_assert(NT / CG == 128, "one box of W a stage");
};

// One output tile, and which blocks of its depth this CTA multiplies.
struct Fp8Tile {
  int expert;
  int row0, rows;
  int col0;
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

// The product of two scales may be past fp32's ends where the result is not. Products and
// totals are therefore held times 2^40: below the normal numbers they then lose at most
// 2^-190 of the product and 2^-165 of a term, less than any result holds. A row that meets a
// product of 2^36 or more (whose totals could overflow) goes on in coarse products and
// totals, times 2^-40: its total is multiplied by 2^-80 once, between two slots, and terms
// below 2^-85 may be lost beside such a product. No total is ever multiplied by more than
// one, so what a row has summed stays what it is, whatever blocks come next (blocks of
// zeros, which have the least scale, among them), and the sums themselves cost nothing more
// (a second factor for every value cost them a tenth, a second loop for such slots 2.5%).
constexpr float kHalfFine = 0x1p20f, kFine = 0x1p40f, kCoarse = 0x1p-40f, kLargest = 0x1p76f;

__device__ __forceinline__ float fine_product(float x, float w) {
  return fabsf(x) < 1.0f ? (x * kFine) * w : x * (w * kFine);
}

// Where even the coarse product is past the largest number every sum but zero has an
// infinite term, as it has with the largest number; infinite scales stay infinite.
__device__ __forceinline__ float coarse_product(float x, float w) {
  const float s = fabsf(x) < 1.0f ? x * (w * kCoarse) : (x * kCoarse) * w;
  return fabsf(s) == INFINITY && fabsf(x) < INFINITY && fabsf(w) < INFINITY ? copysignf(FLT_MAX, s) : s;
}

template <int COLS>
__device__ __forceinline__ void scale_totals(float (&total)[COLS], float f) {
#pragma unroll
  for (int i = 0; i < COLS; ++i) total[i] *= f;
}

// The scale of block kb of the channels from col on (their block of 128; col may lie
// behind the last).
__device__ __forceinline__ const float* channel_scales(const Fp8Args& p, int expert, int64_t col, int kb) {
  const int64_t block = min(col >> 7, static_cast<int64_t>(p.n_blocks) - 1);
  return p.g.w_scale + (static_cast<int64_t>(expert) * p.n_blocks + block) * p.k_blocks + kb;
}

// A block of depth: its four MMAs and the arrivals of their end, by one elected lane of a
// converged warp (one statement: with an election for each, issuing took as long as the
// tensor cores' work).
template <int CG>
__device__ __forceinline__ void mma_block(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint64_t* acc_full,
                                          uint64_t* empty) {
#define ES_BLOCK(group, commit_form, mask)                                                                       \
  asm volatile(                                                                                                  \
      "{\n\t.reg .pred e, z, o;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\telect.sync _|e, 0xffffffff;\n\t"               \
      "setp.ne.b32 z, 0, 0;\n\tsetp.eq.b32 o, 0, 0;\n\t"                                                         \
      "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"                                       \
      "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"                                       \
      "@e tcgen05.mma.cta_group::" group ".kind::f8f6f4 [%0], %1, %2, %3, z;\n\t"                               \
      "@e tcgen05.mma.cta_group::" group ".kind::f8f6f4 [%0], a1, b1, %3, o;\n\t"                               \
      "@e tcgen05.mma.cta_group::" group ".kind::f8f6f4 [%0], a2, b2, %3, o;\n\t"                               \
      "@e tcgen05.mma.cta_group::" group ".kind::f8f6f4 [%0], a3, b3, %3, o;\n\t"                               \
      "@e tcgen05.commit.cta_group::" group ".mbarrier::arrive::one.shared::cluster" commit_form ".b64 [%4]" mask  \
      ";\n\t"                                                                                                    \
      "@e tcgen05.commit.cta_group::" group ".mbarrier::arrive::one.shared::cluster" commit_form ".b64 [%5]" mask  \
      ";\n\t}" ::"r"(d),                                                                                         \
      "l"(a), "l"(b), "r"(idesc), "r"(smem_u32(acc_full)), "r"(smem_u32(empty)), "h"(static_cast<uint16_t>(3))   \
      : "memory")
  if constexpr (CG == 2)
    ES_BLOCK("2", ".multicast::cluster", ", %6");
  else
    ES_BLOCK("1", "", "");
#undef ES_BLOCK
}

// Two totals at once.
__device__ __forceinline__ void fma2(float& t0, float& t1, float a, float b, float s) {
  asm("{\n\t.reg .b64 v, t, f;\n\tmov.b64 v, {%2, %3};\n\tmov.b64 t, {%0, %1};\n\tmov.b64 f, {%4, %4};\n\t"
      "fma.rn.f32x2 t, v, f, t;\n\tmov.b64 {%0, %1}, t;\n\t}"
      : "+f"(t0), "+f"(t1)
      : "f"(a), "f"(b), "f"(s));
}

template <typename T>
__device__ __forceinline__ uint4 pack16(const float* v) {
  alignas(16) T o[16 / sizeof(T)];
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) o[i] = from_f32<T>(v[i]);
  return *reinterpret_cast<uint4*>(o);
}

// Rounds and stores a warp's 32 rows (a lane's each) of COLS channels through the warp's
// 8 KB of shared memory, in blocks of 32 rows x 128 bytes whose 16-byte pieces are swapped
// by the row, as TMA reads them: a whole block is one TMA store, which runs under the next
// tile; a row at a time, or by the warps themselves, the stores of a tile took 5000 cycles.
// What no TMA store may write (rows behind the group's, odd addresses) the warp stores.
template <typename T, int COLS>
__device__ __forceinline__ void store_rows(const Fp8Args& p, const CUtensorMap* map, uint8_t* stage,
                                           const float (&total)[COLS], int row0, int rows, int64_t col0) {
  constexpr int VEC = 16 / sizeof(T), BLOCK = 8 * VEC, PASS = COLS < 2 * BLOCK ? COLS : 2 * BLOCK;
  const int lane = threadIdx.x & 31, j = lane & 7;
  const bool whole = p.wide && rows >= 32;
#pragma unroll
  for (int c = 0; c < COLS; c += PASS) {
    if (lane == 0) bulk_wait_read();
    __syncwarp();
#pragma unroll
    for (int i = 0; i < PASS / VEC; ++i)
      reinterpret_cast<uint4*>(stage + i / 8 * 4096 + lane * 128)[(i & 7) ^ j] = pack16<T>(total + c + i * VEC);
    if (whole) fence_proxy_async();
    __syncwarp();
    if (whole) {
      if (lane == 0) {
#pragma unroll
        for (int i = 0; i < PASS / BLOCK; ++i)
          if (col0 + c + i * BLOCK < p.g.N)
            tma_store_2d(map, stage + i * 4096, static_cast<int>((col0 + c + i * BLOCK) * sizeof(T)), row0);
        bulk_commit();
      }
    } else {
      for (int r = lane >> 3; r < min(rows, 32); r += 4) {
#pragma unroll
        for (int i = 0; i < PASS / BLOCK; ++i) {
          const uint4 v = reinterpret_cast<const uint4*>(stage + i * 4096 + r * 128)[j ^ (r & 7)];
          const int64_t col = col0 + c + i * BLOCK + j * VEC;
          T* out = static_cast<T*>(p.out) + static_cast<int64_t>(row0 + r) * p.g.N + col;
          if (p.wide && col + VEC <= p.g.N) {
            *reinterpret_cast<uint4*>(out) = v;
          } else {
            const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
            for (int q = 0; q < VEC; ++q)
              if (col + q < p.g.N) out[q] = e[q];
          }
        }
      }
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
  constexpr int CG = S::CG, NT = S::NT, STAGES = S::kStages, BUFS = S::kBufs, COLS = S::kCols, BLOCKS = S::kBlocks;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Fp8Ctl ctl;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* out_smem = smem_raw + (base - smem_u32(smem_raw)) + STAGES * S::kStageBytes;
  float* scale_smem = reinterpret_cast<float*>(out_smem + S::kOutBytes);
  int* pre = reinterpret_cast<int*>(out_smem + S::kOutBytes + S::kScaleBytes);
  const int groups = p.g.groups();
  int* lo = pre + groups + 1;
  int* cnt = lo + groups;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank(), csize = cluster_size();
  const uint32_t pair_rank = CG == 2 ? rank : 0;
  const bool leader = pair_rank == 0;

  if (threadIdx.x == 0) {
    prefetch_map(&m.x);
    prefetch_map(&m.x_few);
    if (p.wide) prefetch_map(&m.out);
    prefetch_map(&m.w);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&ctl.full[s], 1);
      mbar_init(&ctl.empty[s], 1);
    }
    for (int b = 0; b < BUFS; ++b) {
      mbar_init(&ctl.acc_full[b], 1);
      mbar_init(&ctl.acc_empty[b], CG * kEpiWarps);
    }
    for (int s = 0; s < kScaleSlots; ++s) {
      mbar_init(&ctl.scale_full[s], 2);
      mbar_init(&ctl.scale_empty[s], kEpiWarps);
    }
    mbar_init(&ctl.red_full, csize * kEpiWarps);
    mbar_init(&ctl.red_empty, csize * kEpiWarps);
    mbar_init(&ctl.drain, 1);
    ctl.abort = 0;
    ctl.progress = 0;
    fence_mbar_init();
  }
  if (warp == 1) tc_alloc<CG>(&ctl.tmem, BUFS * NT);
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
        // X's rows past the tile's are read where its box holds them: their lanes are not stored
        auto x_rows = [&](int r) { return at.rows <= r * 128 ? 0 : at.rows <= r * 128 + kFewRows ? kFewRows : 128; };
        const int mine = x_rows(static_cast<int>(pair_rank));
        const uint32_t bytes = (CG * 128 + x_rows(0) + (CG == 2 ? x_rows(1) : 0)) * 128;
        const int x_row = at.row0 + static_cast<int>(pair_rank) * 128;
        const int w_row = at.col0 + static_cast<int>(pair_rank) * 128;
        const int z = at.expert * p.expert_step;
        for (int kb = at.kb0; kb < at.kb1; ++kb) {
          int go = 0;
          if (lane == 0) {
            go = tc_wait<true>(&ctl.empty[stage], phase ^ 1, &ctl, p.status) ? 1 : 0;
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
          if (lane == 0) {
            if (mine) load_2d<CG>(sa, mine == 128 ? &m.x : &m.x_few, kb * 128, x_row, bar);
            load_3d<CG>(sb, &m.w, kb * 128, w_row, z, bar);
          }
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
        const uint64_t first = operand(base, false);  // of a stage's A; its B lies kABytes behind
        int stage = 0, buf = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int t = t0; t < total_tiles && ok; t += step) {
          const Fp8Tile at = tiles.at(t, rank, csize);
          // D f32, A and B e4m3 (0) and K-major
          constexpr uint32_t idesc = (1u << 4) | ((static_cast<uint32_t>(NT) >> 3) << 17) | ((8u * CG) << 24);
          for (int kb = at.kb0; kb < at.kb1; ++kb) {
            ok = tc_wait_warp<true>(&ctl.full[stage], phase, &ctl, p.status) &&
                 tc_wait_warp<true>(&ctl.acc_empty[buf], acc_phase ^ 1, &ctl, p.status);
            if (!ok) break;
            tc_fence_after();
            const uint64_t da = first + stage * (S::kStageBytes >> 4);
            mma_block<CG>(tmem + buf * NT, da, da + (kABytes >> 4), idesc, &ctl.acc_full[buf], &ctl.empty[stage]);
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
      // -------------------------------------------------------------- scales
      // the two scales' products of kScalesAhead blocks, for 64 rows a warp and each 128
      // channels; eight lanes a row, so that a sector is read once
      const int row0 = (warp - 2) * 64, b = lane & 7;
      int slot = 0;
      uint32_t slot_phase = 0;
      bool ok = true;
      for (int t = t0; t < total_tiles && ok; t += step) {
        const Fp8Tile at = tiles.at(t, rank, csize);
        int source[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = static_cast<int>(pair_rank) * 128 + row0 + i * 32 + lane;
          source[i] = r < at.rows ? static_cast<int>(p.g.source(at.row0 + r)) : -1;
        }
        uint32_t coarse = 0;  // bit (s * 2 + half) * 8 + i: this lane's row is coarse
        for (int kb = at.kb0; kb < at.kb1; kb += kScalesAhead) {
          ok = tc_wait_warp<true>(&ctl.scale_empty[slot], slot_phase ^ 1, &ctl, p.status, true);
          if (!ok) break;
          const bool there = kb + b < at.kb1;
          // either scale times 2^20: where that is past the largest number, the product is looked at again
          float w[BLOCKS];
#pragma unroll
          for (int s = 0; s < BLOCKS; ++s)
            w[s] = there ? *channel_scales(p, at.expert, at.col0 + s * 128, kb + b) * kHalfFine : 0.0f;
          float* to = scale_smem + (slot * kScalesAhead + b) * BLOCKS * kScalePitch + row0 + (lane >> 3);
          const float* from = p.g.x_scale + kb + b;
#pragma unroll 1
          for (int half = 0; half < 2; ++half, to += 32) {
            auto row_scale = [&](int i) {
              const int r = __shfl_sync(0xffffffffu, half ? source[1] : source[0], i * 4 + (lane >> 3));
              return there && r >= 0 ? from[static_cast<int64_t>(r) * p.k_blocks] : 0.0f;
            };
            float x[8];
            bool any = coarse != 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = row_scale(i) * kHalfFine;
#pragma unroll
            for (int s = 0; s < BLOCKS; ++s)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float v = x[i] * w[s];
                to[s * kScalePitch + i * 4] = v;
                any |= !(fabsf(v) < kLargest);
              }
            any = __any_sync(0xffffffffu, any);
            if (any) {
              const uint32_t row = 0xffu << (lane & 24);
#pragma unroll 1
              for (int n = 0; n < 8 * BLOCKS; ++n) {
                const int i = n & 7, s = n >> 3;
                const uint32_t bit = 1u << ((s * 2 + half) * 8 + i);
                const float xs = row_scale(i), ws = there ? *channel_scales(p, at.expert, at.col0 + s * 128, kb + b) : 0.0f;
                const float v = fine_product(xs, ws);
                const bool large = fabsf(v) >= kLargest && fabsf(xs) < INFINITY && fabsf(ws) < INFINITY;
                if (__ballot_sync(0xffffffffu, large) & row) coarse |= bit;
                to[s * kScalePitch + i * 4] = coarse & bit ? coarse_product(xs, ws) : v;
                if (b == 0) ctl.coarse[slot][s][row0 + half * 32 + (lane >> 3) + i * 4] = (coarse & bit) != 0;
              }
            }
            if (lane == 0) ctl.any_coarse[slot][(warp - 2) * 2 + half] = any;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl.scale_full[slot]);
          if (++slot == kScaleSlots) {
            slot = 0;
            slot_phase ^= 1;
          }
        }
      }
      // rows of no expert
      clear_rows(p, p.g.kept(), p.g.rows, blockIdx.x * 64LL + (threadIdx.x - 64), gridDim.x * 64LL);
    }
  } else {
    if constexpr (S::kSplitRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
    // ------------------------------------------------------------- epilogue
    const int quad = warp & 3, set = (warp - 4) >> 2, column = set * COLS;
    int buf = 0;
    uint32_t acc_phase = 0, red_phase = 0;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      int go = 1;
      if (lane == 0) go = tc_wait(bar, parity, &ctl, p.status, true) ? 1 : 0;
      return __shfl_sync(0xffffffffu, go, 0) != 0;
    };
    bool ok = true;
    const int first = static_cast<int>(pair_rank) * 128 + quad * 32;  // this warp's rows of a tile
    int slot = 0;
    uint32_t slot_phase = 0;
    for (int t = t0; t < total_tiles; t += step) {
      const Fp8Tile at = tiles.at(t, rank, csize);
      const int rows = at.rows - first, col0 = at.col0 + column;
      const bool any = rows > 0 && col0 < p.g.N;
      bool coarse = false;
      float total[COLS];
#pragma unroll
      for (int i = 0; i < COLS; ++i) total[i] = 0.0f;
      for (int kb0 = at.kb0; kb0 < at.kb1; kb0 += kScalesAhead) {
        ok = tc_wait_warp<true>(&ctl.scale_full[slot], slot_phase, &ctl, p.status, true);
        if (!ok) break;
        const float* scales =
            scale_smem + (slot * kScalesAhead * BLOCKS + (column >> 7)) * kScalePitch + quad * 32 + lane;
        bool on = coarse;
        if (ctl.any_coarse[slot][quad]) on = ctl.coarse[slot][column >> 7][quad * 32 + lane] != 0;
        if (__any_sync(0xffffffffu, on != coarse)) {
          scale_totals(total, on != coarse ? kCoarse * kCoarse : 1.0f);
          coarse = on;
        }
        const int n = min(at.kb1 - kb0, kScalesAhead);
        for (int i = 0; i < n; ++i) {
          const float s = scales[i * BLOCKS * kScalePitch];
          ok = tc_wait_warp<true>(&ctl.acc_full[buf], acc_phase, &ctl, p.status, true);
          if (!ok) break;
          tc_fence_after();
          const uint32_t acc = tmem + buf * NT + (static_cast<uint32_t>(quad * 32) << 16) + column;
          auto release = [&] {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_done_at(at_rank(smem_u32(&ctl.acc_empty[buf]), CG == 2 ? 0 : rank));
          };
          if (any) {
            // 64 columns at a time: smaller reads wait longer for TMEM (32: 252 us where this takes 242)
#pragma unroll
            for (int c = 0; c < COLS; c += 64) {
              uint32_t v[2][32];
              tmem_ld32_async(acc + c, v[0]);
              tmem_ld32_async(acc + c + 32, v[1]);
              tmem_wait32(v[0]);
              tmem_wait32(v[1]);
              if (c + 64 == COLS) release();
#pragma unroll
              for (int j = 0; j < 64; j += 2)
                fma2(total[c + j], total[c + j + 1], __uint_as_float(v[j >> 5][j & 31]),
                     __uint_as_float(v[j >> 5][(j & 31) + 1]), s);
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
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.scale_empty[slot]);
        if (++slot == kScaleSlots) {
          slot = 0;
          slot_phase ^= 1;
        }
      }
      if (!ok) break;
      scale_totals(total, coarse ? kFine : kCoarse);
      if constexpr (S::SPLIT) {
        // every CTA puts its part into shared memory, [row][channel], and adds up every
        // csize-th piece of four channels, the parts in the CTAs' order
        ok = wait(&ctl.red_empty, red_phase ^ 1);  // the last tile's parts have been read by the whole cluster
        if (!ok) break;
        float* part = reinterpret_cast<float*>(out_smem);
        if (lane < rows) {
          float4* mine = reinterpret_cast<float4*>(part + (first + lane) * S::kPitch + column);
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
        uint8_t* stage = out_smem + (warp - 4) * kWarpOut;
        if (p.out_dtype == ES_BF16) store_rows<__nv_bfloat16, COLS>(p, &m.out, stage, total, at.row0 + first, rows, col0);
        else if (p.out_dtype == ES_F16) store_rows<__half, COLS>(p, &m.out, stage, total, at.row0 + first, rows, col0);
        else store_rows<float, COLS>(p, &m.out, stage, total, at.row0 + first, rows, col0);
      }
    }
  }
  bulk_wait();
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (csize > 1) cluster_sync();
  tc_fence_after();
  if (warp == 1) tc_dealloc<CG>(tmem, BUFS * NT);
}

template <typename S>
int launch(const Fp8Args& p, const Fp8Maps& m, int64_t max_tiles, int csize, cudaStream_t stream) {
  constexpr size_t fixed = 1024 + static_cast<size_t>(S::kStages) * S::kStageBytes + S::kOutBytes + S::kScaleBytes;
  constexpr size_t most = fixed + (3 * kMaxExperts + 1) * sizeof(int);
  static_assert(most + sizeof(Fp8Ctl) <= 227 * 1024, "shared memory of a CTA");
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
  // By the rows of a group, where the tiles then fill the SMs. 64 experts, 2048 x 2816, us for
  // Narrow, Wide: 64 rows a group 87, 108; 96 rows 90, 112; 128 rows 117, 114; 256 rows 196, 168.
  // One matrix of 4096 x 4096: 512 rows 16, 21 (48 wide tiles); 1024 rows 27, 21 (80)
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
  p.wide = g.N * esz % 16 == 0 && g.N * esz <= 0x7fffffffLL && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
  p.status = status;
  Fp8Maps m{};
  if (!bind_context() || !encode_operand(o.x, kInt8, 128, 128, 2, &m.x) ||
      !encode_operand(o.x, kInt8, 128, kFewRows, 2, &m.x_few) || !encode_operand(o.w, kInt8, 128, 128, 3, &m.w))
    return ES_ERR_CUDA;
  if (p.wide && !encode_bytes(y, g.N * esz, g.rows, 128, 32, &m.out)) return ES_ERR_CUDA;
  if (f.path == ES_GROUPED_WIDE) return launch<Fp8Shape<2, 256, false>>(p, m, f.tiles, 2, stream);
  if (f.path == ES_GROUPED_NARROW) return launch<Fp8Shape<1, 128, false>>(p, m, f.tiles, 1, stream);
  return launch<Fp8Shape<1, 128, true>>(p, m, f.tiles, f.split, stream);
}

}  // namespace es
