// Products grouped by expert on the tensor cores (tcgen05 + TMEM + TMA), with
// ragged group sizes: the rows' product (forward, and the gradient of the
// rows with the weights read transposed), the weights' gradient, and the
// product of 8-bit integers.
//
// Orientation. The 128 lanes of the accumulator (256 for a pair of CTAs) are
// the dimension that never is ragged, the output channels; the columns are a
// group's rows:  D[channel, row] = sum_k W[channel, k] X[row, k].  The width
// of an MMA (a multiple of 16, or 32 for a pair) is set tile by tile to the
// rows that are left, so a group of 3 rows costs a 16-wide MMA and no padding,
// and one kernel serves a decode step and a long prompt. For the weights'
// gradient lanes and columns are its two dimensions and the sum runs over the
// group's rows; of a group's last block only the 16-row steps that hold rows
// are multiplied, and the last of them is gathered row by row (tile::gather4)
// with the missing rows pointing outside of the tensor, which reads zeros (so
// that infinities of the next group stay out of it).
//
// Operands are read as they lie: K-major or MN-major, through 128-byte
// swizzled TMA boxes. Routed tokens are first copied into the rows' order: TMA
// row gathers in the main loop (tile::gather4, four rows an instruction) took
// 2.76 ms where the copy and box loads take 1.0 ms (16384 rows, 4096 x 8192,
// bf16). What TMA cannot read (odd addresses or strides) is copied too.
//
// fp32 operands are cut into three bf16 planes, x / 2 = b0 + b1 + b2 (split3). A
// block of depth takes three stages, one for each plane, and the six products
// b_i b_j with i + j <= 2 are made from them (each operand crosses from L2
// once): b0 b0 into one accumulator, the other five, at most 2^-8 of it, into a
// second. What is left out is at most 2^-24 of a product.
//
// Gated products. The two accumulators of a tile are gate and up of the same output
// channels and rows (their operands have maps of their own, `a` and `up`), and the
// epilogue is the activation, the product and, for a training step, the slopes. 60 experts
// of 2048 x 1408 with 69 rows each 112 us, 6.2 TB/s of HBM, which bounds it; a dense
// training step's 8192 rows, 4096 x 8192, bf16, 772 us without the fp32 slopes' 0.5 GB (then
// 808): the epilogue's exp and stores hold up the next tile's MMAs, since TMEM has room for
// one tile.
//
// Long sums. An accumulator truncates what it adds, so sums of one sign come out
// low (measured, relative, bf16 / f16 operands: 7e-7 / 2.5e-6 at a depth of 512, 1.1e-5 /
// 2.3e-5 at 4096, 1.4e-4 / 1.2e-4 at 16384, 1.1e-3 / 8e-4 at 131072). fp32 sums are
// therefore cut into chains of 448, which the epilogue adds in fp32 (6e-7 at any depth).
// 16-bit results keep one chain while its error is a quarter of their rounding
// (one_chain); longer sums (DEEP) are chains of 4096 whose fp32 total stands beside the
// accumulator in TMEM.
//
// Bounds (B200, measured): 16384 rows, 8 experts, 4096 x 8192, bf16 759 us
// forward, the tensor pipe 84% active (on equal groups 88%, as cuBLAS's product
// of that size); 60 experts of 2048 x 2816 with 69 rows each 115 us, 6.2 TB/s of
// HBM; 16 rows over 16 experts of 2048 x 4096 30 us, 5.0 TB/s; 8 bits, 8191 x
// 4096 x 8192 179 to 184 us, 3.0 POP/s, but 16400 rows of 64 experts, 2048 x 1408, 72 us
// with the tensor pipe 33% active: a tile's hand-over takes 11k cycles whatever its
// depth; fp32, 3000 rows, 16 experts, 1000 x 2024 92 us without the planes' 59 us.
// Before the 512 x 256 tile a long group's bound was the L2's bandwidth to the SMs (64
// bytes a clock and SM for 256 x 256).
//
// Roles (12 warps): warp 0 issues the TMA loads, warp 1 the MMAs (an elected
// lane), warps 2-3 clear the output rows of no expert, warps 4-11 read the
// accumulators (TMEM lane quadrant = warp % 4) and write the output. Tiles are
// dealt to the CTAs in turn; where two tiles fit TMEM a tile's epilogue runs
// under the next tile's MMAs (else see drain_held). Every wait is bounded: when one
// runs out the CTA sets ES_ERR_TIMEOUT, drains its copies and MMAs, frees
// TMEM and returns.
#include "activation.cuh"
#include "grouped.cuh"
#include "tc_operands.cuh"
#include "tc_pipe.cuh"

namespace es {
namespace {

constexpr int kEpiWarps = 8;
constexpr int kTcThreads = 128 + 32 * kEpiWarps;
constexpr int kABytes = 16384;  // 128 lanes x 128 bytes of depth
constexpr int kSwizzleRow = 128;
constexpr int kBoxRows = 32;    // rows of one TMA box of X
constexpr int kTileBlock = 8;   // row tiles that share a channel tile's weights in L2
constexpr int kMaxTcStages = 8;

struct TcArgs {
  GroupedArgs g;
  void* out;
  int out_dtype;
  int64_t lanes;      // extent of the lane dimension
  int64_t cols;       // extent of the column dimension (weights' gradient)
  int64_t out_col;    // output stride of a column (rows: of a row)
  int64_t out_expert; // output stride of an expert (weights' gradient)
  int lane_tiles, col_tiles;
  int expert_step;    // 0: every expert has the same matrix
  int plane_experts;  // matrices of one plane of W
  int plane_rows;     // rows of one plane of X (and dY)
  int src_rows;       // rows of the weights' gradient's operands: this row index reads zeros
  uint32_t idesc;     // instruction descriptor without N
  int pairs;          // two neighbouring lanes may be stored together
  int most;           // weights' gradient: groups of more rows than this are the DEEP kernel's
  int activation;     // gated products
  float* slopes;      // (rows, 2 lanes) or NULL
  int32_t* status;
};

// Tensor maps of the operands. The weights' gradient reads a group's last block
// by steps of 16 rows and by gathers of single rows.
struct TcMaps {
  CUtensorMap a, b;
  CUtensorMap up;  // gated products: the second accumulator's lanes
  CUtensorMap a_steps, b_steps, a_rows, b_rows;
};

struct TcCtl {
  uint64_t full[kMaxTcStages];
  uint64_t empty[kMaxTcStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t red_full, red_empty;
  uint64_t scales;
  uint64_t drain;
  uint32_t tmem;
  int abort;
  uint32_t progress;
};

// ------------------------------------------------------------------- kernel

template <int CG_, int MT_, int NT_, int KIND_, bool A_MN_, bool WGRAD_, bool SPLIT_, int PLANES_, bool DEEP_ = false,
          bool GATED_ = false>
struct TcShape {
  static constexpr int CG = CG_;        // CTAs of one MMA
  static constexpr int MT = MT_;        // accumulators of 128 lanes (of each CTA) that share B
  static constexpr int NT = NT_;        // widest MMA
  static constexpr int KIND = KIND_;
  static constexpr bool A_MN = A_MN_;   // lanes contiguous in memory
  static constexpr bool WGRAD = WGRAD_;
  static constexpr bool SPLIT = SPLIT_; // the cluster's CTAs share one tile's depth
  static constexpr int PLANES = PLANES_;
  static constexpr int BK = KIND == kKindI8 ? 128 : 64;  // depth of a stage
  static constexpr bool DEEP = DEEP_;   // an fp32 total in TMEM
  static constexpr int kChain = PLANES > 1 ? 7 : DEEP ? 64 : 1 << 30;  // blocks of depth between fp32 additions
  static constexpr bool GATED = GATED_;  // the two accumulators are gate and up of the same lanes
  static constexpr int kLanes = 128 * (GATED ? 1 : MT) * CG;
  static constexpr int kAccs = PLANES > 1 ? 2 : MT;         // accumulators of a tile
  static constexpr int kTotal = DEEP ? NT : 0;              // columns of the total
  static constexpr int kBufs = 2 * kAccs * NT + kTotal <= 512 ? 2 : 1;  // tiles in TMEM
  static constexpr int kUsed = kBufs * kAccs * NT + kTotal;
  static constexpr int kColumns = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;  // allocated
  static constexpr bool kHeld = kBufs == 1 && PLANES == 1 && !DEEP;  // tiles are held in registers, see drain_held
  static constexpr bool kSums = PLANES > 1 && !WGRAD && !SPLIT;  // the epilogue adds chains in registers
  static constexpr int kStageBytes = MT * kABytes + NT / CG * kSwizzleRow;  // one plane of a block of depth
  static constexpr int kPartBytes = SPLIT ? MT * NT * 128 * 4 : 0;
  static constexpr int kStages =
      (200 * 1024 - kPartBytes) / kStageBytes > kMaxTcStages ? kMaxTcStages : (200 * 1024 - kPartBytes) / kStageBytes;
  static_assert(PLANES == 1 || MT == 1, "planes take the tiles that accumulators would share B with");
  static_assert(kStages > PLANES, "a block's planes and the next block's first");
  static_assert(!GATED || (MT == 2 && KIND == kKindF16 && !WGRAD && !DEEP), "gate and up in 16 bits");
  static_assert(!SPLIT || MT == 1 || GATED, "parts of one accumulator");
  static_assert(kUsed <= 512 && !(DEEP && (MT > 1 || PLANES > 1 || SPLIT)), "one accumulator and its total");

  // Tiles that the other kernel of the same call makes.
  __device__ static __forceinline__ bool skips(int depth, int most) { return WGRAD && (depth > most) != DEEP; }
};

// One output tile, and what of its depth this CTA multiplies.
struct TileAt {
  int expert;
  int64_t lane0;
  int row0;    // first row (rows) or first column (weights' gradient)
  int rows;    // rows or columns of the tile
  int first;   // weights' gradient: the group's first row
  int depth;   // depth of the product
  int kb0, kb1;
};

template <typename S>
struct Tiles {
  const TcArgs& p;
  const int* pre;   // [groups + 1] tiles before each group
  const int* lo;    // [groups]
  const int* cnt;   // [groups]
  int total;

  __device__ __forceinline__ TileAt at(int t, uint32_t rank, uint32_t split) const {
    TileAt r;
    int depth;
    int group, idx, tt;
    if constexpr (S::WGRAD) {
      const int per = p.lane_tiles * p.col_tiles;
      group = t / per;
      idx = t - group * per;
      tt = p.col_tiles;
    } else {
      int a = 0, b = p.g.groups();
      while (b - a > 1) {
        const int m = (a + b) >> 1;
        if (pre[m] <= t) a = m;
        else b = m;
      }
      group = a;
      idx = t - pre[a];
      tt = (cnt[a] + S::NT - 1) / S::NT;
    }
    // blocks of kTileBlock column tiles walk the lane tiles together
    const int block = idx / (kTileBlock * p.lane_tiles);
    const int in = idx - block * kTileBlock * p.lane_tiles;
    const int w = min(kTileBlock, tt - block * kTileBlock);
    const int lane_tile = in / w, col_tile = block * kTileBlock + in % w;
    r.expert = group;
    r.lane0 = static_cast<int64_t>(lane_tile) * S::kLanes;
    if constexpr (S::WGRAD) {
      r.row0 = col_tile * S::NT;
      r.rows = static_cast<int>(min(p.cols - r.row0, static_cast<int64_t>(S::NT)));
      r.first = lo[group];
      depth = cnt[group];
    } else {
      r.row0 = lo[group] + col_tile * S::NT;
      r.rows = min(cnt[group] - col_tile * S::NT, S::NT);
      r.first = 0;
      depth = static_cast<int>(p.g.K);
    }
    r.depth = depth;
    const int nkb = (depth + S::BK - 1) / S::BK;
    if constexpr (S::SPLIT) {
      r.kb0 = static_cast<int>(static_cast<int64_t>(nkb) * rank / split);
      r.kb1 = static_cast<int>(static_cast<int64_t>(nkb) * (rank + 1) / split);
    } else {
      r.kb0 = 0;
      r.kb1 = nkb;
    }
    return r;
  }
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Keeps the compiler from computing a stride's multiples ahead of the loop over
// tiles: they took 60 registers that the held accumulators need.
__device__ __forceinline__ void keep_here(int64_t& stride) { asm volatile("" : "+l"(stride)); }

template <typename T>
__device__ __forceinline__ void pack_cols(const float (&v)[32], uint32_t (&two)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) two[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
}

// Stores columns c < n, packed two to a register, to out + c * stride (out:
// this lane's channel). Two neighbouring lanes (channels) trade registers, so
// that the even one stores both channels of the even columns and the odd one
// of the odd columns, in 4-byte stores.
template <typename T>
__device__ __forceinline__ void store_packed(T* out, int64_t stride, const uint32_t (&two)[16], int n, bool live) {
  keep_here(stride);
  const int odd = threadIdx.x & 1;
  T* o = out - odd + odd * stride;
  const uint32_t take = odd ? 0x3276u : 0x5410u;  // the high halves (theirs, mine), or the low ones (mine, theirs)
#pragma unroll
  for (int c = 0; c < 32; c += 2) {
    const uint32_t theirs = __shfl_xor_sync(0xffffffffu, two[c / 2], 1);
    if (live && c + odd < n) *reinterpret_cast<uint32_t*>(o) = __byte_perm(two[c / 2], theirs, take);
    o += 2 * stride;
  }
}

// Stores v[c] (lane = this thread's channel) to out + c * stride, c < n.
template <typename T>
__device__ __forceinline__ void store_cols(T* out, int64_t stride, const float (&v)[32], int n, bool live,
                                           bool pairs) {
  if constexpr (sizeof(T) == 2) {
    if (pairs) {
      uint32_t two[16];
      pack_cols<T>(v, two);
      store_packed(out, stride, two, n, live);
      return;
    }
  }
  keep_here(stride);
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    if (live && c < n) *out = from_f32<T>(v[c]);
    out += stride;
  }
}

__device__ __forceinline__ void store_typed(void* out, int dtype, int64_t at, int64_t stride, const float (&v)[32],
                                            int n, bool live, bool pairs) {
  if (dtype == ES_BF16)
    store_cols(static_cast<__nv_bfloat16*>(out) + at, stride, v, n, live, pairs);
  else if (dtype == ES_F16)
    store_cols(static_cast<__half*>(out) + at, stride, v, n, live, pairs);
  else
    store_cols(static_cast<float*>(out) + at, stride, v, n, live, false);
}

__device__ __forceinline__ void store_one(void* out, int dtype, int64_t at, float v) {
  if (dtype == ES_BF16)
    static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16(v);
  else if (dtype == ES_F16)
    static_cast<__half*>(out)[at] = __float2half(v);
  else
    static_cast<float*>(out)[at] = v;
}

// Clears the output rows [from, to) with the threads `t` of `nt`.
__device__ __forceinline__ void clear_rows(const TcArgs& p, int64_t from, int64_t to, int64_t t, int64_t nt) {
  const int64_t esz = p.out_dtype == ES_F32 ? 4 : 2;
  char* a = static_cast<char*>(p.out) + from * p.g.N * esz;
  char* b = static_cast<char*>(p.out) + to * p.g.N * esz;
  const int64_t halves = (b - a) / 2;
  const int64_t head = min(halves, static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(a) & 15)) & 15) / 2);
  for (int64_t i = t; i < head; i += nt) reinterpret_cast<uint16_t*>(a)[i] = 0;
  uint4* mid = reinterpret_cast<uint4*>(a + head * 2);
  const int64_t n = (halves - head) / 8;
  for (int64_t i = t; i < n; i += nt) mid[i] = make_uint4(0, 0, 0, 0);
  for (int64_t i = head + n * 8 + t; i < halves; i += nt) reinterpret_cast<uint16_t*>(a)[i] = 0;
}

// A chain's sum from its two accumulators of halved planes: the products of the
// first planes, and the others. An infinity's other planes are zero, so its products
// with a value's lower planes are NaN or of either sign and belong to no sum: where
// the first planes' sum is infinite or NaN it alone is what fp32 arithmetic gives.
__device__ __forceinline__ float plane_sum(float first, float others) {
  return 4.0f * (fabsf(first) < INFINITY ? first + others : first);
}

// A row's scale in two factors, one of them 1: what is above 1 is multiplied last.
// A sum (at least 1, or 0) times a scale of up to 1 neither overflows nor loses
// bits, so that no step is infinite unless the result is.
__device__ __forceinline__ float2 scale_parts(float x) {
  return x > 1.0f ? make_float2(1.0f, x) : make_float2(x, 1.0f);
}

__device__ __forceinline__ float scaled(int sum, float first, float w, float last) {
  return static_cast<float>(sum) * first * w * last;
}

// The 8-bit product's sums times the scales of their rows (xs) and channel.
__device__ __forceinline__ void scale_block(float (&v)[32], const float2* xs, float w) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const float4 x = *reinterpret_cast<const float4*>(xs + i);
    v[i] = scaled(__float_as_int(v[i]), x.x, w, x.y);
    v[i + 1] = scaled(__float_as_int(v[i + 1]), x.z, w, x.w);
  }
}

// Reads one accumulator of an output tile. TMEM holds a single tile of this
// size, so the next tile's MMAs wait for this: a 16-bit tile (packed) and the last
// blocks of 32 columns of an fp32 one are held in registers, a few of them spilled (45 in
// 16 bits, 92 in 8), and stored after the accumulator has been handed back (`release`).
// xs, w: scales of 8-bit operands (I8).
constexpr int kAtOnce32 = 3; // blocks of fp32 tiles that are stored at once: the rest fits the registers

template <typename T, bool I8, typename Release>
__device__ __forceinline__ void drain_held(uint32_t acc, T* out, int64_t stride, int rows, bool live, const float2* xs,
                                           float w, Release release) {
  // all of the accumulator, whatever `rows`: no branch parts the registers' lives
  if constexpr (sizeof(T) == 2) {
    uint32_t held[8][16];
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      float v[32];
      tmem_ld32(acc + b * 32, v);
      if constexpr (I8) scale_block(v, xs + b * 32, w);
      pack_cols<T>(v, held[b]);
    }
    release();
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      store_packed(out, stride, held[b], rows - b * 32, live);
      out += 32 * stride;
    }
  } else {
    float held[8 - kAtOnce32][32];
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      if (b < kAtOnce32) {
        float v[32];
        tmem_ld32(acc + b * 32, v);
        if constexpr (I8) scale_block(v, xs + b * 32, w);
        store_cols(out, stride, v, rows - b * 32, live, false);
        out += 32 * stride;
      } else {
        tmem_ld32(acc + b * 32, held[b - kAtOnce32]);
        if constexpr (I8) scale_block(held[b - kAtOnce32], xs + b * 32, w);
      }
    }
    release();
#pragma unroll
    for (int b = kAtOnce32; b < 8; ++b) {
      store_cols(out, stride, held[b - kAtOnce32], rows - b * 32, live, false);
      out += 32 * stride;
    }
  }
}

__device__ __forceinline__ void store_16(void* out, int dtype, int64_t at, int64_t stride, const float (&v)[32], int n,
                                         bool live, bool pairs) {
  if (dtype == ES_BF16)
    store_cols(static_cast<__nv_bfloat16*>(out) + at, stride, v, n, live, pairs);
  else
    store_cols(static_cast<__half*>(out) + at, stride, v, n, live, pairs);
}

// Activation, product and (for a training step) fp32 slopes of 32 columns, stored.
__device__ __forceinline__ void gated_block(const TcArgs& p, float (&g)[32], const float (&u)[32], int64_t row, int n,
                                            int64_t ch, bool live) {
  float s[32];
  if (p.activation == ES_ACT_GELU) {
    // rolled, through local memory: 32 times erfc's code keeps the compiler from holding
    // the other activations' values in registers (8192 x 4096 x 8192 bf16 1032 us, with silu
    // 852; 69 rows of 60 experts of 2048 x 1408 153 and 123)
    float a[32], d[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) a[i] = g[i];
#pragma unroll 1
    for (int i = 0; i < 32; ++i) activate<ES_ACT_GELU, false>(a[i], a[i], d[i]);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      g[i] = a[i];
      s[i] = d[i];
    }
  } else {
    ES_BY_ACT(p.activation, {
      if constexpr (ACT != ES_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < 32; ++i) activate<ACT, false>(g[i], g[i], s[i]);
      }
    });
  }
  const bool pairs = p.pairs != 0;
  if (p.slopes) {
#pragma unroll
    for (int i = 0; i < 32; ++i) s[i] *= u[i];
    store_cols(p.slopes + row * 2 * p.out_col + ch, 2 * p.out_col, s, n, live, false);
    store_cols(p.slopes + (row * 2 + 1) * p.out_col + ch, 2 * p.out_col, g, n, live, false);
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) g[i] *= u[i];
  store_16(p.out, p.out_dtype, row * p.out_col + ch, p.out_col, g, n, live, pairs);
}

// The epilogue of a gated tile. A warp has every other block of 32 columns of both
// accumulators; where TMEM holds a single tile the last of them is taken into registers
// as it is, so that TMEM is handed back before the last two are worked on. False: given up.
template <typename S>
__device__ __forceinline__ bool gated_tile(const TcArgs& p, TcCtl& ctl, const TileAt& at, uint32_t tmem, int64_t ch,
                                           uint32_t rank, int set, int quad, int& buf, uint32_t& acc_phase) {
  constexpr int PER = S::NT / 64, TAKEN = S::kHeld ? 1 : 0;
  const int lane = threadIdx.x & 31;
  int go = 0;
  if (lane == 0) go = tc_wait(&ctl.acc_full[buf], acc_phase, &ctl, p.status, true) ? 1 : 0;
  if (!__shfl_sync(0xffffffffu, go, 0)) return false;
  tc_fence_after();
  const uint32_t acc = tmem + buf * S::kAccs * S::NT + (static_cast<uint32_t>(quad * 32) << 16) + set * 32;
  float g[32], u[32], last_g[32], last_u[32];
#pragma unroll 1
  for (int i = 0; i < PER; ++i) {
    if (i < PER - TAKEN) {
      tmem_ld32(acc + i * 64, g);
      tmem_ld32(acc + S::NT + i * 64, u);
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        g[j] = last_g[j];
        u[j] = last_u[j];
      }
    }
    if (i == PER - 1 - TAKEN) {
      if constexpr (TAKEN) {
        tmem_ld32(acc + (PER - 1) * 64, last_g);
        tmem_ld32(acc + S::NT + (PER - 1) * 64, last_u);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_done_at(at_rank(smem_u32(&ctl.acc_empty[buf]), S::CG == 2 ? 0 : rank));
    }
    const int c0 = set * 32 + i * 64;
    if (c0 < at.rows) gated_block(p, g, u, at.row0 + c0, at.rows - c0, ch, ch < p.lanes);
  }
  if (++buf == S::kBufs) {
    buf = 0;
    acc_phase ^= 1;
  }
  return true;
}

// The epilogue of a tile whose depth the cluster's CTAs share: each CTA puts
// its part of the sum into shared memory, [column][lane], and every CTA adds
// up every csize-th column, the parts in the CTAs' order. 8-bit products stay
// integers until then (their bits travel as floats). Few columns: the code is
// short and rolled, since a decode step meets it cold. False: given up.
template <typename S>
__device__ __forceinline__ bool split_tile(const TcArgs& p, TcCtl& ctl, const TileAt& at, float* part, uint32_t tmem,
                                           int64_t ch, uint32_t rank, uint32_t csize, int set, int quad, int& buf,
                                           uint32_t& acc_phase, uint32_t& red_phase) {
  constexpr bool I8 = S::KIND == kKindI8;
  const int lane = threadIdx.x & 31;
  const bool live = ch < p.lanes;
  // lane i: the scale of the i-th column that this warp will add up
  float xs = 0.0f, ws = 1.0f;
  const int c_first = rank * 2 + set, c_step = 2 * csize;
  if constexpr (I8) {
    const int c = c_first + lane * c_step;
    const int64_t tok = c < at.rows ? p.g.source(at.row0 + c) : -1;
    if (tok >= 0) xs = p.g.x_scale[tok];
    ws = live ? p.g.w_scale[at.expert * p.lanes + ch] : 0.0f;
  }
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    int go = 1;
    if (lane == 0) go = tc_wait(bar, parity, &ctl, p.status, true) ? 1 : 0;
    return __shfl_sync(0xffffffffu, go, 0) != 0;
  };
  // the last tile's parts have been read by the whole cluster
  if (!wait(&ctl.red_empty, red_phase ^ 1)) return false;
  float* mine = part + quad * 32 + lane;
  for (int s0 = at.kb0; s0 < at.kb1; s0 += min(S::kChain, at.kb1 - s0)) {
    if (!wait(&ctl.acc_full[buf], acc_phase)) return false;
    tc_fence_after();
    const uint32_t acc = tmem + buf * S::kAccs * S::NT + (static_cast<uint32_t>(quad * 32) << 16);
#pragma unroll 1
    for (int c0 = set * 8; c0 < at.rows; c0 += 16) {
      float v[8];
      tmem_ld8(acc + c0, v);
      if constexpr (S::PLANES > 1) {
        float u[8];
        tmem_ld8(acc + S::NT + c0, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = plane_sum(v[i], u[i]) + (s0 > at.kb0 ? mine[(c0 + i) * 128] : 0.0f);
      }
      if constexpr (S::GATED) {
        float u[8];
        tmem_ld8(acc + S::NT + c0, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) mine[(S::NT + c0 + i) * 128] = u[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) mine[(c0 + i) * 128] = v[i];  // columns past the tile's are not read
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) arrive_at(at_rank(smem_u32(&ctl.acc_empty[buf]), rank));
    if (++buf == S::kBufs) {
      buf = 0;
      acc_phase ^= 1;
    }
  }
  __syncwarp();
  if (lane < static_cast<int>(csize)) arrive_at(at_rank(smem_u32(&ctl.red_full), lane));
  if (!wait(&ctl.red_full, red_phase)) return false;
#pragma unroll 1
  for (int c = c_first, i = 0; c < at.rows; c += c_step, ++i) {
    const uint32_t from = smem_u32(mine + c * 128);
    float f[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) f[r] = r < static_cast<int>(csize) ? load_at(at_rank(from, r)) : 0.0f;
    float v = 0.0f;
    if constexpr (I8) {
      int sum = 0;
#pragma unroll
      for (int r = 0; r < 8; ++r) sum += __float_as_int(f[r]);
      const float2 x = scale_parts(__shfl_sync(0xffffffffu, xs, i));
      v = scaled(sum, x.x, ws, x.y);
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r) v += f[r];
    }
    if constexpr (S::GATED) {
      float u = 0.0f, a = 0.0f, s = 0.0f;
      const uint32_t up = smem_u32(mine + (S::NT + c) * 128);
#pragma unroll
      for (int r = 0; r < 8; ++r) u += r < static_cast<int>(csize) ? load_at(at_rank(up, r)) : 0.0f;
      ES_BY_ACT(p.activation, (activate<ACT, false>(v, a, s)));
      if (live && p.slopes) {
        p.slopes[(at.row0 + c) * 2 * p.out_col + ch] = s * u;
        p.slopes[((at.row0 + c) * 2 + 1) * p.out_col + ch] = a;
      }
      v = a * u;
    }
    if (live) store_one(p.out, p.out_dtype, (at.row0 + c) * p.out_col + ch, v);
  }
  __syncwarp();
  if (lane < static_cast<int>(csize)) arrive_at(at_rank(smem_u32(&ctl.red_empty), lane));
  red_phase ^= 1;
  return true;
}

// Registers: the epilogue's two warpgroups take over what the first does not
// need. 128 * kRoleRegs + 256 * kEpiRegs = 384 * kLaunchRegs, which the launch
// has (checked there: a split of more would wait for ever).
constexpr int kRoleRegs = 72, kEpiRegs = 216, kLaunchRegs = 168;
static_assert(128 * kRoleRegs + 256 * kEpiRegs == kTcThreads * kLaunchRegs, "register split");

template <typename S>
__global__ void __launch_bounds__(kTcThreads, 1)
    grouped_tc_kernel(const __grid_constant__ TcArgs p, const __grid_constant__ TcMaps m) {
  constexpr int CG = S::CG, MT = S::MT, NT = S::NT, BK = S::BK, STAGES = S::kStages, PLANES = S::PLANES;
  extern __shared__ uint8_t smem_raw[];
  __shared__ TcCtl ctl;
  __shared__ alignas(16) float2 x_scales[S::KIND == kKindI8 ? 2 : 1][S::KIND == kKindI8 ? NT : 4];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float* part = reinterpret_cast<float*>(smem_raw + (base - smem_u32(smem_raw)) + STAGES * S::kStageBytes);
  int* pre = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(part) + S::kPartBytes);
  const int groups = p.g.groups();
  int* lo = pre + groups + 1;
  int* cnt = lo + groups;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank(), csize = cluster_size();
  const uint32_t pair_rank = CG == 2 ? rank : 0;
  const bool leader = pair_rank == 0;

  if (threadIdx.x == 0) {
    prefetch_map(&m.a);
    prefetch_map(&m.b);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&ctl.full[s], 1);
      mbar_init(&ctl.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&ctl.acc_full[b], 1);
      mbar_init(&ctl.acc_empty[b], CG * kEpiWarps);
    }
    mbar_init(&ctl.scales, kEpiWarps);
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
      const int tiles = S::WGRAD ? 0 : (n + NT - 1) / NT * p.lane_tiles;
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
  const Tiles<S> tiles{p, pre, lo, cnt, S::WGRAD ? groups * p.lane_tiles * p.col_tiles : pre[groups]};
  const int step = static_cast<int>(gridDim.x / csize), t0 = static_cast<int>(blockIdx.x / csize);

  if (warp < 4) {
    if constexpr (S::kHeld) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRoleRegs));
    if (warp == 0) {
      // ------------------------------------------------------------ TMA loads
      int stage = 0, used = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = t0; t < tiles.total && ok; t += step) {
        const TileAt at = tiles.at(t, rank, csize);
        if (S::skips(at.depth, p.most)) continue;
        const int width = (at.rows + 16 * CG - 1) / (16 * CG) * (16 * CG);
        const int half = width / CG;  // columns of this CTA's part of B
        const int lane0 = static_cast<int>(at.lane0) + static_cast<int>(pair_rank) * 128;
        const int col0 = at.row0 + static_cast<int>(pair_rank) * half;
        for (int kb = at.kb0; kb < at.kb1; ++kb) {
          uint32_t bytes;
          int valid = BK;  // weights' gradient: rows of the block
          const int boxes = (half + 63) / 64;
          if constexpr (S::WGRAD) {
            valid = min(at.depth - kb * BK, BK);
            bytes = (2 * MT + boxes) * ((valid + 15) & ~15) * 128u;
          } else {
            bytes = MT * kABytes + (half + kBoxRows - 1) / kBoxRows * (kBoxRows * 128u);
          }
          for (int plane = 0; plane < PLANES; ++plane) {
            int go = 0;
            if (lane == 0) {
              go = tc_wait(&ctl.empty[stage], phase ^ 1, &ctl, p.status) ? 1 : 0;
              if (go && leader) mbar_arrive_expect_tx(&ctl.full[stage], CG * bytes);
              if (go) *reinterpret_cast<volatile uint32_t*>(&ctl.progress) = ++used;
            }
            go = __shfl_sync(0xffffffffu, go, 0);
            if (!go) {
              ok = false;
              break;
            }
            const uint32_t sa = base + stage * S::kStageBytes, sb = sa + MT * kABytes;
            const uint32_t bar = CG == 2 ? at_rank(smem_u32(&ctl.full[stage]), 0) : smem_u32(&ctl.full[stage]);
            if constexpr (S::WGRAD) {
              // operand boxes of 64 lanes (columns) by 64 rows
              const int row = at.first + kb * BK + plane * p.plane_rows;
              const int operands = 2 * MT + boxes;
              auto place = [&](int u, uint32_t& to, int& x) {
                if (u < 2 * MT) {
                  to = sa + u * 8192;
                  x = lane0 + (u >> 1) * 128 * CG + (u & 1) * 64;
                } else {
                  to = sb + (u - 2 * MT) * 8192;
                  x = col0 + (u - 2 * MT) * 64;
                }
              };
              uint32_t to;
              int x;
              if (valid == BK) {
                if (lane < operands) {
                  place(lane, to, x);
                  load_2d<CG>(to, lane < 2 * MT ? &m.a : &m.b, x, row, bar);
                }
              } else {
                // the last block: whole steps of 16 rows, then the rest by
                // gathers of four rows (which cost as much as a box each)
                const int full = valid >> 4, rest = valid & 15;
                for (int i = lane; i < operands * full; i += 32) {
                  const int u = i / full, s = i - u * full;
                  place(u, to, x);
                  load_2d<CG>(to + s * 2048, u < 2 * MT ? &m.a_steps : &m.b_steps, x, row + s * 16, bar);
                }
                for (int i = lane; i < (rest ? operands * 4 : 0); i += 32) {
                  const int u = i >> 2, q = i & 3;
                  place(u, to, x);
                  int r[4];
#pragma unroll
                  for (int j = 0; j < 4; ++j) r[j] = q * 4 + j < rest ? row + full * 16 + q * 4 + j : p.src_rows;
                  load_rows<CG>(to + full * 2048 + q * 512, u < 2 * MT ? &m.a_rows : &m.b_rows, x, r, bar);
                }
              }
            } else {
              const int z = at.expert * p.expert_step + plane * p.plane_experts;
              if constexpr (S::GATED) {
                if constexpr (S::A_MN) {
                  if (lane < 4)
                    load_3d<CG>(sa + lane * 8192, lane < 2 ? &m.a : &m.up, lane0 + (lane & 1) * 64, kb * BK, z, bar);
                } else {
                  if (lane < 2) load_3d<CG>(sa + lane * kABytes, lane ? &m.up : &m.a, kb * BK, lane0, z, bar);
                }
              } else if constexpr (S::A_MN) {
                if (lane < 2 * MT)
                  load_3d<CG>(sa + lane * 8192, &m.a, lane0 + (lane >> 1) * 128 * CG + (lane & 1) * 64, kb * BK, z,
                              bar);
              } else {
                if (lane < MT) load_3d<CG>(sa + lane * kABytes, &m.a, kb * BK, lane0 + lane * 128 * CG, z, bar);
              }
              if (lane * kBoxRows < half)
                load_2d<CG>(sb + lane * (kBoxRows * 128), &m.b, kb * BK,
                            col0 + lane * kBoxRows + plane * p.plane_rows, bar);
            }
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1;
            }
          }
          if (!ok) break;
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
      // the whole warp walks the loop and one elected lane issues: operands
      // that are alike in all lanes go to the uniform registers that the
      // instruction reads (issued by one lane's branch an MMA took 68 cycles)
      if (leader) {
        int stage = 0, buf = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int t = t0; t < tiles.total && ok; t += step) {
          const TileAt at = tiles.at(t, rank, csize);
          if (at.kb0 == at.kb1 || S::skips(at.depth, p.most)) continue;
          const int width = (at.rows + 16 * CG - 1) / (16 * CG) * (16 * CG);
          const uint32_t idesc = p.idesc | (static_cast<uint32_t>(width >> 3) << 17);
          for (int s0 = at.kb0; s0 < at.kb1 && ok; s0 += min(S::kChain, at.kb1 - s0)) {
            const int s1 = s0 + min(S::kChain, at.kb1 - s0);
            ok = tc_wait_warp(&ctl.acc_empty[buf], acc_phase ^ 1, &ctl, p.status);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem + buf * S::kAccs * NT;
            uint32_t more = 0;
            constexpr uint64_t step_a = (S::A_MN ? 2048 : 32) >> 4, step_b = (S::WGRAD ? 2048 : 32) >> 4;
            for (int kb = s0; kb < s1; ++kb) {
              int steps = 4;
              if constexpr (S::WGRAD) steps = (min(at.depth - kb * BK, BK) + 15) >> 4;
              auto product = [&](int sa, int sb, int acc, uint32_t old) {  // of the tiles in stages sa and sb
                const uint64_t da = operand(base + sa * S::kStageBytes, S::A_MN);
                const uint64_t db = operand(base + sb * S::kStageBytes + MT * kABytes, S::WGRAD);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    if (i < steps)
                      mma<CG, S::KIND>(d + (acc + m) * NT, da + m * (kABytes >> 4) + i * step_a, db + i * step_b,
                                       idesc, old | i);
              };
              auto next = [&](int s) { return s + 1 == STAGES ? 0 : s + 1; };
              ok = tc_wait_warp(&ctl.full[stage], phase, &ctl, p.status);
              if (!ok) break;
              tc_fence_after();
              product(stage, stage, 0, more);
              if constexpr (PLANES == 1) {
                commit<CG>(&ctl.empty[stage]);
              } else {
                const int s1st = next(stage), s2nd = next(s1st);
                ok = tc_wait_warp(&ctl.full[s1st], phase ^ (s1st < stage ? 1 : 0), &ctl, p.status);
                if (!ok) break;
                tc_fence_after();
                product(stage, s1st, 1, more);
                product(s1st, stage, 1, 1);
                product(s1st, s1st, 1, 1);
                commit<CG>(&ctl.empty[s1st]);
                ok = tc_wait_warp(&ctl.full[s2nd], phase ^ (s2nd < stage ? 1 : 0), &ctl, p.status);
                if (!ok) break;
                tc_fence_after();
                product(stage, s2nd, 1, 1);
                product(s2nd, stage, 1, 1);
                commit<CG>(&ctl.empty[stage]);
                commit<CG>(&ctl.empty[s2nd]);
                if (s2nd < stage) phase ^= 1;
                stage = s2nd;
              }
              more = 1;
              if (++stage == STAGES) {
                stage = 0;
                phase ^= 1;
              }
            }
            if (!ok) break;
            commit<CG>(&ctl.acc_full[buf]);
            if (++buf == S::kBufs) {
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
    } else if (warp < 4) {
      if constexpr (!S::WGRAD)  // rows of no expert
        clear_rows(p, p.g.kept(), p.g.rows, blockIdx.x * 64LL + (threadIdx.x - 64), gridDim.x * 64LL);
    }
  } else {
    if constexpr (S::kHeld) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
    // ------------------------------------------------------------- epilogue
    // two sets of four warps share the tile's 32-column blocks
    const int quad = warp & 3, set = (warp - 4) >> 2;
    int buf = 0;
    uint32_t acc_phase = 0, red_phase = 0, nth = 0;
    for (int t = t0; t < tiles.total; t += step) {
      const TileAt at = tiles.at(t, rank, csize);
      if (S::skips(at.depth, p.most)) continue;
      const int64_t ch0 = at.lane0 + pair_rank * 128 + quad * 32 + lane;
      const int blocks = (at.rows + 31) / 32;
      if constexpr (S::GATED && !S::SPLIT) {
        if (!gated_tile<S>(p, ctl, at, tmem, ch0, rank, set, quad, buf, acc_phase)) break;
        continue;
      }
      if constexpr (S::SPLIT) {
        if (!split_tile<S>(p, ctl, at, part, tmem, ch0, rank, csize, set, quad, buf, acc_phase, red_phase)) break;
        continue;
      }
      const int64_t out0 = (S::WGRAD ? at.expert * p.out_expert : 0) + at.row0 * p.out_col;
      // scales of 8-bit operands, loaded under the MMAs; two tiles' worth, so
      // that one barrier a tile is enough
      const float2* xs = x_scales[nth & 1];
      float ws[MT];
      if constexpr (S::KIND == kKindI8) {
        const int c = threadIdx.x - 128;
        if (c < NT) {
          const int64_t tok = c < at.rows ? p.g.source(at.row0 + c) : -1;
          x_scales[nth & 1][c] = scale_parts(tok >= 0 ? p.g.x_scale[tok] : 0.0f);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
          ws[m] = ch0 + m * 128 * CG < p.lanes ? p.g.w_scale[at.expert * p.lanes + ch0 + m * 128 * CG] : 0.0f;
        __syncwarp();
        int go = 1;
        if (lane == 0) {
          mbar_arrive(&ctl.scales);
          go = tc_wait(&ctl.scales, nth & 1, &ctl, p.status) ? 1 : 0;
        }
        if (!__shfl_sync(0xffffffffu, go, 0)) break;
        ++nth;
      }
      bool ok = true;
      int s0 = at.kb0;
      float total[S::kSums ? NT / 64 : 1][32];
      do {  // the chains of the sum; one pass over zeros where there is no depth
        const bool any = s0 < at.kb1, first = s0 == at.kb0;
        if (any) {
          int go = 0;
          if (lane == 0) go = tc_wait(&ctl.acc_full[buf], acc_phase, &ctl, p.status, true) ? 1 : 0;
          ok = __shfl_sync(0xffffffffu, go, 0) != 0;
          if (!ok) break;
          tc_fence_after();
        }
        const uint32_t acc = tmem + buf * S::kAccs * NT + (static_cast<uint32_t>(quad * 32) << 16);
        auto release = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_at(at_rank(smem_u32(&ctl.acc_empty[buf]), CG == 2 ? 0 : rank));
        };
        bool released = !any;
        if constexpr (S::kHeld) {
          if (any && (p.pairs || p.out_dtype == ES_F32)) {
            const int64_t ch = ch0 + set * 128 * CG;
            const uint32_t mine = acc + set * NT;
            constexpr bool I8 = S::KIND == kKindI8;
            const float w = I8 ? (set ? ws[MT - 1] : ws[0]) : 1.0f;
            if (p.out_dtype == ES_BF16)
              drain_held<__nv_bfloat16, I8>(mine, static_cast<__nv_bfloat16*>(p.out) + out0 + ch, p.out_col, at.rows,
                                            ch < p.lanes, xs, w, release);
            else if (p.out_dtype == ES_F16)
              drain_held<__half, I8>(mine, static_cast<__half*>(p.out) + out0 + ch, p.out_col, at.rows, ch < p.lanes,
                                     xs, w, release);
            else
              drain_held<float, I8>(mine, static_cast<float*>(p.out) + out0 + ch, p.out_col, at.rows, ch < p.lanes, xs,
                                    w, release);
            released = true;
          }
        }
        if constexpr (S::kSums) {  // the chains' sum stays in registers
#pragma unroll
          for (int i = 0; i < NT / 64; ++i) {
            const int c0 = (set + 2 * i) * 32;
            if (c0 < at.rows) {
              float v[32], u[32];
              tmem_ld32(acc + c0, v);
              tmem_ld32(acc + NT + c0, u);
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const float s = plane_sum(v[j], u[j]);
                total[i][j] = first ? s : total[i][j] + s;
              }
            }
          }
          release();
          released = true;
          if (s0 + S::kChain >= at.kb1) {
#pragma unroll
            for (int i = 0; i < NT / 64; ++i) {
              const int c0 = (set + 2 * i) * 32;
              if (c0 < at.rows)
                store_cols(static_cast<float*>(p.out) + out0 + c0 * p.out_col + ch0, p.out_col, total[i], at.rows - c0,
                           ch0 < p.lanes, false);
            }
          }
        }
        for (int b = set; !S::kSums && b < MT * blocks && (!released || !any); b += 2) {
          const int m = b / blocks, c0 = (b - m * blocks) * 32, n = at.rows - c0;
          const int64_t ch = ch0 + m * 128 * CG;
          const bool live = ch < p.lanes;
          float v[32];
          if (any) {
            tmem_ld32(acc + m * NT + c0, v);
            if constexpr (PLANES > 1) {
              float u[32];
              tmem_ld32(acc + NT + c0, u);
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = plane_sum(v[i], u[i]);
            }
            if constexpr (S::DEEP) {  // each warp has its own part of the total
              const uint32_t total = acc + (S::kBufs - buf) * S::kAccs * NT + c0;
              if (!first) {
                float u[32];
                tmem_ld32(total, u);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] += u[i];
              }
              if (s0 + S::kChain < at.kb1) {
                tmem_st32(total, v);
                continue;
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.0f;
          }
          if constexpr (S::KIND == kKindI8) scale_block(v, xs + c0, m ? ws[MT - 1] : ws[0]);
          const int64_t at0 = out0 + c0 * p.out_col + ch;
          if constexpr (PLANES > 1) {
            float* o = static_cast<float*>(p.out) + at0;
            if (!first && live) {
              int64_t stride = p.out_col;
              keep_here(stride);
              const float* q = o;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                if (i < n) v[i] += *q;
                q += stride;
              }
            }
            store_cols(o, p.out_col, v, n, live, false);
          } else {
            store_typed(p.out, p.out_dtype, at0, p.out_col, v, n, live, p.pairs != 0);
          }
        }
        if (!released) release();
        if (any) {
          if (++buf == S::kBufs) {
            buf = 0;
            acc_phase ^= 1;
          }
          s0 += min(S::kChain, at.kb1 - s0);
        }
      } while (s0 < at.kb1);
      if (!ok) break;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (csize > 1) cluster_sync();
  tc_fence_after();
  if (warp == 1) tc_dealloc<CG>(tmem, S::kColumns);
}

// --------------------------------------------------------------------- host

template <typename S>
int launch(const TcArgs& p, const TcMaps& m, int64_t max_tiles, int csize, cudaStream_t stream) {
  const size_t smem = 1024 + static_cast<size_t>(S::kStages) * S::kStageBytes + S::kPartBytes +
                      (3 * p.g.groups() + 1) * sizeof(int);
  static std::atomic<bool> raised[kMaxAttrDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return ES_ERR_CUDA;
  const bool tracked = dev >= 0 && dev < kMaxAttrDevices;
  if (!tracked || !raised[dev].load(std::memory_order_relaxed)) {
    cudaFuncAttributes attrs;
    if (cudaFuncGetAttributes(&attrs, grouped_tc_kernel<S>) != cudaSuccess) return ES_ERR_CUDA;
    if (S::kHeld && attrs.numRegs < kLaunchRegs) return ES_ERR_UNSUPPORTED;
    const size_t most = 1024 + static_cast<size_t>(S::kStages) * S::kStageBytes + S::kPartBytes +
                        (3 * kMaxExperts + 1) * sizeof(int);
    if (cudaFuncSetAttribute(grouped_tc_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(most)) != cudaSuccess)
      return ES_ERR_CUDA;
    if (tracked) raised[dev].store(true, std::memory_order_relaxed);
  }
  int64_t clusters = kSMs / csize;
  if (clusters > max_tiles) clusters = max_tiles;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * csize));
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = csize;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  // the kernel sets up its barriers and TMEM while the one before it (the rows'
  // copy, their rounding) still runs, and waits for it before its first read
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, grouped_tc_kernel<S>, p, m) != cudaSuccess) {
    cudaGetLastError();
    return ES_ERR_CUDA;
  }
  count_launch();
  return ES_OK;
}

constexpr int64_t kMaxTiles = 0x7fffffffLL;

// The depth up to which a sum with a 16-bit result is one chain: its truncation (1.2e-4 at
// 16384 in f16, 7e-4 at 65536 in bf16, relative, of sums of one sign) is then a quarter of
// half a unit in the result's last place (4.9e-4, 3.9e-3). Longer ones take a half to two
// thirds longer: f16, 4096 rows x 20480 x 4096 780 us (one chain 500), the weights' gradient
// of 4 groups of 65536 rows, 2048 x 2048, 2300 (1570).
int64_t one_chain(int dtype) { return dtype == ES_F16 ? 16384 : 65536; }

// The kernel shape of a rows' product, and its tiles of lanes x cols.
struct RowsForm {
  int path;
  int lanes, cols;
  int split;  // CTAs that share a tile's depth
  int64_t tiles;
};

RowsForm rows_form(const GroupedArgs& g, int dtype) {
  const int64_t R = g.rows, groups = g.groups();
  const int64_t live = groups < R ? groups : R;  // groups that can have rows
  const int64_t mean = R / live;
  auto form = [&](int path, int lanes, int cols) {
    return RowsForm{path, lanes, cols, 1, (R / cols + live) * ((g.N + lanes - 1) / lanes)};
  };
  // By the rows of a group, where the tiles then fill the SMs. 60 experts,
  // 2048 x 2816, bf16, us for Narrow, Middle, Wide: 8 rows 104, 107, 118; 24
  // rows 118, 111, 119; 144 rows 339, 144, 154; 176 rows 397, 173, 160. In 8
  // bits Wide gains from 300 rows (224: 105 and 111, 300: 142 and 126).
  const bool f32 = dtype == ES_F32, i8 = dtype == kInt8;
  const RowsForm wide = form(ES_GROUPED_WIDE, f32 ? 256 : 512, f32 ? 128 : 256);
  const int64_t least = f32 ? 8 : i8 ? 240 : 160;
  const bool one = f32 || i8 || g.K <= one_chain(dtype);
  if (mean > least && wide.tiles >= kSMs / 2) return one ? wide : form(ES_GROUPED_DEEP_WIDE, 256, 256);
  const RowsForm middle = form(ES_GROUPED_MIDDLE, 256, 128);
  if (!f32 && one && mean > 8 && middle.tiles >= kSMs) return middle;
  // few rows, or few tiles: a tile's depth is shared by a cluster while the
  // tiles alone do not fill the SMs
  RowsForm narrow = form(ES_GROUPED_NARROW, 128, 64);
  const int64_t bk = i8 ? 128 : 64, nkb = (g.K + bk - 1) / bk;
  int split = 1;
  while (split < 8 && narrow.tiles * split * 2 <= kSMs && nkb >= split * 4) split *= 2;
  if (split > 1 && (one || g.K <= split * one_chain(dtype))) {
    narrow.path = ES_GROUPED_SPLIT;
    narrow.split = split;
  } else if (!one) {
    narrow.path = ES_GROUPED_DEEP_NARROW;
  }
  return narrow;
}

// The same for a gated product, whose lanes are gate's and up's of one output channel.
RowsForm gated_form(const GroupedArgs& g) {
  const int64_t R = g.rows, groups = g.groups();
  const int64_t live = groups < R ? groups : R;
  const int64_t mean = R / live;
  auto form = [&](int path, int lanes, int cols) {
    return RowsForm{path, lanes, cols, 1, (R / cols + live) * ((g.N + lanes - 1) / lanes)};
  };
  // 60 experts, 2048 x 1408, bf16, us for Narrow, Middle, Wide: 4 rows a group 108, 104, 106;
  // 48 rows 115, 112, 115; 96 rows 155, 121, 127; 144 rows 220, 185, 142; 300 rows 381, 294, 309
  const RowsForm wide = form(ES_GROUPED_WIDE, 256, 256);
  if (mean > 112 && wide.tiles >= kSMs / 2) return wide;
  const RowsForm middle = form(ES_GROUPED_MIDDLE, 128, 128);
  if (middle.tiles >= kSMs) return middle;
  RowsForm narrow = form(ES_GROUPED_NARROW, 128, 64);
  const int64_t nkb = (g.K + 63) / 64;
  while (narrow.split < 8 && narrow.tiles * narrow.split * 2 <= kSMs && nkb >= narrow.split * 4) narrow.split *= 2;
  if (narrow.split > 1) narrow.path = ES_GROUPED_SPLIT;
  return narrow;
}

template <bool A_MN>
int gated_launch(TcArgs& p, const TcMaps& m, cudaStream_t stream) {
  using Wide = TcShape<2, 2, 256, kKindF16, A_MN, false, false, 1, false, true>;
  using Middle = TcShape<1, 2, 128, kKindF16, A_MN, false, false, 1, false, true>;
  using Narrow = TcShape<1, 2, 64, kKindF16, A_MN, false, false, 1, false, true>;
  using Split = TcShape<1, 2, 64, kKindF16, A_MN, false, true, 1, false, true>;
  const RowsForm f = gated_form(p.g);
  p.lane_tiles = static_cast<int>((p.lanes + f.lanes - 1) / f.lanes);
  auto go = [&](auto shape, int csize) {
    using S = decltype(shape);
    if (f.lanes != S::kLanes || f.cols != S::NT) return static_cast<int>(ES_ERR_INVALID);
    p.idesc |= S::CG == 2 ? 16u << 24 : 8u << 24;
    return launch<S>(p, m, f.tiles, csize, stream);
  };
  if (f.path == ES_GROUPED_WIDE) return go(Wide{}, 2);
  if (f.path == ES_GROUPED_MIDDLE) return go(Middle{}, 1);
  if (f.path == ES_GROUPED_NARROW) return go(Narrow{}, 1);
  return go(Split{}, f.split);
}

template <int KIND, bool A_MN, int PLANES>
int rows_launch(TcArgs& p, const TcMaps& m, int dtype, cudaStream_t stream) {
  using Wide = std::conditional_t<PLANES == 1, TcShape<2, 2, 256, KIND, A_MN, false, false, PLANES>,
                                  TcShape<2, 1, 128, KIND, A_MN, false, false, PLANES>>;
  using Middle = TcShape<1, 2, 128, KIND, A_MN, false, false, 1>;
  using Narrow = TcShape<1, 1, 64, KIND, A_MN, false, false, PLANES>;
  using Split = TcShape<1, 1, 64, KIND, A_MN, false, true, PLANES>;
  using DeepWide = TcShape<2, 1, 256, kKindF16, A_MN, false, false, 1, true>;
  using DeepNarrow = TcShape<1, 1, 64, kKindF16, A_MN, false, false, 1, true>;
  const RowsForm f = rows_form(p.g, dtype);
  p.lane_tiles = static_cast<int>((p.lanes + f.lanes - 1) / f.lanes);
  auto go = [&](auto shape, int csize) {
    using S = decltype(shape);
    if (f.lanes != S::kLanes || f.cols != S::NT) return static_cast<int>(ES_ERR_INVALID);
    p.idesc |= S::CG == 2 ? 16u << 24 : 8u << 24;
    return launch<S>(p, m, f.tiles, csize, stream);
  };
  if (f.path == ES_GROUPED_WIDE) return go(Wide{}, 2);
  if (f.path == ES_GROUPED_SPLIT) return go(Split{}, f.split);
  if (f.path == ES_GROUPED_NARROW) return go(Narrow{}, 1);
  if constexpr (PLANES == 1)
    if (f.path == ES_GROUPED_MIDDLE) return go(Middle{}, 1);
  if constexpr (PLANES == 1 && KIND == kKindF16) {
    if (f.path == ES_GROUPED_DEEP_WIDE) return go(DeepWide{}, 2);
    if (f.path == ES_GROUPED_DEEP_NARROW) return go(DeepNarrow{}, 1);
  }
  return ES_ERR_INVALID;
}

uint32_t idesc_of(int dtype, bool a_mn, bool b_mn) {
  // D format (f32 1, s32 2), A and B formats (f16 0, bf16 1, s8 1), majors
  const uint32_t d = dtype == kInt8 ? 2u : 1u;
  const uint32_t ab = dtype == ES_F16 ? 0u : 1u;
  return (d << 4) | (ab << 7) | (ab << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16);
}

// The operands of the rows' product: X (rows, K) and the matrices, lanes
// contiguous (MN-major: K rows of N) or depth contiguous (N rows of K).
struct RowsOperands {
  bool mn;
  Operand x, w;
};

RowsOperands rows_operands(const GroupedArgs& g, int dtype, const void* x, const void* w) {
  RowsOperands o;
  o.mn = dtype != kInt8 && (g.w_n == 1 || g.w_k != 1) && g.N > 1;
  const int64_t depth = g.groups() == 1 || g.w_e == 0 ? 1 : g.num_experts;
  o.x = operand_of(x, dtype, 1, g.order ? g.rows : g.x_rows, g.K, 0, g.x_stride, 1, g.order != nullptr);
  o.w = o.mn ? operand_of(w, dtype, depth, g.K, g.N, g.w_e, g.w_k, g.w_n, false)
             : operand_of(w, dtype, depth, g.N, g.K, g.w_e, g.w_n, g.w_k, false);
  return o;
}

// The operands of the weights' gradient, (rows, K) and (rows, N).
struct WgradOperands {
  Operand x, dy;
};

WgradOperands wgrad_operands(const GroupedArgs& g, int dtype, const void* x, const void* dy, int64_t dy_stride) {
  WgradOperands o;
  o.x = operand_of(x, dtype, 1, g.order ? g.rows : g.x_rows, g.K, 0, g.x_stride, 1, g.order != nullptr);
  o.dy = operand_of(dy, dtype, 1, g.rows, g.N, 0, dy_stride, 1, false);
  return o;
}

bool sizes_ok(const GroupedArgs& g, int dtype) {
  return (dtype == ES_F32 || dtype == ES_BF16 || dtype == ES_F16 || dtype == kInt8) && g.K > 0 && g.N > 0 &&
         g.rows > 0 && g.x_rows > 0 && g.rows * planes_of(dtype) < kMaxTiles;
}

}  // namespace

bool grouped_rows_tc_ok(const GroupedArgs& g, int dtype) {
  return sizes_ok(g, dtype) && (g.rows / 64 + g.groups()) * ((g.N + 127) / 128) < kMaxTiles;
}

int grouped_rows_tc_path(const GroupedArgs& g, int dtype) { return rows_form(g, dtype).path; }

size_t grouped_rows_tc_workspace(const GroupedArgs& g, int dtype, const void* x, const void* w) {
  const RowsOperands o = rows_operands(g, dtype, x, w);
  return o.x.bytes + o.w.bytes;
}

int grouped_rows_tc(const GroupedArgs& g, int dtype, const void* x, const void* w, void* y, int out_dtype,
                    void* workspace, int32_t* status, cudaStream_t stream) {
  RowsOperands o = rows_operands(g, dtype, x, w);
  ES_TRY(lay_out(g, o.x, dtype, true, false, workspace, stream));
  ES_TRY(lay_out(g, o.w, dtype, false, o.w.depth > 1, static_cast<char*>(workspace) + o.x.bytes, stream));
  TcArgs p{};
  p.g = g;
  p.out = y;
  p.out_dtype = out_dtype;
  p.lanes = g.N;
  p.out_col = g.N;
  p.expert_step = o.w.depth > 1 ? 1 : 0;
  p.plane_experts = static_cast<int>(o.w.depth);
  p.plane_rows = static_cast<int>(o.x.rows);
  p.idesc = idesc_of(dtype, o.mn, false);
  p.pairs = g.N % 2 == 0 && (reinterpret_cast<uintptr_t>(y) & 3) == 0;
  p.status = status;
  TcMaps m{};
  const int bk = static_cast<int>(128 / tc_size(dtype));
  if (!bind_context() || !encode_operand(o.w, dtype, o.mn ? 64 : bk, o.mn ? 64 : 128, 3, &m.a) ||
      !encode_operand(o.x, dtype, bk, kBoxRows, 2, &m.b))
    return ES_ERR_CUDA;
  if (dtype == kInt8) return rows_launch<kKindI8, false, 1>(p, m, dtype, stream);
  if (dtype == ES_F32)
    return o.mn ? rows_launch<kKindF16, true, 3>(p, m, dtype, stream)
                : rows_launch<kKindF16, false, 3>(p, m, dtype, stream);
  return o.mn ? rows_launch<kKindF16, true, 1>(p, m, dtype, stream)
              : rows_launch<kKindF16, false, 1>(p, m, dtype, stream);
}

namespace {

// Operands of a gated product: those of the rows' product with the gate, and up. Where F is
// no multiple of 8, up starts at an address that TMA does not take and is copied in every
// call, and the gate too where the rows are not: 69 rows of 60 experts, K 2048, F 1408, 1404,
// 1401: 123, 335, 524 us.
struct GatedOperands {
  RowsOperands gate;
  Operand up;
};

GatedOperands gated_operands(const GroupedArgs& g, int dtype, const void* x, const void* w) {
  const void* up = static_cast<const char*>(w) + g.N * g.w_n * tc_size(dtype);
  return GatedOperands{rows_operands(g, dtype, x, w), rows_operands(g, dtype, x, up).w};
}

}  // namespace

bool grouped_gated_tc_ok(const GroupedArgs& g, int dtype) {
  return (dtype == ES_BF16 || dtype == ES_F16) && grouped_rows_tc_ok(g, dtype) && g.K <= one_chain(dtype);
}

int grouped_gated_tc_path(const GroupedArgs& g) { return gated_form(g).path; }

size_t grouped_gated_tc_workspace(const GroupedArgs& g, int dtype, const void* x, const void* w) {
  const GatedOperands o = gated_operands(g, dtype, x, w);
  return o.gate.x.bytes + o.gate.w.bytes + o.up.bytes;
}

int grouped_gated_tc(const GroupedArgs& g, int dtype, const void* x, const void* w, int activation, void* h,
                     float* slopes, void* workspace, int32_t* status, cudaStream_t stream) {
  GatedOperands o = gated_operands(g, dtype, x, w);
  char* ws = static_cast<char*>(workspace);
  ES_TRY(lay_out(g, o.gate.x, dtype, true, false, ws, stream));
  ws += o.gate.x.bytes;
  ES_TRY(lay_out(g, o.gate.w, dtype, false, o.gate.w.depth > 1, ws, stream));
  ES_TRY(lay_out(g, o.up, dtype, false, o.up.depth > 1, ws + o.gate.w.bytes, stream));
  TcArgs p{};
  p.g = g;
  p.out = h;
  p.out_dtype = dtype;
  p.lanes = g.N;
  p.out_col = g.N;
  p.expert_step = o.up.depth > 1 ? 1 : 0;
  p.plane_experts = static_cast<int>(o.up.depth);
  p.plane_rows = static_cast<int>(o.gate.x.rows);
  p.idesc = idesc_of(dtype, o.gate.mn, false);
  p.pairs = g.N % 2 == 0 && (reinterpret_cast<uintptr_t>(h) & 3) == 0;
  p.activation = activation;
  p.slopes = slopes;
  p.status = status;
  TcMaps m{};
  const int cols = 64, rows = o.gate.mn ? 64 : 128;
  if (!bind_context() || !encode_operand(o.gate.w, dtype, cols, rows, 3, &m.a) ||
      !encode_operand(o.up, dtype, cols, rows, 3, &m.up) ||
      !encode_operand(o.gate.x, dtype, cols, kBoxRows, 2, &m.b))
    return ES_ERR_CUDA;
  return o.gate.mn ? gated_launch<true>(p, m, stream) : gated_launch<false>(p, m, stream);
}

bool grouped_wgrad_tc_ok(const GroupedArgs& g, int dtype) {
  return sizes_ok(g, dtype) && (g.w_n == 1 || g.w_k == 1) &&
         g.groups() * ((g.N + 127) / 128) * ((g.K + 127) / 128) < kMaxTiles;
}

size_t grouped_wgrad_tc_workspace(const GroupedArgs& g, int dtype, const void* x, const void* dy, int64_t dy_stride) {
  const WgradOperands o = wgrad_operands(g, dtype, x, dy, dy_stride);
  return o.x.bytes + o.dy.bytes;
}

int grouped_wgrad_tc(const GroupedArgs& g, int dtype, const void* x, const void* dy, int64_t dy_stride, void* dw,
                     void* workspace, int32_t* status, cudaStream_t stream) {
  WgradOperands o = wgrad_operands(g, dtype, x, dy, dy_stride);
  ES_TRY(lay_out(g, o.x, dtype, true, false, workspace, stream));
  GroupedArgs plain = g;
  plain.order = nullptr;
  ES_TRY(lay_out(plain, o.dy, dtype, true, false, static_cast<char*>(workspace) + o.x.bytes, stream));
  // lanes: the dimension that is contiguous in dw
  const bool n_lanes = g.w_n == 1;
  TcArgs p{};
  p.g = g;
  p.out = dw;
  p.out_dtype = dtype;
  p.lanes = n_lanes ? g.N : g.K;
  p.cols = n_lanes ? g.K : g.N;
  p.out_col = n_lanes ? g.w_k : g.w_n;
  p.out_expert = g.w_e;
  p.plane_rows = static_cast<int>(g.rows);
  p.src_rows = static_cast<int>(g.rows * planes_of(dtype));
  p.idesc = idesc_of(dtype, true, true) | (16u << 24);
  p.pairs = p.lanes % 2 == 0 && p.out_col % 2 == 0 && p.out_expert % 2 == 0 &&
            (reinterpret_cast<uintptr_t>(dw) & 3) == 0;
  p.status = status;
  using Tile = TcShape<2, 2, 256, kKindF16, true, true, false, 1>;
  using Tile32 = TcShape<2, 1, 256, kKindF16, true, true, false, 3>;
  const int lanes = dtype == ES_F32 ? Tile32::kLanes : Tile::kLanes, nt = dtype == ES_F32 ? Tile32::NT : Tile::NT;
  p.lane_tiles = static_cast<int>((p.lanes + lanes - 1) / lanes);
  p.col_tiles = static_cast<int>((p.cols + nt - 1) / nt);
  TcMaps m{};
  const Operand &a = n_lanes ? o.dy : o.x, &b = n_lanes ? o.x : o.dy;
  if (!bind_context() || !encode_operand(a, dtype, 64, 64, 2, &m.a) || !encode_operand(b, dtype, 64, 64, 2, &m.b) ||
      !encode_operand(a, dtype, 64, 16, 2, &m.a_steps) || !encode_operand(b, dtype, 64, 16, 2, &m.b_steps) ||
      !encode_operand(a, dtype, 64, 1, 2, &m.a_rows) || !encode_operand(b, dtype, 64, 1, 2, &m.b_rows))
    return ES_ERR_CUDA;
  const int64_t tiles = static_cast<int64_t>(g.groups()) * p.lane_tiles * p.col_tiles;
  p.most = static_cast<int>(kMaxTiles);
  if (dtype == ES_F32) return launch<Tile32>(p, m, tiles, 2, stream);
  if (g.rows <= one_chain(dtype)) return launch<Tile>(p, m, tiles, 2, stream);
  // groups may be longer than one chain: those have a kernel of their own
  p.most = static_cast<int>(one_chain(dtype));
  ES_TRY(launch<Tile>(p, m, tiles, 2, stream));
  using Deep = TcShape<2, 1, 256, kKindF16, true, true, false, 1, true>;
  p.lane_tiles = static_cast<int>((p.lanes + Deep::kLanes - 1) / Deep::kLanes);
  p.col_tiles = static_cast<int>((p.cols + Deep::NT - 1) / Deep::NT);
  return launch<Deep>(p, m, static_cast<int64_t>(g.groups()) * p.lane_tiles * p.col_tiles, 2, stream);
}

}  // namespace es
