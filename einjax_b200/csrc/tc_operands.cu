// Operands of the tensor-core products as TMA reads them: tensor maps, and the
// copies of what TMA cannot read as it lies.
#include "tc_operands.cuh"

#include <cudaTypedefs.h>

#include <cstring>

namespace es {
namespace {

using Encode = PFN_cuTensorMapEncodeTiled_v12000;

Encode encoder() {
  static const Encode fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess) f = nullptr;
    return reinterpret_cast<Encode>(f);
  }();
  return fn;
}

CUtensorMapDataType map_type(int dtype) {
  return dtype == ES_BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
         : dtype == ES_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                           : CU_TENSOR_MAP_DATA_TYPE_UINT8;
}

struct MapSpec {
  const void* p;
  int dtype;  // ES_BF16, ES_F16, or anything else for bytes
  int64_t d0, d1, d2;
  int64_t s1, s2;  // strides in bytes
  int b0, b1;
};

bool encode_map(const MapSpec& m, int rank, CUtensorMap* map) {
  std::memset(map, 0, sizeof(*map));
  Encode fn = encoder();
  if (!fn) return false;
  cuuint64_t dim[3] = {static_cast<cuuint64_t>(m.d0), static_cast<cuuint64_t>(m.d1), static_cast<cuuint64_t>(m.d2)};
  cuuint64_t stride[2] = {static_cast<cuuint64_t>(m.s1), static_cast<cuuint64_t>(m.s2)};
  cuuint32_t box[3] = {static_cast<cuuint32_t>(m.b0), static_cast<cuuint32_t>(m.b1), 1};
  cuuint32_t one[3] = {1, 1, 1};
  return fn(map, map_type(m.dtype), static_cast<cuuint32_t>(rank), const_cast<void*>(m.p), dim, stride, box, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What a TMA map asks of an address and of the strides (in bytes).
bool tma_ok(const void* p, int64_t s1, int64_t s2 = 16) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s1 > 0 && s1 % 16 == 0 && s1 < (1LL << 40) && s2 > 0 &&
         s2 % 16 == 0 && s2 < (1LL << 40);
}

// ------------------------------------------------- operands laid out for TMA
//
// Copies a (depth, rows, cols) tensor of any strides into rows that TMA can
// read: 16-byte pitch, routed rows in the grouped order, fp32 cut into three
// bf16 planes. A thread writes 16 bytes of one row (of each plane). Bound by
// memory. Matrices of experts without rows are left out.
constexpr int kCopyThreads = 256;

struct LayoutArgs {
  GroupedArgs g;
  const void* src;
  int64_t s_z, s_row, s_col;  // source strides in elements
  int64_t rows, cols, pitch;  // pitch: elements of a row of the copy
  int64_t depth;              // matrices of one plane
  void* out;
  int by_row;   // rows are grouped rows: the source row is theirs, those of no expert are left out
  int by_expert;
  int wide;     // 16-byte loads
};

// Half of x in planes, b0 + b1 + b2 == x / 2 for magnitudes from 2^-109 on (below,
// the third plane ends at bf16's smallest value): each is what is left, rounded to
// 8 bits (to nearest: a rest is at most 2^-8 of its number, twice less than after
// truncation, which the products left out have in their square). Halves, since a
// rounded plane is up to 2^-8 larger than its value: no finite value has an
// infinite plane, and no product of planes overflows where the values' does not. An
// infinity or NaN is its first plane alone; a value below 2^-132 may have none.
__device__ __forceinline__ void split3(float x, uint16_t (&b)[3]) {
  const float h = 0.5f * x;
  const __nv_bfloat16 b0 = __float2bfloat16_rn(h);
  const float r1 = fabsf(h) < INFINITY ? h - __bfloat162float(b0) : 0.0f;
  const __nv_bfloat16 b1 = __float2bfloat16_rn(r1);
  b[0] = __bfloat16_as_ushort(b0);
  b[1] = __bfloat16_as_ushort(b1);
  b[2] = __bfloat16_as_ushort(__float2bfloat16_rn(r1 - __bfloat162float(b1)));
}

template <typename T>
__global__ void __launch_bounds__(kCopyThreads) layout_kernel(const __grid_constant__ LayoutArgs p) {
  let_next_grid_start();
  constexpr bool kSplit = std::is_same<T, float>::value;
  constexpr int VEC = kSplit ? 8 : 16 / sizeof(T);  // elements of a 16-byte store
  const int64_t z = blockIdx.y;
  if (p.by_expert) {
    int64_t lo, hi;
    p.g.bounds(static_cast<int>(z), lo, hi);
    if (hi <= lo) return;
  }
  const int64_t pieces = p.pitch / VEC;
  const int64_t at = blockIdx.x * static_cast<int64_t>(kCopyThreads) + threadIdx.x;
  const int64_t row = at / pieces, c0 = (at - row * pieces) * VEC;
  if (row >= p.rows) return;
  int64_t from = row;
  if (p.by_row) {
    if (row >= p.g.kept()) return;
    from = p.g.source(row);
  }
  const T* src = static_cast<const T*>(p.src) + z * p.s_z + from * p.s_row;
  alignas(16) T v[VEC];
  if (p.wide && from >= 0 && c0 + VEC <= p.cols) {
    constexpr int LOADS = VEC * sizeof(T) / 16;
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(src + c0)[i];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = from >= 0 && c0 + i < p.cols ? src[(c0 + i) * p.s_col] : T(0);
  }
  if constexpr (kSplit) {
    uint16_t b[3][VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      uint16_t s[3];
      split3(v[i], s);
#pragma unroll
      for (int k = 0; k < 3; ++k) b[k][i] = s[k];
    }
    uint16_t* out = static_cast<uint16_t*>(p.out);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      uint4 q;
      q.x = b[k][0] | b[k][1] << 16;
      q.y = b[k][2] | b[k][3] << 16;
      q.z = b[k][4] | b[k][5] << 16;
      q.w = b[k][6] | b[k][7] << 16;
      *reinterpret_cast<uint4*>(out + ((k * p.depth + z) * p.rows + row) * p.pitch + c0) = q;
    }
  } else {
    *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (z * p.rows + row) * p.pitch + c0) =
        *reinterpret_cast<const uint4*>(v);
  }
}

// The common case of routed 16-bit or 8-bit rows: whole pieces of 16 bytes, a
// warp a row, four pieces of a lane in flight (16400 rows of 2048 bytes: 11
// us, 16 with a thread a piece).
__global__ void __launch_bounds__(kCopyThreads) gather_kernel(const __grid_constant__ GroupedArgs g, const uint4* x,
                                                              int64_t stride, int pieces, uint4* out) {
  let_next_grid_start();
  const int lane = threadIdx.x & 31;
  const int64_t r = blockIdx.x * static_cast<int64_t>(kCopyThreads / 32) + (threadIdx.x >> 5);
  if (r >= g.kept()) return;
  const int64_t t = g.source(r);
  const uint4* from = x + t * stride;
  uint4* to = out + r * pieces;
  for (int i0 = lane; i0 < pieces; i0 += 128) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      v[u] = t >= 0 && i0 + u * 32 < pieces ? from[i0 + u * 32] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u * 32 < pieces) to[i0 + u * 32] = v[u];
  }
}

}  // namespace

Operand operand_of(const void* p, int dtype, int64_t depth, int64_t rows, int64_t cols, int64_t s_z, int64_t s_row,
                   int64_t s_col, bool must_copy) {
  const int64_t esz = tc_size(dtype);
  Operand o{p, rows, cols, depth, s_z, s_row, s_col, false, 0, 0};
  o.copy = must_copy || dtype == ES_F32 || (s_col != 1 && cols > 1) ||
           !tma_ok(p, o.row_bytes(esz), o.z_bytes(esz));
  if (o.copy) {
    o.pitch = round_up(cols, 16 / esz);
    o.bytes = round_up(planes_of(dtype) * depth * rows * o.pitch * esz, 256);
  }
  return o;
}

int lay_out(const GroupedArgs& g, Operand& o, int dtype, bool by_row, bool by_expert, void* to, cudaStream_t stream) {
  if (!o.copy) return ES_OK;
  LayoutArgs a{g, o.p, o.s_z, o.s_row, o.s_col, o.rows, o.cols, o.pitch, o.depth, to, by_row, by_expert, 0};
  const int64_t esz = dtype == ES_F32 ? 4 : tc_size(dtype);
  a.wide = (o.s_col == 1 || o.cols == 1) && (reinterpret_cast<uintptr_t>(o.p) & 15) == 0 &&
           (o.s_row * esz % 16 == 0 || (o.rows == 1 && !by_row)) && (o.s_z * esz % 16 == 0 || o.depth == 1);
  if (by_row && a.wide && dtype != ES_F32 && o.cols * esz % 16 == 0) {
    ES_LAUNCH(gather_kernel, static_cast<unsigned>((o.rows + kCopyThreads / 32 - 1) / (kCopyThreads / 32)),
              kCopyThreads, 0, stream, g, static_cast<const uint4*>(o.p), o.s_row * esz / 16,
              static_cast<int>(o.cols * esz / 16), static_cast<uint4*>(to));
    o.p = to;
    return ES_OK;
  }
  const int64_t vec = dtype == ES_F32 ? 8 : 16 / esz;
  const dim3 grid(static_cast<unsigned>((o.rows * (o.pitch / vec) + kCopyThreads - 1) / kCopyThreads),
                  static_cast<unsigned>(o.depth));
  if (dtype == ES_F32)
    ES_LAUNCH((layout_kernel<float>), grid, kCopyThreads, 0, stream, a);
  else if (dtype == kInt8)
    ES_LAUNCH((layout_kernel<int8_t>), grid, kCopyThreads, 0, stream, a);
  else
    ES_LAUNCH((layout_kernel<uint16_t>), grid, kCopyThreads, 0, stream, a);
  o.p = to;
  return ES_OK;
}

// The driver encodes maps for the thread's current context, which a thread has
// only after its first runtime call that needs one (autograd's threads run a
// gradient without any before it).
bool bind_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}

bool encode_bytes(const void* p, int64_t row_bytes, int64_t rows, int box_bytes, int box_rows, CUtensorMap* map) {
  return encode_map(MapSpec{p, kInt8, row_bytes, rows, 1, row_bytes, rows * row_bytes, box_bytes, box_rows}, 2, map);
}

bool encode_operand(const Operand& o, int dtype, int box_cols, int box_rows, int rank, CUtensorMap* map) {
  const int64_t esz = tc_size(dtype), planes = planes_of(dtype);
  const int64_t rows = rank == 2 ? planes * o.rows : o.rows, depth = rank == 3 ? planes * o.depth : 1;
  return encode_map(MapSpec{o.p, dtype == ES_F32 ? ES_BF16 : dtype, o.cols, rows, depth, o.row_bytes(esz),
                            o.z_bytes(esz), box_cols, box_rows},
                    rank, map);
}

}  // namespace es
