// Operands of the tensor-core products as TMA reads them: where they lie, or
// copied into rows that it can read (tc_operands.cu).
#pragma once

#include <cuda.h>

#include "grouped.cuh"

namespace es {

inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// One operand: where it lies, or where it is copied to.
struct Operand {
  const void* p;
  int64_t rows, cols, depth;   // of one plane; cols contiguous
  int64_t s_z, s_row, s_col;   // in elements of the source
  bool copy;
  int64_t pitch;               // of the copy, in elements
  size_t bytes;                // of the copy

  int64_t row_bytes(int64_t esz) const {
    if (copy) return pitch * esz;
    return rows == 1 ? round_up(cols * esz, 16) : s_row * esz;
  }
  int64_t z_bytes(int64_t esz) const {
    if (copy) return rows * pitch * esz;
    return depth == 1 ? round_up(rows * row_bytes(esz), 16) : s_z * esz;
  }
};

// Element size on the tensor cores: planes of fp32 are 16-bit.
inline int64_t tc_size(int dtype) { return dtype == kInt8 ? 1 : 2; }
inline int planes_of(int dtype) { return dtype == ES_F32 ? 3 : 1; }

// The operand p (depth, rows, cols) of an es_dtype or kInt8 (any bytes) with strides in
// elements; it is copied if must_copy, or where TMA cannot read it.
Operand operand_of(const void* p, int dtype, int64_t depth, int64_t rows, int64_t cols, int64_t s_z, int64_t s_row,
                   int64_t s_col, bool must_copy);
// Copies an operand that has to be copied to `to` (Operand::bytes). by_row: its rows are the
// grouped rows of g; by_expert: a matrix an expert, those without rows left out.
int lay_out(const GroupedArgs& g, Operand& o, int dtype, bool by_row, bool by_expert, void* to, cudaStream_t stream);
// Map of contiguous rows of bytes (16-byte address and pitch) in swizzled boxes of box_bytes x box_rows.
bool encode_bytes(const void* p, int64_t row_bytes, int64_t rows, int box_bytes, int box_rows, CUtensorMap* map);
bool bind_context();
bool encode_operand(const Operand& o, int dtype, int box_cols, int box_rows, int rank, CUtensorMap* map);

}  // namespace es
