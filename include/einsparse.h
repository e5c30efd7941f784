/*
 * einsparse — C ABI of the B200 (sm_100a) sparse tensor-relational einsum path.
 *
 * Each entry point replaces one step of einjax's sparse execution path
 * (paths below are relative to the einjax project root). All pointers are
 * device pointers unless stated; all sizes are element counts; every call is
 * asynchronous on `stream` (a cudaStream_t, 0 = legacy default stream) and
 * returns an es_status. No entry point allocates memory: multi-phase steps
 * take a caller-owned workspace whose size the matching *_workspace_size
 * query reports, and data-dependent output sizes are written to a device
 * int64 that the caller reads before allocating the outputs of the *_fill
 * phase. Device-side checks (an index outside its grid) set *error_dev to a
 * non-zero es_status; the caller reads it together with the size. The
 * caller clears *error_dev (and the counts) before a call, except for
 * es_tile_coo_plan, es_tile_dense_plan, es_direct_plan and es_tile_einsum(_ev),
 * which clear their own count and status outputs first.
 *
 * Threading: calls on different streams may run concurrently as long as
 * they do not share a workspace. The library holds no global mutable state
 * apart from a launch counter (es_launch_count).
 */
#ifndef EINSPARSE_H
#define EINSPARSE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum es_status {
  ES_OK = 0,
  ES_ERR_INVALID = 1,     /* bad shape / argument; the reference raises ValueError */
  ES_ERR_INDEX = 2,       /* a coordinate outside the grid its shape defines */
  ES_ERR_WORKSPACE = 3,   /* workspace smaller than *_workspace_size reported */
  ES_ERR_CUDA = 4,        /* CUDA runtime error (launch or async) */
  ES_ERR_UNSUPPORTED = 5, /* dtype / rank / size this build does not handle */
  ES_ERR_TIMEOUT = 6      /* a bounded device-side wait ran out; outputs are invalid */
} es_status;

typedef enum es_dtype { ES_F32 = 0, ES_BF16 = 1, ES_F64 = 2, ES_I32 = 3, ES_I64 = 4, ES_F16 = 5 } es_dtype;

/* Arithmetic of the tile contraction. EXACT: fp32 FFMA (SIMT); TC: tensor
 * cores (bf16 inputs: kind::f16; fp32 inputs: 3-pass split TF32, fp32-level
 * error); AUTO: TC where a tensor-core kernel covers the shape, else EXACT. */
typedef enum es_precision { ES_PREC_AUTO = 0, ES_PREC_EXACT = 1, ES_PREC_TC = 2 } es_precision;

#define ES_MAX_DIMS 8

/* Library version and a count of kernels launched since load (or since the
 * last es_launch_count_reset). */
int es_version(void);
int64_t es_launch_count(void);
void es_launch_count_reset(void);
const char* es_status_string(int status);

/* ---------------------------------------------------------------------------
 * Tiling: element COO -> tile-COO.
 * Replaces SparseTensor.to_relation (tensor/sparse.py:160-219) together with
 * the COO extraction it consumes (tensor/sparse.py:234-270).
 * indices: int32 (nnz, ndim) row-major; values: (nnz) of values_dtype
 * (F32/F64/BF16). Entries equal to zero are dropped (sparse.py:185-187);
 * tiles come out in lexicographic coordinate order (np.unique, :204-206);
 * when a coordinate repeats, the entry that comes last in input order
 * wins (NumPy fancy assignment, :211-212). shape[d] % tile[d] != 0 gives
 * ES_ERR_INVALID (:174-179). Plan writes the tile count T to *num_tiles_dev;
 * fill writes coords int32 (T, ndim) and values (T, prod(tile)) of out_dtype.
 * Either fill output may be NULL: with values_out NULL the call writes the
 * coords (and keeps the value bounds in the workspace); with coords_out NULL
 * it writes the values from the bounds that an earlier coords call left in
 * the same workspace (so the values can be filled later, e.g. while the host
 * waits for other counts).
 * ------------------------------------------------------------------------- */
size_t es_tile_coo_workspace_size(int64_t nnz, int ndim, const int64_t* shape, const int64_t* tile);
int es_tile_coo_plan(const int32_t* indices, const void* values, int values_dtype, int64_t nnz,
                     int ndim, const int64_t* shape, const int64_t* tile,
                     void* workspace, size_t workspace_bytes,
                     int64_t* num_tiles_dev, int32_t* error_dev, void* stream);
int es_tile_coo_fill(const void* values, int values_dtype, int64_t nnz, int ndim,
                     const int64_t* shape, const int64_t* tile,
                     void* workspace, size_t workspace_bytes, int64_t num_tiles,
                     int32_t* coords_out, void* values_out, int out_dtype, void* stream);

/* ---------------------------------------------------------------------------
 * COO ingestion: coalescing repeated coordinates.
 * The reference feeds element COO to its tiling as it comes
 * (_extract_coo, tensor/sparse.py:234-270) and the last repeated coordinate
 * wins there (:211-212); scipy CSR and torch's uncoalesced sparse tensors add
 * repeated coordinates instead. es_coo_coalesce states the policy: it writes
 * one entry per distinct coordinate holding a non-zero value, in row-major
 * coordinate order -- ES_DUP_LAST: the value that comes last in input order;
 * ES_DUP_SUM: the sum of the run, accumulated in float64 in input order (what
 * scipy's sum_duplicates and numpy.add.at compute). Zero entries are dropped
 * before coalescing (tensor/sparse.py:185-187); a sum that cancels to zero is
 * written as 0 (the tiling drops it). indices_out int32 (nnz, ndim) and
 * values_out (nnz) of out_dtype (F32/F64/BF16) are caller buffers of the input
 * size; counts_dev[0] = entries written, counts_dev[1] = non-zero input
 * entries (they differ exactly when a coordinate repeats). A coordinate
 * outside `shape` sets *error_dev to ES_ERR_INDEX. This entry point has no
 * counterpart in the reference (it is the explicit form of its implicit
 * last-wins policy).
 * ------------------------------------------------------------------------- */
typedef enum es_dup_policy { ES_DUP_LAST = 0, ES_DUP_SUM = 1 } es_dup_policy;
size_t es_coo_coalesce_workspace_size(int64_t nnz, int ndim, const int64_t* shape);
int es_coo_coalesce(const int32_t* indices, const void* values, int values_dtype, int64_t nnz,
                    int ndim, const int64_t* shape, int policy,
                    void* workspace, size_t workspace_bytes,
                    int32_t* indices_out, void* values_out, int out_dtype,
                    int64_t* counts_dev, int32_t* error_dev, void* stream);

/* Dense array (row-major `shape`) -> tile-COO of the tiles holding any
 * non-zero. Same result as SparseTensor(dense).to_relation(tile)
 * (tensor/sparse.py:104-117,160-219, via np.nonzero at :260-268). Fill:
 * coords_out or values_out may be NULL (that output is not written; the
 * other one only needs the plan's workspace and the dense array). */
size_t es_tile_dense_workspace_size(int ndim, const int64_t* shape, const int64_t* tile);
int es_tile_dense_plan(const void* dense, int dtype, int ndim, const int64_t* shape,
                       const int64_t* tile, void* workspace, size_t workspace_bytes,
                       int64_t* num_tiles_dev, void* stream);
int es_tile_dense_fill(const void* dense, int dtype, int ndim, const int64_t* shape,
                       const int64_t* tile, void* workspace, size_t workspace_bytes,
                       int64_t num_tiles, int32_t* coords_out, void* values_out, int out_dtype,
                       void* stream);

/* ---------------------------------------------------------------------------
 * Coordinate join. Replaces coordinate_join (execution/sparse_dispatch.py:29-82)
 * and coordinate_join_hash (kernels/pallas_gather.py:19-76).
 * join_keys: nkeys pairs (lhs_dim, rhs_dim); key_extents[k]: the tile-grid
 * extent of key k (coordinates must lie in [0, extent), else ES_ERR_INDEX in
 * *error_dev). Pair order is the reference's: RHS tile j ascending, and for
 * each j every LHS tile with an equal key, LHS index ascending; nkeys == 0
 * gives the LHS-major cross product (:53-59). Plan writes P to *num_pairs_dev;
 * fill writes lhs_idx/rhs_idx as index_dtype (ES_I32 or ES_I64).
 * ------------------------------------------------------------------------- */
size_t es_join_workspace_size(int64_t n_lhs, int64_t n_rhs);
int es_join_plan(const int32_t* lhs_coords, int64_t n_lhs, int lhs_ndim,
                 const int32_t* rhs_coords, int64_t n_rhs, int rhs_ndim,
                 const int32_t* join_keys, int nkeys, const int64_t* key_extents,
                 void* workspace, size_t workspace_bytes,
                 int64_t* num_pairs_dev, int32_t* error_dev, void* stream);
int es_join_fill(int64_t n_lhs, int64_t n_rhs, int nkeys, void* workspace, size_t workspace_bytes,
                 int64_t num_pairs, void* lhs_idx_out, void* rhs_idx_out, int index_dtype,
                 void* stream);

/* Allocation-free coordinate join (no counterpart in the reference; an
 * addition for callers that may not allocate device memory when they join,
 * e.g. code in a host callback or an engine that reserves all memory up
 * front). Same pairs and order as es_join_plan + es_join_fill, but the sort
 * and count scratch comes from a fixed array inside the library (one per
 * GPU, kept until the process exits) instead of a workspace. At most 65536
 * tiles per side, else ES_ERR_UNSUPPORTED. The caller passes the outputs:
 * lhs_idx_out / rhs_idx_out with room for `capacity` pairs and the device
 * int64 *num_pairs_dev that receives P; if P > capacity only `capacity`
 * pairs are written and *error_dev becomes ES_ERR_WORKSPACE. Nothing is
 * allocated or synchronised. Calls whose kernels overlap on one GPU share the
 * array and race: order them on one stream. The first call on a device looks
 * up the array's address (cudaGetSymbolAddress); make it before any stream
 * capture. */
int es_join_static(const int32_t* lhs_coords, int64_t n_lhs, int lhs_ndim,
                   const int32_t* rhs_coords, int64_t n_rhs, int rhs_ndim,
                   const int32_t* join_keys, int nkeys, const int64_t* key_extents,
                   void* lhs_idx_out, void* rhs_idx_out, int index_dtype, int64_t capacity,
                   int64_t* num_pairs_dev, int32_t* error_dev, void* stream);

/* ---------------------------------------------------------------------------
 * Output-tile grouping. Replaces _compute_output_coords + the grouping half of
 * segment_sum (execution/sparse_dispatch.py:174-223, 129-171): the output
 * coordinate of each pair is gathered through agg_keys (pairs (src, dim),
 * src 0 = lhs, 1 = rhs); pairs are stably sorted by it, so inside each group
 * they keep join order (the reference sums each group in pair order,
 * :165-169). Plan writes the group count O to *num_segments_dev; fill writes
 * out_coords int32 (O, out_ndim) sorted lexicographically (:161),
 * seg_offsets int64 (O+1) and the pairs regrouped (seg_lhs_idx,
 * seg_rhs_idx int32, P each; seg_pair_idx int32 = original pair index, may
 * be NULL). lhs_idx/rhs_idx are int32. With seg_strip non-NULL, fill also
 * writes per segment the packed value of its first strip_dims output
 * coordinates (int64, non-decreasing): segments with equal values form a
 * "strip" that shares its lhs-derived coordinates, which es_tile_einsum
 * batches into one tensor-core tile.
 * ------------------------------------------------------------------------- */
size_t es_segments_workspace_size(int64_t num_pairs);
int es_segments_plan(const int32_t* lhs_coords, int lhs_ndim, const int32_t* rhs_coords, int rhs_ndim,
                     const int32_t* lhs_idx, const int32_t* rhs_idx, int64_t num_pairs,
                     const int32_t* agg_keys, int out_ndim, const int64_t* out_extents,
                     void* workspace, size_t workspace_bytes,
                     int64_t* num_segments_dev, int32_t* error_dev, void* stream);
int es_segments_fill(const int32_t* lhs_idx, const int32_t* rhs_idx, int64_t num_pairs, int out_ndim,
                     const int64_t* out_extents, void* workspace, size_t workspace_bytes,
                     int64_t num_segments, int32_t* out_coords, int64_t* seg_offsets,
                     int32_t* seg_lhs_idx, int32_t* seg_rhs_idx, int32_t* seg_pair_idx,
                     int strip_dims, int64_t* seg_strip, void* stream);

/* Per-pair output tile coordinates, int32 (P, out_ndim): the gather of
 * _compute_output_coords (execution/sparse_dispatch.py:174-223). */
int es_output_coords(const int32_t* lhs_coords, int lhs_ndim, const int32_t* rhs_coords, int rhs_ndim,
                     const int32_t* lhs_idx, const int32_t* rhs_idx, int64_t num_pairs,
                     const int32_t* agg_keys, int out_ndim, int32_t* out_coords, void* stream);

/* ---------------------------------------------------------------------------
 * Segmented tile einsum — the per-pair kernel einsum fused with the
 * segment-sum (execution/sparse_dispatch.py:85-126 + 129-171; the batched
 * tile einsum of kernels/pallas_matmul.py:33-113).
 * kernel_string: the per-tile einsum ("ij,jk->ik", "bij,bjk->bik",
 * "ijk,kl->ijl", ...; any two-operand string with an explicit "->").
 * For segment s, out[s_out] = sum over p in [seg_offsets[s], seg_offsets[s+1])
 * of einsum(lhs_values[pair_lhs[p]], rhs_values[pair_rhs[p]]), accumulated
 * in fp32, where s_out = seg_out_index ? seg_out_index[s] : s.
 * seg_offsets == NULL means every pair is its own segment (the unfused
 * per-pair kernel_einsum, output (P, *out_tile)). Output rows that no segment
 * writes are left untouched. lhs_rows / rhs_rows: tiles in each values array
 * (pair indices outside them raise ES_ERR_INDEX in *error_dev and read as
 * zero tiles). Values dtypes: F32 / BF16 / F64 inputs; F32 / BF16 outputs.
 * seg_strip (optional, from es_segments_fill): strip key per segment; the
 * tensor-core path computes up to 8 segments of one strip in one tile.
 * pair_key (optional): the contracted tile coordinate of each pair, with
 * key_extent its range. Contract: inside a segment keys increase strictly,
 * and segments of one strip (seg_strip) pair the same lhs tile with a given
 * key. When given, the tensor-core path may stack up to 128 / Mt strips
 * into one 128-row operand that shares each step's rhs tiles (fp32, Mt 16,
 * 32 or 64, Kt 32 or 64), and splits the contracted range into blocks whose
 * rhs operand fits in L2, adding the blocks' partial sums into the output
 * in block order. A broken contract sets *error_dev to ES_ERR_INVALID.
 * A contraction that is a plain tile matmul after swapping the last two tile
 * dims of an operand ("ik,jk->ij", "ij,ik->jk": the autodiff strings) also
 * takes the tensor-core path; the swapped operand is transposed into the
 * workspace first (a copy, no rounding).
 * workspace: es_tile_einsum_workspace_size bytes (0 for the SIMT path),
 * sized for the same lhs_rows, rhs_rows, num_pairs, num_segments and
 * key_extent (0 when no pair_key is passed). A device-side wait that runs
 * out sets *error_dev to ES_ERR_TIMEOUT.
 * ------------------------------------------------------------------------- */
size_t es_tile_einsum_workspace_size(const char* kernel_string,
                                     const int64_t* lhs_tile, int lhs_nd, const int64_t* rhs_tile, int rhs_nd,
                                     int lhs_dtype, int rhs_dtype, int64_t lhs_rows, int64_t rhs_rows,
                                     int64_t num_pairs, int64_t num_segments, int64_t key_extent, int precision);
int es_tile_einsum(const char* kernel_string,
                   const int64_t* lhs_tile, int lhs_nd, const int64_t* rhs_tile, int rhs_nd,
                   const void* lhs_values, int lhs_dtype, int64_t lhs_rows,
                   const void* rhs_values, int rhs_dtype, int64_t rhs_rows,
                   const int32_t* pair_lhs, const int32_t* pair_rhs, int64_t num_pairs,
                   const int64_t* seg_offsets, int64_t num_segments, const int32_t* seg_out_index,
                   const int64_t* seg_strip, const int32_t* pair_key, int64_t key_extent,
                   void* out_values, int out_dtype, int precision,
                   void* workspace, size_t workspace_bytes, int32_t* error_dev, void* stream);

/* es_tile_einsum that waits for the cudaEvent_t values_ready (NULL: no
 * wait) on `stream` right before its first launch that reads lhs_values or
 * rhs_values: the grouping of the pairs into work items and step records
 * runs first, so values written on another stream (e.g. a tiling's value
 * fill) overlap it. status_host (NULL: none): pinned host int32 that
 * receives *error_dev by an asynchronous copy behind the call's launches,
 * so a caller can check the status later without a copy of its own. */
int es_tile_einsum_ev(const char* kernel_string,
                      const int64_t* lhs_tile, int lhs_nd, const int64_t* rhs_tile, int rhs_nd,
                      const void* lhs_values, int lhs_dtype, int64_t lhs_rows,
                      const void* rhs_values, int rhs_dtype, int64_t rhs_rows,
                      const int32_t* pair_lhs, const int32_t* pair_rhs, int64_t num_pairs,
                      const int64_t* seg_offsets, int64_t num_segments, const int32_t* seg_out_index,
                      const int64_t* seg_strip, const int32_t* pair_key, int64_t key_extent,
                      void* out_values, int out_dtype, int precision,
                      void* workspace, size_t workspace_bytes, int32_t* error_dev, void* stream,
                      void* values_ready, int32_t* status_host);

/* Which path es_tile_einsum takes for these arguments: 1 tensor cores,
 * 0 SIMT, negative es_status if the call would be rejected. Host-side. */
int es_tile_einsum_path(const char* kernel_string, const int64_t* lhs_tile, int lhs_nd,
                        const int64_t* rhs_tile, int rhs_nd, int lhs_dtype, int rhs_dtype, int precision);

/* ---------------------------------------------------------------------------
 * Join + output grouping in one pass for
 *     lhs (batch..., strip..., k) x rhs (batch..., k, col...)
 *         -> out (batch..., strip..., col...)
 * with batch_ndim >= 0 leading batch dims joined pairwise (lhs dim d with rhs
 * dim d), the last lhs coordinate joined with rhs coordinate batch_ndim, and
 * output = the other lhs then the other rhs coordinates (the matmul-like
 * calls of execute_sparse: coordinate_join + _compute_output_coords +
 * segment_sum grouping, execution/sparse_dispatch.py:29-82, 174-223,
 * 129-171). No reference counterpart as one function: it replaces
 * es_join_plan/_fill + es_segments_plan/_fill for these shapes with no sort.
 * Both coordinate arrays must be in lexicographic order without repeats (a
 * relation's invariant); lhs_grid / rhs_grid are the tile-grid extents.
 * plan writes counts_dev[0] = pairs P, [1] = output tiles O, [2] = 1 when a
 * relation is not in lexicographic order (then use the general path); fill
 * writes out_coords (O, out_nd) lexicographic, seg_offsets (O+1), seg_lhs /
 * seg_rhs (P) grouped by output tile (pairs of a tile in ascending k = join
 * order), and optionally seg_strip (O) strip index and seg_key (P) the
 * contracted k. fill takes the same sizes, grids and workspace as plan (the
 * workspace carries the plan's per-(strip, column) offsets).
 * ------------------------------------------------------------------------- */
size_t es_direct_workspace_size(int64_t n_lhs, int lhs_ndim, int64_t n_rhs, int rhs_ndim, int batch_ndim,
                                const int64_t* lhs_grid, const int64_t* rhs_grid);
int es_direct_plan(const int32_t* lhs_coords, int64_t n_lhs, int lhs_ndim, const int32_t* rhs_coords,
                   int64_t n_rhs, int rhs_ndim, int batch_ndim, const int64_t* lhs_grid, const int64_t* rhs_grid,
                   void* workspace, size_t workspace_bytes, int64_t* counts_dev, int32_t* error_dev,
                   void* stream);
int es_direct_fill(const int32_t* lhs_coords, int64_t n_lhs, int lhs_ndim, int64_t n_rhs, int rhs_ndim,
                   int batch_ndim, const int64_t* lhs_grid, const int64_t* rhs_grid, void* workspace,
                   size_t workspace_bytes, int64_t num_pairs, int64_t num_segments, int32_t* out_coords,
                   int64_t* seg_offsets, int32_t* seg_lhs, int32_t* seg_rhs, int64_t* seg_strip, int32_t* seg_key,
                   void* stream);

/* Out tile shape of a kernel string (_infer_output_tile_shape,
 * execution/sparse_dispatch.py:506-545). Host-side; returns the out rank or
 * a negative es_status. */
int es_out_tile_shape(const char* kernel_string, const int64_t* lhs_tile, int lhs_nd,
                      const int64_t* rhs_tile, int rhs_nd, int64_t* out_tile);

/* ---------------------------------------------------------------------------
 * Standalone segment-sum (execution/sparse_dispatch.py:129-171): values
 * (P, tile_elems) grouped by coords (P, nd) int32 with per-dim extents.
 * Plan (es_segsum_plan) writes O; fill writes unique coords (O, nd) sorted
 * lexicographically and the per-group sums, added in row order in fp32.
 * Scatter-add by index (the `.at[idx].add` of autodiff/custom_vjp.py:272-273)
 * is the nd == 1 case with out rows chosen by the caller via es_tile_einsum's
 * seg_out_index; see es_scatter_add_rows.
 * ------------------------------------------------------------------------- */
size_t es_segsum_workspace_size(int64_t num_rows);
int es_segsum_plan(const int32_t* coords, int64_t num_rows, int nd, const int64_t* extents,
                   void* workspace, size_t workspace_bytes, int64_t* num_segments_dev,
                   int32_t* error_dev, void* stream);
int es_segsum_fill(const void* values, int values_dtype, int64_t num_rows, int64_t tile_elems, int nd,
                   const int64_t* extents, void* workspace, size_t workspace_bytes, int64_t num_segments,
                   int32_t* out_coords, void* out_values, int out_dtype, void* stream);

/* Groups of an es_segsum_plan without a reduction: unique coordinates
 * (O, nd) sorted lexicographically into out_coords (may be NULL) and, for
 * each input row r, its group index into row_group[r] (int32, may be NULL).
 * This is the grouping half of segment_sum (execution/sparse_dispatch.py:
 * 154-161: the unique output keys and which key each row belongs to); the
 * sharded path uses it to lay every rank's partial output tiles out in the
 * order of the union of all ranks' output coordinates before the
 * reduce-scatter. Same workspace as the plan, which must have run first. */
int es_segsum_groups(int64_t num_rows, int nd, const int64_t* extents, void* workspace, size_t workspace_bytes,
                     int64_t num_segments, int32_t* out_coords, int32_t* row_group, void* stream);

/* out[idx[r]] += values[r] for r in row order, rows of tile_elems
 * (autodiff/custom_vjp.py:272-273). out must be F32. Deterministic: rows
 * are grouped by a stable sort, each group is summed in row order, then
 * added once. */
size_t es_scatter_add_workspace_size(int64_t num_rows);
int es_scatter_add_rows(const void* values, int values_dtype, const int32_t* idx, int64_t num_rows,
                        int64_t tile_elems, int64_t num_out_rows, void* workspace,
                        size_t workspace_bytes, float* out, int32_t* error_dev, void* stream);

/* ---------------------------------------------------------------------------
 * Sparsity statistics per tiling scheme, the contraction planner's input
 * (tensor/stats.py:25-80 compute_sparsity_stats_coo; the metrics
 * SparseTensor / DenseTensor compute for every scheme, tensor/sparse.py:122-158,
 * tensor/dense.py:44-94). For each of num_schemes tile shapes U
 * (tile_shapes: host int64 (num_schemes, ndim), sides >= 1):
 *   num_tuples_dev[u]            = T(U), tiles holding a non-zero entry;
 *   value_count_dev[u*ndim + l]  = V(l, U), distinct tile coordinates along l.
 * Entries: COO (indices int32 (num_entries, ndim), values of values_dtype or
 * NULL when every entry counts), or with indices == NULL a dense row-major
 * array `values` of `shape` (num_entries = its element count). Zeros do not
 * count; repeated coordinates count once. A coordinate outside the shape sets
 * *error_dev to ES_ERR_INDEX. Tile grids up to 2^32 tiles use a bitmap (the
 * workspace holds up to 512 MB of them per pass, several schemes per pass);
 * larger grids count distinct tile keys after a radix sort of the entries.
 * workspace: es_sparsity_stats_workspace_size bytes for the same arguments.
 * ------------------------------------------------------------------------- */
size_t es_sparsity_stats_workspace_size(int64_t num_entries, int ndim, const int64_t* shape,
                                        const int64_t* tile_shapes, int num_schemes);
int es_sparsity_stats(const int32_t* indices, const void* values, int values_dtype, int64_t num_entries, int ndim,
                      const int64_t* shape, const int64_t* tile_shapes, int num_schemes, void* workspace,
                      size_t workspace_bytes, int64_t* num_tuples_dev, int64_t* value_count_dev,
                      int32_t* error_dev, void* stream);

/* ---------------------------------------------------------------------------
 * Mixture of experts: a contraction with a token x expert matrix of top_k
 * nonzeros a row, whose blocks are ragged in the token axis. No reference
 * counterpart (its relations have fixed tiles).
 *
 * num_tokens tokens choose top_k (<= 32) of num_experts (<= 1024) experts;
 * choice a = token * top_k + j. Row r of the grouped order belongs to choice
 * order[r]; expert e owns the rows offsets[e] to offsets[e + 1] (int32,
 * num_experts + 1); position[a] is the row of choice a. A choice of no expert
 * (-1) has no row (position -1); the rows from offsets[num_experts] on are
 * empty (order -1) and are zero in every output. Value types: ES_F32,
 * ES_BF16, ES_F16; sums in fp32, rounded once. Row strides are in elements,
 * the last dimension is contiguous. Offsets, orders and positions are bounded
 * on the device: what points outside is left out. `status` (may be NULL) is
 * an int32 that the device can write, pinned host memory included: it is left
 * alone unless the call fails on the device (ES_ERR_INDEX, ES_ERR_TIMEOUT).
 * ------------------------------------------------------------------------- */

/* The top_k largest logits of each token, largest first, ties to the lowest
 * expert, and their weights: exp(logit - max) over its sum, over the chosen
 * experts (renormalize != 0) or over all. -inf masks an expert: where fewer
 * than top_k are left the choice is -1 with weight 0. A NaN logit is never
 * chosen and makes every weight of its token NaN. */
int es_route_experts(const void* logits, int dtype, int64_t num_tokens, int num_experts, int64_t row_stride,
                     int top_k, int renormalize, float* weights, int32_t* experts, void* stream);
/* dlogits (num_tokens, num_experts) contiguous, of the logits' type, from the
 * weights and experts of es_route_experts on the same logits. */
int es_route_experts_grad(const void* logits, int dtype, int64_t num_tokens, int num_experts, int64_t row_stride,
                          int top_k, int renormalize, const float* weights, const int32_t* experts,
                          const float* dweights, void* dlogits, void* stream);

/* offsets, order and position of num_choices choices (int32, -1: none), in
 * ascending choice inside an expert. A choice outside [-1, num_experts) counts
 * as -1 and sets *status to ES_ERR_INDEX. */
size_t es_expert_plan_workspace_size(int64_t num_choices, int num_experts);
int es_expert_plan(const int32_t* experts, int64_t num_choices, int num_experts, void* workspace,
                   size_t workspace_bytes, int32_t* offsets, int32_t* order, int32_t* position, int32_t* status,
                   void* stream);

/* y[r] = x[row(r)] w[e(r)] for the num_rows grouped rows: w[e] is (K, N) with
 * any element strides (num_experts == 0: one matrix for all rows, offsets and
 * order NULL), row(r) = order[r] / top_k when order is given (x by token), else r. y
 * (num_rows, N) contiguous, of out_dtype (ES_F32 or the operands' type). Infinities and NaN give what fp32 arithmetic gives, except
 * that a magnitude below 2^-132 may count as zero beside them. fp32 operands
 * keep all their bits from 2^-109 on, sums from 2^-120 on. The tensor
 * cores' sums truncate: of one sign they come out low by up to 8e-7 (fp32
 * operands, any depth), or a quarter of the rounding to the operands' 16-bit
 * type (also where y is ES_F32). The workspace's size goes by the call's own arguments. */
size_t es_grouped_matmul_workspace_size(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const void* w,
                                        int num_experts, int64_t K, int64_t N, int64_t w_expert_stride,
                                        int64_t w_k_stride, int64_t w_n_stride, const int32_t* offsets,
                                        const int32_t* order, int top_k, int64_t num_rows);
int es_grouped_matmul(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const void* w, int num_experts,
                      int64_t K, int64_t N, int64_t w_expert_stride, int64_t w_k_stride, int64_t w_n_stride,
                      const int32_t* offsets, const int32_t* order, int top_k, int64_t num_rows, void* y,
                      int out_dtype, void* workspace, size_t workspace_bytes, int32_t* status, void* stream);
/* The kernel that a rows' product of these sizes runs on (weights contiguous
 * and 16-byte aligned; the rows' gradient is the product with K and N
 * exchanged), -1 for sizes that have none. */
typedef enum es_grouped_path {
  ES_GROUPED_FEW = 0,         /* fp32, few rows a group: weights cut in registers */
  ES_GROUPED_NARROW = 1,      /* 128 channels x 64 rows */
  ES_GROUPED_SPLIT = 2,       /* the same, the depth shared by a cluster */
  ES_GROUPED_MIDDLE = 3,      /* 256 x 128 */
  ES_GROUPED_WIDE = 4,        /* 512 x 256 of a pair of CTAs (fp32: 256 x 128) */
  ES_GROUPED_DEEP_NARROW = 5, /* 16 bits, long sums: chains with an fp32 total, 128 x 64 */
  ES_GROUPED_DEEP_WIDE = 6    /* 256 x 256 */
} es_grouped_path;
int es_grouped_matmul_path(int dtype, int num_experts, int64_t K, int64_t N, int64_t num_rows);
int es_int8_matmul_path(int num_experts, int64_t K, int64_t N, int64_t num_rows);
/* dw[e] = sum over e's rows of x[row(r)]^T dy[r], with dw's element strides
 * (that of K or of N is 1);
 * zero for an expert without rows. dw has the operands' type. */
size_t es_grouped_matmul_wgrad_workspace_size(const void* x, int dtype, int64_t x_rows, int64_t x_stride,
                                              const void* dy, int64_t dy_stride, int num_experts, int64_t K,
                                              int64_t N, const int32_t* offsets, const int32_t* order, int top_k,
                                              int64_t num_rows, void* dw, int64_t dw_expert_stride,
                                              int64_t dw_k_stride, int64_t dw_n_stride);
int es_grouped_matmul_wgrad(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const void* dy,
                            int64_t dy_stride, int num_experts, int64_t K, int64_t N, const int32_t* offsets,
                            const int32_t* order, int top_k, int64_t num_rows, void* dw, int64_t dw_expert_stride,
                            int64_t dw_k_stride, int64_t dw_n_stride, void* workspace, size_t workspace_bytes,
                            int32_t* status, void* stream);

/* h[r] = act(x[row(r)] gate[e(r)]) * (x[row(r)] up[e(r)]) for the num_rows grouped
 * rows, w[e] = [gate | up] (K, 2F) with any element strides; num_experts == 0: one
 * matrix for all rows (offsets and order NULL). h (num_rows, F) contiguous, of the
 * operands' type; slopes (num_rows, 2F) float32, or NULL: [act'(x gate) * (x up)
 * | act(x gate)], the rows of no expert left alone. */
typedef enum es_activation {
  ES_ACT_SILU = 0,      /* g / (1 + exp(-g)) */
  ES_ACT_GELU = 1,      /* g (1 + erf(g / sqrt(2))) / 2 */
  ES_ACT_GELU_TANH = 2, /* g (1 + tanh(sqrt(2 / pi) (g + 0.044715 g^3))) / 2 */
  ES_ACT_RELU = 3
} es_activation;
size_t es_gated_matmul_workspace_size(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const void* w,
                                      int num_experts, int64_t K, int64_t F, int64_t w_expert_stride,
                                      int64_t w_k_stride, int64_t w_n_stride, const int32_t* offsets,
                                      const int32_t* order, int top_k, int64_t num_rows);
int es_gated_matmul(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const void* w, int num_experts,
                    int64_t K, int64_t F, int64_t w_expert_stride, int64_t w_k_stride, int64_t w_n_stride,
                    const int32_t* offsets, const int32_t* order, int top_k, int64_t num_rows, int activation,
                    void* h, float* slopes, void* workspace, size_t workspace_bytes, int32_t* status, void* stream);
/* The kernel of a gated product of these sizes, an es_grouped_path (lanes are those of
 * h) or ES_GATED_TWO: the product in fp32, then a pass for the activation. -1: none. */
#define ES_GATED_TWO 7
int es_gated_matmul_path(int dtype, int num_experts, int64_t K, int64_t F, int64_t num_rows);
/* dy = dh times the slopes (num_rows, 2F), contiguous: the gradient of [x gate | x up],
 * from which es_grouped_matmul and es_grouped_matmul_wgrad make those of x and w.
 * kept_rows (device int32, or NULL for all): the rows from there on are zero. */
int es_gated_matmul_grad(const void* dh, int dtype, int64_t dh_stride, const float* slopes, int64_t num_rows,
                         int64_t F, const int32_t* kept_rows, void* dy, void* stream);

/* out[t] = sum_j weights[t, j] y[position[t, j]] (weights NULL: 1), y
 * (num_rows, width). out (num_tokens, width) contiguous, of out_dtype: y's
 * type, or any when y is ES_F32. */
int es_combine_experts(const void* y, int dtype, int64_t num_rows, int64_t row_stride, const float* weights,
                       const int32_t* position, int64_t num_tokens, int top_k, int64_t width, void* out,
                       int out_dtype, void* stream);
/* dy[position[t, j]] = weights[t, j] dout[t] and dweights[t, j] = <dout[t],
 * y[position[t, j]]>, zero for -1; kept_rows: device int32, the rows that
 * have a choice (offsets + num_experts), the rows from there on are zeroed.
 * Every row below *kept_rows is the position of one choice. dy contiguous. */
int es_combine_experts_grad(const void* y, int dtype, int64_t num_rows, int64_t row_stride, const float* weights,
                            const int32_t* position, const int32_t* kept_rows, int64_t num_tokens, int top_k,
                            int64_t width, const void* dout, int64_t dout_stride, void* dy, float* dweights,
                            void* stream);

/* q[r, i] = rint(x[r, i] / scale[r]), scale[r] = max |x[r]| / 127 in fp32. A
 * row of zeros has scale 0; a row with an infinity or NaN has scale NaN. */
int es_quantize_rows(const void* x, int dtype, int64_t num_rows, int64_t width, int64_t row_stride, int8_t* q,
                     float* scale, void* stream);

/* y[r, n] = x_scale[row(r)] w_scale[e(r), n] sum_k q[row(r), k] wq[e(r), n, k],
 * the sum exact in 32-bit integers (K <= 131071). wq: (num_experts, N, K) int8
 * with contiguous k, w_scale (num_experts, N). num_experts == 0: one matrix
 * for all rows (offsets and order NULL). y (num_rows, N) contiguous. */
size_t es_int8_matmul_workspace_size(const int8_t* q, const float* x_scale, int64_t x_rows, int64_t x_stride,
                                     const int8_t* wq, const float* w_scale, int num_experts, int64_t K, int64_t N,
                                     int64_t w_expert_stride, int64_t w_n_stride, const int32_t* offsets,
                                     const int32_t* order, int top_k, int64_t num_rows);
int es_int8_matmul(const int8_t* q, const float* x_scale, int64_t x_rows, int64_t x_stride, const int8_t* wq,
                   const float* w_scale, int num_experts, int64_t K, int64_t N, int64_t w_expert_stride,
                   int64_t w_n_stride, const int32_t* offsets, const int32_t* order, int top_k, int64_t num_rows,
                   void* y, int out_dtype, void* workspace, size_t workspace_bytes, int32_t* status, void* stream);

/* ---------------------------------------------------------------------------
 * 8-bit floating point (e4m3: 4 exponent and 3 mantissa bits, largest 448, no
 * infinity) with a float32 scale for each block of 128: the serving form beside
 * the 8-bit integers above, with the same groups, orders and status.
 * ------------------------------------------------------------------------- */

/* q[r, i] = e4m3(x[r, i] / s), to nearest, ties to even, s = scale[r, i / 128]
 * the smallest power of two (at least 2^-126) with max |x| <= 448 s over the
 * block. A block with an infinity or NaN has scale and values NaN. activation
 * (es_activation, -1: none): x is (num_rows, 2 width), and act(x[r, i]) *
 * x[r, width + i] is rounded, made in fp32. q (num_rows, width) and scale
 * (num_rows, ceil(width / 128)) contiguous. */
int es_quantize_blocks(const void* x, int dtype, int64_t num_rows, int64_t width, int64_t row_stride, int activation,
                       uint8_t* q, float* scale, void* stream);
/* The same for blocks of 128 x 128 of contiguous matrices (matrices, N, K);
 * scale (matrices, ceil(N / 128), ceil(K / 128)). */
int es_quantize_block_weights(const void* w, int dtype, int64_t matrices, int64_t N, int64_t K, uint8_t* q,
                              float* scale, void* stream);
/* y[r, n] = sum_b x_scale[row(r), b] w_scale[e(r), n / 128, b] sum_{k in b} q[row(r), k] wq[e(r), n, k]
 * over the blocks b of the depth, in fp32, rounded once; any fp32 scales (where a
 * row has a product of two scales of 2^36 or more, its terms below 2^-85 may be lost). wq:
 * (num_experts, N, K) with contiguous k, the scales contiguous. num_experts ==
 * 0: one matrix for all rows (offsets and order NULL). y (num_rows, N)
 * contiguous. */
size_t es_fp8_matmul_workspace_size(const uint8_t* q, const float* x_scale, int64_t x_rows, int64_t x_stride,
                                    const uint8_t* wq, const float* w_scale, int num_experts, int64_t K, int64_t N,
                                    int64_t w_expert_stride, int64_t w_n_stride, const int32_t* offsets,
                                    const int32_t* order, int top_k, int64_t num_rows);
int es_fp8_matmul(const uint8_t* q, const float* x_scale, int64_t x_rows, int64_t x_stride, const uint8_t* wq,
                  const float* w_scale, int num_experts, int64_t K, int64_t N, int64_t w_expert_stride,
                  int64_t w_n_stride, const int32_t* offsets, const int32_t* order, int top_k, int64_t num_rows,
                  void* y, int out_dtype, void* workspace, size_t workspace_bytes, int32_t* status, void* stream);
/* The kernel of a product of these sizes (ES_GROUPED_SPLIT, _NARROW: 128 rows x
 * 128 channels, _WIDE: 256 x 256 of a pair of CTAs), -1 for sizes that have none. */
int es_fp8_matmul_path(int num_experts, int64_t K, int64_t N, int64_t num_rows);

/* ---------------------------------------------------------------------------
 * Norms before and after a block, with its gate and residual scale. Rows of
 * `width` contiguous values (row strides in elements), rms(v) = sqrt(mean(v^2)
 * + eps), all in fp32 and rounded once:
 *   z = h norm_out / rms(h)  (norm_out NULL: z = h),
 *   out = x + scale gate z,   y = out norm_in / rms(out)
 * norm_in NULL: no y. h NULL: out = x is not written, and there is no gate and
 * no norm_out. x, h, gate, out and y have one type (ES_F32, ES_BF16, ES_F16),
 * the norms' weights (width) have it or are ES_F32. out and y (num_rows, width)
 * are contiguous. stats (may be NULL): float32 (num_rows, 2) for the gradient.
 * ------------------------------------------------------------------------- */
typedef enum es_gate {
  ES_GATE_NONE = 0,
  ES_GATE_CHANNEL = 1, /* gate (width) */
  ES_GATE_TOKEN = 2,   /* one value a row, gate_stride elements apart */
  ES_GATE_FULL = 3     /* (num_rows, width), rows gate_stride elements apart */
} es_gate;
int es_residual_norm(const void* x, int64_t x_stride, const void* h, int64_t h_stride, int dtype, int64_t num_rows,
                     int64_t width, const void* norm_in, const void* norm_out, int weight_dtype, const void* gate,
                     int gate_kind, int64_t gate_stride, float scale, float eps, void* out, void* y, float* stats,
                     void* stream);
/* Gradients from dout and dy (NULL: zero) and the forward pass's stats. dx, dh,
 * dgate, dnorm_in, dnorm_out: NULL for what is not wanted; contiguous, of the
 * types and shapes of x, h, gate and the norms. num_columns of the workspace:
 * how many of dnorm_in, dnorm_out and a dgate by channel are wanted. */
size_t es_residual_norm_grad_workspace_size(int dtype, int64_t num_rows, int64_t width, int num_columns);
int es_residual_norm_grad(const void* x, int64_t x_stride, const void* h, int64_t h_stride, int dtype,
                          int64_t num_rows, int64_t width, const void* norm_in, const void* norm_out,
                          int weight_dtype, const void* gate, int gate_kind, int64_t gate_stride, float scale,
                          const float* stats, const void* dout, int64_t dout_stride, const void* dy,
                          int64_t dy_stride, void* dx, void* dh, void* dgate, void* dnorm_in, void* dnorm_out,
                          void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* EINSPARSE_H */
