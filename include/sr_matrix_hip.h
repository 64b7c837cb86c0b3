/*
 * sr_matrix_hip.h -- C ABI of the matrix operators of libsr_states_hip.so:
 * FP8 products with a scale for each block of 128, also of rows in groups with
 * a matrix each, low-rank adapters, and orthogonalised (Muon) updates.
 *
 * The conventions are those of sr_states_hip.h: 0 or an SR_ERR_* code is
 * returned, sr_last_error() holds the message, `stream` is a hipStream_t on
 * the current device, launches are asynchronous on it and nothing
 * synchronizes or allocates.  Pointers are device memory unless said
 * otherwise and are borrowed until the stream has consumed them.  Matrices
 * are row-major with consecutive columns; `ld*` is the distance between rows,
 * in elements.  Dtypes are enum sr_dtype.
 */
#ifndef SR_MATRIX_HIP_H
#define SR_MATRIX_HIP_H

#include "sr_states_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SR_MATRIX_ABI_VERSION 1

/* Values that share a scale along the contracted axis. */
#define SR_BLOCK 128

/* How the scales of a block-scaled matrix are stored: the exponent byte of a
 * power of two (2^(byte - 127)), or any FP32 factor. */
enum sr_scale_type {
  SR_SCALE_E8M0 = 0,
  SR_SCALE_F32 = 1
};

/* One FP8 matrix (rows x k, the contracted axis last) with a scale for each
 * block of 128 columns of one row (block_rows = 1) or of 128 rows
 * (block_rows = 128): scale[r / block_rows * ld_scale + c / 128]. */
typedef struct sr_block_matrix {
  const void* data;
  const void* scale;
  int64_t ld;       /* bytes between rows of data; at most 2^24 */
  int64_t ld_scale; /* elements between rows of scale; at most 2^20 */
  int64_t rows;
  int dtype;        /* SR_E4M3 or SR_E5M2 */
  int scale_type;   /* enum sr_scale_type */
  int block_rows;   /* 1 or 128 */
  int reserved;
} sr_block_matrix;

/* Where one orientation of a block cast goes; data NULL: not wanted. */
typedef struct sr_block_output {
  void* data;       /* FP8 */
  void* scale;      /* E8M0 bytes */
  int64_t ld;
  int64_t ld_scale;
} sr_block_output;

/* Returns SR_MATRIX_ABI_VERSION. */
int sr_matrix_abi_version(void);

/* Quantizes x (rows x cols; FP32, BF16 or FP16) to FP8 `dtype` with a power
 * of two for each block of 128.
 *
 * A block's scale is the smallest 2^e, e >= -127, for which its largest
 * finite |x| is at most 2^e times the format's maximum (1 for a block
 * without a nonzero finite value).  Each value is x 2^-e rounded by `rule`
 * as sr_cast rounds it: counter row * cols + col + seed + offset, saturating,
 * NaN kept.
 *
 * `by_rows` receives blocks along the columns: data rows x cols, scale
 * rows x ceil(cols / 128).  `by_cols` receives blocks along the rows, both
 * transposed: data cols x rows, scale cols x ceil(rows / 128).  Blocks are
 * 1 x 128 along those axes, or 128 x 128 with `square` (one scale row per 128
 * rows of data).  One call fills both. */
int sr_block_cast(const void* x, int64_t ldx, int64_t rows, int64_t cols, int x_dtype, int dtype, int rule,
                  int square, uint32_t seed, uint32_t offset, const sr_block_output* by_rows,
                  const sr_block_output* by_cols, void* stream);

/* out (m x n; FP32, BF16 or FP16) = A B^T of two block-scaled matrices with k
 * contracted values:
 *   out[i,j] = sum over blocks of scale_a scale_b sum in the block of a b
 * summed in FP32 and rounded once.  Both matrices have the same scale type.
 * m = a->rows and n = b->rows. */
int sr_block_matmul(const sr_block_matrix* a, const sr_block_matrix* b, int64_t k, void* out, int64_t ldo,
                    int out_dtype, void* stream);

/* ---- rows sorted into groups ------------------------------------------- */

/* Groups that one call takes. */
#define SR_MATRIX_GROUPS 4096

/* How many rows each of `count` groups has, in order from row 0 on: device
 * memory, int64 where `wide`, else int32, read when the stream comes to it.
 * Sizes below zero count as zero, and groups end where the matrix does. */
typedef struct sr_groups {
  const void* sizes;
  int count;
  int wide;
} sr_groups;

/* Columns of a matrix whose contracted axis is `rows` rows in `groups` groups
 * that each start on a multiple of 128 columns: room for any sizes. */
int64_t sr_grouped_columns(int64_t rows, int64_t groups);

/* sr_block_cast with 1 x 128 blocks, whose blocks along the rows are those of
 * each group by itself: in `by_cols` (wanted; data cols x
 * sr_grouped_columns(rows, count)) a group's columns start on the next
 * multiple of 128 behind the group before, and zeros with a scale of 1 fill
 * what belongs to no row.  `by_rows` is that of sr_block_cast, with the rows
 * behind the last group. */
int sr_grouped_block_cast(const void* x, int64_t ldx, int64_t rows, int64_t cols, int x_dtype, int dtype, int rule,
                          uint32_t seed, uint32_t offset, const sr_groups* groups, const sr_block_output* by_rows,
                          const sr_block_output* by_cols, void* stream);

/* One orientation of the casts of several matrices, `stride` bytes and
 * `stride_scale` scales apart. */
typedef struct sr_block_stack {
  sr_block_output out;
  int64_t stride;
  int64_t stride_scale;
} sr_block_stack;

/* sr_block_cast of `count` matrices (at most SR_MATRIX_GROUPS), each by
 * itself, `x_stride` elements apart.  Value (i, r, c) uses counter
 * (i * rows + r) * cols + c + seed + offset. */
int sr_stacked_block_cast(const void* x, int64_t x_stride, int64_t ldx, int64_t count, int64_t rows, int64_t cols, int x_dtype,
                          int dtype, int rule, int square, uint32_t seed, uint32_t offset, const sr_block_stack* by_rows,
                          const sr_block_stack* by_cols, void* stream);

/* out[t] = a[t] b[i]^T for the rows t of every group i, where b is
 * groups->count matrices, `b_stride` bytes and `b_stride_scale` scales apart;
 * otherwise as sr_block_matmul.  Where 128 rows of a share a scale, they are
 * counted from a's first row, wherever groups start.  Rows behind the last
 * group become zeros with `zero_behind`, and keep what they hold without it. */
int sr_grouped_block_matmul(const sr_block_matrix* a, const sr_block_matrix* b, int64_t b_stride, int64_t b_stride_scale,
                            int64_t k, const sr_groups* groups, void* out, int64_t ldo, int out_dtype, int zero_behind,
                            void* stream);

/* out[i] = a[:, columns of group i] b[:, columns of group i]^T for every group,
 * zeros for one without rows; results are `out_stride` elements apart.  Both
 * matrices have `columns` columns laid out as sr_grouped_block_cast's `by_cols`
 * (a multiple of 128; rows start on 16 bytes).  The values behind a group's
 * rows in its last block of 128 take part: a cast leaves zeros there. */
int sr_grouped_block_contract(const sr_block_matrix* a, const sr_block_matrix* b, int64_t columns, const sr_groups* groups,
                              void* out, int64_t ldo, int64_t out_stride, int out_dtype, void* stream);

/* ---- low-rank adapters ------------------------------------------------- */

/* Adapters that one call takes. */
#define SR_MATRIX_ADAPTERS 65536

/* `count` low-rank updates of one linear layer: a (count x rank x k) and b
 * (count x n x rank), contiguous, of one dtype (FP32, BF16 or FP16; rank 1 to
 * 128). `index` holds each row's adapter (int64 where `wide`, else int32); a
 * row whose number is outside [0, count) has none.  An adapter's update is
 * scaled by its number in `scaling`, or by `scale` where that is NULL. */
typedef struct sr_adapters {
  const void* a;
  const void* b;
  const void* index;
  const float* scaling;
  float scale;
  int count;
  int rank;
  int dtype;
  int wide;
} sr_adapters;

/* FP32 values that sr_adapter_add leaves in `low` for so many rows; 0 for
 * shapes that it refuses. */
int64_t sr_adapter_low(int64_t rows, int64_t k, int64_t rank, int dtype);

/* out[t] = base[t] + s_i (x[t] a_i^T) b_i^T for i = index[t], and base[t] for
 * rows without an adapter.  x (rows x k), base and out (rows x n; out may be
 * base itself) have the adapters' dtype.  `low` receives s_i x[t] a_i^T, in
 * parts, for sr_adapter_backward; with BF16 the second product takes it to
 * 2^-15 of itself, as the gradients' second products take theirs. */
int sr_adapter_add(const sr_adapters* g, const void* x, int64_t ldx, int64_t k, const void* base, int64_t ldbase, int64_t n,
                   int64_t rows, void* out, int64_t ldo, float* low, void* stream);

/* Bytes of workspace for the gradients; 0 for shapes that they refuse. */
int64_t sr_adapter_workspace(int64_t rows, int64_t k, int64_t n, int64_t count, int64_t rank, int dtype);

/* The gradients of sr_adapter_add for dy (rows x n), each where it is not NULL,
 * all of the adapters' dtype:
 *   dx[t] = s_i (dy[t] b_i) a_i                (rows x k; zeros without an adapter)
 *   da_i  = sum over i's rows of (s_i dy[t] b_i)^T x[t]     (count x rank x k)
 *   db_i  = sum over i's rows of dy[t]^T (s_i x[t] a_i^T)   (count x n x rank)
 * Adapters without rows get zeros.  `low` is what sr_adapter_add left. */
int sr_adapter_backward(const sr_adapters* g, const void* x, int64_t ldx, int64_t k, const void* dy, int64_t lddy, int64_t n,
                        int64_t rows, const float* low, void* dx, int64_t lddx, void* da, void* db, void* workspace,
                        void* stream);

/* ---- orthogonalised updates -------------------------------------------- */

/* Newton-Schulz orthogonalisation of a matrix X (rows x cols): X / (|X|_F +
 * eps), then `steps` times X <- a X + (b G + c G^2) X with G = X X^T (X^T X
 * on the right where rows > cols).  The products take FP16 operands scaled by
 * powers of two and sum in FP32; X itself is carried in FP32.  Singular
 * values must stay at or below 2.5 and |b s^2 + c s^4| + 1.5 at or below 7 on
 * the way, which the caller checks (the customary coefficients stay at 1.3
 * and 4.3). */
typedef struct sr_newton_schulz {
  float a, b, c;
  float eps;
  int steps; /* at least 1 */
} sr_newton_schulz;

/* Matrices one launch takes; longer batches run in turn. */
#define SR_MATRIX_BATCH 64

/* Bytes of workspace for `batch` matrices of this shape; 0 for none, and for a
 * shape that the entries below refuse (a side above 2^20, or more than 2^31
 * elements). */
int64_t sr_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols);

/* out[i] = the orthogonalised x[i] (each contiguous rows x cols; x FP32, BF16
 * or FP16; out FP32, BF16 or FP16) for i < batch, `x_stride` and `out_stride`
 * elements apart.  out may be x itself when the dtypes are equal. */
int sr_orthogonalize(const void* x, void* out, int64_t batch, int64_t x_stride, int64_t out_stride, int64_t rows,
                     int64_t cols, int x_dtype, int out_dtype, const sr_newton_schulz* ns, void* workspace,
                     void* stream);

/* One parameter of a Muon step. */
typedef struct sr_muon_row {
  void* p;           /* FP32 or BF16 */
  const void* g;     /* FP32 or BF16 */
  void* u;           /* momentum, any sr_dtype */
  uint32_t key;      /* update key */
  uint32_t offset;   /* flat index of the first element */
} sr_muon_row;

typedef struct sr_muon_hparams {
  float momentum;
  float decay;       /* f32(1 - lr * weight_decay) */
  float neg_lr;      /* f32(-lr * scale of the update) */
  int nesterov;
} sr_muon_hparams;

/* A Muon step of `nrows` contiguous rows x cols parameters (`table` is HOST
 * memory, read during the call):
 *   u = momentum u + g, stored with u's format (counter index + state_key(key, 0) + offset)
 *   v = g + momentum u with nesterov, else u (the unrounded u)
 *   p = decay p + neg_lr orthogonalize(v)
 * `workspace` holds sr_orthogonalize_workspace(nrows, rows, cols) bytes. */
int sr_muon_multi(const sr_muon_row* table, int nrows, int64_t rows, int64_t cols, int p_dtype, int g_dtype,
                  int u_dtype, int u_rule, const sr_muon_hparams* hp, const sr_newton_schulz* ns, void* workspace,
                  void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SR_MATRIX_HIP_H */
