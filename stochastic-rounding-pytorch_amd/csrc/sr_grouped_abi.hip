// sr_grouped_abi.hip -- extern "C" entry points of the grouped casts and products (sr_matrix_hip.h).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/sr_matrix_hip.h"
#include "sr_block_tables.h"
#include "sr_grouped.h"
#include "sr_matrix_launch.h"

namespace {

using sr::aligned_rows;
using sr::blocks;
using sr::check_matrix;
using sr::fail;
using sr::kMaxLd;
using sr::kMaxRows;
using sr::launch;

const sr::GroupedProductTable& products() {
  static const struct Tables {
    sr::GroupedProductTable t{};
    Tables() {
      sr::register_grouped_product_e4m3(t);
      sr::register_grouped_product_e5m2(t);
    }
  } tables;
  return tables.t;
}

const sr::GroupedCastTable& casts() {
  static const struct Tables {
    sr::GroupedCastTable t{};
    Tables() { sr::register_grouped_cast(t); }
  } tables;
  return tables.t;
}

int check_groups(const sr_groups* g) {
  if (!g) return fail(SR_ERR_ARGUMENT, "null argument");
  if (g->count < 0 || g->count > SR_MATRIX_GROUPS)
    return fail(SR_ERR_ARGUMENT, "%d groups: at most %d", g->count, SR_MATRIX_GROUPS);
  if (g->count && !g->sizes) return fail(SR_ERR_ARGUMENT, "null pointer");
  return SR_OK;
}

sr::Groups groups_of(const sr_groups* g) { return {g->sizes, g->count, g->wide != 0}; }

// The checks that every cast makes, and its arguments; *empty where there is nothing to do.
int cast_args(const void* x, int64_t ldx, int64_t rows, int64_t cols, int64_t stored, int x_dtype, int dtype, int rule,
              uint32_t counter_base, const sr_block_output* by_rows, const sr_block_output* by_cols, sr::BlockCastArgs* a) {
  if (x_dtype != SR_F32 && x_dtype != SR_BF16 && x_dtype != SR_F16)
    return fail(SR_ERR_ARGUMENT, "block casts take FP32, BF16 or FP16, not dtype %d", x_dtype);
  if (dtype != SR_E4M3 && dtype != SR_E5M2) return fail(SR_ERR_ARGUMENT, "block casts give E4M3 or E5M2, not dtype %d", dtype);
  if (rule != SR_NEAREST && rule != SR_STOCHASTIC) return fail(SR_ERR_ARGUMENT, "unknown rounding rule %d", rule);
  if (rows < 0 || cols < 0 || rows > kMaxRows || cols > kMaxRows)
    return fail(SR_ERR_ARGUMENT, "%lld x %lld matrix", (long long)rows, (long long)cols);
  const sr_block_output none{};
  a->by_rows = by_rows ? *by_rows : none;
  a->by_cols = by_cols ? *by_cols : none;
  if (!a->by_rows.data && !a->by_cols.data) return fail(SR_ERR_ARGUMENT, "no output");
  if (rows && cols) {
    if (!x || (a->by_rows.data && !a->by_rows.scale) || (a->by_cols.data && !a->by_cols.scale))
      return fail(SR_ERR_ARGUMENT, "null pointer");
    if ((rows > 1 && ldx < cols) || (a->by_rows.data && (a->by_rows.ld < cols || a->by_rows.ld_scale < 0)) ||
        (a->by_cols.data && (a->by_cols.ld < stored || a->by_cols.ld_scale < 0)))
      return fail(SR_ERR_ARGUMENT, "rows overlap");
  }
  a->x = static_cast<const char*>(x);
  a->ldx = ldx;
  a->rows = rows;
  a->cols = cols;
  a->counter_base = counter_base;
  a->tiles_n = static_cast<uint32_t>(blocks(cols));
  return SR_OK;
}

const void* cast_kernel(int x_dtype, int dtype, int rule, sr::GroupedCastKind kind) {
  return casts()[x_dtype == SR_F32 ? 0 : (x_dtype == SR_BF16 ? 1 : 2)][2 * (dtype == SR_E5M2) + (rule == SR_STOCHASTIC)][kind];
}

// `groups` workgroups in launches of fewer than 2^32 threads each; *first is the argument that counts them.
int launch_cast(const void* fn, uint64_t groups, int threads, void* args, uint32_t* first, void* stream) {
  if (groups > 0xFFFFFFFFu) return fail(SR_ERR_ARGUMENT, "%llu workgroups exceed a cast", (unsigned long long)groups);
  constexpr uint64_t kLaunch = 0x7FFFFF / 2;
  for (uint64_t at = 0; at < groups; at += kLaunch) {
    *first = static_cast<uint32_t>(at);
    if (int rc = launch(fn, std::min(kLaunch, groups - at), threads, args, stream)) return rc;
  }
  return SR_OK;
}

// What both products check and pass on.
int product_args(const sr_block_matrix* a, const sr_block_matrix* b, int64_t k, int out_dtype, const sr_groups* groups,
                 sr::GroupedProductArgs* g) {
  if (k < 0 || k > kMaxLd) return fail(SR_ERR_ARGUMENT, "%lld contracted values", (long long)k);
  if (int rc = check_matrix(a, "a", k)) return rc;
  if (int rc = check_matrix(b, "b", k)) return rc;
  if (int rc = check_groups(groups)) return rc;
  if (a->scale_type != b->scale_type) return fail(SR_ERR_ARGUMENT, "a and b have different scale types");
  if (out_dtype != SR_F32 && out_dtype != SR_BF16 && out_dtype != SR_F16)
    return fail(SR_ERR_ARGUMENT, "products are FP32, BF16 or FP16, not dtype %d", out_dtype);
  sr::BlockProductArgs& p = g->p;
  p.a = {static_cast<const char*>(a->data), a->ld, static_cast<int>(a->rows)};
  p.b = {static_cast<const char*>(b->data), b->ld, static_cast<int>(b->rows)};
  p.scale_a = static_cast<const char*>(a->scale);
  p.scale_b = static_cast<const char*>(b->scale);
  p.ld_scale_a = a->ld_scale;
  p.ld_scale_b = b->ld_scale;
  p.shift_a = a->block_rows == 1 ? 0 : 7;
  p.shift_b = b->block_rows == 1 ? 0 : 7;
  p.k = k;
  p.m = static_cast<int>(a->rows);
  p.n = static_cast<int>(b->rows);
  p.out_dtype = out_dtype;
  p.scale_f32 = a->scale_type == SR_SCALE_F32;
  g->groups = groups_of(groups);
  return SR_OK;
}

const sr::GroupedProductKernels& kernels(const sr_block_matrix* a, const sr_block_matrix* b, int out_dtype) {
  const int mode = out_dtype == SR_F32 ? sr::kWide : (a->scale_type == SR_SCALE_F32 ? sr::kFactors : sr::kExponents);
  return products()[a->dtype == SR_E5M2][b->dtype == SR_E5M2][mode];
}

// use(tile's index, its shape).
template <class F>
int with_tile(sr::BlockTile tile, F&& use) {
  switch (tile) {
    case sr::kTile128: return use(sr::kTile128, sr::Tile128{});
    case sr::kTile64x2: return use(sr::kTile64x2, sr::Tile64x2{});
    case sr::kTile64x4: return use(sr::kTile64x4, sr::Tile64x4{});
    default: return use(sr::kTile64, sr::Tile64{});
  }
}

}  // namespace

extern "C" {

int64_t sr_grouped_columns(int64_t rows, int64_t groups) {
  if (rows < 0 || rows > kMaxRows || groups <= 0) return 0;
  return (rows + (SR_BLOCK - 1) * std::min(rows, groups)) / SR_BLOCK * SR_BLOCK;
}

int sr_grouped_block_cast(const void* x, int64_t ldx, int64_t rows, int64_t cols, int x_dtype, int dtype, int rule,
                          uint32_t seed, uint32_t offset, const sr_groups* groups, const sr_block_output* by_rows,
                          const sr_block_output* by_cols, void* stream) {
  if (int rc = check_groups(groups)) return rc;
  const int64_t columns = sr_grouped_columns(rows, groups->count);
  sr::GroupedCastArgs g{};
  if (int rc = cast_args(x, ldx, rows, cols, columns, x_dtype, dtype, rule, seed + offset, by_rows, by_cols, &g.c)) return rc;
  if (!g.c.by_cols.data) return fail(SR_ERR_ARGUMENT, "no output along the groups' rows");
  if (rows == 0 || cols == 0) return SR_OK;
  g.groups = groups_of(groups);
  g.column_blocks = static_cast<uint32_t>(columns / SR_BLOCK);
  const bool rows_too = g.c.by_rows.data;
  // Blocks of the groups and of the rows behind them.
  const uint64_t tiles = std::max<uint64_t>(g.column_blocks, sr_grouped_columns(rows, groups->count + int64_t{1}) / SR_BLOCK) * g.c.tiles_n;
  if (rows_too && static_cast<uint64_t>(blocks(rows)) * g.c.tiles_n >= sr::kWholeTiles)
    return launch_cast(cast_kernel(x_dtype, dtype, rule, sr::kGroupedWhole), tiles, sr::kTileThreads, &g, &g.c.first, stream);
  const uint64_t parts = static_cast<uint64_t>(g.column_blocks) * sr::kColParts +
                         (rows_too ? (static_cast<uint64_t>(rows) + sr::kPartRows - 1) / sr::kPartRows : 0);
  return launch_cast(cast_kernel(x_dtype, dtype, rule, sr::kGroupedParts), parts * g.c.tiles_n, sr::kPartThreads, &g, &g.c.first, stream);
}

int sr_stacked_block_cast(const void* x, int64_t x_stride, int64_t ldx, int64_t count, int64_t rows, int64_t cols, int x_dtype,
                          int dtype, int rule, int square, uint32_t seed, uint32_t offset, const sr_block_stack* by_rows,
                          const sr_block_stack* by_cols, void* stream) {
  sr::StackedCastArgs s{};
  if (count < 0 || count > SR_MATRIX_GROUPS) return fail(SR_ERR_ARGUMENT, "%lld matrices: at most %d", (long long)count, SR_MATRIX_GROUPS);
  if (int rc = cast_args(x, ldx, rows, cols, rows, x_dtype, dtype, rule, seed + offset, by_rows ? &by_rows->out : nullptr,
                         by_cols ? &by_cols->out : nullptr, &s.c))
    return rc;
  if (count == 0 || rows == 0 || cols == 0) return SR_OK;
  s.stride_x = x_stride * (x_dtype == SR_F32 ? 4 : 2);
  if (by_rows) {
    s.rows_data = by_rows->stride;
    s.rows_scale = by_rows->stride_scale;
  }
  if (by_cols) {
    s.cols_data = by_cols->stride;
    s.cols_scale = by_cols->stride_scale;
  }
  const bool rows_too = s.c.by_rows.data, cols_too = s.c.by_cols.data;
  const uint64_t tiles = static_cast<uint64_t>(blocks(rows)) * s.c.tiles_n;
  const sr::GroupedCastKind kind = square ? sr::kStackedSquare
                                   : rows_too && cols_too && tiles * count >= sr::kWholeTiles ? sr::kStackedWhole
                                                                                              : sr::kStackedParts;
  const uint64_t each = tiles * (kind == sr::kStackedParts ? sr::kRowParts * rows_too + sr::kColParts * cols_too : 1);
  if (each > 0xFFFFFFFFu) return fail(SR_ERR_ARGUMENT, "%lld x %lld matrix", (long long)rows, (long long)cols);
  s.each = static_cast<uint32_t>(each);
  return launch_cast(cast_kernel(x_dtype, dtype, rule, kind), each * count,
                     kind == sr::kStackedParts ? sr::kPartThreads : sr::kTileThreads, &s, &s.c.first, stream);
}

int sr_grouped_block_matmul(const sr_block_matrix* a, const sr_block_matrix* b, int64_t b_stride, int64_t b_stride_scale,
                            int64_t k, const sr_groups* groups, void* out, int64_t ldo, int out_dtype, int zero_behind,
                            void* stream) {
  sr::GroupedProductArgs g{};
  if (int rc = product_args(a, b, k, out_dtype, groups, &g)) return rc;
  if (a->rows == 0 || b->rows == 0) return SR_OK;
  if (!out) return fail(SR_ERR_ARGUMENT, "null pointer");
  if (a->rows > 1 && ldo < b->rows) return fail(SR_ERR_ARGUMENT, "rows of the result overlap");
  if (b_stride < 0 || b_stride_scale < 0) return fail(SR_ERR_ARGUMENT, "negative strides");
  g.p.out = static_cast<char*>(out);
  g.p.ldo = ldo;
  g.stride = b_stride;
  g.stride_scale = b_stride_scale * (g.p.scale_f32 ? 4 : 1);
  g.zero_behind = zero_behind != 0;
  const sr::GroupedProductKernels& fn = kernels(a, b, out_dtype);
  const int64_t rows = a->rows, full = std::min<int64_t>(groups->count, rows);  // groups that can have rows
  // Room for any sizes: every group, and the rows behind them, may end inside a tile.
  auto room = [&](int64_t side) { return static_cast<uint64_t>((rows + (side - 1) * (full + g.zero_behind)) / side); };
  const bool async = aligned_rows(a) && aligned_rows(b) && b_stride % 16 == 0;
  // Tiles to expect: one a group where groups are small, and half a tile more than its rows fill where they are large.
  auto tiles = [&](int64_t side) { return std::max(full, rows / side + (full + 1) / 2) * ((g.p.n + side - 1) / side); };
  // Few rows a group to few columns: a wave's own loads have less to wait for than a tile's stages (4 groups by 2048 x 2048: 4
  // rows each 6.9 us and 7.9, 8 rows 7.3 and 7.9, 12 rows 10.4 and 8.0; 16 groups, 8 rows in all, 256 tiles 6.9 and 7.9; 64
  // groups, 12 rows in all, 384 tiles 14.0 and 11.1).
  if (rows <= 8 * full && tiles(64) <= 256) {
    g.p.tiles_n = (g.p.n + 15) / 16;
    return launch(fn.rows, room(16) * g.p.tiles_n, 64 * sr::kRowWaves, &g, stream);
  }
  const sr::BlockTile tile = sr::tile_by_count(tiles);
  if (fn.lean[0] && async && k % SR_BLOCK == 0 && tiles(128) > sr::kLeanTiles) {
    g.p.tiles_n = (g.p.n + 127) / 128;
    return launch(fn.lean[0], room(128) * g.p.tiles_n, 256, &g, stream);
  }
  return with_tile(async || tile == sr::kTile128 ? tile : sr::kTile64, [&](sr::BlockTile index, auto shape) {
    using S = decltype(shape);
    g.p.tiles_n = (g.p.n + S::BN - 1) / S::BN;
    return launch(fn.tile[index][async], room(S::BM) * g.p.tiles_n, S::kThreads, &g, stream);
  });
}

int sr_grouped_block_contract(const sr_block_matrix* a, const sr_block_matrix* b, int64_t columns, const sr_groups* groups,
                              void* out, int64_t ldo, int64_t out_stride, int out_dtype, void* stream) {
  sr::GroupedProductArgs g{};
  if (int rc = product_args(a, b, columns, out_dtype, groups, &g)) return rc;
  if (columns % SR_BLOCK) return fail(SR_ERR_ARGUMENT, "%lld columns of padded groups", (long long)columns);
  if (a->rows == 0 || b->rows == 0 || groups->count == 0) return SR_OK;
  if (!out) return fail(SR_ERR_ARGUMENT, "null pointer");
  if ((a->rows > 1 && ldo < b->rows) || (groups->count > 1 && out_stride < (a->rows - 1) * ldo + b->rows))
    return fail(SR_ERR_ARGUMENT, "rows of the result overlap");
  if (columns && (!aligned_rows(a) || !aligned_rows(b))) return fail(SR_ERR_ARGUMENT, "rows of padded groups start on 16 bytes");
  g.p.out = static_cast<char*>(out);
  g.p.ldo = ldo;
  g.stride_out = out_stride;
  const sr::GroupedProductKernels& fn = kernels(a, b, out_dtype);
  auto tiles = [&](int64_t side) { return groups->count * ((g.p.m + side - 1) / side) * ((g.p.n + side - 1) / side); };
  if (fn.lean[1] && tiles(128) > sr::kLeanTiles) {
    g.p.tiles_m = (g.p.m + 127) / 128;
    g.p.tiles_n = (g.p.n + 127) / 128;
    return launch(fn.lean[1], static_cast<uint64_t>(sr::contract_groups(g.p.tiles_m * g.p.tiles_n)) * groups->count, 256, &g, stream);
  }
  return with_tile(sr::tile_by_count(tiles), [&](sr::BlockTile index, auto shape) {
    using S = decltype(shape);
    g.p.tiles_m = (g.p.m + S::BM - 1) / S::BM;
    g.p.tiles_n = (g.p.n + S::BN - 1) / S::BN;
    return launch(fn.contract[index], static_cast<uint64_t>(sr::contract_groups(g.p.tiles_m * g.p.tiles_n)) * groups->count, S::kThreads, &g, stream);
  });
}

}  // extern "C"
