// sr_matrix_abi.hip -- extern "C" entry points of the block-scaled operators (sr_matrix_hip.h).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/sr_matrix_hip.h"
#include "sr_block_scaled.h"
#include "sr_block_tables.h"
#include "sr_error.h"

namespace {

using sr::fail;

constexpr int64_t kMaxRows = 0x7FFFFFFF - 256;  // row indices of a tile stay in 32 bits
constexpr int64_t kMaxLd = 1 << 24, kMaxScaleLd = 1 << 20;

const sr::BlockProductTable& products() {
  static const struct Tables {
    sr::BlockProductTable t{};
    Tables() {
      sr::register_block_product_e4m3(t);
      sr::register_block_product_e5m2(t);
    }
  } tables;
  return tables.t;
}

const sr::BlockCastTable& casts() {
  static const struct Tables {
    sr::BlockCastTable t{};
    Tables() { sr::register_block_cast(t); }
  } tables;
  return tables.t;
}

int launch(const void* fn, uint64_t groups, int threads, void* arg, void* stream) {
  if (groups > 0x7FFFFFu) return fail(SR_ERR_ARGUMENT, "%llu workgroups exceed a launch", (unsigned long long)groups);
  void* args[] = {arg};
  const hipError_t err = hipLaunchKernel(fn, dim3(static_cast<uint32_t>(groups)), dim3(threads), args, 0,
                                         static_cast<hipStream_t>(stream));
  return err == hipSuccess ? SR_OK : sr::hip_fail(err, "hipLaunchKernel");
}

int64_t blocks(int64_t n) { return (n + SR_BLOCK - 1) / SR_BLOCK; }

int check_matrix(const sr_block_matrix* x, const char* name, int64_t k) {
  if (!x) return fail(SR_ERR_ARGUMENT, "null argument");
  if (x->dtype != SR_E4M3 && x->dtype != SR_E5M2) return fail(SR_ERR_ARGUMENT, "%s must be E4M3 or E5M2", name);
  if (x->scale_type != SR_SCALE_E8M0 && x->scale_type != SR_SCALE_F32)
    return fail(SR_ERR_ARGUMENT, "%s: unknown scale type %d", name, x->scale_type);
  if (x->block_rows != 1 && x->block_rows != SR_BLOCK)
    return fail(SR_ERR_ARGUMENT, "%s: scales cover 1 or %d rows, not %d", name, SR_BLOCK, x->block_rows);
  if (x->rows < 0 || x->rows > kMaxRows) return fail(SR_ERR_ARGUMENT, "%s: %lld rows", name, (long long)x->rows);
  if (x->ld > kMaxLd || (x->rows > 1 && x->ld < k))
    return fail(SR_ERR_ARGUMENT, "%s: %lld bytes between rows of %lld", name, (long long)x->ld, (long long)k);
  if (x->ld_scale > kMaxScaleLd || x->ld_scale < 0)
    return fail(SR_ERR_ARGUMENT, "%s: %lld scales between rows", name, (long long)x->ld_scale);
  if (x->rows && k && (!x->data || !x->scale)) return fail(SR_ERR_ARGUMENT, "%s: null pointer", name);
  return SR_OK;
}

bool aligned_rows(const sr_block_matrix* x) {
  return reinterpret_cast<uintptr_t>(x->data) % 16 == 0 && x->ld % 16 == 0;
}

}  // namespace

extern "C" {

int sr_matrix_abi_version(void) { return SR_MATRIX_ABI_VERSION; }

int sr_block_cast(const void* x, int64_t ldx, int64_t rows, int64_t cols, int x_dtype, int dtype, int rule, int square,
                  uint32_t seed, uint32_t offset, const sr_block_output* by_rows, const sr_block_output* by_cols,
                  void* stream) {
  if (x_dtype != SR_F32 && x_dtype != SR_BF16 && x_dtype != SR_F16)
    return fail(SR_ERR_ARGUMENT, "block casts take FP32, BF16 or FP16, not dtype %d", x_dtype);
  if (dtype != SR_E4M3 && dtype != SR_E5M2) return fail(SR_ERR_ARGUMENT, "block casts give E4M3 or E5M2, not dtype %d", dtype);
  if (rule != SR_NEAREST && rule != SR_STOCHASTIC) return fail(SR_ERR_ARGUMENT, "unknown rounding rule %d", rule);
  if (rows < 0 || cols < 0 || rows > kMaxRows || cols > kMaxRows) return fail(SR_ERR_ARGUMENT, "%lld x %lld matrix", (long long)rows, (long long)cols);
  sr_block_output none{};
  sr::BlockCastArgs a{};
  a.by_rows = by_rows ? *by_rows : none;
  a.by_cols = by_cols ? *by_cols : none;
  if (!a.by_rows.data && !a.by_cols.data) return fail(SR_ERR_ARGUMENT, "no output");
  if (rows == 0 || cols == 0) return SR_OK;
  if (!x || (a.by_rows.data && !a.by_rows.scale) || (a.by_cols.data && !a.by_cols.scale))
    return fail(SR_ERR_ARGUMENT, "null pointer");
  if ((rows > 1 && ldx < cols) || (a.by_rows.data && a.by_rows.ld < cols) || (a.by_cols.data && a.by_cols.ld < rows))
    return fail(SR_ERR_ARGUMENT, "rows overlap");
  a.x = static_cast<const char*>(x);
  a.ldx = ldx;
  a.rows = rows;
  a.cols = cols;
  a.counter_base = seed + offset;
  a.tiles_n = static_cast<uint32_t>(blocks(cols));
  const uint64_t tiles = static_cast<uint64_t>(blocks(rows)) * a.tiles_n;
  const bool rows_too = a.by_rows.data, cols_too = a.by_cols.data;
  const sr::BlockCastKind kind = square ? sr::kCastSquare : (rows_too && cols_too && tiles >= sr::kWholeTiles ? sr::kCastWhole : sr::kCastParts);
  const void* fn = casts()[x_dtype == SR_F32 ? 0 : (x_dtype == SR_BF16 ? 1 : 2)][2 * (dtype == SR_E5M2) + (rule == SR_STOCHASTIC)][kind];
  const uint64_t groups = tiles * (kind == sr::kCastParts ? sr::kRowParts * rows_too + sr::kColParts * cols_too : 1);
  if (groups > 0xFFFFFFFFu) return fail(SR_ERR_ARGUMENT, "%lld x %lld matrix", (long long)rows, (long long)cols);
  constexpr uint64_t kLaunch = 0x7FFFFF / 2;  // a launch has fewer than 2^32 threads
  for (uint64_t first = 0; first < groups; first += kLaunch) {
    a.first = static_cast<uint32_t>(first);
    if (int rc = launch(fn, std::min(kLaunch, groups - first), kind == sr::kCastParts ? sr::kPartThreads : sr::kTileThreads, &a, stream)) return rc;
  }
  return SR_OK;
}

int sr_block_matmul(const sr_block_matrix* a, const sr_block_matrix* b, int64_t k, void* out, int64_t ldo,
                    int out_dtype, void* stream) {
  if (k < 0 || k > kMaxLd) return fail(SR_ERR_ARGUMENT, "%lld contracted values", (long long)k);
  if (int rc = check_matrix(a, "a", k)) return rc;
  if (int rc = check_matrix(b, "b", k)) return rc;
  if (a->scale_type != b->scale_type) return fail(SR_ERR_ARGUMENT, "a and b have different scale types");
  if (out_dtype != SR_F32 && out_dtype != SR_BF16 && out_dtype != SR_F16)
    return fail(SR_ERR_ARGUMENT, "products are FP32, BF16 or FP16, not dtype %d", out_dtype);
  if (a->rows == 0 || b->rows == 0) return SR_OK;
  if (!out) return fail(SR_ERR_ARGUMENT, "null pointer");
  if (a->rows > 1 && ldo < b->rows) return fail(SR_ERR_ARGUMENT, "rows of the result overlap");
  sr::BlockProductArgs g{};
  g.a = {static_cast<const char*>(a->data), a->ld, static_cast<int>(a->rows)};
  g.b = {static_cast<const char*>(b->data), b->ld, static_cast<int>(b->rows)};
  g.scale_a = static_cast<const char*>(a->scale);
  g.scale_b = static_cast<const char*>(b->scale);
  g.ld_scale_a = a->ld_scale;
  g.ld_scale_b = b->ld_scale;
  g.shift_a = a->block_rows == 1 ? 0 : 7;
  g.shift_b = b->block_rows == 1 ? 0 : 7;
  g.k = k;
  g.out = static_cast<char*>(out);
  g.ldo = ldo;
  g.m = static_cast<int>(a->rows);
  g.n = static_cast<int>(b->rows);
  g.out_dtype = out_dtype;
  g.scale_f32 = a->scale_type == SR_SCALE_F32;
  const int mode = out_dtype == SR_F32 ? sr::kWide : (g.scale_f32 ? sr::kFactors : sr::kExponents);
  const sr::BlockProductKernels& fn = products()[a->dtype == SR_E5M2][b->dtype == SR_E5M2][mode];
  if (g.m <= 16) {
    g.tiles_m = 1;
    g.tiles_n = (g.n + 15) / 16;
    return launch(fn.rows, g.tiles_n, 64 * sr::kRowWaves, &g, stream);
  }
  auto tiles = [&](int64_t side) { return ((g.m + side - 1) / side) * ((g.n + side - 1) / side); };
  const bool async = aligned_rows(a) && aligned_rows(b);
  auto launch_tiles = [&](const void* kernel, auto shape) {
    using S = decltype(shape);
    g.tiles_m = (g.m + S::BM - 1) / S::BM;
    g.tiles_n = (g.n + S::BN - 1) / S::BN;
    return launch(kernel, static_cast<uint64_t>(g.tiles_m) * g.tiles_n, S::kThreads, &g, stream);
  };
  const sr::BlockTile tile = sr::tile_by_count(tiles);
  switch (async || tile == sr::kTile128 ? tile : sr::kTile64) {
    case sr::kTile128: return launch_tiles(fn.tile[sr::kTile128][async], sr::Tile128{});
    case sr::kTile64x2: return launch_tiles(fn.tile[sr::kTile64x2][1], sr::Tile64x2{});
    case sr::kTile64x4: return launch_tiles(fn.tile[sr::kTile64x4][1], sr::Tile64x4{});
    default: return launch_tiles(fn.tile[sr::kTile64][async], sr::Tile64{});
  }
}

}  // extern "C"
