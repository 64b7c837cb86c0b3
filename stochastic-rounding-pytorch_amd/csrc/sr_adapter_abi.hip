// sr_adapter_abi.hip -- extern "C" entry points of the adapters (sr_matrix_hip.h).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/sr_matrix_hip.h"
#include "sr_adapter.h"
#include "sr_adapter_tables.h"
#include "sr_matrix_launch.h"

namespace {

using sr::fail;
using sr::launch;

constexpr int kMaxRank = 128;
constexpr int64_t kMaxSide = 1 << 24;        // k and n
constexpr int64_t kPartialBytes = 256 << 20;  // of the gradients' partial sums, at most

const sr::AdapterKernels& kernels(int dtype) {
  static const struct Tables {
    sr::AdapterTable t{};
    Tables() {
      sr::register_adapters_f32(t[SR_F32]);
      sr::register_adapters_bf16(t[SR_BF16]);
      sr::register_adapters_f16(t[SR_F16]);
    }
  } tables;
  return tables.t[dtype];
}

int64_t element(int dtype) { return dtype == SR_F32 ? 4 : 2; }
int chunks_of(int rank) { return (rank + sr::kRankChunk - 1) / sr::kRankChunk; }
int rank_index(int chunks) { return chunks <= 1 ? 0 : (chunks <= 2 ? 1 : (chunks <= 4 ? 2 : 3)); }

bool shape_is_good(int64_t rows, int64_t k, int64_t n, int64_t count, int64_t rank, int dtype) {
  return rows >= 0 && rows <= sr::kMaxRows && k >= 0 && k <= kMaxSide && n >= 0 && n <= kMaxSide && count >= 0 &&
         count <= SR_MATRIX_ADAPTERS && rank >= 1 && rank <= kMaxRank && (dtype == SR_F32 || dtype == SR_BF16 || dtype == SR_F16);
}

// Parts of the contracted axis: so many that few rows give every CU work, at least a step for each wave.
int splits_of(int64_t rows, int64_t k, int dtype) {
  const int64_t tiles = (rows + 15) / 16, steps = (k + kernels(dtype).step - 1) / kernels(dtype).step;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({8, 256 / std::max<int64_t>(tiles, 1), steps / sr::kShrinkWaves})));
}

int64_t low_values(int64_t rows, int64_t k, int rank, int dtype) {
  return splits_of(rows, k, dtype) * rows * chunks_of(rank) * sr::kRankChunk;
}

int check(const sr_adapters* g, int64_t rows, int64_t k, int64_t n) {
  if (!g) return fail(SR_ERR_ARGUMENT, "null argument");
  if (g->dtype != SR_F32 && g->dtype != SR_BF16 && g->dtype != SR_F16)
    return fail(SR_ERR_ARGUMENT, "adapters are FP32, BF16 or FP16, not dtype %d", g->dtype);
  if (g->rank < 1 || g->rank > kMaxRank) return fail(SR_ERR_ARGUMENT, "rank %d: 1 to %d", g->rank, kMaxRank);
  if (!shape_is_good(rows, k, n, g->count, g->rank, g->dtype))
    return fail(SR_ERR_ARGUMENT, "%lld rows, %lld to %lld by %d adapters", (long long)rows, (long long)k, (long long)n, g->count);
  if (rows && (!g->index || (g->count && ((k && !g->a) || (n && !g->b))))) return fail(SR_ERR_ARGUMENT, "null pointer");
  return SR_OK;
}

sr::Adapters adapters_of(const sr_adapters* g, const void* matrices, int64_t rows) {
  sr::Adapters a{};
  a.a = static_cast<const char*>(matrices);
  a.index = g->index;
  a.scaling = g->scaling;
  a.scale = g->scale;
  a.count = g->count;
  a.rank = g->rank;
  a.chunks = chunks_of(g->rank);
  a.wide = g->wide != 0;
  a.rows = rows;
  return a;
}

// Workgroups, or waves, that share the adapters of 16 rows, as a power of two: more of them where there are few otherwise.
int slot_bits_of(int64_t others, int count) {
  const int64_t wanted = std::min<int64_t>(256 / std::max<int64_t>(others, 1), count);
  return wanted >= 4 ? 2 : (wanted >= 2 ? 1 : 0);
}

sr::ShrinkArgs shrink_args(const sr_adapters* g, const void* matrices, const void* x, int64_t ldx, int64_t k, int64_t rows, float* low) {
  sr::ShrinkArgs s{};
  s.g = adapters_of(g, matrices, rows);
  s.x = static_cast<const char*>(x);
  s.ldx = ldx;
  s.k = k;
  s.low = low;
  s.row_tiles = static_cast<int>((rows + 15) / 16);
  s.splits = splits_of(rows, k, g->dtype);
  s.slot_bits = slot_bits_of(static_cast<int64_t>(s.row_tiles) * s.splits, g->count);
  return s;
}

sr::ExpandArgs expand_args(const sr_adapters* g, const void* matrices, const float* low, int splits, const void* base, int64_t ldbase,
                           int64_t n, int64_t rows, void* out, int64_t ldo) {
  sr::ExpandArgs s{};
  s.g = adapters_of(g, matrices, rows);
  s.low = low;
  s.base = static_cast<const char*>(base);
  s.out = static_cast<char*>(out);
  s.ldbase = ldbase;
  s.ldout = ldo;
  s.n = n;
  s.splits = splits;
  return s;
}

// low = the scaled products of x with `matrices` (count x rank x k).
int shrink(const sr_adapters* g, const sr::ShrinkArgs& args, void* stream) {
  sr::ShrinkArgs s = args;
  return launch(kernels(g->dtype).shrink[rank_index(s.g.chunks)], (static_cast<uint64_t>(s.row_tiles) * s.splits) << s.slot_bits,
                64 * sr::kShrinkWaves, &s, stream);
}

// out = base + low by `matrices` (count x n x rank), transposed.
int expand(const sr_adapters* g, const sr::ExpandArgs& args, void* stream) {
  sr::ExpandArgs s = args;
  const int64_t row_tiles = (s.g.rows + 15) / 16, waves = row_tiles * ((s.n + 63) / 64);
  // 64 columns a wave where they give every CU eight waves; 16 and the adapters shared out below that (512 rows to 2048: 12.0
  // us and 12.4 in runs of an adapter, 1024 rows 12.4 and 19.5, 256 rows 12.3 and 10.5).
  const bool wide = waves >= 2048;
  const int64_t groups = wide ? (row_tiles + sr::kExpandTiles - 1) / sr::kExpandTiles : row_tiles;
  s.slot_bits = wide ? 0 : slot_bits_of(1, g->count);
  s.column_tiles = static_cast<int>((s.n + (wide ? 63 : 15)) / (wide ? 64 : 16));
  s.blocks = ((s.column_tiles << s.slot_bits) + sr::kAdapterWaves - 1) / sr::kAdapterWaves;
  return launch(kernels(g->dtype).expand[rank_index(s.g.chunks)][wide], static_cast<uint64_t>(groups) * s.blocks, sr::kAdapterThreads, &s,
                stream);
}

// The one and then the other.  (In one kernel, 16 rows a workgroup, all of b passes each of them: 8192 rows of 2048 to 8192
// took 114 us, and take 73 in two.)
int shrink_and_expand(const sr_adapters* g, const sr::ShrinkArgs& down, const sr::ExpandArgs& up, void* stream) {
  // Bytes of the adapters' a that every workgroup of the one launch would read by itself, a chunk of ranks at a time: one row of
  // 2048 to 2048 takes 7.8 us and 10.1, of 4096 8.5 and 10.2, two of 2048 8.9 and 9.5; one of 8192 12.7 and 10.3, four of 2048
  // 15.1 and 9.6.  More rows can meet more adapters, one after the other (eight rows of 512 12.0 us).
  if (down.g.rows <= 2 && up.n && down.g.rows * down.g.chunks * down.k * element(g->dtype) <= 8192) {
    sr::FewArgs s{down, up, down.splits};
    s.down.splits = 1;
    s.down.slot_bits = s.up.slot_bits = 0;
    constexpr int64_t kColumns = 16 * sr::kShrinkWaves;
    return launch(kernels(g->dtype).few[rank_index(s.down.g.chunks)], static_cast<uint64_t>((up.n + kColumns - 1) / kColumns),
                  64 * sr::kShrinkWaves, &s, stream);
  }
  if (int rc = shrink(g, down, stream)) return rc;
  return up.n ? expand(g, up, stream) : SR_OK;
}

// How the rows of a gradient are parted.
struct Parts {
  int64_t rows;
  int count;
};
Parts parts_of(int64_t rows, int64_t k, int64_t n, int count, int rank, int dtype) {
  const int columns = kernels(dtype).contract_columns[rank_index(chunks_of(rank))];
  const int64_t groups = std::max<int64_t>(1, count * ((k + columns - 1) / columns + (n + columns - 1) / columns));
  const int64_t bytes = std::max<int64_t>(1, int64_t{4} * count * chunks_of(rank) * sr::kRankChunk * (k + n));
  const int64_t lists = (rows + sr::kListRows - 1) / sr::kListRows;
  const int64_t wanted = std::max<int64_t>(1, std::min({lists, (1024 + groups - 1) / groups, kPartialBytes / bytes}));
  const int64_t each = std::max<int64_t>(1, (lists + wanted - 1) / wanted) * sr::kListRows;
  return {each, static_cast<int>(std::max<int64_t>(1, (rows + each - 1) / each))};
}

// Places in the workspace of the gradients.
struct Workspace {
  int64_t a_turned, b_turned, low, partial[2], filled, bytes;
};
Workspace workspace_of(int64_t rows, int64_t k, int64_t n, int count, int rank, int dtype) {
  Workspace w{};
  auto place = [&](int64_t bytes) {
    const int64_t at = w.bytes;
    w.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  const Parts parts = parts_of(rows, k, n, count, rank, dtype);
  const int64_t width = chunks_of(rank) * sr::kRankChunk;
  w.a_turned = place(count * rank * k * element(dtype));
  w.b_turned = place(count * rank * n * element(dtype));
  w.low = place(low_values(rows, n, rank, dtype) * 4);
  if (parts.count > 1) {
    w.partial[0] = place(parts.count * count * width * k * 4);
    w.partial[1] = place(parts.count * count * width * n * 4);
    w.filled = place(int64_t{4} * parts.count * count);
  }
  return w;
}

}  // namespace

extern "C" {

int64_t sr_adapter_low(int64_t rows, int64_t k, int64_t rank, int dtype) {
  return shape_is_good(rows, k, 0, 0, rank, dtype) ? low_values(rows, k, static_cast<int>(rank), dtype) : 0;
}

int64_t sr_adapter_workspace(int64_t rows, int64_t k, int64_t n, int64_t count, int64_t rank, int dtype) {
  if (!shape_is_good(rows, k, n, count, rank, dtype)) return 0;
  return workspace_of(rows, k, n, static_cast<int>(count), static_cast<int>(rank), dtype).bytes;
}

int sr_adapter_add(const sr_adapters* g, const void* x, int64_t ldx, int64_t k, const void* base, int64_t ldbase, int64_t n,
                   int64_t rows, void* out, int64_t ldo, float* low, void* stream) {
  if (int rc = check(g, rows, k, n)) return rc;
  if (rows == 0) return SR_OK;
  if ((rows > 1 && (ldx < k || ldbase < n || ldo < n))) return fail(SR_ERR_ARGUMENT, "rows overlap");
  if ((k && !x) || (n && (!base || !out)) || !low) return fail(SR_ERR_ARGUMENT, "null pointer");
  return shrink_and_expand(g, shrink_args(g, g->a, x, ldx, k, rows, low),
                           expand_args(g, g->b, low, splits_of(rows, k, g->dtype), base, ldbase, n, rows, out, ldo), stream);
}

int sr_adapter_backward(const sr_adapters* g, const void* x, int64_t ldx, int64_t k, const void* dy, int64_t lddy, int64_t n,
                        int64_t rows, const float* low, void* dx, int64_t lddx, void* da, void* db, void* workspace, void* stream) {
  if (int rc = check(g, rows, k, n)) return rc;
  const bool want_x = dx && rows && k, want_a = da && g->count && k, want_b = db && g->count && n;
  if (!want_x && !want_a && !want_b) return SR_OK;
  if (rows > 1 && (ldx < k || lddy < n || (want_x && lddx < k))) return fail(SR_ERR_ARGUMENT, "rows overlap");
  if (!workspace || (rows && ((want_a && !x) || (n && !dy) || (want_b && !low)))) return fail(SR_ERR_ARGUMENT, "null pointer");
  const Workspace w = workspace_of(rows, k, n, g->count, g->rank, g->dtype);
  const sr::AdapterKernels& fn = kernels(g->dtype);
  char* work = static_cast<char*>(workspace);
  auto at = [&](int64_t place) { return reinterpret_cast<float*>(work + place); };
  const bool live = rows && g->count;  // rows can have adapters

  if (live && (want_x || want_a)) {
    sr::TurnArgs t{};
    if (int64_t{g->count} * ((n + 63) / 64 + (k + 63) / 64) * ((g->rank + 63) / 64) > 0x7FFFFF)
      return fail(SR_ERR_ARGUMENT, "%d adapters of %lld to %lld exceed a launch", g->count, (long long)k, (long long)n);
    auto turn = [&](const void* from, int64_t to, int64_t r, int64_t c) {
      const int64_t tiles_n = (c + 63) / 64;
      return sr::TurnOperand{static_cast<const char*>(from), work + to, r, c, static_cast<int>(tiles_n),
                             static_cast<uint32_t>(g->count * ((r + 63) / 64) * tiles_n)};
    };
    t.op[0] = turn(g->b, w.b_turned, n, g->rank);
    if (want_x) t.op[1] = turn(g->a, w.a_turned, g->rank, k);
    const uint64_t tiles = uint64_t{t.op[0].tiles} + t.op[1].tiles;
    if (tiles)
      if (int rc = launch(fn.turn, tiles, 256, &t, stream)) return rc;
  }
  const int splits = splits_of(rows, n, g->dtype);
  if (want_x || (live && want_a)) {
    const sr::ShrinkArgs down = shrink_args(g, work + w.b_turned, dy, lddy, n, rows, at(w.low));
    const sr::ExpandArgs up = expand_args(g, work + w.a_turned, at(w.low), splits, nullptr, 0, k, rows, dx, lddx);
    if (int rc = want_x ? shrink_and_expand(g, down, up, stream) : shrink(g, down, stream)) return rc;
  }
  if (!want_a && !want_b) return SR_OK;

  const Parts parts = parts_of(rows, k, n, g->count, g->rank, g->dtype);
  sr::ContractArgs c{};
  c.g = adapters_of(g, nullptr, rows);
  c.parts = parts.count;
  c.part_rows = parts.rows;
  c.filled = reinterpret_cast<int*>(work + w.filled);
  const int columns = fn.contract_columns[rank_index(c.g.chunks)];
  int used = 0;
  auto operand = [&](const float* values, int value_splits, const void* rows_of, int64_t ld, int64_t cols, void* out, int64_t partial, int turned) {
    c.op[used++] = {values, value_splits, static_cast<const char*>(rows_of), ld, cols, static_cast<char*>(out), at(partial), turned,
                    static_cast<int>((cols + columns - 1) / columns)};
  };
  if (want_a) operand(at(w.low), splits, x, ldx, k, da, w.partial[0], 0);
  if (want_b) operand(low, splits_of(rows, k, g->dtype), dy, lddy, n, db, w.partial[1], 1);
  const uint64_t groups = static_cast<uint64_t>(c.op[0].tiles + c.op[1].tiles) * g->count * parts.count;
  if (int rc = launch(fn.contract[rank_index(c.g.chunks)], groups, sr::kAdapterThreads, &c, stream)) return rc;
  if (parts.count == 1) return SR_OK;
  const int64_t items = sr::finish_items(c.g, c.op[0]) + sr::finish_items(c.g, c.op[1]);
  return launch(fn.finish, static_cast<uint64_t>((items + 255) / 256), 256, &c, stream);
}

}  // extern "C"
