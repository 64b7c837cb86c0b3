// sr_grouped.h -- block casts and products whose rows are sorted into groups, each with a matrix of its own.
//
// The groups' sizes are device memory, and no launch waits for them: a grid has
// room for any sizes, every wave sums them up by itself (64 groups a step), and
// workgroups beyond the tiles that there are end at once.  Sizes below zero
// count as zero and rows beyond the matrix as none, so that no sizes lead out of it.
#pragma once

#include <hip/hip_runtime.h>

#include "sr_block_scaled.h"

namespace sr {

struct Groups {
  const void* sizes;  // `count` numbers, int64 where `wide`, else int32
  int count;
  int wide;
};

__device__ __forceinline__ uint32_t group_size(const Groups& g, int i, uint32_t limit) {
  if (i >= g.count) return 0;
  if (g.wide) {
    const int64_t n = gptr<int64_t>(g.sizes)[i];
    return n < 0 ? 0u : (n < static_cast<int64_t>(limit) ? static_cast<uint32_t>(n) : limit);
  }
  const int32_t n = gptr<int32_t>(g.sizes)[i];
  return n < 0 ? 0u : umin(static_cast<uint32_t>(n), limit);
}

// min(the sum of x over this lane and those before it, limit); every x and the limit are below 2^31.
__device__ __forceinline__ uint32_t scan_capped(uint32_t x, uint32_t limit) {
#define SR_SCAN_STEP(control, rows) \
  x = umin(x + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), control, rows, 0xF, false)), limit)
  SR_SCAN_STEP(0x111, 0xF);  // 1, 2, 4 and 8 lanes back inside 16
  SR_SCAN_STEP(0x112, 0xF);
  SR_SCAN_STEP(0x114, 0xF);
  SR_SCAN_STEP(0x118, 0xF);
  SR_SCAN_STEP(0x142, 0xA);  // lane 15 to the next 16, lane 31 to the upper half
  SR_SCAN_STEP(0x143, 0xC);
#undef SR_SCAN_STEP
  return x;
}

__device__ __forceinline__ uint32_t lane_value(uint32_t x, int lane) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
}

// 64 groups, one a lane: their first row, rows, first tile and tiles of TILE rows, capped at `limit` rows in all.
// PADDED: a group's rows are rounded up to whole tiles before they are counted.
template <int TILE, bool PADDED>
struct GroupChunk {
  uint32_t start, rows, first, tiles;
  uint32_t rows_end, tiles_end;  // of the chunk, uniform

  __device__ __forceinline__ void load(const Groups& g, int chunk, uint32_t rows_before, uint32_t tiles_before, uint32_t limit) {
    const int lane = threadIdx.x & 63;
    uint32_t n = group_size(g, chunk + lane, limit);
    if (PADDED) n = umin((n + TILE - 1) / TILE * TILE, limit);
    const uint32_t end = umin(scan_capped(n, limit) + rows_before, limit);
    start = static_cast<uint32_t>(__shfl_up(static_cast<int>(end), 1));
    if (lane == 0) start = rows_before;
    rows = end - start;
    tiles = (rows + TILE - 1) / TILE;
    first = scan_capped(tiles, 0x7FFFFFFFu) + tiles_before;
    rows_end = lane_value(end, 63);
    tiles_end = lane_value(first, 63);
    first -= tiles;
  }
};

// A tile's group (the groups' count: rows behind the last one), uniform.
struct GroupTile {
  int group;
  uint32_t start, rows;   // the group's
  uint32_t first, tiles;  // its first tile among all and its tiles
};

// All groups' tiles of TILE rows.
template <int TILE>
struct GroupTable {
  GroupChunk<TILE, false> chunk;  // the first 64 groups
  uint32_t rows, tiles;           // of all groups

  __device__ __forceinline__ void load(const Groups& g, uint32_t limit) {
    chunk.load(g, 0, 0, 0, limit);
    rows = chunk.rows_end;
    tiles = chunk.tiles_end;
    for (int at = 64; at < g.count; at += 64) {
      GroupChunk<TILE, false> next;
      next.load(g, at, rows, tiles, limit);
      rows = next.rows_end;
      tiles = next.tiles_end;
    }
  }

  // The group of tile `tile`, counted over all groups and then over the rows behind them.
  __device__ __forceinline__ GroupTile find(const Groups& g, uint32_t tile, uint32_t limit) const {
    if (tile >= tiles) return {g.count, rows, limit - rows, tiles, (limit - rows + TILE - 1) / TILE};
    GroupChunk<TILE, false> c = chunk;
    int at = 0;
    while (c.tiles_end <= tile) {
      at += 64;
      c.load(g, at, c.rows_end, c.tiles_end, limit);
    }
    // The only lane with first <= tile < first + tiles.
    const int lane = __builtin_ctzll(__ballot(tile - c.first < c.tiles));
    return {at + lane, lane_value(c.start, lane), lane_value(c.rows, lane), lane_value(c.first, lane), lane_value(c.tiles, lane)};
  }
};

// The groups where every group's rows are padded to whole blocks.
struct PaddedGroups {
  int group;
  uint32_t start, rows;

  // Group number `number`, the largest ones first where a wave holds them all.
  __device__ __forceinline__ void find(const Groups& g, int number, uint32_t limit) {
    GroupChunk<SR_BLOCK, true> c;
    c.load(g, 0, 0, 0, limit);
    if (g.count <= 64) {
      const int lane = threadIdx.x & 63;
      int larger = 0;
      for (int j = 0; j < g.count; ++j) {
        const uint32_t other = lane_value(c.rows, j);
        larger += other > c.rows || (other == c.rows && j < lane);
      }
      group = __builtin_ctzll(__ballot(lane < g.count && larger == number));
    } else {
      group = number;
    }
    int at = 0;
    while (group >= at + 64) {
      at += 64;
      c.load(g, at, c.rows_end, 0, limit);
    }
    start = lane_value(c.start, group - at);
    rows = lane_value(c.rows, group - at);
  }
};

// ---------------------------------------------------------------------------
// Products.
//
//   rows      out[t] = a[t] b[g]^T for the rows t of group g, b a stack of matrices
//   contract  out[g] = a[:, g] b[:, g]^T over the columns of group g, which start
//             on multiples of 128 and end in zeros.  Every XCD takes an eighth of each
//             result, large groups first: their tiles cost as much as they have
//             rows, and with whole groups to an XCD the unluckiest one set the time
//             (16 groups of 60 to 2000 rows to 2048 x 2048: 99 us and 72)
//
// Both find their group and go on as a plain product does, on the part of the
// operands that the group has: what a plain product measured holds for them
// (sr_block_scaled.h).
// ---------------------------------------------------------------------------
struct GroupedProductArgs {
  BlockProductArgs p;  // m: all rows of a (rows), or of one result (contract)
  Groups groups;
  int64_t stride, stride_scale;  // rows: between matrices of b and of its scales, in bytes
  int64_t stride_out;            // contract: between results, in elements
  int zero_behind;               // rows: rows behind the last group become zeros
};

__device__ __forceinline__ int64_t output_bytes(const BlockProductArgs& p, int64_t elements) {
  return elements * (p.out_dtype == SR_F32 ? 4 : 2);
}

// The product of the group that tile `q` of TILE rows belongs to.
template <int TILE>
__device__ __forceinline__ BlockProductArgs rows_product(const GroupedProductArgs& g, const GroupTile& at) {
  BlockProductArgs p = g.p;
  p.a.base += at.start * p.a.ld;
  p.a.rows = p.m = static_cast<int>(at.rows);
  p.first_a = static_cast<int>(at.start);  // a group may start inside a block of 128 rows
  p.out += output_bytes(p, at.start * p.ldo);
  p.tiles_m = at.tiles;
  if (at.group == g.groups.count) {
    p.k = 0;  // nothing is read
  } else {
    p.b.base += at.group * g.stride;
    p.scale_b += at.group * g.stride_scale;
  }
  return p;
}

template <int MODE, int FA, int FB, class S, bool ASYNC>
__global__ __launch_bounds__(S::kThreads, kProductWaves<S>) void grouped_product_kernel(GroupedProductArgs g) {
  __shared__ __align__(1024) char lds[product_lds<MODE, S>() + 16];
  GroupTable<S::BM> table;
  const uint32_t limit = static_cast<uint32_t>(g.p.m);
  table.load(g.groups, limit);
  const uint32_t behind = g.zero_behind ? (limit - table.rows + S::BM - 1) / S::BM : 0;
  const uint32_t total = (table.tiles + behind) * g.p.tiles_n;
  if (blockIdx.x >= total) return;
  const uint32_t id = xcd_run(blockIdx.x, total);
  const GroupTile at = table.find(g.groups, id / g.p.tiles_n, limit);
  const BlockProductArgs p = rows_product<S::BM>(g, at);
  uint32_t tile_m, tile_n;
  band_tile(id - at.first * p.tiles_n, p.tiles_m, p.tiles_n, tile_m, tile_n);
  product_tile<MODE, FA, FB, S, ASYNC>(p, lds, tile_m * S::BM, tile_n * S::BN);
}

// Groups of few rows: tiles of 16 rows by 16 columns.
template <int MODE, int FA, int FB>
__global__ __launch_bounds__(64 * kRowWaves) void grouped_product_rows_kernel(GroupedProductArgs g) {
  __shared__ f32x4 sums[kRowWaves][64];
  GroupTable<16> table;
  const uint32_t limit = static_cast<uint32_t>(g.p.m);
  table.load(g.groups, limit);
  const uint32_t behind = g.zero_behind ? (limit - table.rows + 15) / 16 : 0;
  const uint32_t total = (table.tiles + behind) * g.p.tiles_n;
  if (blockIdx.x >= total) return;
  const uint32_t id = xcd_run(blockIdx.x, total);
  GroupTile at = table.find(g.groups, id / g.p.tiles_n, limit);
  const uint32_t within = id - at.first * g.p.tiles_n, tile_n = within / at.tiles, tile_m = within - tile_n * at.tiles;
  at.start += tile_m * 16;
  at.rows = umin(at.rows - tile_m * 16, 16);
  product_rows<MODE, FA, FB>(rows_product<16>(g, at), sums, static_cast<int>(tile_n) * 16);
}

// Workgroups of one result, an eighth of them on each XCD.
inline __host__ __device__ uint32_t contract_groups(uint32_t tiles) { return (tiles + 7) / 8 * 8; }

// The product of this workgroup's result and its tile in it; false where there is none.  `scales`: of a row, up to the
// matrix's end.
__device__ __forceinline__ bool contract_product(const GroupedProductArgs& g, BlockProductArgs& p, uint32_t& tile_m, uint32_t& tile_n,
                                                 int& scales) {
  p = g.p;
  const uint32_t tiles = p.tiles_m * p.tiles_n, each = contract_groups(tiles), number = blockIdx.x / each;
  const uint32_t id = xcd_run(blockIdx.x - number * each, each);
  if (id >= tiles) return false;
  PaddedGroups in;
  in.find(g.groups, static_cast<int>(number), static_cast<uint32_t>(p.k));
  const int64_t size = p.scale_f32 ? 4 : 1;
  scales = static_cast<int>((p.k - in.start) / SR_BLOCK);
  p.a.base += in.start;
  p.b.base += in.start;
  p.scale_a += in.start / SR_BLOCK * size;
  p.scale_b += in.start / SR_BLOCK * size;
  p.k = in.rows;
  p.out += output_bytes(p, in.group * g.stride_out);
  band_tile(id, p.tiles_m, p.tiles_n, tile_m, tile_n);
  return true;
}

template <int MODE, int FA, int FB, class S, bool ASYNC>
__global__ __launch_bounds__(S::kThreads, kProductWaves<S>) void grouped_contract_kernel(GroupedProductArgs g) {
  __shared__ __align__(1024) char lds[product_lds<MODE, S>() + 16];
  BlockProductArgs p;
  uint32_t tile_m, tile_n;
  int scales;
  if (!contract_product(g, p, tile_m, tile_n, scales)) return;
  product_tile<MODE, FA, FB, S, ASYNC>(p, lds, tile_m * S::BM, tile_n * S::BN, scales);
}

// ---------------------------------------------------------------------------
// The same products in 128 x 128 tiles with E8M0 scales, over whole blocks of the
// contracted axis.
//
// One stage in LDS, so that three workgroups share a CU: each waits for its loads,
// and what it spends outside its products (its group, its stages' way from
// memory, its results' way out) runs under the others'.  With two stages in LDS
// and two workgroups, a contraction of 16 groups of 512 rows to 2048 x 2048 took 85 us
// and takes 69 so, of 2048 rows 161 and 150; where a CU has one tile at a time it
// loses (one group of 8192 rows: 49 and 67).
// ---------------------------------------------------------------------------
// The chip holds 512 tiles of two workgroups a CU: where there are more of them, this one takes less time (rows of 16
// groups, 2048 x 2048: 624 tiles 28.5 us and 33.8, 1152 55.9 and 59.7, 4672 of 8192 x 2048 202 and 212; contractions of 640
// tiles 34 and 41), up to there more (416 tiles 23.6 and 21.0, contractions of 512 20.1 and 18.0).
constexpr int64_t kLeanTiles = 512;
constexpr int kLeanStages = 16;    // whose scales are in LDS at a time
constexpr int kLeanScaleRow = 20;  // bytes of a row of them: 32 rows' same bytes lie in different banks

template <int FA, int FB, bool CONTRACT>
__global__ __launch_bounds__(256, 3) void grouped_lean_kernel(GroupedProductArgs g) {
  using S = TileShape<128, 128, 2, 2>;
  __shared__ __align__(1024) char lds[S::kStage + (S::BM + S::BN) * kLeanScaleRow];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave_m = wave / S::WN * S::kRowsM, wave_n = wave % S::WN * S::kRowsN;

  // This workgroup's group and tile, and the scales that a row has in memory.
  BlockProductArgs p = g.p;
  uint32_t tile_m, tile_n;
  int scales;
  if constexpr (CONTRACT) {
    if (!contract_product(g, p, tile_m, tile_n, scales)) return;
  } else {
    GroupTable<S::BM> table;
    const uint32_t limit = static_cast<uint32_t>(p.m);
    table.load(g.groups, limit);
    const uint32_t total = (table.tiles + (g.zero_behind ? (limit - table.rows + S::BM - 1) / S::BM : 0)) * p.tiles_n;
    if (blockIdx.x >= total) return;
    const uint32_t id = xcd_run(blockIdx.x, total);
    const GroupTile in = table.find(g.groups, id / p.tiles_n, limit);
    p = rows_product<S::BM>(g, in);
    scales = static_cast<int>(p.k / SR_BLOCK);
    band_tile(id - in.first * p.tiles_n, p.tiles_m, p.tiles_n, tile_m, tile_n);
  }
  const int row0 = tile_m * S::BM, col0 = tile_n * S::BN, stages = static_cast<int>(p.k / SR_BLOCK);
  // Sixteen-row fragments of this wave that the group has.
  const int left = p.m - row0 - wave_m, live = left <= 0 ? 0 : (left >= S::kRowsM ? S::MI : (left + 15) / 16);

  Stager<S> stager;
  stager.init(p.a, p.b, row0, col0, wave, lane);
  // The scales of stages [first, first + kLeanStages), a row for each thread.
  char* marks = lds + S::kStage;
  auto fill = [&](int first) {
    const int r = threadIdx.x;
    const bool of_a = r < S::BM;
    const int row = of_a ? row0 + r : col0 + r - S::BM, rows = of_a ? p.m : p.n;
    const int row_at = (of_a ? p.first_a : 0) + (row < rows ? row : rows - 1);
    const char* from = (of_a ? p.scale_a : p.scale_b) +
                       (row_at >> (of_a ? p.shift_a : p.shift_b)) * (of_a ? p.ld_scale_a : p.ld_scale_b) + first;
    const int there = scales - first;
    char* to = marks + r * kLeanScaleRow;
    if (there >= kLeanStages) {
      const i32x4 v = load_whole_chunk(from, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) reinterpret_cast<int*>(to)[j] = v[j];
    } else {
#pragma unroll 1
      for (int j = 0; j < there; ++j) to[j] = static_cast<char>(gptr<uint8_t>(from)[j]);
    }
  };

  f32x4 acc[S::MI][S::NI] = {};
  const uint32_t fragment = fragment_offset(lane);
  if (stages) {
    stager.load_async(lds, 0, wave);
    fill(0);
  }
  for (int kt = 0; kt < stages; ++kt) {
    stage_barrier();
    if (live > 0) {
      Fragment<kExponents, FB> b[S::NI];
      Scales<kExponents, S::MI, S::NI> marked;
      const char* at = marks + kt % kLeanStages;
#pragma unroll
      for (int i = 0; i < S::MI; ++i)
        marked.a[i] = *reinterpret_cast<const uint8_t*>(at + (wave_m + 16 * i + (lane & 15)) * kLeanScaleRow);
#pragma unroll
      for (int i = 0; i < S::NI; ++i)
        marked.b[i][0] = *reinterpret_cast<const uint8_t*>(at + (S::BM + wave_n + 16 * i + (lane & 15)) * kLeanScaleRow);
      const char* sa = lds + wave_m * kStageBytes;
      const char* sb = lds + (S::BM + wave_n) * kStageBytes;
#pragma unroll
      for (int i = 0; i < S::NI; ++i)
        b[i].set(read_chunk(sb + fragment + i * 16 * kStageBytes), read_chunk(sb + (fragment ^ 64) + i * 16 * kStageBytes));
      auto row = [&](int mi) {
        Fragment<kExponents, FA> a;
        a.set(read_chunk(sa + fragment + mi * 16 * kStageBytes), read_chunk(sa + (fragment ^ 64) + mi * 16 * kStageBytes));
#pragma unroll
        for (int ni = 0; ni < S::NI; ++ni) block_mma<false>(acc[mi][ni], a, b[ni], marked, mi, ni);
      };
#pragma unroll
      for (int mi = 0; mi < S::MI; ++mi) row(mi);
    }
    lds_barrier();  // every wave is done with the stage
    if (kt + 1 < stages) {
      stager.load_async(lds, (kt + 1) * kStageBytes, wave);
      if ((kt + 1) % kLeanStages == 0) fill(kt + 1);
    }
  }

  // The results pass the stage's LDS, 32 rows of a wave at a time: four values of a row at place (place ^ row) of its
  // sixteen, so that neither side's accesses meet in the same banks.
  char* turned = lds + wave * (S::kStage / 4);
  auto place = [&](int row, int four) { return reinterpret_cast<f32x4*>(turned + row * 256 + ((four ^ row) & 15) * 16); };
  with_output(p, row0, col0, S::BM, S::BN, [&](auto out, auto edge) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half * 2 >= live) break;
#pragma unroll
      for (int mi = 0; mi < 2; ++mi)
#pragma unroll
        for (int ni = 0; ni < S::NI; ++ni) *place(16 * mi + (lane & 15), 4 * ni + (lane >> 4)) = acc[2 * half + mi][ni];
      constexpr int kOut = decltype(out)::value;
      if constexpr (kOut != SR_F32 && !decltype(edge)::value) {
        // Eight values a lane, eight lanes a row.  The result is not read again here: its stores pass the caches by.
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = 8 * k + (lane >> 3);
          uint32_t w[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const f32x4 v = *place(row, 2 * (lane & 7) + h);
            const float x[4] = {v[0], v[1], v[2], v[3]};
            uint32_t pair[2];
            encode_group<kOut == SR_BF16 ? ENC_BF16_RN : ENC_F16_RN>(x, 0u, pair);
            w[2 * h] = pair[0];
            w[2 * h + 1] = pair[1];
          }
          uint16_t* to = reinterpret_cast<uint16_t*>(p.out) + (row0 + wave_m + 32 * half + row) * p.ldo + col0 + wave_n + 8 * (lane & 7);
          __builtin_nontemporal_store(eight_halves{w[0], w[1], w[2], w[3]}, (SR_GLOBAL eight_halves*)(to));
        }
        continue;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int row = 4 * k + (lane >> 4);
        store_results<kOut, decltype(edge)::value>(p, row0 + wave_m + 32 * half + row, col0 + wave_n + 4 * (lane & 15), *place(row, lane & 15));
      }
    }
  });
}

// ---------------------------------------------------------------------------
// Casts.
//
// A group's blocks along the rows start at its first row, and its transposed
// columns at a multiple of 128, zeros up to the next: a contraction over them
// then has whole blocks of its own group only.  Tiles of 128 rows of a group do
// both orientations; rows behind the last group are cast along the columns
// alone.
//
// A stack of matrices is cast matrix by matrix in one launch.
// ---------------------------------------------------------------------------
struct GroupedCastArgs {
  BlockCastArgs c;
  Groups groups;
  uint32_t column_blocks;  // of the transposed result
};

// The part of a cast that a group's rows are; `block`: its first block of transposed columns.
__device__ __forceinline__ BlockCastArgs cast_of_group(const BlockCastArgs& c, const GroupTile& at, int element_bytes) {
  BlockCastArgs p = c;
  p.x += static_cast<int64_t>(at.start) * c.ldx * element_bytes;
  p.rows = at.rows;
  p.counter_base += at.start * static_cast<uint32_t>(c.cols);
  if (p.by_rows.data) {
    p.by_rows.data = static_cast<char*>(p.by_rows.data) + at.start * c.by_rows.ld;
    p.by_rows.scale = static_cast<char*>(p.by_rows.scale) + at.start * c.by_rows.ld_scale;
  }
  p.by_cols.data = static_cast<char*>(p.by_cols.data) + static_cast<int64_t>(at.first) * SR_BLOCK;
  p.by_cols.scale = static_cast<char*>(p.by_cols.scale) + at.first;
  return p;
}

// Zeros in block `block` of the transposed columns, for `cols` columns from col0 on.
__device__ __forceinline__ void zero_columns(const BlockCastArgs& c, uint32_t block, int64_t col0, int cols, int threads) {
  for (int i = threadIdx.x; i < cols * 16; i += threads) {
    const int64_t col = col0 + (i >> 4);
    if (col >= c.cols) break;
    char* q = static_cast<char*>(c.by_cols.data) + col * c.by_cols.ld + static_cast<int64_t>(block) * SR_BLOCK + (i & 15) * 8;
    *(SR_GLOBAL eight_bytes*)(q) = eight_bytes{0, 0};
    if ((i & 15) == 0) store_exponent(c.by_cols, col, block, 0);
  }
}

template <int XE, int QE>
__global__ __launch_bounds__(kTileThreads, 4) void grouped_cast_tile_kernel(GroupedCastArgs g) {
  GroupTable<kCastTile> table;
  const uint32_t limit = static_cast<uint32_t>(g.c.rows);
  table.load(g.groups, limit);
  const uint32_t id = g.c.first + blockIdx.x, tile = id / g.c.tiles_n;
  const int64_t col0 = static_cast<int64_t>(id - tile * g.c.tiles_n) * kCastTile;
  if (tile >= table.tiles && tile < g.column_blocks) zero_columns(g.c, tile, col0, kCastTile, kTileThreads);
  const GroupTile at = table.find(g.groups, tile, limit);
  const uint32_t within = tile - at.first;
  if (within >= at.tiles) return;  // behind the rows behind the last group
  if (at.group == g.groups.count) {
    // Rows behind the last group have no place in the transposed result.
    for (int part = 0; part < kCastTile; part += kTileThreads / 16)
      cast_row_part<XE, QE>(g.c, static_cast<int64_t>(at.start) + within * kCastTile + part, col0 / kCastTile);
    return;
  }
  const BlockCastArgs p = cast_of_group(g.c, at, enc_bytes(XE));
  cast_tile<XE, QE, false, 16, true>(p, static_cast<int64_t>(within) * kCastTile, col0, true, true,
                               static_cast<int64_t>(within + 1) * kCastTile);
}

// Workgroups of one orientation each: first kColParts times tiles_n of every
// block of transposed columns, then, where the rows are asked for, those of all
// rows as they lie.
template <int XE, int QE>
__global__ __launch_bounds__(kPartThreads, enc_stochastic(QE) ? 5 : 6) void grouped_cast_parts_kernel(GroupedCastArgs g) {
  constexpr int kCols = 8 * kPartLanes;
  const uint32_t id = g.c.first + blockIdx.x, each = kColParts * g.c.tiles_n, tile = id / each;
  if (tile >= g.column_blocks) {
    const uint32_t row_id = id - each * g.column_blocks, part = row_id / g.c.tiles_n;
    cast_row_part<XE, QE>(g.c, static_cast<int64_t>(part) * kPartRows, row_id - part * g.c.tiles_n);
    return;
  }
  GroupTable<kCastTile> table;
  const uint32_t limit = static_cast<uint32_t>(g.c.rows);
  table.load(g.groups, limit);
  const int64_t col0 = static_cast<int64_t>(id - tile * each) * kCols;
  if (tile >= table.tiles) {
    zero_columns(g.c, tile, col0, kCols, kPartThreads);
    return;
  }
  const GroupTile at = table.find(g.groups, tile, limit);
  const uint32_t within = tile - at.first;
  const BlockCastArgs p = cast_of_group(g.c, at, enc_bytes(XE));
  cast_tile<XE, QE, false, kPartLanes, true>(p, static_cast<int64_t>(within) * kCastTile, col0, false, true,
                                       static_cast<int64_t>(within + 1) * kCastTile);
}

// A stack of matrices of `c`'s shape.
struct StackedCastArgs {
  BlockCastArgs c;
  int64_t stride_x;                                          // between matrices, in bytes
  int64_t rows_data, rows_scale, cols_data, cols_scale;      // of the results
  uint32_t each;                                             // workgroups of a matrix
};

__device__ __forceinline__ BlockCastArgs matrix_of_stack(const StackedCastArgs& s, uint32_t matrix) {
  BlockCastArgs p = s.c;
  p.x += matrix * s.stride_x;
  p.counter_base += matrix * static_cast<uint32_t>(s.c.rows) * static_cast<uint32_t>(s.c.cols);
  if (p.by_rows.data) {
    p.by_rows.data = static_cast<char*>(p.by_rows.data) + matrix * s.rows_data;
    p.by_rows.scale = static_cast<char*>(p.by_rows.scale) + matrix * s.rows_scale;
  }
  if (p.by_cols.data) {
    p.by_cols.data = static_cast<char*>(p.by_cols.data) + matrix * s.cols_data;
    p.by_cols.scale = static_cast<char*>(p.by_cols.scale) + matrix * s.cols_scale;
  }
  return p;
}

template <int XE, int QE, bool SQUARE>
__global__ __launch_bounds__(kTileThreads, SQUARE ? 6 : 4) void stacked_cast_tile_kernel(StackedCastArgs s) {
  const uint32_t id = s.c.first + blockIdx.x, matrix = id / s.each;
  cast_whole<XE, QE, SQUARE>(matrix_of_stack(s, matrix), id - matrix * s.each);
}

template <int XE, int QE>
__global__ __launch_bounds__(kPartThreads, enc_stochastic(QE) ? 5 : 6) void stacked_cast_parts_kernel(StackedCastArgs s) {
  const uint32_t id = s.c.first + blockIdx.x, matrix = id / s.each;
  cast_parts<XE, QE>(matrix_of_stack(s, matrix), id - matrix * s.each);
}

}  // namespace sr
