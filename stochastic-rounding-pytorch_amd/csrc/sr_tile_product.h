// sr_tile_product.h -- tiles of A * B^T on gfx950's matrix cores.
//
// Both operands hold their contracted axis contiguously, so an operand row is
// a run of bytes: FP8 (one per byte) or FP16 (two bytes each).  A workgroup
// computes a BM x BN tile and walks the contracted axis in stages of 128
// bytes: 128 FP8 values, which is one block of the block scales, or 64 FP16
// values.  A stage of both operands lies in LDS, (BM + BN) rows of eight
// 16-byte chunks; two stages alternate, so that the loads of one run under
// the products of the other with one barrier per stage.
//
// LDS layout.  Chunk c of row r lies at position c ^ (r % 8) of its row.  A
// fragment read takes one chunk of each of 16 consecutive rows, and the
// swizzle spreads these over all banks; unswizzled rows are 128 bytes apart,
// and all of them would meet in the same four banks.
//
// Fragments.  Lane l of a wave holds row l % 16 and chunks l / 16 and
// l / 16 + 4 of it.  For FP16 (16x16x32 products) these are two operands, for
// FP8 (16x16x128) the two halves of one.  Which values of the contracted axis
// share a lane does not matter as long as both operands agree.
//
// The second operand's rows are handed to the instruction as its first
// argument: lane l then holds, of each 16x16 tile of the result, row l % 16
// of A and the four consecutive rows 4 (l / 16) .. + 3 of B, which are
// neighbours in a row-major result.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace sr {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
// A 16-byte chunk at any byte address: gfx950's global loads take any alignment.
typedef int chunk_any __attribute__((ext_vector_type(4), aligned(1)));

constexpr int kStageBytes = 128;  // of each operand row
constexpr int kChunk = 16;

// BM x BN results by WM x WN waves.
template <int BM_, int BN_, int WM_, int WN_>
struct TileShape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int kRowsM = BM / WM, kRowsN = BN / WN;      // of one wave
  static constexpr int MI = kRowsM / 16, NI = kRowsN / 16;      // its 16x16 tiles
  static constexpr int kStage = (BM + BN) * kStageBytes;        // bytes of one LDS stage
  static constexpr int kLoads = (BM + BN) / 8 / kWaves;         // chunks a lane stages
  static_assert(BM % 8 == 0 && ((BM + BN) / 8) % kWaves == 0 && kRowsM % 16 == 0 && kRowsN % 16 == 0, "tile shape");
};

// One operand: `rows` rows of `bytes` bytes, `ld` bytes apart.
struct Operand {
  const char* base;
  int64_t ld;
  int rows;
};

// Waits for this wave's loads into LDS and its LDS accesses, then for the
// workgroup's other waves.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The tiles of a grid are numbered so that each XCD, which gets every eighth
// workgroup, works on a contiguous run of them (its own L2 then holds the
// rows that neighbouring tiles share).
__device__ __forceinline__ uint32_t xcd_run(uint32_t id, uint32_t total) {
  const uint32_t xcd = id & 7u, slot = id >> 3, each = total >> 3, extra = total & 7u;
  return xcd * each + (xcd < extra ? xcd : extra) + slot;
}

// Tile (row, column) of run position `id`: bands of up to 8 tile rows, down
// the columns of a band, so that the tiles in flight on an XCD share both
// operands' rows.
__device__ __forceinline__ void band_tile(uint32_t id, uint32_t tm, uint32_t tn, uint32_t& row, uint32_t& col) {
  constexpr uint32_t kBand = 8;
  const uint32_t band = id / (kBand * tn), first = band * kBand;
  const uint32_t height = tm - first < kBand ? tm - first : kBand;
  const uint32_t within = id - first * tn;
  row = first + within % height;
  col = within / height;
}

// The lower triangle's tile of index id: row >= col, counted row by row.
__device__ __forceinline__ void triangle_tile(uint32_t id, uint32_t& row, uint32_t& col) {
  uint32_t r = static_cast<uint32_t>((sqrtf(8.0f * static_cast<float>(id) + 1.0f) - 1.0f) * 0.5f);
  while (r * (r + 1) / 2 > id) --r;
  while ((r + 1) * (r + 2) / 2 <= id) ++r;
  row = r;
  col = id - r * (r + 1) / 2;
}

// The 16 bytes at `at` of a row that ends at `end`; zeros from there on.
__device__ __forceinline__ i32x4 load_chunk(const char* row, int64_t at, int64_t end) {
  if (at + kChunk <= end) {
    const chunk_any v = *(const __attribute__((address_space(1))) chunk_any*)(row + at);
    return i32x4{v[0], v[1], v[2], v[3]};
  }
  uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < kChunk; ++j)
    if (at + j < end)
      words[j >> 2] |= static_cast<uint32_t>(*(const __attribute__((address_space(1))) uint8_t*)(row + at + j)) << (8 * (j & 3));
  return i32x4{(int)words[0], (int)words[1], (int)words[2], (int)words[3]};
}

// Stages of both operands' rows for one workgroup.
template <class S>
struct Stager {
  const char* a;  // this workgroup's first row of either operand
  const char* b;
  int64_t lda, ldb;
  int rows_a, rows_b;  // valid rows from there (at least 1)
  uint32_t offset[S::kLoads];  // this lane's chunk in each of its loads, from a or b

  // `wave` is uniform.  Rows past the operand's end repeat its last row: the
  // results they give are not stored.
  __device__ void init(const Operand& opa, const Operand& opb, int row_a, int row_b, int wave, int lane) {
    lda = opa.ld;
    ldb = opb.ld;
    a = opa.base + row_a * lda;
    b = opb.base + row_b * ldb;
    rows_a = opa.rows - row_a;
    rows_b = opb.rows - row_b;
    const uint32_t chunk = static_cast<uint32_t>((lane & 7) ^ (lane >> 3)) * kChunk;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int r = (i * S::kWaves + wave) * 8 + (lane >> 3);
      const bool of_a = r < S::BM;
      const int valid = of_a ? rows_a : rows_b, at = of_a ? r : r - S::BM;
      offset[i] = static_cast<uint32_t>(at < valid ? at : valid - 1) * static_cast<uint32_t>(of_a ? lda : ldb) + chunk;
    }
  }

  // Asynchronous loads of the stage whose bytes start at k, straight into LDS.
  // Every row has 128 bytes from k, 16-byte aligned.
  __device__ void load_async(char* stage, int64_t k, int wave) const {
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int r0 = (i * S::kWaves + wave) * 8;  // uniform; a load's rows are of one operand
      const char* base = (r0 < S::BM ? a : b) + k;
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(base + offset[i]),
          (__attribute__((address_space(3))) void*)(stage + r0 * kStageBytes), kChunk, 0, 0);
    }
  }

  // The same stage through registers, for rows of any alignment and for a
  // stage that ends inside its 128 bytes: bytes from `end` on become zero.
  __device__ void load(i32x4 (&regs)[S::kLoads], int64_t k, int64_t end, int wave, int lane) const {
    const int64_t chunk = ((lane & 7) ^ (lane >> 3)) * kChunk;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const char* row = ((i * S::kWaves + wave) * 8 < S::BM ? a : b) + (offset[i] - chunk);
      regs[i] = load_chunk(row, k + chunk, end);
    }
  }

  __device__ static void store(char* stage, const i32x4 (&regs)[S::kLoads], int wave, int lane) {
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i)
      *reinterpret_cast<i32x4*>(stage + (i * S::kWaves + wave) * 8 * kStageBytes + lane * kChunk) = regs[i];
  }
};

// Byte offset of this lane's first chunk in a 16-row fragment; the second
// one's differs in bit 6.
__device__ __forceinline__ uint32_t fragment_offset(int lane) {
  return static_cast<uint32_t>((lane & 15) * kStageBytes + (((lane >> 4) ^ (lane & 7)) * kChunk));
}

__device__ __forceinline__ i32x4 read_chunk(const char* p) { return *reinterpret_cast<const i32x4*>(p); }

}  // namespace sr
