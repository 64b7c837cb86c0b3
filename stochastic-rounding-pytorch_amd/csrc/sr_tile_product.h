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
#include <type_traits>
#include <utility>

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

// BM x BN results by WM x WN waves; two stages in LDS.  With GROUPS > 1 so many
// such sets of waves take every GROUPS-th stage each, with stages of their own,
// and add their sums at the end: for launches with few tiles, whose time is
// the latency of one tile's walk.
template <int BM_, int BN_, int WM_, int WN_, int GROUPS_ = 1>
struct TileShape {
  static constexpr int kGroups = GROUPS_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kWaves = WM * WN;                         // of one group
  static constexpr int kThreads = 64 * kWaves * kGroups;
  static constexpr int kMinWaves = kThreads <= 512 ? 2 : (kWaves * kGroups + 3) / 4;  // of a SIMD, for its registers
  static constexpr int kRowsM = BM / WM, kRowsN = BN / WN;      // of one wave
  static constexpr int MI = kRowsM / 16, NI = kRowsN / 16;      // its 16x16 tiles
  static constexpr int kStage = (BM + BN) * kStageBytes;        // bytes of one LDS stage
  static constexpr int kLds = 2 * kStage * kGroups;             // all stages
  static constexpr int kSums = (kGroups - 1) * BM * BN * 4;     // the other groups' sums
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

// The same without waiting for loads, for what only LDS accesses must order.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Walks `stages` stages, a group every kGroups-th: load(stage, buffer) starts a
// stage's loads into one of the group's two buffers, use(stage, buffer) takes
// one that has landed for all its waves.  between(stage) runs on every wave
// before the stages from `stage` on (a multiple of kGroups), when every wave
// is done with those before.  Past the end a group loads the last stage
// again and uses nothing.
template <class S, class Load, class Between, class Use>
__device__ __forceinline__ void walk_stages(int stages, int group, Load&& load, Between&& between, Use&& use) {
  if (stages <= 0) return;
  auto start = [&](int kt, int buffer) { load(kt < stages ? kt : stages - 1, buffer); };
  start(group, 0);
  for (int base = 0, buffer = 0; base < stages; base += S::kGroups, buffer ^= 1) {
    stage_barrier();
    between(base);
    if (base + S::kGroups < stages) start(base + S::kGroups + group, buffer ^ 1);
    if (S::kGroups == 1 || base + group < stages) use(base + group, buffer);
  }
}

// Adds the groups' sums into group 0's, in the groups' order, through LDS that
// every wave is done with; only group 0 may go on to use acc, and after it the LDS.
template <class S>
__device__ __forceinline__ void add_groups(char* lds, int group, f32x4 (&acc)[S::MI][S::NI]) {
  if constexpr (S::kGroups > 1) {
    constexpr int kTiles = S::MI * S::NI, kThreadsOfGroup = S::kThreads / S::kGroups;
    const int t = threadIdx.x - group * kThreadsOfGroup;
    f32x4* sums = reinterpret_cast<f32x4*>(lds);
    if (group > 0) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) sums[((group - 1) * kTiles + i) * kThreadsOfGroup + t] = acc[i / S::NI][i % S::NI];
    }
    lds_barrier();
    if (group == 0) {
#pragma unroll
      for (int g = 0; g < S::kGroups - 1; ++g)
#pragma unroll
        for (int i = 0; i < kTiles; ++i) acc[i / S::NI][i % S::NI] += sums[(g * kTiles + i) * kThreadsOfGroup + t];
    }
    lds_barrier();
  }
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

// The lower triangle's tile of index id, counted row by row: row r has r + 1 tiles.
__device__ __forceinline__ void triangle_tile(uint32_t id, uint32_t& row, uint32_t& col) {
  uint32_t r = static_cast<uint32_t>((sqrtf(8.0f * static_cast<float>(id) + 1.0f) - 1.0f) * 0.5f);
  while (r * (r + 1) / 2 > id) --r;
  while ((r + 1) * (r + 2) / 2 <= id) ++r;
  row = r;
  col = id - r * (r + 1) / 2;
}

// The 16 bytes at `at` of a row, all inside it.
__device__ __forceinline__ i32x4 load_whole_chunk(const char* row, int64_t at) {
  const chunk_any v = *(const __attribute__((address_space(1))) chunk_any*)(row + at);
  return i32x4{v[0], v[1], v[2], v[3]};
}

// The 16 bytes at `at` of a row of `end` bytes (at least 1, the same for the
// wave); zeros from its end on.  Without a branch per lane, at whose end each
// load would wait for memory by itself: a chunk that passes the end is
// read where it still fits and shifted, and rows shorter than a chunk are read
// byte by byte at clamped places.
__device__ __forceinline__ i32x4 load_chunk(const char* row, int64_t at, int64_t end) {
  if (end >= kChunk) {
    const int64_t from = at < end - kChunk ? at : end - kChunk;
    const i32x4 v = load_whole_chunk(row, from);
    const int skip = at - from < kChunk ? static_cast<int>(at - from) : kChunk;  // bytes before the chunk
    const uint64_t lo = static_cast<uint32_t>(v[0]) | static_cast<uint64_t>(static_cast<uint32_t>(v[1])) << 32;
    const uint64_t hi = static_cast<uint32_t>(v[2]) | static_cast<uint64_t>(static_cast<uint32_t>(v[3])) << 32;
    const int bits = 8 * (skip & 7);
    // lo and hi shifted by less than a word, then by a word.
    const uint64_t low = (lo >> bits) | ((hi << 1) << (63 - bits)), high = hi >> bits;
    const uint64_t a = skip >= 16 ? 0 : (skip >= 8 ? high : low), b = skip >= 8 ? 0 : high;
    return i32x4{static_cast<int>(a), static_cast<int>(a >> 32), static_cast<int>(b), static_cast<int>(b >> 32)};
  }
  uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < kChunk; ++j) {
    const int64_t from = at + j < end ? at + j : end - 1;
    const uint32_t byte = *(const __attribute__((address_space(1))) uint8_t*)(row + from);
    words[j >> 2] |= (at + j < end ? byte : 0u) << (8 * (j & 3));
  }
  return i32x4{(int)words[0], (int)words[1], (int)words[2], (int)words[3]};
}

// A buffer over all that follows `base`: its loads take a 32-bit offset per
// lane and a uniform one, and need no address arithmetic.  (The host's pass
// over the kernels knows neither the type nor the builtins.)
#if defined(__HIP_DEVICE_COMPILE__)
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer_of(const char* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, -1, 0x00020000);
}
// 16 bytes of every lane to consecutive places of LDS from `to` on, which is uniform.
__device__ __forceinline__ void chunks_to_lds(Buffer from, char* to, uint32_t offset, uint32_t uniform) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, offset, uniform, 0, 0);
}
#else
typedef const char* Buffer;
__device__ inline Buffer buffer_of(const char* base) { return base; }
__device__ inline void chunks_to_lds(Buffer, char*, uint32_t, uint32_t) {}
#endif

// Stages of both operands' rows for one workgroup.
template <class S>
struct Stager {
  static constexpr int kLoadsA = S::BM / 8 / S::kWaves;  // the others are B's
  static_assert(S::BM / 8 % S::kWaves == 0, "a load's rows are of one operand");
  const char* a;  // this workgroup's first row of either operand
  const char* b;
  Buffer buffer_a, buffer_b;
  uint32_t offset[S::kLoads];  // this lane's chunk in each of its loads, from a or b

  // `wave` is uniform.  Rows past the operand's end repeat its last row: the
  // results they give are not stored.
  __device__ void init(const Operand& opa, const Operand& opb, int row_a, int row_b, int wave, int lane) {
    a = opa.base + row_a * opa.ld;
    b = opb.base + row_b * opb.ld;
    buffer_a = buffer_of(a);
    buffer_b = buffer_of(b);
    const uint32_t chunk = static_cast<uint32_t>((lane & 7) ^ (lane >> 3)) * kChunk;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const bool of_a = i < kLoadsA;
      const int at = ((of_a ? i : i - kLoadsA) * S::kWaves + wave) * 8 + (lane >> 3);
      const int valid = of_a ? opa.rows - row_a : opb.rows - row_b;
      offset[i] = static_cast<uint32_t>(at < valid ? at : valid - 1) * static_cast<uint32_t>(of_a ? opa.ld : opb.ld) + chunk;
    }
  }

  // Asynchronous loads of the stage whose bytes start at k, straight into LDS.
  // Every row has 128 bytes from k, 16-byte aligned.
  __device__ void load_async(char* stage, uint32_t k, int wave) const {
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i)
      chunks_to_lds(i < kLoadsA ? buffer_a : buffer_b, stage + (i * S::kWaves + wave) * 8 * kStageBytes, offset[i], k);
  }

  // The same stage through registers, for rows of any alignment and for a
  // stage that ends inside its 128 bytes: bytes from `end` on become zero.
  __device__ void load(i32x4 (&regs)[S::kLoads], int64_t k, int64_t end, int wave, int lane) const {
    const int64_t chunk = ((lane & 7) ^ (lane >> 3)) * kChunk;
    // Whole stages load without a branch per chunk: at its end a branch waits for its own load.
    if (k + kStageBytes <= end) {
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) regs[i] = load_whole_chunk((i < kLoadsA ? a : b) + offset[i], k);
    } else {
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) regs[i] = load_chunk((i < kLoadsA ? a : b) + (offset[i] - chunk), k + chunk, end);
    }
  }

  // The two together, chunk by chunk.
  __device__ void load_through(char* stage, int64_t k, int64_t end, int wave, int lane) const {
    const int64_t chunk = ((lane & 7) ^ (lane >> 3)) * kChunk;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i)
      *reinterpret_cast<i32x4*>(stage + (i * S::kWaves + wave) * 8 * kStageBytes + lane * kChunk) =
          load_chunk((i < kLoadsA ? a : b) + (offset[i] - chunk), k + chunk, end);
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

// ---------------------------------------------------------------------------
// FP16 products on 256 x 256 tiles by eight waves, for launches that fill the
// chip with them: what a CU reads per product is half of a 128 x 128 tile's.
//
// A wave computes 128 x 64 results as 4 x 2 tiles of 32 x 32.  Each stage is
// two halves of 64 bytes per row.  A half's fragments are read while the
// products of the half before run.  The one barrier per stage stands between
// the halves: by then every wave holds the second half in registers, so the
// buffer is free for the loads of two stages later, and the next stage has had
// a whole stage's time to arrive.
// ---------------------------------------------------------------------------
using TileWide = TileShape<256, 256, 2, 4>;
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct WideTile {
  static constexpr int MI = TileWide::kRowsM / 32, NI = TileWide::kRowsN / 32;

  // One wave's fragments of a half stage: two chunks of its row of each 32-row tile.
  struct Fragments {
    f16x8 a[MI][2], b[NI][2];
    // `a_at`, `b_at`: this lane's first chunk among the stage's bytes, for half 0.
    __device__ __forceinline__ void read(const char* stage, uint32_t a_at, uint32_t b_at, int half) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          b[i][j] = __builtin_bit_cast(f16x8, read_chunk(stage + (b_at ^ (64 * half + 32 * j)) + i * 32 * kStageBytes));
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          a[i][j] = __builtin_bit_cast(f16x8, read_chunk(stage + (a_at ^ (64 * half + 32 * j)) + i * 32 * kStageBytes));
    }
    __device__ __forceinline__ void multiply(f32x16 (&acc)[MI][NI]) const {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
          for (int ni = 0; ni < NI; ++ni)
            acc[mi][ni] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b[ni][j], a[mi][j], acc[mi][ni], 0, 0, 0);
    }
  };

  // Asks the scheduler to issue a half's LDS reads between the first three
  // quarters of the products that run meanwhile: left alone it gathers them at
  // the end, to reuse registers, and then waits for them.
  template <int I = 0>
  static __device__ __forceinline__ void interleave() {
    constexpr int kProducts = 2 * MI * NI, kReads = 2 * (MI + NI), kSlots = 3 * kProducts / 4;
    if constexpr (I == kProducts) {
      __builtin_amdgcn_sched_barrier(0);
    } else {
      constexpr int kNow = I < kSlots ? (I + 1) * kReads / kSlots - I * kReads / kSlots : 0;
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // one matrix instruction
      if constexpr (kNow > 0) __builtin_amdgcn_sched_group_barrier(0x100, kNow, 0);
      interleave<I + 1>();
    }
  }

  // acc += the products of `stages` whole stages (at least 1).  On return every wave is done with the LDS.
  static __device__ __forceinline__ void run(char* lds, const Stager<TileWide>& stager, int stages, int wave, int lane,
                                             f32x16 (&acc)[MI][NI]) {
    const uint32_t at = (lane & 31) * kStageBytes + (((lane >> 5) ^ (lane & 7)) * kChunk);
    const uint32_t at_a = wave / TileWide::WN * TileWide::kRowsM * kStageBytes + at;
    const uint32_t at_b = (TileWide::BM + wave % TileWide::WN * TileWide::kRowsN) * kStageBytes + at;
    auto load = [&](int kt) { stager.load_async(lds + (kt & 1) * TileWide::kStage, kt * kStageBytes, wave); };
    Fragments first, second;
    load(0);
    stage_barrier();
    if (stages > 1) load(1);
    first.read(lds, at_a, at_b, 0);
    auto step = [&](int kt, auto more) {
      second.read(lds + (kt & 1) * TileWide::kStage, at_a, at_b, 1);
      first.multiply(acc);
      interleave();
      stage_barrier();
      if constexpr (decltype(more)::value) load(kt + 2);
      // Past the last stage this reads what the buffer held two stages ago; nothing uses it.
      first.read(lds + (~kt & 1) * TileWide::kStage, at_a, at_b, 0);
      second.multiply(acc);
      interleave();
    };
    int kt = 0;
    for (; kt + 2 < stages; ++kt) step(kt, std::true_type{});
    for (; kt < stages; ++kt) step(kt, std::false_type{});
    stage_barrier();
  }
};

// ---------------------------------------------------------------------------
// Results on their way out.
//
// A matrix instruction leaves a lane four neighbours of one row, and the
// lanes beside it other rows: stored from there, every access would scatter
// over 16 or 32 rows, 8 to 32 bytes each.  So a wave passes 32 rows by CN
// columns at a time through LDS of its own and takes them up as blocks of
// 4 x 4, CN / 4 lanes to a row: a row's lanes then cover whole cache lines, and a
// block turns in registers where the transpose is stored as well.  The rows
// are padded so that neither side's accesses meet in the same banks.  Only
// one wave uses a chunk, so it needs no barrier.
// ---------------------------------------------------------------------------
template <int CN>
struct ResultChunk {
  static constexpr int kRows = 32, kStride = CN + 4, kTurnedStride = kRows + 4;
  static constexpr int kLanes = CN / 4, kBlocks = kRows * CN / 16 / 64;  // lanes of a row; blocks of a lane
  static constexpr int kBytes = kRows * kStride * 4;
  static constexpr int kTurnedLanes = kRows / 4;  // lanes of a turned row
  template <class T>
  static constexpr int turned_bytes() { return CN * kTurnedStride * static_cast<int>(sizeof(T)); }

  // Block `i` of this lane: rows block_row(i) .. + 3, columns block_col() .. + 3.
  static __device__ __forceinline__ int block_row(int i, int lane) { return 4 * (i * (64 / kLanes) + lane / kLanes); }
  static __device__ __forceinline__ int block_col(int lane) { return 4 * (lane % kLanes); }

  static __device__ __forceinline__ void put(float* chunk, int row, int col, const f32x4& v) {
    *reinterpret_cast<f32x4*>(chunk + row * kStride + col) = v;
  }
  static __device__ __forceinline__ f32x4 get(const float* chunk, int row, int col) {
    return *reinterpret_cast<const f32x4*>(chunk + row * kStride + col);
  }

  // The transpose: columns become rows of 32 values of T.
  template <class T, class T4>
  static __device__ __forceinline__ void put_turned(T* turned, int col, int row, const T4& v) {
    *reinterpret_cast<T4*>(turned + col * kTurnedStride + row) = v;
  }
  // Turned block `i` of this lane: four values of column turned_col(i) from row turned_row() on.
  static constexpr int kTurnedBlocks = CN * kTurnedLanes / 64;
  static __device__ __forceinline__ int turned_col(int i, int lane) { return i * (64 / kTurnedLanes) + lane / kTurnedLanes; }
  static __device__ __forceinline__ int turned_row(int lane) { return 4 * (lane % kTurnedLanes); }
  template <class T, class T4>
  static __device__ __forceinline__ T4 get_turned(const T* turned, int i, int lane) {
    return *reinterpret_cast<const T4*>(turned + turned_col(i, lane) * kTurnedStride + turned_row(lane));
  }
};

// The 32-row chunks of a wave of S's results: for each, fills it from the
// accumulators and calls use(its number, chunk), the number as a constant.
// 16 x 16 tiles acc[MI][NI] of f32x4, or 32 x 32 ones of f32x16.
// (Folds, not loops: accumulators live in registers only where every index is
// known, and the unroller gives up on bodies this long.)
template <class S, class F, int... C>
__device__ __forceinline__ void chunks_of(float* chunk, int lane, const f32x4 (&acc)[S::MI][S::NI], F&& use,
                                          std::integer_sequence<int, C...>) {
  using Chunk = ResultChunk<S::kRowsN>;
  ([&] {
#pragma unroll
    for (int mi = 0; mi < 2; ++mi)
#pragma unroll
      for (int ni = 0; ni < S::NI; ++ni)
        Chunk::put(chunk, mi * 16 + (lane & 15), ni * 16 + 4 * (lane >> 4), acc[2 * C + mi][ni]);
    use(std::integral_constant<int, C>{}, chunk);
  }(), ...);
}

template <class S, class F, int... C>
__device__ __forceinline__ void chunks_of(float* chunk, int lane, const f32x16 (&acc)[WideTile::MI][WideTile::NI], F&& use,
                                          std::integer_sequence<int, C...>) {
  using Chunk = ResultChunk<S::kRowsN>;
  ([&] {
#pragma unroll
    for (int ni = 0; ni < WideTile::NI; ++ni)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        Chunk::put(chunk, lane & 31, ni * 32 + 8 * q + 4 * (lane >> 5),
                   f32x4{acc[C][ni][4 * q], acc[C][ni][4 * q + 1], acc[C][ni][4 * q + 2], acc[C][ni][4 * q + 3]});
    use(std::integral_constant<int, C>{}, chunk);
  }(), ...);
}

template <class S, class Acc, class F>
__device__ __forceinline__ void for_each_chunk(float* chunk, int lane, const Acc& acc, F&& use) {
  chunks_of<S>(chunk, lane, acc, use, std::make_integer_sequence<int, S::kRowsM / 32>{});
}

}  // namespace sr
