// sr_block_scaled.h -- kernels of the FP8 block-scaled cast and product.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/sr_matrix_hip.h"
#include "sr_kernels.h"
#include "sr_tile_product.h"

namespace sr {

// ---------------------------------------------------------------------------
// Cast to FP8 with a power of two for each block of 128.
//
// Sixteen lanes share a row, eight values each (one 16-byte load of BF16): its
// maximum is four rotations inside them.  Blocks along the columns need
// 128 rows: a thread holds four neighbouring ones, the columns' maxima cross LDS
// once, and the encoded bytes are turned 4 x 4 in registers and cross it
// once.  Rows leave as 128 bytes of sixteen lanes, columns as 128 bytes of 32.
//
// Three kernels:
//   square   square blocks: both orientations hold the same bytes
//   whole    both orientations of a tile from one read of it, with one hash for
//            each value
//   parts    workgroups of one orientation each, smaller than a tile: for one
//            orientation alone, and for both of so few tiles that the chip's CUs
//            would idle (parts against whole, nearest: 128 tiles 5.6 us and 6.4, 192
//            level at 6.8, 256 7.6 and 7.0; stochastic: 128 tiles 7.4 and 8.9, 192
//            10.2 and 9.4, 256 11.5 and 9.6)
//
// 8192 x 2048 BF16 to E4M3, calls one after the other; 67 MB with both results (13
// us at a copy's rate), 50 with one (10): whole 17 us nearest, 23.5 stochastic,
// square 14 and 18, rows alone 11 and 15, columns alone 12 and 16.  The stochastic
// ones are bound by arithmetic, half of it the hash (31 operations for a value
// of both orientations, of which the hash is 17).
// ---------------------------------------------------------------------------
constexpr int kCastTile = 128;

struct BlockCastArgs {
  const char* x;
  int64_t ldx, rows, cols;
  sr_block_output by_rows, by_cols;
  uint32_t counter_base;  // seed + offset (mod 2^32)
  uint32_t tiles_n;       // blocks of 128 columns
  uint32_t first;         // the launch's first workgroup
};

// The format of encoding QE.
template <int QE>
struct CastFormat {
  static constexpr bool kE4M3 = QE == ENC_E4M3_RN || QE == ENC_E4M3_SR;
  using F = std::conditional_t<kE4M3, E4M3, E5M2>;
  static constexpr int kTop = kE4M3 ? 8 : 15;  // the largest value is 1.75 2^kTop
};

// The exponent e of a block's scale 2^e from the bits of its largest finite
// magnitude: with amax = f 2^E, 1 <= f < 2, e = E - top, one more where
// f > 1.75; 0 where amax is 0.  Subnormal amax are far below 2^(top - 127),
// where e stays at -127.
template <int QE>
__device__ __forceinline__ int block_exponent(uint32_t amax) {
  const int e = static_cast<int>(amax >> 23) - 127 - CastFormat<QE>::kTop + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return amax == 0 ? 0 : (e > -127 ? e : -127);
}

// 2^-e, e in [-127, 120]: always a normal number.
__device__ __forceinline__ float inverse_scale(int e) { return bits_f32(static_cast<uint32_t>(127 - e) << 23); }

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t umin(uint32_t a, uint32_t b) { return a < b ? a : b; }

constexpr uint32_t kInfBits = 0x7F800000u;

__device__ __forceinline__ uint32_t magnitude(float x) { return f32_bits(x) & 0x7FFFFFFFu; }

__device__ __forceinline__ uint32_t finite_magnitude(float x) {
  const uint32_t a = magnitude(x);
  return a < kInfBits ? a : 0u;
}

// The largest finite magnitude of eight values; `finite`: all of them are.
__device__ __forceinline__ uint32_t largest(const float (&x)[8], bool finite) {
  uint32_t m = 0;
  if (finite) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) m = umax(umax(m, magnitude(x[j])), magnitude(x[j + 1]));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) m = umax(m, finite_magnitude(x[j]));
  }
  return m;
}

// Byte j of each of four words, for j = 0..3: a 4 x 4 byte transpose.
__device__ __forceinline__ void transpose_bytes(uint32_t (&w)[4]) {
  const uint32_t lo01 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), hi01 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
  const uint32_t lo23 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), hi23 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
}

// The largest of the 16 lanes of a row, in all of them.
__device__ __forceinline__ uint32_t max_of_16(uint32_t m) {
  m = umax(m, __builtin_amdgcn_update_dpp(0u, m, 0x128, 0xF, 0xF, true));  // rotations by 8, 4, 2, 1 lanes
  m = umax(m, __builtin_amdgcn_update_dpp(0u, m, 0x124, 0xF, 0xF, true));
  m = umax(m, __builtin_amdgcn_update_dpp(0u, m, 0x122, 0xF, 0xF, true));
  return umax(m, __builtin_amdgcn_update_dpp(0u, m, 0x121, 0xF, 0xF, true));
}

// Eight values of two bytes, and eight bytes, in one access each that promises one element's alignment (rows start
// anywhere; sr_group_access.h's types of these sizes promise more, their groups being of larger elements).
typedef uint32_t eight_halves __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t eight_bytes __attribute__((ext_vector_type(2), aligned(1)));

// Eight values from `p`, of which the first `live` are there; zeros for the rest.
template <int XE>
__device__ __forceinline__ void load_eight(const char* p, int live, float (&x)[8]) {
  if (live == 8) {
    uint32_t w[2 * group_words(XE)];
    if constexpr (enc_bytes(XE) == 4) {
      load_words<16, true>(p, w);
      load_words<16, true>(p + 16, w + 4);
    } else {
      const eight_halves values = *(const SR_GLOBAL eight_halves*)(p);
      __builtin_memcpy(w, &values, 16);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t words[group_words(XE)];
      float v[4];
#pragma unroll
      for (int j = 0; j < group_words(XE); ++j) words[j] = w[h * group_words(XE) + j];
      decode_group<XE>(words, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * h + j] = v[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < live ? decode<XE>(load1<XE>(p, j)) : 0.0f;
  }
}

// The hashes of eight consecutive counters.
template <int QE>
__device__ __forceinline__ void hash_eight(uint32_t counter, uint32_t (&hash)[2][4]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) hash[j >> 2][j & 3] = enc_stochastic(QE) ? h32(counter + static_cast<uint32_t>(j)) : 0u;
}

// Four values, scaled into the format's range, as FP8.  Where they are finite
// and (stochastic) zeros or at least the format's smallest normal number, the
// rule is an addition: the random bits as far below the format's last bit as
// FP32 has bits, and a truncation, after which the convert is exact.  The
// general rule takes the rest (4% of the waves' groups of normally
// distributed values for stochastic E4M3, next to none for the others).
template <int QE>
__device__ __forceinline__ uint32_t encode_scaled(const float (&y)[4], const uint32_t (&hash)[4], bool finite) {
  using F = typename CastFormat<QE>::F;
  uint32_t bits[4], word[1];
#pragma unroll
  for (int j = 0; j < 4; ++j) bits[j] = f32_bits(y[j]);
  bool plain = finite;
  if constexpr (enc_stochastic(QE)) {
    uint32_t smallest = 0xFFFFFFFFu;  // of 2 |y| - 1, for zeros the largest of all
#pragma unroll
    for (int j = 0; j < 4; j += 2) smallest = umin(umin(smallest, 2 * bits[j] - 1), 2 * bits[j + 1] - 1);
    plain = plain && smallest >= (static_cast<uint32_t>(127 + F::kEmin) << 24) - 1;
  }
  if (plain) {
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (enc_stochastic(QE)) {
      constexpr int kShift = 9 + F::kM;
#pragma unroll
      for (int j = 0; j < 4; ++j) bits[j] = (bits[j] + (~hash[j] >> kShift)) & ~(0xFFFFFFFFu >> kShift);
    }
    if constexpr (CastFormat<QE>::kE4M3) {
      const int low = __builtin_amdgcn_cvt_pk_fp8_f32(bits_f32(bits[0]), bits_f32(bits[1]), 0, false);
      word[0] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(bits_f32(bits[2]), bits_f32(bits[3]), low, true));
    } else {
      const int low = __builtin_amdgcn_cvt_pk_bf8_f32(bits_f32(bits[0]), bits_f32(bits[1]), 0, false);
      word[0] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_bf8_f32(bits_f32(bits[2]), bits_f32(bits[3]), low, true));
    }
#endif
  } else {
    encode_group_with<QE>(bits, hash, word);
  }
  return word[0];
}

// One row's eight values under their block's scale.
template <int QE>
__device__ __forceinline__ void encode_row(const float (&x)[8], int e, const uint32_t (&hash)[2][4], bool finite,
                                           uint32_t (&words)[2]) {
  const float inv = inverse_scale(e);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float y[4] = {x[4 * h] * inv, x[4 * h + 1] * inv, x[4 * h + 2] * inv, x[4 * h + 3] * inv};
    words[h] = encode_scaled<QE>(y, hash[h], finite);
  }
}

// Stores the first `live` of eight bytes.
__device__ __forceinline__ void store_eight(char* q, const uint32_t (&words)[2], int live) {
  if (live == 8) {
    *(SR_GLOBAL eight_bytes*)(q) = eight_bytes{words[0], words[1]};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < live) *gptr_mut<uint8_t>(q + j) = static_cast<uint8_t>(words[j >> 2] >> (8 * (j & 3)));
  }
}

__device__ __forceinline__ void store_exponent(const sr_block_output& to, int64_t row, int64_t col, int e) {
  *gptr_mut<uint8_t>(static_cast<char*>(to.scale) + row * to.ld_scale + col) = static_cast<uint8_t>(e + 127);
}

template <class T>
__device__ __forceinline__ int live_of(T at, T end, int width) {
  return at >= end ? 0 : (end - at < width ? static_cast<int>(end - at) : width);
}

// The tile of 128 rows and 8 LANES columns from (row0, col0), by a workgroup
// of 32 LANES threads, of which LANES share four neighbouring rows.
template <int XE, int QE, bool SQUARE, int LANES>
__device__ __forceinline__ void cast_tile(const BlockCastArgs& a, int64_t row0, int64_t col0, bool want_rows, bool want_cols) {
  constexpr int kGroups = 32, kThreads = kGroups * LANES, kCols = 8 * LANES;
  constexpr int kTurn = 32 / LANES;
  __shared__ uint32_t turned[kCols * 32];
  __shared__ __align__(16) uint32_t partial[SQUARE ? 1 : kGroups][kCols];
  __shared__ __align__(16) int exponents[kCols];
  __shared__ uint32_t whole[kThreads / 64];
  const int t = threadIdx.x, group = t / LANES, lane = t % LANES;
  const int64_t r0 = row0 + 4 * group, c = col0 + 8 * lane;
  const int live = live_of(c, a.cols, 8);

  float x[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    load_eight<XE>(a.x + ((r0 + i) * a.ldx + c) * enc_bytes(XE), r0 + i < a.rows ? live : 0, x[i]);

  uint32_t m[8] = {}, any = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) m[j] = umax(umax(m[j], magnitude(x[i][j])), magnitude(x[i + 1][j]));
    any = umax(any, m[j]);
  }
  const bool finite = any < kInfBits;
  int tile_exp = 0;  // SQUARE
  int col_exp[8];    // otherwise, of this thread's columns
  {
    if (!finite) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        m[j] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m[j] = umax(m[j], finite_magnitude(x[i][j]));
      }
    }
    if constexpr (SQUARE) {
      uint32_t tile = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) tile = umax(tile, m[j]);
      tile = max_of_16(tile);
      tile = umax(tile, __shfl_xor(tile, 16));
      tile = umax(tile, __shfl_xor(tile, 32));
      if ((t & 63) == 0) whole[t >> 6] = tile;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kThreads / 64; ++w) tile = umax(tile, whole[w]);
      tile_exp = block_exponent<QE>(tile);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) partial[group][8 * lane + j] = m[j];
      __syncthreads();
      if (t < kCols) {
        uint32_t col = 0;
#pragma unroll
        for (int h = 0; h < kGroups; ++h) col = umax(col, partial[h][t]);
        const int e = block_exponent<QE>(col);
        exponents[t] = e;
        if (col0 + t < a.cols) store_exponent(a.by_cols, col0 + t, row0 / kCastTile, e);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) col_exp[j] = exponents[8 * lane + j];
    }
  }

  uint32_t by_col[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = r0 + i;
    uint32_t hash[2][4], words[2];
    hash_eight<QE>(a.counter_base + static_cast<uint32_t>(r) * static_cast<uint32_t>(a.cols) + static_cast<uint32_t>(c), hash);
    if constexpr (SQUARE) {
      encode_row<QE>(x[i], tile_exp, hash, finite, words);
      if (want_rows && r < a.rows) store_eight(static_cast<char*>(a.by_rows.data) + r * a.by_rows.ld + c, words, live);
    } else {
      if (want_rows) {
        const int e = block_exponent<QE>(max_of_16(largest(x[i], finite)));
        encode_row<QE>(x[i], e, hash, finite, words);
        if (r < a.rows) {
          store_eight(static_cast<char*>(a.by_rows.data) + r * a.by_rows.ld + c, words, live);
          if (lane == 0) store_exponent(a.by_rows, r, col0 / kCastTile, e);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = x[i][4 * h + j] * inverse_scale(col_exp[4 * h + j]);
        words[h] = encode_scaled<QE>(y, hash[h], finite);
      }
    }
    by_col[0][i] = words[0];
    by_col[1][i] = words[1];
  }
  if constexpr (SQUARE) {
    if (t == 0) {
      if (want_rows) store_exponent(a.by_rows, row0 / kCastTile, col0 / kCastTile, tile_exp);
      if (want_cols) store_exponent(a.by_cols, col0 / kCastTile, row0 / kCastTile, tile_exp);
    }
    if (!want_cols) return;
  }

  // Column 8 lane + j, rows r0 .. r0 + 3, at word group ^ (kTurn lane) of its column's 32: the lanes of a wave then
  // meet in a bank two at a time, and those that read a column below do not.
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    transpose_bytes(by_col[h]);
#pragma unroll
    for (int j = 0; j < 4; ++j) turned[(8 * lane + 4 * h + j) * 32 + (group ^ (kTurn * lane))] = by_col[h][j];
  }
  __syncthreads();
  const int word_at = t & 31, part = t >> 5;
  const int64_t r = row0 + 4 * word_at;
  const int live_r = live_of(r, a.rows, 4);
#pragma unroll
  for (int k = 0; k < kCols * 32 / kThreads; ++k) {
    const int col = kThreads / 32 * k + part;
    if (col0 + col >= a.cols) break;
    const uint32_t word = turned[col * 32 + (word_at ^ (kTurn * (col >> 3)))];
    char* q = static_cast<char*>(a.by_cols.data) + (col0 + col) * a.by_cols.ld + r;
    if (live_r == 4) {
      *(SR_GLOBAL group4*)(q) = word;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < live_r) *gptr_mut<uint8_t>(q + j) = static_cast<uint8_t>(word >> (8 * j));
    }
  }
}

constexpr int kTileThreads = 512, kPartThreads = 256;
constexpr uint64_t kWholeTiles = 256;  // see above

template <int XE, int QE, bool SQUARE>
__global__ __launch_bounds__(kTileThreads, SQUARE ? 6 : 4) void block_cast_tile_kernel(BlockCastArgs a) {
  const uint32_t tile = a.first + blockIdx.x;
  cast_tile<XE, QE, SQUARE, 16>(a, static_cast<int64_t>(tile / a.tiles_n) * kCastTile,
                              static_cast<int64_t>(tile % a.tiles_n) * kCastTile, a.by_rows.data != nullptr,
                              a.by_cols.data != nullptr);
}

// The workgroups of a band of 128 rows: where the row orientation is asked
// for, eight times tiles_n of 16 rows x 128 columns, along the rows first; then
// two times tiles_n of 64 columns.
constexpr int kPartRows = kPartThreads / 16, kPartLanes = 8;
constexpr int kRowParts = kCastTile / kPartRows, kColParts = kCastTile / (8 * kPartLanes);

template <int XE, int QE>
__global__ __launch_bounds__(kPartThreads, enc_stochastic(QE) ? 5 : 6) void block_cast_parts_kernel(BlockCastArgs a) {
  const uint32_t row_parts = a.by_rows.data ? kRowParts : 0, parts = row_parts + (a.by_cols.data ? kColParts : 0);
  const uint32_t id = a.first + blockIdx.x, band = id / (parts * a.tiles_n), within = id - band * parts * a.tiles_n;
  const int64_t row0 = static_cast<int64_t>(band) * kCastTile;
  if (within >= row_parts * a.tiles_n) {
    cast_tile<XE, QE, false, kPartLanes>(a, row0, static_cast<int64_t>(within - row_parts * a.tiles_n) * 8 * kPartLanes, false, true);
    return;
  }
  const uint32_t part = within / a.tiles_n;
  const int64_t block = within - part * a.tiles_n;
  const int lane = threadIdx.x & 15;
  const int64_t r = row0 + kPartRows * part + (threadIdx.x >> 4), c = block * kCastTile + 8 * lane;
  if (r >= a.rows) return;  // sixteen lanes together
  const int live = live_of(c, a.cols, 8);
  float x[8];
  load_eight<XE>(a.x + (r * a.ldx + c) * enc_bytes(XE), live, x);
  uint32_t any = largest(x, true);
  const bool finite = any < kInfBits;
  if (!finite) any = largest(x, false);
  const int e = block_exponent<QE>(max_of_16(any));
  uint32_t hash[2][4], words[2];
  hash_eight<QE>(a.counter_base + static_cast<uint32_t>(r) * static_cast<uint32_t>(a.cols) + static_cast<uint32_t>(c), hash);
  encode_row<QE>(x, e, hash, finite, words);
  store_eight(static_cast<char*>(a.by_rows.data) + r * a.by_rows.ld + c, words, live);
  if (lane == 0) store_exponent(a.by_rows, r, block, e);
}

// ---------------------------------------------------------------------------
// Product of two block-scaled matrices: out = sum over blocks of
// scale_a scale_b (sum over the block of a b).
//
// Both operands have the contracted axis last, so that a stage, 128 bytes of
// every row of a tile, is one scaled block of each row and one 16x16x128
// instruction per 16 x 16 results.  Tiles of 128 x 128 results and of 64 x 64
// (see tile_by_count); rows of at most 16 take the kernel at the end.
//
// 8192 x 8192 x 2048 takes 144 us (1900 TFLOP/s) when the card is rested: the matrix
// cores work 43% of the cycles and the LDS 33%, and every stage of a workgroup
// waits once for its loads.  Call after call it takes 145 to 175 as the clock
// falls under the load (1.7 GHz after 20 calls, 2.4 at rest; zeros as data: 122), and
// 256 x 256 tiles are level.  Small ones are bound by latency: 4.3 us of
// arguments, first stage and result, then 0.5 to 1 us a stage (501 x 2304 x 768: 6.7
// us).
// ---------------------------------------------------------------------------
struct BlockProductArgs {
  Operand a, b;
  const char* scale_a;
  const char* scale_b;
  int64_t ld_scale_a, ld_scale_b;
  int shift_a, shift_b;  // log2 of the rows that share a scale: 0 or 7
  int64_t k;
  char* out;
  int64_t ldo;
  int m, n, out_dtype;
  int scale_f32;  // the scales are FP32 factors, not E8M0 bytes
  uint32_t tiles_m, tiles_n;
};

// Format selector of the f8f6f4 matrix instructions.
template <int DT>
constexpr int kFormatCode = DT == SR_E4M3 ? 0 : 1;

// Four consecutive results of row `row`, as OUT.  EDGE: they may lie outside the result, wholly or in part.
template <int OUT, bool EDGE>
__device__ __forceinline__ void store_results(const BlockProductArgs& g, int row, int col, const f32x4& v) {
  if (EDGE && (row >= g.m || col >= g.n)) return;
  const int live = EDGE && g.n - col < 4 ? g.n - col : 4;
  const int64_t at = row * g.ldo + col;
  if constexpr (OUT == SR_F32) {
    float* p = reinterpret_cast<float*>(g.out) + at;
    if (live == 4) {
      uint32_t w[4];
      __builtin_memcpy(w, &v, 16);
      *(SR_GLOBAL group16*)(p) = group16{w[0], w[1], w[2], w[3]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < live) *gptr_mut<float>(p + j) = v[j];
    }
  } else {
    const float x[4] = {v[0], v[1], v[2], v[3]};
    uint32_t w[2];
    encode_group<OUT == SR_BF16 ? ENC_BF16_RN : ENC_F16_RN>(x, 0u, w);
    uint16_t* p = reinterpret_cast<uint16_t*>(g.out) + at;
    if (live == 4) {
      *(SR_GLOBAL group8*)(p) = group8{w[0], w[1]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < live) *gptr_mut<uint16_t>(p + j) = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

// Calls store(OUT, EDGE) for the result's type and whether the rows x cols from (row0, col0) pass its edges.
template <class F>
__device__ __forceinline__ void with_output(const BlockProductArgs& g, int row0, int col0, int rows, int cols, F&& store) {
  auto typed = [&](auto out) {
    if (row0 + rows <= g.m && col0 + cols <= g.n) store(out, std::false_type{});
    else store(out, std::true_type{});
  };
  if (g.out_dtype == SR_F32) typed(std::integral_constant<int, SR_F32>{});
  else if (g.out_dtype == SR_BF16) typed(std::integral_constant<int, SR_BF16>{});
  else typed(std::integral_constant<int, SR_F16>{});
}

// Stores a workgroup's results through its LDS, which every wave is done with.
template <int LDS, class S, class Acc>
__device__ __forceinline__ void store_chunks(const BlockProductArgs& g, char* lds, int row0, int col0, int wave, int lane,
                                             const Acc& acc) {
  using Chunk = ResultChunk<S::kRowsN>;
  static_assert(S::kWaves * Chunk::kBytes <= LDS, "a chunk per wave");
  const int wave_row = row0 + wave / S::WN * S::kRowsM, wave_col = col0 + wave % S::WN * S::kRowsN;
  float* chunk = reinterpret_cast<float*>(lds + wave * Chunk::kBytes);
  with_output(g, row0, col0, S::BM, S::BN, [&](auto out, auto edge) {
    for_each_chunk<S>(chunk, lane, acc, [&](auto number, const float* from) {
      constexpr int first = 32 * decltype(number)::value;
#pragma unroll
      for (int i = 0; i < Chunk::kBlocks; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = Chunk::block_row(i, lane) + k, col = Chunk::block_col(lane);
          store_results<decltype(out)::value, decltype(edge)::value>(g, wave_row + first + row, wave_col + col,
                                                                     Chunk::get(from, row, col));
        }
    });
  });
}

// How a product multiplies and scales.
//   kExponents  FP8 instructions, which apply E8M0 scales inside their sum
//   kFactors    FP8 instructions per block, FP32 scales applied to the block's sum
//   kWide       FP16 instructions on the widened values (exact), scales of
//               either type applied to the block's sum
// The FP8 instructions round inside: 1.5e-5 of the result's norm for one dot
// of 128 E4M3 values (measured; 1.2e-5 for E5M2 x E4M3, 9e-6 for E5M2), alike
// in the 16x16x128 and the half as fast 16x16x32 forms.  That disappears in a
// BF16 or FP16 result (1.7e-3, 2e-4) but not in an FP32 one, which therefore
// takes the FP16 instructions (4e-8) at half the rate.
enum ProductMode { kExponents, kFactors, kWide, kProductModes };

// A block's sum times two FP32 scales.  It lies between 2^-32 and 2^39 or is 0,
// but the scales' product, or that of the sum and one scale, can leave FP32's
// range on the way to a result inside it (2^100 by 2^30 with a small sum gave
// infinity, with a sum of 0 NaN).  Scales between 2^-62 and 2^62, and zeros, are
// `near`: their product is safe, and one multiplication and the fused one into
// the result do.  A tile that has others looks at its scales' largest and
// smallest products, and where these are no normal numbers it sums again with
// each scale as two factors of about half its exponent.  With T the result's
// exponent and S the sum's, both partial products below are then near
// 2^((T + S) / 2) and 2^((T - S) / 2): inside the range wherever 2^T is.  (A tile
// that sums again takes four times as long; one that only looks, 1 to 2 us more.)
struct ScaleRange {
  uint32_t high = 0, low = 0xFFFFFFFFu;  // magnitudes; the lowest is of those that are not 0, less one
  __device__ __forceinline__ void add(uint32_t bits) {
    const uint32_t m = bits & 0x7FFFFFFFu;
    high = umax(high, m);
    low = umin(low, m - 1);
  }
  __device__ __forceinline__ void add(const ScaleRange& other) {
    high = umax(high, other.high);
    low = umin(low, other.low);
  }
  __device__ __forceinline__ bool near() const { return high <= (189u << 23) && low >= (65u << 23) - 1; }
  __device__ __forceinline__ bool zeros() const { return low == 0xFFFFFFFFu; }
  // Whether every product with a factor of `other`'s is 0 or a normal number.
  __device__ __forceinline__ bool normal_with(const ScaleRange& other) const {
    if (zeros() || other.zeros()) return umax(high, other.high) < kInfBits;
    return bits_f32(high) * bits_f32(other.high) <= 0x1p127f && bits_f32(low + 1) * bits_f32(other.low + 1) >= 0x1p-126f;
  }
};

// The power of two with half the exponent of `s`, rounded down; subnormal numbers, infinities and NaN count as 2^-127
// and 2^128.
__device__ __forceinline__ uint32_t half_power_bits(float s) { return (((f32_bits(s) >> 23 & 255u) + 127u) >> 1) << 23; }

// acc + part * sa * sb; FAR: any scales, otherwise such as have a normal product.
template <bool FAR>
__device__ __forceinline__ float add_scaled(float acc, float part, float sa, float sb) {
  if constexpr (FAR) {
    const uint32_t a = half_power_bits(sa), b = half_power_bits(sb);
    // s 2^-h is exact: 2^-h as the power of two with the opposite exponent.
    const float rest_a = sa * bits_f32((254u << 23) - a), rest_b = sb * bits_f32((254u << 23) - b);
    return fmaf(part * rest_a * rest_b, bits_f32(a) * bits_f32(b), acc);
  } else {
    return fmaf(part, sa * sb, acc);
  }
}

// The FP32 value of an E8M0 byte.
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
  return bits_f32(byte == 0 ? 0x00400000u : (byte == 255 ? 0x7FC00000u : byte << 23));
}

// The scales of a workgroup's rows, 32 bytes of each at a time, in LDS beside
// the stages: 32 exponent bytes where the instructions take them, else 8 FP32
// factors.  Read from memory stage by stage they would cost more than they
// weigh: the scales of one stage lie in a cache line of their own for every
// row, and an access to 64 lines takes 64 cycles (measured at
// 8192 x 8192 x 2048 on 128 x 128 tiles: 202 us with a load per fragment and
// stage, 144 so).  Rows are 36 bytes apart: 32 rows' same bytes then lie in
// different banks.
template <int MODE, class S>
struct ScaleArea {
  static constexpr int kRow = 36, kFill = 32, kBytes = (S::BM + S::BN) * kRow;
  static constexpr int kPeriod = MODE == kExponents ? kFill : kFill / 4;

  // Row r of the area for blocks [first, first + kPeriod), of which `total` - first are there (values past them mean
  // nothing): rows of A, then of B; rows past the operand's end repeat its last one.
  static __device__ __forceinline__ void row(const BlockProductArgs& g, int row0, int col0, int r, int first, int total,
                                             int (&words)[8]) {
    const int size = g.scale_f32 ? 4 : 1;
    const bool of_a = r < S::BM;
    const int at = of_a ? row0 + r : col0 + r - S::BM, rows = of_a ? g.m : g.n;
    const char* from = (of_a ? g.scale_a : g.scale_b) +
                       (((at < rows ? at : rows - 1) >> (of_a ? g.shift_a : g.shift_b)) * (of_a ? g.ld_scale_a : g.ld_scale_b) + first) * size;
    const int64_t end = static_cast<int64_t>(total - first) * size;
    const i32x4 lo = load_chunk(from, 0, end);
    if (MODE == kWide && !g.scale_f32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) words[j] = static_cast<int>(f32_bits(e8m0_value(lo[j >> 2] >> (8 * (j & 3)) & 255)));
      return;
    }
    const i32x4 hi = load_chunk(from, 16, end);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      words[j] = lo[j];
      words[4 + j] = hi[j];
    }
  }

  // These blocks of every row.  Sets *far where a factor is not a near one.
  static __device__ void fill(char* area, int* far, const BlockProductArgs& g, int row0, int col0, int first, int total) {
    ScaleRange range;
    for (int r = threadIdx.x; r < S::BM + S::BN; r += S::kThreads) {
      int words[8];
      row(g, row0, col0, r, first, total, words);
      int* to = reinterpret_cast<int*>(area + r * kRow);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (MODE != kExponents) range.add(j < total - first ? words[j] : 0);
        to[j] = words[j];
      }
    }
    if (MODE != kExponents && !range.near()) *far = 1;
  }

  // Whether every product of a factor of A and one of B that a tile's rows hold is 0 or a normal number, for tiles with
  // factors that are not near ones: what the ordinary walk summed is right then.  `scratch`: LDS, an entry a wave.
  // Every wave is done with the LDS, before and after.
  static __device__ bool products_are_normal(ScaleRange* scratch, const BlockProductArgs& g, int row0, int col0, int total) {
    static_assert(S::BM + S::BN <= S::kThreads && S::BM % 64 == 0 && S::BN % 64 == 0, "a row for a thread, waves of one operand");
    ScaleRange range;
    if (static_cast<int>(threadIdx.x) < S::BM + S::BN) {
      for (int first = 0; first < total; first += kPeriod) {
        int words[8];
        row(g, row0, col0, threadIdx.x, first, total, words);
#pragma unroll
        for (int j = 0; j < 8; ++j) range.add(j < total - first ? words[j] : 0);
      }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) range.add(ScaleRange{__shfl_xor(range.high, d), __shfl_xor(range.low, d)});
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = range;
    lds_barrier();
    ScaleRange sides[2];
#pragma unroll
    for (int w = 0; w < (S::BM + S::BN) / 64; ++w) sides[w * 64 < S::BM ? 0 : 1].add(scratch[w]);
    lds_barrier();
    return sides[0].normal_with(sides[1]);
  }
};

// The scales one lane needs for one block of the contracted axis.  kExponents:
// the exponent byte of its row of each fragment.  Otherwise: the factor of its
// row of A and of each of the four rows of B whose results it holds.
template <int MODE, int MI, int NI>
struct Scales {
  static constexpr bool kExp = MODE == kExponents;
  static constexpr int kPerB = kExp ? 1 : 4;
  using Value = std::conditional_t<kExp, int, float>;
  Value a[MI], b[NI][kPerB];

  // From memory, in the matrices' own type.
  static __device__ __forceinline__ Value read(const char* p, bool f32) {
    if constexpr (kExp) return *reinterpret_cast<const uint8_t*>(p);
    else if constexpr (MODE == kFactors) return *reinterpret_cast<const float*>(p);
    else return f32 ? *reinterpret_cast<const float*>(p) : e8m0_value(*reinterpret_cast<const uint8_t*>(p));
  }

  // From the area.  `wave_m`, `wave_n`: this wave's first rows of A and B in it; `slot`: the block's place in a row.
  template <class S>
  __device__ __forceinline__ void load(const char* area, int wave_m, int wave_n, int slot, int lane) {
    using T = std::conditional_t<kExp, uint8_t, float>;
    constexpr int kRow = ScaleArea<MODE, S>::kRow;
    const char* at = area + slot * sizeof(T);
    const char* pa = at + (wave_m + (lane & 15)) * kRow;
    const char* pb = at + (S::BM + wave_n + (kExp ? lane & 15 : 4 * (lane >> 4))) * kRow;
#pragma unroll
    for (int i = 0; i < MI; ++i) a[i] = *reinterpret_cast<const T*>(pa + i * 16 * kRow);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < kPerB; ++j) b[i][j] = *reinterpret_cast<const T*>(pb + (i * 16 + j) * kRow);
  }
};

// One row's 32 values of a lane, as the instructions take them.
template <int MODE, int FMT>
struct Fragment {
  i32x8 v;
  __device__ void set(const i32x4& lo, const i32x4& hi) { v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
};

template <int FMT>
struct Fragment<kWide, FMT> {
  f16x8 v[4];
  __device__ void set(const i32x4& lo, const i32x4& hi) {
    const int w[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f16x2 pair;
        if constexpr (FMT == SR_E4M3)
          pair = j & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[2 * i + j / 2], 1.0f, true)
                       : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[2 * i + j / 2], 1.0f, false);
        else
          pair = j & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w[2 * i + j / 2], 1.0f, true)
                       : __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w[2 * i + j / 2], 1.0f, false);
        v[i][2 * j] = pair[0];
        v[i][2 * j + 1] = pair[1];
      }
    }
  }
};

// One block of 128 of a 16 x 16 tile of results: B's rows first (see
// sr_tile_product.h).
template <bool FAR, int MODE, int FA, int FB, int MI, int NI>
__device__ __forceinline__ void block_mma(f32x4& acc, const Fragment<MODE, FA>& a, const Fragment<MODE, FB>& b,
                                          const Scales<MODE, MI, NI>& s, int mi, int ni) {
  if constexpr (MODE == kExponents) {
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.v, a.v, acc, kFormatCode<FB>, kFormatCode<FA>, 0,
                                                           s.b[ni][0], 0, s.a[mi]);
  } else {
    f32x4 part{};
    if constexpr (MODE == kFactors) {
      part = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.v, a.v, part, kFormatCode<FB>, kFormatCode<FA>, 0, 0x7F,
                                                              0, 0x7F);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) part = __builtin_amdgcn_mfma_f32_16x16x32_f16(b.v[i], a.v[i], part, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = add_scaled<FAR>(acc[j], part[j], s.a[mi], s.b[ni][j]);
  }
}

// A tile's sums once more where products of its scales leave FP32's normal range: a stage at a time by the first group of waves,
// with few values in registers, so that the ordinary walk keeps its own.  Every wave is done with the LDS, before and
// after.
template <int MODE, int FA, int FB, class S>
__device__ __forceinline__ void sum_far_scales(const BlockProductArgs& g, char* lds, char* area, int* far, int row0, int col0,
                                               int wave, int group, int stages, f32x4 (&acc)[S::MI][S::NI]) {
  using Area = ScaleArea<MODE, S>;
  const int wave_m = wave / S::WN * S::kRowsM, wave_n = wave % S::WN * S::kRowsN;
  int lane = threadIdx.x & 63;
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(lane));  // nothing computed from it is kept over the ordinary walk
#endif
  Stager<S> stager;
  stager.init(g.a, g.b, row0, col0, wave, lane);
  const uint32_t fragment = fragment_offset(lane);
#pragma unroll
  for (int mi = 0; mi < S::MI; ++mi)
#pragma unroll
    for (int ni = 0; ni < S::NI; ++ni) acc[mi][ni] = f32x4{};
  for (int kt = 0; kt < stages; ++kt) {
    if (kt % Area::kPeriod == 0) Area::fill(area, far, g, row0, col0, kt, stages);
    if (group == 0) stager.load_through(lds, static_cast<int64_t>(kt) * kStageBytes, g.k, wave, lane);
    lds_barrier();
    if (group == 0) {
#pragma unroll
      for (int mi = 0; mi < S::MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < S::NI; ++ni) {
          const int row = wave_m + 16 * mi, col = wave_n + 16 * ni;
          const char* sa = lds + row * kStageBytes;
          const char* sb = lds + (S::BM + col) * kStageBytes;
          Scales<MODE, 1, 1> scales;
          scales.template load<S>(area, row, col, kt % Area::kPeriod, lane);
          Fragment<MODE, FA> a;
          Fragment<MODE, FB> b;
          a.set(read_chunk(sa + fragment), read_chunk(sa + (fragment ^ 64)));
          b.set(read_chunk(sb + fragment), read_chunk(sb + (fragment ^ 64)));
          block_mma<true>(acc[mi][ni], a, b, scales, 0, 0);
          asm volatile("" ::: "memory");  // the next tile's reads stay behind this one's
        }
    }
    lds_barrier();
  }
}

// Waves of a SIMD: as many workgroups of a small tile as its stages leave room for in a CU (three with unaligned rows'
// registers), two of the large one.
template <class S>
constexpr int kProductWaves = S::BM > 64 ? S::kMinWaves : (S::kGroups > 1 ? 4 : 3);

template <int MODE, int FA, int FB, class S, bool ASYNC>
__global__ __launch_bounds__(S::kThreads, kProductWaves<S>) void block_product_kernel(BlockProductArgs g) {
  static_assert(ASYNC || S::kGroups == 1, "groups take aligned rows");
  using Area = ScaleArea<MODE, S>;
  constexpr int kStages = S::kLds + Area::kBytes, kChunks = S::kWaves * ResultChunk<S::kRowsN>::kBytes;
  constexpr int kLds = kStages > kChunks ? kStages : kChunks;
  static_assert(S::kSums <= kLds, "the groups' sums");
  // One array: beside a second one the compiler lets the stages' asynchronous loads land before any read of LDS.
  __shared__ __align__(1024) char lds[kLds + 16];
  int* far = reinterpret_cast<int*>(lds + kLds);  // a scale so far is not a near one
  const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = all % S::kWaves, group = all / S::kWaves;
  if (MODE != kExponents && threadIdx.x == 0) *far = 0;  // a barrier comes before the first fill
  uint32_t tile_m, tile_n;
  band_tile(xcd_run(blockIdx.x, g.tiles_m * g.tiles_n), g.tiles_m, g.tiles_n, tile_m, tile_n);
  const int row0 = tile_m * S::BM, col0 = tile_n * S::BN;
  const int wave_m = wave / S::WN * S::kRowsM, wave_n = wave % S::WN * S::kRowsN;

  Stager<S> stager;
  stager.init(g.a, g.b, row0, col0, wave, lane);
  char* own = lds + group * 2 * S::kStage;  // this group's stages
  char* area = lds + S::kLds;

  f32x4 acc[S::MI][S::NI] = {};
  const uint32_t fragment = fragment_offset(lane);
  const int stages = static_cast<int>((g.k + kStageBytes - 1) / kStageBytes);
  auto multiply = [&](const char* stage, int kt) {
    Scales<MODE, S::MI, S::NI> scales;
    scales.template load<S>(area, wave_m, wave_n, kt & (Area::kPeriod - 1), lane);
    const char* sa = stage + wave_m * kStageBytes + fragment;
    const char* sb = stage + (S::BM + wave_n) * kStageBytes + fragment;
    const char* sa2 = stage + wave_m * kStageBytes + (fragment ^ 64);
    const char* sb2 = stage + (S::BM + wave_n) * kStageBytes + (fragment ^ 64);
    Fragment<MODE, FB> b[S::NI];
#pragma unroll
    for (int ni = 0; ni < S::NI; ++ni)
      b[ni].set(read_chunk(sb + ni * 16 * kStageBytes), read_chunk(sb2 + ni * 16 * kStageBytes));
#pragma unroll
    for (int mi = 0; mi < S::MI; ++mi) {
      Fragment<MODE, FA> a;
      a.set(read_chunk(sa + mi * 16 * kStageBytes), read_chunk(sa2 + mi * 16 * kStageBytes));
#pragma unroll
      for (int ni = 0; ni < S::NI; ++ni) block_mma<false>(acc[mi][ni], a, b[ni], scales, mi, ni);
    }
  };

  auto refill = [&](int kt) {
    if ((kt & (Area::kPeriod - 1)) == 0) {
      Area::fill(area, far, g, row0, col0, kt, stages);
      lds_barrier();
    }
  };
  if constexpr (ASYNC) {
    const int whole = static_cast<int>(g.k / kStageBytes);
    walk_stages<S>(
        whole, group, [&](int kt, int buffer) { stager.load_async(own + buffer * S::kStage, kt * kStageBytes, wave); }, refill,
        [&](int kt, int buffer) { multiply(own + buffer * S::kStage, kt); });
    if (whole < stages) {  // the contracted axis ends inside a stage
      stage_barrier();
      refill(whole);
      if (group == 0) stager.load_through(lds, static_cast<int64_t>(whole) * kStageBytes, g.k, wave, lane);
      lds_barrier();
      if (group == 0) multiply(lds, whole);
    }
  } else {
    // Two sets of registers, so that a stage's loads have two stages' time, where they are small enough (of the 128
    // tile, with FP16 instructions, two did not fit: 4096 x 4096 x 1000 took 129 us so).
    constexpr bool kTwo = S::kLoads <= 4;
    i32x4 even[S::kLoads], odd[kTwo ? S::kLoads : 1];
    auto load = [&](i32x4 (&regs)[S::kLoads], int kt) {
      if (kt < stages) stager.load(regs, static_cast<int64_t>(kt) * kStageBytes, g.k, wave, lane);
    };
    auto step = [&](int kt, i32x4 (&next)[S::kLoads], i32x4 (&after)[S::kLoads]) {
      lds_barrier();
      refill(kt);
      load(after, kTwo ? kt + 2 : kt + 1);
      multiply(lds + (kt & 1) * S::kStage, kt);
      if (kt + 1 < stages) stager.store(lds + (~kt & 1) * S::kStage, next, wave, lane);
    };
    load(even, 0);
    if constexpr (kTwo) load(odd, 1);
    if (stages > 0) stager.store(lds, even, wave, lane);
    if constexpr (kTwo) {
      for (int kt = 0; kt < stages; kt += 2) {
        step(kt, odd, even);
        if (kt + 1 < stages) step(kt + 1, even, odd);
      }
    } else {
      for (int kt = 0; kt < stages; ++kt) step(kt, even, even);
    }
  }
  stage_barrier();
  if constexpr (MODE != kExponents) {
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(*far), 0) &&
        !Area::products_are_normal(reinterpret_cast<ScaleRange*>(lds), g, row0, col0, stages))
      sum_far_scales<MODE, FA, FB, S>(g, lds, area, far, row0, col0, wave, group, stages, acc);
  }
  add_groups<S>(lds, group, acc);
  if (group == 0) store_chunks<kLds, S>(g, lds, row0, col0, wave, lane, acc);
}

// Few rows of A (at most 16): one 16-column tile of the result per workgroup,
// whose waves take the blocks of the contracted axis in turn and add their
// sums through LDS in wave order.  The operands go from memory to registers:
// each byte of B is used once.  1 x 8192 x 2048 takes 5.5 us (3.1 TB/s of B), of
// which a launch and its arguments are about 3.
constexpr int kRowWaves = 8;

template <int MODE, int FA, int FB>
__global__ __launch_bounds__(64 * kRowWaves) void block_product_rows_kernel(BlockProductArgs g) {
  __shared__ f32x4 sums[kRowWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col0 = static_cast<int>(xcd_run(blockIdx.x, g.tiles_n)) * 16;
  const int row_a = (lane & 15) < g.m ? lane & 15 : g.m - 1;
  const int row_b = col0 + (lane & 15) < g.n ? col0 + (lane & 15) : g.n - 1;
  const char* pa = g.a.base + row_a * g.a.ld;
  const char* pb = g.b.base + row_b * g.b.ld;
  const int size = g.scale_f32 ? 4 : 1;
  const char* scale_a = g.scale_a + (row_a >> g.shift_a) * g.ld_scale_a * size;
  const char* scale_b[Scales<MODE, 1, 1>::kPerB];
#pragma unroll
  for (int j = 0; j < Scales<MODE, 1, 1>::kPerB; ++j) {
    const int r = col0 + (MODE == kExponents ? lane & 15 : 4 * (lane >> 4) + j);
    scale_b[j] = g.scale_b + ((r < g.n ? r : g.n - 1) >> g.shift_b) * g.ld_scale_b * size;
  }
  f32x4 acc{};
  const int whole = static_cast<int>(g.k / kStageBytes);
  auto block = [&](int kb, auto load) {
    Scales<MODE, 1, 1> s;
    s.a[0] = Scales<MODE, 1, 1>::read(scale_a + static_cast<int64_t>(kb) * size, g.scale_f32);
#pragma unroll
    for (int j = 0; j < Scales<MODE, 1, 1>::kPerB; ++j)
      s.b[0][j] = Scales<MODE, 1, 1>::read(scale_b[j] + static_cast<int64_t>(kb) * size, g.scale_f32);
    const int64_t at = static_cast<int64_t>(kb) * kStageBytes + (lane >> 4) * kChunk;
    Fragment<MODE, FA> a;
    Fragment<MODE, FB> b;
    a.set(load(pa, at), load(pa, at + 64));
    b.set(load(pb, at), load(pb, at + 64));
    block_mma<true>(acc, a, b, s, 0, 0);
  };
  // A wave's blocks are few, so that the loads of two run together.
  auto inside = [](const char* row, int64_t at) { return load_whole_chunk(row, at); };
  int kb = wave;
  for (; kb + kRowWaves < whole; kb += 2 * kRowWaves) {
    block(kb, inside);
    block(kb + kRowWaves, inside);
  }
  if (kb < whole) block(kb, inside);
  if (g.k % kStageBytes && whole % kRowWaves == wave)
    block(whole, [&](const char* row, int64_t at) { return load_chunk(row, at, g.k); });
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kRowWaves; ++w) acc += sums[w][lane];
  with_output(g, 0, col0, 16, 16, [&](auto out, auto edge) {
    store_results<decltype(out)::value, decltype(edge)::value>(g, lane & 15, col0 + 4 * (lane >> 4), acc);
  });
}

}  // namespace sr
