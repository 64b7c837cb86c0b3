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
// A workgroup takes a 128 x 128 tile of x into registers, each thread 4 x 4
// values of each of four 32-row bands, so that one read serves both
// orientations: row blocks reduce over half a wave, column blocks over
// the bands and, through LDS, over the eight half-waves.  Encoded bytes of
// the transposed orientation are turned 4 x 4 in registers and cross LDS
// once; both outputs leave as whole 128-byte runs.
// ---------------------------------------------------------------------------
constexpr int kCastTile = 128, kCastThreads = 256;

struct BlockCastArgs {
  const char* x;
  int64_t ldx, rows, cols;
  sr_block_output by_rows, by_cols;
  uint32_t counter_base;  // seed + offset (mod 2^32)
  uint32_t tiles_n;
};

// The exponent e of a block's scale 2^e from the bits of its largest finite
// magnitude: with amax = f 2^E, 1 <= f < 2, and the format's maximum
// 1.75 2^top, e = E - top, one more where f > 1.75; 0 where amax is 0.
// Subnormal amax are far below 2^(top - 127), where e stays at -127.
template <int TOP>
__device__ __forceinline__ int block_exponent(uint32_t amax) {
  const int e = static_cast<int>(amax >> 23) - 127 - TOP + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return amax == 0 ? 0 : (e > -127 ? e : -127);
}

// 2^-e, e in [-127, 120]: always a normal number.
__device__ __forceinline__ float inverse_scale(int e) { return bits_f32(static_cast<uint32_t>(127 - e) << 23); }

__device__ __forceinline__ uint32_t finite_magnitude(float x) {
  const uint32_t a = f32_bits(x) & 0x7FFFFFFFu;
  return a < 0x7F800000u ? a : 0u;
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Byte j of each of four words, for j = 0..3: a 4 x 4 byte transpose.
__device__ __forceinline__ void transpose_bytes(uint32_t (&w)[4]) {
  const uint32_t lo01 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), hi01 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
  const uint32_t lo23 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), hi23 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
}

template <int XE, int QE, bool SQUARE>
__global__ __launch_bounds__(kCastThreads) void block_cast_kernel(BlockCastArgs a) {
  constexpr int TOP = (QE == ENC_E4M3_RN || QE == ENC_E4M3_SR) ? 8 : 15;
  constexpr int XB = enc_bytes(XE);
  __shared__ uint32_t turned[kCastTile * 32];
  __shared__ uint32_t partial[8][kCastTile];
  __shared__ uint32_t whole[8];
  const int t = threadIdx.x, half = t >> 5, lane = t & 31;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / a.tiles_n) * kCastTile;
  const int64_t col0 = static_cast<int64_t>(blockIdx.x % a.tiles_n) * kCastTile;
  const int64_t c = col0 + 4 * lane;
  const int live = c >= a.cols ? 0 : (a.cols - c < 4 ? static_cast<int>(a.cols - c) : 4);

  // Rows of this thread: band k, row 32 k + 4 half + i.
  float x[4][4][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = row0 + 32 * k + 4 * half + i;
      const char* p = a.x + (r * a.ldx + c) * XB;
      if (r < a.rows && live == 4) {
        uint32_t w[group_words(XE)];
        load_words<4 * XB, true>(p, w);
        decode_group<XE>(w, x[k][i]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[k][i][j] = r < a.rows && j < live ? decode<XE>(load1<XE>(p, j)) : 0.0f;
      }
    }
  }

  const bool want_rows = a.by_rows.data != nullptr, want_cols = a.by_cols.data != nullptr;
  uint32_t tile_max = 0;  // SQUARE
  int col_exp[4];         // of this thread's four columns
  if (SQUARE || want_cols) {
    uint32_t m[4] = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = umax(m[j], finite_magnitude(x[k][i][j]));
    if constexpr (SQUARE) {
      tile_max = umax(umax(m[0], m[1]), umax(m[2], m[3]));
#pragma unroll
      for (int d = 16; d; d >>= 1) tile_max = umax(tile_max, __shfl_xor(tile_max, d, 32));
      if (lane == 0) whole[half] = tile_max;
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 8; ++h) tile_max = umax(tile_max, whole[h]);
#pragma unroll
      for (int j = 0; j < 4; ++j) col_exp[j] = block_exponent<TOP>(tile_max);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) partial[half][4 * lane + j] = m[j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int h = 0; h < 8; ++h) m[j] = umax(m[j], partial[h][4 * lane + j]);
        col_exp[j] = block_exponent<TOP>(m[j]);
      }
    }
  }

#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t hash[4][4], by_col[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = row0 + 32 * k + 4 * half + i;
      const uint32_t counter = a.counter_base + static_cast<uint32_t>(r) * static_cast<uint32_t>(a.cols) + static_cast<uint32_t>(c);
#pragma unroll
      for (int j = 0; j < 4; ++j) hash[i][j] = enc_stochastic(QE) ? h32(counter + static_cast<uint32_t>(j)) : 0u;
      uint32_t bits[4], word[1];
      if (want_rows) {
        int e;
        if constexpr (SQUARE) {
          e = col_exp[0];
        } else {
          uint32_t m = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) m = umax(m, finite_magnitude(x[k][i][j]));
#pragma unroll
          for (int d = 16; d; d >>= 1) m = umax(m, __shfl_xor(m, d, 32));
          e = block_exponent<TOP>(m);
        }
        const float inv = inverse_scale(e);
#pragma unroll
        for (int j = 0; j < 4; ++j) bits[j] = f32_bits(x[k][i][j] * inv);
        encode_group_with<QE>(bits, hash[i], word);
        if (r < a.rows) {
          char* q = static_cast<char*>(a.by_rows.data) + r * a.by_rows.ld + c;
          if (live == 4) {
            store_words<4>(q, word);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (j < live) *gptr_mut<uint8_t>(q + j) = static_cast<uint8_t>(word[0] >> (8 * j));
          }
          if constexpr (!SQUARE)
            if (lane == 0)
              *gptr_mut<uint8_t>(static_cast<char*>(a.by_rows.scale) + r * a.by_rows.ld_scale + col0 / kCastTile) =
                  static_cast<uint8_t>(e + 127);
        }
      }
      if (want_cols) {
#pragma unroll
        for (int j = 0; j < 4; ++j) bits[j] = f32_bits(x[k][i][j] * inverse_scale(col_exp[j]));
        encode_group_with<QE>(bits, hash[i], word);
        by_col[i] = word[0];
      }
    }
    if (want_cols) {
      transpose_bytes(by_col);
      // Column 4 lane + j, rows 32 k + 4 half .. + 3, at word (row / 4) ^ lane of its column: the lanes of a
      // half-wave meet in different banks here, and those that read a column below do too.
#pragma unroll
      for (int j = 0; j < 4; ++j) turned[(4 * lane + j) * 32 + ((8 * k + half) ^ lane)] = by_col[j];
    }
  }

  if (SQUARE && t == 0) {
    const uint8_t byte = static_cast<uint8_t>(block_exponent<TOP>(tile_max) + 127);
    const int64_t rb = row0 / kCastTile, cb = col0 / kCastTile;
    if (want_rows) *gptr_mut<uint8_t>(static_cast<char*>(a.by_rows.scale) + rb * a.by_rows.ld_scale + cb) = byte;
    if (want_cols) *gptr_mut<uint8_t>(static_cast<char*>(a.by_cols.scale) + cb * a.by_cols.ld_scale + rb) = byte;
  }
  if (!want_cols) return;
  if constexpr (!SQUARE) {
    if (half == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < live)
          *gptr_mut<uint8_t>(static_cast<char*>(a.by_cols.scale) + (c + j) * a.by_cols.ld_scale + row0 / kCastTile) =
              static_cast<uint8_t>(col_exp[j] + 127);
    }
  }
  __syncthreads();
  const int64_t r = row0 + 4 * lane;
  const int live_r = r >= a.rows ? 0 : (a.rows - r < 4 ? static_cast<int>(a.rows - r) : 4);
#pragma unroll
  for (int k = 0; k < kCastTile / 8; ++k) {
    const int col = 8 * k + half;
    if (col0 + col >= a.cols) break;
    const uint32_t word[1] = {turned[col * 32 + (lane ^ (col >> 2))]};
    char* q = static_cast<char*>(a.by_cols.data) + (col0 + col) * a.by_cols.ld + r;
    if (live_r == 4) {
      store_words<4>(q, word);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < live_r) *gptr_mut<uint8_t>(q + j) = static_cast<uint8_t>(word[0] >> (8 * j));
    }
  }
}

// ---------------------------------------------------------------------------
// Product of two block-scaled matrices.
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

// Four consecutive results of row `row`.
__device__ __forceinline__ void store_results(const BlockProductArgs& g, int row, int col, const f32x4& v) {
  if (row >= g.m || col >= g.n) return;
  const int live = g.n - col < 4 ? g.n - col : 4;
  const int64_t at = row * g.ldo + col;
  if (g.out_dtype == SR_F32) {
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
    return;
  }
  uint32_t code[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    code[j] = g.out_dtype == SR_BF16 ? bf16_rn(f32_bits(v[j])) : minifloat_encode<F16, false>(f32_bits(v[j]), 0u);
  uint16_t* p = reinterpret_cast<uint16_t*>(g.out) + at;
  if (live == 4) {
    *(SR_GLOBAL group8*)(p) = group8{code[0] | code[1] << 16, code[2] | code[3] << 16};
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < live) *gptr_mut<uint16_t>(p + j) = static_cast<uint16_t>(code[j]);
  }
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

// The FP32 value of an E8M0 byte.
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
  return bits_f32(byte == 0 ? 0x00400000u : (byte == 255 ? 0x7FC00000u : byte << 23));
}

// The scales one lane needs for one block of the contracted axis.  kExponents:
// the exponent byte of its row of each fragment.  Otherwise: the factor of its
// row of A and of each of the four rows of B whose results it holds.  Rows
// past the end repeat the last one.
template <int MODE, int MI, int NI>
struct Scales {
  static constexpr bool kExp = MODE == kExponents;
  static constexpr int kPerB = kExp ? 1 : 4;
  using Value = std::conditional_t<kExp, int, float>;
  Value a[MI], b[NI][kPerB];

  struct Places {
    const char* a;  // of the first scale row of this workgroup's tile
    const char* b;
    uint32_t offset_a[MI], offset_b[NI][kPerB];  // bytes; a tile spans at most 2^8 rows of at most 2^20 scales
    uint32_t size;                               // of one scale
    bool shared_b;

    __device__ void init(const BlockProductArgs& g, int tile_row, int tile_col, int wave_row, int wave_col, int lane) {
      size = kExp ? 1 : (MODE == kFactors || g.scale_f32 ? 4 : 1);
      const int first_a = tile_row >> g.shift_a, first_b = tile_col >> g.shift_b;
      a = g.scale_a + first_a * g.ld_scale_a * size;
      b = g.scale_b + first_b * g.ld_scale_b * size;
      shared_b = g.shift_b != 0;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int r = wave_row + i * 16 + (lane & 15);
        offset_a[i] = static_cast<uint32_t>(((r < g.m ? r : g.m - 1) >> g.shift_a) - first_a) *
                      static_cast<uint32_t>(g.ld_scale_a) * size;
      }
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < kPerB; ++j) {
          const int r = wave_col + i * 16 + (kExp ? lane & 15 : 4 * (lane >> 4) + j);
          offset_b[i][j] = static_cast<uint32_t>(((r < g.n ? r : g.n - 1) >> g.shift_b) - first_b) *
                           static_cast<uint32_t>(g.ld_scale_b) * size;
        }
    }

    __device__ Value read(const char* p) const {
      if constexpr (kExp) return *gptr<uint8_t>(p);
      else if constexpr (MODE == kFactors) return *gptr<float>(p);
      else return size == 4 ? *gptr<float>(p) : e8m0_value(*gptr<uint8_t>(p));
    }
  };

  __device__ void load(const Places& at, int64_t kb) {
    const char* pa = at.a + kb * at.size;
    const char* pb = at.b + kb * at.size;
#pragma unroll
    for (int i = 0; i < MI; ++i) a[i] = at.read(pa + at.offset_a[i]);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
#pragma unroll
      for (int j = 0; j < kPerB; ++j) b[i][j] = j && at.shared_b ? b[i][0] : at.read(pb + at.offset_b[i][j]);
    }
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
template <int MODE, int FA, int FB, int MI, int NI>
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
    for (int j = 0; j < 4; ++j) acc[j] = fmaf(part[j], s.a[mi] * s.b[ni][j], acc[j]);
  }
}

template <int MODE, int FA, int FB, class S, bool ASYNC>
__global__ __launch_bounds__(S::kThreads, 2) void block_product_kernel(BlockProductArgs g) {
  __shared__ __align__(1024) char lds[2 * S::kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t tile_m, tile_n;
  band_tile(xcd_run(blockIdx.x, g.tiles_m * g.tiles_n), g.tiles_m, g.tiles_n, tile_m, tile_n);
  const int row0 = tile_m * S::BM, col0 = tile_n * S::BN;
  const int wave_m = wave / S::WN * S::kRowsM, wave_n = wave % S::WN * S::kRowsN;

  Stager<S> stager;
  stager.init(g.a, g.b, row0, col0, wave, lane);
  Scales<MODE, S::MI, S::NI> scales, next;
  typename Scales<MODE, S::MI, S::NI>::Places places;
  places.init(g, row0, col0, row0 + wave_m, col0 + wave_n, lane);

  f32x4 acc[S::MI][S::NI] = {};
  const uint32_t fragment = fragment_offset(lane);
  auto multiply = [&](const char* stage) {
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
      for (int ni = 0; ni < S::NI; ++ni) block_mma(acc[mi][ni], a, b[ni], scales, mi, ni);
    }
  };

  // Stage kt lies in buffer kt % 2.  At its barrier it has landed for every
  // wave, and every wave is done with the other buffer.
  const int stages = static_cast<int>((g.k + kStageBytes - 1) / kStageBytes);
  if constexpr (ASYNC) {
    const int whole = static_cast<int>(g.k / kStageBytes);
    if (whole > 0) {
      scales.load(places, 0);
      stager.load_async(lds, 0, wave);
    }
    for (int kt = 0; kt < whole; ++kt) {
      stage_barrier();
      if (kt + 1 < whole) {
        next.load(places, kt + 1);
        stager.load_async(lds + (~kt & 1) * S::kStage, static_cast<int64_t>(kt + 1) * kStageBytes, wave);
      }
      multiply(lds + (kt & 1) * S::kStage);
      scales = next;
    }
    if (whole < stages) {  // the contracted axis ends inside a stage
      char* stage = lds + (whole & 1) * S::kStage;
      i32x4 regs[S::kLoads];
      scales.load(places, whole);
      stager.load(regs, static_cast<int64_t>(whole) * kStageBytes, g.k, wave, lane);
      stager.store(stage, regs, wave, lane);
      stage_barrier();
      multiply(stage);
    }
  } else {
    i32x4 regs[S::kLoads];
    if (stages > 0) {
      scales.load(places, 0);
      stager.load(regs, 0, g.k, wave, lane);
      stager.store(lds, regs, wave, lane);
    }
    for (int kt = 0; kt < stages; ++kt) {
      stage_barrier();
      const bool more = kt + 1 < stages;
      if (more) {
        next.load(places, kt + 1);
        stager.load(regs, static_cast<int64_t>(kt + 1) * kStageBytes, g.k, wave, lane);
      }
      multiply(lds + (kt & 1) * S::kStage);
      if (more) stager.store(lds + (~kt & 1) * S::kStage, regs, wave, lane);
      scales = next;
    }
  }

#pragma unroll
  for (int mi = 0; mi < S::MI; ++mi)
#pragma unroll
    for (int ni = 0; ni < S::NI; ++ni)
      store_results(g, row0 + wave_m + mi * 16 + (lane & 15), col0 + wave_n + ni * 16 + 4 * (lane >> 4), acc[mi][ni]);
}

// Few rows of A (at most 16): one 16-column tile of the result per workgroup,
// whose waves take the blocks of the contracted axis in turn and add their
// sums through LDS in wave order.  The operands go from memory to registers:
// each byte of B is used once.
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
  typename Scales<MODE, 1, 1>::Places places;
  places.init(g, 0, col0, 0, col0, lane);
  f32x4 acc{};
  const int stages = static_cast<int>((g.k + kStageBytes - 1) / kStageBytes);
  for (int kb = wave; kb < stages; kb += kRowWaves) {
    Scales<MODE, 1, 1> s;
    s.load(places, kb);
    const int64_t at = static_cast<int64_t>(kb) * kStageBytes + (lane >> 4) * kChunk;
    Fragment<MODE, FA> a;
    Fragment<MODE, FB> b;
    a.set(load_chunk(pa, at, g.k), load_chunk(pa, at + 64, g.k));
    b.set(load_chunk(pb, at, g.k), load_chunk(pb, at + 64, g.k));
    block_mma(acc, a, b, s, 0, 0);
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kRowWaves; ++w) acc += sums[w][lane];
  store_results(g, lane & 15, col0 + 4 * (lane >> 4), acc);
}

}  // namespace sr
