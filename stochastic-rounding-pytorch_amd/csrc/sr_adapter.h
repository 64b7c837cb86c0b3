// sr_adapter.h -- low-rank updates of rows that each have an adapter of their own:
//
//   y[t] = base[t] + s_i (x[t] a_i^T) b_i^T,  i = index[t]
//
// with a_i (rank x k) and b_i (n x rank), and their gradients.  Rows lie in any
// order: a tile of 16 rows goes once through each adapter that it meets, and
// keeps of every pass only the rows that are the adapter's.  Nothing of one
// adapter reaches a row of another, infinities and NaN included.
//
//   shrink    low[t] = s_i x[t] a_i^T in FP32
//   expand    y[t] = base[t] + low[t] b_i^T
//   contract  sums over an adapter's rows t of low[t][r] x[t][c]: the gradients
//             of a (low of dy and b, with x) and of b (low of x and a, with dy)
//
// The input's gradient is shrink by b^T and expand by a^T.
//
// Numbers.  Products of x and the adapters run on their type's matrix
// instructions; what follows takes `low` as FP32.  With BF16 operands a value
// of it enters as two BF16 parts, truncated and rest, which keep 15 bits: far
// below the result's rounding unless the ranks cancel.  FP16 has no exponents for
// that, so FP16 operands widen to FP32 there.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/sr_matrix_hip.h"
#include "sr_group_access.h"
#include "sr_math.h"
#include "sr_tile_product.h"

namespace sr {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
// Sixteen and eight bytes at the alignment of one element.
typedef uint32_t halves8 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t halves4 __attribute__((ext_vector_type(2), aligned(2)));
typedef float floats4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kAdapterWaves = 4, kAdapterThreads = 64 * kAdapterWaves;
constexpr int kRankChunk = 16;  // ranks of one matrix instruction's result

struct Adapters {
  const char* a;         // count x rank x k, or for gradients its transpose or b's
  const void* index;     // the rows' adapters, int64 where `wide`, else int32; none where outside [0, count)
  const float* scaling;  // one for each adapter, or null:
  float scale;           // for all
  int count, rank, chunks;  // chunks: of 16 ranks
  int wide;
  int64_t rows;
};

__device__ __forceinline__ int adapter_of(const Adapters& g, int64_t row) {
  if (row >= g.rows) return -1;
  if (g.wide) {
    const int64_t i = gptr<int64_t>(g.index)[row];
    return i >= 0 && i < g.count ? static_cast<int>(i) : -1;
  }
  const int i = gptr<int32_t>(g.index)[row];
  return i >= 0 && i < g.count ? i : -1;
}

__device__ __forceinline__ float adapter_scale(const Adapters& g, int adapter) {
  return g.scaling ? gptr<float>(g.scaling)[adapter < 0 ? 0 : adapter] : g.scale;
}

// Eight values of the contracted axis, as a matrix instruction takes them.  Which ones share a lane does not matter as
// long as both operands agree: lane q of a row's four takes 16 bytes at 16 q of each 64, so that an access covers 64
// neighbouring bytes of a row.
template <int XE>
struct Eight {
  uint32_t w[enc_bytes(XE) * 2];
};

constexpr int kEightSpan = 32;  // values of a row that its four lanes' eights are

// Lane q's of the 32 values from place `at` of a row on.
template <int XE>
__device__ __forceinline__ Eight<XE> load_eight_whole(const char* row, int64_t at, int q) {
  Eight<XE> e;
  if constexpr (enc_bytes(XE) == 2) {
    const halves8 v = *(const SR_GLOBAL halves8*)(row + 2 * at + 16 * q);
    __builtin_memcpy(e.w, &v, 16);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const floats4 v = *(const SR_GLOBAL floats4*)(row + 4 * at + 64 * h + 16 * q);
      __builtin_memcpy(e.w + 4 * h, &v, 16);
    }
  }
  return e;
}

// The same with zeros from place `end` on.
template <int XE>
__device__ __forceinline__ Eight<XE> load_eight_to(const char* row, int64_t at, int q, int64_t end) {
  Eight<XE> e{};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t c = at + (enc_bytes(XE) == 2 ? 8 * q + j : 16 * (j >> 2) + 4 * q + (j & 3));
    if (c < end) {
      if constexpr (enc_bytes(XE) == 2) e.w[j >> 1] |= static_cast<uint32_t>(gptr<uint16_t>(row)[c]) << (16 * (j & 1));
      else e.w[j] = gptr<uint32_t>(row)[c];
    }
  }
  return e;
}

// acc[4 q + e][i] += sum over the eight places of first and second: see sr_tile_product.h.
template <int XE>
__device__ __forceinline__ void mma_eight(f32x4& acc, const Eight<XE>& first, const Eight<XE>& second) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (XE == ENC_BF16_RN) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, first), __builtin_bit_cast(bf16x8, second), acc, 0, 0, 0);
  } else if constexpr (XE == ENC_F16_RN) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, first), __builtin_bit_cast(f16x8, second), acc, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_f32(first.w[j]), bits_f32(second.w[j]), acc, 0, 0, 0);
  }
#endif
}

// Two FP32 values as BF16, rounded to nearest, and the upper halves of two words.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}
__device__ __forceinline__ uint32_t upper_halves(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }
__device__ __forceinline__ uint32_t lower_halves(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x05040100u); }

// x as two BF16 values of its sign, of which neither is zero unless x is: beside an infinite factor a zero would turn an
// infinite sum into NaN.  The upper half of `upper` is x cut off below its magnitude, one step less where x is a BF16 value itself,
// and `rest` what that leaves (infinite with x).  A rest below 2^-134 rounds to zero, which a magnitude of x below 2^-110
// can leave.
struct TwoParts {
  uint32_t upper;
  float rest;
  __device__ __forceinline__ explicit TwoParts(float x) {
    upper = f32_bits(x) - (x != 0.0f);
    rest = x - bits_f32(upper & 0xFFFF0000u);
  }
};

// Four values in T at `p`, of which `live` are there.
template <int XE>
__device__ __forceinline__ f32x4 load_four(const char* p, int live) {
  f32x4 x{};
  if constexpr (enc_bytes(XE) == 4) {
    if (live >= 4) {
      const floats4 v = *(const SR_GLOBAL floats4*)(p);
      return f32x4{v[0], v[1], v[2], v[3]};
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < live) x[j] = gptr<float>(p)[j];
  } else {
    uint32_t w[2] = {0, 0};
    if (live >= 4) {
      const halves4 v = *(const SR_GLOBAL halves4*)(p);
      w[0] = v[0];
      w[1] = v[1];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < live) w[j >> 1] |= static_cast<uint32_t>(gptr<uint16_t>(p)[j]) << (16 * (j & 1));
    }
    if constexpr (XE == ENC_BF16_RN) {
      x = f32x4{bits_f32(w[0] << 16), bits_f32(w[0] & 0xFFFF0000u), bits_f32(w[1] << 16), bits_f32(w[1] & 0xFFFF0000u)};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)))));
    }
  }
  return x;
}

template <int XE>
__device__ __forceinline__ void store_four(char* p, const f32x4& x, int live) {
  if constexpr (enc_bytes(XE) == 4) {
    if (live >= 4) {
      *(SR_GLOBAL floats4*)(p) = floats4{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < live) gptr_mut<float>(p)[j] = x[j];
    }
  } else {
    uint32_t w[2];
    if constexpr (XE == ENC_BF16_RN) {
      w[0] = pack_bf16(x[0], x[1]);
      w[1] = pack_bf16(x[2], x[3]);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[h] = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(x[2 * h]))) |
               static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(x[2 * h + 1]))) << 16;
    }
    if (live >= 4) {
      *(SR_GLOBAL halves4*)(p) = halves4{w[0], w[1]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < live) gptr_mut<uint16_t>(p)[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

__device__ __forceinline__ int live_four(int64_t at, int64_t end) { return at >= end ? 0 : (end - at < 4 ? static_cast<int>(end - at) : 4); }

// Calls use(adapter, number) for every adapter that 16 rows meet, in the order of their first rows; `mine` is this
// lane's.  Uniform.
template <class F>
__device__ __forceinline__ void for_each_adapter(int mine, F&& use) {
  uint32_t todo = static_cast<uint32_t>(__ballot(mine >= 0)) & 0xFFFFu;
  for (int number = 0; todo; ++number) {
    const int adapter = __builtin_amdgcn_readlane(mine, __builtin_ctz(todo));
    todo &= ~static_cast<uint32_t>(__ballot(mine == adapter));
    use(adapter, number);
  }
}

// Whether the adapters of 64 rows, one a lane, do not come in runs in ascending order: `order` then receives the rows in
// the order of their adapters, between which they keep their own.  For a whole workgroup, whose waves hold the same.
// (8192 rows of 2048 to 2048 in ascending or descending runs 26.5 us without a look and 26.9 with it; in runs of 100 rows in any
// order, whose ends are put in order though they need none, 34.2 and 37.9; mixed row by row 96 and 58.)
__device__ __forceinline__ bool order_rows(int mine, int* order) {
  const int lane = threadIdx.x & 63, above = __shfl_up(mine, 1);
  if (__ballot(lane > 0 && mine < above) == 0) return false;
  if (threadIdx.x < 64) {
    int place = 0;
    for (int j = 0; j < 64; ++j) {
      const int other = __builtin_amdgcn_readlane(mine, j);
      place += other < mine || (other == mine && j < lane);
    }
    order[place] = lane;
  }
  __syncthreads();
  return true;
}

// ---------------------------------------------------------------------------
// shrink: a workgroup takes 16 rows, one of `splits` parts of the contracted axis
// and, of the adapters that the rows meet, every `slots`-th.  Its eight waves
// share these adapters out as far as they go, and the part's steps beyond that.
// Partial sums of the parts lie behind each other in `low`, for expand and
// contract to add in order; a row is written by its adapter's workgroup alone.
//
// 8192 x 2048 BF16, rank 16: 16 us, 6.5 of them bytes; the rest is the chain of
// index, rows, sums and launch (twice as many values of x take 7 us more).  Loads of
// x ahead of the index, and more of them together, are level.  One row of 2048:
// 3.8 us; 64 rows with 32 adapters: 8.4, in one part for the whole axis 10 to 15%
// more, without slots 40%.
// ---------------------------------------------------------------------------
struct ShrinkArgs {
  Adapters g;
  const char* x;
  int64_t ldx, k;
  float* low;  // splits x rows x 16 chunks
  int row_tiles, splits, slot_bits;  // 2^slot_bits slots
};

constexpr int kShrinkWaves = 8;
template <int XE>
constexpr int kShrinkStep = 4 * 32 / enc_bytes(XE);  // values of the contracted axis that a wave takes at once: 128 bytes of a row

// Wave c ends with chunk c's sums of the rows that this workgroup writes: use(row, c, the four of this lane's row from
// rank 4 (lane / 16) of the chunk on).
template <int XE, int RC, class F>
__device__ __forceinline__ void shrink_tile(const ShrinkArgs& s, f32x4 (&sums)[kShrinkWaves][RC][64], int (&order)[64], int tile,
                                            int split, int slot, F&& use) {
  constexpr int kStep = kShrinkStep<XE>, kEights = kStep / kEightSpan;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, q = lane >> 4;
  const int slots = 1 << s.slot_bits;
  // A quarter of 64 rows, which are taken in the order of their adapters where that is another.
  const int64_t row0 = static_cast<int64_t>(tile >> 2) * 64;
  const int all = adapter_of(s.g, row0 + lane);
  int place = (tile & 3) * 16 + i;
  if (row0 + 64 <= s.g.rows && order_rows(all, order)) place = order[place];
  const int64_t row = row0 + place;
  const int mine = __shfl(all, place);
  const char* x = s.x + (row < s.g.rows ? row : s.g.rows - 1) * s.ldx * enc_bytes(XE);
  int met = 0;          // by this workgroup
  bool owned = mine < 0 && slot == 0;  // this lane's row is written here
  for_each_adapter(mine, [&](int adapter, int number) {
    if ((number & (slots - 1)) != slot) return;
    ++met;
    owned |= mine == adapter;
  });
  if (met == 0 && slot > 0) return;
  const int share_bits = met >= 8 ? 0 : (met >= 4 ? 1 : (met >= 2 ? 2 : 3)), shares = 1 << share_bits;  // waves of one adapter

  const int64_t steps = (s.k + kStep - 1) / kStep, part = (steps + s.splits - 1) / s.splits;
  const int64_t begin = split * part, end = begin + part < steps ? begin + part : steps;
  const int64_t each = (part + shares - 1) >> share_bits, first = begin + (wave & (shares - 1)) * each;
  const int64_t last = first + each < end ? first + each : end;
  const int64_t whole = s.k / kStep < last ? s.k / kStep : last;

  f32x4 acc[RC] = {};
  for_each_adapter(mine, [&](int adapter, int number) {
    if ((number & (slots - 1)) != slot || ((number >> s.slot_bits) & ((kShrinkWaves >> share_bits) - 1)) != wave >> share_bits) return;
    const char* rows[RC];
#pragma unroll
    for (int c = 0; c < RC; ++c) {
      const int rank = c * kRankChunk + i;
      rows[c] = s.g.a + (static_cast<int64_t>(adapter) * s.g.rank + (rank < s.g.rank ? rank : s.g.rank - 1)) * s.k * enc_bytes(XE);
    }
    f32x4 sum[RC] = {};
    // So many steps' loads go out together.
    constexpr int kTogether = RC == 1 ? 4 : (RC == 2 ? 2 : 1);
    auto step = [&](int64_t kt, auto together, auto load) {
      constexpr int kSteps = decltype(together)::value;
      Eight<XE> v[kSteps][kEights], m[kSteps][RC][kEights];
#pragma unroll
      for (int u = 0; u < kSteps; ++u)
#pragma unroll
        for (int e = 0; e < kEights; ++e) {
          const int64_t at = (kt + u) * kStep + kEightSpan * e;
          v[u][e] = load(x, at);
#pragma unroll
          for (int c = 0; c < RC; ++c)
            if (c < s.g.chunks) m[u][c][e] = load(rows[c], at);
        }
#pragma unroll
      for (int u = 0; u < kSteps; ++u)
#pragma unroll
        for (int c = 0; c < RC; ++c) {
          if (c < s.g.chunks) {
#pragma unroll
            for (int e = 0; e < kEights; ++e) mma_eight<XE>(sum[c], m[u][c][e], v[u][e]);
          }
        }
    };
    auto inside = [&](const char* p, int64_t c) { return load_eight_whole<XE>(p, c, q); };
    int64_t kt = first;
    for (; kt + kTogether <= whole; kt += kTogether) step(kt, std::integral_constant<int, kTogether>{}, inside);
    for (; kt < whole; ++kt) step(kt, std::integral_constant<int, 1>{}, inside);
    if (whole < last && first <= whole)
      step(whole, std::integral_constant<int, 1>{}, [&](const char* p, int64_t c) { return load_eight_to<XE>(p, c, q, s.k); });
#pragma unroll
    for (int c = 0; c < RC; ++c)
      if (mine == adapter) acc[c] = sum[c];
  });
#pragma unroll
  for (int c = 0; c < RC; ++c) sums[wave][c][lane] = acc[c];
  __syncthreads();
  // Wave c adds chunk c.
  if (wave >= s.g.chunks || !owned || row >= s.g.rows) return;
  f32x4 total = sums[0][wave][lane];
#pragma unroll
  for (int w = 1; w < kShrinkWaves; ++w) total += sums[w][wave][lane];
  const float scale = adapter_scale(s.g, mine);
  const int rank = wave * kRankChunk + 4 * q;
  f32x4 out{};
#pragma unroll
  for (int j = 0; j < 4; ++j) out[j] = mine >= 0 && rank + j < s.g.rank ? total[j] * scale : 0.0f;
  use(row, wave, out);
}

// Part `split` of a row's chunk.
__device__ __forceinline__ void store_low(const ShrinkArgs& s, int64_t row, int split, int chunk, int q, const f32x4& v) {
  *(SR_GLOBAL floats4*)(s.low + (split * s.g.rows + row) * s.g.chunks * kRankChunk + chunk * kRankChunk + 4 * q) =
      floats4{v[0], v[1], v[2], v[3]};
}

template <int XE, int RC>
__global__ __launch_bounds__(64 * kShrinkWaves) void adapter_shrink_kernel(ShrinkArgs s) {
  __shared__ f32x4 sums[kShrinkWaves][RC][64];
  __shared__ int order[64];
  const int tile = blockIdx.x % s.row_tiles, unit = blockIdx.x / s.row_tiles;
  const int slot = unit & ((1 << s.slot_bits) - 1), split = unit >> s.slot_bits, q = (threadIdx.x & 63) >> 4;
  shrink_tile<XE, RC>(s, sums, order, tile, split, slot,
                      [&](int64_t row, int chunk, const f32x4& v) { store_low(s, row, split, chunk, q, v); });
}

// Sixteen ranks of `low` and of the adapters as the products with FP32 values take them.  With BF16, 32 places of the
// contracted axis are the sixteen ranks twice, by the truncated parts and by the rests; else four instructions take four
// ranks each.
template <int XE>
struct Sixteen {
  static constexpr bool kParts = XE == ENC_BF16_RN;
  uint32_t w[4];  // eight BF16 values, or four FP32 ones

  // A lane's part of the 64 bytes that expand lays out for a row of low.
  __device__ __forceinline__ void of_lds(const char* p) {
    const i32x4 v = read_chunk(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = static_cast<uint32_t>(v[j]);
  }

  // Those of a row of b, of which `rank` are there.
  static __device__ __forceinline__ Sixteen of_row(const char* row, int rank, int c, int q) {
    Sixteen s;
    if constexpr (kParts) {
      const int at = c * kRankChunk;
      const Eight<XE> e = at + 16 <= rank ? load_eight_whole<XE>(row, at, q & 1) : load_eight_to<XE>(row, at, q & 1, rank);
#pragma unroll
      for (int j = 0; j < 4; ++j) s.w[j] = e.w[j];
    } else {
      const int at = c * kRankChunk + 4 * q;
      const f32x4 v = load_four<XE>(row + at * enc_bytes(XE), live_four(at, rank));
#pragma unroll
      for (int j = 0; j < 4; ++j) s.w[j] = f32_bits(v[j]);
    }
    return s;
  }

  __device__ __forceinline__ void mma(f32x4& acc, const Sixteen& second) const {
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (kParts) {
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, second.w), acc, 0, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_f32(w[j]), bits_f32(second.w[j]), acc, 0, 0, 0);
    }
#endif
  }
};

// ---------------------------------------------------------------------------
// expand: a workgroup takes TILES times 16 rows, whose `low` it adds up and lays out
// in LDS once; its waves take 16 NT columns each.  Their instructions take the
// rows of b in an order that leaves a lane runs of 16 bytes, four lanes side by side.
// All of base is on its way before anything waits, and the adapter met last
// stays in registers.  Where 64 rows do not come in runs of one adapter they are
// taken in the order of their adapters, so that each adapter is read about once,
// here and in shrink (8192 rows of 8 adapters in any order, 2048 to 2048, rank 16: 96
// us and 58 in all; in runs 27).  With slots so many waves take every slots-th of the
// adapters that 16 rows meet, and write only these rows.
//
// 8192 rows to 8192 columns, rank 16: 58 us, at the rate of a large copy 52.  With
// `low` read by every wave instead of once a workgroup it took 70, and with tiles
// one after the other, each waiting for its own loads, 108.
// ---------------------------------------------------------------------------
struct ExpandArgs {
  Adapters g;  // a: count x n x rank
  const float* low;
  const char* base;  // or null: zeros
  char* out;
  int64_t ldbase, ldout, n;
  int splits, slot_bits;
  int column_tiles;  // of 16 NT
  int blocks;        // of kAdapterWaves column tiles and slots
};

// N neighbouring values of a row as they lie.
template <int XE, int N>
struct Run {
  static constexpr int kWords = N * enc_bytes(XE) / 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const char* p) {
#pragma unroll
    for (int h = 0; h < kWords; h += 4) {
      if constexpr (enc_bytes(XE) == 4) {
        const floats4 v = *(const SR_GLOBAL floats4*)(p + 4 * h);
        __builtin_memcpy(w + h, &v, 16);
      } else if constexpr (kWords >= 4) {
        const halves8 v = *(const SR_GLOBAL halves8*)(p + 4 * h);
        __builtin_memcpy(w + h, &v, 16);
      } else {
        const halves4 v = *(const SR_GLOBAL halves4*)(p);
        __builtin_memcpy(w, &v, 8);
      }
    }
  }
  __device__ __forceinline__ void load(const char* p, int live) {
#pragma unroll
    for (int h = 0; h < kWords; ++h) w[h] = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j < live) {
        if constexpr (enc_bytes(XE) == 2) w[j >> 1] |= static_cast<uint32_t>(gptr<uint16_t>(p)[j]) << (16 * (j & 1));
        else w[j] = gptr<uint32_t>(p)[j];
      }
    }
  }
  __device__ __forceinline__ float value(int j) const {
    if constexpr (enc_bytes(XE) == 4) return bits_f32(w[j]);
    else if constexpr (XE == ENC_BF16_RN) return bits_f32(j & 1 ? w[j >> 1] & 0xFFFF0000u : w[j >> 1] << 16);
    else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)))));
  }
  __device__ __forceinline__ void set(int j, float lo, float hi) {  // values j and j + 1, j even
    if constexpr (enc_bytes(XE) == 4) {
      w[j] = f32_bits(lo);
      w[j + 1] = f32_bits(hi);
    } else if constexpr (XE == ENC_BF16_RN) {
      w[j >> 1] = pack_bf16(lo, hi);
    } else {
      w[j >> 1] = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(lo))) |
                  static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(hi))) << 16;
    }
  }
  __device__ __forceinline__ void store(char* p) const {
#pragma unroll
    for (int h = 0; h < kWords; h += 4) {
      if constexpr (enc_bytes(XE) == 4)
        *(SR_GLOBAL floats4*)(p + 4 * h) = floats4{bits_f32(w[h]), bits_f32(w[h + 1]), bits_f32(w[h + 2]), bits_f32(w[h + 3])};
      else if constexpr (kWords >= 4) *(SR_GLOBAL halves8*)(p + 4 * h) = halves8{w[h], w[h + 1], w[h + 2], w[h + 3]};
      else *(SR_GLOBAL halves4*)(p) = halves4{w[0], w[1]};
    }
  }
  __device__ __forceinline__ void store(char* p, int live) const {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j < live) {
        if constexpr (enc_bytes(XE) == 2) gptr_mut<uint16_t>(p)[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
        else gptr_mut<uint32_t>(p)[j] = w[j];
      }
    }
  }
};

constexpr int kLowBytes = 64;  // of 16 ranks of a row in LDS

// Lays four values of a row's `low`, from rank `rank` of their chunk on, out for Sixteen::of_lds.
template <int XE>
__device__ __forceinline__ void put_low(char* chunk, int rank, const f32x4& v) {
  if constexpr (Sixteen<XE>::kParts) {
    // Sixteen truncated parts, then the sixteen rests.
    uint32_t* w = reinterpret_cast<uint32_t*>(chunk + 2 * rank);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const TwoParts lo(v[2 * h]), hi(v[2 * h + 1]);
      w[h] = upper_halves(lo.upper, hi.upper);
      w[8 + h] = pack_bf16(lo.rest, hi.rest);
    }
  } else {
    *reinterpret_cast<f32x4*>(chunk + 4 * rank) = v;
  }
}

// 16 NT columns of a wave: a lane's are kRuns runs of kRun, each beside those of its row's other three lanes.
template <int XE, int RC, int NT>
struct Columns {
  static constexpr int kSize = enc_bytes(XE), kRun = NT == 1 ? 4 : 16 / kSize, kRuns = 4 * NT / kRun;
  using Base = Run<XE, kRun>[kRuns];
  int64_t n0, col;
  bool edge;
  int held;
  Sixteen<XE> b[NT][RC];

  __device__ __forceinline__ void start(const ExpandArgs& s, int64_t first, int q) {
    n0 = first;
    col = n0 + q * kRun;
    edge = n0 + 16 * NT > s.n;
    held = -1;
  }
  __device__ __forceinline__ int live(const ExpandArgs& s, int run) const {
    const int64_t at = col + 4 * run * kRun;
    return at >= s.n ? 0 : (s.n - at < kRun ? static_cast<int>(s.n - at) : kRun);
  }
  __device__ __forceinline__ void load(const ExpandArgs& s, int64_t row, Base& base) const {
    if (!s.base) return;
    const char* p = s.base + ((row < s.g.rows ? row : s.g.rows - 1) * s.ldbase + col) * kSize;
    if (edge) {
#pragma unroll
      for (int run = 0; run < kRuns; ++run) base[run].load(p + 4 * run * kRun * kSize, live(s, run));
    } else {
#pragma unroll
      for (int run = 0; run < kRuns; ++run) base[run].load(p + 4 * run * kRun * kSize);
    }
  }
  __device__ __forceinline__ void hold(const ExpandArgs& s, int adapter, int i, int q) {
    if (adapter == held) return;
    held = adapter;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      // Four of the run's columns, as result rows 4 q .. 4 q + 3 of the instruction.
      constexpr int kFours = kRun / 4;
      const int64_t n = n0 + t / kFours * 4 * kRun + (i >> 2) * kRun + t % kFours * 4 + (i & 3);
      const char* row = s.g.a + (static_cast<int64_t>(adapter) * s.n + (n < s.n ? n : s.n - 1)) * s.g.rank * kSize;
#pragma unroll
      for (int c = 0; c < RC; ++c)
        if (c < s.g.chunks) b[t][c] = Sixteen<XE>::of_row(row, s.g.rank, c, q);
    }
  }
  // The results of 16 rows; `low`: this lane's row in LDS.
  __device__ __forceinline__ void results(const ExpandArgs& s, int64_t row, int mine, const char* low_row, const Base& base,
                                          uint32_t slot, int i, int q) {
    const uint32_t slots = 1u << s.slot_bits;
    f32x4 sum[NT] = {};
    bool owned = mine < 0 && slot == 0;
    for_each_adapter(mine, [&](int adapter, int number) {
      if ((number & (slots - 1)) != slot) return;
      hold(s, adapter, i, q);
      owned |= mine == adapter;
      Sixteen<XE> low[RC];
#pragma unroll
      for (int c = 0; c < RC; ++c)
        if (c < s.g.chunks) low[c].of_lds(low_row + c * kLowBytes + 16 * q);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 part = {};
#pragma unroll
        for (int c = 0; c < RC; ++c)
          if (c < s.g.chunks) b[t][c].mma(part, low[c]);
        if (mine == adapter) sum[t] = part;
      }
    });
    if (!owned || row >= s.g.rows) return;
    char* p = s.out + (row * s.ldout + col) * kSize;
#pragma unroll
    for (int run = 0; run < kRuns; ++run) {
      Run<XE, kRun> out = base[run];
      if (!s.base || mine >= 0) {
#pragma unroll
        for (int j = 0; j < kRun; j += 2) {
          const int at = run * kRun + j;
          const float lo = sum[at >> 2][at & 3], hi = sum[at >> 2][(at & 3) + 1];
          if (s.base) out.set(j, base[run].value(j) + lo, base[run].value(j + 1) + hi);
          else out.set(j, lo, hi);
        }
      }
      if (edge) out.store(p + 4 * run * kRun * kSize, live(s, run));
      else out.store(p + 4 * run * kRun * kSize);
    }
  }
};

template <int XE, int RC, int NT, int TILES>
__global__ __launch_bounds__(kAdapterThreads) void adapter_expand_kernel(ExpandArgs s) {
  constexpr int kRows = 16 * TILES;
  __shared__ __align__(16) char lows[kRows * RC * kLowBytes];
  __shared__ int indices[kRows], order[kRows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, q = lane >> 4;
  const uint32_t group = blockIdx.x / s.blocks, unit = (blockIdx.x - group * s.blocks) * kAdapterWaves + wave;
  const uint32_t slot = unit & ((1u << s.slot_bits) - 1);
  const int64_t row0 = static_cast<int64_t>(group) * kRows;
  Columns<XE, RC, NT> columns;
  columns.start(s, static_cast<int64_t>(unit >> s.slot_bits) * 16 * NT, q);

  typename Columns<XE, RC, NT>::Base base[TILES];
#pragma unroll
  for (int tile = 0; tile < TILES; ++tile) columns.load(s, row0 + tile * 16 + i, base[tile]);
  const int64_t width = s.g.chunks * kRankChunk, stride = s.g.rows * width;
  if (threadIdx.x < kRows) indices[threadIdx.x] = adapter_of(s.g, row0 + threadIdx.x);
  // Four values at a time, all of the group's rows side by side.
  const int64_t fours = (s.g.rows - row0 < kRows ? s.g.rows - row0 : kRows) * width / 4;
  for (int64_t at = threadIdx.x; at < fours; at += kAdapterThreads) {
    const float* from = s.low + row0 * width + 4 * at;
    const floats4 v = *(const SR_GLOBAL floats4*)(from);
    f32x4 sum{v[0], v[1], v[2], v[3]};
    for (int p = 1; p < s.splits; ++p) {
      const floats4 more = *(const SR_GLOBAL floats4*)(from + p * stride);
      sum += f32x4{more[0], more[1], more[2], more[3]};
    }
    const int row = static_cast<int>(4 * at / width), place = static_cast<int>(4 * at - row * width);
    put_low<XE>(lows + (row * RC + place / kRankChunk) * kLowBytes, place % kRankChunk, sum);
  }
  __syncthreads();
  bool mixed = false;
  if constexpr (kRows == 64) mixed = order_rows(indices[lane], order);
  if (columns.n0 >= s.n) return;
  int rows[TILES];
#pragma unroll
  for (int tile = 0; tile < TILES; ++tile) {
    rows[tile] = mixed ? order[tile * 16 + i] : tile * 16 + i;
    if (mixed) columns.load(s, row0 + rows[tile], base[tile]);
  }
#pragma unroll
  for (int tile = 0; tile < TILES; ++tile)
    columns.results(s, row0 + rows[tile], indices[rows[tile]], lows + rows[tile] * RC * kLowBytes, base[tile], slot, i, q);
}

// ---------------------------------------------------------------------------
// Both in one, for a few rows: every workgroup goes through the rows' adapters by
// itself, and on to 16 columns a wave.  One launch; the adapters' a comes from the
// caches after the first (one row of 2048 to 2048, rank 8: 7.4 us a call, 9.6 in two).
// ---------------------------------------------------------------------------
struct FewArgs {
  ShrinkArgs down;  // in one part
  ExpandArgs up;
  int parts;        // of `low` as a backward pass adds them up: all but the first become zeros
};

template <int XE, int RC>
__global__ __launch_bounds__(64 * kShrinkWaves) void adapter_few_kernel(FewArgs s) {
  __shared__ f32x4 sums[kShrinkWaves][RC][64];
  __shared__ int order[64];
  __shared__ __align__(16) char lows[16 * RC * kLowBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, q = lane >> 4;
  Columns<XE, RC, 1> columns;
  typename Columns<XE, RC, 1>::Base base;
  columns.start(s.up, (static_cast<int64_t>(blockIdx.x) * kShrinkWaves + wave) * 16, q);
  columns.load(s.up, i, base);
  shrink_tile<XE, RC>(s.down, sums, order, 0, 0, 0, [&](int64_t row, int chunk, const f32x4& v) {
    put_low<XE>(lows + (row * RC + chunk) * kLowBytes, 4 * q, v);
    if (blockIdx.x == 0) {
      store_low(s.down, row, 0, chunk, q, v);
      for (int part = 1; part < s.parts; ++part) store_low(s.down, row, part, chunk, q, f32x4{});
    }
  });
  __syncthreads();
  if (columns.n0 < s.up.n) columns.results(s.up, i, adapter_of(s.up.g, i), lows + i * RC * kLowBytes, base, 0, i, q);
}

// ---------------------------------------------------------------------------
// contract: out[i][r][c] = sum over the rows t of adapter i of low[t][r] x[t][c].
//
// A workgroup takes an adapter, 16 CJ columns and one part of the rows.  It
// first lists the part's rows that are the adapter's, in order; its waves then
// take 32 of them at a time in turn, turned in registers so that rows are the
// contracted axis, and add their sums in wave order.  Parts leave FP32 sums
// and whether they had rows at all, for `finish` to add in order.
//
// 8191 rows by 2048 and 2304 columns, rank 32, 4 adapters: 30 us for 71 MB (14 at a copy's
// rate); 50 without the next rows' loads under this step's products.  Without
// parts one adapter of all rows takes 113 us a backward pass and not 59.
// ---------------------------------------------------------------------------
struct ContractOperand {
  const float* low;  // splits x rows x 16 chunks
  int splits;
  const char* x;
  int64_t ldx, cols;
  char* out;         // count x rank x cols, or count x cols x rank where `turned`
  float* partial;    // parts x count x (16 chunks) x cols
  int turned;
  int tiles;         // of 16 CJ columns
};

struct ContractArgs {
  Adapters g;
  ContractOperand op[2];
  int parts;             // 1: results go straight to out
  int64_t part_rows;     // a multiple of kListRows
  int* filled;           // parts x count
};

constexpr int kListRows = 1024;

// Eight rows of CJ columns, and their transpose: CJ eights of one column each.
template <int XE, int CJ>
struct Turned {
  static constexpr int kWords = CJ * enc_bytes(XE) / 4;
  Run<XE, CJ> rows[8];

  __device__ __forceinline__ uint32_t word(int e, int h) const { return rows[e].w[h]; }
  __device__ __forceinline__ void clear(int e) {
#pragma unroll
    for (int h = 0; h < kWords; ++h) rows[e].w[h] = 0;
  }
  // Column j of all eight rows as BF16 pairs.
  __device__ __forceinline__ void halves(int j, uint32_t (&w)[4]) const {
#pragma unroll
    for (int p = 0; p < 4; ++p)
      w[p] = j & 1 ? upper_halves(word(2 * p, j >> 1), word(2 * p + 1, j >> 1)) : lower_halves(word(2 * p, j >> 1), word(2 * p + 1, j >> 1));
  }
  // Column j of row e as FP32.
  __device__ __forceinline__ float value(int j, int e) const { return rows[e].value(j); }
};

template <int XE, int RC, int CJ>
__global__ __launch_bounds__(kAdapterThreads) void adapter_contract_kernel(ContractArgs s) {
  constexpr int kSize = enc_bytes(XE);
  constexpr bool kParts = XE == ENC_BF16_RN;
  __shared__ __align__(16) uint32_t list[kListRows];  // rows past `at`; behind its end the first row, for loads that nothing uses
  __shared__ uint32_t counts[kAdapterWaves];
  __shared__ f32x4 sums[CJ * RC][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, q = lane >> 4;
  uint32_t id = blockIdx.x;
  const uint32_t tiles = s.op[0].tiles + s.op[1].tiles;
  const uint32_t part = id / (tiles * s.g.count);
  id -= part * tiles * s.g.count;
  const int adapter = static_cast<int>(id / tiles);
  id -= adapter * tiles;
  const bool second = id >= static_cast<uint32_t>(s.op[0].tiles);
  const ContractOperand& op = s.op[second];
  const int64_t c0 = static_cast<int64_t>(second ? id - s.op[0].tiles : id) * 16 * CJ + i * CJ;  // this lane's first column
  const int live = c0 >= op.cols ? 0 : (op.cols - c0 < CJ ? static_cast<int>(op.cols - c0) : CJ);
  const bool edge = c0 - i * CJ + 16 * CJ > op.cols;
  const int64_t width = s.g.chunks * kRankChunk, stride = s.g.rows * width;
  const int64_t begin = part * s.part_rows, end = begin + s.part_rows < s.g.rows ? begin + s.part_rows : s.g.rows;

  f32x4 acc[CJ][RC] = {};
  bool any = false;
  for (int64_t at = begin; at < end; at += kListRows) {
    // Each thread looks at four neighbouring rows.
    constexpr int kOwn = kListRows / kAdapterThreads;
    uint32_t own = 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      const int64_t row = at + threadIdx.x * kOwn + j;
      if (row < end && adapter_of(s.g, row) == adapter) own |= 1u << j;
    }
    uint32_t before = __builtin_popcount(own);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t up = static_cast<uint32_t>(__shfl_up(static_cast<int>(before), d));
      if (lane >= d) before += up;
    }
    __syncthreads();  // the list of before is done with
    if (lane == 63) counts[wave] = before;
    __syncthreads();
    uint32_t total = 0, place = before - __builtin_popcount(own);
#pragma unroll
    for (int w = 0; w < kAdapterWaves; ++w) {
      if (w < wave) place += counts[w];
      total += counts[w];
    }
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
      if (own >> j & 1) list[place++] = threadIdx.x * kOwn + j;
    for (uint32_t k = total + threadIdx.x; k < (total + 31) / 32 * 32; k += kAdapterThreads) list[k] = 0;
    __syncthreads();
    any |= total > 0;

    struct Step {
      Turned<XE, CJ> x;
      float low[RC][8];
    };
    auto fetch = [&](uint32_t first, Step& step) {
      uint32_t places[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const i32x4 v = read_chunk(reinterpret_cast<const char*>(list + first + q * 8 + 4 * h));
#pragma unroll
        for (int j = 0; j < 4; ++j) places[4 * h + j] = static_cast<uint32_t>(v[j]);
      }
      const char* from = op.x + (at * op.ldx + c0) * kSize;
      if (edge) {
#pragma unroll
        for (int e = 0; e < 8; ++e) step.x.rows[e].load(from + places[e] * op.ldx * kSize, live);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) step.x.rows[e].load(from + places[e] * op.ldx * kSize);
      }
      const float* low = op.low + at * width + i;
#pragma unroll
      for (int c = 0; c < RC; ++c)
        if (c < s.g.chunks) {
#pragma unroll
          for (int e = 0; e < 8; ++e) step.low[c][e] = *gptr<float>(low + places[e] * width + c * kRankChunk);
        }
      for (int k = 1; k < op.splits; ++k)
#pragma unroll
        for (int c = 0; c < RC; ++c)
          if (c < s.g.chunks) {
#pragma unroll
            for (int e = 0; e < 8; ++e) step.low[c][e] += *gptr<float>(low + k * stride + places[e] * width + c * kRankChunk);
          }
    };
    auto use = [&](uint32_t first, Step& step) {
      if (first + 32 > total) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (first + q * 8 + e < total) continue;
          step.x.clear(e);
#pragma unroll
          for (int c = 0; c < RC; ++c) step.low[c][e] = 0;
        }
      }
      if constexpr (kParts) {
        Eight<XE> upper[RC], rest[RC];
#pragma unroll
        for (int c = 0; c < RC; ++c)
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const TwoParts lo(step.low[c][2 * p]), hi(step.low[c][2 * p + 1]);
            upper[c].w[p] = upper_halves(lo.upper, hi.upper);
            rest[c].w[p] = pack_bf16(lo.rest, hi.rest);
          }
#pragma unroll
        for (int j = 0; j < CJ; ++j) {
          Eight<XE> column;
          step.x.halves(j, column.w);
#pragma unroll
          for (int c = 0; c < RC; ++c) {
            if (c < s.g.chunks) {
              mma_eight<XE>(acc[j][c], upper[c], column);
              mma_eight<XE>(acc[j][c], rest[c], column);
            }
          }
        }
      } else {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int j = 0; j < CJ; ++j) {
            const float v = step.x.value(j, e);
#pragma unroll
            for (int c = 0; c < RC; ++c)
              if (c < s.g.chunks) acc[j][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(step.low[c][e], v, acc[j][c], 0, 0, 0);
          }
#endif
      }
    };
    // A step's loads run under the products of the one before, where the sums leave registers for both.
    constexpr uint32_t kStride = 32 * kAdapterWaves;
    uint32_t first = wave * 32;
    if constexpr (RC <= 2) {
      Step even, odd;
      if (first < total) fetch(first, even);
      for (; first < total; first += 2 * kStride) {
        if (first + kStride < total) fetch(first + kStride, odd);
        use(first, even);
        if (first + 2 * kStride < total) fetch(first + 2 * kStride, even);
        if (first + kStride < total) use(first + kStride, odd);
      }
    } else {
      for (; first < total; first += kStride) {
        Step step;
        fetch(first, step);
        use(first, step);
      }
    }
  }

  for (int w = 1; w < kAdapterWaves; ++w) {
    __syncthreads();
    if (wave == w) {
#pragma unroll
      for (int j = 0; j < CJ; ++j)
#pragma unroll
        for (int c = 0; c < RC; ++c) sums[j * RC + c][lane] = acc[j][c];
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int j = 0; j < CJ; ++j)
#pragma unroll
        for (int c = 0; c < RC; ++c) acc[j][c] += sums[j * RC + c][lane];
    }
  }
  if (wave > 0) return;
  if (s.parts > 1) {
    if (c0 == 0 && !second && q == 0) s.filled[part * s.g.count + adapter] = any;
    if (!any) return;
    float* to = op.partial + (static_cast<int64_t>(part) * s.g.count + adapter) * width * op.cols;
#pragma unroll
    for (int c = 0; c < RC; ++c) {
      if (c >= s.g.chunks) break;
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < CJ; j += 4)
          store_four<ENC_F32>(reinterpret_cast<char*>(to + (c * kRankChunk + 4 * q + e) * op.cols + c0 + j),
                              f32x4{acc[j][c][e], acc[j + 1][c][e], acc[j + 2][c][e], acc[j + 3][c][e]}, live_four(c0 + j, op.cols));
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < RC; ++c) {
    if (c >= s.g.chunks) break;
    const int rank = c * kRankChunk + 4 * q;
    if (op.turned) {
#pragma unroll
      for (int j = 0; j < CJ; ++j)
        if (j < live)
          store_four<XE>(op.out + ((adapter * op.cols + c0 + j) * s.g.rank + rank) * kSize, acc[j][c], live_four(rank, s.g.rank));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (rank + e < s.g.rank) {
#pragma unroll
          for (int j = 0; j < CJ; j += 4)
            store_four<XE>(op.out + ((static_cast<int64_t>(adapter) * s.g.rank + rank + e) * op.cols + c0 + j) * kSize,
                           f32x4{acc[j][c][e], acc[j + 1][c][e], acc[j + 2][c][e], acc[j + 3][c][e]}, live_four(c0 + j, op.cols));
        }
    }
  }
}

// Threads that finish an operand's results.
inline __host__ __device__ int64_t finish_items(const Adapters& g, const ContractOperand& op) {
  if (!op.out) return 0;
  return g.count * (op.turned ? op.cols * ((g.rank + 3) / 4) : (op.cols + 3) / 4 * g.rank);
}

// Adds the parts' sums: a thread takes four columns of one rank, or of a turned result four ranks of one column.
template <int XE>
__global__ __launch_bounds__(256) void adapter_finish_kernel(ContractArgs s) {
  const int64_t width = s.g.chunks * kRankChunk;
  int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t firsts = finish_items(s.g, s.op[0]);
  if (id >= firsts + finish_items(s.g, s.op[1])) return;  // an operand that is not there has no sizes to divide by
  const bool second = id >= firsts;
  if (second) id -= firsts;
  const ContractOperand& op = s.op[second];
  const int64_t quads = (op.cols + 3) / 4, ranks = (s.g.rank + 3) / 4;
  int64_t adapter, rank, col;
  if (op.turned) {
    // Neighbouring threads take neighbouring columns, whose partial sums lie side by side.
    col = id % op.cols;
    rank = id / op.cols % ranks * 4;
    adapter = id / op.cols / ranks;
  } else {
    col = id % quads * 4;
    rank = id / quads % s.g.rank;
    adapter = id / quads / s.g.rank;
  }
  // Eight parts' loads go out together; what a part without rows holds means nothing.
  constexpr int kTogether = 8;
  f32x4 sum{};
  const int live = live_four(col, op.cols);
  for (int first = 0; first < s.parts; first += kTogether) {
    f32x4 values[kTogether];
    int filled[kTogether];
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      const int64_t p = first + j < s.parts ? first + j : s.parts - 1;
      filled[j] = gptr<int>(s.filled)[p * s.g.count + adapter];
      const float* from = op.partial + ((p * s.g.count + adapter) * width + rank) * op.cols + col;
      if (op.turned) {
#pragma unroll
        for (int e = 0; e < 4; ++e) values[j][e] = *gptr<float>(from + e * op.cols);  // ranks up to `width` are there
      } else {
        // The places of the last column stand in for those behind it.
#pragma unroll
        for (int e = 0; e < 4; ++e) values[j][e] = *gptr<float>(from + (e < live ? e : live - 1));
      }
    }
#pragma unroll
    for (int j = 0; j < kTogether; ++j)
      if (first + j < s.parts && filled[j]) sum += values[j];
  }
  if (op.turned)
    store_four<XE>(op.out + ((adapter * op.cols + col) * s.g.rank + rank) * enc_bytes(XE), sum, live_four(rank, s.g.rank));
  else
    store_four<XE>(op.out + ((adapter * s.g.rank + rank) * op.cols + col) * enc_bytes(XE), sum, live_four(col, op.cols));
}

// ---------------------------------------------------------------------------
// The adapters turned, for the input's gradient: to[i][c][r] = from[i][r][c], tiles of 64 x 64 through LDS.
// ---------------------------------------------------------------------------
struct TurnOperand {
  const char* from;
  char* to;
  int64_t rows, cols;
  int tiles_n;
  uint32_t tiles;  // of all matrices
};

struct TurnArgs {
  TurnOperand op[2];
};

template <int SIZE>
__global__ __launch_bounds__(256) void adapter_turn_kernel(TurnArgs s) {
  using T = std::conditional_t<SIZE == 4, uint32_t, uint16_t>;
  __shared__ T tile[64][64 + 4 / SIZE];
  const bool second = blockIdx.x >= s.op[0].tiles;
  const TurnOperand& op = s.op[second];
  const uint32_t id = blockIdx.x - (second ? s.op[0].tiles : 0);
  const uint32_t tiles_m = static_cast<uint32_t>((op.rows + 63) / 64), each = tiles_m * op.tiles_n;
  const uint32_t matrix = id / each, within = id - matrix * each;
  const int64_t r0 = static_cast<int64_t>(within / op.tiles_n) * 64, c0 = static_cast<int64_t>(within % op.tiles_n) * 64;
  const T* from = reinterpret_cast<const T*>(op.from) + matrix * op.rows * op.cols;
  T* to = reinterpret_cast<T*>(op.to) + matrix * op.rows * op.cols;
  const int column = threadIdx.x & 63, first = threadIdx.x >> 6;
  // Places past the matrix's edges repeat its last ones, so that no load waits for a condition.
  const int64_t col = c0 + column < op.cols ? c0 + column : op.cols - 1;
  T values[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int64_t row = r0 + 4 * r + first;
    values[r] = gptr<T>(from)[(row < op.rows ? row : op.rows - 1) * op.cols + col];
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) tile[4 * r + first][column] = values[r];
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 64; c += 4)
    if (c0 + c + first < op.cols && r0 + column < op.rows) gptr_mut<T>(to)[(c0 + c + first) * op.rows + r0 + column] = tile[column][c + first];
}

}  // namespace sr
