// sr_newton_schulz.h -- kernels of the Newton-Schulz orthogonalisation and of the Muon update around it.
//
// The iteration.  X0 = V / (|V|_F + eps), then X <- a X + (b G + c G^2) X with
// G = X X^T, on the orientation with at most as many rows (m) as columns (n).
// G and P = b G + c G^2 are symmetric, so only the tiles of their lower
// triangle are computed and each is stored twice.
//
// Numbers.  The products take FP16 operands and sum in FP32.  Every operand
// is held times 2^13: singular values stay near 1, so entries are at most a
// few units and typical ones 1/sqrt(mn), and 2^13 puts both inside FP16's
// normal range.  X itself is carried in FP32 beside its FP16 copy H:
//
//   X' = a X + P H
//
// A rounding error of X that lies in the space of small singular values
// grows by a (about 3.4) in every step; with a X exact to FP32, the error of
// H meets P instead, which is near 0 there.  (On a rank-16 matrix with noise
// of 1e-3, the result's error in the Frobenius norm is 4e-4; with X held in
// FP16 alone it is 4e-2.)  P is stored as P + s I with s = 1.5, and s H is
// subtracted in FP32: on the large singular values P lies between -3 and 0,
// and half the magnitude halves the rounding of its diagonal.
//
// The norm.  Squares of FP32 values need twice its exponents (a norm above 1.8e19
// would overflow, values below 1e-23 would vanish), so they are summed in
// FP64, and X is V 2^-h times a factor near one, 2^h being the norm's power of two.
//
// Workspace.  Rows and columns are padded to multiples of 64 with zeros, which
// every step keeps, so the products have no edges along their contracted
// axis.  Per padded element: X in FP32, H, and two buffers of H^T, which one
// step reads while it writes the other.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/sr_matrix_hip.h"
#include "sr_kernels.h"
#include "sr_tile_product.h"

namespace sr {

constexpr float kNsScale = 8192.0f, kNsInverse = 1.0f / 8192.0f;  // 2^13
constexpr float kNsProduct = kNsInverse * kNsInverse;             // of a product of two scaled operands
constexpr float kNsShift = 1.5f;
constexpr int kNsPad = 64;        // rows and columns of the workspace are padded to it
constexpr int kNsPartials = 256;  // partial sums of squares per matrix
constexpr int kNsThreads = 256;
constexpr int kNsLoadThreads = 1024;

// The matrices of one launch.
struct MatrixTable {
  uint64_t p[SR_MATRIX_BATCH];  // parameters, or results
  uint64_t g[SR_MATRIX_BATCH];  // gradients, or inputs
  uint64_t u[SR_MATRIX_BATCH];  // momenta
  uint32_t counter[SR_MATRIX_BATCH];
};

struct NsArgs {
  int rows, cols;  // of the matrices
  int m, n;        // padded: m <= n, X is m x n, transposed where rows > cols
  int tall;
  int partials;    // partial sums per matrix in use
  int keep;        // the first kernel writes V
  float a, b, c, eps;
  float* x;
  _Float16* h;
  const _Float16* ht;
  _Float16* ht_next;
  _Float16* g;
  _Float16* p;
  double* partial;
  float momentum, decay, neg_lr;  // Muon
  int nesterov;
  int muon, out_dtype;  // last step: update p in out_dtype, or store the result
};

// Sum over the workgroup's THREADS threads, in a fixed order; the same in all of them.
template <int THREADS>
__device__ __forceinline__ double group_sum(double v, double* scratch) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  v = scratch[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) v += scratch[w];
  return v;
}

// What divides V, from the sum of its squares: V / (|V|_F + eps) = (V 2^-shift) * factor.
struct NsDivisor {
  int shift;
  float factor;
  __device__ __forceinline__ float operator()(float v) const { return ldexpf(v, -shift) * factor; }
};

// The sum is a normal number of FP64, 0, infinite or NaN.  A divisor of 0 has only zeros to divide, which stay.
__device__ __forceinline__ NsDivisor ns_divisor(double sum, float eps) {
  uint64_t bits;
  __builtin_memcpy(&bits, &sum, 8);
  const int exponent = static_cast<int>(bits >> 52) & 0x7FF;
  int h = 0;
  if (exponent != 0 && exponent != 0x7FF) {  // sum = [1, 4) 2^2h
    h = (exponent - 1023) >> 1;
    bits -= static_cast<uint64_t>(static_cast<int64_t>(2 * h)) << 52;
    __builtin_memcpy(&sum, &bits, 8);
  }
  const float divisor = sqrtf(static_cast<float>(sum)) + ldexpf(eps, -h);
  return {h, divisor == 0.0f ? 0.0f : 1.0f / divisor};
}

// How many of the columns col .. col + 3 of row `row` the caller's matrices have.
__device__ __forceinline__ int live_four(const NsArgs& a, int row, int col) {
  return row >= a.rows || col >= a.cols ? 0 : (a.cols - col < 4 ? a.cols - col : 4);
}

// The values of columns col .. col + 3 of row `row` of a matrix of the
// caller's with encoding E; zeros outside.  Without a branch per lane, at whose
// end each load would wait for memory by itself: what passes the edges is
// read where it still fits and shifted (1023 x 767 took 3 us longer with branches).
template <int E>
__device__ __forceinline__ f32x4 load_four(const NsArgs& a, const void* from, int row, int col) {
  const int live = live_four(a, row, col);
  f32x4 v{};
  if (a.cols < 4) {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < live) v[j] = decode<E>(load1<E>(from, static_cast<int64_t>(row) * a.cols + col + j));
    return v;
  }
  const int at_row = row < a.rows ? row : a.rows - 1, at_col = col < a.cols - 4 ? col : a.cols - 4, shift = col - at_col;
  uint32_t w[group_words(E)];
  float r[4];
  load_group<E>(from, static_cast<int64_t>(at_row) * a.cols + at_col, w);
  decode_group<E>(w, r);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float x = 0.0f;
#pragma unroll
    for (int s = 3; s >= 0; --s)
      if (j + s < 4) x = shift == s ? r[j + s] : x;
    v[j] = j < live ? x : 0.0f;
  }
  return v;
}

// Loads what the kernel will need of its arguments at once: they may lie in
// host memory, where each load that waits by itself costs a microsecond or two.
__device__ __forceinline__ void need_arguments(const NsArgs& a) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" ::"s"(a.m), "s"(a.n), "s"(a.a), "s"(a.b), "s"(a.c), "s"(a.x), "s"(a.h), "s"(a.ht), "s"(a.ht_next),
               "s"(a.g), "s"(a.p));
#endif
}

__device__ __forceinline__ void need_arguments(const NsArgs& a, const MatrixTable& t, int matrix) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" ::"s"(a.m), "s"(a.n), "s"(a.rows), "s"(a.cols), "s"(a.tall), "s"(a.keep), "s"(a.partials), "s"(a.eps),
               "s"(a.x), "s"(a.h), "s"(a.ht_next), "s"(a.partial), "s"(a.momentum), "s"(a.nesterov), "s"(t.g[matrix]),
               "s"(t.u[matrix]), "s"(t.counter[matrix]));
#endif
}

// Partial sums of the squares of V, which is the gradient (GE) or, with
// UE >= 0, what the momentum update makes of it; V itself in FP32, in the
// workspace's orientation, where a.keep asks for it.  64 x 64 tiles, of which a
// workgroup takes every gridDim.x-th; a tile's loads come before its stores,
// which might change what a later load reads for all that the compiler knows.
template <int GE, int UE>
__global__ __launch_bounds__(kNsLoadThreads) void ns_load_kernel(NsArgs a, MatrixTable t) {
  __shared__ float turned[kNsPad][kNsPad + 1];
  __shared__ double scratch[kNsLoadThreads / 64];
  constexpr int kRows = kNsLoadThreads / 16, kPasses = kNsPad / kRows;
  const int matrix = blockIdx.y;
  need_arguments(a, t, matrix);
  const void* g = reinterpret_cast<const void*>(t.g[matrix]);
  void* u = reinterpret_cast<void*>(t.u[matrix]);
  float* x = a.x + static_cast<int64_t>(matrix) * a.m * a.n;
  const int tiles_c = (a.tall ? a.m : a.n) / kNsPad, tiles = (a.m / kNsPad) * (a.n / kNsPad);
  const int tr = threadIdx.x >> 4, tc = 4 * (threadIdx.x & 15);
  double sum = 0.0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int r0 = tile / tiles_c * kNsPad, c = tile % tiles_c * kNsPad + tc;
    f32x4 v[kPasses], old[kPasses];
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
      const int r = r0 + kRows * pass + tr;
      v[pass] = load_four<GE>(a, g, r, c);
      if constexpr (UE >= 0) old[pass] = load_four<UE>(a, u, r, c);
    }
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
      const int r = r0 + kRows * pass + tr;
      if constexpr (UE >= 0) {
        const int64_t i = static_cast<int64_t>(r) * a.cols + c;
        const uint32_t counter = t.counter[matrix] + static_cast<uint32_t>(i);
        const int live = live_four(a, r, c);
        float uv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float gv = v[pass][j];
          uv[j] = old[pass][j] * a.momentum + gv;
          v[pass][j] = j < live ? (a.nesterov ? uv[j] * a.momentum + gv : uv[j]) : 0.0f;
        }
        if (live == 4) {
          uint32_t w[group_words(UE)];
          encode_group<UE>(uv, counter, w);
          store_group<UE>(u, i, w);
        } else {
#pragma unroll
          for (int j = 0; j < 3; ++j)
            if (j < live) store1<UE>(u, i + j, encode<UE>(uv[j], counter + static_cast<uint32_t>(j)));
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = fma(static_cast<double>(v[pass][j]), static_cast<double>(v[pass][j]), sum);
      if (!a.keep) continue;
      if (a.tall) {
#pragma unroll
        for (int j = 0; j < 4; ++j) turned[tc + j][kRows * pass + tr] = v[pass][j];
      } else {
        *reinterpret_cast<f32x4*>(x + static_cast<int64_t>(r) * a.n + c) = v[pass];
      }
    }
    if (a.keep && a.tall) {
      __syncthreads();
#pragma unroll
      for (int pass = 0; pass < kPasses; ++pass) {
        const int row = kRows * pass + tr;
        *reinterpret_cast<f32x4*>(x + static_cast<int64_t>(c - tc + row) * a.n + r0 + tc) =
            f32x4{turned[row][tc], turned[row][tc + 1], turned[row][tc + 2], turned[row][tc + 3]};
      }
      __syncthreads();
    }
  }
  sum = group_sum<kNsLoadThreads>(sum, scratch);
  if (threadIdx.x == 0) a.partial[matrix * kNsPartials + blockIdx.x] = sum;
}

// X = V / (|V|_F + eps) and its FP16 copies H and H^T, one 64 x 64 tile per
// workgroup.  V comes from the caller's matrices (GE), which is less to read
// and spares writing it in FP32 first, or with GE < 0 from X.  Bound by memory:
// 8192 x 2048 BF16 takes 18 us for the sum and 36 for the rest (168 MB, 4.7
// TB/s); 40 and 31 where the first wrote V for the second.
template <int GE>
__global__ __launch_bounds__(kNsThreads) void ns_scale_kernel(NsArgs a, MatrixTable t) {
  __shared__ float turned[kNsPad][kNsPad + 1];
  __shared__ double scratch[4];
  const int matrix = blockIdx.y;
  need_arguments(a, t, matrix);
  const int64_t base = static_cast<int64_t>(matrix) * a.m * a.n;
  float* x = a.x + base;
  _Float16* h = a.h + base;
  _Float16* ht = a.ht_next + base;
  const bool flip = GE >= 0 && a.tall;  // V's tiles lie as H^T's
  const int tiles_c = (flip ? a.m : a.n) / kNsPad;
  const int r0 = blockIdx.x / tiles_c * kNsPad, c0 = blockIdx.x % tiles_c * kNsPad;
  const int tr = threadIdx.x >> 4, tc = 4 * (threadIdx.x & 15);
  f32x4 v[4];
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int r = r0 + 16 * pass + tr, c = c0 + tc;
    if constexpr (GE >= 0)
      v[pass] = load_four<GE>(a, reinterpret_cast<const void*>(t.g[matrix]), r, c);
    else
      v[pass] = *reinterpret_cast<const f32x4*>(x + static_cast<int64_t>(r) * a.n + c);
  }
  static_assert(kNsPartials <= kNsThreads, "a partial sum for each thread");
  const double sum = static_cast<int>(threadIdx.x) < a.partials ? a.partial[matrix * kNsPartials + threadIdx.x] : 0.0;
  const NsDivisor scaled = ns_divisor(group_sum<kNsThreads>(sum, scratch), a.eps);
  auto store_x = [&](int row, int col, const f32x4& y, const f16x4& w) {
    const int64_t i = static_cast<int64_t>(row) * a.n + col;
    *reinterpret_cast<f32x4*>(x + i) = y;
    *reinterpret_cast<f16x4*>(h + i) = w;
  };
  auto store_turned = [&](int row, int col, const f16x4& w) {
    *reinterpret_cast<f16x4*>(ht + static_cast<int64_t>(row) * a.m + col) = w;
  };
  auto halves = [](const f32x4& y) {
    f16x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = static_cast<_Float16>(y[j] * kNsScale);
    return w;
  };
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int row = 16 * pass + tr;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[pass][j] = scaled(v[pass][j]);
      turned[tc + j][row] = v[pass][j];
    }
    if (flip) store_turned(r0 + row, c0 + tc, halves(v[pass]));
    else store_x(r0 + row, c0 + tc, v[pass], halves(v[pass]));
  }
  __syncthreads();
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int row = 16 * pass + tr;
    const f32x4 y{turned[row][tc], turned[row][tc + 1], turned[row][tc + 2], turned[row][tc + 3]};
    if (flip) store_x(c0 + row, r0 + tc, y, halves(y));
    else store_turned(c0 + row, r0 + tc, halves(y));
  }
}

// Stores four consecutive values of row `row` of the result with encoding E, or
// (MUON) of the parameter, whose values were `old`, updated by them.
template <int E, bool MUON>
__device__ __forceinline__ void finish(const NsArgs& a, void* out, int row, int col, const f32x4& y, const f32x4& old) {
  const int live = live_four(a, row, col);
  if (!live) return;
  const int64_t i = static_cast<int64_t>(row) * a.cols + col;
  float r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = MUON ? fmaf(y[j], a.neg_lr, old[j] * a.decay) : y[j];
  if (live == 4) {
    uint32_t w[group_words(E)];
    encode_group<E>(r, 0u, w);
    store_group<E>(out, i, w);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < live) store1<E>(out, i + j, encode<E>(r[j], 0u));
  }
}

enum NsOp { kNsGram, kNsPolynomial, kNsStep, kNsLast };

// A workgroup's tile and operands.
struct NsTile {
  Operand a, b;
  int matrix, row0, col0, stages;
  bool mirrored;  // a tile below the diagonal, to be stored twice
};

template <int OP, class S>
__device__ __forceinline__ NsTile ns_tile(const NsArgs& a, uint32_t tiles_m, uint32_t tiles_n, uint32_t tiles,
                                          uint32_t matrices) {
  constexpr bool kSymmetric = OP == kNsGram || OP == kNsPolynomial;
  NsTile r;
  const uint32_t id = xcd_run(blockIdx.x, tiles * matrices);
  r.matrix = id / tiles;
  uint32_t tile_m, tile_n;
  if constexpr (kSymmetric) {
    static_assert(S::BM == S::BN, "a triangle of square tiles");
    triangle_tile(id % tiles, tile_m, tile_n);
  } else {
    band_tile(id % tiles, tiles_m, tiles_n, tile_m, tile_n);
  }
  r.row0 = tile_m * S::BM;
  r.col0 = tile_n * S::BN;
  r.mirrored = tile_n * S::BN < tile_m * S::BM;  // left of the diagonal blocks, which are computed whole
  const int64_t base = static_cast<int64_t>(r.matrix) * a.m * a.n, square = static_cast<int64_t>(r.matrix) * a.m * a.m;
  if constexpr (OP == kNsGram) {
    r.a = r.b = {reinterpret_cast<const char*>(a.h + base), 2 * static_cast<int64_t>(a.n), a.m};
    r.stages = a.n / (kStageBytes / 2);
  } else {
    r.a = {reinterpret_cast<const char*>((OP == kNsPolynomial ? a.g : a.p) + square), 2 * static_cast<int64_t>(a.m), a.m};
    r.b = r.a;
    if constexpr (!kSymmetric) r.b = {reinterpret_cast<const char*>(a.ht + base), 2 * static_cast<int64_t>(a.m), a.n};
    r.stages = a.m / (kStageBytes / 2);
  }
  return r;
}

// Stores a workgroup's sums through its LDS, which every wave is done with.
//   kNsGram, kNsPolynomial  the FP16 matrix, and its transpose where `mirrored`
//   kNsStep                 X, H and H^T
//   kNsLast                 the results (E, MUON), transposed where TURNED
template <int OP, bool TURNED, int E, bool MUON, int LDS, class S, class Acc>
__device__ __forceinline__ void ns_store(const NsArgs& a, const MatrixTable& t, const NsTile& tile, char* lds, int wave,
                                         int lane, const Acc& acc) {
  constexpr bool kSymmetric = OP == kNsGram || OP == kNsPolynomial;
  using Chunk = ResultChunk<S::kRowsN>;
  using T = std::conditional_t<OP == kNsLast, float, _Float16>;
  using T4 = std::conditional_t<OP == kNsLast, f32x4, f16x4>;
  constexpr bool kTurns = OP != kNsLast || TURNED;
  constexpr int kWaveBytes = Chunk::kBytes + (kTurns ? Chunk::template turned_bytes<T>() : 0);
  static_assert(S::kWaves * kWaveBytes <= LDS, "a chunk and its transpose per wave");
  const int width = kSymmetric ? a.m : a.n;
  const int64_t base = static_cast<int64_t>(tile.matrix) * a.m * a.n, square = static_cast<int64_t>(tile.matrix) * a.m * a.m;
  const int wave_row = tile.row0 + wave / S::WN * S::kRowsM, wave_col = tile.col0 + wave % S::WN * S::kRowsN;
  float* chunk = reinterpret_cast<float*>(lds + wave * kWaveBytes);
  T* turned = reinterpret_cast<T*>(lds + wave * kWaveBytes + Chunk::kBytes);
  _Float16* out = (OP == kNsGram ? a.g : a.p) + square;  // kSymmetric
  void* result = reinterpret_cast<void*>(t.p[tile.matrix]);  // kNsLast

  // What the sums of a chunk are combined with: G, or X and the parameter, of all of the lane's rows.  A chunk's loads
  // go out before the stores of the one before it: memory operations are waited for in their order, so that loads
  // behind stores wait for these too.
  using Old = std::conditional_t<OP == kNsPolynomial, f16x4, f32x4>;
  Old old[2][Chunk::kBlocks][4];
  // (The registers of wide tiles do not hold two chunks of X and the parameter.)
  constexpr bool kAhead = !(MUON && std::is_same_v<S, TileWide>);
  f32x4 parameter[2][Chunk::kBlocks][4], across[2][Chunk::kTurnedBlocks];
  constexpr int kChunks = S::kRowsM / 32;
  // The workspace's sizes are multiples of 64, so a chunk of 32 x 32 or 32 x 64 is inside or outside as a whole.
  auto inside = [&](int number) { return wave_row + 32 * number < a.m && wave_col < width; };
  auto load = [&](int number) {
    const bool in = inside(number);
    const int row0 = in ? wave_row + 32 * number : 0, col = (in ? wave_col : 0) + Chunk::block_col(lane);
#pragma unroll
    for (int i = 0; i < Chunk::kBlocks; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int row = row0 + Chunk::block_row(i, lane) + k;
        if constexpr (OP == kNsPolynomial)
          old[number & 1][i][k] = *reinterpret_cast<const f16x4*>(a.g + square + static_cast<int64_t>(row) * a.m + col);
        else if constexpr (OP != kNsGram)
          old[number & 1][i][k] = *reinterpret_cast<const f32x4*>(a.x + base + static_cast<int64_t>(row) * a.n + col);
      }
  };
  auto load_parameter = [&](int number) {
    const bool in = inside(number);
    const int row0 = in ? wave_row + 32 * number : 0, col0 = in ? wave_col : 0;
    if constexpr (MUON && TURNED) {
#pragma unroll
      for (int i = 0; i < Chunk::kTurnedBlocks; ++i) {
        const int row = col0 + Chunk::turned_col(i, lane), col = row0 + Chunk::turned_row(lane);
        across[number & 1][i] = load_four<E>(a, result, row, col);
      }
    } else if constexpr (MUON) {
      const int col = col0 + Chunk::block_col(lane);
#pragma unroll
      for (int i = 0; i < Chunk::kBlocks; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = row0 + Chunk::block_row(i, lane) + k;
          parameter[number & 1][i][k] = load_four<E>(a, result, row, col);
        }
    }
  };

  auto use = [&](auto number, const float* from) {
    constexpr int kNumber = decltype(number)::value;
    constexpr int kLoad = kAhead ? kNumber + 1 : kNumber;
    if constexpr (kLoad < kChunks) {
      load(kLoad);
      load_parameter(kLoad);
    }
    if (!inside(kNumber)) return;
    const int row0 = wave_row + 32 * kNumber, col = wave_col + Chunk::block_col(lane);
#pragma unroll
    for (int i = 0; i < Chunk::kBlocks; ++i) {
      const int r0 = Chunk::block_row(i, lane);
      T4 block[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int row = row0 + r0 + k;
        const f32x4 v = Chunk::get(from, r0 + k, Chunk::block_col(lane));
        if constexpr (OP == kNsGram) {
#pragma unroll
          for (int j = 0; j < 4; ++j) block[k][j] = static_cast<_Float16>(v[j] * kNsInverse);
          *reinterpret_cast<f16x4*>(out + static_cast<int64_t>(row) * a.m + col) = block[k];
        } else if constexpr (OP == kNsPolynomial) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = fmaf(a.c * kNsInverse, v[j], a.b * static_cast<float>(old[kNumber & 1][i][k][j]));
            block[k][j] = static_cast<_Float16>(row == col + j ? p + kNsShift * kNsScale : p);
          }
          *reinterpret_cast<f16x4*>(out + static_cast<int64_t>(row) * a.m + col) = block[k];
        } else {
          f32x4 y;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = old[kNumber & 1][i][k][j], h = static_cast<float>(static_cast<_Float16>(x * kNsScale)) * kNsInverse;
            y[j] = fmaf(v[j], kNsProduct, fmaf(-kNsShift, h, a.a * x));
          }
          if constexpr (OP == kNsStep) {
            const int64_t at = base + static_cast<int64_t>(row) * a.n + col;
#pragma unroll
            for (int j = 0; j < 4; ++j) block[k][j] = static_cast<_Float16>(y[j] * kNsScale);
            *reinterpret_cast<f32x4*>(a.x + at) = y;
            *reinterpret_cast<f16x4*>(a.h + at) = block[k];
          } else {
            block[k] = y;
            if constexpr (!TURNED) finish<E, MUON>(a, result, row, col, y, parameter[kNumber & 1][i][k]);
          }
        }
      }
      if constexpr (kTurns) {
        if (!kSymmetric || tile.mirrored) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            Chunk::template put_turned<T, T4>(turned, Chunk::block_col(lane) + j, r0,
                                              T4{block[0][j], block[1][j], block[2][j], block[3][j]});
        }
      }
    }
    if constexpr (OP == kNsLast && TURNED) {
#pragma unroll
      for (int i = 0; i < Chunk::kTurnedBlocks; ++i)
        finish<E, MUON>(a, result, wave_col + Chunk::turned_col(i, lane), row0 + Chunk::turned_row(lane),
                        Chunk::template get_turned<T, T4>(turned, i, lane), across[kNumber & 1][i]);
    } else if constexpr (kTurns) {
      if (!kSymmetric || tile.mirrored) {
        _Float16* to = kSymmetric ? out : a.ht_next + base;
#pragma unroll
        for (int i = 0; i < Chunk::kTurnedBlocks; ++i)
          *reinterpret_cast<f16x4*>(to + static_cast<int64_t>(wave_col + Chunk::turned_col(i, lane)) * a.m + row0 +
                                    Chunk::turned_row(lane)) = Chunk::template get_turned<T, T4>(turned, i, lane);
      }
    }
  };
  if constexpr (kAhead) {
    load(0);
    load_parameter(0);
  }
  for_each_chunk<S>(chunk, lane, acc, use);
}

// Bytes of LDS of a kernel that has `stages` bytes of stages.
template <int OP, bool TURNED, class S>
constexpr int ns_lds(int stages) {
  const int turned = OP == kNsLast ? (TURNED ? ResultChunk<S::kRowsN>::template turned_bytes<float>() : 0)
                                   : ResultChunk<S::kRowsN>::template turned_bytes<_Float16>();
  const int chunks = S::kWaves * (ResultChunk<S::kRowsN>::kBytes + turned);
  return stages > chunks ? stages : chunks;
}

// Calls store(E, MUON) with the last step's encoding and kind; other steps have neither.
template <int OP, class F>
__device__ __forceinline__ void with_result(const NsArgs& a, F&& store) {
  using std::integral_constant;
  if constexpr (OP != kNsLast) {
    store(integral_constant<int, ENC_F32>{}, std::false_type{});
  } else if (a.muon) {
    if (a.out_dtype == SR_F32) store(integral_constant<int, ENC_F32>{}, std::true_type{});
    else store(integral_constant<int, ENC_BF16_RN>{}, std::true_type{});
  } else {
    if (a.out_dtype == SR_F32) store(integral_constant<int, ENC_F32>{}, std::false_type{});
    else if (a.out_dtype == SR_BF16) store(integral_constant<int, ENC_BF16_RN>{}, std::false_type{});
    else store(integral_constant<int, ENC_F16_RN>{}, std::false_type{});
  }
}

// One launch of products: S-shaped tiles of every matrix.
//   kNsGram        G = H H^T, the lower triangle's tiles
//   kNsPolynomial  P + s I = b G + c G^2 + s I, the same tiles
//   kNsStep        X <- a X - s H + (P + s I) H, and the new H and H^T
//   kNsLast        the same into the results or the parameters; TURNED where
//                  these are the transpose of the workspace's orientation
// Few tiles are bound by the latency of a tile's walk (768 x 2304: G 12.6 us, P
// 7.2, step 11.6), many by what a CU reads from its L2 (G of 8 x 2048 x 2048
// 108 us, 676 TFLOP/s of the computed half and diagonal; G of 2048 x 8192, 528
// tiles of 64 x 64 on 256 CUs, 77 us with the matrix cores busy 20% of the cycles).
template <int OP, class S, bool TURNED>
__global__ __launch_bounds__(S::kThreads, S::kMinWaves) void ns_product_kernel(NsArgs a, uint32_t tiles_m, uint32_t tiles_n,
                                                                    uint32_t tiles, uint32_t matrices, MatrixTable t) {
  constexpr int kLds = ns_lds<OP, TURNED, S>(S::kLds);
  static_assert(S::kSums <= kLds, "the groups' sums");
  __shared__ __align__(1024) char lds[kLds];
  const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = all % S::kWaves, group = all / S::kWaves;
  char* own = lds + group * 2 * S::kStage;  // this group's stages
  need_arguments(a);
  const NsTile tile = ns_tile<OP, S>(a, tiles_m, tiles_n, tiles, matrices);
  const int wave_m = wave / S::WN * S::kRowsM, wave_n = wave % S::WN * S::kRowsN;
  const int stages = tile.stages;
  Stager<S> stager;
  stager.init(tile.a, tile.b, tile.row0, tile.col0, wave, lane);

  f32x4 acc[S::MI][S::NI] = {};
  const uint32_t fragment = fragment_offset(lane);
  walk_stages<S>(
      stages, group, [&](int kt, int buffer) { stager.load_async(own + buffer * S::kStage, kt * kStageBytes, wave); },
      [](int) {},
      [&](int, int buffer) {
        const char* stage = own + buffer * S::kStage;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const char* sa = stage + wave_m * kStageBytes + (fragment ^ (64 * ks));
          const char* sb = stage + (S::BM + wave_n) * kStageBytes + (fragment ^ (64 * ks));
          f16x8 fb[S::NI];
#pragma unroll
          for (int ni = 0; ni < S::NI; ++ni)
            fb[ni] = __builtin_bit_cast(f16x8, read_chunk(sb + ni * 16 * kStageBytes));
#pragma unroll
          for (int mi = 0; mi < S::MI; ++mi) {
            const f16x8 fa = __builtin_bit_cast(f16x8, read_chunk(sa + mi * 16 * kStageBytes));
#pragma unroll
            for (int ni = 0; ni < S::NI; ++ni)
              acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb[ni], fa, acc[mi][ni], 0, 0, 0);
          }
        }
      });
  stage_barrier();
  add_groups<S>(lds, group, acc);
  if (group > 0) return;
  with_result<OP>(a, [&](auto encoding, auto muon) {
    ns_store<OP, TURNED, decltype(encoding)::value, decltype(muon)::value, kLds, S>(a, t, tile, lds, wave, lane, acc);
  });
}

// The same launches on wide tiles.  The step of 8192 x 2048 takes 92 us: 51 for
// the product (1355 TFLOP/s) and the rest for 192 MB of X, H and H^T at 4.6
// TB/s.
template <int OP, bool TURNED>
__global__ __launch_bounds__(TileWide::kThreads, 2) void ns_wide_kernel(NsArgs a, uint32_t tiles_m, uint32_t tiles_n,
                                                                        uint32_t tiles, uint32_t matrices, MatrixTable t) {
  constexpr int kLds = ns_lds<OP, TURNED, TileWide>(2 * TileWide::kStage);
  __shared__ __align__(1024) char lds[kLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  need_arguments(a);
  const NsTile tile = ns_tile<OP, TileWide>(a, tiles_m, tiles_n, tiles, matrices);
  Stager<TileWide> stager;
  stager.init(tile.a, tile.b, tile.row0, tile.col0, wave, lane);
  f32x16 acc[WideTile::MI][WideTile::NI] = {};
  WideTile::run(lds, stager, tile.stages, wave, lane, acc);
  with_result<OP>(a, [&](auto encoding, auto muon) {
    ns_store<OP, TURNED, decltype(encoding)::value, decltype(muon)::value, kLds, TileWide>(a, t, tile, lds, wave, lane, acc);
  });
}

// ---------------------------------------------------------------------------
// Small matrices: all steps of one matrix in one workgroup.
//
// With at most 64 rows (padded) and 768 columns, H fits the LDS and X the
// registers of sixteen waves, so that the steps need no memory and no further
// launches: 64 x 576 takes 32 us so, and a chain of 16 launches of 3 to 5 us
// each took 70.  Wave w
// computes tile (w / 4, w % 4) of G and P, and of X the column tiles w, w + 16, ...:
// lane l holds rows 16 i + 4 (l / 16) .. + 3 of its column 16 t + l % 16.
//
// LDS rows are runs of 16-byte chunks, chunk c of row r at place c ^ (r % 8) of
// its group of eight, as in the stages above.  G and P are symmetric, so a
// lane's four values of a column are stored as four neighbours of that row.
// The step needs H with its rows as the contracted axis: the transposing LDS
// read gives lane i of sixteen the values at column i of four rows, when lane i
// points at columns 4 (i % 4) .. + 3 of row i / 4.
// ---------------------------------------------------------------------------
constexpr int kSmallRows = 64, kSmallCols = 768, kSmallThreads = 1024;
constexpr int kSmallTiles = kSmallCols / 16 / 16;  // column tiles of a wave, at most

#if defined(__HIP_DEVICE_COMPILE__)
typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f16x4 read_turned(const char* p) {
  return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}
#else
__device__ inline f16x4 read_turned(const char*) { return {}; }
#endif

// Byte offset of column `col` (a multiple of 4) of row `row` in rows of `stride` bytes.
__device__ __forceinline__ int swizzled(int row, int col, int stride) {
  return row * stride + (((col >> 3) ^ (row & 7)) << 4) + ((col & 4) << 1);
}

// One value of the result, in the caller's orientation.
template <int E, bool MUON>
__device__ __forceinline__ void finish_one(const NsArgs& a, void* out, int row, int col, float y) {
  if (row >= a.rows || col >= a.cols) return;
  const int64_t i = static_cast<int64_t>(row) * a.cols + col;
  const float r = MUON ? fmaf(y, a.neg_lr, decode<E>(load1<E>(out, i)) * a.decay) : y;
  store1<E>(out, i, encode<E>(r, 0u));
}

__global__ __launch_bounds__(kSmallThreads, 4) void ns_small_kernel(NsArgs a, int steps, MatrixTable t) {
  __shared__ __align__(1024) char small_lds[2 * (2 * kSmallRows * kSmallRows + kSmallRows * kSmallCols)];
  __shared__ double scratch[16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int across = lane & 15, quarter = lane >> 4;
  const int matrix = blockIdx.x, n = a.n;
  char* gram = small_lds;                           // 64 x 64
  char* poly = gram + kSmallRows * kSmallRows * 2;  // 64 x 64
  char* h = poly + kSmallRows * kSmallRows * 2;     // 64 x n
  const int stride = 2 * n;
  const float* from = a.x + static_cast<int64_t>(matrix) * a.m * n;

  double sum = static_cast<int>(threadIdx.x) < a.partials ? a.partial[matrix * kNsPartials + threadIdx.x] : 0.0;
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) scratch[wave] = sum;
  f32x4 x[kSmallTiles][4];
#pragma unroll
  for (int c = 0; c < kSmallTiles; ++c) {
    const int col = 16 * (wave + 16 * c) + across;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[c][i][j] = 16 * (wave + 16 * c) < n ? from[(16 * i + 4 * quarter + j) * n + col] : 0.0f;
  }
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int w = 0; w < 16; ++w) sum += scratch[w];
  const NsDivisor scaled = ns_divisor(sum, a.eps);

  // Places in H whose swizzle does not change over the loops: 16 rows further are 16 strides, 16 column tiles further
  // (the wave's next) 512 bytes, 64 columns further 128 bytes.
  uint32_t own_h[4];  // of this lane's column of its first tile, row 4 quarter + j
#pragma unroll
  for (int j = 0; j < 4; ++j)
    own_h[j] = swizzled(4 * quarter + j, (16 * wave + across) & ~3, stride) + 2 * (across & 3);
  uint32_t turned_h[2];  // what it points at in the transposing reads of rows 0 .. 3 and 4 .. 7
#pragma unroll
  for (int u = 0; u < 2; ++u) turned_h[u] = swizzled(8 * quarter + across / 4 + 4 * u, 16 * wave + 4 * (across & 3), stride);
  uint32_t chunk_h[2], chunk_s[2];  // chunk 4 u + quarter of row `across` of H, and of G or P
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    chunk_h[u] = swizzled(across, 8 * (4 * u + quarter), stride);
    chunk_s[u] = swizzled(across, 8 * (4 * u + quarter), 2 * kSmallRows);
  }
  const uint32_t rows16 = 16 * stride;

  // H = X in FP16; every wave its column tiles.
  auto store_h = [&] {
#pragma unroll
    for (int c = 0; c < kSmallTiles; ++c) {
      if (16 * (wave + 16 * c) >= n) break;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<_Float16*>(h + own_h[j] + i * rows16 + 512 * c) = static_cast<_Float16>(x[c][i][j] * kNsScale);
    }
  };
#pragma unroll
  for (int c = 0; c < kSmallTiles; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[c][i][j] = scaled(x[c][i][j]);
  store_h();
  __syncthreads();

  const int tile_i = wave >> 2, tile_j = wave & 3;
  auto fragment = [](const char* p) { return __builtin_bit_cast(f16x8, read_chunk(p)); };
  // Where a lane's four values of a symmetric tile belong: row of tile j, columns of tile i.
  const int own = swizzled(16 * tile_j + across, 16 * tile_i + 4 * quarter, 2 * kSmallRows);
  for (int step = 0; step < steps; ++step) {
    f32x4 sums[2] = {};
    const char *rows_i = h + tile_i * rows16, *rows_j = h + tile_j * rows16;
    for (int k = 0; k < stride; k += 128) {  // 64 columns, which n is a multiple of
#pragma unroll
      for (int u = 0; u < 2; ++u)
        sums[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fragment(rows_i + chunk_h[u] + k), fragment(rows_j + chunk_h[u] + k),
                                                         sums[u], 0, 0, 0);
    }
    f16x4 g;
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = static_cast<_Float16>((sums[0][j] + sums[1][j]) * kNsInverse);
    *reinterpret_cast<f16x4*>(gram + own) = g;
    __syncthreads();
    f32x4 square{};
#pragma unroll
    for (int k = 0; k < 2; ++k)
      square = __builtin_amdgcn_mfma_f32_16x16x32_f16(fragment(gram + 32 * kSmallRows * tile_i + chunk_s[k]),
                                                      fragment(gram + 32 * kSmallRows * tile_j + chunk_s[k]), square, 0, 0, 0);
    f16x4 p;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float v = fmaf(a.c * kNsInverse, square[j], a.b * static_cast<float>(g[j]));
      p[j] = static_cast<_Float16>(16 * tile_j + across == 16 * tile_i + 4 * quarter + j ? v + kNsShift * kNsScale : v);
    }
    *reinterpret_cast<f16x4*>(poly + own) = p;
    __syncthreads();
    f16x8 left[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) left[i][k] = fragment(poly + 32 * kSmallRows * i + chunk_s[k]);
#pragma unroll
    for (int c = 0; c < kSmallTiles; ++c) {
      if (16 * (wave + 16 * c) >= n) break;
      f16x8 right[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const char* rows = h + 2 * k * rows16 + 512 * c;
        right[k] = __builtin_shufflevector(read_turned(rows + turned_h[0]), read_turned(rows + turned_h[1]), 0, 1, 2, 3, 4, 5, 6, 7);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x4 v{};
#pragma unroll
        for (int k = 0; k < 2; ++k) v = __builtin_amdgcn_mfma_f32_16x16x32_f16(left[i][k], right[k], v, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float own_h = static_cast<float>(static_cast<_Float16>(x[c][i][j] * kNsScale)) * kNsInverse;
          x[c][i][j] = fmaf(v[j], kNsProduct, fmaf(-kNsShift, own_h, a.a * x[c][i][j]));
        }
      }
    }
    // A wave reads and writes only its own columns of H in the step, and all of it in the next G.
    if (step + 1 < steps) {
      store_h();
      __syncthreads();
    }
  }

  void* out = reinterpret_cast<void*>(t.p[matrix]);
  with_result<kNsLast>(a, [&](auto encoding, auto muon) {
#pragma unroll
    for (int c = 0; c < kSmallTiles; ++c) {
      const int col = 16 * (wave + 16 * c) + across;
      if (16 * (wave + 16 * c) >= n) break;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = 16 * i + 4 * quarter + j;
          finish_one<decltype(encoding)::value, decltype(muon)::value>(a, out, a.tall ? col : row, a.tall ? row : col, x[c][i][j]);
        }
    }
  });
}

}  // namespace sr
