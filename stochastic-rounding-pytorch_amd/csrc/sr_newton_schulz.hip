// sr_newton_schulz.hip -- kernels and extern "C" entry points of the orthogonalised updates (sr_matrix_hip.h).
#include "sr_newton_schulz.h"

#include "sr_block_tables.h"
#include "sr_error.h"

namespace {

using sr::fail;
using sr::NsArgs;

constexpr int64_t kMaxSide = 1 << 20, kMaxElements = int64_t{1} << 31;

int64_t padded(int64_t n) { return (n + sr::kNsPad - 1) / sr::kNsPad * sr::kNsPad; }
int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// Bytes of each part of the workspace of `batch` padded m x n matrices.
struct Layout {
  int64_t x, h, square, partial;
  Layout(int64_t batch, int64_t m, int64_t n)
      : x(aligned(batch * m * n * 4)), h(aligned(batch * m * n * 2)), square(aligned(batch * m * m * 2)),
        partial(aligned(batch * sr::kNsPartials * 8)) {}
  int64_t total() const { return x + 3 * h + 2 * square + partial; }
};

bool fits(int64_t rows, int64_t cols) { return rows <= kMaxSide && cols <= kMaxSide && rows * cols <= kMaxElements; }

int check_shape(int64_t batch, int64_t rows, int64_t cols, const sr_newton_schulz* ns) {
  if (batch < 0 || rows < 0 || cols < 0) return fail(SR_ERR_ARGUMENT, "negative size");
  if (!fits(rows, cols))
    return fail(SR_ERR_ARGUMENT, "%lld x %lld matrices are too large", (long long)rows, (long long)cols);
  if (!ns) return fail(SR_ERR_ARGUMENT, "null argument");
  if (ns->steps < 1) return fail(SR_ERR_ARGUMENT, "%d steps", ns->steps);
  return SR_OK;
}

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? SR_OK : sr::hip_fail(err, what);
}

template <int GE>
void load_momentum(const NsArgs& a, const sr::MatrixTable& t, int ue, dim3 grid, hipStream_t s) {
  switch (ue) {
#define SR_CASE(E) \
  case sr::E: sr::ns_load_kernel<GE, sr::E><<<grid, sr::kNsLoadThreads, 0, s>>>(a, t); break;
    SR_CASE(ENC_F32)
    SR_CASE(ENC_BF16_RN)
    SR_CASE(ENC_BF16_SR)
    SR_CASE(ENC_F16_RN)
    SR_CASE(ENC_F16_SR)
    SR_CASE(ENC_E4M3_RN)
    SR_CASE(ENC_E4M3_SR)
    SR_CASE(ENC_E5M2_RN)
    SR_CASE(ENC_E5M2_SR)
#undef SR_CASE
  }
}

template <int OP, class S, bool TURNED = false>
int product(const NsArgs& a, int matrices, const sr::MatrixTable& t, hipStream_t s) {
  constexpr bool kSymmetric = OP == sr::kNsGram || OP == sr::kNsPolynomial;
  const uint32_t tm = (a.m + S::BM - 1) / S::BM, tn = ((kSymmetric ? a.m : a.n) + S::BN - 1) / S::BN;
  const uint32_t tiles = kSymmetric ? tm * (tm + 1) / 2 : tm * tn;
  if (static_cast<uint64_t>(tiles) * matrices > 0x3FFFFFu) return fail(SR_ERR_ARGUMENT, "%u tiles exceed a launch", tiles);
  if constexpr (std::is_same_v<S, sr::TileWide>) {
    sr::ns_wide_kernel<OP, TURNED><<<tiles * matrices, S::kThreads, 0, s>>>(a, tm, tn, tiles, matrices, t);
  } else {
    sr::ns_product_kernel<OP, S, TURNED><<<tiles * matrices, S::kThreads, 0, s>>>(a, tm, tn, tiles, matrices, t);
  }
  return launched("Newton-Schulz product launch");
}

// The symmetric launches stop at 128 x 128 tiles, and the others take 256 x
// 256 ones where these fill the chip: a triangle has few large tiles (8
// matrices of 2048 x 2048: G 122 us on 256 x 256 tiles and 102 on 128 x 128,
// the step 200 and 244).
template <int OP, bool TURNED = false>
int product_by_size(const NsArgs& a, int matrices, const sr::MatrixTable& t, hipStream_t s) {
  constexpr bool kSymmetric = OP == sr::kNsGram || OP == sr::kNsPolynomial;
  if constexpr (OP == sr::kNsLast && !TURNED) {
    if (a.tall) return product_by_size<OP, true>(a, matrices, t, s);
  }
  auto tiles = [&](int64_t side) {
    const int64_t tm = (a.m + side - 1) / side, tn = (a.n + side - 1) / side;
    return (kSymmetric ? tm * (tm + 1) / 2 : tm * tn) * matrices;
  };
  if constexpr (!kSymmetric) {
    if (tiles(256) >= 256) return product<OP, sr::TileWide, TURNED>(a, matrices, t, s);
  }
  switch (sr::tile_by_count(tiles)) {
    case sr::kTile128: return product<OP, sr::Tile128, TURNED>(a, matrices, t, s);
    case sr::kTile64x2: return product<OP, sr::Tile64x2, TURNED>(a, matrices, t, s);
    case sr::kTile64x4: return product<OP, sr::Tile64x4, TURNED>(a, matrices, t, s);
    default: return product<OP, sr::Tile64, TURNED>(a, matrices, t, s);
  }
}

// The whole update of up to SR_MATRIX_BATCH matrices.  `ue` is the momentum's
// encoding, or -1 for none.
int run(NsArgs a, const sr::MatrixTable& t, int matrices, int g_dtype, int ue, const sr_newton_schulz& ns,
        void* workspace, hipStream_t s) {
  a.m = static_cast<int>(padded(a.rows < a.cols ? a.rows : a.cols));
  a.n = static_cast<int>(padded(a.rows < a.cols ? a.cols : a.rows));
  a.tall = a.rows > a.cols;
  a.a = ns.a;
  a.b = ns.b;
  a.c = ns.c;
  a.eps = ns.eps;
  const Layout layout(matrices, a.m, a.n);
  char* w = static_cast<char*>(workspace);
  a.x = reinterpret_cast<float*>(w);
  w += layout.x;
  a.h = reinterpret_cast<_Float16*>(w);
  _Float16* turned[2] = {reinterpret_cast<_Float16*>(w + layout.h), reinterpret_cast<_Float16*>(w + 2 * layout.h)};
  w += 3 * layout.h;
  a.g = reinterpret_cast<_Float16*>(w);
  a.p = reinterpret_cast<_Float16*>(w + layout.square);
  a.partial = reinterpret_cast<double*>(w + 2 * layout.square);

  const int64_t tiles = static_cast<int64_t>(a.m / sr::kNsPad) * (a.n / sr::kNsPad);
  a.partials = static_cast<int>(tiles < sr::kNsPartials ? tiles : sr::kNsPartials);
  const dim3 grid(a.partials, matrices), all(static_cast<uint32_t>(tiles), matrices);
  const bool small = a.m == sr::kSmallRows && a.n <= sr::kSmallCols;
  a.keep = ue >= 0 || small;
  if (ue < 0) {
    if (g_dtype == SR_F32) sr::ns_load_kernel<sr::ENC_F32, -1><<<grid, sr::kNsLoadThreads, 0, s>>>(a, t);
    else if (g_dtype == SR_BF16) sr::ns_load_kernel<sr::ENC_BF16_RN, -1><<<grid, sr::kNsLoadThreads, 0, s>>>(a, t);
    else sr::ns_load_kernel<sr::ENC_F16_RN, -1><<<grid, sr::kNsLoadThreads, 0, s>>>(a, t);
  } else if (g_dtype == SR_F32) {
    load_momentum<sr::ENC_F32>(a, t, ue, grid, s);
  } else {
    load_momentum<sr::ENC_BF16_RN>(a, t, ue, grid, s);
  }
  if (int rc = launched("ns_load_kernel launch")) return rc;
  if (small) {
    sr::ns_small_kernel<<<matrices, sr::kSmallThreads, 0, s>>>(a, ns.steps, t);
    return launched("ns_small_kernel launch");
  }
  a.ht_next = turned[0];
  if (ue >= 0) sr::ns_scale_kernel<-1><<<all, sr::kNsThreads, 0, s>>>(a, t);
  else if (g_dtype == SR_F32) sr::ns_scale_kernel<sr::ENC_F32><<<all, sr::kNsThreads, 0, s>>>(a, t);
  else if (g_dtype == SR_BF16) sr::ns_scale_kernel<sr::ENC_BF16_RN><<<all, sr::kNsThreads, 0, s>>>(a, t);
  else sr::ns_scale_kernel<sr::ENC_F16_RN><<<all, sr::kNsThreads, 0, s>>>(a, t);
  if (int rc = launched("ns_scale_kernel launch")) return rc;
  for (int step = 0; step < ns.steps; ++step) {
    a.ht = turned[step & 1];
    a.ht_next = turned[~step & 1];
    if (int rc = product_by_size<sr::kNsGram>(a, matrices, t, s)) return rc;
    if (int rc = product_by_size<sr::kNsPolynomial>(a, matrices, t, s)) return rc;
    if (int rc = step + 1 < ns.steps ? product_by_size<sr::kNsStep>(a, matrices, t, s)
                                     : product_by_size<sr::kNsLast>(a, matrices, t, s))
      return rc;
  }
  return SR_OK;
}

int momentum_enc(int dtype, int rule) {
  if (rule != SR_NEAREST && rule != SR_STOCHASTIC) return -1;
  switch (dtype) {
    case SR_F32: return sr::ENC_F32;
    case SR_BF16: return rule == SR_STOCHASTIC ? sr::ENC_BF16_SR : sr::ENC_BF16_RN;
    case SR_F16: return rule == SR_STOCHASTIC ? sr::ENC_F16_SR : sr::ENC_F16_RN;
    case SR_E4M3: return rule == SR_STOCHASTIC ? sr::ENC_E4M3_SR : sr::ENC_E4M3_RN;
    case SR_E5M2: return rule == SR_STOCHASTIC ? sr::ENC_E5M2_SR : sr::ENC_E5M2_RN;
    default: return -1;
  }
}

}  // namespace

extern "C" {

int64_t sr_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0 || !fits(rows, cols)) return 0;
  const int64_t m = padded(rows < cols ? rows : cols), n = padded(rows < cols ? cols : rows);
  return Layout(batch < SR_MATRIX_BATCH ? batch : SR_MATRIX_BATCH, m, n).total();
}

int sr_orthogonalize(const void* x, void* out, int64_t batch, int64_t x_stride, int64_t out_stride, int64_t rows,
                     int64_t cols, int x_dtype, int out_dtype, const sr_newton_schulz* ns, void* workspace,
                     void* stream) {
  if (int rc = check_shape(batch, rows, cols, ns)) return rc;
  for (int dtype : {x_dtype, out_dtype})
    if (dtype != SR_F32 && dtype != SR_BF16 && dtype != SR_F16)
      return fail(SR_ERR_ARGUMENT, "orthogonalize takes and gives FP32, BF16 or FP16, not dtype %d", dtype);
  if (batch == 0 || rows == 0 || cols == 0) return SR_OK;
  if (!x || !out || !workspace) return fail(SR_ERR_ARGUMENT, "null pointer");
  if (batch > 1 && out_stride < rows * cols) return fail(SR_ERR_ARGUMENT, "results overlap");
  const int64_t x_size = x_dtype == SR_F32 ? 4 : 2, out_size = out_dtype == SR_F32 ? 4 : 2;
  for (int64_t first = 0; first < batch; first += SR_MATRIX_BATCH) {
    const int count = static_cast<int>(batch - first < SR_MATRIX_BATCH ? batch - first : SR_MATRIX_BATCH);
    sr::MatrixTable t{};
    for (int i = 0; i < count; ++i) {
      t.g[i] = reinterpret_cast<uint64_t>(x) + static_cast<uint64_t>((first + i) * x_stride * x_size);
      t.p[i] = reinterpret_cast<uint64_t>(out) + static_cast<uint64_t>((first + i) * out_stride * out_size);
    }
    NsArgs a{};
    a.rows = static_cast<int>(rows);
    a.cols = static_cast<int>(cols);
    a.out_dtype = out_dtype;
    if (int rc = run(a, t, count, x_dtype, -1, *ns, workspace, static_cast<hipStream_t>(stream))) return rc;
  }
  return SR_OK;
}

int sr_muon_multi(const sr_muon_row* table, int nrows, int64_t rows, int64_t cols, int p_dtype, int g_dtype,
                  int u_dtype, int u_rule, const sr_muon_hparams* hp, const sr_newton_schulz* ns, void* workspace,
                  void* stream) {
  if (int rc = check_shape(nrows, rows, cols, ns)) return rc;
  if ((p_dtype != SR_F32 && p_dtype != SR_BF16) || (g_dtype != SR_F32 && g_dtype != SR_BF16))
    return fail(SR_ERR_ARGUMENT, "parameter and gradient must be FP32 or BF16");
  const int ue = momentum_enc(u_dtype, u_rule);
  if (ue < 0) return fail(SR_ERR_ARGUMENT, "unsupported state dtype or rule");
  if (!hp) return fail(SR_ERR_ARGUMENT, "null hyperparameters");
  if (nrows == 0 || rows == 0 || cols == 0) return SR_OK;
  if (!table || !workspace) return fail(SR_ERR_ARGUMENT, "null pointer");
  for (int i = 0; i < nrows; ++i)
    if (!table[i].p || !table[i].g || !table[i].u) return fail(SR_ERR_ARGUMENT, "row %d: null pointer", i);
  for (int first = 0; first < nrows; first += SR_MATRIX_BATCH) {
    const int count = nrows - first < SR_MATRIX_BATCH ? nrows - first : SR_MATRIX_BATCH;
    sr::MatrixTable t{};
    for (int i = 0; i < count; ++i) {
      const sr_muon_row& row = table[first + i];
      t.p[i] = reinterpret_cast<uint64_t>(row.p);
      t.g[i] = reinterpret_cast<uint64_t>(row.g);
      t.u[i] = reinterpret_cast<uint64_t>(row.u);
      t.counter[i] = sr::state_key(row.key, 0) + row.offset;
    }
    NsArgs a{};
    a.rows = static_cast<int>(rows);
    a.cols = static_cast<int>(cols);
    a.momentum = hp->momentum;
    a.decay = hp->decay;
    a.neg_lr = hp->neg_lr;
    a.nesterov = hp->nesterov;
    a.muon = 1;
    a.out_dtype = p_dtype;
    if (int rc = run(a, t, count, g_dtype, ue, *ns, workspace, static_cast<hipStream_t>(stream))) return rc;
  }
  return SR_OK;
}

}  // extern "C"
