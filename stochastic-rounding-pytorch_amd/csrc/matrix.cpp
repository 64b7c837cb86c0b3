// Native entries of the matrix operators: block casts and products, the
// block-scaled linear layer, and orthogonalisation.
//
// The operators' small calls are bound by the host: through Python checks and
// ctypes a block cast took 30 us around a kernel of 6.  This CPython extension
// makes the tensor checks, allocates the results and calls the C ABI's entry
// points through the addresses the Python side binds once.
//
// bind(block_cast, block_matmul, orthogonalize, orthogonalize_workspace, grouped_columns, grouped_block_cast,
//      stacked_block_cast, grouped_block_matmul, grouped_block_contract, adapter_low, adapter_workspace, adapter_add,
//      adapter_backward, last_error)
//   Keep the addresses of these sr_ entry points, taken from the loaded library.
//
// block_cast(x, code, rule, square, axes, seed, offset, stream) -> tuple or int
//   The (data, scale) pairs of x for each character of `axes` ("1", "0", "10"
//   or "01"), flat; or the entry's status where that is not 0.
//
// block_matmul(a_data, a_scale, b_data, b_scale, out_code, out, stream) -> tensor or int
//   a b^T into a new tensor of sr_dtype out_code, or into `out` (not None).
//
// linear_forward(x, weight, formats, seed, need_x, need_weight, stream) -> tuple or int
//   (y, x_t data, x_t scale, w_t data, w_t scale): the product of x's and
//   weight's casts, and those the gradients need (None where not needed).
//   `formats` is (code, rule) of input, weight and gradient, flat, and `seed`
//   holds their three streams.
// linear_backward(dy, x_t data, x_t scale, w_t data, w_t scale, formats, seed, dx_code, dw_code, stream)
//   -> (dx, dw) or int; None for the gradients whose operands are None.
//
// orthogonalize(x, out_code, a, b, c, eps, steps, batch limit bytes, stream) -> tensor or int
//
// grouped_cast(x, sizes, code, rule, square, axes, seed, offset, stream) -> tuple or int
//   As block_cast, of a matrix whose rows are in groups of `sizes`, or (None) of a stack of matrices.
// grouped_matmul(a_data, a_scale, b_data, b_scale, sizes, out_code, out, stream) -> tensor or int
//   Each group's rows of a by its matrix of b, or its columns of a by its columns of b where b is a matrix.
// grouped_linear(x, weight, sizes, formats, seed, stream) -> tensor or int
//   The grouped layer, recorded for autograd in grad mode.
// adapter_add(base, x, a, b, index, scaling, scale, out, stream) -> tensor or int
//   base plus each row's low-rank update, into `out` where it is not None; else recorded for autograd in grad mode.
//
// The last two are nodes of the autograd graph themselves: through a Python function a training step of a small layer
// took 119 us, of which its kernels are 58, and one of small adapters 101.
//
// Errors of the tensors raise TypeError or ValueError before anything is
// launched.  Every entry runs with the first tensor's device current and the
// GIL released around the launch; `stream` is the raw handle of a stream on
// that device.

#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <optional>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "../../include/sr_matrix_hip.h"

namespace {

using CastFn = decltype(&sr_block_cast);
using MatmulFn = decltype(&sr_block_matmul);
using OrthogonalizeFn = decltype(&sr_orthogonalize);
using WorkspaceFn = decltype(&sr_orthogonalize_workspace);
CastFn g_cast = nullptr;
MatmulFn g_matmul = nullptr;
OrthogonalizeFn g_orthogonalize = nullptr;
WorkspaceFn g_workspace = nullptr;
decltype(&sr_grouped_columns) g_columns = nullptr;
decltype(&sr_grouped_block_cast) g_grouped_cast = nullptr;
decltype(&sr_stacked_block_cast) g_stacked_cast = nullptr;
decltype(&sr_grouped_block_matmul) g_grouped_matmul = nullptr;
decltype(&sr_grouped_block_contract) g_grouped_contract = nullptr;
decltype(&sr_adapter_low) g_adapter_low = nullptr;
decltype(&sr_adapter_workspace) g_adapter_workspace = nullptr;
decltype(&sr_adapter_add) g_adapter_add = nullptr;
decltype(&sr_adapter_backward) g_adapter_backward = nullptr;
decltype(&sr_last_error) g_last_error = nullptr;
PyObject* g_out_of_memory = nullptr;  // torch.OutOfMemoryError

// A refusal, raised as `type`.
struct Refusal : std::runtime_error {
  PyObject* type;
  Refusal(PyObject* t, const std::string& message) : std::runtime_error(message), type(t) {}
};
// A nonzero status of the C ABI, whose message sr_last_error() holds.
struct Status {
  int code;
};

[[noreturn]] void value_error(const std::string& message) { throw Refusal(PyExc_ValueError, message); }
[[noreturn]] void type_error(const std::string& message) { throw Refusal(PyExc_TypeError, message); }

int dtype_code(c10::ScalarType type) {
  switch (type) {
    case c10::ScalarType::Float: return SR_F32;
    case c10::ScalarType::BFloat16: return SR_BF16;
    case c10::ScalarType::Half: return SR_F16;
    case c10::ScalarType::Float8_e4m3fn: return SR_E4M3;
    case c10::ScalarType::Float8_e5m2: return SR_E5M2;
    default: return -1;
  }
}
c10::ScalarType scalar_type(int code) {
  constexpr c10::ScalarType types[] = {c10::ScalarType::Float, c10::ScalarType::BFloat16, c10::ScalarType::Half,
                                       c10::ScalarType::Float8_e4m3fn, c10::ScalarType::Float8_e5m2};
  return types[code];
}
bool wide(int code) { return code == SR_F32 || code == SR_BF16 || code == SR_F16; }
std::string name_of(c10::ScalarType type) {
  // The names Python shows; the ones that reach a message here are torch's own otherwise.
  switch (type) {
    case c10::ScalarType::Double: return "torch.float64";
    case c10::ScalarType::Float: return "torch.float32";
    case c10::ScalarType::BFloat16: return "torch.bfloat16";
    case c10::ScalarType::Half: return "torch.float16";
    case c10::ScalarType::Float8_e4m3fn: return "torch.float8_e4m3fn";
    case c10::ScalarType::Float8_e5m2: return "torch.float8_e5m2";
    default: return c10::toString(type);
  }
}

void* address(unsigned long long value) { return reinterpret_cast<void*>(static_cast<uintptr_t>(value)); }

const at::Tensor& tensor(PyObject* object) {
  if (!THPVariable_Check(object)) type_error(std::string("expected a tensor, got ") + Py_TYPE(object)->tp_name);
  return THPVariable_Unpack(object);
}

// Device memory of a tensor that has elements.  A lazily negated view (torch's negative bit) holds other values than its
// memory: inputs are resolved before they come here.
void* memory(const at::Tensor& x) {
  if (x.is_neg()) value_error("lazily negated views cannot be used: call resolve_neg()");
  void* p = const_cast<void*>(x.const_data_ptr());
  if (!p && x.numel()) value_error("tensors without device memory cannot be used");
  return p;
}

int64_t blocks(int64_t n) { return (n + SR_BLOCK - 1) / SR_BLOCK; }

// The distance between rows of a matrix with consecutive columns; an empty one has any strides.
int64_t row_stride(const at::Tensor& x, const std::string& what) {
  const int64_t rows = x.size(0), cols = x.size(1);
  if (!x.numel()) return std::max<int64_t>(cols, 1);
  const int64_t stride = rows > 1 ? x.stride(0) : std::max<int64_t>(cols, 1);
  if ((cols > 1 && x.stride(1) != 1) || stride < cols)
    value_error(what + " requires consecutive columns and rows that do not overlap");
  return stride;
}

struct Scaled {
  at::Tensor data, scale;
};

// Rows start on 16 bytes, which the product's asynchronous loads need.
Scaled new_scaled(int64_t rows, int64_t k, int code, bool square, const at::Device& device) {
  const auto options = at::TensorOptions().device(device);
  return {at::empty_strided({rows, k}, {(k + 15) / 16 * 16, 1}, options.dtype(scalar_type(code))),
          at::empty({square ? blocks(rows) : rows, blocks(k)}, options.dtype(c10::ScalarType::Float8_e8m0fnu))};
}

void checked(int status) {
  if (status) throw Status{status};
}

// The casts of x: by_rows (axis 1) and by_cols (axis 0), where asked for.  The caller has x's device current.
void cast_into(const at::Tensor& given, int code, int rule, bool square, uint32_t seed, uint32_t offset, Scaled* by_rows,
               Scaled* by_cols, void* stream) {
  const at::Tensor x = given.resolve_neg();
  const int x_code = dtype_code(x.scalar_type());
  if (!wide(x_code)) type_error("expected FP32, BF16 or FP16 input, got " + name_of(x.scalar_type()));
  if (x.dim() != 2) value_error("block_cast takes a matrix, not " + std::to_string(x.dim()) + " dimensions");
  if (!x.is_cuda()) value_error("block_cast requires a GPU tensor");
  const int64_t stride = row_stride(x, "block_cast"), rows = x.size(0), cols = x.size(1);
  sr_block_output out[2] = {};
  if (by_rows) {
    *by_rows = new_scaled(rows, cols, code, square, x.device());
    out[0] = {memory(by_rows->data), memory(by_rows->scale), by_rows->data.stride(0), std::max<int64_t>(blocks(cols), 1)};
  }
  if (by_cols) {
    *by_cols = new_scaled(cols, rows, code, square, x.device());
    out[1] = {memory(by_cols->data), memory(by_cols->scale), by_cols->data.stride(0), std::max<int64_t>(blocks(rows), 1)};
  }
  if (rows && cols)
    checked(g_cast(memory(x), stride, rows, cols, x_code, code, rule, square, seed, offset, by_rows ? &out[0] : nullptr,
                   by_cols ? &out[1] : nullptr, stream));
}

// The distance between matrices of a stack, and a matrix of it.
int64_t stack_stride(const at::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : 0; }
at::Tensor matrix_of(const at::Tensor& x) { return x.dim() == 3 ? x.select(0, 0) : x; }

sr_block_matrix operand(const at::Tensor& data, const at::Tensor& scale, const std::string& name) {
  const int code = dtype_code(data.scalar_type());
  if (code != SR_E4M3 && code != SR_E5M2) type_error(name + ": data must be FP8 (E4M3 or E5M2), got " + name_of(data.scalar_type()));
  const bool e8m0 = scale.scalar_type() == c10::ScalarType::Float8_e8m0fnu;
  if (!e8m0 && scale.scalar_type() != c10::ScalarType::Float)
    type_error(name + ": scales must be torch.float8_e8m0fnu or torch.float32, got " + name_of(scale.scalar_type()));
  if (data.dim() != 2 || scale.dim() != 2) value_error(name + ": data and scales must be matrices");
  if (!data.is_cuda() || scale.device() != data.device())
    value_error(name + ": data and scales must be on the same GPU device");
  const int64_t rows = data.size(0), k = data.size(1);
  if (scale.size(1) != blocks(k) || (scale.size(0) != rows && scale.size(0) != blocks(rows))) {
    auto shape = [](int64_t a, int64_t b) { return std::to_string(a) + " x " + std::to_string(b); };
    value_error(name + ": scales of a " + shape(rows, k) + " matrix are " + shape(rows, blocks(k)) + " or " +
                shape(blocks(rows), blocks(k)) + ", not " + shape(scale.size(0), scale.size(1)));
  }
  return {memory(data), memory(scale), row_stride(data, name + ": data"), row_stride(scale, name + ": scale"), rows, code,
          e8m0 ? SR_SCALE_E8M0 : SR_SCALE_F32, scale.size(0) == rows ? 1 : SR_BLOCK, 0};
}

// First and one past the last byte a matrix touches.
std::pair<uintptr_t, uintptr_t> span(const at::Tensor& x) {
  const auto start = reinterpret_cast<uintptr_t>(x.const_data_ptr());
  if (!x.numel()) return {start, start};
  int64_t last = 0;
  for (int64_t d = 0; d < x.dim(); ++d) last += (x.size(d) - 1) * x.stride(d);
  return {start, start + static_cast<uintptr_t>((last + 1) * x.element_size())};
}

std::string shape_of(at::IntArrayRef shape) {
  std::string text;
  for (int64_t n : shape) text += (text.empty() ? "" : " x ") + std::to_string(n);
  return text;
}

// Makes `out` a new tensor of this shape and dtype where it is not defined, and else checks that it can take the result
// of these operands; sets out_code.  Returns the distance between its rows.
int64_t result_of(at::Tensor& out, at::IntArrayRef shape, int& out_code, const Scaled& a, const Scaled& b, const char* name) {
  if (!out.defined()) {
    if (out_code < 0) out_code = SR_BF16;
    out = at::empty(shape, at::TensorOptions().device(a.data.device()).dtype(scalar_type(out_code)));
    return shape.back();
  }
  if (!wide(dtype_code(out.scalar_type())) || (out_code >= 0 && dtype_code(out.scalar_type()) != out_code))
    type_error("out has dtype " + name_of(out.scalar_type()));
  out_code = dtype_code(out.scalar_type());
  if (out.sizes() != shape || out.device() != a.data.device())
    value_error("out must be a " + shape_of(shape) + " tensor on " + a.data.device().str());
  int64_t stride = std::max<int64_t>(shape.back(), 1);
  if (out.numel()) {
    stride = row_stride(matrix_of(out), "out");
    if (out.dim() == 3 && out.size(0) > 1 && out.stride(0) < (out.size(1) - 1) * stride + out.size(2))
      value_error("out requires matrices that do not overlap");
  }
  const auto [start, end] = span(out);
  for (const at::Tensor* t : {&a.data, &a.scale, &b.data, &b.scale}) {
    const auto [first, last] = span(*t);
    if (start < last && first < end) value_error("out must not overlap the operands");
  }
  // As torch's own out= functions: the write is not differentiable, and whoever saved the tensor must notice it.
  if (out.requires_grad() && c10::GradMode::is_enabled())
    throw Refusal(PyExc_RuntimeError,
                  std::string("out requires grad, and ") + name + " records no gradients: call it under torch.no_grad()");
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
  return stride;
}

// The caller has the operands' device current.
at::Tensor matmul(const Scaled& a, const Scaled& b, int out_code, at::Tensor out, void* stream) {
  const sr_block_matrix left = operand(a.data, a.scale, "a"), right = operand(b.data, b.scale, "b");
  const int64_t k = a.data.size(1), m = left.rows, n = right.rows;
  if (b.data.device() != a.data.device()) value_error("a and b must be on the same GPU device");
  if (b.data.size(1) != k)
    value_error("a and b contract " + std::to_string(k) + " and " + std::to_string(b.data.size(1)) + " values");
  if (left.scale_type != right.scale_type) type_error("a and b must have scales of one type");
  const int64_t stride = result_of(out, {m, n}, out_code, a, b, "block_matmul");
  if (m && n) checked(g_matmul(&left, &right, k, memory(out), stride, out_code, stream));
  return out;
}

// x as rows of its last size, copied only where its layout needs it.
at::Tensor as_rows(const at::Tensor& x) {
  int64_t rows = 1;
  for (int64_t d = 0; d + 1 < x.dim(); ++d) rows *= x.size(d);
  const int64_t cols = x.size(-1);
  at::Tensor flat = x.dim() == 2 ? x : x.reshape({rows, cols});
  if ((cols > 1 && flat.stride(1) != 1) || (rows > 1 && flat.stride(0) < cols)) flat = flat.contiguous();
  return flat;
}

// ---- rows sorted into groups ----

// The groups that a tensor of sizes describes, on `device`.
sr_groups groups_of(const at::Tensor& sizes, const at::Device& device) {
  const bool wide = sizes.scalar_type() == c10::ScalarType::Long;
  if (!wide && sizes.scalar_type() != c10::ScalarType::Int) type_error("sizes must be torch.int32 or torch.int64, got " + name_of(sizes.scalar_type()));
  if (sizes.dim() != 1 || !sizes.is_contiguous()) value_error("sizes must be one row of consecutive numbers");
  if (sizes.device() != device) value_error("sizes must be on the same GPU device");
  if (sizes.size(0) > SR_MATRIX_GROUPS)
    value_error(std::to_string(sizes.size(0)) + " groups: at most " + std::to_string(SR_MATRIX_GROUPS));
  return {memory(sizes), static_cast<int>(sizes.size(0)), wide};
}

// The casts of the rows of x, blocks along the rows ending with each group.
void cast_groups_into(const at::Tensor& given, const at::Tensor& sizes, int code, int rule, uint32_t seed, uint32_t offset,
                      Scaled* by_rows, Scaled* by_cols, void* stream) {
  const at::Tensor x = given.resolve_neg();
  const int x_code = dtype_code(x.scalar_type());
  if (!wide(x_code)) type_error("expected FP32, BF16 or FP16 input, got " + name_of(x.scalar_type()));
  if (x.dim() != 2) value_error("groups are rows of a matrix, not of " + std::to_string(x.dim()) + " dimensions");
  if (!x.is_cuda()) value_error("grouped_block_cast requires a GPU tensor");
  const sr_groups groups = groups_of(sizes, x.device());
  const int64_t stride = row_stride(x, "grouped_block_cast"), rows = x.size(0), cols = x.size(1);
  const int64_t columns = g_columns(rows, groups.count);
  if (by_cols) *by_cols = new_scaled(cols, columns, code, false, x.device());
  if (!by_cols || !columns) {  // nothing depends on the groups
    if (by_rows) cast_into(x, code, rule, false, seed, offset, by_rows, nullptr, stream);
    return;
  }
  sr_block_output out[2] = {};
  if (by_rows) {
    *by_rows = new_scaled(rows, cols, code, false, x.device());
    out[0] = {memory(by_rows->data), memory(by_rows->scale), by_rows->data.stride(0), std::max<int64_t>(blocks(cols), 1)};
  }
  out[1] = {memory(by_cols->data), memory(by_cols->scale), by_cols->data.stride(0), blocks(columns)};
  if (cols)
    checked(g_grouped_cast(memory(x), stride, rows, cols, x_code, code, rule, seed, offset, &groups, by_rows ? &out[0] : nullptr,
                           &out[1], stream));
}

// A stack of matrices, rows on 16 bytes.
Scaled new_stack(int64_t count, int64_t rows, int64_t k, int code, bool square, const at::Device& device) {
  const auto options = at::TensorOptions().device(device);
  const int64_t ld = (k + 15) / 16 * 16;
  return {at::empty_strided({count, rows, k}, {rows * ld, ld, 1}, options.dtype(scalar_type(code))),
          at::empty({count, square ? blocks(rows) : rows, blocks(k)}, options.dtype(c10::ScalarType::Float8_e8m0fnu))};
}

// The casts of every matrix of x.
void cast_stack_into(const at::Tensor& given, int code, int rule, bool square, uint32_t seed, uint32_t offset, Scaled* by_rows,
                     Scaled* by_cols, void* stream) {
  const at::Tensor x = given.resolve_neg();
  const int x_code = dtype_code(x.scalar_type());
  if (!wide(x_code)) type_error("expected FP32, BF16 or FP16 input, got " + name_of(x.scalar_type()));
  if (x.dim() != 3) value_error("a stack of matrices has three dimensions, not " + std::to_string(x.dim()));
  if (!x.is_cuda()) value_error("grouped_block_cast requires a GPU tensor");
  const int64_t count = x.size(0), rows = x.size(1), cols = x.size(2);
  if (count > SR_MATRIX_GROUPS) value_error(std::to_string(count) + " matrices: at most " + std::to_string(SR_MATRIX_GROUPS));
  sr_block_stack out[2] = {};
  auto make = [&](Scaled* to, sr_block_stack& stack, int64_t r, int64_t c) {
    if (!to) return;
    *to = new_stack(count, r, c, code, square, x.device());
    stack = {{memory(to->data), memory(to->scale), to->data.stride(1), std::max<int64_t>(blocks(c), 1)},
             to->data.stride(0),
             to->scale.size(1) * to->scale.size(2)};
  };
  make(by_rows, out[0], rows, cols);
  make(by_cols, out[1], cols, rows);
  if (x.numel())
    checked(g_stacked_cast(memory(x), stack_stride(x), row_stride(matrix_of(x), "grouped_block_cast"), count, rows, cols, x_code,
                           code, rule, square, seed, offset, by_rows ? &out[0] : nullptr, by_cols ? &out[1] : nullptr, stream));
}

// The caller has the operands' device current.
at::Tensor grouped_product(const Scaled& a, const Scaled& b, const at::Tensor& sizes, int out_code, at::Tensor out, void* stream) {
  const bool stacked = b.data.dim() == 3;
  const sr_block_matrix left = operand(a.data, a.scale, "a");
  if (stacked && (b.scale.dim() != 3 || b.scale.size(0) != b.data.size(0)))
    value_error("b: a stack of matrices has a stack of as many scales");
  const sr_groups groups = groups_of(sizes, a.data.device());
  const int64_t k = a.data.size(1);
  if (b.data.device() != a.data.device()) value_error("a and b must be on the same GPU device");
  if (b.data.dim() < 2 || b.data.size(-1) != k)
    value_error("a and b contract " + std::to_string(k) + " and " + std::to_string(b.data.dim() ? b.data.size(-1) : 0) + " values");
  if (stacked && b.data.size(0) != groups.count)
    value_error("b has " + std::to_string(b.data.size(0)) + " matrices for " + std::to_string(groups.count) + " groups");
  const int64_t m = left.rows, n = b.data.size(-2), count = groups.count;
  const bool given = out.defined();
  if (given) {
    const auto [start, end] = span(out);
    const auto [first, last] = span(sizes);
    if (start < last && first < end) value_error("out must not overlap the sizes");
  }
  if (stacked) {
    sr_block_matrix right{};
    if (count) {
      right = operand(matrix_of(b.data), matrix_of(b.scale), "b");
      if (left.scale_type != right.scale_type) type_error("a and b must have scales of one type");
    }
    const int64_t stride = result_of(out, {m, n}, out_code, a, b, "grouped_block_matmul");  // after every refusal
    if (!m || !n) return out;
    if (!count) return given ? out : out.zero_();
    checked(g_grouped_matmul(&left, &right, stack_stride(b.data), stack_stride(b.scale), k, &groups, memory(out), stride, out_code,
                             !given, stream));
    return out;
  }
  const sr_block_matrix right = operand(b.data, b.scale, "b");
  if (left.scale_type != right.scale_type) type_error("a and b must have scales of one type");
  if (k % SR_BLOCK) value_error("the columns of padded groups are a multiple of " + std::to_string(SR_BLOCK) + ", not " + std::to_string(k));
  for (const sr_block_matrix* x : {&left, &right})
    if (k && (reinterpret_cast<uintptr_t>(x->data) % 16 || x->ld % 16)) value_error("rows of padded groups must start on 16 bytes");
  const int64_t stride = result_of(out, {count, m, n}, out_code, a, b, "grouped_block_matmul");
  if (out.numel())
    checked(g_grouped_contract(&left, &right, k, &groups, memory(out), stride, out.size(0) > 1 ? out.stride(0) : m * stride, out_code,
                               stream));
  return out;
}

// A stack with consecutive columns and rows that do not overlap, copied only where its layout needs it.
at::Tensor as_stack(const at::Tensor& x) {
  const bool copy = (x.size(2) > 1 && x.stride(2) != 1) || (x.size(1) > 1 && x.stride(1) < x.size(2));
  return copy ? x.contiguous() : x;
}

// ---- low-rank adapters ----

// The adapters of rows (..., k), checked; `a`, `b` and `index` are made contiguous.
struct AdapterSet {
  at::Tensor a, b, index, scaling;
  sr_adapters g{};
  int64_t rows = 0, k = 0, n = 0;

  AdapterSet(const at::Tensor& x, const at::Tensor& given_a, const at::Tensor& given_b, const at::Tensor& given_index,
             const at::Tensor& given_scaling, double scale) {
    const int code = dtype_code(x.scalar_type());
    if (!wide(code)) type_error("expected FP32, BF16 or FP16 input, got " + name_of(x.scalar_type()));
    if (!x.is_cuda()) value_error("adapter_add requires GPU tensors");
    for (const auto& [t, name] : {std::pair<const at::Tensor&, const char*>{given_a, "a"}, {given_b, "b"}}) {
      if (t.scalar_type() != x.scalar_type()) type_error(std::string(name) + " must have x's dtype, got " + name_of(t.scalar_type()));
      if (t.device() != x.device()) value_error(std::string(name) + " must be on x's device");
      if (t.dim() != 3) value_error(std::string(name) + " is a stack of matrices, not " + std::to_string(t.dim()) + " dimensions");
    }
    if (x.dim() < 1) value_error("x has rows of values");
    k = x.size(-1);
    n = given_b.size(1);
    rows = 1;
    for (int64_t d = 0; d + 1 < x.dim(); ++d) rows *= x.size(d);
    const int64_t count = given_a.size(0), rank = given_a.size(1);
    if (given_b.size(0) != count || given_b.size(2) != rank || given_a.size(2) != k)
      value_error("x of " + std::to_string(k) + " values, a " + shape_of(given_a.sizes()) + " and b " + shape_of(given_b.sizes()) +
                  " do not match");
    if (rank < 1 || rank > 128) value_error("adapters have rank 1 to 128, not " + std::to_string(rank));
    if (count > SR_MATRIX_ADAPTERS) value_error(std::to_string(count) + " adapters: at most " + std::to_string(SR_MATRIX_ADAPTERS));
    if (given_index.scalar_type() != c10::ScalarType::Int && given_index.scalar_type() != c10::ScalarType::Long)
      type_error("index must be torch.int32 or torch.int64, got " + name_of(given_index.scalar_type()));
    if (given_index.device() != x.device()) value_error("index must be on x's device");
    if (given_index.dim() != x.dim() - 1 || given_index.sizes() != x.sizes().slice(0, x.dim() - 1))
      value_error("index must hold an adapter for each row of x");
    if (given_scaling.defined()) {
      if (given_scaling.scalar_type() != c10::ScalarType::Float) type_error("scaling must be torch.float32, got " + name_of(given_scaling.scalar_type()));
      if (given_scaling.device() != x.device() || given_scaling.dim() != 1 || given_scaling.size(0) != count)
        value_error("scaling must hold a number for each adapter on x's device");
      scaling = given_scaling.detach().resolve_neg().contiguous();
    }
    a = given_a.detach().resolve_neg().contiguous();
    b = given_b.detach().resolve_neg().contiguous();
    index = given_index.contiguous();
    g = {memory(a), memory(b), memory(index), scaling.defined() && count ? static_cast<const float*>(memory(scaling)) : nullptr,
         static_cast<float>(scale), static_cast<int>(count), static_cast<int>(rank), code, index.scalar_type() == c10::ScalarType::Long};
  }
};

// base plus the updates; `low` is what the gradients need.
at::Tensor add_adapters(const at::Tensor& base, const at::Tensor& x, const AdapterSet& set, at::Tensor out, at::Tensor& low, void* stream) {
  if (base.scalar_type() != x.scalar_type()) type_error("base must have x's dtype, got " + name_of(base.scalar_type()));
  if (base.device() != x.device()) value_error("base must be on x's device");
  auto shape = x.sizes().vec();
  shape.back() = set.n;
  if (base.sizes() != at::IntArrayRef(shape)) value_error("base must be " + shape_of(shape) + ", not " + shape_of(base.sizes()));
  const at::Tensor rows = as_rows(x.detach().resolve_neg()), from = as_rows(base.detach().resolve_neg());
  const bool given = out.defined();
  at::Tensor to;  // out as rows
  if (given) {
    if (out.scalar_type() != x.scalar_type()) type_error("out has dtype " + name_of(out.scalar_type()));
    if (out.sizes() != base.sizes() || out.device() != x.device()) value_error("out must be a " + shape_of(shape) + " tensor on " + x.device().str());
    if (out.is_neg()) value_error("lazily negated views cannot be used: call resolve_neg()");
    if (out.requires_grad() && c10::GradMode::is_enabled())
      throw Refusal(PyExc_RuntimeError, "out requires grad, and a given out records no gradients: call adapter_add under torch.no_grad()");
    to = out.dim() == 2 ? out : out.view({set.rows, set.n});
    row_stride(to, "out");
    const auto [start, end] = span(out);
    const bool same = from.const_data_ptr() == to.const_data_ptr() && from.sizes() == to.sizes() && from.strides() == to.strides();
    for (const at::Tensor* t : {&rows, &set.a, &set.b, &set.index, &set.scaling, &from}) {
      if (!t->defined() || (t == &from && same)) continue;
      const auto [first, last] = span(*t);
      if (start < last && first < end) value_error("out must not overlap the operands, but for base itself");
    }
    if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
  } else {
    out = at::empty(shape, x.options());
    to = out.view({set.rows, set.n});
  }
  low = at::empty({g_adapter_low(set.rows, set.k, set.g.rank, set.g.dtype)}, x.options().dtype(c10::ScalarType::Float));
  checked(g_adapter_add(&set.g, memory(rows), row_stride(rows, "x"), set.k, memory(from), row_stride(from, "base"), set.n, set.rows,
                        memory(to), row_stride(to, "out"), static_cast<float*>(memory(low)), stream));
  return out;
}

// ---- nodes of the autograd graph ----

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The engine runs a node on the stream of its forward pass; who calls one directly has it run on the caller's, where its
// workspace and results belong too.
void* current_stream(const at::Device& device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }

// The engine checks the gradients that it passes; a node that is called directly may get any tensor.
void check_gradient(const at::Tensor& dy, at::IntArrayRef shape, int dtype, const at::Device& device) {
  if (dtype_code(dy.scalar_type()) != dtype || dy.sizes() != shape || dy.device() != device)
    value_error("the gradient must be a " + shape_of(shape) + " tensor of " + name_of(scalar_type(dtype)) + " on " + device.str());
}

// Runs a node's gradients: a failed launch becomes an error here, where the message of this thread's last one is, and
// the gradients cannot be differentiated again.
template <class Body>
variable_list gradients(const char* name, Body&& body) {
  const bool recorded = c10::GradMode::is_enabled();
  variable_list out;
  try {
    const at::AutoGradMode off(false);
    out = body();
  } catch (const Status& status) {
    throw std::runtime_error(std::string(name) + " failed (" + std::to_string(status.code) + "): " + g_last_error());
  }
  if (!recorded) return out;
  for (at::Tensor& t : out)
    if (t.defined()) t = t.detach().set_requires_grad(true);
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate twice: the gradients of ") + name + " have none", static_cast<int64_t>(out.size()));
  return (*error)(std::move(out));
}

struct GroupedLinear : torch::autograd::Function<GroupedLinear> {
  struct Options {
    int format[6];
    uint32_t seed[3];
    void* stream;
  };
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const at::Tensor& sizes, bool need_x,
                            bool need_w, const Options& o) {
    Scaled qx, qx_t, qw, qw_t;
    const at::Tensor rows = as_rows(x.detach()), weight = as_stack(w.detach());
    cast_groups_into(rows, sizes, o.format[0], o.format[1], o.seed[0], 0, &qx, need_w ? &qx_t : nullptr, o.stream);
    cast_stack_into(weight, o.format[2], o.format[3], true, o.seed[1], 0, &qw, need_x ? &qw_t : nullptr, o.stream);
    if (need_x || need_w) {
      ctx->save_for_backward({sizes, qx_t.data, qx_t.scale, qw_t.data, qw_t.scale});
      ctx->saved_data["rule"] = std::vector<int64_t>{o.format[4], o.format[5], o.seed[2], dtype_code(x.scalar_type()), dtype_code(w.scalar_type()),
                                                     x.size(0), w.size(1)};
    }
    return grouped_product(qx, qw, sizes, dtype_code(x.scalar_type()), at::Tensor(), o.stream);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return gradients("grouped_block_linear", [&] {
      const variable_list saved = ctx->get_saved_variables();
      const std::vector<int64_t> rule = ctx->saved_data["rule"].toIntVector();
      const at::Tensor& dy = grads[0];
      at::Tensor dx, dw;
      if (dy.defined()) {
        const c10::DeviceGuard guard(dy.device());
        void* stream = current_stream(dy.device());
        check_gradient(dy, {rule[5], rule[6]}, static_cast<int>(rule[3]), saved[0].device());
        const Scaled x{saved[1], saved[2]}, w{saved[3], saved[4]};
        const bool need_x = w.data.defined() && ctx->needs_input_grad(0), need_w = x.data.defined() && ctx->needs_input_grad(1);
        Scaled by_rows, by_cols;
        cast_groups_into(as_rows(dy.detach()), saved[0], static_cast<int>(rule[0]), static_cast<int>(rule[1]),
                         static_cast<uint32_t>(rule[2]), 0, need_x ? &by_rows : nullptr, need_w ? &by_cols : nullptr, stream);
        if (need_x) dx = grouped_product(by_rows, w, saved[0], static_cast<int>(rule[3]), at::Tensor(), stream);
        if (need_w) dw = grouped_product(by_cols, x, saved[0], static_cast<int>(rule[4]), at::Tensor(), stream);
      }
      return variable_list{dx, dw, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    });
  }
};

struct AdapterAdd : torch::autograd::Function<AdapterAdd> {
  struct Options {
    at::Tensor scaling;  // or undefined: `scale` for all
    double scale;
    void* stream;
  };
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& base, const at::Tensor& x, const at::Tensor& a, const at::Tensor& b,
                            const at::Tensor& index, const Options& o) {
    at::Tensor low;
    const at::Tensor y = add_adapters(base, x, AdapterSet(x, a, b, index, o.scaling, o.scale), at::Tensor(), low, o.stream);
    ctx->save_for_backward({x, a, b, index, o.scaling, low});
    ctx->saved_data["scale"] = o.scale;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return gradients("adapter_add", [&] {
      const variable_list saved = ctx->get_saved_variables();
      const at::Tensor &x = saved[0], &a = saved[1], &b = saved[2], &dy = grads[0];
      at::Tensor dbase, dx, da, db;
      const bool need_x = ctx->needs_input_grad(1), need_a = ctx->needs_input_grad(2), need_b = ctx->needs_input_grad(3);
      if (dy.defined()) {
        const c10::DeviceGuard guard(dy.device());
        void* stream = current_stream(dy.device());
        if (ctx->needs_input_grad(0)) dbase = dy;
        if (need_x || need_a || need_b) {
          const AdapterSet set(x, a, b, saved[3], saved[4], ctx->saved_data["scale"].toDouble());
          auto shape = x.sizes().vec();
          shape.back() = set.n;
          check_gradient(dy, shape, set.g.dtype, x.device());
          const at::Tensor low = saved[5].contiguous();  // a hook of saved tensors may have put another in its place
          if (low.scalar_type() != c10::ScalarType::Float || low.device() != x.device() ||
              low.numel() != g_adapter_low(set.rows, set.k, set.g.rank, set.g.dtype))
            value_error("the tensors kept for the backward pass have changed their types or sizes");
          const at::Tensor rows = as_rows(x.detach().resolve_neg()), from = as_rows(dy.detach().resolve_neg());
          if (need_x) dx = at::empty(x.sizes(), x.options());
          if (need_a) da = at::empty(a.sizes(), a.options());
          if (need_b) db = at::empty(b.sizes(), b.options());
          const at::Tensor workspace = at::empty({g_adapter_workspace(set.rows, set.k, set.n, set.g.count, set.g.rank, set.g.dtype)},
                                                 x.options().dtype(c10::ScalarType::Byte));
          auto place = [](const at::Tensor& t) { return t.defined() ? memory(t) : nullptr; };
          checked(g_adapter_backward(&set.g, memory(rows), row_stride(rows, "x"), set.k, memory(from), row_stride(from, "dy"), set.n,
                                     set.rows, static_cast<const float*>(memory(low)), place(dx), set.k, place(da), place(db),
                                     memory(workspace), stream));
        }
      }
      return variable_list{dbase, dx, da, db, at::Tensor(), at::Tensor()};
    });
  }
};

bool bound() {
  return g_cast && g_matmul && g_orthogonalize && g_workspace && g_columns && g_grouped_cast && g_stacked_cast &&
         g_grouped_matmul && g_grouped_contract && g_adapter_low && g_adapter_workspace && g_adapter_add && g_adapter_backward &&
         g_last_error;
}

// Runs `body` as the entries promise; nullptr with an exception set, the
// status, or what `result` makes of the outcome.
template <class Body, class Result>
PyObject* run(const at::Device& device, Body body, Result result) {
  if (!bound()) {
    PyErr_SetString(PyExc_RuntimeError, "the native entries are not bound to the library");
    return nullptr;
  }
  int status = 0;
  std::string message;
  PyObject* type = nullptr;
  std::optional<python_error> raised;  // by a hook of saved tensors, in Python
  Py_BEGIN_ALLOW_THREADS
  try {
    const c10::OptionalDeviceGuard guard(device.is_cuda() ? c10::optional<at::Device>(device) : c10::nullopt);
    body();
  } catch (const Refusal& refusal) {
    type = refusal.type;
    message = refusal.what();
  } catch (const Status& s) {
    status = s.code;
  } catch (python_error& error) {
    raised.emplace(std::move(error));
  } catch (const c10::OutOfMemoryError& error) {
    type = g_out_of_memory;
    message = error.what_without_backtrace();
  } catch (const std::exception& error) {
    type = PyExc_RuntimeError;
    message = error.what();
  } catch (...) {
    type = PyExc_RuntimeError;
    message = "unknown C++ exception in a native entry";
  }
  Py_END_ALLOW_THREADS
  if (raised) {
    raised->restore();
    return nullptr;
  }
  if (type) {
    PyErr_SetString(type, message.c_str());
    return nullptr;
  }
  if (status) return PyLong_FromLong(status);
  return result();
}

PyObject* wrap(const at::Tensor& x) {
  if (!x.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(x);
}

// A tuple of the tensors; None in the place of undefined ones.
PyObject* wrap_all(std::initializer_list<const at::Tensor*> tensors) {
  PyObject* tuple = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
  if (!tuple) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor* t : tensors) {
    PyObject* item = wrap(*t);
    if (!item) {
      Py_DECREF(tuple);
      return nullptr;
    }
    PyTuple_SET_ITEM(tuple, i++, item);
  }
  return tuple;
}

// The casts of the axes `wanted`, flat.
PyObject* wrap_casts(const std::string& wanted, const Scaled& by_rows, const Scaled& by_cols) {
  const Scaled &first = wanted[0] == '1' ? by_rows : by_cols, &second = wanted[0] == '1' ? by_cols : by_rows;
  if (wanted.size() == 1) return wrap_all({&first.data, &first.scale});
  return wrap_all({&first.data, &first.scale, &second.data, &second.scale});
}

PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long at[14];
  if (!PyArg_ParseTuple(args, "KKKKKKKKKKKKKK", &at[0], &at[1], &at[2], &at[3], &at[4], &at[5], &at[6], &at[7], &at[8], &at[9],
                        &at[10], &at[11], &at[12], &at[13]))
    return nullptr;
  auto keep = [](auto& function, unsigned long long value) {
    function = reinterpret_cast<std::remove_reference_t<decltype(function)>>(address(value));
  };
  keep(g_cast, at[0]);
  keep(g_matmul, at[1]);
  keep(g_orthogonalize, at[2]);
  keep(g_workspace, at[3]);
  keep(g_columns, at[4]);
  keep(g_grouped_cast, at[5]);
  keep(g_stacked_cast, at[6]);
  keep(g_grouped_matmul, at[7]);
  keep(g_grouped_contract, at[8]);
  keep(g_adapter_low, at[9]);
  keep(g_adapter_workspace, at[10]);
  keep(g_adapter_add, at[11]);
  keep(g_adapter_backward, at[12]);
  keep(g_last_error, at[13]);
  if (!bound()) {
    PyErr_SetString(PyExc_ValueError, "null entry point address");
    return nullptr;
  }
  PyObject* torch = PyImport_ImportModule("torch");
  g_out_of_memory = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
  Py_XDECREF(torch);
  if (!g_out_of_memory) return nullptr;
  Py_RETURN_NONE;
}

PyObject* block_cast(PyObject*, PyObject* args) {
  PyObject* object;
  int code, rule, square;
  const char* axes;
  unsigned long long seed, offset, stream;
  if (!PyArg_ParseTuple(args, "OiiisKKK", &object, &code, &rule, &square, &axes, &seed, &offset, &stream)) return nullptr;
  const at::Tensor& x = tensor(object);
  const std::string wanted(axes);
  Scaled by_rows, by_cols;
  return run(
      x.device(),
      [&] {
        cast_into(x, code, rule, square, static_cast<uint32_t>(seed), static_cast<uint32_t>(offset),
                  wanted.find('1') != std::string::npos ? &by_rows : nullptr,
                  wanted.find('0') != std::string::npos ? &by_cols : nullptr, address(stream));
      },
      [&] { return wrap_casts(wanted, by_rows, by_cols); });
}

PyObject* block_matmul(PyObject*, PyObject* args) {
  PyObject *a_data, *a_scale, *b_data, *b_scale, *out_object;
  int out_code;
  unsigned long long stream;
  if (!PyArg_ParseTuple(args, "OOOOiOK", &a_data, &a_scale, &b_data, &b_scale, &out_code, &out_object, &stream)) return nullptr;
  for (PyObject* object : {a_data, a_scale, b_data, b_scale})
    if (!THPVariable_Check(object)) type_error("operands must be BlockScaled pairs of tensors");
  const Scaled a{tensor(a_data), tensor(a_scale)}, b{tensor(b_data), tensor(b_scale)};
  at::Tensor out;
  if (out_object != Py_None) out = tensor(out_object);
  const bool given = out.defined();
  at::Tensor result;
  return run(
      a.data.device(), [&] { result = matmul(a, b, out_code, out, address(stream)); },
      [&]() -> PyObject* {
        if (!given) return wrap(result);
        Py_INCREF(out_object);
        return out_object;
      });
}

PyObject* linear_forward(PyObject*, PyObject* args) {
  PyObject *x_object, *w_object;
  int format[6], need_x, need_w;
  unsigned long long seed[3], stream;
  if (!PyArg_ParseTuple(args, "OO(iiiiii)(KKK)ppK", &x_object, &w_object, &format[0], &format[1], &format[2], &format[3],
                        &format[4], &format[5], &seed[0], &seed[1], &seed[2], &need_x, &need_w, &stream))
    return nullptr;
  const at::Tensor &x = tensor(x_object), &w = tensor(w_object);
  Scaled qx, qx_t, qw, qw_t;
  at::Tensor y;
  return run(
      x.device(),
      [&] {
        const at::Tensor rows = as_rows(x.detach()), weight = as_rows(w.detach());
        cast_into(rows, format[0], format[1], false, static_cast<uint32_t>(seed[0]), 0, &qx, need_w ? &qx_t : nullptr, address(stream));
        cast_into(weight, format[2], format[3], true, static_cast<uint32_t>(seed[1]), 0, &qw, need_x ? &qw_t : nullptr, address(stream));
        y = matmul(qx, qw, dtype_code(x.scalar_type()), at::Tensor(), address(stream));
        if (x.dim() != 2) {
          auto shape = x.sizes().vec();
          shape.back() = w.size(0);
          y = y.view(shape);
        }
      },
      [&] { return wrap_all({&y, &qx_t.data, &qx_t.scale, &qw_t.data, &qw_t.scale}); });
}

PyObject* linear_backward(PyObject*, PyObject* args) {
  PyObject *dy_object, *x_data, *x_scale, *w_data, *w_scale;
  int code, rule, dx_code, dw_code;
  unsigned long long seed, stream;
  if (!PyArg_ParseTuple(args, "OOOOOiiKiiK", &dy_object, &x_data, &x_scale, &w_data, &w_scale, &code, &rule, &seed, &dx_code,
                        &dw_code, &stream))
    return nullptr;
  const at::Tensor& dy = tensor(dy_object);
  const bool need_w = x_data != Py_None, need_x = w_data != Py_None;
  Scaled x, w, by_rows, by_cols;
  if (need_w) x = {tensor(x_data), tensor(x_scale)};
  if (need_x) w = {tensor(w_data), tensor(w_scale)};
  at::Tensor dx, dw;
  return run(
      dy.device(),
      [&] {
        const at::Tensor rows = as_rows(dy.detach());
        cast_into(rows, code, rule, false, static_cast<uint32_t>(seed), 0, need_x ? &by_rows : nullptr,
                  need_w ? &by_cols : nullptr, address(stream));
        if (need_x) {
          dx = matmul(by_rows, w, dx_code, at::Tensor(), address(stream));
          if (dy.dim() != 2) {
            auto shape = dy.sizes().vec();
            shape.back() = w.data.size(0);
            dx = dx.view(shape);
          }
        }
        if (need_w) dw = matmul(by_cols, x, dw_code, at::Tensor(), address(stream));
      },
      [&] { return wrap_all({&dx, &dw}); });
}

PyObject* grouped_cast(PyObject*, PyObject* args) {
  PyObject *object, *sizes_object;
  int code, rule, square;
  const char* axes;
  unsigned long long seed, offset, stream;
  if (!PyArg_ParseTuple(args, "OOiiisKKK", &object, &sizes_object, &code, &rule, &square, &axes, &seed, &offset, &stream))
    return nullptr;
  const at::Tensor& x = tensor(object);
  at::Tensor sizes;
  if (sizes_object != Py_None) sizes = tensor(sizes_object);
  const std::string wanted(axes);
  Scaled by_rows, by_cols;
  return run(
      x.device(),
      [&] {
        Scaled* rows = wanted.find('1') != std::string::npos ? &by_rows : nullptr;
        Scaled* cols = wanted.find('0') != std::string::npos ? &by_cols : nullptr;
        const uint32_t s = static_cast<uint32_t>(seed), o = static_cast<uint32_t>(offset);
        if (!sizes.defined()) {
          cast_stack_into(x, code, rule, square, s, o, rows, cols, address(stream));
        } else {
          if (square) value_error("groups of rows take blocks of one row");
          cast_groups_into(x, sizes, code, rule, s, o, rows, cols, address(stream));
        }
      },
      [&] { return wrap_casts(wanted, by_rows, by_cols); });
}

PyObject* grouped_matmul(PyObject*, PyObject* args) {
  PyObject *a_data, *a_scale, *b_data, *b_scale, *sizes_object, *out_object;
  int out_code;
  unsigned long long stream;
  if (!PyArg_ParseTuple(args, "OOOOOiOK", &a_data, &a_scale, &b_data, &b_scale, &sizes_object, &out_code, &out_object, &stream))
    return nullptr;
  for (PyObject* object : {a_data, a_scale, b_data, b_scale})
    if (!THPVariable_Check(object)) type_error("operands must be BlockScaled pairs of tensors");
  const Scaled a{tensor(a_data), tensor(a_scale)}, b{tensor(b_data), tensor(b_scale)};
  const at::Tensor& sizes = tensor(sizes_object);
  at::Tensor out;
  if (out_object != Py_None) out = tensor(out_object);
  const bool given = out.defined();
  at::Tensor result;
  return run(
      a.data.device(), [&] { result = grouped_product(a, b, sizes, out_code, out, address(stream)); },
      [&]() -> PyObject* {
        if (!given) return wrap(result);
        Py_INCREF(out_object);
        return out_object;
      });
}

// No operand may carry a tangent of forward-mode differentiation: the result would lose it without a word.
void refuse_tangents(std::initializer_list<const at::Tensor*> operands, const char* name) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const at::Tensor* t : operands)
    if (t->defined() && t->_fw_grad(0).defined())
      throw Refusal(PyExc_NotImplementedError, std::string(name) + " has no forward-mode derivatives, and an operand has a tangent");
}

PyObject* grouped_linear(PyObject*, PyObject* args) {
  PyObject *x_object, *w_object, *sizes_object;
  GroupedLinear::Options o;
  unsigned long long seed[3], stream;
  if (!PyArg_ParseTuple(args, "OOO(iiiiii)(KKK)K", &x_object, &w_object, &sizes_object, &o.format[0], &o.format[1], &o.format[2],
                        &o.format[3], &o.format[4], &o.format[5], &seed[0], &seed[1], &seed[2], &stream))
    return nullptr;
  for (int k = 0; k < 3; ++k) o.seed[k] = static_cast<uint32_t>(seed[k]);
  o.stream = address(stream);
  const at::Tensor &x = tensor(x_object), &w = tensor(w_object), &sizes = tensor(sizes_object);
  at::Tensor y;
  return run(
      x.device(),
      [&] {
        refuse_tangents({&x, &w}, "grouped_block_linear");
        const bool recorded = c10::GradMode::is_enabled();
        y = GroupedLinear::apply(x, w, sizes, recorded && x.requires_grad(), recorded && w.requires_grad(), o);
      },
      [&] { return wrap(y); });
}

PyObject* adapter_add(PyObject*, PyObject* args) {
  PyObject *base_object, *x_object, *a_object, *b_object, *index_object, *scaling_object, *out_object;
  double scale;
  unsigned long long stream;
  if (!PyArg_ParseTuple(args, "OOOOOOdOK", &base_object, &x_object, &a_object, &b_object, &index_object, &scaling_object, &scale,
                        &out_object, &stream))
    return nullptr;
  const at::Tensor &base = tensor(base_object), &x = tensor(x_object), &a = tensor(a_object), &b = tensor(b_object),
                   &index = tensor(index_object);
  at::Tensor scaling, out, low, result;
  if (scaling_object != Py_None) scaling = tensor(scaling_object);
  if (out_object != Py_None) out = tensor(out_object);
  const bool given = out.defined();
  return run(
      x.device(),
      [&] {
        refuse_tangents({&base, &x, &a, &b, &scaling, &out}, "adapter_add");
        const bool recorded = c10::GradMode::is_enabled() &&
                              (base.requires_grad() || x.requires_grad() || a.requires_grad() || b.requires_grad());
        if (recorded && given)
          throw Refusal(PyExc_RuntimeError, "a given out records no gradients: call adapter_add under torch.no_grad()");
        if (recorded) result = AdapterAdd::apply(base, x, a, b, index, AdapterAdd::Options{scaling, scale, address(stream)});
        else result = add_adapters(base, x, AdapterSet(x, a, b, index, scaling, scale), out, low, address(stream));
      },
      [&]() -> PyObject* {
        if (!given) return wrap(result);
        Py_INCREF(out_object);
        return out_object;
      });
}

PyObject* orthogonalize(PyObject*, PyObject* args) {
  PyObject* object;
  int out_code;
  sr_newton_schulz ns{};
  unsigned long long limit, stream;
  if (!PyArg_ParseTuple(args, "OiffffiKK", &object, &out_code, &ns.a, &ns.b, &ns.c, &ns.eps, &ns.steps, &limit, &stream))
    return nullptr;
  const at::Tensor& x = tensor(object);
  at::Tensor out;
  return run(
      x.device(),
      [&] {
        if (!wide(dtype_code(x.scalar_type()))) type_error("expected FP32, BF16 or FP16 input, got " + name_of(x.scalar_type()));
        if (x.dim() < 2) value_error("orthogonalize takes matrices, not " + std::to_string(x.dim()) + " dimensions");
        if (!x.is_cuda()) value_error("orthogonalize requires a GPU tensor");
        const auto options = at::TensorOptions().device(x.device());
        out = at::empty(x.sizes(), options.dtype(scalar_type(out_code)));
        if (!x.numel()) return;
        const at::Tensor from = x.detach().resolve_neg().contiguous();
        const int64_t rows = x.size(-2), cols = x.size(-1), size = rows * cols, batch = x.numel() / size;
        const int64_t one = std::max<int64_t>(g_workspace(1, rows, cols), 1);
        const int64_t each = std::min<int64_t>({batch, SR_MATRIX_BATCH, std::max<int64_t>(static_cast<int64_t>(limit) / one, 1)});
        const at::Tensor workspace = at::empty({g_workspace(each, rows, cols)}, options.dtype(c10::ScalarType::Byte));
        for (int64_t first = 0; first < batch; first += each)
          checked(g_orthogonalize(static_cast<const char*>(memory(from)) + first * size * from.element_size(),
                                  static_cast<char*>(memory(out)) + first * size * out.element_size(),
                                  std::min(each, batch - first), size, size, rows, cols, dtype_code(x.scalar_type()), out_code,
                                  &ns, memory(workspace), address(stream)));
      },
      [&] { return wrap(out); });
}

// Every entry behind one guard for what happens outside run().
template <PyObject* (*Entry)(PyObject*, PyObject*)>
PyObject* guarded(PyObject* self, PyObject* args) {
  try {
    return Entry(self, args);
  } catch (const Refusal& refusal) {
    PyErr_SetString(refusal.type, refusal.what());
  } catch (const std::exception& error) {
    PyErr_SetString(PyExc_RuntimeError, error.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception in a native entry");
  }
  return nullptr;
}

PyMethodDef methods[] = {
    {"bind", guarded<bind>, METH_VARARGS, "Keep the addresses of the C ABI's entry points."},
    {"block_cast", guarded<block_cast>, METH_VARARGS, "Cast a matrix to FP8 with block scales."},
    {"block_matmul", guarded<block_matmul>, METH_VARARGS, "Multiply two block-scaled matrices."},
    {"linear_forward", guarded<linear_forward>, METH_VARARGS, "Forward pass of the block-scaled linear layer."},
    {"linear_backward", guarded<linear_backward>, METH_VARARGS, "Gradients of the block-scaled linear layer."},
    {"grouped_cast", guarded<grouped_cast>, METH_VARARGS, "Cast rows in groups, or a stack of matrices, to FP8 with block scales."},
    {"grouped_matmul", guarded<grouped_matmul>, METH_VARARGS, "Multiply each group's rows by its matrix, or contract its columns."},
    {"grouped_linear", guarded<grouped_linear>, METH_VARARGS, "The grouped linear layer."},
    {"adapter_add", guarded<adapter_add>, METH_VARARGS, "Add each row's low-rank update."},
    {"orthogonalize", guarded<orthogonalize>, METH_VARARGS, "Orthogonalise matrices."},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_matrix", "Native entries of the matrix operators.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__matrix(void) { return PyModule_Create(&module); }
