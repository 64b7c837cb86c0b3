// Native entries of the matrix operators: block casts and products, the
// block-scaled linear layer, and orthogonalisation.
//
// The operators' small calls are bound by the host: through Python checks and
// ctypes a block cast took 30 us around a kernel of 6.  This CPython extension
// makes the tensor checks, allocates the results and calls the C ABI's entry
// points through the addresses the Python side binds once.
//
// bind(block_cast, block_matmul, orthogonalize, orthogonalize_workspace)
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
// Errors of the tensors raise TypeError or ValueError before anything is
// launched.  Every entry runs with the first tensor's device current and the
// GIL released around the launch; `stream` is the raw handle of a stream on
// that device.

#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <stdexcept>
#include <string>

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

// The distance between rows of a matrix with consecutive columns.
int64_t row_stride(const at::Tensor& x, const std::string& what) {
  const int64_t rows = x.size(0), cols = x.size(1);
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

// The caller has the operands' device current.
at::Tensor matmul(const Scaled& a, const Scaled& b, int out_code, at::Tensor out, void* stream) {
  const sr_block_matrix left = operand(a.data, a.scale, "a"), right = operand(b.data, b.scale, "b");
  const int64_t k = a.data.size(1), m = left.rows, n = right.rows;
  if (b.data.device() != a.data.device()) value_error("a and b must be on the same GPU device");
  if (b.data.size(1) != k)
    value_error("a and b contract " + std::to_string(k) + " and " + std::to_string(b.data.size(1)) + " values");
  if (left.scale_type != right.scale_type) type_error("a and b must have scales of one type");
  const auto options = at::TensorOptions().device(a.data.device());
  int64_t stride = n;
  if (out.defined()) {
    if (!wide(dtype_code(out.scalar_type())) || (out_code >= 0 && dtype_code(out.scalar_type()) != out_code))
      type_error("out has dtype " + name_of(out.scalar_type()));
    out_code = dtype_code(out.scalar_type());
    if (out.dim() != 2 || out.size(0) != m || out.size(1) != n || out.device() != a.data.device())
      value_error("out must be a " + std::to_string(m) + " x " + std::to_string(n) + " tensor on " + a.data.device().str());
    stride = row_stride(out, "out");
    const auto [start, end] = span(out);
    for (const at::Tensor* t : {&a.data, &a.scale, &b.data, &b.scale}) {
      const auto [first, last] = span(*t);
      if (start < last && first < end) value_error("out must not overlap the operands");
    }
    // As torch's own out= functions: the write is not differentiable, and whoever saved the tensor must notice it.
    if (out.requires_grad() && c10::GradMode::is_enabled())
      throw Refusal(PyExc_RuntimeError, "out requires grad, and block_matmul records no gradients: call it under torch.no_grad()");
    if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
  } else {
    if (out_code < 0) out_code = SR_BF16;
    out = at::empty({m, n}, options.dtype(scalar_type(out_code)));
  }
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

bool bound() { return g_cast && g_matmul && g_orthogonalize && g_workspace; }

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
  Py_BEGIN_ALLOW_THREADS
  try {
    const c10::OptionalDeviceGuard guard(device.is_cuda() ? c10::optional<at::Device>(device) : c10::nullopt);
    body();
  } catch (const Refusal& refusal) {
    type = refusal.type;
    message = refusal.what();
  } catch (const Status& s) {
    status = s.code;
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

PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long cast, matmul, orthogonalize, workspace;
  if (!PyArg_ParseTuple(args, "KKKK", &cast, &matmul, &orthogonalize, &workspace)) return nullptr;
  g_cast = reinterpret_cast<CastFn>(address(cast));
  g_matmul = reinterpret_cast<MatmulFn>(address(matmul));
  g_orthogonalize = reinterpret_cast<OrthogonalizeFn>(address(orthogonalize));
  g_workspace = reinterpret_cast<WorkspaceFn>(address(workspace));
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
      [&]() -> PyObject* {
        const Scaled &first = wanted[0] == '1' ? by_rows : by_cols, &second = wanted[0] == '1' ? by_cols : by_rows;
        if (wanted.size() == 1) return wrap_all({&first.data, &first.scale});
        return wrap_all({&first.data, &first.scale, &second.data, &second.scale});
      });
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
    {"orthogonalize", guarded<orthogonalize>, METH_VARARGS, "Orthogonalise matrices."},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_matrix", "Native entries of the matrix operators.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__matrix(void) { return PyModule_Create(&module); }
