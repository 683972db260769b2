// The Python binding of the fp8 linears on torch tensors (ignite_xdna_b200/fp8.py): argument checks,
// outputs, the tensors' device and its current stream, then the C ABI. It is native because a decode
// step makes these calls a token at a time: the same work in Python around ctypes took 16 to 20 us per
// call, several times the kernels.
//
// The C ABI's functions come as addresses from the library that the package has loaded, so this module
// links against torch only.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/ixb200.h"

namespace {

decltype(&ixb_fp8_quantize) fp8_quantize = nullptr;
decltype(&ixb_rmsnorm_quant) rmsnorm_quant = nullptr;
decltype(&ixb_fp8_linear) fp8_linear = nullptr;
decltype(&ixb_fp8_linear_swiglu) fp8_linear_swiglu = nullptr;
decltype(&ixb_last_error) last_error = nullptr;
PyObject* error_class = nullptr;    // IxbError(code, message)
PyObject* out_of_memory = nullptr;  // torch.OutOfMemoryError

constexpr int64_t kBlock = 128;
int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }

// A Python error on its way out.
struct Raised {};

[[noreturn]] void raise(PyObject* type, const char* format, ...) {
  char text[512];
  va_list args;
  va_start(args, format);
  vsnprintf(text, sizeof text, format, args);
  va_end(args);
  PyErr_SetString(type, text);
  throw Raised{};
}

void check(int rc) {
  if (rc >= 0) return;
  if (PyObject* e = PyObject_CallFunction(error_class, "is", rc, last_error())) {
    PyErr_SetObject(error_class, e);
    Py_DECREF(e);
  }
  throw Raised{};
}

std::string shape(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) raise(PyExc_TypeError, "%s: a tensor is needed, got %s", name, Py_TYPE(o)->tp_name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided) raise(PyExc_ValueError, "%s: a strided tensor is needed", name);
  if (t.is_neg()) raise(PyExc_ValueError, "%s: its memory holds the negated values (call resolve_neg() first)", name);
  if (t.requires_grad() && at::GradMode::is_enabled())
    raise(PyExc_ValueError, "%s requires grad: these operators have no backward pass (call them under torch.no_grad())", name);
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
    raise(PyExc_ValueError, "%s has a forward-mode tangent, which these operators would drop: they have no derivative", name);
  return t;
}

int type_of(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return IXB_BF16;
    case at::kHalf: return IXB_F16;
    case at::kFloat: return IXB_F32;
    default: raise(PyExc_TypeError, "%s: bfloat16, float16 or float32 is needed, got %s", name, c10::toString(t.scalar_type()));
  }
}

void same_type(const at::Tensor& t, at::ScalarType type, const char* name) {
  if (t.scalar_type() != type)
    raise(PyExc_TypeError, "%s: %s is needed, got %s", name, c10::toString(type), c10::toString(t.scalar_type()));
}

// A matrix whose rows are contiguous and do not overlap. Returns the stride between rows; the one of a
// single row says nothing, so it gets the least that fits.
int64_t rows_of(const at::Tensor& t, const char* name) {
  if (t.dim() != 2 || !t.is_cuda())
    raise(PyExc_ValueError, "%s: a two-dimensional CUDA tensor is needed, got %s on %s", name, shape(t).c_str(),
          t.device().str().c_str());
  const int64_t rows = t.size(0), cols = t.size(1);
  if (rows > INT_MAX || cols > INT_MAX) raise(PyExc_ValueError, "%s: too large, %s", name, shape(t).c_str());
  if (cols > 1 && t.stride(1) != 1) raise(PyExc_ValueError, "%s: the values of a row must be contiguous", name);
  if (rows <= 1) return (cols + 15) / 16 * 16;
  if (t.stride(0) < cols)
    raise(PyExc_ValueError, "%s: rows overlap (stride %lld below %lld)", name, (long long)t.stride(0), (long long)cols);
  return t.stride(0);
}

void same_shape(const at::Tensor& t, int64_t rows, int64_t cols, const char* name) {
  if (t.size(0) != rows || t.size(1) != cols)
    raise(PyExc_ValueError, "%s: shape (%lld, %lld) is needed, got %s", name, (long long)rows, (long long)cols, shape(t).c_str());
}

void same_device(const at::Tensor& a, const at::Tensor& b, const char* name) {
  if (a.device() != b.device())
    raise(PyExc_ValueError, "%s: on %s, the others on %s", name, b.device().str().c_str(), a.device().str().c_str());
}

// Whether two matrices with contiguous rows have a byte in common. Exact where their rows are equally far apart
// (two column ranges of one matrix) or either has one row; elsewhere matrices whose spans meet count as sharing.
bool shares_memory(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  struct Rows {
    int64_t begin, width, pitch, rows;  // bytes
    explicit Rows(const at::Tensor& t) {
      const int64_t size = (int64_t)t.element_size();
      begin = (int64_t)reinterpret_cast<intptr_t>(t.const_data_ptr());
      width = t.size(1) * size;
      rows = t.size(0);
      pitch = rows > 1 ? t.stride(0) * size : width;
    }
    int64_t end() const { return begin + (rows - 1) * pitch + width; }
  } x(a), y(b);
  if (x.begin >= y.end() || y.begin >= x.end()) return false;
  if (x.rows == 1) x.pitch = y.pitch;
  if (y.rows == 1) y.pitch = x.pitch;
  if (x.pitch != y.pitch || x.width > x.pitch || y.width > y.pitch) return true;
  // the spans meet and both repeat every `pitch` bytes: the rows miss one another if neither's columns, taken
  // around the pitch, reach into the other's
  const int64_t d = ((y.begin - x.begin) % x.pitch + x.pitch) % x.pitch;  // from x's columns to y's
  return d < x.width || d + y.width > x.pitch;
}

// An e4m3 matrix of K columns with a scale per `rows` rows and 128 columns.
struct Operand {
  const uint8_t* q;
  int64_t ld;
  const uint8_t* s;
  int64_t lds;
};
Operand operand(const at::Tensor& first, PyObject* qo, PyObject* so, const char* name, const char* scale_name, int64_t rows,
                int64_t K) {
  const at::Tensor &q = tensor(qo, name), &s = tensor(so, scale_name);
  Operand o;
  o.ld = rows_of(q, name);
  same_type(q, at::kFloat8_e4m3fn, name);
  if (q.size(1) != K)
    raise(PyExc_ValueError, "%s: %lld columns are needed, got %s", name, (long long)K, shape(q).c_str());
  o.lds = rows_of(s, scale_name);
  same_type(s, at::kFloat8_e8m0fnu, scale_name);
  same_shape(s, (q.size(0) + rows - 1) / rows, blocks(K), scale_name);
  same_device(first, q, name);
  same_device(first, s, scale_name);
  o.q = static_cast<const uint8_t*>(q.const_data_ptr());
  o.s = static_cast<const uint8_t*>(s.const_data_ptr());
  return o;
}

at::Tensor matrix(int64_t rows, int64_t cols, const at::Tensor& like, at::ScalarType type) {
  return at::Tensor(at::detail::empty_cuda({rows, cols}, type, like.device(), std::nullopt));
}
// An empty scale matrix whose rows start on 4 bytes, which the products read a word at a time.
at::Tensor scales(int64_t rows, int64_t cols, const at::Tensor& like) {
  const int64_t n = blocks(cols);
  return at::Tensor(at::detail::empty_strided_cuda({rows, n}, {(n + 3) / 4 * 4, 1}, at::kFloat8_e8m0fnu, like.device()));
}
uint8_t* bytes(const at::Tensor& t) { return static_cast<uint8_t*>(t.mutable_data_ptr()); }

// The tensors' device for the launch, and its current stream.
struct OnDevice {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit OnDevice(const at::Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
};

PyObject* tuple(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = Py_None;
    if (t.defined()) o = THPVariable_Wrap(t);
    else Py_INCREF(o);
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// Runs `body`; C++ exceptions become Python ones and do not cross into the interpreter.
template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F&& body) {
  try {
    if (got != want) raise(PyExc_TypeError, "%zd arguments are needed, got %zd", want, got);
    if (!error_class) raise(PyExc_RuntimeError, "bind() has not been called");
    return body();
  } catch (const Raised&) {
    return nullptr;
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(out_of_memory, e.what_without_backtrace());
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

int int_of(PyObject* o, const char* name) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  if (v < INT_MIN || v > INT_MAX) raise(PyExc_ValueError, "%s: %ld is out of range", name, v);
  return (int)v;
}

PyObject* py_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {  // x, block_rows
  return guarded(n, 2, [&] {
    const at::Tensor& x = tensor(a[0], "x");
    const int type = type_of(x, "x");
    const int block_rows = int_of(a[1], "block_rows");
    const int64_t ldx = rows_of(x, "x");
    const int64_t M = x.size(0), K = x.size(1);
    OnDevice on(x);
    const at::Tensor q = matrix(M, K, x, at::kFloat8_e4m3fn), s = scales(block_rows == 1 ? M : blocks(M), K, x);
    check(fp8_quantize(x.const_data_ptr(), type, ldx, (int)M, (int)K, block_rows, bytes(q), K, bytes(s), s.stride(0), on.stream));
    return tuple({q, s});
  });
}

PyObject* py_rmsnorm_quant(PyObject*, PyObject* const* a, Py_ssize_t n) {  // x, weight, eps, residual, position
  return guarded(n, 5, [&] {
    const at::Tensor &x = tensor(a[0], "x"), &w = tensor(a[1], "weight");
    const int type = type_of(x, "x");
    const int64_t ldx = rows_of(x, "x"), M = x.size(0), K = x.size(1);
    if (w.dim() != 1 || w.size(0) != K || !w.is_contiguous() || !w.is_cuda())
      raise(PyExc_ValueError, "weight: a contiguous CUDA tensor of %lld values is needed, got %s on %s", (long long)K,
            shape(w).c_str(), w.device().str().c_str());
    const int weight_type = type_of(w, "weight");
    if (weight_type != type && weight_type != IXB_F32)
      raise(PyExc_TypeError, "weight: %s or Float is needed, got %s", c10::toString(x.scalar_type()), c10::toString(w.scalar_type()));
    same_device(x, w, "weight");
    const double eps = PyFloat_AsDouble(a[2]);
    if (eps == -1.0 && PyErr_Occurred()) throw Raised{};
    const bool keep = a[3] != Py_None, e4m3 = a[4] == Py_None;
    const int position = e4m3 ? 0 : int_of(a[4], "position");
    const void* r = nullptr;
    int64_t ldr = 0;
    if (keep) {
      const at::Tensor& t = tensor(a[3], "residual");
      ldr = rows_of(t, "residual");
      same_type(t, x.scalar_type(), "residual");
      same_shape(t, M, K, "residual");
      same_device(x, t, "residual");
      r = t.const_data_ptr();
    }
    OnDevice on(x);
    at::Tensor h, s;
    if (keep) h = matrix(M, K, x, x.scalar_type());
    if (e4m3) s = scales(M, K, x);
    const at::Tensor q = matrix(M, K, x, e4m3 ? at::kFloat8_e4m3fn : at::kChar);
    // no rows: an empty tensor has no address, and the entry wants to see a residual with its output
    if (M > 0)
      check(rmsnorm_quant(x.const_data_ptr(), ldx, r, ldr, w.const_data_ptr(), type, weight_type, (int)M, (int)K, (float)eps,
                          position, keep ? h.mutable_data_ptr() : nullptr, K, bytes(q), K, e4m3 ? bytes(s) : nullptr,
                          e4m3 ? s.stride(0) : 0, on.stream));
    return tuple({q, s, h});
  });
}

PyObject* py_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {  // x, x_scale, w, w_scale, out_dtype, out
  return guarded(n, 6, [&] {
    const at::Tensor &x = tensor(a[0], "x"), &w = tensor(a[2], "w");
    rows_of(x, "x");
    rows_of(w, "w");
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
    const Operand ox = operand(x, a[0], a[1], "x", "x_scale", 1, K);
    const Operand ow = operand(x, a[2], a[3], "w", "w_scale", kBlock, K);
    OnDevice on(x);
    at::Tensor out;
    int64_t ldo = N;
    if (a[5] == Py_None) {
      if (!THPDtype_Check(a[4])) raise(PyExc_TypeError, "out_dtype: a torch.dtype is needed, got %s", Py_TYPE(a[4])->tp_name);
      const at::ScalarType type = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
      if (type != at::kBFloat16 && type != at::kHalf && type != at::kFloat)
        raise(PyExc_TypeError, "out_dtype: bfloat16, float16 or float32 is needed, got %s", c10::toString(type));
      out = matrix(M, N, x, type);
    } else {
      out = tensor(a[5], "out");
      type_of(out, "out");
      ldo = rows_of(out, "out");
      if (ldo < N) ldo = N;
      same_shape(out, M, N, "out");
      same_device(x, out, "out");
      for (int i = 0; i < 4; ++i)
        if (shares_memory(THPVariable_Unpack(a[i]), out)) raise(PyExc_ValueError, "out shares memory with an input");
      // what autograd has saved of it is no longer what it saved
      if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
    }
    check(fp8_linear(ox.q, ox.ld, ox.s, ox.lds, ow.q, ow.ld, ow.s, ow.lds, out.mutable_data_ptr(), type_of(out, "out"), ldo, (int)M,
                     (int)N, (int)K, on.stream));
    return THPVariable_Wrap(out);
  });
}

PyObject* py_linear_swiglu(PyObject*, PyObject* const* a, Py_ssize_t n) {  // x, x_scale, gate, gate_scale, up, up_scale
  return guarded(n, 6, [&] {
    const at::Tensor &x = tensor(a[0], "x"), &gate = tensor(a[2], "gate"), &up = tensor(a[4], "up");
    rows_of(x, "x");
    rows_of(gate, "gate");
    const int64_t M = x.size(0), K = x.size(1), N = gate.size(0);
    const Operand ox = operand(x, a[0], a[1], "x", "x_scale", 1, K);
    const Operand og = operand(x, a[2], a[3], "gate", "gate_scale", kBlock, K);
    const Operand ou = operand(x, a[4], a[5], "up", "up_scale", kBlock, K);
    if (up.size(0) != N)
      raise(PyExc_ValueError, "gate and up have %lld and %lld rows", (long long)N, (long long)up.size(0));
    OnDevice on(x);
    const at::Tensor q = matrix(M, N, x, at::kFloat8_e4m3fn), s = scales(M, N, x);
    check(fp8_linear_swiglu(ox.q, ox.ld, ox.s, ox.lds, og.q, og.ld, og.s, og.lds, ou.q, ou.ld, ou.s, ou.lds, bytes(q), N, bytes(s),
                            s.stride(0), (int)M, (int)N, (int)K, on.stream));
    return tuple({q, s});
  });
}

PyObject* py_shares_memory(PyObject*, PyObject* const* a, Py_ssize_t n) {  // two matrices with contiguous rows
  return guarded(n, 2, [&] {
    const at::Tensor &x = tensor(a[0], "a"), &y = tensor(a[1], "b");
    if (x.dim() != 2 || y.dim() != 2) raise(PyExc_ValueError, "matrices are needed");
    return PyBool_FromLong(shares_memory(x, y));
  });
}

PyObject* py_bind(PyObject*, PyObject* args) {  // two error classes, five addresses
  PyObject *cls, *oom;
  unsigned long long p[5];
  if (!PyArg_ParseTuple(args, "OOKKKKK", &cls, &oom, &p[0], &p[1], &p[2], &p[3], &p[4])) return nullptr;
  last_error = reinterpret_cast<decltype(last_error)>(p[0]);
  fp8_quantize = reinterpret_cast<decltype(fp8_quantize)>(p[1]);
  rmsnorm_quant = reinterpret_cast<decltype(rmsnorm_quant)>(p[2]);
  fp8_linear = reinterpret_cast<decltype(fp8_linear)>(p[3]);
  fp8_linear_swiglu = reinterpret_cast<decltype(fp8_linear_swiglu)>(p[4]);
  Py_INCREF(cls);
  Py_INCREF(oom);
  Py_XDECREF(error_class);
  Py_XDECREF(out_of_memory);
  error_class = cls;
  out_of_memory = oom;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_VARARGS, "bind(error_class, out_of_memory, last_error, quantize, rmsnorm_quant, linear, linear_swiglu): addresses of the C ABI"},
    {"quantize", (PyCFunction)(void*)py_quantize, METH_FASTCALL, nullptr},
    {"rmsnorm_quant", (PyCFunction)(void*)py_rmsnorm_quant, METH_FASTCALL, nullptr},
    {"linear", (PyCFunction)(void*)py_linear, METH_FASTCALL, nullptr},
    {"shares_memory", (PyCFunction)(void*)py_shares_memory, METH_FASTCALL, nullptr},
    {"linear_swiglu", (PyCFunction)(void*)py_linear_swiglu, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ixb_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ixb_torch() { return PyModule_Create(&module); }
