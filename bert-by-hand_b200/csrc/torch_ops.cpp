// Python module _bbh_ops: the 8-bit linear path's unit operators on torch tensors, over the C ABI
// of libbbh.so. It checks types, shapes, strides and devices, allocates what the caller did
// not give, and launches on the current stream of the tensors' device. A call on small tensors is
// mostly host work: 3.3 to 5 us here where the same steps in Python with ctypes took 9 to 13.
//
// Arguments are positional (bbh.py has the signatures and the documentation). TypeError and
// ValueError say what is wrong with a tensor, BBHError (given by bbh.py) what the C ABI
// refused; errors of torch's own are torch's (torch.OutOfMemoryError where an output cannot be
// allocated). No gradient is recorded.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <string>

#include "../../include/bbh.h"

namespace {

PyObject* g_bbh_error = nullptr;  // bbh.BBHError

struct Refused : std::exception {
  PyObject* type;
  std::string text;
  Refused(PyObject* t, std::string s) : type(t), text(std::move(s)) {}
  const char* what() const noexcept override { return text.c_str(); }
};
struct Failed : std::exception {  // a BBH_ERR_* of the C ABI
  int code;
  explicit Failed(int c) : code(c) {}
};

[[noreturn]] void type_error(const std::string& s) { throw Refused(PyExc_TypeError, s); }
[[noreturn]] void value_error(const std::string& s) { throw Refused(PyExc_ValueError, s); }
void check(int rc) {
  if (rc != BBH_OK) throw Failed(rc);
}

// The interpreter is free while this lives: an allocation may wait for the device and a launch for room in the
// queue, and what they wait for (a host function of a stream in front, another thread) may need the interpreter.
// Between the reading of the arguments and the wrapping of results; a throw takes the lock back first.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  NoGil() = default;
  NoGil(const NoGil&) = delete;
  NoGil& operator=(const NoGil&) = delete;
  ~NoGil() { PyEval_RestoreThread(state); }
};

// Runs f, turning its exceptions into Python's.
template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F f) {
  try {
    if (n != want) type_error("wrong number of arguments");
    return f();
  } catch (const Refused& e) {
    PyErr_SetString(e.type, e.what());
  } catch (const Failed& e) {
    if (PyObject* o = PyObject_CallFunction(g_bbh_error, "is", e.code, bbh_last_error())) {
      PyErr_SetObject(g_bbh_error, o);
      Py_DECREF(o);
    }
  } catch (const std::exception&) {
    torch::translate_exception_to_python(std::current_exception());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

const at::Tensor* tensor(PyObject* o, const char* what) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) type_error(std::string(what) + " must be a tensor");
  return &THPVariable_Unpack(o);
}
const at::Tensor& given(PyObject* o, const char* what) {
  const at::Tensor* t = tensor(o, what);
  if (!t) type_error(std::string(what) + " must be a tensor");
  return *t;
}
const at::Tensor& on_gpu(PyObject* o, const char* what) {
  const at::Tensor& t = given(o, what);
  if (!t.is_cuda()) value_error("expected a CUDA tensor");
  return t;
}

int dtype_code(at::ScalarType t) {
  if (t == at::kHalf) return BBH_F16;
  if (t == at::kBFloat16) return BBH_BF16;
  type_error("expected float16 or bfloat16");
}
at::ScalarType dtype_of(PyObject* o) {
  if (!THPDtype_Check(o)) type_error("dtype must be a torch.dtype");
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
int as_int(int64_t v) {
  if (v > INT32_MAX) value_error("a size exceeds 2^31 - 1");
  return static_cast<int>(v);
}

// A 2-D operand: the pointer and row stride the C ABI takes.
struct Rows {
  void* p = nullptr;
  int64_t ld = 0;
};
template <typename T>
T* ptr(const Rows& r) {
  return static_cast<T*>(r.p);
}
void two_d(const at::Tensor& t, const char* what) {
  if (t.dim() != 2) value_error(std::string("expected a 2-D tensor: ") + what);
}
Rows rows(const at::Tensor& t, const at::Device& dev, at::ScalarType type, int64_t m, int64_t d, const char* what) {
  if (t.scalar_type() != type) type_error(std::string(what) + " must be " + c10::toString(type));
  if (t.dim() != 2 || t.size(0) != m || t.size(1) != d)
    value_error(std::string(what) + " must be [" + std::to_string(m) + ", " + std::to_string(d) + "]");
  if (t.device() != dev) value_error(std::string(what) + " must be on " + dev.str());
  if (t.stride(1) != 1 && d > 1) value_error(std::string("the rows of ") + what + " must have unit stride");
  // the stride of a single row says nothing
  return {t.data_ptr(), m > 1 ? t.stride(0) : (d + 15) / 16 * 16};
}
// A contiguous vector of n elements, or null.
template <typename T>
T* vec(const at::Tensor* t, const at::Device& dev, at::ScalarType type, int64_t n, const char* what) {
  if (!t) return nullptr;
  if (t->scalar_type() != type) type_error(std::string(what) + " must be " + c10::toString(type));
  if (t->dim() != 1 || t->size(0) != n || (n > 1 && t->stride(0) != 1))
    value_error(std::string(what) + " must be contiguous [" + std::to_string(n) + "]");
  if (t->device() != dev) value_error(std::string(what) + " must be on " + dev.str());
  return static_cast<T*>(t->data_ptr());
}

at::Tensor make(at::IntArrayRef size, at::ScalarType type, const at::Device& dev) {
  return at::Tensor(at::detail::empty_cuda(size, type, dev, std::nullopt));
}
// int8 [m, d] whose rows start at multiples of 128 bytes, or of the next smaller power of two from 16 on that
// lengthens them by a quarter at most. linear_i8 reads the rows in pieces of 128 bytes, which then lie in one
// cache line: 8192 x 4096 x 1000 takes 27.1 us with rows 1024 bytes apart, 34.3 with 1008.
at::Tensor make_i8(int64_t m, int64_t d, const at::Device& dev) {
  int64_t unit = 128;
  auto padded = [&] { return (d + unit - 1) / unit * unit; };
  while (unit > 16 && (padded() - d) * 4 > d) unit /= 2;
  return at::Tensor(at::detail::empty_strided_cuda({m, d}, {padded(), 1}, at::kChar, dev));
}
void* stream_of(const at::Device& dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

PyObject* tuple(std::initializer_list<PyObject*> items) {
  PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(items.size()));
  Py_ssize_t i = 0;
  for (PyObject* o : items) PyTuple_SET_ITEM(t, i++, o);
  return t;
}
// The caller's object, or the tensor made in its place.
PyObject* result(PyObject* o, const at::Tensor& made) { return o == Py_None ? THPVariable_Wrap(made) : Py_NewRef(o); }

using U16 = uint16_t;

// The operands that both norms have in common.
struct NormArgs {
  const at::Tensor& x;
  at::Device dev;
  at::ScalarType type;
  int code;
  int64_t m, d;
  Rows xr, rr, sr;
  at::Tensor sum;
  bool residual;
  U16* weight;

  NormArgs(PyObject* ox, PyObject* ow, PyObject* ores, PyObject* osum)
      : x(on_gpu(ox, "x")), dev(x.device()), type(x.scalar_type()) {
    two_d(x, "x");
    code = dtype_code(type);
    m = x.size(0);
    d = x.size(1);
    xr = rows(x, dev, type, m, d, "x");
    weight = vec<U16>(tensor(ow, "weight"), dev, type, d, "weight");
    const at::Tensor* r = tensor(ores, "residual");
    const at::Tensor* s = tensor(osum, "sum_out");
    residual = r != nullptr;
    if (!r) {
      if (s) value_error("sum_out needs a residual");
      return;
    }
    rr = rows(*r, dev, type, m, d, "residual");
    if (s) sr = rows(*s, dev, type, m, d, "sum_out");
  }
  void make_sum(PyObject* osum) {  // after the device guard
    if (!residual || osum != Py_None) return;
    sum = make({m, d}, type, dev);
    sr = {sum.data_ptr(), d};
  }
};

// x, weight, eps, residual, out, sum_out -> y | (y, sum)
PyObject* rmsnorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> PyObject* {
    NormArgs k(a[0], a[1], a[3], a[5]);
    const double eps = PyFloat_AsDouble(a[2]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    Rows yr;
    if (a[4] != Py_None) yr = rows(given(a[4], "out"), k.dev, k.type, k.m, k.d, "out");
    at::Tensor y;
    {
      const NoGil no_gil;
      const c10::cuda::CUDAGuard on(k.dev);
      k.make_sum(a[5]);
      if (a[4] == Py_None) {
        y = make({k.m, k.d}, k.type, k.dev);
        yr = {y.data_ptr(), k.d};
      }
      check(bbh_rmsnorm(ptr<U16>(k.xr), k.xr.ld, ptr<U16>(k.rr), k.rr.ld, k.weight, ptr<U16>(yr), yr.ld, ptr<U16>(k.sr),
                        k.sr.ld, as_int(k.m), as_int(k.d), static_cast<float>(eps), k.code, stream_of(k.dev)));
    }
    PyObject* oy = result(a[4], y);
    return k.residual ? tuple({oy, result(a[5], k.sum)}) : oy;
  });
}

// x, weight, eps, residual, sum_out -> (q, scale) | (q, scale, sum)
PyObject* rmsnorm_i8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    NormArgs k(a[0], a[1], a[3], a[4]);
    const double eps = PyFloat_AsDouble(a[2]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    at::Tensor q, scale;
    {
      const NoGil no_gil;
      const c10::cuda::CUDAGuard on(k.dev);
      k.make_sum(a[4]);
      q = make_i8(k.m, k.d, k.dev);
      scale = make({k.m}, at::kFloat, k.dev);
      check(bbh_rmsnorm_i8(ptr<U16>(k.xr), k.xr.ld, ptr<U16>(k.rr), k.rr.ld, k.weight, static_cast<int8_t*>(q.data_ptr()),
                           q.stride(0), static_cast<float*>(scale.data_ptr()), ptr<U16>(k.sr), k.sr.ld, as_int(k.m),
                           as_int(k.d), static_cast<float>(eps), k.code, stream_of(k.dev)));
    }
    PyObject *oq = THPVariable_Wrap(q), *os = THPVariable_Wrap(scale);
    return k.residual ? tuple({oq, os, result(a[4], k.sum)}) : tuple({oq, os});
  });
}

// x -> (q, scale)
PyObject* quantize_i8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 1, [&]() -> PyObject* {
    const at::Tensor& x = on_gpu(a[0], "x");
    const at::Device dev = x.device();
    two_d(x, "x");
    const int code = dtype_code(x.scalar_type());
    const int64_t m = x.size(0), d = x.size(1);
    const Rows xr = rows(x, dev, x.scalar_type(), m, d, "x");
    at::Tensor q, scale;
    {
      const NoGil no_gil;
      const c10::cuda::CUDAGuard on(dev);
      q = make_i8(m, d, dev);
      scale = make({m}, at::kFloat, dev);
      check(bbh_quantize_i8(ptr<U16>(xr), xr.ld, static_cast<int8_t*>(q.data_ptr()), q.stride(0),
                            static_cast<float*>(scale.data_ptr()), as_int(m), as_int(d), code, stream_of(dev)));
    }
    return tuple({THPVariable_Wrap(q), THPVariable_Wrap(scale)});
  });
}

// q, scale, dtype, out -> y
PyObject* dequantize_i8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    const at::Tensor& q = on_gpu(a[0], "q");
    const at::Device dev = q.device();
    two_d(q, "q");
    const int64_t m = q.size(0), d = q.size(1);
    const Rows qr = rows(q, dev, at::kChar, m, d, "q");
    const at::Tensor* out = tensor(a[3], "out");
    const at::ScalarType type = out ? out->scalar_type() : dtype_of(a[2]);
    const int code = dtype_code(type);
    float* scale = vec<float>(&given(a[1], "scale"), dev, at::kFloat, m, "scale");
    Rows yr;
    if (out) yr = rows(*out, dev, type, m, d, "out");
    at::Tensor y;
    {
      const NoGil no_gil;
      const c10::cuda::CUDAGuard on(dev);
      if (!out) {
        y = make({m, d}, type, dev);
        yr = {y.data_ptr(), d};
      }
      check(bbh_dequantize_i8(ptr<int8_t>(qr), qr.ld, scale, ptr<U16>(yr), yr.ld, as_int(m), as_int(d), code,
                              stream_of(dev)));
    }
    return result(a[3], y);
  });
}

// A, a_scale, W, w_scale, bias, gelu, dtype, out -> C
PyObject* linear_i8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const at::Tensor &A = on_gpu(a[0], "A"), &W = given(a[2], "W");
    const at::Device dev = A.device();
    two_d(A, "A");
    two_d(W, "W");
    const int64_t M = A.size(0), K = A.size(1), N = W.size(0);
    const Rows ar = rows(A, dev, at::kChar, M, K, "A"), wr = rows(W, dev, at::kChar, N, K, "W");
    const at::Tensor* out = tensor(a[7], "out");
    const at::ScalarType type = out ? out->scalar_type() : dtype_of(a[6]);
    const int code = dtype_code(type);
    float* sa = vec<float>(&given(a[1], "a_scale"), dev, at::kFloat, M, "a_scale");
    float* sw = vec<float>(&given(a[3], "w_scale"), dev, at::kFloat, N, "w_scale");
    U16* bias = vec<U16>(tensor(a[4], "bias"), dev, type, N, "bias");
    const int gelu = PyObject_IsTrue(a[5]);
    if (gelu < 0) return nullptr;
    Rows cr;
    if (out) cr = rows(*out, dev, type, M, N, "out");
    at::Tensor C;
    {
      const NoGil no_gil;
      const c10::cuda::CUDAGuard on(dev);
      if (!out) {
        C = make({M, N}, type, dev);
        cr = {C.data_ptr(), N};
      }
      check(bbh_linear_i8(ptr<int8_t>(ar), ar.ld, sa, ptr<int8_t>(wr), wr.ld, sw, bias, ptr<U16>(cr), cr.ld, as_int(M),
                          as_int(N), as_int(K), gelu, code, stream_of(dev)));
    }
    return result(a[7], C);
  });
}

PyObject* set_error(PyObject*, PyObject* cls) {
  Py_XDECREF(g_bbh_error);
  g_bbh_error = Py_NewRef(cls);
  Py_RETURN_NONE;
}

#define BBH_FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {BBH_FAST(rmsnorm),       BBH_FAST(rmsnorm_i8), BBH_FAST(quantize_i8),
                           BBH_FAST(dequantize_i8), BBH_FAST(linear_i8),  {"set_error", set_error, METH_O, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_bbh_ops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bbh_ops() { return PyModule_Create(&g_module); }
