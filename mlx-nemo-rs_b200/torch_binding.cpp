// torch_binding.cpp -- the CPython/libtorch side of fp8.py: argument checks,
// output allocation and the C ABI calls of the 8-bit linears and the
// LayerNorm on torch CUDA tensors.
//
// A streaming chunk's operators take 2 to 8 us on the device.  Checked and
// allocated from Python they cost 12 to 23 us of host time a call; here about
// a third of that.  Every refusal raises NrpError with the ABI's codes.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>
#include <tuple>
#include <utility>

#include "../include/nemo_relpos.h"

namespace {

using at::ScalarType;
using at::Tensor;

PyObject* g_error = nullptr;            // NrpError
PyTypeObject* g_fp8 = nullptr;          // Fp8Tensor
PyObject* g_default_context = nullptr;  // Context.default
constexpr int kMaxDevices = 64;
PyObject* g_context[kMaxDevices] = {};  // default contexts in use, kept alive
nrp_context* g_handle[kMaxDevices] = {};

struct Refused {
  int code;
  std::string msg;
};
struct PythonError {};  // a Python exception is set

[[noreturn]] void fail(const std::string& msg, int code = NRP_ERR_INVALID) {
  throw Refused{code, msg};
}

std::string shape_of(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}
std::string type_name(ScalarType t) { return c10::toString(t); }

const Tensor& tensor(const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) fail(std::string(name) + ": a CUDA tensor is needed");
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda()) fail(std::string(name) + ": a CUDA tensor is needed");
  return t;
}
// A contiguous tensor of the type on the device.
const Tensor& checked(const char* name, PyObject* o, ScalarType type, int dev) {
  const Tensor& t = tensor(name, o);
  if (t.get_device() != dev)
    fail(std::string(name) + ": on device " + std::to_string(t.get_device()) +
         ", the others on device " + std::to_string(dev));
  if (t.scalar_type() != type)
    fail(std::string(name) + ": dtype " + type_name(t.scalar_type()) + ", " + type_name(type) +
             " needed",
         NRP_ERR_UNSUPPORTED);
  if (!t.is_contiguous() || t.is_neg() || t.is_conj())
    fail(std::string(name) + ": shape " + shape_of(t.sizes()) + ", strides " +
         shape_of(t.strides()) + ": must be contiguous");
  return t;
}
struct Size {
  int64_t rows, cols;
};
Size size_of(const char* name, const Tensor& t) {
  const auto s = t.sizes();
  if (s.empty() || s.back() == 0 || s.back() > INT32_MAX)
    fail(std::string(name) + ": shape " + shape_of(s) + ": no columns, or too many");
  return {t.numel() / s.back(), s.back()};
}
const void* vector(const char* name, PyObject* o, int64_t n, ScalarType type, int dev) {
  const Tensor& t = checked(name, o, type, dev);
  if (t.numel() != n)
    fail(std::string(name) + ": " + std::to_string(t.numel()) + " values, " + std::to_string(n) +
         " needed");
  return t.const_data_ptr();
}
int dtype_code(const char* name, ScalarType t) {
  if (t == ScalarType::Float) return NRP_DTYPE_F32;
  if (t == ScalarType::BFloat16) return NRP_DTYPE_BF16;
  fail(std::string(name) + ": dtype " + type_name(t), NRP_ERR_UNSUPPORTED);
}
ScalarType dtype_arg(const char* name, PyObject* o) {
  if (!THPDtype_Check(o)) fail(std::string(name) + ": dtype must be a torch.dtype");
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
int rows32(const char* name, int64_t rows) {
  if (rows > INT32_MAX) fail(std::string(name) + ": " + std::to_string(rows) + " rows");
  return static_cast<int>(rows);
}

int64_t blocks(int64_t n) { return (n + 127) / 128; }
Tensor empty(at::IntArrayRef shape, ScalarType type, int dev) {
  if (c10::cuda::current_device() == dev) {
    // the same in fewer steps (no device guard, no options)
    const auto meta = c10::scalarTypeToTypeMeta(type);
    int64_t bytes = static_cast<int64_t>(meta.itemsize());
    for (int64_t n : shape) bytes *= n;
    c10::Allocator* allocator = c10::cuda::CUDACachingAllocator::get();
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(
        c10::make_intrusive<c10::StorageImpl>(c10::StorageImpl::use_byte_size_t(), bytes,
                                              allocator->allocate(bytes), allocator, true),
        c10::DispatchKeySet(c10::DispatchKey::CUDA), meta);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
    return t;
  }
  return at::detail::empty_cuda(shape, type,
                                c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(dev)),
                                std::nullopt);
}
// Two f32 tensors of one shape, and a matrix' codes and scales: each with a storage
// of its own (one of both would save 0.5 us, but resize_ of one would grow into the
// other, and either keep and save both).
std::pair<Tensor, Tensor> empty_two(at::IntArrayRef shape, int dev) {
  Tensor first = empty(shape, ScalarType::Float, dev);
  return {std::move(first), empty(shape, ScalarType::Float, dev)};
}
std::pair<Tensor, Tensor> empty_codes(at::IntArrayRef shape, Size n, int64_t block_rows, int dev) {
  Tensor codes = empty(shape, ScalarType::Float8_e4m3fn, dev);
  return {std::move(codes), empty({block_rows == 1 ? n.rows : blocks(n.rows), blocks(n.cols)},
                                  ScalarType::Float, dev)};
}
// out= of the given shape and type, or a new tensor.
Tensor output(const char* name, PyObject* out, at::IntArrayRef shape, ScalarType type, int dev) {
  dtype_code(name, type);
  if (out == Py_None) return empty(shape, type, dev);
  const Tensor& t = checked(name, out, type, dev);
  if (t.sizes() != shape)
    fail(std::string(name) + ": shape " + shape_of(t.sizes()) + ", " + shape_of(shape) + " needed");
  return t;
}

// A Python int's value; -1 for another object, or one past 64 bits.
int64_t int_or_none(PyObject* o) {
  const int64_t v = PyLong_Check(o) ? PyLong_AsLongLong(o) : -1;
  if (v == -1 && PyErr_Occurred()) PyErr_Clear();
  return v;
}

// A tensor of the caller's that a call has written: autograd sees by its version
// that a value it saved is gone.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

bool is_fp8(PyObject* o) { return PyObject_TypeCheck(o, g_fp8) && PyTuple_GET_SIZE(o) == 3; }
struct Codes {
  const Tensor* codes;
  uint8_t* q;
  float* s;
  Size size;
};
// A valid Fp8Tensor with the given block rows (0: any).
Codes codes_of(const char* name, PyObject* o, int64_t block_rows, int dev,
               int64_t* block = nullptr) {
  if (!is_fp8(o)) fail(std::string(name) + ": an Fp8Tensor is needed");
  const int64_t br = int_or_none(PyTuple_GET_ITEM(o, 2));
  if (block_rows ? br != block_rows : br != 1 && br != 128)
    fail(std::string(name) + ": block_rows " + std::to_string(br) + ", " +
         (block_rows ? std::to_string(block_rows) : "1 or 128") + " needed");
  const std::string sub = std::string(name) + " codes";
  const Tensor& c = checked(sub.c_str(), PyTuple_GET_ITEM(o, 0), ScalarType::Float8_e4m3fn, dev);
  const Size size = size_of(sub.c_str(), c);
  const std::string sc = std::string(name) + " scales";
  const void* s = vector(sc.c_str(), PyTuple_GET_ITEM(o, 1),
                         (br == 1 ? size.rows : blocks(size.rows)) * blocks(size.cols),
                         ScalarType::Float, dev);
  if (block) *block = br;
  return {&c, static_cast<uint8_t*>(c.data_ptr()),
          static_cast<float*>(const_cast<void*>(s)), size};
}
void codes_written(PyObject* o) {
  written(THPVariable_Unpack(PyTuple_GET_ITEM(o, 0)));
  written(THPVariable_Unpack(PyTuple_GET_ITEM(o, 1)));
}
int codes_device(const char* name, PyObject* o) {
  if (!is_fp8(o)) fail(std::string(name) + ": an Fp8Tensor is needed");
  return tensor(name, PyTuple_GET_ITEM(o, 0)).get_device();
}

// The handle of a Context object, which must be the device's.
nrp_context* handle_of(PyObject* ctx, int dev) {
  PyObject* handle = PyObject_GetAttrString(ctx, "handle");
  PyObject* value = handle ? PyObject_GetAttrString(handle, "value") : nullptr;
  PyObject* device = value ? PyObject_GetAttrString(ctx, "device") : nullptr;
  nrp_context* h = value ? static_cast<nrp_context*>(PyLong_AsVoidPtr(value)) : nullptr;
  const long d = device ? PyLong_AsLong(device) : -1;
  Py_XDECREF(handle);
  Py_XDECREF(value);
  Py_XDECREF(device);
  if (PyErr_Occurred()) throw PythonError{};
  if (d != dev)
    fail("context of device " + std::to_string(d) + ", tensors on device " + std::to_string(dev));
  return h;
}
// ctx, or the device's default context, which is looked up once and kept.
nrp_context* context_of(PyObject* ctx, int dev) {
  if (ctx != Py_None) return handle_of(ctx, dev);
  if (dev >= kMaxDevices) fail("device " + std::to_string(dev), NRP_ERR_UNSUPPORTED);
  if (!g_handle[dev]) {
    PyObject* c = PyObject_CallFunction(g_default_context, "i", dev);
    if (!c) throw PythonError{};
    if (g_handle[dev]) {  // another thread came here meanwhile
      Py_DECREF(c);
    } else {
      g_handle[dev] = handle_of(c, dev);
      g_context[dev] = c;  // (the reference stays)
    }
  }
  return g_handle[dev];
}

void* stream_of(int dev) {
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
}
// Runs an ABI call without the GIL and leaves the thread's current device as
// it was (the library makes the context's current).
template <typename F>
void call(int dev, F&& f) {
  struct Unlocked {
    PyThreadState* save = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(save); }  // also when a CUDA call throws
  };
  int rc;
  std::string msg;
  {
    Unlocked unlocked;
    const auto current = c10::cuda::current_device();
    rc = f();
    if (rc < 0) msg = nrp_last_error();
    if (current != dev) c10::cuda::set_device(current);
  }
  if (rc < 0) fail(msg, rc);
}

PyObject* new_fp8(const Tensor& codes, const Tensor& scales, int64_t block_rows) {
  PyObject* t = PyTuple_New(3);
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(codes));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(scales));
  PyTuple_SET_ITEM(t, 2, PyLong_FromLongLong(block_rows));
  PyObject* args = PyTuple_Pack(1, t);
  PyObject* r = args ? PyTuple_Type.tp_new(g_fp8, args, nullptr) : nullptr;
  Py_XDECREF(args);
  Py_DECREF(t);
  if (!r) throw PythonError{};
  return r;
}
PyObject* tuple_of(const Tensor& a, const Tensor& b, const Tensor& c) {
  PyObject* t = PyTuple_New(3);
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(b));
  PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(c));
  return t;
}

// ------------------------------------------------------------- the calls
// quantize(x, block_rows, ctx, out)
PyObject* quantize(PyObject* const* a) {
  const Tensor& t = tensor("quantize", a[0]);
  const int dev = t.get_device();
  const int dt = dtype_code("quantize", t.scalar_type());
  checked("quantize", a[0], t.scalar_type(), dev);
  const Size n = size_of("quantize", t);
  const int64_t br = int_or_none(a[1]);
  if (br != 1 && br != 128)
    fail("quantize: block_rows " + std::to_string(br) + " (supported: 1, 128)",
         NRP_ERR_UNSUPPORTED);
  Tensor codes, scales;
  Codes q{};
  if (a[3] == Py_None) {
    std::tie(codes, scales) = empty_codes(t.sizes(), n, br, dev);
    q.q = static_cast<uint8_t*>(codes.data_ptr());
    q.s = static_cast<float*>(scales.data_ptr());
  } else {
    q = codes_of("quantize out", a[3], br, dev);
    if (q.size.rows != n.rows || q.size.cols != n.cols)
      fail("quantize out: codes " + shape_of(q.codes->sizes()) + " for " + shape_of(t.sizes()));
  }
  nrp_context* ctx = context_of(a[2], dev);
  call(dev, [&] {
    return nrp_fp8_quantize(ctx, stream_of(dev), dt, t.const_data_ptr(), n.rows,
                            static_cast<int>(n.cols), static_cast<int>(br), q.q, q.s);
  });
  if (a[3] != Py_None) {
    codes_written(a[3]);
    return Py_NewRef(a[3]);
  }
  return new_fp8(codes, scales, br);
}

// dequantize(q, dtype, ctx, out)
PyObject* dequantize(PyObject* const* a) {
  const int dev = codes_device("dequantize", a[0]);
  int64_t br = 0;
  const Codes q = codes_of("dequantize", a[0], 0, dev, &br);
  const ScalarType type = dtype_arg("dequantize", a[1]);
  const int dt = dtype_code("dequantize", type);
  const Tensor out = output("dequantize out", a[3], q.codes->sizes(), type, dev);
  nrp_context* ctx = context_of(a[2], dev);
  call(dev, [&] {
    return nrp_fp8_dequantize(ctx, stream_of(dev), q.q, q.s, q.size.rows,
                              static_cast<int>(q.size.cols), static_cast<int>(br), dt,
                              out.data_ptr());
  });
  if (a[3] != Py_None) written(out);
  return THPVariable_Wrap(out);
}

// product(x, w, bias, dtype, ctx, out, codes, trans): fp8_linear, or the
// input's gradient
PyObject* product(PyObject* const* a) {
  const bool trans = a[7] == Py_True;
  const char* name = trans ? "fp8_linear_input_grad" : "fp8_linear";
  const int dev = codes_device(name, a[1]);
  const Codes w = codes_of(name, a[1], 128, dev);
  const int64_t red = trans ? w.size.rows : w.size.cols;
  const int64_t cols = trans ? w.size.cols : w.size.rows;
  const Tensor* x;
  const void* src = nullptr;
  Size n;
  ScalarType type = ScalarType::BFloat16;
  uint8_t* xq;
  float* xs;
  Tensor buf;
  if (is_fp8(a[0])) {
    if (a[6] != Py_None)
      fail(std::string(name) + ": codes= takes the codes of a tensor that the call quantises");
    const Codes q = codes_of(name, a[0], 1, dev);
    x = q.codes;
    n = q.size;
    xq = q.q;
    xs = q.s;
    if (a[3] != Py_None) type = dtype_arg(name, a[3]);
  } else {
    type = tensor(name, a[0]).scalar_type();
    dtype_code(name, type);
    x = &checked(name, a[0], type, dev);
    n = size_of(name, *x);
    if (a[3] != Py_None && dtype_arg(name, a[3]) != type)
      fail(std::string(name) + ": input " + type_name(type) + ", output " +
               type_name(dtype_arg(name, a[3])),
           NRP_ERR_UNSUPPORTED);
    src = x->const_data_ptr();
    if (a[6] == Py_None) {  // not wanted: both in one buffer of this call
      const int64_t bytes = (n.rows * n.cols + 15) / 16 * 16;
      buf = empty({bytes + 4 * n.rows * blocks(n.cols)}, ScalarType::Byte, dev);
      xq = static_cast<uint8_t*>(buf.data_ptr());
      xs = reinterpret_cast<float*>(xq + bytes);
    } else {
      const Codes q = codes_of(name, a[6], 1, dev);
      if (q.size.rows != n.rows || q.size.cols != n.cols)
        fail(std::string(name) + ": codes " + shape_of(q.codes->sizes()) + " for " +
             shape_of(x->sizes()));
      xq = q.q;
      xs = q.s;
    }
  }
  const int dt = dtype_code(name, type);
  if (n.cols != red)
    fail(std::string(name) + ": input " + shape_of(x->sizes()) + ", weight " +
         shape_of(w.codes->sizes()));
  const void* bias =
      a[2] == Py_None ? nullptr : vector("fp8_linear bias", a[2], cols, type, dev);
  c10::DimVector shape(x->sizes().begin(), x->sizes().end());
  shape.back() = cols;
  const Tensor out = output(name, a[5], shape, type, dev);
  nrp_context* ctx = context_of(a[4], dev);
  const int m = rows32(name, n.rows), r = static_cast<int>(red), c = static_cast<int>(cols);
  call(dev, [&] {
    return trans ? nrp_fp8_linear_input_grad(ctx, stream_of(dev), dt, src, xq, xs, m, r, w.q, w.s,
                                             c, out.data_ptr())
                 : nrp_fp8_linear(ctx, stream_of(dev), dt, src, xq, xs, m, r, w.q, w.s, c, bias,
                                  out.data_ptr());
  });
  if (a[5] != Py_None) written(out);
  if (a[6] != Py_None) codes_written(a[6]);
  return THPVariable_Wrap(out);
}

// weight_grad(dy, x, bias, dtype, ctx, out, bias_out)
PyObject* weight_grad(PyObject* const* a) {
  const char* name = "fp8_linear_weight_grad";
  const int dev = tensor("fp8_linear_weight_grad dy", a[0]).get_device();
  const Tensor& dy = checked("fp8_linear_weight_grad dy", a[0], ScalarType::BFloat16, dev);
  const Size n = size_of("fp8_linear_weight_grad dy", dy);
  const Codes x = codes_of("fp8_linear_weight_grad input", a[1], 1, dev);
  if (x.size.rows != n.rows)
    fail(std::string(name) + ": " + std::to_string(n.rows) + " rows of dy, " +
         std::to_string(x.size.rows) + " of x");
  const int want = PyObject_IsTrue(a[2]);
  if (want < 0) throw PythonError{};
  const ScalarType type = dtype_arg(name, a[3]);
  const int dt = dtype_code(name, type);
  const Tensor dw = output("fp8_linear_weight_grad out", a[5], {n.cols, x.size.cols}, type, dev);
  Tensor db;
  if (want || a[6] != Py_None)
    db = output("fp8_linear_weight_grad bias_out", a[6], {n.cols}, type, dev);
  nrp_context* ctx = context_of(a[4], dev);
  const int m = rows32(name, n.rows);
  call(dev, [&] {
    return nrp_fp8_linear_weight_grad(ctx, stream_of(dev), dy.const_data_ptr(), x.q, x.s, m,
                                      static_cast<int>(n.cols), static_cast<int>(x.size.cols), dt,
                                      dw.data_ptr(), db.defined() ? db.data_ptr() : nullptr);
  });
  if (a[5] != Py_None) written(dw);
  if (a[6] != Py_None) written(db);
  PyObject* t = PyTuple_New(2);
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(dw));
  PyTuple_SET_ITEM(t, 1, db.defined() ? THPVariable_Wrap(db) : Py_NewRef(Py_None));
  return t;
}

// layer_norm(x, gamma, beta, eps, ctx, out)
PyObject* layer_norm(PyObject* const* a) {
  const Tensor& t = tensor("layer_norm", a[0]);
  const int dev = t.get_device();
  const ScalarType type = t.scalar_type();
  const int dt = dtype_code("layer_norm", type);
  checked("layer_norm", a[0], type, dev);
  const Size n = size_of("layer_norm", t);
  const void* g = vector("layer_norm gamma", a[1], n.cols, ScalarType::Float, dev);
  const void* b = vector("layer_norm beta", a[2], n.cols, ScalarType::Float, dev);
  const double eps = PyFloat_AsDouble(a[3]);
  if (eps == -1.0 && PyErr_Occurred()) throw PythonError{};
  const Tensor y = output("layer_norm out", a[5], t.sizes(), type, dev);
  const auto rows = t.sizes().slice(0, t.sizes().size() - 1);
  const auto [mean, rstd] = empty_two(rows, dev);
  nrp_context* ctx = context_of(a[4], dev);
  float* const stats[2] = {static_cast<float*>(mean.data_ptr()),
                           static_cast<float*>(rstd.data_ptr())};
  call(dev, [&] {
    return nrp_layer_norm(ctx, stream_of(dev), dt, t.const_data_ptr(), n.rows,
                          static_cast<int>(n.cols), static_cast<const float*>(g),
                          static_cast<const float*>(b), static_cast<float>(eps), y.data_ptr(),
                          stats[0], stats[1]);
  });
  if (a[5] != Py_None) written(y);
  return tuple_of(y, mean, rstd);
}

// layer_norm_backward(dy, x, mean, rstd, gamma, ctx, out)
PyObject* layer_norm_backward(PyObject* const* a) {
  const char* name = "layer_norm_backward";
  const Tensor& dy = tensor("layer_norm_backward dy", a[0]);
  const int dev = dy.get_device();
  const ScalarType type = dy.scalar_type();
  const int dt = dtype_code("layer_norm_backward dy", type);
  checked("layer_norm_backward dy", a[0], type, dev);
  const Size n = size_of("layer_norm_backward dy", dy);
  const void* x;
  const float* xs = nullptr;
  Size nx;
  if (is_fp8(a[1])) {
    const Codes q = codes_of("layer_norm_backward input", a[1], 1, dev);
    x = q.q;
    xs = q.s;
    nx = q.size;
  } else {
    const Tensor& t = checked("layer_norm_backward input", a[1], type, dev);
    x = t.const_data_ptr();
    nx = size_of("layer_norm_backward input", t);
  }
  if (nx.rows != n.rows || nx.cols != n.cols)
    fail(std::string(name) + ": dy " + shape_of(dy.sizes()) + " and an input of other size");
  const void* mu = vector("layer_norm_backward mean", a[2], n.rows, ScalarType::Float, dev);
  const void* rs = vector("layer_norm_backward rstd", a[3], n.rows, ScalarType::Float, dev);
  const void* g = vector("layer_norm_backward gamma", a[4], n.cols, ScalarType::Float, dev);
  const Tensor dx = output("layer_norm_backward out", a[6], dy.sizes(), type, dev);
  const auto [dgamma, dbeta] = empty_two({n.cols}, dev);
  int64_t bytes = 0;
  const int cols = static_cast<int>(n.cols);
  if (const int rc = nrp_layer_norm_backward_workspace(n.rows, cols, &bytes); rc < 0)
    fail(nrp_last_error(), rc);
  Tensor ws;
  if (bytes) ws = empty({bytes}, ScalarType::Byte, dev);
  nrp_context* ctx = context_of(a[5], dev);
  float* const sums[2] = {static_cast<float*>(dgamma.data_ptr()),
                          static_cast<float*>(dbeta.data_ptr())};
  call(dev, [&] {
    return nrp_layer_norm_backward(
        ctx, stream_of(dev), dt, x, xs, dy.const_data_ptr(), static_cast<const float*>(mu),
        static_cast<const float*>(rs), static_cast<const float*>(g), n.rows, cols, dx.data_ptr(),
        sums[0], sums[1], bytes ? ws.data_ptr() : nullptr, bytes);
  });
  if (a[6] != Py_None) written(dx);
  return tuple_of(dx, dgamma, dbeta);
}

// ----------------------------------------------------------------- module
template <PyObject* (*F)(PyObject* const*), int kArgs>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != kArgs) {
    PyErr_Format(PyExc_TypeError, "%d arguments needed, got %zd", kArgs, nargs);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused& r) {
    PyObject* e = PyObject_CallFunction(g_error, "is", r.code, r.msg.c_str());
    if (e) {
      PyErr_SetObject(g_error, e);
      Py_DECREF(e);
    }
    return nullptr;
  } catch (const PythonError&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// setup(NrpError, Fp8Tensor, Context.default)
PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 3 || !PyType_Check(args[1]) ||
      !PyType_IsSubtype(reinterpret_cast<PyTypeObject*>(args[1]), &PyTuple_Type)) {
    PyErr_SetString(PyExc_TypeError, "setup(NrpError, Fp8Tensor, Context.default)");
    return nullptr;
  }
  Py_XSETREF(g_error, Py_NewRef(args[0]));
  PyTypeObject* old = g_fp8;
  g_fp8 = reinterpret_cast<PyTypeObject*>(Py_NewRef(args[1]));
  Py_XDECREF(reinterpret_cast<PyObject*>(old));
  Py_XSETREF(g_default_context, Py_NewRef(args[2]));
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef g_methods[] = {
    {"setup", FAST(setup), nullptr},
    {"quantize", FAST((entry<quantize, 4>)), nullptr},
    {"dequantize", FAST((entry<dequantize, 4>)), nullptr},
    {"product", FAST((entry<product, 8>)), nullptr},
    {"weight_grad", FAST((entry<weight_grad, 7>)), nullptr},
    {"layer_norm", FAST((entry<layer_norm, 6>)), nullptr},
    {"layer_norm_backward", FAST((entry<layer_norm_backward, 7>)), nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_nrp_torch", nullptr, -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__nrp_torch() { return PyModule_Create(&g_module); }
