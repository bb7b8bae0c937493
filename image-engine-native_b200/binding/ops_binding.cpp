// The fast path of iec/ops.py: reads the tensors' pointers, shapes and
// strides without going through Python for each, fills the argument struct
// and calls the library. A call of the smallest sizes is bound by this host
// work (5.6 us through Python attributes and ctypes for a 2 us kernel).
//
// Every function returns the call's iec_status, or -1 without calling where
// something is not as the fast path takes it (an output to be allocated, a
// type, shape, stride or device that does not fit): iec/ops.py then goes
// through its checks one by one and says what is wrong.
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/iec_cuda.h"

namespace {

struct {
  iec_status (*group_norm)(iec_ops*, const iec_group_norm_args*, void*);
  iec_status (*group_norm_fp8)(iec_ops*, const iec_group_norm_args*, void*);
  iec_status (*quantize_fp8)(iec_ops*, const iec_quantize_fp8_args*, void*);
  iec_status (*matmul_fp8)(iec_ops*, const iec_matmul_fp8_args*, void*);
} lib;

constexpr int64_t BLOCK = 128;
int64_t blocks(int64_t k) { return (k + BLOCK - 1) / BLOCK; }

// The handle, its device and the stream of a call.
struct Call {
  iec_ops* ops = nullptr;
  int device = -1;
  void* stream = nullptr;
  bool ok = true;
  Call(PyObject* handle, PyObject* dev, PyObject* st) {
    ops = reinterpret_cast<iec_ops*>(PyLong_AsVoidPtr(handle));
    device = (int)PyLong_AsLong(dev);
    if (st == Py_None)
      stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    else
      stream = PyLong_AsVoidPtr(st);
    if (!stream) stream = reinterpret_cast<void*>(1);  // cudaStreamLegacy: torch's default stream is the handle 0
    if (PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
  }
  const at::Tensor* tensor(PyObject* o) {
    if (THPVariable_Check(o)) {
      const at::Tensor& t = THPVariable_Unpack(o);
      const bool lost = t.requires_grad() && c10::GradMode::is_enabled();  // its gradient
      if (t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device && !lost) return &t;
    }
    ok = false;
    return nullptr;
  }
  // A rows x cols matrix of contiguous rows; its row stride.
  void* matrix(PyObject* o, int64_t rows, int64_t cols, at::ScalarType type, size_t* step) {
    const at::Tensor* t = tensor(o);
    if (!t || t->dim() != 2 || t->scalar_type() != type || t->size(0) != rows || t->size(1) != cols ||
        (cols > 1 && t->stride(1) != 1) || (rows > 1 && t->stride(0) < 0)) {
      ok = false;
      return nullptr;
    }
    *step = (size_t)(rows > 1 ? t->stride(0) : std::max<int64_t>(cols, 1));
    return t->data_ptr();
  }
  // n contiguous floats, null for None.
  const float* vector(PyObject* o, int64_t n) {
    if (o == Py_None) return nullptr;
    const at::Tensor* t = tensor(o);
    if (!t || t->dim() != 1 || t->scalar_type() != at::kFloat || t->size(0) != n || (n > 1 && t->stride(0) != 1)) {
      ok = false;
      return nullptr;
    }
    return static_cast<const float*>(t->data_ptr());
  }
  int dtype(const at::Tensor& t) {
    switch (t.scalar_type()) {
      case at::kHalf: return IEC_F16;
      case at::kBFloat16: return IEC_BF16;
      case at::kFloat: return IEC_F32;
      default: ok = false; return 0;
    }
  }
  // Maps x ... x channels with the pixels at one stride.
  void* maps(PyObject* o, size_t* n, size_t* pixels, size_t* c, size_t* step, size_t* map_step) {
    const at::Tensor* t = tensor(o);
    if (!t || t->dim() < 2) {
      ok = false;
      return nullptr;
    }
    const int64_t d = t->dim(), channels = t->size(d - 1);
    int64_t px = 1, st = channels;
    if (channels > 1 && t->stride(d - 1) != 1) ok = false;
    for (int64_t i = d - 2; i > 0; i--) {
      if (t->size(i) == 1) continue;
      if (px == 1)
        st = t->stride(i);
      else if (t->stride(i) != st * px)
        ok = false;
      px *= t->size(i);
    }
    const int64_t ms = t->size(0) > 1 ? t->stride(0) : channels;
    if (st < 0 || ms < 0) ok = false;
    *n = (size_t)t->size(0);
    *pixels = (size_t)px;
    *c = (size_t)channels;
    *step = (size_t)st;
    *map_step = (size_t)ms;
    return t->data_ptr();
  }
  PyObject* result(iec_status status) { return PyLong_FromLong((long)status); }
  // Numbers; anything else leaves the fast path.
  int64_t integer(PyObject* o) {
    const long long v = PyLong_Check(o) ? PyLong_AsLongLong(o) : -1;
    if (!PyLong_Check(o) || v < INT32_MIN || v > INT32_MAX) ok = false;
    if (PyErr_Occurred()) PyErr_Clear();
    return v;
  }
  float number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return (float)v;
  }
};

PyObject* slow() { return PyLong_FromLong(-1); }

// (handle, device, stream, x, groups, gamma, beta, eps, act, out or codes, scales)
template <bool FP8>
PyObject* group_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != (FP8 ? 11 : 10)) return slow();
  Call call(a[0], a[1], a[2]);
  iec_group_norm_args args = {};
  args.x = call.maps(a[3], &args.n, &args.pixels, &args.c, &args.x_stride, &args.x_map_stride);
  if (!call.ok) return slow();
  const at::Tensor& x = THPVariable_Unpack(a[3]);
  args.dtype = call.dtype(x);
  const int64_t groups = call.integer(a[4]);
  args.groups = groups > 0 ? (size_t)groups : 0;
  args.gamma = call.vector(a[5], (int64_t)args.c);
  args.beta = call.vector(a[6], (int64_t)args.c);
  args.eps = call.number(a[7]);
  args.act = (int)call.integer(a[8]);
  if (FP8) {
    const int64_t rows = (int64_t)(args.n * args.pixels), c = (int64_t)args.c;
    args.codes = static_cast<uint8_t*>(call.matrix(a[9], rows, c, at::kFloat8_e4m3fn, &args.code_stride));
    args.scales = static_cast<float*>(call.matrix(a[10], blocks(c), rows, at::kFloat, &args.scale_stride));
    return call.ok ? call.result(lib.group_norm_fp8(call.ops, &args, call.stream)) : slow();
  }
  size_t on = 0, opx = 0, oc = 0;
  args.out = call.maps(a[9], &on, &opx, &oc, &args.out_stride, &args.out_map_stride);
  if (!call.ok) return slow();
  const at::Tensor& out = THPVariable_Unpack(a[9]);
  if (out.scalar_type() != x.scalar_type() || out.sizes() != x.sizes()) return slow();
  return call.result(lib.group_norm(call.ops, &args, call.stream));
}

// (handle, device, stream, x, block_rows, codes, scales)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) return slow();
  Call call(a[0], a[1], a[2]);
  const at::Tensor* x = call.tensor(a[3]);
  if (!x || x->dim() != 2) return slow();
  iec_quantize_fp8_args args = {};
  const int64_t rows = x->size(0), k = x->size(1), block_rows = call.integer(a[4]);
  args.x = call.matrix(a[3], rows, k, x->scalar_type(), &args.x_stride);
  args.dtype = call.dtype(*x);
  args.rows = (size_t)rows;
  args.k = (size_t)k;
  args.block_rows = block_rows > 0 ? (size_t)block_rows : 0;
  args.codes = static_cast<uint8_t*>(call.matrix(a[5], rows, k, at::kFloat8_e4m3fn, &args.code_stride));
  args.scales = static_cast<float*>(
      call.matrix(a[6], blocks(k), block_rows == BLOCK ? blocks(rows) : rows, at::kFloat, &args.scale_stride));
  return call.ok ? call.result(lib.quantize_fp8(call.ops, &args, call.stream)) : slow();
}

// (handle, device, stream, a, a_scales, w, w_scales, bias, act, residual, out)
PyObject* matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 11) return slow();
  Call call(a[0], a[1], a[2]);
  const at::Tensor *ta = call.tensor(a[3]), *tw = call.tensor(a[5]), *out = call.tensor(a[10]);
  if (!call.ok || ta->dim() != 2 || tw->dim() != 2) return slow();
  iec_matmul_fp8_args args = {};
  const int64_t m = ta->size(0), k = ta->size(1), cols = tw->size(0);
  args.a = static_cast<const uint8_t*>(call.matrix(a[3], m, k, at::kFloat8_e4m3fn, &args.a_stride));
  args.a_scales = static_cast<const float*>(call.matrix(a[4], blocks(k), m, at::kFloat, &args.a_scale_stride));
  args.w = static_cast<const uint8_t*>(call.matrix(a[5], cols, k, at::kFloat8_e4m3fn, &args.w_stride));
  args.w_scales =
      static_cast<const float*>(call.matrix(a[6], blocks(k), blocks(cols), at::kFloat, &args.w_scale_stride));
  args.bias = call.vector(a[7], cols);
  args.act = (int)call.integer(a[8]);
  if (a[9] != Py_None) args.residual = call.matrix(a[9], m, cols, out->scalar_type(), &args.residual_stride);
  args.out = call.matrix(a[10], m, cols, out->scalar_type(), &args.out_stride);
  args.dtype = call.dtype(*out);
  args.m = (size_t)m;
  args.n = (size_t)cols;
  args.k = (size_t)k;
  return call.ok ? call.result(lib.matmul_fp8(call.ops, &args, call.stream)) : slow();
}

// The library's entry points, by address.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "bind takes four addresses");
    return nullptr;
  }
  void* at[4];
  for (int i = 0; i < 4; i++) at[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  lib.group_norm = reinterpret_cast<decltype(lib.group_norm)>(at[0]);
  lib.group_norm_fp8 = reinterpret_cast<decltype(lib.group_norm_fp8)>(at[1]);
  lib.quantize_fp8 = reinterpret_cast<decltype(lib.quantize_fp8)>(at[2]);
  lib.matmul_fp8 = reinterpret_cast<decltype(lib.matmul_fp8)>(at[3]);
  Py_RETURN_NONE;
}

// C++ exceptions (a tensor without storage, say) leave the fast path too.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  try {
    return F(self, a, n);
  } catch (const std::exception&) {
    PyErr_Clear();
    return slow();
  }
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<F>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<bind>("bind"),         method<group_norm<false>>("group_norm"),
                         method<group_norm<true>>("group_norm_fp8"), method<quantize>("quantize_fp8"),
                         method<matmul>("matmul_fp8"), {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops_binding() { return PyModule_Create(&module); }
