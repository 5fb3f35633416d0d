// mx_python.cpp -- the Python entry points of the operators on MX blocks
// (ptwm_amd.api serves them from here).
//
// The smallest calls cost the host more than the GPU, and reading a tensor's
// size, type and address through Python's attributes cost more than the launch:
// 3 us for five tensors.  Here they are read from the tensor itself; checks and
// errors are the same as the rest of the package's: TypeError for what is not a
// tensor of the wanted type, ValueError for sizes, strides and devices,
// NativeError for a refusal of the library.
#define PY_SSIZE_T_CLEAN
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstring>
#include <initializer_list>
#include <string>

#include "../../include/ptwm_mi355x.h"

namespace {

struct Failed {};  // a Python error is set

[[noreturn]] void fail(PyObject* type, const char* format, ...) {
  va_list args;
  va_start(args, format);
  PyErr_FormatV(type, format, args);
  va_end(args);
  throw Failed();
}

// The arguments of a call by position or name; nullptr where one is absent or None.
template <size_t N>
void take_args(const char* (&names)[N], size_t required, PyObject* const* args, Py_ssize_t n, PyObject* keywords,
               PyObject* (&out)[N]) {
  if ((size_t)n > N) fail(PyExc_TypeError, "takes at most %zu arguments (%zd given)", N, n);
  for (size_t i = 0; i < N; ++i) out[i] = i < (size_t)n ? args[i] : nullptr;
  const Py_ssize_t nk = keywords ? PyTuple_GET_SIZE(keywords) : 0;
  for (Py_ssize_t k = 0; k < nk; ++k) {
    PyObject* key = PyTuple_GET_ITEM(keywords, k);
    size_t i = 0;
    while (i < N && PyUnicode_CompareWithASCIIString(key, names[i]) != 0) ++i;
    if (i == N) fail(PyExc_TypeError, "got an unexpected keyword argument '%U'", key);
    if (out[i]) fail(PyExc_TypeError, "got multiple values for argument '%s'", names[i]);
    out[i] = args[n + k];
  }
  for (size_t i = 0; i < N; ++i) {
    if (out[i] == Py_None) out[i] = nullptr;
    if (!out[i] && i < required) fail(PyExc_TypeError, "missing argument '%s'", names[i]);
  }
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) fail(PyExc_TypeError, "%s: expected a device tensor", name);
  return THPVariable_Unpack(o);
}

typedef std::initializer_list<at::ScalarType> Types;
const Types kReal = {at::kBFloat16, at::kHalf, at::kFloat};
const Types kE4m3 = {at::kFloat8_e4m3fn};
const Types kCodes = {at::kFloat8_e4m3fn, at::kByte};
const Types kScales = {at::kFloat8_e8m0fnu, at::kByte};
const Types kWeight = {at::kByte, at::kFloat4_e2m1fn_x2};

// Public dtype codes (dtype.rs:79-103).
uint32_t code_of(at::ScalarType t) {
  return t == at::kFloat ? 1 : t == at::kHalf ? 4 : t == at::kBFloat16 ? 6 : 29;
}

void check_place(const at::Tensor& t, const char* name, int64_t device, const Types& types) {
  bool wanted = false;
  for (at::ScalarType s : types) wanted = wanted || t.scalar_type() == s;
  if (!wanted) {
    std::string list;
    for (at::ScalarType s : types) list += (list.empty() ? "" : ", ") + std::string(c10::toString(s));
    fail(PyExc_TypeError, "%s: dtype %s is not one of %s", name, c10::toString(t.scalar_type()), list.c_str());
  }
  if (t.is_neg()) fail(PyExc_ValueError, "%s: a lazily negated view, resolve it first (Tensor.resolve_neg)", name);
  if (!t.is_cuda()) fail(PyExc_ValueError, "%s: tensor is not on a GPU device", name);
  if (t.get_device() != device)
    fail(PyExc_ValueError, "%s: tensor is on device %d, call names device %lld", name, (int)t.get_device(),
         (long long)device);
}

struct Rows {
  uint64_t ptr = 0, stride = 0;
};

// A matrix of the given size and one of the types, whose rows are contiguous and do not overlap.
Rows matrix(const at::Tensor& t, const char* name, int64_t rows, int64_t cols, int64_t device, const Types& types) {
  check_place(t, name, device, types);
  if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols) {
    std::string shape;
    for (int64_t s : t.sizes()) shape += (shape.empty() ? "" : ", ") + std::to_string(s);
    fail(PyExc_ValueError, "%s: shape (%s) is not (%lld, %lld)", name, shape.c_str(), (long long)rows,
         (long long)cols);
  }
  if ((t.stride(1) != 1 && cols > 1) || (t.stride(0) < cols && rows > 1))
    fail(PyExc_ValueError, "%s: rows must be contiguous and must not overlap", name);
  return {reinterpret_cast<uint64_t>(t.data_ptr()), (uint64_t)t.stride(0)};
}

uint64_t vector(const at::Tensor& t, const char* name, int64_t n, int64_t device, const Types& types) {
  check_place(t, name, device, types);
  if (t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
    fail(PyExc_ValueError, "%s: expected %lld contiguous elements", name, (long long)n);
  return reinterpret_cast<uint64_t>(t.data_ptr());
}

// The first input: rows of whole blocks of 32.
const at::Tensor& input(PyObject* o, const char* name) {
  const at::Tensor& t = tensor(o, name);
  if (t.dim() != 2) fail(PyExc_ValueError, "%s: expected a matrix, a row a token", name);
  if (t.size(1) == 0 || t.size(1) % 32)
    fail(PyExc_ValueError, "%s: %lld columns are not whole blocks of 32", name, (long long)t.size(1));
  return t;
}

int64_t device_of(PyObject* o) {
  if (!o) return 0;
  const long long d = PyLong_AsLongLong(o);
  if (d == -1 && PyErr_Occurred()) throw Failed();
  if (d < 0 || d > 0x7FFFFFFF) fail(PyExc_ValueError, "device_ordinal: %lld is not a device", d);
  return d;
}

// The library's entry points, from the file that ptwm_amd._native loads.
decltype(&ptwm_mi355x_rms_norm_mx_cuda) g_norm;
decltype(&ptwm_mi355x_swiglu_mx_cuda) g_swiglu;
decltype(&ptwm_mi355x_mxfp4_linear_cuda) g_linear;

PyObject* g_stream;  // torch's current stream of a device
PyObject* g_error;   // NativeError

uint64_t stream_of(int64_t device) {
  PyObject* d = PyLong_FromLongLong(device);
  if (!d) throw Failed();
  PyObject* s = PyObject_CallOneArg(g_stream, d);
  Py_DECREF(d);
  if (!s) throw Failed();
  const unsigned long long v = PyLong_AsUnsignedLongLong(s);
  Py_DECREF(s);
  if (PyErr_Occurred()) throw Failed();
  return v;
}

PyObject* done(int64_t rc, const char* what) {
  if (rc == 0) Py_RETURN_NONE;
  PyObject* e = PyObject_CallFunction(g_error, "Ls", (long long)rc, what);
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  return nullptr;
}

// Runs a call; C++ and HIP errors inside torch's accessors become Python's.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const Failed&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyObject* rms_norm_mx_cuda(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* keywords) {
  return guarded([&]() -> PyObject* {
    static const char* names[] = {"x", "weight", "out", "out_scales", "device_ordinal", "residual", "sum_out", "eps"};
    PyObject* a[8];
    take_args(names, 4, args, n, keywords, a);
    const int64_t device = device_of(a[4]);
    const at::Tensor& x = input(a[0], "x");
    const int64_t rows = x.size(0), cols = x.size(1);
    const Rows xr = matrix(x, "x", rows, cols, device, kReal);
    const Types same = {x.scalar_type()};
    const at::Tensor& weight = tensor(a[1], "weight");
    const uint64_t w = vector(weight, "weight", cols, device, kReal);
    Rows residual, sum;
    if (a[5]) residual = matrix(tensor(a[5], "residual"), "residual", rows, cols, device, same);
    if (a[6]) sum = matrix(tensor(a[6], "sum_out"), "sum_out", rows, cols, device, same);
    const Rows out = matrix(tensor(a[2], "out"), "out", rows, cols, device, kCodes);
    const Rows scales = matrix(tensor(a[3], "out_scales"), "out_scales", rows, cols / 32, device, kScales);
    const double eps = a[7] ? PyFloat_AsDouble(a[7]) : 1e-6;
    if (eps == -1.0 && PyErr_Occurred()) throw Failed();
    if (rows == 0) Py_RETURN_NONE;
    return done(g_norm(code_of(x.scalar_type()), xr.ptr, xr.stride, residual.ptr,
                                             residual.stride, code_of(weight.scalar_type()), w, (float)eps, sum.ptr,
                                             sum.stride, out.ptr, out.stride, scales.ptr, scales.stride, rows, cols,
                                             stream_of(device), (uint32_t)device),
                "rms_norm_mx_cuda");
  });
}

PyObject* swiglu_mx_cuda(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* keywords) {
  return guarded([&]() -> PyObject* {
    static const char* names[] = {"gate", "up", "out", "out_scales", "device_ordinal"};
    PyObject* a[5];
    take_args(names, 4, args, n, keywords, a);
    const int64_t device = device_of(a[4]);
    const at::Tensor& gate = input(a[0], "gate");
    const int64_t rows = gate.size(0), cols = gate.size(1);
    const Rows g = matrix(gate, "gate", rows, cols, device, kReal);
    const Rows u = matrix(tensor(a[1], "up"), "up", rows, cols, device, {gate.scalar_type()});
    const Rows out = matrix(tensor(a[2], "out"), "out", rows, cols, device, kCodes);
    const Rows scales = matrix(tensor(a[3], "out_scales"), "out_scales", rows, cols / 32, device, kScales);
    if (rows == 0) Py_RETURN_NONE;
    return done(g_swiglu(code_of(gate.scalar_type()), g.ptr, g.stride, u.ptr, u.stride, out.ptr,
                                           out.stride, scales.ptr, scales.stride, rows, cols, stream_of(device),
                                           (uint32_t)device),
                "swiglu_mx_cuda");
  });
}

PyObject* mxfp4_linear_cuda(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* keywords) {
  return guarded([&]() -> PyObject* {
    static const char* names[] = {"x", "weight", "scales", "out", "device_ordinal", "x_scales", "bias"};
    PyObject* a[7];
    take_args(names, 4, args, n, keywords, a);
    const int64_t device = device_of(a[4]);
    const at::Tensor& x = input(a[0], "x");
    const int64_t tokens = x.size(0), cols = x.size(1);
    const bool eight = x.scalar_type() == at::kFloat8_e4m3fn;
    if (eight != (a[5] != nullptr))
      fail(PyExc_ValueError, "x_scales: wanted with float8_e4m3fn activations, and only there");
    const Rows xr = matrix(x, "x", tokens, cols, device, eight ? kE4m3 : kReal);
    Rows xs;
    if (eight) xs = matrix(tensor(a[5], "x_scales"), "x_scales", tokens, cols / 32, device, kScales);
    const at::Tensor& weight = tensor(a[1], "weight");
    const int64_t rows = weight.dim() ? weight.size(0) : 0;
    const Rows w = matrix(weight, "weight", rows, cols / 2, device, kWeight);
    const Rows s = matrix(tensor(a[2], "scales"), "scales", rows, cols / 32, device, kScales);
    const at::Tensor& out = tensor(a[3], "out");
    const Rows o = matrix(out, "out", tokens, rows, device, kReal);
    const uint64_t bias = a[6] ? vector(tensor(a[6], "bias"), "bias", rows, device, {out.scalar_type()}) : 0;
    if (tokens == 0 || rows == 0) Py_RETURN_NONE;
    return done(g_linear(code_of(x.scalar_type()), xr.ptr, xr.stride, xs.ptr, xs.stride, w.ptr,
                                              w.stride, s.ptr, s.stride, code_of(out.scalar_type()), bias, o.ptr,
                                              o.stride, tokens, rows, cols, stream_of(device), (uint32_t)device),
                "mxfp4_linear_cuda");
  });
}

PyDoc_STRVAR(kNormDoc,
             "rms_norm_mx_cuda(x, weight, out, out_scales, device_ordinal=0, residual=None, sum_out=None, eps=1e-06)\n"
             "--\n\n"
             "Root-mean-square norm with an output in 8 bits (library addition):\n"
             "``s = x + residual``, ``y = s * rsqrt(mean(s**2) + eps) * weight`` for\n"
             "every row, in 32 bits.  ``out`` [rows, cols] (float8_e4m3fn or uint8)\n"
             "receives y's codes and ``out_scales`` [rows, cols / 32] (float8_e8m0fnu\n"
             "or uint8) a power of two for each block of 32: the smallest with which\n"
             "the block's largest magnitude is at most 448.  ``sum_out`` receives ``s``\n"
             "in x's dtype and may be ``x`` or ``residual`` itself.  x: float32,\n"
             "float16 or bfloat16, rows at any stride; weight: any of the three.\n"
             "Queued on torch's current stream; nothing is waited for.");
PyDoc_STRVAR(kSwigluDoc,
             "swiglu_mx_cuda(gate, up, out, out_scales, device_ordinal=0)\n--\n\n"
             "Gated activation with an output in 8 bits (library addition):\n"
             "``y = gate / (1 + exp(-gate)) * up`` in 32 bits, to ``out`` and\n"
             "``out_scales`` as rms_norm_mx_cuda writes them.  gate and up: float32,\n"
             "float16 or bfloat16, rows at any stride (the halves of one matrix, say).\n"
             "Queued on torch's current stream; nothing is waited for.");
PyDoc_STRVAR(kLinearDoc,
             "mxfp4_linear_cuda(x, weight, scales, out, device_ordinal=0, x_scales=None, bias=None)\n--\n\n"
             "``out = x @ W.T (+ bias)`` with MXFP4 weights (library addition):\n"
             "``weight`` [rows, cols / 2] holds e2m1 codes, the first of two in the low\n"
             "nibble, and ``scales`` [rows, cols / 32] their E8M0 bytes, as a decode\n"
             "restores them.  x [tokens, cols] is float32, float16, bfloat16, or\n"
             "float8_e4m3fn with ``x_scales`` [tokens, cols / 32]; out [tokens, rows]\n"
             "is float32, float16 or bfloat16, bias [rows] of out's dtype.  Sums are\n"
             "held in 32 bits.  Rows may lie at any stride, but are contiguous.\n"
             "Queued on torch's current stream; nothing is waited for.");

PyMethodDef kMethods[] = {
    {"rms_norm_mx_cuda", (PyCFunction)(void (*)(void))rms_norm_mx_cuda, METH_FASTCALL | METH_KEYWORDS, kNormDoc},
    {"swiglu_mx_cuda", (PyCFunction)(void (*)(void))swiglu_mx_cuda, METH_FASTCALL | METH_KEYWORDS, kSwigluDoc},
    {"mxfp4_linear_cuda", (PyCFunction)(void (*)(void))mxfp4_linear_cuda, METH_FASTCALL | METH_KEYWORDS, kLinearDoc},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "ptwm_amd._mx", "Operators on MX blocks.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mx(void) {
  PyObject* torch_c = PyImport_ImportModule("torch._C");
  if (!torch_c) return nullptr;
  g_stream = PyObject_GetAttrString(torch_c, "_cuda_getCurrentRawStream");
  Py_DECREF(torch_c);
  PyObject* native = g_stream ? PyImport_ImportModule("ptwm_amd._native") : nullptr;
  if (!native) return nullptr;
  g_error = PyObject_GetAttrString(native, "NativeError");
  PyObject* path = g_error ? PyObject_GetAttrString(native, "LIB_PATH") : nullptr;
  Py_DECREF(native);
  const char* file = path ? PyUnicode_AsUTF8(path) : nullptr;
  if (!file) return nullptr;
  void* lib = dlopen(file, RTLD_NOW | RTLD_LOCAL);
  Py_DECREF(path);
  if (lib) {
    g_norm = reinterpret_cast<decltype(g_norm)>(dlsym(lib, "ptwm_mi355x_rms_norm_mx_cuda"));
    g_swiglu = reinterpret_cast<decltype(g_swiglu)>(dlsym(lib, "ptwm_mi355x_swiglu_mx_cuda"));
    g_linear = reinterpret_cast<decltype(g_linear)>(dlsym(lib, "ptwm_mi355x_mxfp4_linear_cuda"));
  }
  if (!g_norm || !g_swiglu || !g_linear) {
    PyErr_SetString(PyExc_ImportError, "the library lacks the operators on MX blocks");
    return nullptr;
  }
  return PyModule_Create(&kModule);
}
