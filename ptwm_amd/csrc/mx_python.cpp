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
#include <ATen/ops/empty.h>
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
decltype(&ptwm_mi355x_mxfp4_quantise_cuda) g_quantise;
decltype(&ptwm_mi355x_mxfp4_matmul_cuda) g_matmul;
decltype(&ptwm_mi355x_mxfp4_moe_workspace) g_moe_workspace;
decltype(&ptwm_mi355x_mxfp4_moe_cuda) g_moe;

PyObject* g_stream;  // torch's current stream of a device
PyObject* g_error;   // NativeError
PyObject* g_memory;  // torch.OutOfMemoryError

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
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(g_memory, e.what_without_backtrace());
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

PyObject* mxfp4_quantise_cuda(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* keywords) {
  return guarded([&]() -> PyObject* {
    static const char* names[] = {"x", "codes", "scales", "device_ordinal", "saturate"};
    PyObject* a[5];
    take_args(names, 3, args, n, keywords, a);
    const int64_t device = device_of(a[3]);
    const at::Tensor& x = input(a[0], "x");
    const int64_t rows = x.size(0), cols = x.size(1);
    const Rows xr = matrix(x, "x", rows, cols, device, kReal);
    const Rows codes = matrix(tensor(a[1], "codes"), "codes", rows, cols / 2, device, kWeight);
    const Rows scales = matrix(tensor(a[2], "scales"), "scales", rows, cols / 32, device, kScales);
    const int saturate = a[4] ? PyObject_IsTrue(a[4]) : 1;
    if (saturate < 0) throw Failed();
    if (rows == 0) Py_RETURN_NONE;
    return done(g_quantise(code_of(x.scalar_type()), xr.ptr, xr.stride, codes.ptr, codes.stride, scales.ptr,
                           scales.stride, rows, cols, saturate, stream_of(device), (uint32_t)device),
                "mxfp4_quantise_cuda");
  });
}

PyObject* mxfp4_matmul_cuda(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* keywords) {
  return guarded([&]() -> PyObject* {
    static const char* names[] = {"x", "x_scales", "weight", "scales", "out", "device_ordinal", "bias"};
    PyObject* a[7];
    take_args(names, 5, args, n, keywords, a);
    const int64_t device = device_of(a[5]);
    const at::Tensor& x = tensor(a[0], "x");
    if (x.dim() != 2) fail(PyExc_ValueError, "x: expected a matrix, a row a token");
    const int64_t tokens = x.size(0), half = x.size(1);
    if (half == 0 || half % 16) fail(PyExc_ValueError, "x: %lld bytes of codes are not whole blocks of 16", (long long)half);
    const Rows xr = matrix(x, "x", tokens, half, device, kWeight);
    const Rows xs = matrix(tensor(a[1], "x_scales"), "x_scales", tokens, half / 16, device, kScales);
    const at::Tensor& weight = tensor(a[2], "weight");
    const int64_t rows = weight.dim() ? weight.size(0) : 0;
    const Rows w = matrix(weight, "weight", rows, half, device, kWeight);
    const Rows s = matrix(tensor(a[3], "scales"), "scales", rows, half / 16, device, kScales);
    const at::Tensor& out = tensor(a[4], "out");
    const Rows o = matrix(out, "out", tokens, rows, device, kReal);
    const uint64_t bias = a[6] ? vector(tensor(a[6], "bias"), "bias", rows, device, {out.scalar_type()}) : 0;
    if (tokens == 0 || rows == 0) Py_RETURN_NONE;
    return done(g_matmul(xr.ptr, xr.stride, xs.ptr, xs.stride, w.ptr, w.stride, s.ptr, s.stride,
                         code_of(out.scalar_type()), bias, o.ptr, o.stride, tokens, rows, half * 2,
                         stream_of(device), (uint32_t)device),
                "mxfp4_matmul_cuda");
  });
}

// A stack of matrices [experts, rows, cols] whose rows are contiguous and do not overlap: address, rows' and experts'
// strides.
void stack(PyObject* o, const char* name, int64_t experts, int64_t rows, int64_t cols, int64_t device,
           const Types& types, uint64_t& ptr, uint64_t& stride, uint64_t& expert) {
  const at::Tensor& t = tensor(o, name);
  check_place(t, name, device, types);
  if (t.dim() != 3 || t.size(0) != experts || t.size(1) != rows || t.size(2) != cols) {
    std::string shape;
    for (int64_t s : t.sizes()) shape += (shape.empty() ? "" : ", ") + std::to_string(s);
    fail(PyExc_ValueError, "%s: shape (%s) is not (%lld, %lld, %lld)", name, shape.c_str(), (long long)experts,
         (long long)rows, (long long)cols);
  }
  if ((t.stride(2) != 1 && cols > 1) || (t.stride(1) < cols && rows > 1))
    fail(PyExc_ValueError, "%s: rows must be contiguous and must not overlap", name);
  ptr = reinterpret_cast<uint64_t>(t.data_ptr()), stride = (uint64_t)t.stride(1), expert = (uint64_t)t.stride(0);
}

// One product's weights: codes, scales and an optional bias [experts, rows] at any strides.
ptwm_mi355x_experts experts_of(PyObject* codes, const char* name, PyObject* scales, const char* scales_name,
                               PyObject* bias, const char* bias_name, int64_t experts, int64_t rows, int64_t cols,
                               int64_t device, at::ScalarType bias_type) {
  ptwm_mi355x_experts w = {};
  stack(codes, name, experts, rows, cols / 2, device, kWeight, w.codes, w.codes_stride, w.codes_expert);
  stack(scales, scales_name, experts, rows, cols / 32, device, kScales, w.scales, w.scales_stride, w.scales_expert);
  if (bias) {
    const at::Tensor& b = tensor(bias, bias_name);
    check_place(b, bias_name, device, {bias_type});
    if (b.dim() != 2 || b.size(0) != experts || b.size(1) != rows)
      fail(PyExc_ValueError, "%s: shape is not (%lld, %lld)", bias_name, (long long)experts, (long long)rows);
    w.bias = reinterpret_cast<uint64_t>(b.data_ptr());
    w.bias_stride = (uint64_t)b.stride(1), w.bias_expert = (uint64_t)b.stride(0);
  }
  return w;
}

PyObject* mxfp4_moe_cuda(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* keywords) {
  return guarded([&]() -> PyObject* {
    static const char* names[] = {"x",         "router",    "gate",           "gate_scales", "up",        "up_scales",
                                  "down",      "down_scales", "out",          "top_k",       "device_ordinal",
                                  "router_bias", "gate_bias", "up_bias",      "down_bias",   "experts",   "weights"};
    PyObject* a[17];
    take_args(names, 10, args, n, keywords, a);
    ptwm_mi355x_mxfp4_moe c = {};
    const int64_t device = device_of(a[10]);
    const at::Tensor& x = input(a[0], "x");
    const int64_t tokens = x.size(0), cols = x.size(1);
    const Rows xr = matrix(x, "x", tokens, cols, device, kReal);
    const at::Tensor& router = tensor(a[1], "router");
    const int64_t experts = router.dim() ? router.size(0) : 0;
    const Rows r = matrix(router, "router", experts, cols, device, kReal);
    const at::Tensor& gate = tensor(a[2], "gate");
    const int64_t inner = gate.dim() == 3 ? gate.size(1) : 0;
    if (inner == 0 || inner % 32)
      fail(PyExc_ValueError, "gate: expected [experts, inner, cols / 2] with inner in whole blocks of 32");
    const at::Tensor& out = tensor(a[8], "out");
    const Rows o = matrix(out, "out", tokens, cols, device, kReal);
    const int64_t top_k = PyLong_AsLongLong(a[9]);
    if (top_k == -1 && PyErr_Occurred()) throw Failed();
    if (top_k < 1 || top_k > 32 || top_k > experts || experts > 1024)
      fail(PyExc_ValueError, "top_k: %lld of %lld experts, up to 32 of up to 1024 can be chosen", (long long)top_k,
           (long long)experts);
    if (cols > 131072 || inner > 131072) fail(PyExc_ValueError, "x, gate: rows and inner sizes up to 131072 are taken");
    const at::ScalarType type = out.scalar_type();
    c.gate = experts_of(a[2], "gate", a[3], "gate_scales", a[12], "gate_bias", experts, inner, cols, device, type);
    c.up = experts_of(a[4], "up", a[5], "up_scales", a[13], "up_bias", experts, inner, cols, device, type);
    c.down = experts_of(a[6], "down", a[7], "down_scales", a[14], "down_bias", experts, cols, inner, device, type);
    if (a[11]) c.router_bias = vector(tensor(a[11], "router_bias"), "router_bias", experts, device, {router.scalar_type()});
    const auto chosen = [&](PyObject* t, const char* name, at::ScalarType kind) -> uint64_t {
      if (!t) return 0;
      const Rows m = matrix(tensor(t, name), name, tokens, top_k, device, {kind});
      if (!THPVariable_Unpack(t).is_contiguous()) fail(PyExc_ValueError, "%s: must be contiguous", name);
      return m.ptr;
    };
    c.experts_out = chosen(a[15], "experts", at::kInt);
    c.weights_out = chosen(a[16], "weights", at::kFloat);
    if (tokens == 0) Py_RETURN_NONE;
    c.x = xr.ptr, c.x_stride = xr.stride, c.router = r.ptr, c.router_stride = r.stride;
    c.out = o.ptr, c.out_stride = o.stride;
    c.tokens = tokens, c.experts = experts, c.top_k = top_k, c.cols = cols, c.inner = inner;
    c.x_dtype = code_of(x.scalar_type()), c.router_dtype = code_of(router.scalar_type()), c.out_dtype = code_of(type);
    const int64_t bytes = g_moe_workspace(&c);
    if (bytes < 0) return done(bytes, "mxfp4_moe_cuda");
    // from torch's allocator: the current stream's, or a captured graph's own, so no two calls at once share it
    const at::Tensor workspace =
        at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, (at::DeviceIndex)device));
    c.workspace = reinterpret_cast<uint64_t>(workspace.data_ptr()), c.workspace_bytes = bytes;
    return done(g_moe(&c, stream_of(device), (uint32_t)device), "mxfp4_moe_cuda");
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

PyDoc_STRVAR(kQuantiseDoc,
             "mxfp4_quantise_cuda(x, codes, scales, device_ordinal=0, saturate=True)\n--\n\n"
             "Values to MXFP4 (library addition): ``codes`` [rows, cols / 2] (uint8 or\n"
             "float4_e2m1fn_x2) receives e2m1 codes, the first of two in the low nibble,\n"
             "``scales`` [rows, cols / 32] (float8_e8m0fnu or uint8) a power of two for\n"
             "each block of 32.  With ``saturate`` the scale leaves a block's largest\n"
             "magnitude in [4, 8) and what is above 6 becomes 6; without it the scale is\n"
             "the smallest with which nothing is above 6.  Codes are rounded to nearest,\n"
             "ties to even.  A block with an infinity or NaN gets the scale NaN.\n"
             "x [rows, cols]: float32, float16 or bfloat16, rows at any stride.\n"
             "Queued on torch's current stream; nothing is waited for.");
PyDoc_STRVAR(kMatmulDoc,
             "mxfp4_matmul_cuda(x, x_scales, weight, scales, out, device_ordinal=0, bias=None)\n--\n\n"
             "``out = x @ W.T (+ bias)`` with both matrices in MXFP4 (library addition):\n"
             "``x`` [tokens, cols / 2] and ``weight`` [rows, cols / 2] hold e2m1 codes,\n"
             "``x_scales`` and ``scales`` their E8M0 bytes, as mxfp4_quantise_cuda writes\n"
             "them and a decode restores them.  out [tokens, rows] is float32, float16 or\n"
             "bfloat16, bias [rows] of out's dtype.  Products are exact, sums are held in\n"
             "32 bits.  Rows may lie at any stride, but are contiguous.\n"
             "Queued on torch's current stream; nothing is waited for.");
PyDoc_STRVAR(kMoeDoc,
             "mxfp4_moe_cuda(x, router, gate, gate_scales, up, up_scales, down, down_scales, out, top_k,\n"
             "               device_ordinal=0, router_bias=None, gate_bias=None, up_bias=None, down_bias=None,\n"
             "               experts=None, weights=None)\n--\n\n"
             "A mixture-of-experts layer on MXFP4 experts for a few tokens (library\n"
             "addition).  A token's logits are ``x @ router.T (+ router_bias)``, summed in\n"
             "64 bits; its top_k experts are those with the largest, the lowest index of\n"
             "equal ones, weighted by a softmax over them.  ``out`` is the weighted sum of\n"
             "``h @ down[e].T (+ down_bias[e])`` with ``h = silu(x @ gate[e].T\n"
             "(+ gate_bias[e])) * (x @ up[e].T (+ up_bias[e]))``.  A logit of minus\n"
             "infinity keeps an expert out, with the weight 0.\n\n"
             "x, out [tokens, cols] and router [experts, cols]: float32, float16 or\n"
             "bfloat16 each; router_bias [experts] of router's dtype.  gate and up\n"
             "[experts, inner, cols / 2] and down [experts, cols, inner / 2] hold e2m1\n"
             "codes, with scales [..., / 32], as a decode restores them; their rows are\n"
             "contiguous, at any stride: views of one tensor, its halves or every second\n"
             "row, will do.  gate_bias, up_bias [experts, inner] and down_bias [experts,\n"
             "cols]: out's dtype, any strides.  ``experts`` (int32) and ``weights``\n"
             "(float32) [tokens, top_k], contiguous, receive the choice, largest first.\n"
             "out may be x.  Up to 32 of up to 1024 experts; more than 64 tokens take\n"
             "several passes over the weights.  The workspace comes from torch's\n"
             "allocator.  Queued on torch's current stream; nothing is waited for.");

PyMethodDef kMethods[] = {
    {"rms_norm_mx_cuda", (PyCFunction)(void (*)(void))rms_norm_mx_cuda, METH_FASTCALL | METH_KEYWORDS, kNormDoc},
    {"swiglu_mx_cuda", (PyCFunction)(void (*)(void))swiglu_mx_cuda, METH_FASTCALL | METH_KEYWORDS, kSwigluDoc},
    {"mxfp4_linear_cuda", (PyCFunction)(void (*)(void))mxfp4_linear_cuda, METH_FASTCALL | METH_KEYWORDS, kLinearDoc},
    {"mxfp4_quantise_cuda", (PyCFunction)(void (*)(void))mxfp4_quantise_cuda, METH_FASTCALL | METH_KEYWORDS, kQuantiseDoc},
    {"mxfp4_matmul_cuda", (PyCFunction)(void (*)(void))mxfp4_matmul_cuda, METH_FASTCALL | METH_KEYWORDS, kMatmulDoc},
    {"mxfp4_moe_cuda", (PyCFunction)(void (*)(void))mxfp4_moe_cuda, METH_FASTCALL | METH_KEYWORDS, kMoeDoc},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "ptwm_amd._mx", "Operators on MX blocks.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mx(void) {
  PyObject* torch_c = PyImport_ImportModule("torch._C");
  if (!torch_c) return nullptr;
  g_stream = PyObject_GetAttrString(torch_c, "_cuda_getCurrentRawStream");
  g_memory = g_stream ? PyObject_GetAttrString(torch_c, "OutOfMemoryError") : nullptr;
  Py_DECREF(torch_c);
  PyObject* native = g_memory ? PyImport_ImportModule("ptwm_amd._native") : nullptr;
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
    g_quantise = reinterpret_cast<decltype(g_quantise)>(dlsym(lib, "ptwm_mi355x_mxfp4_quantise_cuda"));
    g_matmul = reinterpret_cast<decltype(g_matmul)>(dlsym(lib, "ptwm_mi355x_mxfp4_matmul_cuda"));
    g_moe_workspace = reinterpret_cast<decltype(g_moe_workspace)>(dlsym(lib, "ptwm_mi355x_mxfp4_moe_workspace"));
    g_moe = reinterpret_cast<decltype(g_moe)>(dlsym(lib, "ptwm_mi355x_mxfp4_moe_cuda"));
  }
  if (!g_norm || !g_swiglu || !g_linear || !g_quantise || !g_matmul || !g_moe_workspace || !g_moe) {
    PyErr_SetString(PyExc_ImportError, "the library lacks the operators on MX blocks");
    return nullptr;
  }
  return PyModule_Create(&kModule);
}
