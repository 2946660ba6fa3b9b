// The host side of the 8-bit activation path's eager calls: argument checks,
// output tensors, the current stream and the call into libfp4x.so, as the
// Python module _fp4x_host.  fp4x_kernels.py holds the public functions and
// their documentation.
//
// Why it is compiled: at a few rows the kernels take 3 to 5 us and the launch
// itself 3.3 us of host time, so what is added around it is the call's time.
// The same code in Python (ctypes, torch.empty_strided) takes 7.5 us for
// quantize_q8, 7.7 for w8a8_linear and 10.5 for rms_norm_q8 with a residual.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <climits>
#include <string>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/fp4x.h"

namespace {

using at::Tensor;

// A Python exception of a given type, thrown through the functions below.
struct Refused {
  PyObject* type;
  std::string why;
};
[[noreturn]] void value_error(const std::string& why) { throw Refused{PyExc_ValueError, "fp4x: " + why}; }
[[noreturn]] void type_error(const std::string& why) { throw Refused{PyExc_TypeError, "fp4x: " + why}; }
[[noreturn]] void other_gpu() {
  throw Refused{PyExc_RuntimeError, "fp4x: HIP kernels need GPU tensors, all on one GPU"};
}

void check(int rc, const char* what) {
  if (rc != FP4X_OK)
    throw Refused{rc == FP4X_ERR_ARG ? PyExc_ValueError : PyExc_RuntimeError,
                  std::string("fp4x ") + what + ": " + fp4x_last_error()};
}

// Runs f without the interpreter's lock: a launch waits when its queue is full.
template <class F>
int launch(F f) {
  PyThreadState* st = PyEval_SaveThread();
  const int rc = f();
  PyEval_RestoreThread(st);
  return rc;
}

const Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) type_error(std::string(what) + " must be a tensor");
  return THPVariable_Unpack(o);
}
const Tensor* optional_tensor(PyObject* o, const char* what) {
  return o == Py_None ? nullptr : &tensor(o, what);
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return FP4X_DT_BF16;
    case at::kFloat: return FP4X_DT_F32;
    case at::kHalf: return FP4X_DT_F16;
    default: type_error(std::string("unsupported dtype ") + at::toString(t) + " (bf16, fp16 or fp32)");
  }
}

int to_int(int64_t v) {
  if (v > INT_MAX) value_error("a tensor has more than 2^31 - 1 rows or columns");
  return (int)v;
}

void on_gpu(const Tensor& t) {
  if (!t.is_cuda()) other_gpu();
}
void same_gpu(const Tensor& t, const Tensor& as) {
  if (!t.is_cuda() || t.get_device() != as.get_device()) other_gpu();
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

Tensor make(at::IntArrayRef size, at::IntArrayRef stride, at::ScalarType t, const Tensor& like) {
  return at::detail::empty_strided_cuda(size, stride, t, like.device());
}
Tensor rows(int64_t m, int64_t h, at::ScalarType t, const Tensor& like) { return make({m, h}, {h, 1}, t, like); }

// 2-D rows with unit column stride; copied where they have another.
Tensor rows2(const Tensor& t, const char* what) {
  if (t.dim() != 2) value_error(std::string(what) + " must be 2-D");
  return t.stride(1) == 1 || t.size(1) == 1 ? t : t.contiguous();
}

// A tensor of a given type over part of a storage.
Tensor part(const c10::Storage& storage, int64_t at_byte, at::IntArrayRef size, at::IntArrayRef stride, at::ScalarType t) {
  Tensor x = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(storage), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                      c10::scalarTypeToTypeMeta(t));
  x.unsafeGetTensorImpl()->set_sizes_and_strides(size, stride, at_byte / (int64_t)c10::elementSize(t));
  return x;
}

// An output in 8 bits.  Code rows start on 16 bytes, as w8a8_linear reads them;
// a row of another length is padded.  Up to 1 MiB codes and scales are one
// allocation, which takes 0.4 us less than two of the 5 that such a call takes;
// torch's allocator serves requests of that size from blocks of 2 MiB, so what a
// caller who keeps only one of them holds in vain stays below its granularity.
// Above, where the kernel takes longer than the host, each has its own: a
// weight's scales do not keep its codes, nor a saved tensor the other one.
constexpr int64_t kShared = 1 << 20;
// The stride of code rows with scales per 128 values: they start on a cache line where that adds a sixteenth at most.  The
// products read a row 128 bytes at a time, and a line that two of those share is asked for twice: 250 x [13310 x 2500] take
// 20.3 us with rows of both operands 2512 bytes apart, 17.2 with 2560; 4096 x [16384 x 2500] 172 and 155.
int64_t line_rows(int64_t k) {
  const int64_t lines = (k + 127) & -128;
  return (lines - k) * 16 <= k ? lines : (k + 15) & -16;
}
struct Codes {
  int fmt;
  Tensor q, s;
};
Codes make_codes(int64_t m, int64_t h, PyObject* fmt, const Tensor& like) {
  int f = -1;
  if (PyUnicode_Check(fmt)) {
    if (PyUnicode_CompareWithASCIIString(fmt, "int8") == 0) f = FP4X_Q8_INT8;
    else if (PyUnicode_CompareWithASCIIString(fmt, "e4m3") == 0) f = FP4X_Q8_E4M3;
    else if (PyUnicode_CompareWithASCIIString(fmt, "mx8") == 0) f = FP4X_Q8_MX8;
    else if (PyUnicode_CompareWithASCIIString(fmt, "e4m3_g128") == 0) f = FP4X_Q8_E4M3_G128;
  }
  if (f < 0) value_error("fmt is one of 'int8', 'e4m3', 'mx8' and 'e4m3_g128'");
  const int64_t ld = f == FP4X_Q8_E4M3_G128 ? line_rows(h) : (h + 15) & -16, blocks = f == FP4X_Q8_E4M3_G128 ? (h + 127) / 128 : h / 32;
  const int64_t bytes = m * ld + m * (f == FP4X_Q8_MX8 ? blocks : f == FP4X_Q8_E4M3_G128 ? 4 * blocks : 4);
  const at::ScalarType qt = f == FP4X_Q8_INT8 ? at::kChar : at::kFloat8_e4m3fn;
  Codes c;
  c.fmt = f;
  if (bytes > kShared) {
    c.q = part(make({m * ld}, {1}, at::kByte, like).storage(), 0, {m, h}, {ld, 1}, qt);   // whole rows, the last too
    c.s = f == FP4X_Q8_MX8         ? rows(m, blocks, at::kByte, like)
          : f == FP4X_Q8_E4M3_G128 ? make({m, blocks}, {1, m}, at::kFloat, like)
                                   : make({m}, {1}, at::kFloat, like);
    return c;
  }
  const c10::Storage both = make({bytes}, {1}, at::kByte, like).storage();
  c.q = part(both, 0, {m, h}, {ld, 1}, qt);
  c.s = f == FP4X_Q8_MX8         ? part(both, m * ld, {m, blocks}, {blocks, 1}, at::kByte)
        : f == FP4X_Q8_E4M3_G128 ? part(both, m * ld, {m, blocks}, {1, m}, at::kFloat)
                                 : part(both, m * ld, {m}, {1}, at::kFloat);
  return c;
}

PyObject* pack(std::initializer_list<Tensor> ts) {
  PyObject* t = PyTuple_New((Py_ssize_t)ts.size());
  if (!t) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor& x : ts) {
    PyObject* o = THPVariable_Wrap(x);
    if (!o) {
      Py_DECREF(t);
      return nullptr;
    }
    PyTuple_SET_ITEM(t, i++, o);
  }
  return t;
}

double number(PyObject* o, const char* what) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    type_error(std::string(what) + " must be a number");
  }
  return v;
}

// rms_norm_q8(x, w, eps, residual, fmt, w_offset, normed, residual_out)
PyObject* rms_norm_q8(PyObject* const* a) {
  const Tensor &x0 = tensor(a[0], "x"), &w0 = tensor(a[1], "the norm weight");
  on_gpu(x0);
  same_gpu(w0, x0);
  const Tensor x = rows2(x0, "x");
  const int64_t m = x.size(0), h = x.size(1);
  const int dt = dtype_code(x.scalar_type());
  if (w0.dim() != 1 || w0.size(0) != h) value_error("the norm weight must have " + std::to_string(h) + " values");
  const Tensor w = w0.contiguous();
  const double eps = number(a[2], "eps"), off = number(a[5], "w_offset");
  const int normed = PyObject_IsTrue(a[6]);
  if (normed < 0) return nullptr;
  const c10::DeviceGuard guard(x.device());
  const Tensor *r0 = optional_tensor(a[3], "the residual"), *ro = optional_tensor(a[7], "residual_out");
  if (ro && !r0) value_error("residual_out needs a residual");
  Tensor r, out, y;
  int rdt = dt;
  if (r0) {
    same_gpu(*r0, x);
    if (r0->sizes() != x.sizes()) value_error("the residual must have x's shape");
    r = rows2(*r0, "the residual");
    rdt = dtype_code(r.scalar_type());
    if (!ro) {
      out = rows(m, h, r.scalar_type(), x);
    } else {
      same_gpu(*ro, x);
      if (ro->sizes() != x.sizes() || ro->scalar_type() != r.scalar_type() || (h > 1 && ro->stride(1) != 1))
        value_error("residual_out must have the residual's shape and type and unit column stride");
      out = *ro;
    }
  }
  if (normed) y = rows(m, h, x.scalar_type(), x);
  const Codes c = make_codes(m, h, a[4], x);
  const int M = to_int(m), H = to_int(h), wdt = dtype_code(w.scalar_type());
  void* st = stream_of(x);
  check(launch([&] {
          return fp4x_rms_norm_q8(x.data_ptr(), x.stride(0), dt, r0 ? r.data_ptr() : nullptr, r0 ? r.stride(0) : 0, rdt,
                                  w.data_ptr(), wdt, (float)off, eps, M, H, c.fmt, c.q.data_ptr(), c.q.stride(0),
                                  c.s.data_ptr(), r0 ? out.data_ptr() : nullptr, r0 ? out.stride(0) : 0,
                                  normed ? y.data_ptr() : nullptr, h, st);
        }),
        "rms_norm_q8");
  if (r0) return normed ? pack({c.q, c.s, out, y}) : pack({c.q, c.s, out});
  return normed ? pack({c.q, c.s, y}) : pack({c.q, c.s});
}

// silu_mul_q8(gate, up, fmt)
PyObject* silu_mul_q8(PyObject* const* a) {
  const Tensor& g0 = tensor(a[0], "gate");
  on_gpu(g0);
  const Tensor* u0 = optional_tensor(a[1], "up");
  if (u0) same_gpu(*u0, g0);
  const Tensor g = rows2(g0, "gate");
  const int dt = dtype_code(g.scalar_type());
  const int64_t m = g.size(0);
  int64_t f = g.size(1);
  const void* up;
  int64_t ldu = g.stride(0);
  Tensor u;
  if (!u0) {
    if (f & 1) value_error("gate and up side by side need an even number of columns");
    f >>= 1;
    up = static_cast<const char*>(g.data_ptr()) + f * (int64_t)g.element_size();
  } else {
    if (u0->sizes() != g.sizes() || u0->scalar_type() != g.scalar_type())
      value_error("up must have gate's shape and type");
    u = rows2(*u0, "up");
    up = u.data_ptr();
    ldu = u.stride(0);
  }
  const c10::DeviceGuard guard(g.device());
  const Codes c = make_codes(m, f, a[2], g);
  const int M = to_int(m), H = to_int(f);
  void* st = stream_of(g);
  check(launch([&] {
          return fp4x_silu_mul_q8(g.data_ptr(), g.stride(0), up, ldu, dt, M, H, c.fmt, c.q.data_ptr(), c.q.stride(0),
                                  c.s.data_ptr(), st);
        }),
        "silu_mul_q8");
  return pack({c.q, c.s});
}

// quantize_q8(x, fmt)
PyObject* quantize_q8(PyObject* const* a) {
  const Tensor& x0 = tensor(a[0], "x");
  on_gpu(x0);
  const Tensor x = rows2(x0, "x");
  const int64_t m = x.size(0), h = x.size(1);
  const int dt = dtype_code(x.scalar_type());
  const c10::DeviceGuard guard(x.device());
  const Codes c = make_codes(m, h, a[1], x);
  const int M = to_int(m), H = to_int(h);
  void* st = stream_of(x);
  check(launch([&] {
          return fp4x_quantize_q8(x.data_ptr(), x.stride(0), dt, M, H, c.fmt, c.q.data_ptr(), c.q.stride(0),
                                  c.s.data_ptr(), st);
        }),
        "quantize_q8");
  return pack({c.q, c.s});
}

// Code rows that start on 16 bytes, less than 2^24 apart, and can be read to
// the next 16-byte boundary past their end: q itself as the functions above lay
// it out, a copy otherwise.  The last two dimensions are rows and columns.
Tensor codes16(const Tensor& q, const char* what, at::ScalarType type = at::kChar, int64_t dims = 2) {
  if (q.scalar_type() != type)
    type_error(std::string(what) + " must be " + (type == at::kChar ? "int8" : "float8_e4m3fn") + ", got " + at::toString(q.scalar_type()));
  if (q.dim() != dims) value_error(std::string(what) + " must be " + std::to_string(dims) + "-D");
  const int64_t e = dims == 3 ? q.size(0) : 1, n = q.size(-2), k = q.size(-1), ld = q.stride(-2), up = (k + 15) & -16;
  const int64_t step = dims == 3 ? q.stride(0) : 0;
  if ((reinterpret_cast<uintptr_t>(q.data_ptr()) & 15) == 0 && (ld & 15) == 0 && (step & 15) == 0 &&
      (q.stride(-1) == 1 || k == 1) && k <= ld && ld < 1 << 24 &&
      (k == up || (uint64_t)(q.storage_offset() + (e - 1) * step + (n - 1) * ld + up) <= q.storage().nbytes()))
    return q;
  const int64_t to = type == at::kChar ? up : line_rows(k);
  const c10::Storage whole = make({e * n * to}, {1}, at::kByte, q).storage();    // whole rows, the last too
  const Tensor c = dims == 3 ? part(whole, 0, {e, n, k}, {n * to, to, 1}, type) : part(whole, 0, {n, k}, {to, 1}, type);
  c.copy_(q);
  return c;
}

Tensor scales(const Tensor& s, int64_t n, const char* what) {
  if (s.scalar_type() != at::kFloat || s.numel() != n)
    value_error(std::string(what) + " must be " + std::to_string(n) + " fp32 scales");
  return s.contiguous();
}

// w8a8_linear(xq, xs, wq, ws, bias, out_dtype)
PyObject* w8a8_linear(PyObject* const* a) {
  const Tensor &x0 = tensor(a[0], "xq"), &xs0 = tensor(a[1], "xs"), &w0 = tensor(a[2], "wq"), &ws0 = tensor(a[3], "ws");
  on_gpu(x0);
  same_gpu(xs0, x0);
  same_gpu(w0, x0);
  same_gpu(ws0, x0);
  if (!THPDtype_Check(a[5])) type_error("out_dtype must be a torch.dtype");
  const at::ScalarType ot = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
  const int odt = dtype_code(ot);
  const c10::DeviceGuard guard(x0.device());
  const Tensor x = codes16(x0, "xq"), w = codes16(w0, "wq");
  const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
  if (w.size(1) != k)
    value_error("activation K=" + std::to_string(k) + " does not match weight K=" + std::to_string(w.size(1)));
  const Tensor xs = scales(xs0, m, "xs"), ws = scales(ws0, n, "ws");
  Tensor b;
  if (const Tensor* b0 = optional_tensor(a[4], "the bias")) {
    same_gpu(*b0, x);
    if (b0->dim() != 1 || b0->size(0) != n) value_error("the bias must have " + std::to_string(n) + " values");
    b = b0->to(at::kFloat).contiguous();
  }
  const Tensor out = rows(m, n, ot, x);
  const int M = to_int(m), N = to_int(n), K = to_int(k);
  void* st = stream_of(x);
  check(launch([&] {
          return fp4x_w8a8_linear(x.data_ptr(), x.stride(0), static_cast<const float*>(xs.data_ptr()), w.data_ptr(),
                                  w.stride(0), static_cast<const float*>(ws.data_ptr()),
                                  b.defined() ? static_cast<const float*>(b.data_ptr()) : nullptr, out.data_ptr(), n,
                                  odt, M, N, K, st);
        }),
        "w8a8_linear");
  return THPVariable_Wrap(out);
}

// The scales of `m` activation rows of k values per 128: any strides.
const Tensor& scales128(const Tensor& s, int64_t m, int64_t k, const char* what) {
  const int64_t b = (k + 127) / 128;
  if (s.scalar_type() != at::kFloat || s.dim() != 2 || s.size(0) != m || s.size(1) != b)
    value_error(std::string(what) + " must be fp32 scales [" + std::to_string(m) + ", " + std::to_string(b) + "]");
  return s;
}
// Those of weights [.., n, k] per 128 x 128.
Tensor scales128x128(const Tensor& s, const Tensor& w, const char* what) {
  const int64_t nb = (w.size(-2) + 127) / 128, kb = (w.size(-1) + 127) / 128;
  if (s.scalar_type() != at::kFloat || s.dim() != w.dim() || s.size(-2) != nb || s.size(-1) != kb ||
      (w.dim() == 3 && s.size(0) != w.size(0)))
    value_error(std::string(what) + " must be fp32 scales [" + (w.dim() == 3 ? std::to_string(w.size(0)) + ", " : "") +
                std::to_string(nb) + ", " + std::to_string(kb) + "]");
  return s.contiguous();
}
Tensor ints(const Tensor& t, const Tensor& as, const char* what) {
  same_gpu(t, as);
  if (t.scalar_type() != at::kInt) type_error(std::string(what) + " must be int32, got " + at::toString(t.scalar_type()));
  return t.contiguous();
}
int64_t whole(PyObject* o, const char* what) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    type_error(std::string(what) + " must be a whole number");
  }
  return v;
}

// quantize_f8(w)
PyObject* quantize_f8(PyObject* const* a) {
  const Tensor& w0 = tensor(a[0], "w");
  on_gpu(w0);
  if (w0.dim() != 2 && w0.dim() != 3) value_error("w must be 2-D, or 3-D with the experts first");
  const int dt = dtype_code(w0.scalar_type());
  const c10::DeviceGuard guard(w0.device());
  const Tensor w = w0.stride(-1) == 1 || w0.size(-1) == 1 ? w0 : w0.contiguous();
  const bool ex = w.dim() == 3;
  const int64_t e = ex ? w.size(0) : 1, n = w.size(-2), k = w.size(-1), ld = line_rows(k);
  const int64_t nb = (n + 127) / 128, kb = (k + 127) / 128;
  const c10::Storage codes = make({e * n * ld}, {1}, at::kByte, w).storage();    // whole rows, the last too
  const Tensor q = ex ? part(codes, 0, {e, n, k}, {n * ld, ld, 1}, at::kFloat8_e4m3fn)
                      : part(codes, 0, {n, k}, {ld, 1}, at::kFloat8_e4m3fn);
  const Tensor s = ex ? make({e, nb, kb}, {nb * kb, kb, 1}, at::kFloat, w) : rows(nb, kb, at::kFloat, w);
  const int E = to_int(e), N = to_int(n), K = to_int(k);
  void* st = stream_of(w);
  check(launch([&] {
          return fp4x_quantize_f8(w.data_ptr(), w.stride(-2), ex ? w.stride(0) : 0, dt, E, N, K, q.data_ptr(), ld, n * ld,
                                  static_cast<float*>(s.data_ptr()), st);
        }),
        "quantize_f8");
  return pack({q, s});
}

// f8_linear(xq, xs, wq, ws, bias, out_dtype)
PyObject* f8_linear(PyObject* const* a) {
  const Tensor &x0 = tensor(a[0], "xq"), &xs0 = tensor(a[1], "xs"), &w0 = tensor(a[2], "wq"), &ws0 = tensor(a[3], "ws");
  on_gpu(x0);
  same_gpu(xs0, x0);
  same_gpu(w0, x0);
  same_gpu(ws0, x0);
  if (!THPDtype_Check(a[5])) type_error("out_dtype must be a torch.dtype");
  const at::ScalarType ot = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
  const int odt = dtype_code(ot);
  const c10::DeviceGuard guard(x0.device());
  const Tensor x = codes16(x0, "xq", at::kFloat8_e4m3fn), w = codes16(w0, "wq", at::kFloat8_e4m3fn);
  const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
  if (w.size(1) != k)
    value_error("activation K=" + std::to_string(k) + " does not match weight K=" + std::to_string(w.size(1)));
  const Tensor xs = scales128(xs0, m, k, "xs"), ws = scales128x128(ws0, w, "ws");
  Tensor b;
  if (const Tensor* b0 = optional_tensor(a[4], "the bias")) {
    same_gpu(*b0, x);
    if (b0->dim() != 1 || b0->size(0) != n) value_error("the bias must have " + std::to_string(n) + " values");
    b = b0->to(at::kFloat).contiguous();
  }
  const Tensor out = rows(m, n, ot, x);
  const int M = to_int(m), N = to_int(n), K = to_int(k);
  void* st = stream_of(x);
  check(launch([&] {
          return fp4x_f8_linear(x.data_ptr(), x.stride(0), static_cast<const float*>(xs.data_ptr()), xs.stride(0),
                                xs.stride(1), w.data_ptr(), w.stride(0), static_cast<const float*>(ws.data_ptr()),
                                b.defined() ? static_cast<const float*>(b.data_ptr()) : nullptr, out.data_ptr(), n, odt,
                                M, N, K, st);
        }),
        "f8_linear");
  return THPVariable_Wrap(out);
}

// f8_linear_experts(xq, xs, wq, ws, offsets, tokens, out_dtype)
PyObject* f8_linear_experts(PyObject* const* a) {
  const Tensor &x0 = tensor(a[0], "xq"), &xs0 = tensor(a[1], "xs"), &w0 = tensor(a[2], "wq"), &ws0 = tensor(a[3], "ws");
  const Tensor& o0 = tensor(a[4], "offsets");
  const Tensor* t0 = optional_tensor(a[5], "tokens");
  on_gpu(x0);
  same_gpu(xs0, x0);
  same_gpu(w0, x0);
  same_gpu(ws0, x0);
  if (!THPDtype_Check(a[6])) type_error("out_dtype must be a torch.dtype");
  const at::ScalarType ot = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
  const int odt = dtype_code(ot);
  const c10::DeviceGuard guard(x0.device());
  const Tensor x = codes16(x0, "xq", at::kFloat8_e4m3fn), w = codes16(w0, "wq", at::kFloat8_e4m3fn, 3);
  const int64_t m = x.size(0), k = x.size(1), e = w.size(0), n = w.size(1);
  if (w.size(2) != k)
    value_error("activation K=" + std::to_string(k) + " does not match weight K=" + std::to_string(w.size(2)));
  const Tensor xs = scales128(xs0, m, k, "xs"), ws = scales128x128(ws0, w, "ws");
  const Tensor off = ints(o0, x, "offsets");
  if (off.dim() != 1 || off.size(0) != e + 1) value_error("offsets must have " + std::to_string(e + 1) + " values");
  Tensor tok;
  if (t0) {
    tok = ints(*t0, x, "tokens");
    if (tok.dim() != 1) value_error("tokens must be 1-D");
  }
  const int64_t p = t0 ? tok.size(0) : m;
  const Tensor out = rows(p, n, ot, x);
  const int X = to_int(m), E = to_int(e), P = to_int(p), N = to_int(n), K = to_int(k);
  void* st = stream_of(x);
  check(launch([&] {
          return fp4x_f8_linear_experts(x.data_ptr(), x.stride(0), static_cast<const float*>(xs.data_ptr()), xs.stride(0),
                                        xs.stride(1), X, t0 ? static_cast<const int*>(tok.data_ptr()) : nullptr,
                                        static_cast<const int*>(off.data_ptr()), E, w.data_ptr(), w.stride(1), w.stride(0),
                                        static_cast<const float*>(ws.data_ptr()), out.data_ptr(), n, odt, P, N, K, st);
        }),
        "f8_linear_experts");
  return THPVariable_Wrap(out);
}

// expert_sort(ids, experts)
PyObject* expert_sort(PyObject* const* a) {
  const Tensor& i0 = tensor(a[0], "ids");
  const int64_t e = whole(a[1], "experts");
  on_gpu(i0);
  if (i0.dim() != 2) value_error("ids must be 2-D");
  const bool wide = i0.scalar_type() == at::kLong;
  if (!wide && i0.scalar_type() != at::kInt) type_error(std::string("ids must be int64 or int32, got ") + at::toString(i0.scalar_type()));
  if (e < 1 || e > 4096) value_error("1 to 4096 experts, got " + std::to_string(e));
  const int64_t t = i0.size(0), k = i0.size(1);
  if (k < 1) value_error("a token needs at least one id");
  if (t > (1 << 30) / k) value_error("more than 2^30 ids");
  const c10::DeviceGuard guard(i0.device());
  const Tensor ids = i0.stride(1) == 1 || k == 1 ? i0 : i0.contiguous();
  const int64_t p = t * k, off = (e + 4) / 4 * 16, need = fp4x_expert_sort_workspace(t, (int)k, (int)e);
  Tensor offsets, tokens, slots, ws;
  if (off + 8 * p <= kShared) {                    // one allocation, as the codes and scales above
    const c10::Storage all = make({off + 8 * p}, {1}, at::kByte, ids).storage();
    offsets = part(all, 0, {e + 1}, {1}, at::kInt);
    tokens = part(all, off, {p}, {1}, at::kInt);
    slots = part(all, off + 4 * p, {t, k}, {k, 1}, at::kInt);
  } else {
    offsets = make({e + 1}, {1}, at::kInt, ids);
    tokens = make({p}, {1}, at::kInt, ids);
    slots = rows(t, k, at::kInt, ids);
  }
  if (need) ws = make({need}, {1}, at::kByte, ids);
  void* st = stream_of(ids);
  check(launch([&] {
          return fp4x_expert_sort(ids.data_ptr(), wide, ids.stride(0), t, (int)k, (int)e,
                                  static_cast<int*>(offsets.data_ptr()), static_cast<int*>(tokens.data_ptr()),
                                  static_cast<int*>(slots.data_ptr()), need ? ws.data_ptr() : nullptr, need, st);
        }),
        "expert_sort");
  return pack({offsets, tokens, slots});
}

// expert_rows(x, tokens)
PyObject* expert_rows(PyObject* const* a) {
  const Tensor &x0 = tensor(a[0], "x"), &t0 = tensor(a[1], "tokens");
  on_gpu(x0);
  const c10::DeviceGuard guard(x0.device());
  const Tensor x = rows2(x0, "x"), tok = ints(t0, x, "tokens");
  if (tok.dim() != 1) value_error("tokens must be 1-D");
  const int64_t size = (int64_t)x.element_size(), t = x.size(0), h = x.size(1), p = tok.size(0);
  if (size != 1 && size != 2 && size != 4) type_error(std::string("elements of 1, 2 or 4 bytes, got ") + at::toString(x.scalar_type()));
  const Tensor out = rows(p, h, x.scalar_type(), x);
  const int T = to_int(t), P = to_int(p), H = to_int(h);
  void* st = stream_of(x);
  check(launch([&] {
          return fp4x_expert_rows(x.data_ptr(), x.stride(0), (int)size, T, static_cast<const int*>(tok.data_ptr()), P, H,
                                  out.data_ptr(), h, st);
        }),
        "expert_rows");
  return THPVariable_Wrap(out);
}

// The weights of slots [t, k], of a float type of their own.
Tensor weights_of(const Tensor& w, const Tensor& slots) {
  same_gpu(w, slots);
  if (w.sizes() != slots.sizes()) value_error("the weights must have the slots' shape");
  return w.contiguous();
}

// expert_combine(y, slots, weights)
PyObject* expert_combine(PyObject* const* a) {
  const Tensor &y0 = tensor(a[0], "y"), &s0 = tensor(a[1], "slots");
  const Tensor* w0 = optional_tensor(a[2], "the weights");
  on_gpu(y0);
  const c10::DeviceGuard guard(y0.device());
  const Tensor y = rows2(y0, "y"), slots = ints(s0, y, "slots");
  if (slots.dim() != 2 || slots.size(1) < 1) value_error("slots must be 2-D, at least one per token");
  const int dt = dtype_code(y.scalar_type());
  const int64_t p = y.size(0), h = y.size(1), t = slots.size(0), k = slots.size(1);
  Tensor w;
  int wdt = dt;
  if (w0) {
    w = weights_of(*w0, slots);
    wdt = dtype_code(w.scalar_type());
  }
  const Tensor out = rows(t, h, y.scalar_type(), y);
  const int P = to_int(p), H = to_int(h), T = to_int(t), k_ = to_int(k);
  void* st = stream_of(y);
  check(launch([&] {
          return fp4x_expert_combine(y.data_ptr(), y.stride(0), dt, P, static_cast<const int*>(slots.data_ptr()),
                                     w0 ? w.data_ptr() : nullptr, wdt, out.data_ptr(), h, T, k_, H, st);
        }),
        "expert_combine");
  return THPVariable_Wrap(out);
}

// expert_combine_grad(dout, y, slots, weights, tokens)
PyObject* expert_combine_grad(PyObject* const* a) {
  const Tensor &d0 = tensor(a[0], "dout"), &y0 = tensor(a[1], "y"), &s0 = tensor(a[2], "slots");
  const Tensor &w0 = tensor(a[3], "the weights"), &t0 = tensor(a[4], "tokens");
  on_gpu(y0);
  same_gpu(d0, y0);
  const c10::DeviceGuard guard(y0.device());
  const Tensor y = rows2(y0, "y"), d = rows2(d0, "dout"), slots = ints(s0, y, "slots"), tok = ints(t0, y, "tokens");
  if (slots.dim() != 2 || slots.size(1) < 1) value_error("slots must be 2-D, at least one per token");
  const Tensor w = weights_of(w0, slots);
  const int dt = dtype_code(y.scalar_type()), wdt = dtype_code(w.scalar_type());
  const int64_t p = y.size(0), h = y.size(1), t = slots.size(0), k = slots.size(1);
  if (d.size(0) != t || d.size(1) != h || d.scalar_type() != y.scalar_type())
    value_error("dout must have a row per token, of y's length and type");
  if (tok.dim() != 1 || tok.size(0) != p) value_error("tokens must have a value per row of y");
  const Tensor dy = rows(p, h, y.scalar_type(), y), dw = rows(t, k, w.scalar_type(), y);
  const int P = to_int(p), H = to_int(h), T = to_int(t), k_ = to_int(k);
  void* st = stream_of(y);
  check(launch([&] {
          return fp4x_expert_combine_grad(d.data_ptr(), d.stride(0), y.data_ptr(), y.stride(0), dt, P,
                                          static_cast<const int*>(slots.data_ptr()), static_cast<const int*>(tok.data_ptr()),
                                          w.data_ptr(), wdt, dy.data_ptr(), h, dw.data_ptr(), T, k_, H, st);
        }),
        "expert_combine_grad");
  return pack({dy, dw});
}

template <PyObject* (*F)(PyObject* const*), int ARGS>
PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != ARGS) {
    PyErr_Format(PyExc_TypeError, "fp4x: %d arguments expected, got %zd", ARGS, n);
    return nullptr;
  }
  try {
    return F(a);
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.why.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject* const*), int ARGS>
constexpr PyMethodDef method(const char* name) {
  return {name, (PyCFunction)(void (*)())entry<F, ARGS>, METH_FASTCALL, nullptr};
}
PyMethodDef kMethods[] = {method<rms_norm_q8, 8>("rms_norm_q8"), method<silu_mul_q8, 3>("silu_mul_q8"),
                          method<quantize_q8, 2>("quantize_q8"), method<w8a8_linear, 6>("w8a8_linear"),
                          method<quantize_f8, 1>("quantize_f8"), method<f8_linear, 6>("f8_linear"),
                          method<f8_linear_experts, 7>("f8_linear_experts"), method<expert_sort, 2>("expert_sort"),
                          method<expert_rows, 2>("expert_rows"), method<expert_combine, 3>("expert_combine"),
                          method<expert_combine_grad, 5>("expert_combine_grad"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fp4x_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fp4x_host() {
  PyObject* m = PyModule_Create(&kModule);
  if (m && PyModule_AddIntConstant(m, "ABI_VERSION", FP4X_ABI_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
