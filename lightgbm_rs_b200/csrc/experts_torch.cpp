// Python module lightgbm_rs_b200._experts: the expert-layer entry points on torch tensors.
// It checks tensors, makes results and scratch with torch's allocator, and calls the C ABI on
// torch's current stream. A call through ctypes and torch's Python functions took 9 to 19 us
// of host time for kernels of 2 to 4 us; a served row pays that at every layer.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <sstream>
#include <string>

#include "lgbm_b200.h"

namespace {

using at::Tensor;

PyObject* g_error_type = nullptr;  // lightgbm_rs_b200._lib.LightGBMError

// Raised as LightGBMError(code, message).
struct Refused {
  int code;
  std::string msg;
};

template <typename... Parts>
[[noreturn]] void refuse(int code, const Parts&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw Refused{code, s.str()};
}

void check(int rc) {
  if (rc != LGBM_B200_OK) throw Refused{rc, lgbm_b200_last_error()};
}

std::string describe(const Tensor& t) {
  std::ostringstream s;
  s << t.sizes() << " " << t.scalar_type() << " on " << t.device();
  return s.str();
}

int dtype_of(const char* what, const Tensor& t, bool halves) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return LGBM_B200_DTYPE_BF16;
    case at::kHalf: return LGBM_B200_DTYPE_F16;
    case at::kFloat:
      if (!halves) return LGBM_B200_DTYPE_F32;
      break;
    default: break;
  }
  refuse(LGBM_B200_INVALID_ARGUMENT, what, ": want a tensor of ",
         halves ? "bfloat16 or float16" : "float32, bfloat16 or float16", ", got ", describe(t));
}

Tensor tensor(const char* what, PyObject* o) {
  if (!THPVariable_Check(o)) refuse(LGBM_B200_INVALID_ARGUMENT, what, ": want a torch tensor");
  Tensor t = THPVariable_Unpack(o);
  // nothing is recorded for autograd: a result would lose the gradient without a word
  if (t.requires_grad() && at::GradMode::is_enabled())
    refuse(LGBM_B200_INVALID_ARGUMENT, what, ": an input requires a gradient, which autograd does "
           "not get through here; call under torch.no_grad() and use the _backward functions");
  return t;
}

// A [rows, width] matrix with a contiguous last axis.
struct Matrix {
  Tensor t;
  int dtype;
  int64_t rows, width, pitch;
  const void* p() const { return t.data_ptr(); }
};

// `reads`: its values are wanted, else only its shape.
Matrix matrix(const char* what, Tensor t, bool halves, bool reads = true) {
  Matrix m;
  m.dtype = dtype_of(what, t, halves);
  if (t.dim() != 2 || !t.is_cuda())
    refuse(LGBM_B200_INVALID_ARGUMENT, what, ": want a 2-D CUDA tensor, got ", describe(t));
  m.rows = t.size(0);
  m.width = t.size(1);
  m.pitch = m.rows > 1 ? t.stride(0) : m.width;
  if ((m.width > 1 && t.stride(1) != 1) || m.pitch < m.width) {
    if (reads) t = t.contiguous();
    m.pitch = m.width;
  }
  m.t = std::move(t);
  return m;
}

// A contiguous tensor of exactly this type, shape and device.
Tensor same(const char* what, Tensor t, c10::Device dev, at::ScalarType type, at::IntArrayRef shape) {
  if (t.scalar_type() != type || t.device() != dev || t.sizes() != shape)
    refuse(LGBM_B200_INVALID_ARGUMENT, what, ": want ", shape, " ", type, " on ", dev, ", got ",
           describe(t));
  return t.is_contiguous() ? t : t.contiguous();
}

Tensor make(c10::Device dev, at::ScalarType type, at::IntArrayRef shape) {
  return at::detail::empty_cuda(shape, type, dev, std::nullopt);
}

// Contiguous tensors cut out of one block of memory, which lives as long as any of them: small
// results of one call cost one allocation. Offsets and sizes in bytes are multiples of 16.
class Block {
 public:
  Block(c10::Device dev, int64_t bytes) : base_(make(dev, at::kByte, {bytes})) {}
  static int64_t bytes(int64_t elements) { return (elements * 4 + 15) / 16 * 16; }
  Tensor cut(at::ScalarType type, at::IntArrayRef shape) {  // 4-byte elements
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(
        c10::Storage(base_.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA),
        c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(at_ / 4);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
    at_ += bytes(t.numel());
    return t;
  }

 private:
  Tensor base_;
  int64_t at_ = 0;
};

// The device made current, and its current stream.
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(c10::Device dev)
      : guard(dev), stream(c10::cuda::getCurrentCUDAStream(dev.index()).stream()) {}
};

// Scratch of a call; freed to torch's allocator, which hands it out again behind the call on
// the same stream.
struct Scratch {
  Tensor t;
  int64_t bytes;
  Scratch(c10::Device dev, int64_t n) : bytes(n) {
    if (n > 0) t = make(dev, at::kByte, {n});
  }
  void* p() const { return bytes > 0 ? t.data_ptr() : nullptr; }
};

int64_t whole(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
uint64_t counter(const char* what, PyObject* o) {
  const unsigned long long v = PyLong_AsUnsignedLongLong(o);
  if (v == (unsigned long long)-1 && PyErr_Occurred()) {
    if (!PyErr_ExceptionMatches(PyExc_OverflowError)) throw python_error();
    PyErr_Clear();
    refuse(LGBM_B200_INVALID_ARGUMENT, what, ": seed and offset are 64-bit counters");
  }
  return v;
}
bool flag(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}

PyObject* wrap(Tensor t) { return THPVariable_Wrap(std::move(t)); }
template <typename... T>
PyObject* wrap_all(T... t) {
  PyObject* out = PyTuple_New(sizeof...(T));
  if (!out) throw python_error();
  Py_ssize_t i = 0;
  auto put = [&](Tensor v) {
    PyObject* o = Py_None;
    if (v.defined()) o = wrap(std::move(v));
    else Py_INCREF(o);
    PyTuple_SET_ITEM(out, i++, o);
  };
  (put(std::move(t)), ...);
  return out;
}

// route(logits, k, normalize) -> (weights, experts, position, rows, offsets)
PyObject* route(PyObject* const* a) {
  const char* what = "route";
  const Matrix l = matrix(what, tensor(what, a[0]), false);
  const int64_t k = whole(a[1]);
  const bool normalize = flag(a[2]);
  if (k < 1 || k > l.width)
    refuse(LGBM_B200_INVALID_ARGUMENT, what, ": k ", k, " of ", l.width, " experts");
  if (l.width > INT32_MAX) refuse(LGBM_B200_CAPABILITY_UNAVAILABLE, what, ": too many experts");
  const auto dev = l.t.device();
  On on(dev);
  const int64_t slots = l.rows * k;
  Block block(dev, 4 * Block::bytes(slots) + Block::bytes(l.width + 1));
  Tensor weights = block.cut(at::kFloat, {l.rows, k}), chosen = block.cut(at::kInt, {l.rows, k}),
         position = block.cut(at::kInt, {l.rows, k}), rows = block.cut(at::kInt, {slots}),
         offsets = block.cut(at::kInt, {l.width + 1});
  Scratch ws(dev, lgbm_b200_experts_route_workspace(l.rows, (int32_t)l.width, (int32_t)k));
  check(lgbm_b200_experts_route(l.p(), l.dtype, l.rows, (int32_t)l.width, l.pitch, (int32_t)k,
                                normalize, weights.data_ptr<float>(), chosen.data_ptr<int32_t>(),
                                position.data_ptr<int32_t>(), rows.data_ptr<int32_t>(),
                                offsets.data_ptr<int32_t>(), ws.p(), ws.bytes, on.stream));
  return wrap_all(weights, chosen, position, rows, offsets);
}

// route_backward(dweights, logits, weights, experts, normalize) -> dlogits
PyObject* route_backward(PyObject* const* a) {
  const char* what = "route_backward";
  const Matrix l = matrix(what, tensor(what, a[1]), false);
  const auto dev = l.t.device();
  Tensor weights = tensor(what, a[2]);
  if (weights.dim() != 2)
    refuse(LGBM_B200_INVALID_ARGUMENT, what, ": weights ", describe(weights));
  const int64_t k = weights.size(1);
  const int64_t shape[2] = {l.rows, k};
  weights = same("route_backward: weights", weights, dev, at::kFloat, shape);
  const Tensor dweights =
      same("route_backward: dweights", tensor(what, a[0]), dev, at::kFloat, shape);
  const Tensor chosen =
      same("route_backward: experts", tensor(what, a[3]), dev, at::kInt, shape);
  On on(dev);
  Tensor out = make(dev, l.t.scalar_type(), {l.rows, l.width});
  check(lgbm_b200_experts_route_backward(
      dweights.data_ptr<float>(), weights.data_ptr<float>(), chosen.data_ptr<int32_t>(), l.p(),
      l.dtype, l.rows, (int32_t)l.width, l.pitch, (int32_t)k, flag(a[4]), out.data_ptr(),
      on.stream));
  return wrap(out);
}

// What the products share: x, w [E, outer, inner], offsets, rows (None: x's own).
struct Product {
  Matrix x;
  Tensor w, offsets, index;
  int64_t experts, outer, inner, rows;
  const int32_t* ip() const { return index.defined() ? index.data_ptr<int32_t>() : nullptr; }
};

void index_rows(const char* what, Product& p, PyObject* rows) {
  p.rows = p.x.rows;
  if (rows == Py_None) return;
  Tensor t = tensor(what, rows);
  if (t.dim() != 1) refuse(LGBM_B200_INVALID_ARGUMENT, what, ": rows ", describe(t));
  p.index = same("rows", t, p.x.t.device(), at::kInt, t.sizes());
  p.rows = t.size(0);
}

Product product(const char* what, PyObject* x, PyObject* w, PyObject* offsets, PyObject* rows,
                bool reads_x, bool reads_w) {
  Product p;
  p.x = matrix(what, tensor(what, x), true, reads_x);
  const auto dev = p.x.t.device();
  p.w = tensor(what, w);
  if (p.w.dim() != 3 || p.w.scalar_type() != p.x.t.scalar_type() || p.w.device() != dev)
    refuse(LGBM_B200_INVALID_ARGUMENT, what, ": want w [experts, outer, inner] like x, got ",
           describe(p.w), " with x ", describe(p.x.t));
  if (reads_w && !p.w.is_contiguous()) p.w = p.w.contiguous();
  p.experts = p.w.size(0);
  p.outer = p.w.size(1);
  p.inner = p.w.size(2);
  if (p.x.width != p.inner)
    refuse(LGBM_B200_LENGTH_MISMATCH, what, ": x is ", p.x.width, " wide, w takes ", p.inner);
  p.offsets = same("offsets", tensor(what, offsets), dev, at::kInt, {p.experts + 1});
  index_rows(what, p, rows);
  if (p.experts > INT32_MAX || p.outer > INT32_MAX || p.inner > INT32_MAX)
    refuse(LGBM_B200_CAPABILITY_UNAVAILABLE, what, ": w ", describe(p.w));
  return p;
}

// grouped_matmul(x, w, offsets, rows) -> y
PyObject* grouped_matmul(PyObject* const* a) {
  const char* what = "grouped_matmul";
  const Product p = product(what, a[0], a[1], a[2], a[3], true, true);
  const auto dev = p.x.t.device();
  On on(dev);
  Tensor y = make(dev, p.x.t.scalar_type(), {p.rows, p.outer});
  Scratch ws(dev, lgbm_b200_experts_matmul_workspace(
                      p.x.p(), p.x.pitch, p.ip(), p.w.data_ptr(), p.rows, (int32_t)p.experts,
                      (int32_t)p.inner, (int32_t)p.outer));
  check(lgbm_b200_experts_matmul(p.x.p(), p.x.rows, p.x.pitch, p.ip(), p.w.data_ptr(),
                                 p.offsets.data_ptr<int32_t>(), p.x.dtype, p.rows,
                                 (int32_t)p.experts, (int32_t)p.inner, (int32_t)p.outer,
                                 y.data_ptr(), ws.p(), ws.bytes, on.stream));
  return wrap(y);
}

// grouped_matmul_backward(dy, x, w, offsets, rows, wide_dw, need_dx, need_dw) -> (dx, dw)
PyObject* grouped_matmul_backward(PyObject* const* a) {
  const char* what = "grouped_matmul_backward";
  const bool need_dx = flag(a[6]), need_dw = flag(a[7]);
  const Product p = product(what, a[1], a[2], a[3], a[4], need_dw, need_dx);
  const Matrix dy = matrix(what, tensor(what, a[0]), true);
  const auto dev = p.x.t.device();
  const auto type = p.x.t.scalar_type();
  if (dy.dtype != p.x.dtype || dy.t.device() != dev)
    refuse(LGBM_B200_INVALID_ARGUMENT, what, ": dy ", describe(dy.t), ", x ", describe(p.x.t));
  if (dy.rows != p.rows || dy.width != p.outer)
    refuse(LGBM_B200_LENGTH_MISMATCH, what, ": dy ", describe(dy.t), ", want [", p.rows, ", ",
           p.outer, "]");
  const bool wide = flag(a[5]);
  const int32_t experts = (int32_t)p.experts, inner = (int32_t)p.inner, outer = (int32_t)p.outer;
  On on(dev);
  Tensor dx, dw;
  if (need_dx) dx = make(dev, type, {p.rows, p.inner});
  if (need_dw) dw = make(dev, wide ? at::kFloat : type, {p.experts, p.outer, p.inner});
  if (dx.defined() || dw.defined()) {
    Scratch ws(dev, lgbm_b200_experts_matmul_backward_workspace(
                        dy.p(), dy.pitch, p.x.p(), p.x.pitch, p.ip(), p.w.data_ptr(), p.rows,
                        experts, inner, outer, dx.defined(), dw.defined()));
    check(lgbm_b200_experts_matmul_backward(
        dy.p(), dy.pitch, p.x.p(), p.x.rows, p.x.pitch, p.ip(), p.w.data_ptr(),
        p.offsets.data_ptr<int32_t>(), p.x.dtype, wide ? LGBM_B200_DTYPE_F32 : p.x.dtype, p.rows,
        experts, inner, outer, dx.defined() ? dx.data_ptr() : nullptr,
        dw.defined() ? dw.data_ptr() : nullptr, ws.p(), ws.bytes, on.stream));
  }
  return wrap_all(dx, dw);
}

// grouped_matmul_w4(x, q, scales, offsets, zeros, rows, group_size) -> y
PyObject* grouped_matmul_w4(PyObject* const* a) {
  const char* what = "grouped_matmul_w4";
  Product p;
  p.x = matrix(what, tensor(what, a[0]), true);
  const auto dev = p.x.t.device();
  Tensor q = tensor(what, a[1]);
  const int64_t size = whole(a[6]);
  if (q.dim() != 3 || (size != 32 && size != 64 && size != 128))
    refuse(LGBM_B200_INVALID_ARGUMENT, what, ": q ", describe(q), ", groups of ", size);
  p.inner = p.x.width;
  p.experts = q.size(0);
  p.outer = q.size(1);
  if (p.experts > INT32_MAX || p.outer > INT32_MAX || p.inner > INT32_MAX)
    refuse(LGBM_B200_CAPABILITY_UNAVAILABLE, what, ": q ", describe(q));
  q = same("grouped_matmul_w4: q", q, dev, at::kByte,
           {p.experts, p.outer, (p.inner + 31) / 32 * 16});
  const int64_t shape[3] = {p.experts, p.outer, (p.inner + size - 1) / size};
  const Tensor scales = same("grouped_matmul_w4: scales", tensor(what, a[2]), dev,
                             p.x.t.scalar_type(), shape);
  Tensor zeros;
  if (a[4] != Py_None)
    zeros = same("grouped_matmul_w4: zeros", tensor(what, a[4]), dev, at::kByte, shape);
  const Tensor offsets =
      same("grouped_matmul_w4: offsets", tensor(what, a[3]), dev, at::kInt, {p.experts + 1});
  index_rows(what, p, a[5]);
  On on(dev);
  Tensor y = make(dev, p.x.t.scalar_type(), {p.rows, p.outer});
  check(lgbm_b200_experts_matmul_w4(
      p.x.p(), p.x.rows, p.x.pitch, p.ip(), q.data_ptr<uint8_t>(), scales.data_ptr(),
      zeros.defined() ? zeros.data_ptr<uint8_t>() : nullptr, (int32_t)size,
      offsets.data_ptr<int32_t>(), p.x.dtype, p.rows, (int32_t)p.experts, (int32_t)p.inner,
      (int32_t)p.outer, y.data_ptr(), on.stream));
  return wrap(y);
}

// position [T, k] and weights [T, k] or None
struct Slots {
  Tensor position, weights;
  int64_t tokens, k;
  const float* wp() const { return weights.defined() ? weights.data_ptr<float>() : nullptr; }
};

Slots slots(const char* what, c10::Device dev, PyObject* position, PyObject* weights) {
  Slots s;
  s.position = tensor(what, position);
  if (s.position.dim() != 2)
    refuse(LGBM_B200_INVALID_ARGUMENT, what, ": position ", describe(s.position));
  s.position = same("position", s.position, dev, at::kInt, s.position.sizes());
  s.tokens = s.position.size(0);
  s.k = s.position.size(1);
  if (s.k > INT32_MAX) refuse(LGBM_B200_CAPABILITY_UNAVAILABLE, what, ": k ", s.k);
  if (weights != Py_None)
    s.weights = same("weights", tensor(what, weights), dev, at::kFloat, s.position.sizes());
  return s;
}

// combine(y, position, weights) -> out
PyObject* combine(PyObject* const* a) {
  const char* what = "combine";
  const Matrix y = matrix(what, tensor(what, a[0]), false);
  const auto dev = y.t.device();
  const Slots s = slots(what, dev, a[1], a[2]);
  if (y.width > INT32_MAX) refuse(LGBM_B200_CAPABILITY_UNAVAILABLE, what, ": y ", describe(y.t));
  On on(dev);
  Tensor out = make(dev, y.t.scalar_type(), {s.tokens, y.width});
  check(lgbm_b200_experts_combine(y.p(), y.dtype, y.rows, (int32_t)y.width, y.pitch,
                                  s.position.data_ptr<int32_t>(), s.wp(), s.tokens, (int32_t)s.k,
                                  out.data_ptr(), on.stream));
  return wrap(out);
}

// combine_backward(dout, y, position, weights) -> (dy, dweights)
PyObject* combine_backward(PyObject* const* a) {
  const char* what = "combine_backward";
  const Matrix y = matrix(what, tensor(what, a[1]), false);
  const Matrix dout = matrix(what, tensor(what, a[0]), false);
  const auto dev = y.t.device();
  const Slots s = slots(what, dev, a[2], a[3]);
  if (dout.dtype != y.dtype || dout.t.device() != dev)
    refuse(LGBM_B200_INVALID_ARGUMENT, what, ": dout ", describe(dout.t), ", y ", describe(y.t));
  if (dout.rows != s.tokens || dout.width != y.width)
    refuse(LGBM_B200_LENGTH_MISMATCH, what, ": dout ", describe(dout.t), ", y ", describe(y.t),
           ", ", s.tokens, " tokens");
  if (y.width > INT32_MAX) refuse(LGBM_B200_CAPABILITY_UNAVAILABLE, what, ": y ", describe(y.t));
  On on(dev);
  Tensor dy = make(dev, y.t.scalar_type(), {y.rows, y.width}), dw;
  if (s.weights.defined()) dw = make(dev, at::kFloat, {s.tokens, s.k});
  check(lgbm_b200_experts_combine_backward(
      dout.p(), y.p(), y.dtype, y.rows, (int32_t)y.width, dout.pitch, y.pitch,
      s.position.data_ptr<int32_t>(), s.wp(), s.tokens, (int32_t)s.k, dy.data_ptr(),
      dw.defined() ? dw.data_ptr<float>() : nullptr, on.stream));
  return wrap_all(dy, dw);
}

// An array of any shape as rows of one pitch: contiguous (one row) or a 2-D row pitch.
struct Walk {
  Tensor t;
  bool flat;
  int64_t rows, width, pitch;
};
Walk walk(const Tensor& t) {
  if (t.dim() == 2 && !t.is_contiguous() && t.stride(1) == 1 && t.stride(0) >= t.size(1))
    return {t, false, t.size(0), t.size(1), t.stride(0)};
  return {t.is_contiguous() ? t : t.contiguous(), true, 1, t.numel(), t.numel()};
}

// dropout(x, p, seed, offset, residual) -> out
PyObject* dropout(PyObject* const* a) {
  const char* what = "dropout";
  const Tensor x = tensor(what, a[0]);
  const int dtype = dtype_of(what, x, false);
  if (!x.is_cuda()) refuse(LGBM_B200_INVALID_ARGUMENT, what, ": want a CUDA tensor");
  const double p = PyFloat_AsDouble(a[1]);
  if (p == -1.0 && PyErr_Occurred()) throw python_error();
  const uint64_t seed = counter(what, a[2]), offset = counter(what, a[3]);
  Walk w = walk(x), r{};
  if (a[4] != Py_None) {
    const Tensor res = tensor(what, a[4]);
    if (res.sizes() != x.sizes() || res.scalar_type() != x.scalar_type() ||
        res.device() != x.device())
      refuse(LGBM_B200_LENGTH_MISMATCH, what, ": residual ", describe(res), ", x ", describe(x));
    r = walk(res);
    if (w.flat != r.flat) {  // one of them has a row pitch: both as rows
      Walk& f = w.flat ? w : r;
      f.rows = x.size(0);
      f.width = f.pitch = x.size(1);
    }
  }
  On on(x.device());
  Tensor out = make(x.device(), x.scalar_type(), x.sizes());
  check(lgbm_b200_experts_dropout(w.t.data_ptr(), r.t.defined() ? r.t.data_ptr() : nullptr, dtype,
                                  w.rows, w.width, w.pitch, r.pitch, p, seed, offset,
                                  out.data_ptr(), on.stream));
  return wrap(out);
}

// errors() -> bits
PyObject* errors(PyObject* const*) {
  uint32_t bits = 0;
  int rc;
  Py_BEGIN_ALLOW_THREADS  // it waits for the device
  rc = lgbm_b200_experts_errors(&bits);
  Py_END_ALLOW_THREADS
  check(rc);
  return PyLong_FromUnsignedLong(bits);
}

// One Python entry point: the argument count, the GIL (kept: nothing here waits but errors, which
// releases it), and C++ exceptions as Python ones.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused& r) {
    PyObject* value = PyObject_CallFunction(g_error_type, "is", r.code, r.msg.c_str());
    if (value) {
      PyErr_SetObject(g_error_type, value);
      Py_DECREF(value);
    }
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyMethodDef g_methods[] = {
    {"route", (PyCFunction)(void (*)())entry<route, 3>, METH_FASTCALL, nullptr},
    {"route_backward", (PyCFunction)(void (*)())entry<route_backward, 5>, METH_FASTCALL, nullptr},
    {"grouped_matmul", (PyCFunction)(void (*)())entry<grouped_matmul, 4>, METH_FASTCALL, nullptr},
    {"grouped_matmul_backward", (PyCFunction)(void (*)())entry<grouped_matmul_backward, 8>,
     METH_FASTCALL, nullptr},
    {"grouped_matmul_w4", (PyCFunction)(void (*)())entry<grouped_matmul_w4, 7>, METH_FASTCALL,
     nullptr},
    {"combine", (PyCFunction)(void (*)())entry<combine, 3>, METH_FASTCALL, nullptr},
    {"combine_backward", (PyCFunction)(void (*)())entry<combine_backward, 4>, METH_FASTCALL,
     nullptr},
    {"dropout", (PyCFunction)(void (*)())entry<dropout, 5>, METH_FASTCALL, nullptr},
    {"errors", (PyCFunction)(void (*)())entry<errors, 0>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_experts", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__experts(void) {
  PyObject* lib = PyImport_ImportModule("lightgbm_rs_b200._lib");
  if (!lib) return nullptr;
  g_error_type = PyObject_GetAttrString(lib, "LightGBMError");
  Py_DECREF(lib);
  return g_error_type ? PyModule_Create(&g_module) : nullptr;
}
