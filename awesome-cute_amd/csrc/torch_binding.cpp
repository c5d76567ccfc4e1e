// The calls of marlin.py and streamk.py on tensors, in C++: checks, sizes,
// pointers, the current stream, the output's allocation and the library call.
//
// Bound: host time.  A product of a few rows takes the GPU 3 to 10 us; the same
// steps in Python through ctypes took the host 5.8 us for `mul` and 12.5 us for
// a layer, so a decoder's linear layers ran at the host's pace.  Here they take
// 3.3 and 5.0 us (of which the output's allocation 1.2), the launch itself
// about 2.5: one row through the sixteen layers of four blocks of a 7B model
// 206 -> 122 us on one box, 189 -> 135 on another.
//
// Tensors are allocated and the library is entered with the interpreter lock
// released, as torch's own calls and ctypes do: a launch may wait for room in
// the stream's queue, a stream's first call allocates, and an allocation may
// wait for another thread's.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/GradMode.h>
#include <c10/core/InferenceMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <pybind11/pybind11.h>

#include "../../include/feedforward_amd.h"
#include "../../include/marlin_amd.h"
#include "../../include/marlin_amd_convert.h"
#include "../../include/streamk_amd.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

const at::Tensor* tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a torch.Tensor", name);
    return nullptr;
  }
  return &THPVariable_Unpack(o);
}

// an argument that may be None; false with an exception set
bool optional(PyObject* o, const char* name, at::Tensor* out) {
  if (o == Py_None) return true;
  const at::Tensor* const t = tensor(o, name);
  if (!t) return false;
  *out = *t;
  return true;
}

bool to_int(PyObject* o, int* v) {
  const long x = PyLong_AsLong(o);
  if (x == -1 && PyErr_Occurred()) return false;
  if (x != (int)x) {
    PyErr_SetString(PyExc_OverflowError, "argument does not fit into a C int");
    return false;
  }
  *v = (int)x;
  return true;
}

void* current_stream(int dev) { return (void*)c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream(); }

bool differentiated(std::initializer_list<const at::Tensor*> inputs) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : inputs)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Whether something records the operators of torch's dispatcher: a dispatch mode (make_fx, fake
// tensors, a counter), torch.jit.trace, or a tensor of its own kind.  A launch behind the dispatcher
// is nothing to them, and all that they would see of a call is its output's allocation; the caller,
// in Python, gets NotImplemented and takes the call's operator, which comes back here with one
// argument more (`Call::inner`) once nobody looks on.
bool looked_on(std::initializer_list<const at::Tensor*> inputs) {
  if (c10::impl::TorchDispatchModeTLS::any_modes_set() || at::tracer::impl::is_dispatch_enabled()) return true;
  for (const at::Tensor* t : inputs)
    if (t->defined() && t->key_set().has(c10::DispatchKey::Python)) return true;
  return false;
}

// The arguments that a call came with: `want`, or one more
struct Call {
  bool inner = false;
  bool takes(Py_ssize_t nargs, Py_ssize_t want, const char* name) {
    inner = nargs == want + 1;
    if (nargs == want || inner) return true;
    PyErr_Format(PyExc_TypeError, "%s takes %d arguments", name, (int)want);
    return false;
  }
};

// No kernel carries tangents along, and a result without one would count as a constant
void refuse_tangents(std::initializer_list<const at::Tensor*> inputs) {
  for (const at::Tensor* t : inputs)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), "forward-mode differentiation is not supported");
}

// The result of a product with 4-bit weights, which have no gradients, for inputs that want some: a
// backward pass that gets there is told.  (The node's edges go on to the inputs, so that it is on the
// way of every gradient that is asked for; without it a sum with the product would pass back
// the gradient of its other terms alone.)
at::Tensor without_gradients(const at::Tensor& out, std::initializer_list<const at::Tensor*> inputs) {
  variable_list all = {out};
  for (const at::Tensor* t : inputs) all.push_back(*t);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "products with 4-bit weights have no gradients", (int64_t)all.size());
  return (*error)(std::move(all))[0];
}

constexpr int kMulTensors = 5;
const char* const kMulNames[kMulTensors] = {"A", "B", "C", "s", "workspace"};

bool check_mul(const at::Tensor* const* t) {
  for (int i = 0; i < kMulTensors; i++)
    if (!t[i]->is_cuda()) {
      PyErr_Format(PyExc_RuntimeError, "%s must be a GPU tensor", kMulNames[i]);
      return false;
    }
  for (int i = 0; i < kMulTensors; i++)
    if (!t[i]->is_contiguous()) {
      PyErr_Format(PyExc_RuntimeError, "%s must be contiguous", kMulNames[i]);
      return false;
    }
  return true;
}

struct Hints {
  int thread_k = -1, thread_n = -1, sms = -1, max_par = 16, cute = 1;
};

// C (m, n) = A (m, k) * dequantised B; false with an exception set
bool enqueue_mul(const at::Tensor& A, const at::Tensor& B, const at::Tensor& C, const at::Tensor& s,
                 const at::Tensor& workspace, int64_t m, int64_t n, int64_t k, const Hints& h) {
  const int dev = A.get_device();
  char err[512];
  int rc;
  void* const st = current_stream(dev);
  const void *pa = A.data_ptr(), *pb = B.data_ptr(), *ps = s.data_ptr();
  void *pc = C.data_ptr(), *pw = workspace.data_ptr();
  const int s_rows = (int)s.size(0);
  const long long ws = workspace.numel();
  Py_BEGIN_ALLOW_THREADS
  rc = marlin_mul(pa, pb, pc, ps, (int)m, (int)n, (int)k, s_rows, pw, ws, dev, st, h.thread_k,
                  h.thread_n, h.sms, h.max_par, h.cute, err, sizeof(err));
  Py_END_ALLOW_THREADS
  if (rc == 0) return true;
  if (err[0])
    PyErr_SetString(PyExc_RuntimeError, err);
  else
    PyErr_Format(PyExc_RuntimeError, "marlin_mul failed with code %d", rc);
  return false;
}

// mul(A, B, C, s, workspace, thread_k, thread_n, sms, max_par, cute_version)
PyObject* py_mul(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Call call;
  if (!call.takes(nargs, 10, "mul")) return nullptr;
  const at::Tensor* t[kMulTensors];
  for (int i = 0; i < kMulTensors; i++)
    if (!(t[i] = tensor(args[i], kMulNames[i]))) return nullptr;
  if (!call.inner && looked_on({t[0], t[1], t[2], t[3], t[4]})) Py_RETURN_NOTIMPLEMENTED;
  Hints h;
  if (!to_int(args[5], &h.thread_k) || !to_int(args[6], &h.thread_n) || !to_int(args[7], &h.sms) ||
      !to_int(args[8], &h.max_par))
    return nullptr;
  h.cute = PyObject_IsTrue(args[9]);
  if (h.cute < 0 || !check_mul(t)) return nullptr;
  if (!enqueue_mul(*t[0], *t[1], *t[2], *t[3], *t[4], t[0]->size(0), t[2]->size(1), t[0]->size(1), h))
    return nullptr;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// linear(A, B, s, workspace, cute_version) -> C: the last dimension of A times
// the weight, rows of any shape
PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Call call;
  if (!call.takes(nargs, 5, "linear")) return nullptr;
  const at::Tensor *A = tensor(args[0], "A"), *B = tensor(args[1], "B"), *s = tensor(args[2], "s"),
                   *workspace = tensor(args[3], "workspace");
  if (!A || !B || !s || !workspace) return nullptr;
  if (!call.inner && looked_on({A, B, s, workspace})) Py_RETURN_NOTIMPLEMENTED;
  Hints h;
  h.cute = PyObject_IsTrue(args[4]);
  if (h.cute < 0) return nullptr;
  if (A->dim() < 1 || s->dim() < 2) {
    PyErr_SetString(PyExc_IndexError, "A needs a last dimension and s two");
    return nullptr;
  }
  const int64_t n = s->size(1), k = A->size(-1);
  c10::SmallVector<int64_t, 6> shape(A->sizes().begin(), A->sizes().end());
  shape.back() = n;
  at::Tensor C, rows;
  {
    pybind11::gil_scoped_release unlocked;
    C = at::empty(shape, A->options().requires_grad(false).memory_format(c10::nullopt));
    // (a copy where the leading dimensions do not fold into one)
    if (!A->is_contiguous() || k == 0) rows = A->reshape({-1, k});
  }
  if (rows.defined()) A = &rows;
  const at::Tensor* const t[kMulTensors] = {A, B, &C, s, workspace};
  if (!check_mul(t)) return nullptr;
  if (!enqueue_mul(*A, *B, C, *s, *workspace, A->numel() / k, n, k, h)) return nullptr;
  return THPVariable_Wrap(std::move(C));
  END_HANDLE_TH_ERRORS
}

// The operands of a gated projection with 4-bit weights: A (rows, k), B (k/16, 4n), C (rows, n),
// s (groups, 2n); false with an exception set.
bool enqueue_gated(const at::Tensor& A, const at::Tensor& B, const at::Tensor& C, const at::Tensor& s,
                   const at::Tensor& workspace, int act, int max_par) {
  const at::Tensor* const t[kMulTensors] = {&A, &B, &C, &s, &workspace};
  if (!check_mul(t)) return false;
  for (int i = 0; i < kMulTensors; i++) {
    const bool whole = i == 1 || i == 4;
    if (t[i]->scalar_type() != (whole ? at::kInt : at::kHalf)) {
      PyErr_Format(PyExc_ValueError, "%s must be of type torch.%s", kMulNames[i], whole ? "int32" : "half");
      return false;
    }
    if (t[i]->device() != A.device() || t[i]->is_neg()) {
      PyErr_Format(PyExc_ValueError, "%s must be a plain tensor on A's device", kMulNames[i]);
      return false;
    }
  }
  constexpr int64_t most = 0x7fffffff;
  if (A.dim() != 2 || B.dim() != 2 || C.dim() != 2 || s.dim() != 2 || A.size(0) != C.size(0) ||
      A.size(0) > most || A.size(1) > most || C.size(1) > most / 2 || s.size(0) > most ||
      B.size(0) != A.size(1) / 16 || B.size(1) != 4 * C.size(1) || s.size(1) != 2 * C.size(1)) {
    PyErr_SetString(PyExc_ValueError,
                    "a gated product takes A (m, k), B (k/16, 4n), C (m, n) and s (groups, 2n)");
    return false;
  }
  const int dev = A.get_device();
  char err[512];
  int rc;
  void* const st = current_stream(dev);
  const void *pa = A.data_ptr(), *pb = B.data_ptr(), *ps = s.data_ptr();
  void *pc = C.data_ptr(), *pw = workspace.data_ptr();
  const int m = (int)A.size(0), n = (int)C.size(1), k = (int)A.size(1), groups = (int)s.size(0);
  const long long ws = workspace.numel();
  Py_BEGIN_ALLOW_THREADS
  rc = feedforward_gated_w4(pa, pb, pc, ps, m, n, k, groups, pw, ws, act, dev, st, max_par, err, sizeof(err));
  Py_END_ALLOW_THREADS
  if (rc == 0) return true;
  PyErr_SetString(PyExc_RuntimeError, err);
  return false;
}

// gated_mul(A, B, C, s, workspace, activation, max_par)
PyObject* py_gated_mul(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Call call;
  if (!call.takes(nargs, 7, "gated_mul")) return nullptr;
  const at::Tensor* t[kMulTensors];
  for (int i = 0; i < kMulTensors; i++)
    if (!(t[i] = tensor(args[i], kMulNames[i]))) return nullptr;
  int act, max_par;
  if (!to_int(args[5], &act) || !to_int(args[6], &max_par)) return nullptr;
  refuse_tangents({t[0], t[2], t[3]});
  // (as torch's functions with an `out` do)
  TORCH_CHECK(call.inner || !differentiated({t[0], t[2], t[3]}),
              "gated_mul writes into C and has no gradients, but an argument requires one");
  if (!call.inner && looked_on({t[0], t[1], t[2], t[3], t[4]})) Py_RETURN_NOTIMPLEMENTED;
  if (!enqueue_gated(*t[0], *t[1], *t[2], *t[3], *t[4], act, max_par)) return nullptr;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// gated_linear(A, B, s, workspace, activation) -> C, rows of any shape
PyObject* py_gated_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Call call;
  if (!call.takes(nargs, 5, "gated_linear")) return nullptr;
  const at::Tensor *A = tensor(args[0], "A"), *B = tensor(args[1], "B"), *s = tensor(args[2], "s"),
                   *workspace = tensor(args[3], "workspace");
  if (!A || !B || !s || !workspace) return nullptr;
  int act;
  if (!to_int(args[4], &act)) return nullptr;
  refuse_tangents({A, s});
  if (!call.inner && looked_on({A, B, s, workspace})) Py_RETURN_NOTIMPLEMENTED;
  if (A->dim() < 1 || s->dim() != 2 || s->size(1) % 2 != 0 || A->size(-1) == 0) {
    PyErr_SetString(PyExc_ValueError, "A needs a last dimension, s two and an even number of columns");
    return nullptr;
  }
  const int64_t n = s->size(1) / 2, k = A->size(-1);
  c10::SmallVector<int64_t, 6> shape(A->sizes().begin(), A->sizes().end());
  shape.back() = n;
  at::Tensor C, rows, out;
  {
    pybind11::gil_scoped_release unlocked;
    C = at::empty(shape, A->options().requires_grad(false).memory_format(c10::nullopt));
    // (a copy where the leading dimensions do not fold into one)
    rows = A->reshape({-1, k});
    if (!rows.is_contiguous()) rows = rows.contiguous();
    out = C.view({rows.size(0), n});
  }
  if (!enqueue_gated(rows, *B, out, *s, *workspace, act, 16)) return nullptr;
  return THPVariable_Wrap(!call.inner && differentiated({A, s}) ? without_gradients(C, {A, s}) : std::move(C));
  END_HANDLE_TH_ERRORS
}

// without_gradients(out, A): out as the result of products of A
PyObject* py_without_gradients(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "without_gradients takes 2 arguments");
    return nullptr;
  }
  const at::Tensor *out = tensor(args[0], "out"), *A = tensor(args[1], "A");
  if (!out || !A) return nullptr;
  return THPVariable_Wrap(differentiated({A}) ? without_gradients(*out, {A}) : *out);
  END_HANDLE_TH_ERRORS
}

// dense(A, B, C or None) -> C (m, n) = A (m, k) * B (n, k)^T
PyObject* py_dense(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Call call;
  if (!call.takes(nargs, 3, "dense")) return nullptr;
  const at::Tensor* in[2];
  for (int i = 0; i < 2; i++) {
    const char* const name = i ? "B" : "A";
    if (!(in[i] = tensor(args[i], name))) return nullptr;
    if (!call.inner && looked_on({in[i]})) Py_RETURN_NOTIMPLEMENTED;
    if (in[i]->scalar_type() != at::kHalf || !in[i]->is_cuda() || !in[i]->is_contiguous() ||
        in[i]->dim() != 2) {
      PyErr_Format(PyExc_ValueError, "%s must be a contiguous 2-d torch.half tensor on the GPU", name);
      return nullptr;
    }
  }
  const at::Tensor &A = *in[0], &B = *in[1];
  const int64_t m = A.size(0), k = A.size(1), n = B.size(0);
  if (B.size(1) != k) {
    PyErr_SetString(PyExc_ValueError, "A and B must have the same k");
    return nullptr;
  }
  at::Tensor C;
  if (args[2] == Py_None) {
    pybind11::gil_scoped_release unlocked;
    C = at::empty({m, n}, A.options().requires_grad(false));
  } else {
    const at::Tensor* c = tensor(args[2], "C");
    if (!c) return nullptr;
    if (c->dim() != 2 || c->size(0) != m || c->size(1) != n || c->scalar_type() != at::kHalf ||
        !c->is_contiguous() || c->device() != A.device()) {
      PyErr_SetString(PyExc_ValueError, "C must be a contiguous (m, n) torch.half tensor on A's device");
      return nullptr;
    }
    C = *c;
  }
  const int dev = A.get_device();
  void* const st = current_stream(dev);
  const void *pa = A.data_ptr(), *pb = B.data_ptr();
  void* pc = C.data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = streamk_gemm_tn(pa, pb, pc, (int)m, (int)n, (int)k, dev, st);
  Py_END_ALLOW_THREADS
  if (rc == STREAMK_ERR_SHAPE) {
    PyErr_Format(PyExc_ValueError,
                 "shape (m=%lld, n=%lld, k=%lld) not supported: n must be a multiple of 256, k of 64",
                 (long long)m, (long long)n, (long long)k);
    return nullptr;
  }
  if (rc != STREAMK_OK) {
    PyErr_Format(PyExc_RuntimeError, "streamk_gemm_tn: %s", streamk_amd_last_error());
    return nullptr;
  }
  if (args[2] == Py_None) return THPVariable_Wrap(std::move(C));
  Py_INCREF(args[2]);
  return args[2];
  END_HANDLE_TH_ERRORS
}

// ---- dense feed-forward products (feedforward_amd.h) with fp16 or bfloat16 tensors.  A pass that
// takes several launches makes all of them here, its temporaries among them: they come from torch's
// allocator on the current stream and go back to it in that stream's order.  The autograd functions
// are C++ as well: as Python's they took the host 50 us more a pass than the kernels of a small one.

// a matrix as the kernels address it: rows that start on 16 bytes, at most kFarthest elements apart
constexpr int64_t kFarthest = 1 << 21;
struct Matrix {
  at::Tensor t;
  void* there = nullptr;  // (without a tensor)
  long long ld = 0;
  Matrix(void* at, long long ld) : there(at), ld(ld) {}
  // y as `rows` rows of `width`.  (One that is whole is taken without a view: views of all the
  // operands take the host 5 us of a backward pass.)
  Matrix(const at::Tensor& y, int64_t rows, int64_t width) : t(y) {
    if (y.is_contiguous() && (reinterpret_cast<uintptr_t>(y.data_ptr()) & 15) == 0 && width % 8 == 0) {
      ld = width;
      return;
    }
    const at::Tensor x = y.reshape({rows, width});
    t = x;
    const bool one = rows <= 1;
    const bool apart = !one && (x.stride(0) % 8 != 0 || x.stride(0) < x.size(1) || x.stride(0) > kFarthest);
    if (x.numel() != 0 && ((x.size(1) > 1 && x.stride(1) != 1) || apart ||
                           (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) != 0)) {
      t = at::empty(x.sizes(), x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
      t.copy_(x);
    }
    ld = t.size(0) <= 1 || t.numel() == 0 ? (t.size(1) + 7) / 8 * 8 : t.stride(0);
  }
  void* at() const { return t.defined() ? t.data_ptr() : there; }
};

// a gradient whose memory holds its values: autograd may hand over a view that is to be read negated
at::Tensor plain_values(const at::Tensor& grad) { return grad.defined() ? grad.resolve_neg() : grad; }

void feedforward_check(int rc) {
  TORCH_CHECK_VALUE(rc != FEEDFORWARD_ERR_SHAPE, feedforward_last_error());
  TORCH_CHECK(rc == FEEDFORWARD_OK, feedforward_last_error());
}

// x (..., k) and w (rows, k)
void check_dense(const at::Tensor& x, const at::Tensor& w) {
  for (const at::Tensor* t : {&x, &w}) {
    const char* const name = t == &x ? "x" : "weight";
    TORCH_CHECK_VALUE(t->is_cuda() && (t->scalar_type() == at::kHalf || t->scalar_type() == at::kBFloat16), name,
                      " must be a torch.half or torch.bfloat16 tensor on the GPU");
    TORCH_CHECK_VALUE(t->layout() == at::kStrided && !t->is_neg() && !t->is_conj(), name, " must be a plain tensor");
  }
  TORCH_CHECK_VALUE(x.scalar_type() == w.scalar_type() && x.device() == w.device(),
                    "x and weight must have one type and one device");
  TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1) && w.size(1) != 0,
                    "weight must have two dimensions, the second one x's last, not 0");
  TORCH_CHECK_VALUE(w.size(0) <= 0x7fffffff && w.size(1) <= 0x7fffffff && x.numel() / w.size(1) <= 0x7fffffff,
                    "a size does not fit into a C int");
}

int type_code(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat ? FEEDFORWARD_FP32 : t.scalar_type() == at::kBFloat16 ? FEEDFORWARD_BF16 : FEEDFORWARD_FP16;
}
void* at_of(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

using Maybe = std::optional<at::Tensor>;
Maybe maybe(const at::Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }

at::TensorOptions options_as(const at::Tensor& like) {
  return like.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous);
}
at::Tensor empty_as(const at::Tensor& like, at::IntArrayRef shape) { return at::empty(shape, options_as(like)); }

at::Tensor empty_rows(const at::Tensor& x, int64_t columns) {
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = columns;
  return empty_as(x, shape);
}

// A backward pass that is captured into a graph while an eager graph of the same leaves is alive:
// a leaf's accumulator lives as long as any graph that ends in it and belongs to the stream that was
// current when it was made.  The engine would make that stream wait for the captured one, which draws
// it into the capture without a way back, and the capture's end takes the process with it.  Refused
// here, before the engine gets there.
void check_capture(at::ArrayRef<at::Tensor> inputs, int dev) {
  const c10::hip::HIPStream now = c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev);
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(now.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
  for (const at::Tensor& t : inputs) {
    if (!t.defined() || !t.requires_grad() || !t.is_leaf()) continue;
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto stream = accumulator ? accumulator->stream() : std::nullopt;
    // (by number: torch names the device of one of them CUDA, of the other HIP)
    TORCH_CHECK(!stream || (stream->id() == now.id() && stream->device_index() == dev),
                "the stream is being captured, and an eager graph of the same leaf, made on another stream, is "
                "alive: free what was computed from it before the capture, or compute it on this stream");
  }
}

// The gradients that a backward pass returns, where that is itself to be differentiated: no kernel
// does, and whoever asks for it is told.  `from`: what they are made of, to which the edges of the
// node that tells go on -- without these it is on the way to no input, and a second derivative
// that has another path to its input would be that path's alone.
variable_list once_differentiable(variable_list&& grads, const char* name, std::initializer_list<const variable_list*> from) {
  if (!c10::GradMode::is_enabled()) return std::move(grads);
  const size_t count = grads.size();
  variable_list all;
  for (at::Tensor& g : grads) all.push_back(g.defined() ? g.detach().set_requires_grad(true) : g);
  for (const variable_list* list : from) all.insert(all.end(), list->begin(), list->end());
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " is differentiable once",
                                                               (int64_t)all.size());
  variable_list marked = (*error)(std::move(all));
  marked.resize(count);
  return marked;
}

// What stands for the inputs of the node that runs, where the backward pass has not kept them: nothing but their edges
variable_list inputs_of_the_node() {
  variable_list out;
  if (!c10::GradMode::is_enabled()) return out;
  if (const auto node = torch::autograd::get_current_node())
    for (const torch::autograd::Edge& edge : node->next_edges())
      if (edge.is_valid()) torch::autograd::impl::set_gradient_edge(out.emplace_back(at::empty({0})), edge);
  return out;
}

// Scratch for a product's partial sums, where its plan has any: its own, or memory that is there
struct Room {
  at::Tensor t;
  void* there = nullptr;
  long long bytes;
  Room(void* at, long long bytes) : there(at), bytes(bytes) {}
  Room(const at::Tensor& like, int64_t m, int64_t n, int64_t k, int gated, int turned)
      : bytes(feedforward_product_bytes((int)m, (int)n, (int)k, gated, turned, like.get_device())) {
    if (bytes > 0) t = at::empty({bytes / 4}, options_as(like).dtype(at::kFloat));
  }
  void* at() const { return t.defined() ? t.data_ptr() : there; }
};

// act(x G^T) * (x U^T), and with `keep` both sums (otherwise undefined)
std::pair<at::Tensor, at::Tensor> gated_forward(const at::Tensor& x, const at::Tensor& w, int act, bool keep) {
  check_dense(x, w);
  TORCH_CHECK_VALUE(w.size(0) % 2 == 0, "weight must hold the rows of gate and, behind them, as many of up");
  const int64_t n = w.size(0) / 2, k = w.size(1), m = x.numel() / k, ldpre = (n + 15) / 16 * 32;
  const int dev = x.get_device();
  at::Tensor h = empty_rows(x, n), pre;
  if (keep) pre = at::empty({m, ldpre}, options_as(x).dtype(at::kFloat));
  const Matrix a(x, m, k), b(w, 2 * n, k);
  const Room room(x, m, n, k, true, FEEDFORWARD_ROWS);
  feedforward_check(feedforward_gated(a.at(), b.at(), h.data_ptr(), keep ? (float*)pre.data_ptr() : nullptr, (int)m,
                                      (int)n, (int)k, a.ld, b.ld, n, ldpre, type_code(x), act, room.at(), room.bytes,
                                      dev, current_stream(dev)));
  return {h, pre};
}

at::Tensor linear_forward(const at::Tensor& x, const at::Tensor& w) {
  check_dense(x, w);
  const int64_t n = w.size(0), k = w.size(1), m = x.numel() / k;
  const int dev = x.get_device();
  at::Tensor y = empty_rows(x, n);
  const Matrix a(x, m, k), b(w, n, k);
  const Room room(x, m, n, k, false, FEEDFORWARD_ROWS);
  feedforward_check(feedforward_product(a.at(), b.at(), y.data_ptr(), (int)m, (int)n, (int)k, a.ld, b.ld, n,
                                        FEEDFORWARD_ROWS, type_code(x), room.at(), room.bytes, dev,
                                        current_stream(dev)));
  return y;
}

// The gradients of x (m, k) and w (r, k) from that of their product, d (m, r): dx = d w and
// dw = d^T x, sums over r and over m, times `scale`.  x and w need be there for the other's gradient alone.
// `shared`, if there: room for one of the two at a time.
void product_grads(const at::Tensor& x, const at::Tensor& w, const Matrix& d, const at::Tensor& dx,
                   const at::Tensor& dw, float scale = 1.f, const Room* shared = nullptr) {
  const at::Tensor &as_x = x.defined() ? x : dx, &as_w = w.defined() ? w : dw, &like = dx.defined() ? dx : dw;
  if (!like.defined()) return;
  const int64_t k = like.size(-1), m = as_x.defined() ? as_x.numel() / k : 0, r = as_w.defined() ? as_w.size(0) : 0;
  const int type = type_code(like), dev = like.get_device();
  void* const st = current_stream(dev);
  if (dx.defined()) {
    const Matrix b(w, r, k);
    const Room room = shared ? *shared : Room(like, m, k, r, false, FEEDFORWARD_TURN_B);
    feedforward_check(feedforward_product_scaled(d.at(), b.at(), dx.data_ptr(), (int)m, (int)k, (int)r, d.ld, b.ld, k,
                                                 FEEDFORWARD_TURN_B, type, scale, room.at(), room.bytes, dev, st));
  }
  if (dw.defined()) {
    const Matrix a(x, m, k);
    const Room room = shared ? *shared : Room(like, r, k, m, false, FEEDFORWARD_TURN_BOTH);
    feedforward_check(feedforward_product_scaled(d.at(), a.at(), dw.data_ptr(), (int)r, (int)k, (int)m, d.ld, a.ld, k,
                                                 FEEDFORWARD_TURN_BOTH, type, scale, room.at(), room.bytes, dev, st));
  }
}

// -> (dx, dweight), undefined where not wanted
std::pair<at::Tensor, at::Tensor> gated_backward(const at::Tensor& dh, const at::Tensor& pre, const at::Tensor& x,
                                                 const at::Tensor& w, int act, bool want_x, bool want_w) {
  check_dense(x, w);
  const int64_t n = w.size(0) / 2, k = w.size(1), m = x.numel() / k, ldpre = (n + 15) / 16 * 32;
  TORCH_CHECK_VALUE(dh.scalar_type() == x.scalar_type() && dh.device() == x.device() && dh.dim() >= 1 &&
                        dh.size(-1) == n && dh.numel() == m * n && pre.scalar_type() == at::kFloat &&
                        pre.device() == x.device() && pre.numel() == m * ldpre && pre.is_contiguous(),
                    "dh and the sums must be those of x and weight");
  const int dev = x.get_device();
  check_capture({x, w}, dev);
  at::Tensor dx, dw;
  if (want_x) dx = empty_as(x, x.sizes());
  if (want_w) dw = empty_as(w, w.sizes());
  if (m == 0 || n == 0) {
    if (want_x) dx.zero_();
    if (want_w) dw.zero_();
  } else if (want_x || want_w) {
    const int64_t ld = (2 * n + 63) / 64 * 64;  // rows of whole cache lines
    const Matrix d(plain_values(dh), m, n), dgu(empty_as(x, {m, ld}), m, ld);
    feedforward_check(feedforward_gated_grad(d.at(), (const float*)pre.data_ptr(), dgu.at(), (int)m, (int)n, d.ld,
                                             ldpre, ld, type_code(x), act, dev, current_stream(dev)));
    product_grads(x, w, dgu, dx, dw);
  }
  return {dx, dw};
}

std::pair<at::Tensor, at::Tensor> linear_backward(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& w,
                                                  bool want_x, bool want_w) {
  check_dense(x, w);
  const int64_t n = w.size(0), k = w.size(1), m = x.numel() / k;
  TORCH_CHECK_VALUE(dy.scalar_type() == x.scalar_type() && dy.device() == x.device() && dy.dim() >= 1 &&
                        dy.size(-1) == n && dy.numel() == m * n,
                    "dy must be that of x and weight");
  const int dev = x.get_device();
  check_capture({x, w}, dev);
  at::Tensor dx, dw;
  if (want_x) dx = empty_as(x, x.sizes());
  if (want_w) dw = empty_as(w, w.sizes());
  if (m == 0 || n == 0) {
    if (want_x) dx.zero_();
    if (want_w) dw.zero_();
  } else if (want_x || want_w) {
    product_grads(x, w, Matrix(plain_values(dy), m, n), dx, dw);
  }
  return {dx, dw};
}

struct GatedFunction : torch::autograd::Function<GatedFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, int64_t act) {
    auto [h, pre] = gated_forward(x, w, (int)act, true);
    ctx->save_for_backward({x, w, pre});
    ctx->saved_data["act"] = act;
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(3);
    if (grads[0].defined()) {
      c10::AutoGradMode off(false);
      std::tie(out[0], out[1]) = gated_backward(grads[0], saved[2], saved[0], saved[1], (int)ctx->saved_data["act"].toInt(),
                                                ctx->needs_input_grad(0), ctx->needs_input_grad(1));
    }
    return once_differentiable(std::move(out), "gated", {&grads, &saved});
  }
};

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w) {
    ctx->save_for_backward({x, w});
    return linear_forward(x, w);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(2);
    if (grads[0].defined()) {
      c10::AutoGradMode off(false);
      std::tie(out[0], out[1]) = linear_backward(grads[0], saved[0], saved[1], ctx->needs_input_grad(0), ctx->needs_input_grad(1));
    }
    return once_differentiable(std::move(out), "linear", {&grads, &saved});
  }
};

PyObject* tuple_of(std::initializer_list<at::Tensor> tensors) {
  PyObject* const tuple = PyTuple_New((Py_ssize_t)tensors.size());
  if (!tuple) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : tensors) PyTuple_SET_ITEM(tuple, i++, THPVariable_Wrap(t));  // (None where undefined)
  return tuple;
}

bool takes(Py_ssize_t nargs, Py_ssize_t want, const char* name) {
  if (nargs == want) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %d arguments", name, (int)want);
  return false;
}

// gated_dense(x, weight, activation) -> h, with what its gradients need where they are wanted
PyObject* py_gated_dense(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Call call;
  if (!call.takes(nargs, 3, "gated_dense")) return nullptr;
  const at::Tensor *x = tensor(args[0], "x"), *w = tensor(args[1], "weight");
  int act;
  if (!x || !w || !to_int(args[2], &act)) return nullptr;
  at::Tensor h;
  refuse_tangents({x, w});
  if (!call.inner && looked_on({x, w})) Py_RETURN_NOTIMPLEMENTED;
  {
    pybind11::gil_scoped_release unlocked;
    h = !call.inner && differentiated({x, w}) ? GatedFunction::apply(*x, *w, (int64_t)act) : gated_forward(*x, *w, act, false).first;
  }
  return THPVariable_Wrap(std::move(h));
  END_HANDLE_TH_ERRORS
}

// linear_dense(x, weight) -> x weight^T, likewise
PyObject* py_linear_dense(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Call call;
  if (!call.takes(nargs, 2, "linear_dense")) return nullptr;
  const at::Tensor *x = tensor(args[0], "x"), *w = tensor(args[1], "weight");
  if (!x || !w) return nullptr;
  at::Tensor y;
  refuse_tangents({x, w});
  if (!call.inner && looked_on({x, w})) Py_RETURN_NOTIMPLEMENTED;
  {
    pybind11::gil_scoped_release unlocked;
    y = !call.inner && differentiated({x, w}) ? LinearFunction::apply(*x, *w) : linear_forward(*x, *w);
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// gated_sums(x, weight, activation) -> (h, both sums), gated_grads(dh, sums, x, weight, activation, want_x,
// want_weight) and linear_grads(dy, x, weight, want_x, want_weight) -> (dx, dweight), None where not
// wanted: the passes by themselves, for compilers
bool to_bool(PyObject* o, bool* v) {
  const int is = PyObject_IsTrue(o);
  *v = is > 0;
  return is >= 0;
}

PyObject* py_gated_sums(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (!takes(nargs, 3, "gated_sums")) return nullptr;
  const at::Tensor *x = tensor(args[0], "x"), *w = tensor(args[1], "weight");
  int act;
  if (!x || !w || !to_int(args[2], &act)) return nullptr;
  std::pair<at::Tensor, at::Tensor> out;
  {
    pybind11::gil_scoped_release unlocked;
    out = gated_forward(*x, *w, act, true);
  }
  return tuple_of({out.first, out.second});
  END_HANDLE_TH_ERRORS
}

PyObject* py_gated_grads(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (!takes(nargs, 7, "gated_grads")) return nullptr;
  const at::Tensor *dh = tensor(args[0], "dh"), *pre = tensor(args[1], "sums"), *x = tensor(args[2], "x"),
                   *w = tensor(args[3], "weight");
  int act;
  bool want_x, want_w;
  if (!dh || !pre || !x || !w || !to_int(args[4], &act) || !to_bool(args[5], &want_x) || !to_bool(args[6], &want_w))
    return nullptr;
  std::pair<at::Tensor, at::Tensor> out;
  {
    pybind11::gil_scoped_release unlocked;
    out = gated_backward(*dh, *pre, *x, *w, act, want_x, want_w);
  }
  return tuple_of({out.first, out.second});
  END_HANDLE_TH_ERRORS
}

PyObject* py_linear_grads(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (!takes(nargs, 5, "linear_grads")) return nullptr;
  const at::Tensor *dy = tensor(args[0], "dy"), *x = tensor(args[1], "x"), *w = tensor(args[2], "weight");
  bool want_x, want_w;
  if (!dy || !x || !w || !to_bool(args[3], &want_x) || !to_bool(args[4], &want_w)) return nullptr;
  std::pair<at::Tensor, at::Tensor> out;
  {
    pybind11::gil_scoped_release unlocked;
    out = linear_backward(*dy, *x, *w, want_x, want_w);
  }
  return tuple_of({out.first, out.second});
  END_HANDLE_TH_ERRORS
}

// ---- dropout, and products with an epilogue

// What makes a mask: with p = 0 there is none, and whatever seed was given is let go.
struct Drop {
  double p = 0.0;
  int64_t seed = 0, site = 0;
  at::Tensor seed_at;  // or undefined

  bool on() const { return p != 0.0; }
  void check(const at::Tensor& x) const {
    TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "the probability of dropout must be 0 to 1, not ", p);
    TORCH_CHECK_VALUE(site >= 0 && site <= 0xffffffffLL, "site must be 0 to 2^32 - 1, not ", site);
    TORCH_CHECK_VALUE(!seed_at.defined() || (seed_at.scalar_type() == at::kLong && seed_at.numel() == 1 &&
                                             seed_at.layout() == at::kStrided && seed_at.device() == x.device()),
                      "a seed that is a tensor must be one torch.int64 on the device of x");
  }
  feedforward_drop plain() const {
    return {p, (long long)seed, seed_at.defined() ? (const long long*)seed_at.data_ptr() : nullptr, (unsigned)site};
  }
};

bool to_int64(PyObject* o, const char* name, int64_t* v) {
  int past = 0;
  const long long x = PyLong_AsLongLongAndOverflow(o, &past);
  if (x == -1 && PyErr_Occurred()) return false;
  if (past != 0) {
    PyErr_Format(PyExc_ValueError, "%s does not fit into 64 bits", name);
    return false;
  }
  *v = x;
  return true;
}

// p, seed (an int, a tensor or None) and site
bool drop_arguments(PyObject* const* args, Drop* out) {
  out->p = PyFloat_AsDouble(args[0]);
  if (PyErr_Occurred()) return false;
  if (!to_int64(args[2], "site", &out->site)) return false;
  if (!out->on()) return true;
  if (args[1] == Py_None) {
    PyErr_SetString(PyExc_ValueError, "dropout needs a seed");
    return false;
  }
  if (THPVariable_Check(args[1])) {
    out->seed_at = THPVariable_Unpack(args[1]);
    return true;
  }
  return to_int64(args[1], "seed", &out->seed);
}

// the tensors behind the first `want` arguments
bool leaves_behind(PyObject* const* args, Py_ssize_t nargs, Py_ssize_t want, const char* name, std::vector<at::Tensor>* out) {
  if (nargs < want) return takes(nargs, want, name);
  for (Py_ssize_t i = want; i < nargs; i++) {
    const at::Tensor* const t = tensor(args[i], "leaves");
    if (!t) return false;
    out->push_back(*t);
  }
  return true;
}

// What a forward pass keeps besides the tensors that it saves, as one object (an entry of the context's
// dictionary for each takes the host 0.1 to 0.2 us, both ways).  The leaves are what gradients go to that the
// backward pass has no other use for: check_capture wants them, and a leaf's accumulator, which the
// graph holds, holds the leaf.
struct Kept : torch::CustomClassHolder {
  int act = 0;
  int64_t k = 0;
  Drop drop;  // (its seed in memory is saved: if that has been written since, asking for it raises)
  std::vector<at::Tensor> leaves;
  bool there[2] = {};  // of a product the bias and the residual, of dropout the input and the residual
  void leaf(const at::Tensor& t) {
    if (t.defined() && t.is_leaf() && t.requires_grad()) leaves.push_back(t);
  }
  void input(int i, const at::Tensor& t) {
    there[i] = t.defined();
    leaf(t);
  }
};
void keep(AutogradContext* ctx, c10::intrusive_ptr<Kept> kept) {
  kept->drop.seed_at = at::Tensor();
  ctx->saved_data["kept"] = c10::IValue::make_capsule(std::move(kept));
}
c10::intrusive_ptr<Kept> kept_by(AutogradContext* ctx) {
  return c10::static_intrusive_pointer_cast<Kept>(ctx->saved_data.at("kept").toCapsule());
}

struct FullInputs {
  at::Tensor x, w, bias, residual;  // (the last two may be undefined)
  int act = 0;
  Drop drop;
  int64_t m = 0, n = 0, k = 0;

  void check() {
    check_dense(x, w);
    n = w.size(0), k = w.size(1), m = x.numel() / k;
    for (const at::Tensor* t : {&bias, &residual}) {
      if (!t->defined()) continue;
      const char* const name = t == &bias ? "bias" : "residual";
      TORCH_CHECK_VALUE(t->scalar_type() == x.scalar_type() && t->device() == x.device(), name,
                        " must have the type and the device of x");
      TORCH_CHECK_VALUE(t->layout() == at::kStrided && !t->is_neg(), name, " must be a plain tensor");
    }
    TORCH_CHECK_VALUE(!bias.defined() || (bias.dim() == 1 && bias.size(0) == n), "bias must have one dimension, the rows of weight");
    if (residual.defined()) {
      bool fits = residual.dim() == x.dim() && residual.size(-1) == n;
      for (int64_t i = 0; fits && i + 1 < x.dim(); i++) fits = residual.size(i) == x.size(i);
      TORCH_CHECK_VALUE(fits, "residual must have the result's shape");
    }
    drop.check(x);
  }
};

// residual + drop(act(x w^T + bias)), and, with an activation and anything to keep, the slopes that a backward
// pass takes, 16 bits each (otherwise undefined): those of feedforward_linear_train, or of feedforward_linear
enum class Keep { kNothing, kSlopes, kSteps };
std::pair<at::Tensor, at::Tensor> full_forward(FullInputs& in, Keep keep) {
  in.check();
  const int dev = in.x.get_device();
  at::Tensor y = empty_rows(in.x, in.n), slopes;
  if (keep != Keep::kNothing && in.act != 0) slopes = at::empty({in.m, in.n}, options_as(in.x).dtype(at::kShort));
  const Matrix a(in.x, in.m, in.k), b(in.w, in.n, in.k);
  std::optional<Matrix> bias, residual;
  if (in.bias.defined()) bias.emplace(in.bias, 1, in.n);
  if (in.residual.defined()) residual.emplace(in.residual, in.m, in.n);
  const Room room(in.x, in.m, in.n, in.k, FEEDFORWARD_FULL, FEEDFORWARD_ROWS);
  const feedforward_drop drop = in.drop.plain();
  const auto linear = keep == Keep::kSteps ? feedforward_linear : feedforward_linear_train;
  feedforward_check(linear(a.at(), b.at(), y.data_ptr(), bias ? bias->at() : nullptr, residual ? residual->at() : nullptr,
                           at_of(slopes), (int)in.m, (int)in.n, (int)in.k, a.ld, b.ld, in.n, residual ? residual->ld : 0,
                           in.n, type_code(in.x), in.act, &drop, room.at(), room.bytes, dev, current_stream(dev)));
  return {y, slopes};
}

// What a backward pass takes of a product: x (m, k) where its weight's gradient is wanted, w (n, k) where x's is
struct FullGrads {
  at::Tensor slopes, x, w;
  int act = 0;
  Drop drop;
  int64_t k = 0;
};

// -> (dx, dweight, dbias), undefined where not wanted.  (The residual's gradient is dy.)
std::array<at::Tensor, 3> full_backward(const at::Tensor& dy, const FullGrads& in, const std::array<bool, 3>& want,
                                        at::ArrayRef<at::Tensor> leaves) {
  const int64_t n = dy.size(-1), m = n > 0 ? dy.numel() / n : 0, k = in.k;
  const at::Tensor& slopes = in.slopes;
  const int dev = dy.get_device();
  check_capture(leaves, dev);
  std::array<at::Tensor, 3> out;
  if (want[0]) out[0] = empty_rows(dy, k);
  if (want[1]) out[1] = empty_as(dy, {n, k});
  if (want[2]) out[2] = empty_as(dy, {n});
  if (m == 0 || n == 0) {
    for (at::Tensor& g : out)
      if (g.defined()) g.zero_();
    return out;
  }
  const bool products = want[0] || want[1];
  if (!products && !want[2]) return out;
  const Matrix d(plain_values(dy), m, n);
  // One allocation holds what lives no longer than this call: the sums' gradient, which without an
  // activation and a mask is dy, the bias's partial sums, and room for the products, one after the other.
  // (Each of its own takes the host 1.2 us of a pass that on small problems is the host's.)
  const bool other = products && (in.act != 0 || in.drop.on());
  const int64_t ld = (n + 63) / 64 * 64;  // rows of whole cache lines
  const long long dz_bytes = other ? 2 * m * ld : 0;
  const long long sum_bytes = want[2] ? (feedforward_linear_grad_bytes((int)m, (int)n) + 255) / 256 * 256 : 0;
  const auto product_bytes = [&](int64_t rows, int64_t sum, int turned) {
    return feedforward_product_bytes((int)rows, (int)k, (int)sum, 0, turned, dev);
  };
  const long long room_bytes = std::max(want[0] ? product_bytes(m, n, FEEDFORWARD_TURN_B) : 0,
                                        want[1] ? product_bytes(n, m, FEEDFORWARD_TURN_BOTH) : 0);
  at::Tensor scratch;
  if (dz_bytes + sum_bytes + room_bytes > 0)
    scratch = at::empty({dz_bytes + sum_bytes + room_bytes}, options_as(dy).dtype(at::kByte));
  char* const base = (char*)at_of(scratch);
  const Matrix dz = other ? Matrix(base, ld) : d;
  float factor = 1.f;
  if (other || want[2]) {
    const feedforward_drop drop = in.drop.plain();
    feedforward_check(feedforward_linear_backward(d.at(), at_of(slopes), other ? base : nullptr, at_of(out[2]), (int)m,
                                                  (int)n, d.ld, n, ld, type_code(dy), &drop,
                                                  sum_bytes ? base + dz_bytes : nullptr, sum_bytes, &factor, dev,
                                                  current_stream(dev)));
  }
  const Room room(room_bytes > 0 ? base + dz_bytes + sum_bytes : nullptr, room_bytes);
  if (products) product_grads(in.x, in.w, dz, out[0], out[1], factor, &room);
  return out;
}

// ... as they come from elsewhere than a forward pass that has checked them
void check_full_grads(const at::Tensor& dy, FullGrads* in) {
  check_dense(in->x, in->w);
  in->k = in->w.size(1);
  TORCH_CHECK_VALUE(dy.scalar_type() == in->x.scalar_type() && dy.device() == in->x.device() &&
                        dy.layout() == at::kStrided && dy.dim() >= 1 && dy.size(-1) == in->w.size(0) &&
                        dy.numel() == in->x.numel() / in->k * in->w.size(0),
                    "dy must be that of x and weight");
  const at::Tensor& slopes = in->slopes;
  TORCH_CHECK_VALUE(slopes.defined() == (in->act != 0) &&
                        (!slopes.defined() || (slopes.scalar_type() == at::kShort && slopes.device() == dy.device() &&
                                            slopes.numel() == dy.numel() && slopes.is_contiguous())),
                    "the slopes must be those of x and weight");
  in->drop.check(dy);
}

struct FullFunction : torch::autograd::Function<FullFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const Maybe& bias,
                            const Maybe& residual, int64_t act, double p, int64_t seed, int64_t site,
                            const Maybe& seed_at) {
    FullInputs in{x, w, bias.value_or(at::Tensor()), residual.value_or(at::Tensor()), (int)act,
                  Drop{p, seed, site, seed_at.value_or(at::Tensor())}};
    // Each operand is saved for the other's gradient, and the slopes for those of what they belong to: the residual's is
    // dy whatever they are.  (Operands of a frozen layer need not live until the backward pass.)
    const bool dx = x.requires_grad(), dw = w.requires_grad();
    auto [y, slopes] = full_forward(in, dx || dw || (in.bias.defined() && in.bias.requires_grad()) ? Keep::kSlopes : Keep::kNothing);
    ctx->save_for_backward({dw ? x : at::Tensor(), dx ? w : at::Tensor(), slopes, in.drop.seed_at});
    auto kept = c10::make_intrusive<Kept>();
    kept->act = in.act;
    kept->k = in.k;
    kept->drop = in.drop;
    kept->leaf(x);
    kept->leaf(w);
    kept->input(0, in.bias);
    kept->input(1, in.residual);
    keep(ctx, std::move(kept));
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(9);
    if (grads[0].defined()) {
      c10::AutoGradMode off(false);
      const auto kept = kept_by(ctx);
      FullGrads in{saved[2], saved[0], saved[1], kept->act, kept->drop, kept->k};
      in.drop.seed_at = saved[3];
      // (the context counts the inputs that are there)
      const std::array<bool, 3> want = {ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                        kept->there[0] && ctx->needs_input_grad(2)};
      auto g = full_backward(grads[0], in, want, kept->leaves);
      for (int i = 0; i < 3; i++) out[i] = g[i];
      if (kept->there[1] && ctx->needs_input_grad(2 + kept->there[0])) out[3] = grads[0];
    }
    const variable_list inputs = inputs_of_the_node();
    return once_differentiable(std::move(out), "linear", {&grads, &saved, &inputs});
  }
};

struct DropoutInputs {
  at::Tensor x, residual;  // (the latter may be undefined)
  Drop drop;

  void check() const {
    for (const at::Tensor* t : {&x, &residual}) {
      if (!t->defined()) continue;
      const char* const name = t == &x ? "x" : "residual";
      const auto type = t->scalar_type();
      TORCH_CHECK_VALUE(t->is_cuda() && (type == at::kHalf || type == at::kBFloat16 || type == at::kFloat), name,
                        " must be a torch.half, torch.bfloat16 or torch.float tensor on the GPU");
      TORCH_CHECK_VALUE(t->layout() == at::kStrided && !t->is_neg(), name, " must be a plain tensor");
    }
    TORCH_CHECK_VALUE(!residual.defined() || (residual.scalar_type() == x.scalar_type() &&
                                              residual.device() == x.device() && residual.sizes() == x.sizes()),
                      "residual must have the type, the device and the shape of x");
    drop.check(x);
  }
};

at::Tensor dropout_forward(const DropoutInputs& in) {
  in.check();
  const int dev = in.x.get_device();
  at::Tensor y = empty_as(in.x, in.x.sizes());
  const at::Tensor x = in.x.contiguous(), residual = in.residual.defined() ? in.residual.contiguous() : in.residual;
  const feedforward_drop drop = in.drop.plain();
  feedforward_check(feedforward_dropout(x.data_ptr(), at_of(residual), y.data_ptr(), x.numel(), type_code(x), &drop, dev,
                                        current_stream(dev)));
  return y;
}

// the gradient of x
at::Tensor dropout_backward(const at::Tensor& dy, const Drop& drop, at::ArrayRef<at::Tensor> leaves) {
  check_capture(leaves, dy.get_device());
  return dropout_forward({plain_values(dy), at::Tensor(), drop});
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const Maybe& residual, double p, int64_t seed,
                            int64_t site, const Maybe& seed_at) {
    const DropoutInputs in{x, residual.value_or(at::Tensor()), Drop{p, seed, site, seed_at.value_or(at::Tensor())}};
    at::Tensor y = dropout_forward(in);
    ctx->save_for_backward({in.drop.seed_at});
    auto kept = c10::make_intrusive<Kept>();
    kept->drop = in.drop;
    kept->input(0, x);
    kept->input(1, in.residual);
    keep(ctx, std::move(kept));
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(6);
    if (grads[0].defined()) {
      c10::AutoGradMode off(false);
      const auto kept = kept_by(ctx);
      Drop drop = kept->drop;
      drop.seed_at = saved[0];
      if (ctx->needs_input_grad(0)) out[0] = dropout_backward(grads[0], drop, kept->leaves);
      if (kept->there[1] && ctx->needs_input_grad(1)) out[1] = grads[0];
    }
    return once_differentiable(std::move(out), "dropout", {&grads, &saved});
  }
};

// x, weight, bias, residual (the last two may be None), activation, p, seed and site
bool full_arguments(PyObject* const* args, FullInputs* in) {
  const at::Tensor *x = tensor(args[0], "x"), *w = x ? tensor(args[1], "weight") : nullptr;
  if (!x || !w || !optional(args[2], "bias", &in->bias) || !optional(args[3], "residual", &in->residual) ||
      !to_int(args[4], &in->act) || !drop_arguments(args + 5, &in->drop))
    return false;
  in->x = *x;
  in->w = *w;
  return true;
}

// linear_full(x, weight, bias, residual, activation, p, seed, site) -> y, with what its gradients need where
// they are wanted
PyObject* py_linear_full(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Call call;
  FullInputs in;
  if (!call.takes(nargs, 8, "linear_full") || !full_arguments(args, &in)) return nullptr;
  refuse_tangents({&in.x, &in.w, &in.bias, &in.residual});
  if (!call.inner && looked_on({&in.x, &in.w, &in.bias, &in.residual, &in.drop.seed_at})) Py_RETURN_NOTIMPLEMENTED;
  at::Tensor y;
  {
    pybind11::gil_scoped_release unlocked;
    y = !call.inner && differentiated({&in.x, &in.w, &in.bias, &in.residual})
            ? FullFunction::apply(in.x, in.w, maybe(in.bias), maybe(in.residual), (int64_t)in.act, in.drop.p,
                                  in.drop.seed, in.drop.site, maybe(in.drop.seed_at))
            : full_forward(in, Keep::kNothing).first;
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// dropout(x, residual, p, seed, site) -> y, likewise
PyObject* py_dropout(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Call call;
  DropoutInputs in;
  if (!call.takes(nargs, 5, "dropout")) return nullptr;
  const at::Tensor* const x = tensor(args[0], "x");
  if (!x || !optional(args[1], "residual", &in.residual) || !drop_arguments(args + 2, &in.drop)) return nullptr;
  in.x = *x;
  refuse_tangents({&in.x, &in.residual});
  if (!call.inner && looked_on({&in.x, &in.residual, &in.drop.seed_at})) Py_RETURN_NOTIMPLEMENTED;
  at::Tensor y;
  {
    pybind11::gil_scoped_release unlocked;
    y = !call.inner && differentiated({&in.x, &in.residual})
            ? DropoutFunction::apply(in.x, maybe(in.residual), in.drop.p, in.drop.seed, in.drop.site, maybe(in.drop.seed_at))
            : dropout_forward(in);
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// dropout_grad(dy, p, seed, site, leaves) -> dx, for compilers
PyObject* py_dropout_grad(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Drop drop;
  std::vector<at::Tensor> leaves;
  if (!leaves_behind(args, nargs, 4, "dropout_grad", &leaves)) return nullptr;
  const at::Tensor* const dy = tensor(args[0], "dy");
  if (!dy || !drop_arguments(args + 1, &drop)) return nullptr;
  at::Tensor dx;
  {
    pybind11::gil_scoped_release unlocked;
    dx = dropout_backward(*dy, drop, leaves);
  }
  return THPVariable_Wrap(std::move(dx));
  END_HANDLE_TH_ERRORS
}

// linear_full_kept(... as linear_full) -> (y, the slopes or None) and linear_full_grads(dy, slopes, x, weight,
// activation, p, seed, site, want_x, want_weight, want_bias, more leaves) -> (dx, dweight, dbias), None where not
// wanted: the passes by themselves, for compilers.  linear_full_slopes: linear_full_kept with slopes in the form of the C
// entry feedforward_linear.
template <Keep KEEP>
PyObject* py_linear_full_kept(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  FullInputs in;
  if (!takes(nargs, 8, KEEP == Keep::kSteps ? "linear_full_slopes" : "linear_full_kept") || !full_arguments(args, &in))
    return nullptr;
  std::pair<at::Tensor, at::Tensor> out;
  {
    pybind11::gil_scoped_release unlocked;
    out = full_forward(in, KEEP);
  }
  return tuple_of({out.first, out.second});
  END_HANDLE_TH_ERRORS
}

PyObject* py_linear_full_grads(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  std::vector<at::Tensor> leaves;
  if (!leaves_behind(args, nargs, 11, "linear_full_grads", &leaves)) return nullptr;
  const at::Tensor *dy = tensor(args[0], "dy"), *x = dy ? tensor(args[2], "x") : nullptr,
                   *w = x ? tensor(args[3], "weight") : nullptr;
  FullGrads in;
  std::array<bool, 3> want;
  if (!w || !optional(args[1], "slopes", &in.slopes) || !to_int(args[4], &in.act) || !drop_arguments(args + 5, &in.drop))
    return nullptr;
  in.x = *x;
  in.w = *w;
  for (int i = 0; i < 3; i++)
    if (!to_bool(args[8 + i], &want[i])) return nullptr;
  leaves.push_back(in.x);
  leaves.push_back(in.w);
  std::array<at::Tensor, 3> g;
  {
    pybind11::gil_scoped_release unlocked;
    check_full_grads(*dy, &in);
    g = full_backward(*dy, in, want, leaves);
  }
  return tuple_of({g[0], g[1], g[2]});
  END_HANDLE_TH_ERRORS
}

// ---- the norms around a block, fp16, bfloat16 or fp32

// rows of d neighbouring elements, any distance apart that is not less
struct Rows {
  at::Tensor t;
  long long ld = 0;
  Rows() = default;
  Rows(const at::Tensor& x, int64_t rows, int64_t d) {
    if (!x.defined()) return;
    if (x.is_contiguous()) {
      t = x;
      ld = d;
      return;
    }
    t = x.reshape({rows, d});
    if (t.numel() != 0 && ((d > 1 && t.stride(1) != 1) || (rows > 1 && t.stride(0) < d)))
      t = t.contiguous();
    ld = rows > 1 && t.numel() != 0 ? t.stride(0) : d;
  }
  void* at() const { return t.defined() ? t.data_ptr() : nullptr; }
};

struct NormInputs {
  at::Tensor residual, block, post, gate, pre;  // (the last four may be undefined)
  int64_t rows = 0, d = 0, rows_per_gate = 1;

  void check() {
    const std::pair<const char*, const at::Tensor*> all[] = {
        {"residual", &residual}, {"block", &block}, {"post_weight", &post}, {"gate", &gate}, {"pre_weight", &pre}};
    for (const auto& [name, t] : all) {
      if (!t->defined()) continue;
      const auto type = t->scalar_type();
      TORCH_CHECK_VALUE(t->is_cuda() && (type == at::kHalf || type == at::kBFloat16 || type == at::kFloat), name,
                        " must be a torch.half, torch.bfloat16 or torch.float tensor on the GPU");
      TORCH_CHECK_VALUE(t->layout() == at::kStrided && !t->is_neg(), name, " must be a plain tensor");
      TORCH_CHECK_VALUE(type == residual.scalar_type() && t->device() == residual.device(), name,
                        " must have the residual's type and device");
    }
    const int64_t dims = residual.dim();
    TORCH_CHECK_VALUE(dims >= 1 && residual.size(-1) != 0, "residual needs a last dimension, not 0");
    d = residual.size(-1);
    rows = residual.numel() / d;
    TORCH_CHECK_VALUE(rows <= 0x7fffffff && d <= 0x7fffffff, "a size does not fit into a C int");
    TORCH_CHECK_VALUE(!block.defined() || block.sizes() == residual.sizes(), "block must have the residual's shape");
    for (const at::Tensor* w : {&post, &pre})
      TORCH_CHECK_VALUE(!w->defined() || (w->dim() == 1 && w->size(0) == d), w == &post ? "post_weight" : "pre_weight",
                        " must have one dimension, the residual's last");
    TORCH_CHECK_VALUE(block.defined() || (!post.defined() && !gate.defined()), "post_weight and gate belong to a block");
    TORCH_CHECK_VALUE(block.defined() || pre.defined(), "there is neither a block nor a pre_weight");
    rows_per_gate = rows > 0 ? rows : 1;
    if (!gate.defined()) return;
    // (d), or the residual's leading dimensions, ones for the others, and d
    bool fits = gate.dim() >= 1 && gate.size(-1) == d && (gate.dim() == 1 || gate.dim() == dims);
    if (fits && gate.dim() > 1) {
      int64_t ones = dims - 1, shared = 1;
      while (ones > 0 && gate.size(ones - 1) == 1) shared *= residual.size(--ones);
      for (int64_t i = 0; i < ones; i++) fits = fits && gate.size(i) == residual.size(i);
      rows_per_gate = shared > 0 ? shared : 1;
    }
    TORCH_CHECK_VALUE(fits, "gate must have the shape (d,), or the residual's with ones for its last dimensions but d");
  }
  int dev() const { return residual.get_device(); }
  Rows gate_rows() const { return gate.defined() ? Rows(gate, gate.numel() / d, d) : Rows(); }
};

at::Tensor weight_of(const at::Tensor& w) { return w.defined() ? w.contiguous() : w; }

struct NormOutputs {
  at::Tensor y, r, lengths;
};

NormOutputs norm_forward(NormInputs& in, double scale, double eps, bool keep) {
  in.check();
  const int dev = in.dev();
  NormOutputs out;
  if (in.pre.defined()) out.y = empty_as(in.residual, in.residual.sizes());
  if (in.block.defined()) out.r = empty_as(in.residual, in.residual.sizes());
  if (keep) out.lengths = at::empty({in.rows, 2}, options_as(in.residual).dtype(at::kFloat));
  const Rows res(in.residual, in.rows, in.d), block(in.block, in.rows, in.d), gate = in.gate_rows();
  const at::Tensor post = weight_of(in.post), pre = weight_of(in.pre);
  feedforward_check(feedforward_norm(res.at(), res.ld, block.at(), block.ld, at_of(post), gate.at(), gate.ld,
                                     (int)in.rows_per_gate, at_of(pre), (float)scale, (float)eps, at_of(out.r),
                                     at_of(out.y), (float*)at_of(out.lengths), in.rows, (int)in.d,
                                     type_code(in.residual), dev, current_stream(dev)));
  return out;
}

// The gradients of residual, block, post, gate and pre, undefined where not wanted; `in.residual` is the
// forward pass's r.  dy or dr may be undefined; `leaf` is the residual that went in, or undefined.
std::array<at::Tensor, 5> norm_backward(const at::Tensor& dy, const at::Tensor& dr, NormInputs& in,
                                        const at::Tensor& lengths, double scale, const at::Tensor& leaf,
                                        const std::array<bool, 5>& want) {
  in.check();
  for (const at::Tensor* g : {&dy, &dr})
    TORCH_CHECK_VALUE(!g->defined() || (g->sizes() == in.residual.sizes() && g->scalar_type() == in.residual.scalar_type() &&
                                        g->device() == in.residual.device()),
                      "dy and dr must be gradients of the outputs");
  TORCH_CHECK_VALUE(lengths.defined() && lengths.scalar_type() == at::kFloat && lengths.is_contiguous() &&
                        lengths.numel() == 2 * in.rows && lengths.device() == in.residual.device(),
                    "lengths must be those of the forward pass");
  const int dev = in.dev();
  check_capture({leaf, in.block, in.post, in.gate, in.pre}, dev);
  std::array<at::Tensor, 5> out;
  const at::Tensor* const like[5] = {&in.residual, &in.block, &in.post, &in.gate, &in.pre};
  for (int i = 0; i < 5; i++)
    if (want[i] && like[i]->defined()) out[i] = empty_as(*like[i], like[i]->sizes());
  // without dy nothing comes back through the last norm
  const bool back = in.pre.defined() && dy.defined();
  if (in.rows == 0 || (!back && !dr.defined())) {
    for (at::Tensor& g : out)
      if (g.defined()) g.zero_();
    return out;
  }
  if (out[4].defined() && !back) out[4].zero_();
  at::Tensor partials;
  long long bytes = 0;
  if (out[2].defined() || out[3].defined() || (out[4].defined() && back)) {
    bytes = feedforward_norm_grad_bytes(in.rows, (int)in.d, (int)in.rows_per_gate, type_code(in.residual));
    if (bytes > 0) partials = at::empty({bytes / 4}, options_as(in.residual).dtype(at::kFloat));
  }
  const Rows gdy(back ? plain_values(dy) : at::Tensor(), in.rows, in.d), gdr(plain_values(dr), in.rows, in.d), r(in.residual, in.rows, in.d),
      block(in.block, in.rows, in.d), gate = in.gate_rows();
  const at::Tensor post = weight_of(in.post), pre = back ? weight_of(in.pre) : at::Tensor();
  feedforward_check(feedforward_norm_grad(
      gdy.at(), gdy.ld, gdr.at(), gdr.ld, r.at(), r.ld, block.at(), block.ld, at_of(post), gate.at(), gate.ld,
      (int)in.rows_per_gate, at_of(pre), (float)scale, (const float*)lengths.data_ptr(), at_of(out[0]), at_of(out[1]),
      at_of(out[2]), at_of(out[3]), back ? at_of(out[4]) : nullptr, at_of(partials), bytes, in.rows, (int)in.d,
      type_code(in.residual), dev, current_stream(dev)));
  return out;
}

// outputs y and r, those of them that there are
struct NormFunction : torch::autograd::Function<NormFunction> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& residual, const Maybe& block, const Maybe& post,
                               const Maybe& gate, const Maybe& pre, double scale, double eps) {
    NormInputs in{residual, block.value_or(at::Tensor()), post.value_or(at::Tensor()), gate.value_or(at::Tensor()),
                  pre.value_or(at::Tensor())};
    const NormOutputs out = norm_forward(in, scale, eps, true);
    // (with a block the backward pass takes r and no values of the residual: it may be overwritten, and
    // where it is no leaf -- a leaf's accumulator, which the graph holds, holds the leaf --, go)
    ctx->save_for_backward({in.block.defined() ? out.r : residual, in.block, in.post, in.gate, in.pre, out.lengths});
    if (residual.is_leaf() && residual.requires_grad()) ctx->saved_data["leaf"] = residual;
    // (without a block the residual itself is what the norm took, and it is not multiplied)
    ctx->saved_data["scale"] = in.block.defined() ? scale : 1.0;
    ctx->set_materialize_grads(false);
    variable_list outputs;
    if (out.y.defined()) outputs.push_back(out.y);
    if (out.r.defined()) outputs.push_back(out.r);
    return outputs;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    NormInputs in{saved[0], saved[1], saved[2], saved[3], saved[4]};
    const bool norm = in.pre.defined();
    const at::Tensor dy = norm ? grads[0] : at::Tensor(), dr = in.block.defined() ? grads[norm ? 1 : 0] : at::Tensor();
    const auto leaf = ctx->saved_data.find("leaf");
    std::array<bool, 5> want;
    // (the context counts the inputs that are there)
    const at::Tensor* const inputs[5] = {&in.residual, &in.block, &in.post, &in.gate, &in.pre};
    for (int i = 0, at = 0; i < 5; i++) want[i] = inputs[i]->defined() && ctx->needs_input_grad(at++);
    variable_list out(7);
    {
      c10::AutoGradMode off(false);
      auto g = norm_backward(dy, dr, in, saved[5], ctx->saved_data["scale"].toDouble(),
                             leaf != ctx->saved_data.end() ? leaf->second.toTensor() : at::Tensor(), want);
      for (int i = 0; i < 5; i++) out[i] = g[i];
    }
    return once_differentiable(std::move(out), "residual_norm", {&grads, &saved});
  }
};

bool norm_arguments(PyObject* const* args, NormInputs* in) {
  const at::Tensor* const residual = tensor(args[0], "residual");
  if (!residual || !optional(args[1], "block", &in->block) || !optional(args[2], "post_weight", &in->post) ||
      !optional(args[3], "gate", &in->gate) || !optional(args[4], "pre_weight", &in->pre))
    return false;
  in->residual = *residual;
  return true;
}

// residual_norm(residual, block, post, gate, pre, scale, eps) -> (y, r); block, post, gate and pre may
// be None, and so are then r (without a block) and y (without pre)
PyObject* py_residual_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  NormInputs in;
  if (!takes(nargs, 7, "residual_norm") || !norm_arguments(args, &in)) return nullptr;
  refuse_tangents({&in.residual, &in.block, &in.post, &in.gate, &in.pre});
  if (looked_on({&in.residual, &in.block, &in.post, &in.gate, &in.pre})) Py_RETURN_NOTIMPLEMENTED;
  const double scale = PyFloat_AsDouble(args[5]), eps = PyFloat_AsDouble(args[6]);
  if (PyErr_Occurred()) return nullptr;
  NormOutputs out;
  {
    pybind11::gil_scoped_release unlocked;
    if (differentiated({&in.residual, &in.block, &in.post, &in.gate, &in.pre})) {
      const variable_list v = NormFunction::apply(in.residual, maybe(in.block), maybe(in.post),
                                                  maybe(in.gate), maybe(in.pre), scale, eps);
      if (in.pre.defined()) out.y = v[0];
      if (in.block.defined()) out.r = v.back();
    } else {
      out = norm_forward(in, scale, eps, false);
    }
  }
  return tuple_of({out.y, out.r});
  END_HANDLE_TH_ERRORS
}

// norm_lengths(... as residual_norm) -> (y, r, lengths) and norm_grads(dy, dr, r, block, post, gate, pre,
// lengths, scale, and which of the five are wanted) -> five gradients, None where not wanted and for what
// is None: the passes by themselves, for compilers
PyObject* py_norm_lengths(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  NormInputs in;
  if (!takes(nargs, 7, "norm_lengths") || !norm_arguments(args, &in)) return nullptr;
  const double scale = PyFloat_AsDouble(args[5]), eps = PyFloat_AsDouble(args[6]);
  if (PyErr_Occurred()) return nullptr;
  NormOutputs out;
  {
    pybind11::gil_scoped_release unlocked;
    out = norm_forward(in, scale, eps, true);
  }
  return tuple_of({out.y, out.r, out.lengths});
  END_HANDLE_TH_ERRORS
}

PyObject* py_norm_grads(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  NormInputs in;
  at::Tensor dy, dr;
  if (!takes(nargs, 14, "norm_grads") || !optional(args[0], "dy", &dy) || !optional(args[1], "dr", &dr) ||
      !norm_arguments(args + 2, &in))
    return nullptr;
  const at::Tensor* const lengths = tensor(args[7], "lengths");
  const double scale = PyFloat_AsDouble(args[8]);
  if (!lengths || PyErr_Occurred()) return nullptr;
  std::array<bool, 5> want;
  for (int i = 0; i < 5; i++)
    if (!to_bool(args[9 + i], &want[i])) return nullptr;
  std::array<at::Tensor, 5> g;
  {
    pybind11::gil_scoped_release unlocked;
    g = norm_backward(dy, dr, in, *lengths, scale, at::Tensor(), want);
  }
  return tuple_of({g[0], g[1], g[2], g[3], g[4]});
  END_HANDLE_TH_ERRORS
}

// What the conversion kernels may take: plain tensors on one GPU, 16-byte aligned,
// without gradients.  (That nothing looks on is the caller's to know.)
//
// Bound: host time for layers up to about 3000 x 3000; the two kernels of a
// 1024 x 1024 one take 12 us, the same checks in Python and two calls through
// ctypes took 32 for quantising and packing, here 17 (4096 x 4096: 38.8 -> 33.3).
const at::Tensor* plain(PyObject* o) {
  return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
}
bool convertible(const at::Tensor& t, const at::Device& dev) {
  return t.device() == dev && !t.is_neg() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0 &&
         !(t.requires_grad() && c10::GradMode::is_enabled());
}
// 1 launched, 0 not a problem for the kernels, -1 with an exception set
int converted(int rc) {
  if (rc == MARLIN_OK) return 1;
  if (rc == MARLIN_ERR_PROB_SHAPE) return 0;
  PyErr_Format(PyExc_RuntimeError, "weight conversion failed with code %d: %s", rc,
               marlin_amd_convert_last_error());
  return -1;
}

// quantize(w, groupsize) -> (fake, q, s), or None where the tensor operations have to do it
PyObject* py_quantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  int gs;
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "quantize takes 2 arguments");
    return nullptr;
  }
  const at::Tensor* const pw = plain(args[0]);
  if (!to_int(args[1], &gs)) {  // what else a group size may be, the tensor operations say
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (!pw || pw->dim() != 2 || pw->scalar_type() != at::kHalf || !pw->is_cuda() || pw->numel() == 0)
    Py_RETURN_NONE;
  const at::Tensor& w = *pw;
  const int64_t k = w.size(0), n = w.size(1);
  if (gs == -1 && k == (int)k) gs = (int)k;
  const bool by_column = !w.is_contiguous();
  if (gs <= 0 || k % gs != 0 || k != (int)k || n != (int)n || !convertible(w, w.device()) ||
      (by_column ? !(w.stride(0) == 1 && w.stride(1) == k && gs % 4 == 0) : n % 4 != 0))
    Py_RETURN_NONE;
  const int dev = w.get_device();
  void* const st = current_stream(dev);
  at::Tensor fake, q, s;
  int rc;
  {
    pybind11::gil_scoped_release unlocked;
    const auto plain_options = w.options().requires_grad(false);
    fake = at::empty_like(w, plain_options, at::MemoryFormat::Preserve);
    q = at::empty_like(fake, plain_options.dtype(at::kInt), at::MemoryFormat::Preserve);
    s = at::empty({k / gs, n}, plain_options);
    rc = marlin_amd_quantize(w.data_ptr(), (int)k, (int)n, gs, by_column, fake.data_ptr(), q.data_ptr(),
                             s.data_ptr(), dev, st);
  }
  const int done = converted(rc);
  if (done < 0) return nullptr;
  if (done == 0) Py_RETURN_NONE;
  PyObject* const out[3] = {THPVariable_Wrap(std::move(fake)), THPVariable_Wrap(std::move(q)),
                            THPVariable_Wrap(std::move(s))};
  PyObject* const tuple = PyTuple_New(3);
  if (!tuple) return nullptr;
  for (int i = 0; i < 3; i++) PyTuple_SET_ITEM(tuple, i, out[i]);
  return tuple;
  END_HANDLE_TH_ERRORS
}

// whether `read` has no bytes between the first and the last of the contiguous `written`: a
// kernel would read what it is overwriting, the tensor operations read everything first
bool apart(const at::Tensor& written, const at::Tensor& read) {
  const char* const lo = (const char*)written.data_ptr();
  const char* const hi = lo + written.numel() * written.element_size();
  int64_t last = 0;
  for (int64_t d = 0; d < read.dim(); d++) last += (read.size(d) - 1) * read.stride(d);
  const char* const at = (const char*)read.data_ptr();
  return at >= hi || at + (last + 1) * read.element_size() <= lo;
}

// pack(w (k, n), s (groups, n), B, packed, k, n, groupsize or -1) -> whether B and the packed
// scales have been written; False where the tensor operations have to do it
PyObject* py_pack(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  int k, n, gs;
  if (nargs != 7) {
    PyErr_SetString(PyExc_TypeError, "pack takes 7 arguments");
    return nullptr;
  }
  const at::Tensor *pw = plain(args[0]), *ps = plain(args[1]), *pb = plain(args[2]), *pp = plain(args[3]);
  if (!to_int(args[4], &k) || !to_int(args[5], &n) || !to_int(args[6], &gs)) {
    PyErr_Clear();
    Py_RETURN_FALSE;
  }
  if (!pw || !ps || !pb || !pp || !pw->is_cuda() || (gs <= 0 && gs != -1)) Py_RETURN_FALSE;
  const at::Tensor &w = *pw, &s = *ps, &B = *pb, &packed = *pp;
  const auto is = [](const at::Tensor& t, at::ScalarType type, int64_t rows, int64_t columns) {
    return t.scalar_type() == type && t.dim() == 2 && t.size(0) == rows && t.size(1) == columns;
  };
  const int64_t groups = gs == -1 ? 1 : k / gs;
  const bool by_column = !w.is_contiguous();
  const at::Device on = w.device();
  if (!is(w, at::kHalf, k, n) || !is(s, at::kHalf, groups, n) || !is(packed, at::kHalf, groups, n) ||
      !is(B, at::kInt, k / 16, 2 * (int64_t)n) || (by_column && !(w.stride(0) == 1 && w.stride(1) == k)) ||
      !B.is_contiguous() || !packed.is_contiguous() || !convertible(w, on) || !convertible(B, on) ||
      !convertible(packed, on) || s.device() != on || s.requires_grad() || s.is_neg() ||
      // (writes to inference tensors elsewhere are refused by the tensor operations)
      (!c10::InferenceMode::is_enabled() && (B.is_inference() || packed.is_inference())) ||
      !apart(B, w) || !apart(B, s) || !apart(B, packed) || !apart(packed, w) || !apart(packed, s))
    Py_RETURN_FALSE;
  const int dev = w.get_device();
  void* const st = current_stream(dev);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = marlin_amd_pack(w.data_ptr(), k, n, gs, by_column, s.data_ptr(), s.stride(0), s.stride(1),
                       B.data_ptr(), packed.data_ptr(), dev, st);
  Py_END_ALLOW_THREADS
  const int done = converted(rc);
  if (done < 0) return nullptr;
  if (done == 0) Py_RETURN_FALSE;
  // written in place, as an assignment to them would be
  for (const at::Tensor* t : {&B, &packed})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"mul", (PyCFunction)(void (*)(void))py_mul, METH_FASTCALL, nullptr},
    {"linear", (PyCFunction)(void (*)(void))py_linear, METH_FASTCALL, nullptr},
    {"residual_norm", (PyCFunction)(void (*)(void))py_residual_norm, METH_FASTCALL, nullptr},
    {"norm_grads", (PyCFunction)(void (*)(void))py_norm_grads, METH_FASTCALL, nullptr},
    {"gated_dense", (PyCFunction)(void (*)(void))py_gated_dense, METH_FASTCALL, nullptr},
    {"gated_grads", (PyCFunction)(void (*)(void))py_gated_grads, METH_FASTCALL, nullptr},
    {"linear_dense", (PyCFunction)(void (*)(void))py_linear_dense, METH_FASTCALL, nullptr},
    {"linear_full", (PyCFunction)(void (*)(void))py_linear_full, METH_FASTCALL, nullptr},
    {"linear_full_kept", (PyCFunction)(void (*)(void))py_linear_full_kept<Keep::kSlopes>, METH_FASTCALL, nullptr},
    {"linear_full_slopes", (PyCFunction)(void (*)(void))py_linear_full_kept<Keep::kSteps>, METH_FASTCALL, nullptr},
    {"linear_full_grads", (PyCFunction)(void (*)(void))py_linear_full_grads, METH_FASTCALL, nullptr},
    {"dropout", (PyCFunction)(void (*)(void))py_dropout, METH_FASTCALL, nullptr},
    {"dropout_grad", (PyCFunction)(void (*)(void))py_dropout_grad, METH_FASTCALL, nullptr},
    {"gated_sums", (PyCFunction)(void (*)(void))py_gated_sums, METH_FASTCALL, nullptr},
    {"norm_lengths", (PyCFunction)(void (*)(void))py_norm_lengths, METH_FASTCALL, nullptr},
    {"linear_grads", (PyCFunction)(void (*)(void))py_linear_grads, METH_FASTCALL, nullptr},
    {"gated_mul", (PyCFunction)(void (*)(void))py_gated_mul, METH_FASTCALL, nullptr},
    {"gated_linear", (PyCFunction)(void (*)(void))py_gated_linear, METH_FASTCALL, nullptr},
    {"without_gradients", (PyCFunction)(void (*)(void))py_without_gradients, METH_FASTCALL, nullptr},
    {"quantize", (PyCFunction)(void (*)(void))py_quantize, METH_FASTCALL, nullptr},
    {"pack", (PyCFunction)(void (*)(void))py_pack, METH_FASTCALL, nullptr},
    {"dense", (PyCFunction)(void (*)(void))py_dense, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_marlin_torch", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__marlin_torch(void) { return PyModule_Create(&module); }
