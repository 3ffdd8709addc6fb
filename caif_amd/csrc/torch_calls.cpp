// Native side of caif_amd/torch_ops.py: the per-call work around an entry point of the C ABI (argument checks, result and
// workspace allocation, current stream) for torch tensors.  In Python that work took 8.5 us of a call whose launch costs
// the host 3 to 4 us: a one-row linear of 1408 x 2048 (2.9 MB of weight) took 12.1 us a call, bound by the host; from here
// it takes 6.5 (host 5.1).
//
// The entry points are the ones the ctypes layer has loaded (caif_amd/capi.py hands their addresses to bind()), so there
// is one copy of libcaifx.so in the process and no state here besides those addresses.  A non-zero status is returned as a
// Python int; the caller turns it into the exception.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <initializer_list>
#include <stdexcept>
#include <vector>

#include "caifx.h"

namespace {

// ------------------------------------------------------------------ entry points
#define ENTRIES(X)                                                                                                      \
  X(caifx_qlinear_forward) X(caifx_qlinear_forward_add) X(caifx_qlinear_backward_input)                                  \
  X(caifx_qlinear_backward_input_add) X(caifx_qlinear_workspace_bytes) X(caifx_qlinear_grouped_forward)                  \
  X(caifx_qlinear_grouped_backward_input) X(caifx_qlinear_grouped_backward_input_add)                                    \
  X(caifx_qlinear_grouped_workspace_bytes) X(caifx_qlinear_grouped_fresh) X(caifx_silu) X(caifx_silu_backward) X(caifx_multiply) X(caifx_add)           \
  X(caifx_silu_multiply) X(caifx_swiglu_backward) X(caifx_moe_dispatch_map_workspace_bytes)                              \
  X(caifx_moe_build_dispatch_map) X(caifx_moe_dispatch) X(caifx_moe_combine) X(caifx_moe_combine_backward_grad_expert)   \
  X(caifx_moe_combine_backward_grad_weights) X(caifx_moe_dispatch_backward) X(caifx_moe_dispatch_fresh)                  \
  X(caifx_moe_combine_backward_grad_expert_fresh) X(caifx_quantize_int8_per_channel)           \
  X(caifx_quantize_int8_per_tensor) X(caifx_quantize_to_int4) X(caifx_adapters_forward) X(caifx_adapters_backward)         \
  X(caifx_adapters_workspace_bytes) X(caifx_checkpoint_pack) X(caifx_checkpoint_unpack) X(caifx_silu_multiply_checkpoint)   \
  X(caifx_swiglu_backward_checkpoint) X(caifx_mxfp4_quantize) X(caifx_mxfp4_dequantize) X(caifx_mxfp4_matmul)               \
  X(caifx_mxfp4_matmul_workspace_bytes) X(caifx_gated_forward) X(caifx_gated_backward) X(caifx_gated_workspace_bytes)

struct Api {
#define X(name) decltype(&::name) name = nullptr;
  ENTRIES(X)
#undef X
} api;

PyObject *bind(PyObject *, PyObject *table)
{
  // every address is looked up before any is taken
  Api fresh;
#define X(name)                                                                                   \
  {                                                                                               \
    PyObject *v = PyDict_GetItemString(table, #name);                                             \
    const unsigned long long p = v ? PyLong_AsUnsignedLongLong(v) : 0;                            \
    if (p == 0 || PyErr_Occurred()) {                                                             \
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "missing entry point " #name);   \
      return nullptr;                                                                             \
    }                                                                                             \
    fresh.name = reinterpret_cast<decltype(&::name)>(p);                                          \
  }
  ENTRIES(X)
#undef X
  api = fresh;
  Py_RETURN_NONE;
}

// ------------------------------------------------------------------ arguments
struct Error {
  PyObject *type;
  const char *what;
};

const at::Tensor &tensor(PyObject *o)
{
  if (!THPVariable_Check(o)) throw Error{PyExc_TypeError, "expected a torch tensor"};
  return THPVariable_Unpack(o);
}

// device memory, contiguous: the C ABI sees raw pointers
const at::Tensor &device_tensor(PyObject *o)
{
  const at::Tensor &t = tensor(o);
  if (!t.is_cuda()) throw Error{PyExc_RuntimeError, "host backend not supported"};
  if (!t.is_contiguous()) throw Error{PyExc_RuntimeError, "tensor must be contiguous"};
  return t;
}

int64_t integer(PyObject *o)
{
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Error{nullptr, nullptr};
  return v;
}

int code_of(at::ScalarType t)
{
  switch (t) {
    case at::kFloat: return CAIFX_F32;
    case at::kHalf: return CAIFX_F16;
    case at::kBFloat16: return CAIFX_BF16;
    default: throw Error{PyExc_KeyError, "tensor must be fp32, fp16 or bf16"};
  }
}

at::ScalarType type_of(int64_t code)
{
  switch (code) {
    case CAIFX_F32: return at::kFloat;
    case CAIFX_F16: return at::kHalf;
    case CAIFX_BF16: return at::kBFloat16;
    default: throw Error{PyExc_KeyError, "unknown dtype code"};
  }
}

// an attribute of a Python weight object; names are interned once
struct Attr {
  PyObject *name;
  explicit Attr(const char *s) : name(PyUnicode_InternFromString(s)) {}
};

struct Owned {
  PyObject *p;
  explicit Owned(PyObject *q) : p(q)
  {
    if (!p) throw Error{nullptr, nullptr};
  }
  ~Owned() { Py_DECREF(p); }
  Owned(const Owned &) = delete;
  Owned &operator=(const Owned &) = delete;
};

int64_t int_attr(PyObject *o, const Attr &a) { return integer(Owned(PyObject_GetAttr(o, a.name)).p); }

// data pointer of a tensor attribute, null for None (the weight object keeps the tensor alive)
void *ptr_attr(PyObject *o, const Attr &a)
{
  Owned v(PyObject_GetAttr(o, a.name));
  return v.p == Py_None ? nullptr : tensor(v.p).data_ptr();
}

struct WeightAttrs {
  Attr wq{"wq"}, scales{"scales"}, wq_ptrs{"wq_ptrs"}, scales_ptrs{"scales_ptrs"}, weights{"weights"}, n{"N"}, k{"K"},
      kind{"w_kind"}, period{"scale_period"}, group{"group_size"};
};
const WeightAttrs &attrs()
{
  static const WeightAttrs a;
  return a;
}

// the launch itself without the interpreter lock: it can wait for room in the queue.  It takes the entry point and its
// arguments, so whatever can throw (sizes, data pointers, the stream) is evaluated while the lock is held.
struct Unlocked {
  PyThreadState *state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};
template <typename... P, typename... A> int launch(int (*entry)(P...), A... args)
{
  const Unlocked without_lock;
  return entry(args...);
}

void *stream() { return static_cast<void *>(c10::hip::getCurrentHIPStream().stream()); }

at::Tensor bytes_like(const at::Tensor &x, size_t n)
{
  return at::empty({static_cast<int64_t>(n)}, x.options().dtype(at::kByte));
}

// the kernels write the caller's workspace by its address: anything but gapless memory of the input's device would be a fault
void check_workspace(PyObject *given, const at::Tensor &x)
{
  if (given == Py_None) return;
  const at::Tensor &t = tensor(given);
  if (t.numel() > 0 && (t.device() != x.device() || !t.is_contiguous()))
    throw Error{PyExc_ValueError, "the workspace must be contiguous and on the input's device"};
}

// the caller's workspace, or one of the size the library asks for (none for zero bytes)
struct Workspace {
  at::Tensor held;
  void *p = nullptr;
  size_t bytes = 0;
  template <typename Query> Workspace(PyObject *given, const at::Tensor &x, Query query)
  {
    if (given != Py_None) {
      const at::Tensor &t = tensor(given);
      p = t.data_ptr();
      bytes = static_cast<size_t>(t.numel());
    } else if ((bytes = query()) > 0) {
      // the workspace is optional: on a card that is full up to the result the calls run without it, as those kernels do that
      // never asked for one
      try {
        held = bytes_like(x, bytes);
        p = held.data_ptr();
      } catch (const c10::OutOfMemoryError &) {
        bytes = 0;
      }
    }
  }
};

PyObject *result(int status, const at::Tensor &t)
{
  if (status != CAIFX_OK) return PyLong_FromLong(status);
  return THPVariable_Wrap(t);
}

// argument count, C++ and Python errors
template <typename F> PyObject *guarded(Py_ssize_t have, Py_ssize_t want, F f)
{
  if (have != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, have);
    return nullptr;
  }
  try {
    return f();
  } catch (const Error &e) {
    if (e.type) PyErr_SetString(e.type, e.what);
    return nullptr;
  } catch (const c10::Error &e) {
    // torch's own out-of-memory type where there is one
    PyObject *type = PyExc_RuntimeError;
    if (std::strstr(e.what_without_backtrace(), "out of memory")) {
      PyObject *torch = PyImport_ImportModule("torch");
      PyObject *oom = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
      Py_XDECREF(torch);
      PyErr_Clear();
      if (oom) {
        PyErr_SetString(oom, e.what_without_backtrace());
        Py_DECREF(oom);
        return nullptr;
      }
    }
    PyErr_SetString(type, e.what_without_backtrace());
    return nullptr;
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// the codes and scales of a weight in microscaled 4 bits, [N, K]: the kernels take both sizes from N and K
void check_mxfp4(PyObject *w, int64_t N, int64_t K, const at::Tensor &x)
{
  const int64_t blocks = (K + CAIFX_MXFP4_BLOCK - 1) / CAIFX_MXFP4_BLOCK;
  Owned codes(PyObject_GetAttr(w, attrs().wq.name)), scales(PyObject_GetAttr(w, attrs().scales.name));
  const at::Tensor &c = device_tensor(codes.p), &s = device_tensor(scales.p);
  if (c.scalar_type() != at::kByte || s.scalar_type() != at::kByte || c.numel() != N * 16 * blocks || s.numel() != N * blocks)
    throw Error{PyExc_ValueError, "a W_MXFP4 weight's codes are uint8 [N, 16 * ceil(K / 32)], its scales uint8 [N, ceil(K / 32)]"};
  if (c.device() != x.device() || s.device() != x.device()) throw Error{PyExc_RuntimeError, "tensors must be on one device"};
}

// ------------------------------------------------------------------ frozen linear
// qlinear(backward, x, weight, compute_dtype, out_dtype, out, workspace, addend) -> result or status
PyObject *qlinear(PyObject *, PyObject *const *a, Py_ssize_t n)
{
  return guarded(n, 8, [&]() -> PyObject * {
    const bool backward = integer(a[0]) != 0;
    const at::Tensor &x = device_tensor(a[1]);
    PyObject *w = a[2];
    const WeightAttrs &at_ = attrs();
    const int64_t N = int_attr(w, at_.n), K = int_attr(w, at_.k);
    const int64_t in = backward ? N : K, out_dim = backward ? K : N;
    if (in <= 0) throw Error{PyExc_ValueError, "the weight has no elements"};
    const int64_t M = x.numel() / in;
    const int compute = static_cast<int>(integer(a[3])), od = static_cast<int>(integer(a[4]));
    const int xd = code_of(x.scalar_type());
    const int kind = static_cast<int>(int_attr(w, at_.kind));
    const int64_t period = int_attr(w, at_.period);
    const int group = static_cast<int>(int_attr(w, at_.group));
    check_workspace(a[6], x);
    c10::OptionalDeviceGuard guard;
    if (kind == CAIFX_W_MXFP4) {
      check_mxfp4(w, N, K, x);
      if (x.numel() != M * in) throw Error{PyExc_ValueError, "the input's size is not a multiple of the reduction length"};
      for (const int i : {5, 7})
        if (a[i] != Py_None && (device_tensor(a[i]).numel() != M * out_dim || tensor(a[i]).scalar_type() != type_of(od) || tensor(a[i]).device() != x.device()))
          throw Error{PyExc_ValueError, "the result and the addend must have the result's dtype and rows x columns elements, on the input's device"};
      guard.reset_device(x.device());
    }
    const void *wq = ptr_attr(w, at_.wq), *scales = ptr_attr(w, at_.scales);
    const at::Tensor y = a[5] != Py_None ? tensor(a[5]) : at::empty({M, out_dim}, x.options().dtype(type_of(od)));
    const Workspace ws(a[6], x, [&] { return api.caifx_qlinear_workspace_bytes(M, N, K, xd, compute, kind, backward ? 1 : 0); });
    if (a[7] != Py_None) {
      const at::Tensor &add = tensor(a[7]);
      if (add.scalar_type() != y.scalar_type() || add.numel() != y.numel())
        throw Error{PyExc_AssertionError, "the addend must have the result's dtype and size"};
      const auto fn = backward ? api.caifx_qlinear_backward_input_add : api.caifx_qlinear_forward_add;
      return result(launch(fn, M, N, K, x.data_ptr(), xd, compute, wq, kind, scales, period, group, y.data_ptr(), od, add.data_ptr(), ws.p, ws.bytes, stream()), y);
    }
    const auto fn = backward ? api.caifx_qlinear_backward_input : api.caifx_qlinear_forward;
    return result(launch(fn, M, N, K, x.data_ptr(), xd, compute, wq, kind, scales, period, group, y.data_ptr(), od, ws.p, ws.bytes, stream()), y);
  });
}

// grouped(backward, x, offsets, weights, compute_dtype, out_dtype, out, workspace, addend) -> result or status
PyObject *grouped(PyObject *, PyObject *const *a, Py_ssize_t n)
{
  return guarded(n, 9, [&]() -> PyObject * {
    const bool backward = integer(a[0]) != 0;
    const at::Tensor &x = device_tensor(a[1]);
    const at::Tensor &offsets = device_tensor(a[2]);
    PyObject *w = a[3];
    const WeightAttrs &at_ = attrs();
    const int64_t N = int_attr(w, at_.n), K = int_attr(w, at_.k);
    const int64_t in = backward ? N : K, out_dim = backward ? K : N;
    if (in <= 0) throw Error{PyExc_ValueError, "the weight has no elements"};
    const int64_t rows = x.numel() / in;
    const int compute = static_cast<int>(integer(a[4])), od = static_cast<int>(integer(a[5]));
    const int xd = code_of(x.scalar_type());
    const int kind = static_cast<int>(int_attr(w, at_.kind));
    Owned list(PyObject_GetAttr(w, at_.weights.name));
    const Py_ssize_t E = PySequence_Size(list.p);
    if (E < 0) throw Error{nullptr, nullptr};
    // sizes and dtypes are checked here, before anything is launched
    check_workspace(a[7], x);
    if (x.numel() != rows * in) throw Error{PyExc_ValueError, "the input's size is not a multiple of the reduction length"};
    if (offsets.scalar_type() != at::kInt || offsets.numel() != E + 1) throw Error{PyExc_ValueError, "offsets must be int32 [experts + 1]"};
    if (a[6] != Py_None) {
      const at::Tensor &o = device_tensor(a[6]);
      if (o.scalar_type() != type_of(od) || o.numel() != rows * out_dim)
        throw Error{PyExc_ValueError, "the result tensor must have the result's dtype and rows x columns elements"};
    }
    const at::Tensor y = a[6] != Py_None ? tensor(a[6]) : at::empty({rows, out_dim}, x.options().dtype(type_of(od)));
    const int64_t period = int_attr(w, at_.period);
    const int group = static_cast<int>(int_attr(w, at_.group));
    const auto wq = static_cast<const void *const *>(ptr_attr(w, at_.wq_ptrs));
    const auto scales = static_cast<const void *const *>(ptr_attr(w, at_.scales_ptrs));
    const Workspace ws(a[7], x, [&] {
      return api.caifx_qlinear_grouped_workspace_bytes(static_cast<int>(E), rows, N, K, xd, compute, kind, backward ? 1 : 0);
    });
    const auto off = static_cast<const int32_t *>(offsets.data_ptr());
    const void *addend = nullptr;
    if (a[8] != Py_None) {
      if (!backward) throw Error{PyExc_AssertionError, "the forward takes no addend"};
      const at::Tensor &add = tensor(a[8]);
      if (add.scalar_type() != y.scalar_type() || add.numel() != y.numel())
        throw Error{PyExc_AssertionError, "the addend must have the result's dtype and size"};
      addend = add.data_ptr();
    }
    // a fresh result's rows outside the segments are zero
    if (a[6] == Py_None)
      return result(launch(api.caifx_qlinear_grouped_fresh, backward ? 1 : 0, static_cast<int>(E), off, rows, N, K, x.data_ptr(), xd, compute, wq, kind, scales,
                           period, group, y.data_ptr(), od, addend, ws.p, ws.bytes, stream()), y);
    if (addend) {
      return result(launch(api.caifx_qlinear_grouped_backward_input_add, static_cast<int>(E), off, rows, N, K, x.data_ptr(), xd, compute, wq, kind, scales,
                                                                 period, group, y.data_ptr(), od, addend, ws.p, ws.bytes, stream()), y);
    }
    const auto fn = backward ? api.caifx_qlinear_grouped_backward_input : api.caifx_qlinear_grouped_forward;
    return result(launch(fn, static_cast<int>(E), off, rows, N, K, x.data_ptr(), xd, compute, wq, kind, scales, period, group, y.data_ptr(), od, ws.p,
                     ws.bytes, stream()), y);
  });
}

PyObject *pair(int status, const at::Tensor &x, const at::Tensor &y)
{
  if (status != CAIFX_OK) return PyLong_FromLong(status);
  Owned p(THPVariable_Wrap(x)), q(THPVariable_Wrap(y));
  return PyTuple_Pack(2, p.p, q.p);
}

// ------------------------------------------------------------------ quantise
// quantize_int8(x, per_channel) -> (codes, scales) or status
PyObject *quantize_int8(PyObject *, PyObject *const *a, Py_ssize_t n)
{
  return guarded(n, 2, [&]() -> PyObject * {
    const at::Tensor &x = device_tensor(a[0]);
    if (x.scalar_type() != at::kFloat) throw Error{PyExc_RuntimeError, "QuantizeInt8: input must be fp32"};
    const int per_channel = PyObject_IsTrue(a[1]);
    if (per_channel < 0) throw Error{nullptr, nullptr};
    if (per_channel && x.dim() != 2) throw Error{PyExc_RuntimeError, "QuantizeInt8 PerChannel: input must be 2D"};
    const at::Tensor q = at::empty(x.sizes(), x.options().dtype(at::kChar));
    const at::Tensor s = at::empty({per_channel ? x.size(1) : 1}, x.options());
    const auto in = static_cast<const float *>(x.data_ptr());
    if (!per_channel) return pair(launch(api.caifx_quantize_int8_per_tensor, in, q.data_ptr(), s.data_ptr(), x.numel(), stream()), q, s);
    const int64_t rows = x.size(0), cols = x.size(1);
    if (rows > INT32_MAX || cols > INT32_MAX) throw Error{PyExc_OverflowError, "QuantizeInt8 PerChannel: too many rows or columns"};
    return pair(launch(api.caifx_quantize_int8_per_channel, in, q.data_ptr(), s.data_ptr(), static_cast<int>(rows), static_cast<int>(cols), stream()), q, s);
  });
}

// quantize_int4(x, group_size) -> (packed, fp16 scales) or status
PyObject *quantize_int4(PyObject *, PyObject *const *a, Py_ssize_t n)
{
  return guarded(n, 2, [&]() -> PyObject * {
    const at::Tensor &x = device_tensor(a[0]);
    if (x.scalar_type() != at::kFloat) throw Error{PyExc_RuntimeError, "QuantizeInt4PerGroup: input must be fp32"};
    const int64_t group = integer(a[1]), count = x.numel();
    if (group == 0) throw Error{PyExc_RuntimeError, "QuantizeInt4PerGroup: group_size must be > 0"};
    if (group > INT32_MAX || group < INT32_MIN) throw Error{PyExc_OverflowError, "QuantizeInt4PerGroup: group_size out of range"};
    const int64_t groups = group > 0 ? (count + group - 1) / group : 0;      // a negative size is the library's error
    const at::Tensor packed = at::empty({(count + 1) / 2}, x.options().dtype(at::kByte));
    const at::Tensor s = at::empty({groups}, x.options().dtype(at::kHalf));
    return pair(launch(api.caifx_quantize_to_int4, static_cast<const float *>(x.data_ptr()), packed.data_ptr(), s.data_ptr(), count, static_cast<int>(group), stream()), packed, s);
  });
}

// ------------------------------------------------------------------ element-wise
// elementwise(op, a, b or None, out or None): 0 silu, 1 silu_backward, 2 multiply, 3 add, 4 silu_multiply
PyObject *elementwise(PyObject *, PyObject *const *a, Py_ssize_t n)
{
  return guarded(n, 4, [&]() -> PyObject * {
    const at::Tensor &x = device_tensor(a[1]);
    const void *b = a[2] == Py_None ? nullptr : device_tensor(a[2]).data_ptr();
    if (a[3] != Py_None) {
      const at::Tensor &o = tensor(a[3]);
      if (!o.is_cuda()) throw Error{PyExc_RuntimeError, "host backend not supported"};
      if (o.scalar_type() != x.scalar_type() || o.numel() != x.numel() || !o.is_contiguous())
        throw Error{o.is_contiguous() ? PyExc_ValueError : PyExc_RuntimeError,
                    o.is_contiguous() ? "out must be a contiguous tensor of the input's dtype and size" : "tensor must be contiguous"};
    }
    const at::Tensor y = a[3] != Py_None ? tensor(a[3]) : at::empty_like(x);
    const int dt = code_of(x.scalar_type());
    const int64_t op = integer(a[0]);
    if (op == 0) return result(launch(api.caifx_silu, x.data_ptr(), y.data_ptr(), x.numel(), dt, stream()), y);
    const auto fn = op == 1 ? api.caifx_silu_backward : op == 2 ? api.caifx_multiply : op == 3 ? api.caifx_add : api.caifx_silu_multiply;
    return result(launch(fn, x.data_ptr(), b, y.data_ptr(), x.numel(), dt, stream()), y);
  });
}

// swiglu_backward(gate, up, grad_hidden, out_gate, out_up) -> (grad_gate, grad_up) or status
PyObject *swiglu_backward(PyObject *, PyObject *const *a, Py_ssize_t n)
{
  return guarded(n, 5, [&]() -> PyObject * {
    const at::Tensor &gate = device_tensor(a[0]), &up = device_tensor(a[1]), &gh = device_tensor(a[2]);
    if (gate.sizes() != up.sizes() || gate.sizes() != gh.sizes() || gate.scalar_type() != up.scalar_type() || gate.scalar_type() != gh.scalar_type())
      throw Error{PyExc_AssertionError, "gate, up and grad_hidden must have one shape and dtype"};
    const at::Tensor gg = a[3] != Py_None ? tensor(a[3]) : at::empty_like(gate);
    const at::Tensor gu = a[4] != Py_None ? tensor(a[4]) : at::empty_like(gate);
    const int dt = code_of(gate.scalar_type());
    const int st = launch(api.caifx_swiglu_backward, gate.data_ptr(), up.data_ptr(), gh.data_ptr(), gg.data_ptr(), gu.data_ptr(), gate.numel(), dt, stream());
    if (st != CAIFX_OK) return PyLong_FromLong(st);
    Owned p(THPVariable_Wrap(gg)), q(THPVariable_Wrap(gu));
    return PyTuple_Pack(2, p.p, q.p);
  });
}

// ------------------------------------------------------------------ MoE token routing
// moe_build_dispatch_map(expert_indices, num_experts, capacity) -> (map, offsets) or status
PyObject *moe_build_dispatch_map(PyObject *, PyObject *const *a, Py_ssize_t n)
{
  return guarded(n, 3, [&]() -> PyObject * {
    const at::Tensor &ids = device_tensor(a[0]);
    if (ids.scalar_type() != at::kInt || ids.dim() != 2) throw Error{PyExc_AssertionError, "expert_indices must be int32 [tokens, top_k]"};
    const int64_t tokens = ids.size(0);
    const int top_k = static_cast<int>(ids.size(1)), E = static_cast<int>(integer(a[1]));
    const at::Tensor map = at::empty_like(ids);
    const at::Tensor offsets = at::empty({E + 1}, ids.options());
    size_t nb = api.caifx_moe_dispatch_map_workspace_bytes(tokens, top_k, E);
    if (nb < 4 * static_cast<size_t>(E)) nb = 4 * static_cast<size_t>(E);
    const at::Tensor ws = bytes_like(ids, nb);
    const int capacity = static_cast<int>(integer(a[2]));
    return pair(launch(api.caifx_moe_build_dispatch_map, static_cast<const int32_t *>(ids.data_ptr()), tokens, top_k, E, capacity,
                                                 static_cast<int32_t *>(map.data_ptr()), static_cast<int32_t *>(offsets.data_ptr()), ws.data_ptr(),
                                                 nb, stream()), map, offsets);
  });
}

// rows x columns: the tensor that gives the number of tokens has no other rank
const at::Tensor &matrix(const at::Tensor &t)
{
  if (t.dim() != 2) throw Error{PyExc_ValueError, "expected a two-dimensional tensor"};
  return t;
}

// the second extent of a tensor of two dimensions or more
int64_t columns(const at::Tensor &t)
{
  if (t.dim() < 2) throw Error{PyExc_IndexError, "expected a tensor of at least two dimensions"};
  return t.size(1);
}

const int32_t *ints(PyObject *o) { return static_cast<const int32_t *>(device_tensor(o).data_ptr()); }

// moe_dispatch(x, ids, map, offsets, total_rows, out)
PyObject *moe_dispatch(PyObject *, PyObject *const *a, Py_ssize_t n)
{
  return guarded(n, 6, [&]() -> PyObject * {
    const at::Tensor &x = device_tensor(a[0]), &ids = device_tensor(a[1]), &offsets = device_tensor(a[3]);
    const int64_t tokens = matrix(x).size(0), dim = x.size(1), top_k = columns(ids);
    const bool fresh = a[5] == Py_None;
    const at::Tensor buf = fresh ? at::empty({integer(a[4]), dim}, x.options()) : tensor(a[5]);
    const int32_t *i1 = ints(a[1]); const int32_t *i2 = ints(a[2]); const int32_t *i3 = ints(a[3]); const int dt = code_of(x.scalar_type());
    if (fresh)
      return result(launch(api.caifx_moe_dispatch_fresh, x.data_ptr(), i1, i2, i3, buf.data_ptr(), buf.size(0), tokens, dim,
                                               static_cast<int>(top_k), static_cast<int>(offsets.numel() - 1), dt, stream()), buf);
    return result(launch(api.caifx_moe_dispatch, x.data_ptr(), i1, i2, i3, buf.data_ptr(), tokens, dim,
                                         static_cast<int>(top_k), static_cast<int>(offsets.numel() - 1), dt, stream()), buf);
  });
}

// moe_combine(expert_buffer, ids, weights, map, offsets, out)
PyObject *moe_combine(PyObject *, PyObject *const *a, Py_ssize_t n)
{
  return guarded(n, 6, [&]() -> PyObject * {
    const at::Tensor &buf = device_tensor(a[0]), &ids = device_tensor(a[1]), &w = device_tensor(a[2]), &offsets = device_tensor(a[4]);
    const int64_t tokens = matrix(ids).size(0), dim = columns(buf), top_k = ids.size(1);
    const at::Tensor y = a[5] != Py_None ? tensor(a[5]) : at::empty({tokens, dim}, buf.options());
    const int32_t *i1 = ints(a[1]); const int32_t *i3 = ints(a[3]); const int32_t *i4 = ints(a[4]); const int dt = code_of(buf.scalar_type());
    return result(launch(api.caifx_moe_combine, buf.data_ptr(), i1, w.data_ptr(), i3, i4, y.data_ptr(), tokens, dim,
                                        static_cast<int>(top_k), static_cast<int>(offsets.numel() - 1), dt, stream()), y);
  });
}

// moe_combine_backward_grad_expert(grad_output, ids, weights, map, offsets, total_rows, out)
PyObject *moe_combine_backward_grad_expert(PyObject *, PyObject *const *a, Py_ssize_t n)
{
  return guarded(n, 7, [&]() -> PyObject * {
    const at::Tensor &g = device_tensor(a[0]), &ids = device_tensor(a[1]), &w = device_tensor(a[2]), &offsets = device_tensor(a[4]);
    const int64_t tokens = matrix(g).size(0), dim = g.size(1), top_k = columns(ids);
    const bool fresh = a[6] == Py_None;
    const at::Tensor buf = fresh ? at::empty({integer(a[5]), dim}, g.options()) : tensor(a[6]);
    const int32_t *i1 = ints(a[1]); const int32_t *i3 = ints(a[3]); const int32_t *i4 = ints(a[4]); const int dt = code_of(g.scalar_type());
    if (fresh)
      return result(launch(api.caifx_moe_combine_backward_grad_expert_fresh, g.data_ptr(), i1, w.data_ptr(), i3, i4, buf.data_ptr(), buf.size(0), tokens,
                                                                   dim, static_cast<int>(top_k), static_cast<int>(offsets.numel() - 1), dt, stream()), buf);
    return result(launch(api.caifx_moe_combine_backward_grad_expert, g.data_ptr(), i1, w.data_ptr(), i3, i4, buf.data_ptr(), tokens, dim,
                                                             static_cast<int>(top_k), static_cast<int>(offsets.numel() - 1),
                                                             dt, stream()), buf);
  });
}

// moe_dispatch_backward(grad_expert_buffer, ids, map, offsets, out)
PyObject *moe_dispatch_backward(PyObject *, PyObject *const *a, Py_ssize_t n)
{
  return guarded(n, 5, [&]() -> PyObject * {
    const at::Tensor &g = device_tensor(a[0]), &ids = device_tensor(a[1]), &offsets = device_tensor(a[3]);
    const int64_t tokens = matrix(ids).size(0), dim = columns(g), top_k = ids.size(1);
    const at::Tensor y = a[4] != Py_None ? tensor(a[4]) : at::empty({tokens, dim}, g.options());
    const int32_t *i1 = ints(a[1]); const int32_t *i2 = ints(a[2]); const int32_t *i3 = ints(a[3]); const int dt = code_of(g.scalar_type());
    return result(launch(api.caifx_moe_dispatch_backward, g.data_ptr(), i1, i2, i3, y.data_ptr(), tokens, dim,
                                                  static_cast<int>(top_k), static_cast<int>(offsets.numel() - 1), dt,
                                                  stream()), y);
  });
}

// moe_combine_backward_grad_weights(grad_output, expert_buffer, ids, map, offsets)
PyObject *moe_combine_backward_grad_weights(PyObject *, PyObject *const *a, Py_ssize_t n)
{
  return guarded(n, 5, [&]() -> PyObject * {
    const at::Tensor &g = device_tensor(a[0]), &buf = device_tensor(a[1]), &ids = device_tensor(a[2]), &offsets = device_tensor(a[4]);
    const int64_t tokens = matrix(ids).size(0), top_k = ids.size(1), dim = columns(g);
    const at::Tensor y = at::empty({tokens, top_k}, g.options());
    const int32_t *i2 = ints(a[2]); const int32_t *i3 = ints(a[3]); const int32_t *i4 = ints(a[4]); const int dt = code_of(g.scalar_type());
    return result(launch(api.caifx_moe_combine_backward_grad_weights, g.data_ptr(), buf.data_ptr(), i2, i3, i4, y.data_ptr(), tokens, dim,
                                                              static_cast<int>(top_k), static_cast<int>(offsets.numel() - 1),
                                                              dt, stream()), y);
  });
}

// ------------------------------------------------------------------ low-rank adapters, activation checkpoints
// These calls run on the device their first tensor lives on, whichever is current, and on that device's current stream.
struct Device {
  at::Device at;
  c10::DeviceGuard guard;
  explicit Device(const at::Tensor &t) : at(t.device()), guard(at) {}
  void *stream() const { return static_cast<void *>(c10::hip::getCurrentHIPStream(at.index()).stream()); }
  // device memory of this device, contiguous, of the type and number of elements that the call takes
  const at::Tensor &operand(PyObject *o, at::ScalarType type, int64_t elements, const char *what) const
  {
    const at::Tensor &t = device_tensor(o);
    if (t.device() != at) throw Error{PyExc_RuntimeError, "tensors must be on one device"};
    if (t.scalar_type() != type || t.numel() != elements) throw Error{PyExc_ValueError, what};
    return t;
  }
  const at::Tensor *optional(PyObject *o, at::ScalarType type, int64_t elements, const char *what) const
  {
    return o == Py_None ? nullptr : &operand(o, type, elements, what);
  }
};

void *data(const at::Tensor *t) { return t ? t->data_ptr() : nullptr; }

bool truth(PyObject *o)
{
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Error{nullptr, nullptr};
  return v != 0;
}

// the factors of the adapters: a [L, rank, K], b [L, N, rank]
struct Factors {
  int64_t L, rank, K, N;
  Factors(const Device &d, const at::Tensor &a, const at::Tensor &b, at::ScalarType type)
  {
    if (a.dim() != 3 || b.dim() != 3 || a.size(0) != b.size(0) || a.size(1) != b.size(2))
      throw Error{PyExc_ValueError, "the factors must be a [adapters, rank, K] and b [adapters, N, rank]"};
    if (a.scalar_type() != type || b.scalar_type() != type) throw Error{PyExc_ValueError, "the factors must have the activations' dtype"};
    if (a.device() != d.at || b.device() != d.at) throw Error{PyExc_RuntimeError, "tensors must be on one device"};
    L = a.size(0), rank = a.size(1), K = a.size(2), N = b.size(1);
    if (L > INT32_MAX || rank > INT32_MAX) throw Error{PyExc_OverflowError, "too many adapters"};
    if (a.numel() == 0 || b.numel() == 0) throw Error{PyExc_ValueError, "the factors have no elements"};
  }
};

int64_t rows_of(const at::Tensor &t, int64_t columns)
{
  if (t.dim() == 0 || t.size(t.dim() - 1) != columns) throw Error{PyExc_ValueError, "a row of activations must be as long as the factors' rows"};
  return t.numel() / columns;
}

// a result that the caller gives may be the base, place for place, and shares no memory with what else is read while it is written
void apart(const at::Tensor &out, const at::Tensor *base, std::initializer_list<const at::Tensor *> inputs)
{
  const auto from = [](const at::Tensor &t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); };
  const auto meet = [&](const at::Tensor &t) { return from(out) < from(t) + t.nbytes() && from(t) < from(out) + out.nbytes(); };
  bool wrong = base && from(*base) != from(out) && meet(*base);
  for (const at::Tensor *t : inputs) wrong = wrong || (t && meet(*t));
  if (wrong) throw Error{PyExc_ValueError, "out must be base itself or share no memory with the inputs"};
}

struct Scratch {
  at::Tensor held;
  size_t bytes;
  Scratch(const at::Tensor &x, size_t n) : bytes(n)
  {
    if (n > 0) held = bytes_like(x, n);
  }
  void *p() const { return bytes ? held.data_ptr() : nullptr; }
};

// adapters_forward(x, ids, a, b, scaling, base, keep_hidden, out) -> y, (y, hidden) or status
PyObject *adapters_forward(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  return guarded(n, 8, [&]() -> PyObject * {
    const at::Tensor &x = device_tensor(v[0]), &a = device_tensor(v[2]), &b = device_tensor(v[3]);
    const Device d(x);
    const int dt = code_of(x.scalar_type());
    const Factors f(d, a, b, x.scalar_type());
    const int64_t M = rows_of(x, f.K);
    const at::Tensor &ids = d.operand(v[1], at::kInt, M, "ids must be int32, one per row");
    const at::Tensor &scaling = d.operand(v[4], at::kFloat, f.L, "scaling must be fp32, one per adapter");
    const at::Tensor *base = d.optional(v[5], x.scalar_type(), M * f.N, "base must have the activations' dtype and rows x N elements");
    const bool keep = truth(v[6]);
    const at::Tensor *out = d.optional(v[7], x.scalar_type(), M * f.N, "out must have the activations' dtype and rows x N elements");
    if (out) apart(*out, base, {&x, &ids, &a, &b, &scaling});
    const at::Tensor y = out ? *out : at::empty({M, f.N}, x.options());
    const at::Tensor hidden = keep ? at::empty({M, f.rank}, x.options().dtype(at::kFloat)) : at::Tensor();
    const int L = static_cast<int>(f.L), r = static_cast<int>(f.rank);
    const Scratch ws(x, api.caifx_adapters_workspace_bytes(M, f.N, f.K, r, L, dt, 0));
    const int st = launch(api.caifx_adapters_forward, M, f.N, f.K, r, L, x.data_ptr(), static_cast<const int32_t *>(ids.data_ptr()), a.data_ptr(),
                          b.data_ptr(), static_cast<const float *>(scaling.data_ptr()), data(base), y.data_ptr(),
                          static_cast<float *>(keep ? hidden.data_ptr() : nullptr), dt, ws.p(), ws.bytes, d.stream());
    return keep ? pair(st, y, hidden) : result(st, y);
  });
}

// adapters_backward(dy, x or codes, scales or None, hidden, ids, a, b, scaling, base, need_dx, need_a, need_b, out) -> (dx, grad_a, grad_b), None for
// what is not needed, or status
PyObject *adapters_backward(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  return guarded(n, 13, [&]() -> PyObject * {
    const at::Tensor &dy = device_tensor(v[0]), &a = device_tensor(v[5]), &b = device_tensor(v[6]);
    const Device d(dy);
    const int dt = code_of(dy.scalar_type());
    const Factors f(d, a, b, dy.scalar_type());
    const int64_t M = rows_of(dy, f.N), groups = (f.K + CAIFX_CHECKPOINT_GROUP - 1) / CAIFX_CHECKPOINT_GROUP;
    const bool packed = v[2] != Py_None, need_x = truth(v[9]), need_a = truth(v[10]), need_b = truth(v[11]);
    // what no wanted result reads may be left out
    const at::Tensor *x = need_a || v[1] != Py_None
                              ? &d.operand(v[1], packed ? at::kChar : dy.scalar_type(), M * f.K,
                                           "x must have rows x K elements of the gradient's dtype, or be int8 codes with scales")
                              : nullptr;
    const at::Tensor *scales = d.optional(v[2], at::kFloat, M * groups, "the checkpoint's scales must be fp32, one per 128 values of a row");
    const at::Tensor *hidden = need_b || v[3] != Py_None ? &d.operand(v[3], at::kFloat, M * f.rank, "hidden must be fp32 [rows, rank]") : nullptr;
    const at::Tensor &ids = d.operand(v[4], at::kInt, M, "ids must be int32, one per row");
    const at::Tensor &scaling = d.operand(v[7], at::kFloat, f.L, "scaling must be fp32, one per adapter");
    const at::Tensor *base = d.optional(v[8], dy.scalar_type(), M * f.K, "base must have the gradient's dtype and rows x K elements");
    const at::Tensor *out = d.optional(v[12], dy.scalar_type(), M * f.K, "out must have the gradient's dtype and rows x K elements");
    if (out && !need_x) throw Error{PyExc_ValueError, "out is for dx, which is not needed"};
    if (out) apart(*out, base, {&dy, need_a ? x : nullptr, need_a ? scales : nullptr, need_b ? hidden : nullptr, &ids, &a, &b, &scaling});
    const at::Tensor dx = out ? *out : need_x ? at::empty({M, f.K}, dy.options()) : at::Tensor();
    const at::Tensor ga = need_a ? at::empty_like(a) : at::Tensor(), gb = need_b ? at::empty_like(b) : at::Tensor();
    const int L = static_cast<int>(f.L), r = static_cast<int>(f.rank);
    const Scratch ws(dy, api.caifx_adapters_workspace_bytes(M, f.N, f.K, r, L, dt, 1));
    const auto at = [](const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
    const int st = launch(api.caifx_adapters_backward, M, f.N, f.K, r, L, dy.data_ptr(), data(x), static_cast<const float *>(data(scales)),
                          static_cast<const float *>(data(hidden)), static_cast<const int32_t *>(ids.data_ptr()), a.data_ptr(), b.data_ptr(),
                          static_cast<const float *>(scaling.data_ptr()), data(base), at(dx), at(ga), at(gb), dt, ws.p(), ws.bytes, d.stream());
    if (st != CAIFX_OK) return PyLong_FromLong(st);
    const auto wrap = [](const at::Tensor &t) { return t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None); };
    Owned p(wrap(dx)), q(wrap(ga)), t(wrap(gb));
    return PyTuple_Pack(3, p.p, q.p, t.p);
  });
}

// rows and columns of an activation, and its checkpoint's tensors
struct Packed {
  int64_t rows = 0, cols = 0, groups = 0;
  explicit Packed(const at::Tensor &t)
  {
    if (t.dim() == 0) throw Error{PyExc_ValueError, "an activation has at least one dimension"};
    cols = t.size(t.dim() - 1);
    rows = cols > 0 ? t.numel() / cols : 0;
    groups = (cols + CAIFX_CHECKPOINT_GROUP - 1) / CAIFX_CHECKPOINT_GROUP;
  }
  static at::Tensor codes(const at::Tensor &like) { return at::empty(like.sizes(), like.options().dtype(at::kChar)); }
  at::Tensor scales(const at::Tensor &like) const
  {
    std::vector<int64_t> shape = like.sizes().vec();
    shape.back() = groups;
    return at::empty(shape, like.options().dtype(at::kFloat));
  }
};

float *floats(const at::Tensor &t) { return static_cast<float *>(t.data_ptr()); }

// checkpoint_pack(x) -> (codes, scales) or status
PyObject *checkpoint_pack(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  return guarded(n, 1, [&]() -> PyObject * {
    const at::Tensor &x = device_tensor(v[0]);
    const Device d(x);
    const int dt = code_of(x.scalar_type());
    const Packed p(x);
    const at::Tensor codes = Packed::codes(x), scales = p.scales(x);
    return pair(launch(api.caifx_checkpoint_pack, x.data_ptr(), codes.data_ptr(), floats(scales), p.rows, p.cols, dt, d.stream()), codes, scales);
  });
}

// checkpoint_unpack(codes, scales, dtype code) -> values or status
PyObject *checkpoint_unpack(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  return guarded(n, 3, [&]() -> PyObject * {
    const at::Tensor &codes = device_tensor(v[0]);
    const Device d(codes);
    if (codes.scalar_type() != at::kChar) throw Error{PyExc_ValueError, "a checkpoint's codes are int8"};
    const Packed p(codes);
    const at::Tensor &scales = d.operand(v[1], at::kFloat, p.rows * p.groups, "the checkpoint's scales must be fp32, one per 128 values of a row");
    const int dt = static_cast<int>(integer(v[2]));
    const at::Tensor y = at::empty(codes.sizes(), codes.options().dtype(type_of(dt)));
    return result(launch(api.caifx_checkpoint_unpack, codes.data_ptr(), floats(scales), y.data_ptr(), p.rows, p.cols, dt, d.stream()), y);
  });
}

// silu_multiply_checkpoint(gate, up) -> (hidden, gate codes, gate scales, up codes, up scales) or status
PyObject *silu_multiply_checkpoint(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  return guarded(n, 2, [&]() -> PyObject * {
    const at::Tensor &gate = device_tensor(v[0]);
    const Device d(gate);
    const int dt = code_of(gate.scalar_type());
    const at::Tensor &up = d.operand(v[1], gate.scalar_type(), gate.numel(), "gate and up must have one shape and dtype");
    if (up.sizes() != gate.sizes()) throw Error{PyExc_ValueError, "gate and up must have one shape and dtype"};
    const Packed p(gate);
    const at::Tensor hidden = at::empty_like(gate), gc = Packed::codes(gate), gs = p.scales(gate), uc = Packed::codes(gate), us = p.scales(gate);
    const int st = launch(api.caifx_silu_multiply_checkpoint, gate.data_ptr(), up.data_ptr(), hidden.data_ptr(), gc.data_ptr(), floats(gs), uc.data_ptr(),
                          floats(us), p.rows, p.cols, dt, d.stream());
    if (st != CAIFX_OK) return PyLong_FromLong(st);
    Owned o1(THPVariable_Wrap(hidden)), o2(THPVariable_Wrap(gc)), o3(THPVariable_Wrap(gs)), o4(THPVariable_Wrap(uc)), o5(THPVariable_Wrap(us));
    return PyTuple_Pack(5, o1.p, o2.p, o3.p, o4.p, o5.p);
  });
}

// swiglu_backward_checkpoint(gate codes, gate scales, up codes, up scales, grad_hidden, with_hidden) -> (grad_gate, grad_up[, hidden]) or status
PyObject *swiglu_backward_checkpoint(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  return guarded(n, 6, [&]() -> PyObject * {
    const at::Tensor &grad = device_tensor(v[4]);
    const Device d(grad);
    const int dt = code_of(grad.scalar_type());
    const Packed p(grad);
    const char *codes_are = "a checkpoint's codes are int8, of the gradient's shape", *scales_are = "the checkpoint's scales must be fp32, one per 128 values of a row";
    const at::Tensor &gc = d.operand(v[0], at::kChar, grad.numel(), codes_are), &uc = d.operand(v[2], at::kChar, grad.numel(), codes_are);
    const at::Tensor &gs = d.operand(v[1], at::kFloat, p.rows * p.groups, scales_are), &us = d.operand(v[3], at::kFloat, p.rows * p.groups, scales_are);
    if (Packed(gc).cols != p.cols || Packed(uc).cols != p.cols) throw Error{PyExc_ValueError, codes_are};
    const bool with = truth(v[5]);
    const at::Tensor gg = at::empty_like(grad), gu = at::empty_like(grad), hidden = with ? at::empty_like(grad) : at::Tensor();
    const int st = launch(api.caifx_swiglu_backward_checkpoint, gc.data_ptr(), floats(gs), uc.data_ptr(), floats(us), grad.data_ptr(), gg.data_ptr(),
                          gu.data_ptr(), with ? hidden.data_ptr() : nullptr, p.rows, p.cols, dt, d.stream());
    if (!with) return pair(st, gg, gu);
    if (st != CAIFX_OK) return PyLong_FromLong(st);
    Owned o1(THPVariable_Wrap(gg)), o2(THPVariable_Wrap(gu)), o3(THPVariable_Wrap(hidden));
    return PyTuple_Pack(3, o1.p, o2.p, o3.p);
  });
}

// ------------------------------------------------------------------ microscaled 4-bit floating point, gated feed-forward block
// the last extent of a tensor of at least one dimension
int64_t last(const at::Tensor &t)
{
  if (t.dim() == 0) throw Error{PyExc_ValueError, "expected a tensor of at least one dimension"};
  return t.size(t.dim() - 1);
}

// codes and scales of rows of values; the scales decide the number of blocks
struct Micro {
  const at::Tensor &codes, &scales;
  int64_t rows, blocks;
  Micro(const Device &d, PyObject *c, PyObject *s) : codes(device_tensor(c)), scales(device_tensor(s))
  {
    if (codes.device() != d.at || scales.device() != d.at) throw Error{PyExc_RuntimeError, "tensors must be on one device"};
    if (codes.scalar_type() != at::kByte || scales.scalar_type() != at::kByte) throw Error{PyExc_ValueError, "codes and scales are uint8"};
    blocks = last(scales);
    if (codes.dim() != scales.dim() || last(codes) != 16 * blocks || codes.numel() != 16 * scales.numel())
      throw Error{PyExc_ValueError, "codes must have 16 bytes for every scale"};
    rows = blocks > 0 ? scales.numel() / blocks : 0;
  }
};

// mxfp4_quantize(x) -> (codes, scales) or status
PyObject *mxfp4_quantize(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  return guarded(n, 1, [&]() -> PyObject * {
    const at::Tensor &x = device_tensor(v[0]);
    const Device d(x);
    const int dt = code_of(x.scalar_type());
    const int64_t cols = last(x), rows = cols > 0 ? x.numel() / cols : 0, blocks = (cols + CAIFX_MXFP4_BLOCK - 1) / CAIFX_MXFP4_BLOCK;
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = 16 * blocks;
    const at::Tensor codes = at::empty(shape, x.options().dtype(at::kByte));
    shape.back() = blocks;
    const at::Tensor scales = at::empty(shape, x.options().dtype(at::kByte));
    return pair(launch(api.caifx_mxfp4_quantize, x.data_ptr(), codes.data_ptr(), scales.data_ptr(), rows, cols, dt, d.stream()), codes, scales);
  });
}

// mxfp4_dequantize(codes, scales, columns, dtype code) -> values or status
PyObject *mxfp4_dequantize(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  return guarded(n, 4, [&]() -> PyObject * {
    const Device d(device_tensor(v[0]));
    const Micro m(d, v[0], v[1]);
    const int64_t cols = integer(v[2]);
    if (cols < 0 || (cols + CAIFX_MXFP4_BLOCK - 1) / CAIFX_MXFP4_BLOCK != m.blocks) throw Error{PyExc_ValueError, "columns do not fill the blocks there are"};
    const int dt = static_cast<int>(integer(v[3]));
    std::vector<int64_t> shape = m.scales.sizes().vec();
    shape.back() = cols;
    const at::Tensor y = at::empty(shape, m.codes.options().dtype(type_of(dt)));
    return result(launch(api.caifx_mxfp4_dequantize, m.codes.data_ptr(), m.scales.data_ptr(), y.data_ptr(), m.rows, cols, dt, d.stream()), y);
  });
}

// mxfp4_matmul(a codes, a scales, b codes, b scales, result's dtype code, out) -> y or status
PyObject *mxfp4_matmul(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  return guarded(n, 6, [&]() -> PyObject * {
    const Device d(device_tensor(v[0]));
    const Micro a(d, v[0], v[1]), b(d, v[2], v[3]);
    if (a.blocks != b.blocks) throw Error{PyExc_ValueError, "both operands must have rows of one length"};
    const int dt = static_cast<int>(integer(v[4]));
    const at::Tensor *out = d.optional(v[5], type_of(dt), a.rows * b.rows, "out must have the result's dtype and M x N elements");
    if (out) apart(*out, nullptr, {&a.codes, &a.scales, &b.codes, &b.scales});
    const at::Tensor y = out ? *out : at::empty({a.rows, b.rows}, a.codes.options().dtype(type_of(dt)));
    const int64_t K = CAIFX_MXFP4_BLOCK * a.blocks;
    const Scratch ws(a.codes, api.caifx_mxfp4_matmul_workspace_bytes(a.rows, b.rows, K));
    return result(launch(api.caifx_mxfp4_matmul, a.rows, b.rows, K, a.codes.data_ptr(), a.scales.data_ptr(), b.codes.data_ptr(), b.scales.data_ptr(),
                         y.data_ptr(), dt, ws.p(), ws.bytes, d.stream()), y);
  });
}

// the two weights of a gated block
struct Gated {
  int64_t N, K;
  int kind;
  const void *gate, *gate_scales, *up, *up_scales;
  Gated(const Device &d, const at::Tensor &x, PyObject *g, PyObject *u)
  {
    const WeightAttrs &w = attrs();
    N = int_attr(g, w.n), K = int_attr(g, w.k), kind = static_cast<int>(int_attr(g, w.kind));
    if (N <= 0 || K <= 0) throw Error{PyExc_ValueError, "the weight has no elements"};
    if (int_attr(u, w.n) != N || int_attr(u, w.k) != K || int_attr(u, w.kind) != kind) throw Error{PyExc_ValueError, "both weights must have one shape and kind"};
    for (PyObject *o : {g, u}) {
      if (kind == CAIFX_W_MXFP4) {
        check_mxfp4(o, N, K, x);
      } else if (kind == CAIFX_W_F16 || kind == CAIFX_W_BF16) {
        const Owned t(PyObject_GetAttr(o, w.wq.name));
        d.operand(t.p, kind == CAIFX_W_F16 ? at::kHalf : at::kBFloat16, N * K, "a stored weight has N x K elements of its kind's type");
      }
    }
    gate = ptr_attr(g, w.wq), up = ptr_attr(u, w.wq);
    gate_scales = kind == CAIFX_W_MXFP4 ? ptr_attr(g, w.scales) : nullptr;
    up_scales = kind == CAIFX_W_MXFP4 ? ptr_attr(u, w.scales) : nullptr;
  }
};

// gated_forward(x, gate weight, up weight, keep) -> hidden, (hidden, gate, up) or status
PyObject *gated_forward(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  return guarded(n, 4, [&]() -> PyObject * {
    const at::Tensor &x = device_tensor(v[0]);
    const Device d(x);
    const int dt = code_of(x.scalar_type());
    const Gated w(d, x, v[1], v[2]);
    if (last(x) != w.K) throw Error{PyExc_ValueError, "a row of activations must be as long as the weights' rows"};
    const int64_t M = x.numel() / w.K;
    const bool keep = truth(v[3]);
    const at::Tensor hidden = at::empty({M, w.N}, x.options());
    const at::Tensor gate = keep ? at::empty_like(hidden) : at::Tensor(), up = keep ? at::empty_like(hidden) : at::Tensor();
    const Scratch ws(x, api.caifx_gated_workspace_bytes(M, w.N, w.K, w.kind, dt, 0));
    const int st = launch(api.caifx_gated_forward, M, w.N, w.K, x.data_ptr(), w.gate, w.gate_scales, w.up, w.up_scales, w.kind, hidden.data_ptr(),
                          keep ? gate.data_ptr() : nullptr, keep ? up.data_ptr() : nullptr, dt, ws.p(), ws.bytes, d.stream());
    if (!keep) return result(st, hidden);
    if (st != CAIFX_OK) return PyLong_FromLong(st);
    Owned o1(THPVariable_Wrap(hidden)), o2(THPVariable_Wrap(gate)), o3(THPVariable_Wrap(up));
    return PyTuple_Pack(3, o1.p, o2.p, o3.p);
  });
}

// gated_backward(grad_hidden, gate, up, gate weight, up weight, need_dx) -> (dx or None, grad_gate, grad_up) or status
PyObject *gated_backward(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  return guarded(n, 6, [&]() -> PyObject * {
    const at::Tensor &grad = device_tensor(v[0]);
    const Device d(grad);
    const int dt = code_of(grad.scalar_type());
    const Gated w(d, grad, v[3], v[4]);
    if (last(grad) != w.N) throw Error{PyExc_ValueError, "a row of gradients must have a value for each of the weights' rows"};
    const int64_t M = grad.numel() / w.N;
    const char *same = "gate and up must have the gradient's dtype and number of elements";
    const at::Tensor &gate = d.operand(v[1], grad.scalar_type(), grad.numel(), same), &up = d.operand(v[2], grad.scalar_type(), grad.numel(), same);
    const bool need = truth(v[5]);
    const at::Tensor gg = at::empty({M, w.N}, grad.options()), gu = at::empty({M, w.N}, grad.options());
    const at::Tensor dx = need ? at::empty({M, w.K}, grad.options()) : at::Tensor();
    const Scratch ws(grad, need ? api.caifx_gated_workspace_bytes(M, w.N, w.K, w.kind, dt, 1) : 0);
    const int st = launch(api.caifx_gated_backward, M, w.N, w.K, grad.data_ptr(), gate.data_ptr(), up.data_ptr(), w.gate, w.gate_scales, w.up, w.up_scales,
                          w.kind, gg.data_ptr(), gu.data_ptr(), need ? dx.data_ptr() : nullptr, dt, ws.p(), ws.bytes, d.stream());
    if (st != CAIFX_OK) return PyLong_FromLong(st);
    Owned o1(need ? THPVariable_Wrap(dx) : Py_NewRef(Py_None)), o2(THPVariable_Wrap(gg)), o3(THPVariable_Wrap(gu));
    return PyTuple_Pack(3, o1.p, o2.p, o3.p);
  });
}

PyMethodDef methods[] = {
    {"bind", bind, METH_O, nullptr},
#define M(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr},
    M(qlinear) M(grouped) M(quantize_int8) M(quantize_int4) M(elementwise) M(swiglu_backward) M(moe_build_dispatch_map) M(moe_dispatch) M(moe_combine)
    M(moe_combine_backward_grad_expert) M(moe_dispatch_backward) M(moe_combine_backward_grad_weights)
    M(adapters_forward) M(adapters_backward) M(checkpoint_pack) M(checkpoint_unpack) M(silu_multiply_checkpoint) M(swiglu_backward_checkpoint)
    M(mxfp4_quantize) M(mxfp4_dequantize) M(mxfp4_matmul) M(gated_forward) M(gated_backward)
#undef M
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "caifx_torch_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit_caifx_torch_calls() { return PyModule_Create(&module); }
