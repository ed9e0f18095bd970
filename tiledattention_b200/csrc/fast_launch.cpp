// One-call host launcher for the common case of tiledattention_b200.sdpa: the reference's
// per-call Python path (src/tiledattention/sdpa.py:14-48 -> kernels/flash_fwd.py:821-973)
// costs ~35 us at S=512; this module does the checks, the output allocation, the stream
// lookup and the ta_sdpa_fwd call in one CPython call.
//
//   launch(q, k, v, causal: bool, scale: float, want_lse: bool) -> o | (o, lse) | None
//
// scale == -1.0 selects the default 1/sqrt(D). The device status word of each device is
// registered once with set_status(device_index, address); a device without one takes the
// full path (which creates and registers it).
//
// It returns None, having launched nothing, for every case it does not take: inputs the
// contract rejects, head dims outside {64, 128, 256} and multiples of 8 up to 256, strides a
// tensor map cannot describe, or any non-OK status from ta_sdpa_fwd (all of which are
// reported before a launch). The caller then runs the full Python path, which raises the
// reference's error for the case or copies / pads the inputs. ta_sdpa_fwd is bound once
// through set_entry(address) with the address of the symbol in the already-loaded native
// library, so the two share one copy of the library's state.
//
// rotary(), kv8_append() and sdpa_kv8() do the same for the operators around a decoder's
// attention: None (nothing launched) where the Python path has to raise, copy or differentiate.
//
// The same module registers the torch operators of the reference's native-op slot
// (torch-ext/torch_binding.cpp:6-19: TORCH_LIBRARY + ops.impl(..., kCUDA, ...)) in C++:
//   tiledattention_b200::sdpa_fwd(Tensor q, Tensor k, Tensor v, bool causal, float scale)
//       -> Tensor
//   tiledattention_b200::sdpa_fwd_partial(Tensor q, Tensor k, Tensor v, bool causal,
//       float scale, int kv_begin, int kv_end, int n_split) -> (Tensor, Tensor)
// with CUDA kernels over the C ABI (copying strides a tensor map cannot describe, padding
// head dims that are not multiples of 8) and Meta kernels for shape propagation. Errors are
// raised with TORCH_CHECK, as the reference's op stub does (tiledattention.cu:13-33).
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/constant_pad_nd.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "tiledattention_b200.h"

#include <cmath>
#include <cstdint>

namespace {

using SdpaFwdFn = decltype(&ta_sdpa_fwd);
using SdpaPartialFn = decltype(&ta_sdpa_fwd_partial);
using LastErrorFn = decltype(&ta_last_error);

SdpaFwdFn g_entry = nullptr;
SdpaPartialFn g_partial = nullptr;
LastErrorFn g_last_error = nullptr;
decltype(&ta_rotary) g_rotary = nullptr;
decltype(&ta_kv8_append) g_kv8_append = nullptr;
decltype(&ta_sdpa_kv8_workspace) g_kv8_workspace = nullptr;
decltype(&ta_sdpa_kv8) g_sdpa_kv8 = nullptr;
constexpr int kMaxDevices = 64;
unsigned int* g_status[kMaxDevices] = {};
unsigned long long g_launches = 0;  // launches taken by this module (read by the tests)

constexpr int kDtypeF16 = TA_DTYPE_F16;
constexpr int kDtypeBf16 = TA_DTYPE_BF16;

// Tensor-map compatible: unit inner stride, 16-byte aligned base and outer strides.
bool tma_ok(const at::Tensor& t) {
  if (t.stride(3) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  const int64_t esz = t.element_size();
  for (int d = 0; d < 3; ++d)
    if (t.size(d) > 1 && (t.stride(d) * esz) % 16) return false;
  return true;
}

PyObject* set_entry(PyObject*, PyObject* arg) {
  const unsigned long long addr = PyLong_AsUnsignedLongLong(arg);
  if (PyErr_Occurred()) return nullptr;
  g_entry = reinterpret_cast<SdpaFwdFn>(static_cast<uintptr_t>(addr));
  Py_RETURN_NONE;
}

// bind_ops(partial_address, last_error_address): the other entry points the torch
// operators call.
PyObject* bind_ops(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "bind_ops(partial_address, last_error_address)");
    return nullptr;
  }
  const unsigned long long a = PyLong_AsUnsignedLongLong(args[0]);
  const unsigned long long b = PyLong_AsUnsignedLongLong(args[1]);
  if (PyErr_Occurred()) return nullptr;
  g_partial = reinterpret_cast<SdpaPartialFn>(static_cast<uintptr_t>(a));
  g_last_error = reinterpret_cast<LastErrorFn>(static_cast<uintptr_t>(b));
  Py_RETURN_NONE;
}

PyObject* set_status(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "set_status(device_index, address)");
    return nullptr;
  }
  const long idx = PyLong_AsLong(args[0]);
  const unsigned long long addr = PyLong_AsUnsignedLongLong(args[1]);
  if (PyErr_Occurred()) return nullptr;
  if (idx < 0 || idx >= kMaxDevices) Py_RETURN_NONE;
  g_status[idx] = reinterpret_cast<unsigned int*>(static_cast<uintptr_t>(addr));
  Py_RETURN_NONE;
}

PyObject* launches(PyObject*, PyObject*) { return PyLong_FromUnsignedLongLong(g_launches); }

PyObject* launch(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 6 || g_entry == nullptr) Py_RETURN_NONE;
  for (int i = 0; i < 3; ++i)
    if (!THPVariable_Check(args[i])) Py_RETURN_NONE;
  if (!PyBool_Check(args[3]) || !PyFloat_Check(args[4]) || !PyBool_Check(args[5]))
    Py_RETURN_NONE;
  try {
    const at::Tensor& q = THPVariable_Unpack(args[0]);
    const at::Tensor& k = THPVariable_Unpack(args[1]);
    const at::Tensor& v = THPVariable_Unpack(args[2]);
    const bool causal = args[3] == Py_True;
    const bool want_lse = args[5] == Py_True;
    double scale = PyFloat_AS_DOUBLE(args[4]);
    if (scale != -1.0 && !(scale > 0.0)) Py_RETURN_NONE;

    if (q.dim() != 4 || !q.is_cuda() || !k.is_cuda() || !v.is_cuda()) Py_RETURN_NONE;
    if (q.sizes() != k.sizes() || q.sizes() != v.sizes()) Py_RETURN_NONE;
    const auto st = q.scalar_type();
    if (k.scalar_type() != st || v.scalar_type() != st) Py_RETURN_NONE;
    int dtype;
    if (st == at::kHalf)
      dtype = kDtypeF16;
    else if (st == at::kBFloat16)
      dtype = kDtypeBf16;
    else
      Py_RETURN_NONE;
    const c10::Device dev = q.device();
    if (k.device() != dev || v.device() != dev) Py_RETURN_NONE;
    const int dev_idx = dev.index();
    if (dev_idx < 0 || dev_idx >= kMaxDevices || g_status[dev_idx] == nullptr) Py_RETURN_NONE;
    if (q.requires_grad() || k.requires_grad() || v.requires_grad()) Py_RETURN_NONE;

    const int64_t B = q.size(0), H = q.size(1), S = q.size(2), D = q.size(3);
    if (B <= 0 || H <= 0 || S <= 0 || D <= 0 || B * H > INT32_MAX || S > INT32_MAX)
      Py_RETURN_NONE;
    if (!(D == 64 || D == 128 || D == 256 || (D % 8 == 0 && D < 256))) Py_RETURN_NONE;
    if (!tma_ok(q) || !tma_ok(k) || !tma_ok(v)) Py_RETURN_NONE;
    if (scale == -1.0) scale = 1.0 / std::sqrt(static_cast<double>(D));

    c10::cuda::CUDAGuard guard(dev);
    at::Tensor o = at::empty({B, H, S, D}, q.options());
    at::Tensor lse;
    if (want_lse) lse = at::empty({B, H, S}, q.options().dtype(at::kFloat));
    const int64_t qs[4] = {q.stride(0), q.stride(1), q.stride(2), q.stride(3)};
    const int64_t ks[4] = {k.stride(0), k.stride(1), k.stride(2), k.stride(3)};
    const int64_t vs[4] = {v.stride(0), v.stride(1), v.stride(2), v.stride(3)};
    const int64_t os[4] = {o.stride(0), o.stride(1), o.stride(2), o.stride(3)};
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev_idx).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_entry(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                 want_lse ? lse.data_ptr<float>() : nullptr, static_cast<int>(B),
                 static_cast<int>(H), static_cast<int>(S), static_cast<int>(D), qs, ks, vs, os,
                 dtype, causal ? 1 : 0, static_cast<float>(scale),
                 g_status[dev_idx], stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) Py_RETURN_NONE;
    ++g_launches;
    if (!want_lse) return THPVariable_Wrap(std::move(o));
    PyObject* po = THPVariable_Wrap(std::move(o));
    if (po == nullptr) return nullptr;
    PyObject* pl = THPVariable_Wrap(std::move(lse));
    if (pl == nullptr) {
      Py_DECREF(po);
      return nullptr;
    }
    PyObject* tup = PyTuple_Pack(2, po, pl);
    Py_DECREF(po);
    Py_DECREF(pl);
    return tup;
  } catch (python_error& e) {  // of Python code that torch called: its own, not ours to answer
    e.restore();
    return nullptr;
  } catch (const std::exception&) {
    // Any ATen error (e.g. out of memory on the output): leave it to the full path, which
    // raises it through torch's own error translation.
    Py_RETURN_NONE;
  }
}

// ---------------------------------------------------------------- rotary and the 8-bit cache

// bind_serving(rotary, kv8_append, sdpa_kv8_workspace, sdpa_kv8): entry points by address.
PyObject* bind_serving(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 4) {
    PyErr_SetString(PyExc_TypeError, "bind_serving takes four addresses");
    return nullptr;
  }
  uintptr_t a[4];
  for (int i = 0; i < 4; ++i) {
    a[i] = static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(args[i]));
    if (PyErr_Occurred()) return nullptr;
  }
  g_rotary = reinterpret_cast<decltype(g_rotary)>(a[0]);
  g_kv8_append = reinterpret_cast<decltype(g_kv8_append)>(a[1]);
  g_kv8_workspace = reinterpret_cast<decltype(g_kv8_workspace)>(a[2]);
  g_sdpa_kv8 = reinterpret_cast<decltype(g_sdpa_kv8)>(a[3]);
  Py_RETURN_NONE;
}

// The tensor of a Python argument, or null.
const at::Tensor* tensor_arg(PyObject* o) {
  return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
}

struct Strides4 {
  int64_t v[4];
  explicit Strides4(const at::Tensor& t)
      : v{t.stride(0), t.stride(1), t.stride(2), t.stride(3)} {}
};

int dtype_code(const at::Tensor& t) {
  const auto st = t.scalar_type();
  return st == at::kHalf ? kDtypeF16 : st == at::kBFloat16 ? kDtypeBf16 : -1;
}

bool fits_int(int64_t n) { return n > 0 && n <= INT32_MAX; }

// A contiguous int32 vector of n entries on dev (unit stride where n > 1).
bool int_vector(const at::Tensor* t, int64_t n, c10::Device dev) {
  return t && t->dim() == 1 && t->size(0) == n && t->scalar_type() == at::kInt &&
         t->device() == dev && (n <= 1 || t->stride(0) == 1);
}

// rotary(q, k, positions, inv_freq) on tensors as the kernel takes them: false, having done
// nothing, for everything else.
struct RotaryHow {
  bool interleaved;
  double magnitude;
  bool inverse;
};
bool rotary_launch(const at::Tensor& q, const at::Tensor* k, const at::Tensor& pos,
                   const at::Tensor& freq, const RotaryHow& how, at::Tensor& qo, at::Tensor& ko) {
  if (g_rotary == nullptr || q.dim() != 4 || !q.is_cuda() || !std::isfinite(how.magnitude))
    return false;
  const int dtype = dtype_code(q);
  const c10::Device dev = q.device();
  const int64_t B = q.size(0), H = q.size(1), S = q.size(2), D = q.size(3);
  if (dtype < 0 || !fits_int(B) || !fits_int(H) || !fits_int(S) || !fits_int(D) || q.stride(3) != 1)
    return false;
  if (k && (k->dim() != 4 || k->device() != dev || dtype_code(*k) != dtype || k->size(0) != B ||
            !fits_int(k->size(1)) || k->size(2) != S || k->size(3) != D || k->stride(3) != 1))
    return false;
  const auto pt = pos.scalar_type();
  if (pos.device() != dev || (pt != at::kInt && pt != at::kLong)) return false;
  const bool row = pos.dim() == 1;
  if (!(row ? pos.size(0) == S
            : pos.dim() == 2 && (pos.size(0) == B || pos.size(0) == 1) && pos.size(1) == S))
    return false;
  if (freq.device() != dev || freq.scalar_type() != at::kDouble || freq.dim() != 1 ||
      freq.size(0) < 1 || 2 * freq.size(0) > D || (freq.size(0) > 1 && freq.stride(0) != 1))
    return false;
  c10::cuda::CUDAGuard guard(dev);
  qo = at::empty({B, H, S, D}, q.options());
  if (k) ko = at::empty({B, k->size(1), S, D}, k->options());
  const Strides4 qs(q), qos(qo), ks(k ? *k : q), kos(k ? ko : qo);
  const int64_t ps[2] = {row || pos.size(0) == 1 ? 0 : pos.stride(0), pos.stride(row ? 0 : 1)};
  const int rc = g_rotary(
      q.data_ptr(), qo.data_ptr(), qs.v, qos.v, static_cast<int>(H), k ? k->data_ptr() : nullptr,
      k ? ko.data_ptr() : nullptr, k ? ks.v : nullptr, k ? kos.v : nullptr,
      k ? static_cast<int>(k->size(1)) : 0, static_cast<int>(B), static_cast<int>(S),
      static_cast<int>(D), static_cast<int>(2 * freq.size(0)), pos.data_ptr(), pt == at::kLong, ps,
      freq.data_ptr<double>(), how.interleaved, how.inverse, static_cast<float>(how.magnitude),
      dtype, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  if (rc != 0) return false;
  ++g_launches;
  return true;
}

// The differentiable form: a rotation's gradient is the rotation the other way, and so is the
// gradient's.
struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                const at::Tensor& q,
                                                const std::optional<at::Tensor>& k,
                                                const at::Tensor& pos, const at::Tensor& freq,
                                                bool interleaved, double magnitude, bool inverse) {
    at::Tensor qo, ko;
    TORCH_CHECK(rotary_launch(q, k ? &*k : nullptr, pos, freq,
                              {interleaved, magnitude, inverse}, qo, ko),
                "rotary: ", g_last_error ? g_last_error() : "", " (launch)");
    ctx->save_for_backward({pos, freq});
    ctx->set_materialize_grads(false);  // of an unused output: undefined, not zeros to be turned
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["inverse"] = inverse;
    ctx->saved_data["has_k"] = k.has_value();
    if (!k) return {qo};
    return {qo, ko};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool interleaved = ctx->saved_data["interleaved"].toBool();
    const double magnitude = ctx->saved_data["magnitude"].toDouble();
    const bool inverse = !ctx->saved_data["inverse"].toBool();
    const bool has_k = ctx->saved_data["has_k"].toBool();
    // A gradient that nobody needs, or that never came, costs nothing.
    at::Tensor gq = ctx->needs_input_grad(0) ? grads[0] : at::Tensor();
    at::Tensor gk = has_k && ctx->needs_input_grad(1) ? grads[1] : at::Tensor();
    for (at::Tensor* g : {&gq, &gk})
      if (g->defined() && g->stride(3) != 1) *g = g->contiguous();
    const std::optional<at::Tensor> none, second = gk.defined() ? std::optional<at::Tensor>(gk) : none;
    if (gq.defined()) {
      auto out = apply(gq, second, saved[0], saved[1], interleaved, magnitude, inverse);
      gq = out[0];
      if (gk.defined()) gk = out[1];
    } else if (gk.defined()) {
      gk = apply(gk, none, saved[0], saved[1], interleaved, magnitude, inverse)[0];
    }
    return {gq, gk, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// A tensor that carries a forward-mode tangent: the Python path turns that too.
bool has_tangent(const at::Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }

PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 7) Py_RETURN_NONE;
  const at::Tensor* q = tensor_arg(args[0]);
  const bool has_k = args[1] != Py_None;
  const at::Tensor* k = has_k ? tensor_arg(args[1]) : nullptr;
  const at::Tensor* pos = tensor_arg(args[2]);
  const at::Tensor* freq = tensor_arg(args[3]);
  if (!q || (has_k && !k) || !pos || !freq) Py_RETURN_NONE;
  if (!PyBool_Check(args[4]) || !PyFloat_Check(args[5]) || !PyBool_Check(args[6])) Py_RETURN_NONE;
  const RotaryHow how{args[4] == Py_True, PyFloat_AS_DOUBLE(args[5]), args[6] == Py_True};
  at::Tensor qo, ko;
  try {
    if (has_tangent(*q) || (k && has_tangent(*k))) Py_RETURN_NONE;
    if (at::GradMode::is_enabled() && (q->requires_grad() || (k && k->requires_grad()))) {
      auto out = RotaryFunction::apply(*q, k ? std::optional<at::Tensor>(*k) : std::nullopt, *pos, *freq, how.interleaved,
                                       how.magnitude, how.inverse);
      qo = out[0];
      if (k) ko = out[1];
    } else if (!rotary_launch(*q, k, *pos, *freq, how, qo, ko)) {
      Py_RETURN_NONE;
    }
  } catch (python_error& e) {  // of Python code that torch called: its own, not ours to answer
    e.restore();
    return nullptr;
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
  PyObject* out = PyTuple_New(2);
  if (out == nullptr) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(qo)));
  if (k) {
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(ko)));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(out, 1, Py_None);
  }
  return out;
}

// The cache's four tensors (args) and the page table, where they are as the kernels take them.
struct CacheArgs {
  const at::Tensor* t[4];  // k, v, k_scale, v_scale
  const at::Tensor* table;
  int64_t pages, heads, page, dim;
};
bool cache_args(PyObject* const* args, PyObject* table, int64_t B, c10::Device dev, CacheArgs& c) {
  for (int i = 0; i < 4; ++i) {
    c.t[i] = tensor_arg(args[i]);
    if (!c.t[i] || c.t[i]->device() != dev || !c.t[i]->is_contiguous() ||
        c.t[i]->requires_grad() || c.t[i]->dim() != (i < 2 ? 4 : 2) ||
        c.t[i]->scalar_type() != (i < 2 ? at::kFloat8_e4m3fn : at::kFloat))
      return false;
  }
  c.pages = c.t[0]->size(0);
  c.heads = c.t[0]->size(1);
  c.page = c.t[0]->size(2);
  c.dim = c.t[0]->size(3);
  if (c.t[1]->sizes() != c.t[0]->sizes() || !fits_int(c.pages) || !fits_int(c.heads) ||
      !fits_int(c.page) || !fits_int(c.dim))
    return false;
  for (int i = 2; i < 4; ++i)
    if (c.t[i]->size(0) != c.pages || c.t[i]->size(1) != c.heads) return false;
  c.table = tensor_arg(table);
  return c.table && c.table->dim() == 2 && c.table->size(0) == B && fits_int(c.table->size(1)) &&
         c.table->scalar_type() == at::kInt && c.table->device() == dev &&
         (c.table->size(1) == 1 || c.table->stride(1) == 1);
}

// kv8_append(k, v, cache.k, cache.v, cache.k_scale, cache.v_scale, table, starts, counts)
PyObject* kv8_append(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 9 || g_kv8_append == nullptr) Py_RETURN_NONE;
  const at::Tensor* k = tensor_arg(args[0]);
  const at::Tensor* v = tensor_arg(args[1]);
  const at::Tensor* starts = tensor_arg(args[7]);
  const at::Tensor* counts = args[8] != Py_None ? tensor_arg(args[8]) : nullptr;
  if (!k || !v || !starts || (args[8] != Py_None && !counts)) Py_RETURN_NONE;
  try {
    if (k->dim() != 4 || v->dim() != 4 || !k->is_cuda()) Py_RETURN_NONE;
    const int dtype = dtype_code(*k);
    const c10::Device dev = k->device();
    const int64_t B = k->size(0), H = k->size(1), T = k->size(2), D = k->size(3);
    if (dtype < 0 || dtype_code(*v) != dtype || v->device() != dev || v->sizes() != k->sizes() ||
        !fits_int(B) || !fits_int(H) || !fits_int(T) || !fits_int(D) || !tma_ok(*k) || !tma_ok(*v))
      Py_RETURN_NONE;
    CacheArgs c;
    if (!cache_args(args + 2, args[6], B, dev, c) || c.heads != H || c.dim != D) Py_RETURN_NONE;
    if (!int_vector(starts, B, dev) || (counts && !int_vector(counts, B, dev))) Py_RETURN_NONE;
    const int idx = dev.index();
    if (idx < 0 || idx >= kMaxDevices || g_status[idx] == nullptr) Py_RETURN_NONE;
    c10::cuda::CUDAGuard guard(dev);
    const Strides4 ks(*k), vs(*v);
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(idx).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_kv8_append(k->data_ptr(), v->data_ptr(), ks.v, vs.v, c.t[0]->data_ptr(),
                      c.t[1]->data_ptr(), c.t[2]->data_ptr<float>(), c.t[3]->data_ptr<float>(),
                      static_cast<int>(c.pages), static_cast<int>(c.page),
                      c.table->data_ptr<int>(), c.table->stride(0),
                      static_cast<int>(c.table->size(1)), starts->data_ptr<int>(),
                      counts ? counts->data_ptr<int>() : nullptr, static_cast<int>(B),
                      static_cast<int>(H), static_cast<int>(T), static_cast<int>(D), dtype,
                      g_status[idx], stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) Py_RETURN_NONE;
    ++g_launches;
    Py_RETURN_TRUE;
  } catch (python_error& e) {  // of Python code that torch called: its own, not ours to answer
    e.restore();
    return nullptr;
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// sdpa_kv8(q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, lengths, counts, causal,
//          scale, want_lse); scale -1.0: the default 1/sqrt(D)
PyObject* sdpa_kv8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 11 || g_sdpa_kv8 == nullptr) Py_RETURN_NONE;
  const at::Tensor* q = tensor_arg(args[0]);
  const at::Tensor* lengths = tensor_arg(args[6]);
  const at::Tensor* counts = args[7] != Py_None ? tensor_arg(args[7]) : nullptr;
  if (!q || !lengths || (args[7] != Py_None && !counts)) Py_RETURN_NONE;
  if (!PyBool_Check(args[8]) || !PyFloat_Check(args[9]) || !PyBool_Check(args[10])) Py_RETURN_NONE;
  double scale = PyFloat_AS_DOUBLE(args[9]);
  const bool want_lse = args[10] == Py_True;
  try {
    if (q->dim() != 4 || !q->is_cuda()) Py_RETURN_NONE;
    const int dtype = dtype_code(*q);
    const c10::Device dev = q->device();
    const int64_t B = q->size(0), H = q->size(1), T = q->size(2), D = q->size(3);
    if (dtype < 0 || !fits_int(B) || !fits_int(H) || !fits_int(T) || !fits_int(D) || !tma_ok(*q))
      Py_RETURN_NONE;
    CacheArgs c;
    if (!cache_args(args + 1, args[5], B, dev, c) || c.dim != D || H % c.heads != 0) Py_RETURN_NONE;
    if (!int_vector(lengths, B, dev) || (counts && !int_vector(counts, B, dev))) Py_RETURN_NONE;
    const int idx = dev.index();
    if (idx < 0 || idx >= kMaxDevices || g_status[idx] == nullptr) Py_RETURN_NONE;
    if (scale == -1.0) scale = 1.0 / std::sqrt(static_cast<double>(D));
    if (!(scale > 0.0) || !std::isfinite(scale)) Py_RETURN_NONE;
    c10::cuda::CUDAGuard guard(dev);
    const int b = static_cast<int>(B), h = static_cast<int>(H), t = static_cast<int>(T),
              d = static_cast<int>(D), hk = static_cast<int>(c.heads);
    const int64_t bytes = g_kv8_workspace(b, h, hk, t, d);
    at::Tensor o = at::empty({B, H, T, D}, q->options());
    at::Tensor lse;
    if (want_lse) lse = at::empty({B, H, T}, q->options().dtype(at::kFloat));
    at::Tensor work = at::empty({bytes}, q->options().dtype(at::kByte));
    const Strides4 qs(*q), os(o);
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(idx).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_sdpa_kv8(q->data_ptr(), qs.v, o.data_ptr(), os.v,
                    want_lse ? lse.data_ptr<float>() : nullptr, c.t[0]->data_ptr(),
                    c.t[1]->data_ptr(), c.t[2]->data_ptr<float>(), c.t[3]->data_ptr<float>(),
                    static_cast<int>(c.pages), static_cast<int>(c.page), c.table->data_ptr<int>(),
                    c.table->stride(0), static_cast<int>(c.table->size(1)),
                    lengths->data_ptr<int>(), counts ? counts->data_ptr<int>() : nullptr, b, h, hk,
                    t, d, dtype, args[8] == Py_True, static_cast<float>(scale), work.data_ptr(),
                    bytes, g_status[idx], stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) Py_RETURN_NONE;
    ++g_launches;
    if (!want_lse) return THPVariable_Wrap(std::move(o));
    PyObject* out = PyTuple_New(2);
    if (out == nullptr) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(o)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(lse)));
    return out;
  } catch (python_error& e) {  // of Python code that torch called: its own, not ours to answer
    e.restore();
    return nullptr;
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// ---------------------------------------------------------------- torch operators

const char* last_error() {
  const char* e = g_last_error ? g_last_error() : nullptr;
  return e && *e ? e : "native call failed";
}

// Inputs as the kernels take them: validated, head dim padded with zeros to the next native
// size unless it is a multiple of 8, strides a tensor map cannot describe copied.
struct Inputs {
  at::Tensor q, k, v;
  int64_t D, kd;
  int dtype;
};

Inputs prepare(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const char* op) {
  TORCH_CHECK(q.dim() == 4, op, ": q, k, v must be [B, H, S, D] tensors");
  TORCH_CHECK(q.sizes() == k.sizes() && q.sizes() == v.sizes(), op,
              ": q, k, v must have identical shapes");
  TORCH_CHECK(q.is_cuda() && k.device() == q.device() && v.device() == q.device(), op,
              ": q, k, v must be CUDA tensors on one device");
  const auto st = q.scalar_type();
  TORCH_CHECK(k.scalar_type() == st && v.scalar_type() == st, op,
              ": q, k, v must share one dtype");
  TORCH_CHECK(st == at::kHalf || st == at::kBFloat16, op,
              ": dtype must be torch.float16 or torch.bfloat16");
  Inputs in{q, k, v, q.size(3), 0, st == at::kBFloat16 ? kDtypeBf16 : kDtypeF16};
  TORCH_CHECK(in.D >= 1 && in.D <= 256, op, ": head dim ", in.D, " is not in [1, 256]");
  in.kd = in.D % 8 == 0 ? in.D : (in.D <= 64 ? 64 : (in.D <= 128 ? 128 : 256));
  at::Tensor* ts[3] = {&in.q, &in.k, &in.v};
  for (at::Tensor* t : ts) {
    if (in.kd != in.D) *t = at::constant_pad_nd(*t, {0, in.kd - in.D}, 0);
    if (!tma_ok(*t)) *t = t->contiguous();
  }
  return in;
}

unsigned int* status_of(const at::Tensor& t) {
  const int idx = t.device().index();
  return idx >= 0 && idx < kMaxDevices ? g_status[idx] : nullptr;
}

at::Tensor sdpa_fwd_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                         bool causal, double scale) {
  TORCH_CHECK(scale > 0.0, "sdpa_fwd: scale must be positive");
  TORCH_CHECK(g_entry != nullptr, "sdpa_fwd: native library not bound");
  c10::cuda::CUDAGuard guard(q.device());
  if (q.numel() == 0) return at::empty(q.sizes(), q.options());
  Inputs in = prepare(q, k, v, "sdpa_fwd");
  const int64_t B = q.size(0), H = q.size(1), S = q.size(2);
  at::Tensor o = at::empty({B, H, S, in.kd}, q.options());
  const int64_t qs[4] = {in.q.stride(0), in.q.stride(1), in.q.stride(2), in.q.stride(3)};
  const int64_t ks[4] = {in.k.stride(0), in.k.stride(1), in.k.stride(2), in.k.stride(3)};
  const int64_t vs[4] = {in.v.stride(0), in.v.stride(1), in.v.stride(2), in.v.stride(3)};
  const int64_t os[4] = {o.stride(0), o.stride(1), o.stride(2), o.stride(3)};
  const int rc = g_entry(in.q.data_ptr(), in.k.data_ptr(), in.v.data_ptr(), o.data_ptr(), nullptr,
                         static_cast<int>(B), static_cast<int>(H), static_cast<int>(S),
                         static_cast<int>(in.kd), qs, ks, vs, os, in.dtype, causal ? 1 : 0,
                         static_cast<float>(scale), status_of(q),
                         c10::cuda::getCurrentCUDAStream(q.device().index()).stream());
  TORCH_CHECK(rc == TA_OK, "sdpa_fwd: ", last_error());
  return in.kd == in.D ? o : o.narrow(3, 0, in.D).contiguous();
}

std::tuple<at::Tensor, at::Tensor> sdpa_fwd_partial_cuda(const at::Tensor& q, const at::Tensor& k,
                                                         const at::Tensor& v, bool causal,
                                                         double scale, int64_t kv_begin,
                                                         int64_t kv_end, int64_t n_split) {
  TORCH_CHECK(scale > 0.0, "sdpa_fwd_partial: scale must be positive");
  TORCH_CHECK(n_split >= 1, "sdpa_fwd_partial: n_split must be at least 1");
  TORCH_CHECK(g_partial != nullptr, "sdpa_fwd_partial: native library not bound");
  c10::cuda::CUDAGuard guard(q.device());
  const int64_t B = q.size(0), H = q.size(1), S = q.size(2);
  auto f32 = q.options().dtype(at::kFloat);
  if (q.numel() == 0)
    return {at::empty({n_split, B, H, S, q.size(3)}, f32), at::empty({n_split, B, H, S}, f32)};
  Inputs in = prepare(q, k, v, "sdpa_fwd_partial");
  at::Tensor o = at::empty({n_split, B, H, S, in.kd}, f32);
  at::Tensor lse = at::empty({n_split, B, H, S}, f32);
  const int64_t qs[4] = {in.q.stride(0), in.q.stride(1), in.q.stride(2), in.q.stride(3)};
  const int64_t ks[4] = {in.k.stride(0), in.k.stride(1), in.k.stride(2), in.k.stride(3)};
  const int64_t vs[4] = {in.v.stride(0), in.v.stride(1), in.v.stride(2), in.v.stride(3)};
  const int rc = g_partial(in.q.data_ptr(), in.k.data_ptr(), in.v.data_ptr(),
                           o.data_ptr<float>(), lse.data_ptr<float>(), static_cast<int>(B),
                           static_cast<int>(H), static_cast<int>(S), static_cast<int>(in.kd), qs,
                           ks, vs, in.dtype, causal ? 1 : 0, static_cast<float>(scale),
                           static_cast<int>(kv_begin), static_cast<int>(kv_end),
                           static_cast<int>(n_split), status_of(q),
                           c10::cuda::getCurrentCUDAStream(q.device().index()).stream());
  TORCH_CHECK(rc == TA_OK, "sdpa_fwd_partial: ", last_error());
  if (in.kd != in.D) o = o.narrow(4, 0, in.D).contiguous();
  return {o, lse};
}

at::Tensor sdpa_fwd_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, bool, double) {
  return at::empty(q.sizes(), q.options());
}

std::tuple<at::Tensor, at::Tensor> sdpa_fwd_partial_meta(const at::Tensor& q, const at::Tensor&,
                                                         const at::Tensor&, bool, double,
                                                         int64_t, int64_t, int64_t n_split) {
  auto f32 = q.options().dtype(at::kFloat);
  return {at::empty({n_split, q.size(0), q.size(1), q.size(2), q.size(3)}, f32),
          at::empty({n_split, q.size(0), q.size(1), q.size(2)}, f32)};
}

PyMethodDef kMethods[] = {
    {"set_entry", reinterpret_cast<PyCFunction>(set_entry), METH_O,
     "Bind ta_sdpa_fwd by its address in the loaded native library."},
    {"bind_ops", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(bind_ops)),
     METH_FASTCALL, "Bind the entry points the torch operators call."},
    {"bind_serving", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(bind_serving)),
     METH_FASTCALL, "Bind the rotary and 8-bit cache entry points."},
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(rotary)),
     METH_FASTCALL, "Checked single-call rotary launch; None when the full path must run."},
    {"kv8_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(kv8_append)),
     METH_FASTCALL, "Checked single-call cache append; None when the full path must run."},
    {"sdpa_kv8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(sdpa_kv8)),
     METH_FASTCALL, "Checked single-call cache attention; None when the full path must run."},
    {"set_status", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(set_status)),
     METH_FASTCALL, "Register the device status word of a device."},
    {"launches", reinterpret_cast<PyCFunction>(launches), METH_NOARGS,
     "Number of launches this module has made."},
    {"launch", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(launch)),
     METH_FASTCALL, "Checked single-call sdpa launch; None when the full path must run."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fast_launch", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

TORCH_LIBRARY(tiledattention_b200, m) {
  m.def("sdpa_fwd(Tensor q, Tensor k, Tensor v, bool causal, float scale) -> Tensor");
  m.def(
      "sdpa_fwd_partial(Tensor q, Tensor k, Tensor v, bool causal, float scale, int kv_begin, "
      "int kv_end, int n_split) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(tiledattention_b200, CUDA, m) {
  m.impl("sdpa_fwd", &sdpa_fwd_cuda);
  m.impl("sdpa_fwd_partial", &sdpa_fwd_partial_cuda);
}

TORCH_LIBRARY_IMPL(tiledattention_b200, Meta, m) {
  m.impl("sdpa_fwd", &sdpa_fwd_meta);
  m.impl("sdpa_fwd_partial", &sdpa_fwd_partial_meta);
}

PyMODINIT_FUNC PyInit__fast_launch() { return PyModule_Create(&kModule); }
