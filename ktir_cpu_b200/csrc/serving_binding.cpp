// The serving operators' Python binding (module ktir_cpu_b200._serving).
//
// A call of few tokens keeps the GPU busy for a few microseconds, less than it
// takes to check nine tensors and fill a descriptor from Python (12 to 16 us).
// Here the same check reads the tensors directly; a call that does not pass it
// returns NotImplemented, and serving.py says what was wrong.  The module
// allocates outputs and workspaces and calls the C ABI; kernels are in
// libktir_b200.so.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <map>
#include <utility>

#include "../../include/ktir_b200.h"

namespace {

constexpr int MAX_DEVICES = 64;
at::Tensor g_status[MAX_DEVICES];                                  // touched under the GIL only
using Key = std::pair<int, cudaStream_t>;
struct Workspaces {
  int64_t parts;                            // bytes at the start that need not be zero; counters behind them
  std::map<Key, at::Tensor> kept;           // by device and stream
  struct Captured {
    unsigned long long capture = 0;
    at::Tensor t;
  };
  std::map<Key, Captured> captured;
};
Workspaces g_decode = {KTIR_PAGED_DECODE_PARTS_BYTES, {}, {}}, g_prompt = {KTIR_PROMPT_PARTS_BYTES, {}, {}};

struct Failed {};   // a Python exception is set

bool capturing() { return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None; }

int32_t* status_of(int dev) {
  at::Tensor& t = g_status[dev];
  if (!t.defined()) {
    if (capturing()) {
      PyErr_SetString(PyExc_RuntimeError, "call a serving operator once on this device before capturing it");
      throw Failed();
    }
    t = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, dev));
    c10::cuda::device_synchronize();   // whichever stream uses it next finds it cleared
  }
  return t.data_ptr<int32_t>();
}

int dtype_of(const at::Tensor& t) {
  return t.scalar_type() == at::kHalf ? KTIR_F16 : t.scalar_type() == at::kBFloat16 ? KTIR_BF16 : -1;
}

// one argument: a tensor, or none where that is allowed
struct Arg {
  const at::Tensor* t = nullptr;
  bool ok = true;
  Arg(PyObject* o, bool optional = false) {
    if (o == Py_None) {
      ok = optional;
    } else if (THPVariable_Check(o)) {
      t = &THPVariable_Unpack(o);
    } else {
      ok = false;
    }
  }
  explicit operator bool() const { return t != nullptr; }
  const at::Tensor* operator->() const { return t; }
  const at::Tensor& operator*() const { return *t; }
};

// Is a level of forward mode open?  Asked once per call: a look at each tensor's tangent
// costs append, whose arguments are views, 0.2 us.
bool g_forward = false;

// a gradient, or a tangent of forward mode, that the operators would lose
bool differentiated(const at::Tensor& t) {
  return (t.requires_grad() && at::GradMode::is_enabled()) || (g_forward && t._fw_grad(0).defined());
}

// a tensor of head vectors of the call's type and device
bool vectors(const at::Tensor& t, const at::Tensor& like, int dims) {
  return t.dim() == dims && t.scalar_type() == like.scalar_type() && t.device() == like.device() &&
         t.stride(dims - 1) == 1 && !differentiated(t);
}

// an int32 index array of n entries on the call's device
bool index(const at::Tensor& t, const at::Tensor& like, int64_t n) {
  return t.scalar_type() == at::kInt && t.device() == like.device() && t.dim() == 1 && t.size(0) == n &&
         (n <= 1 || t.stride(0) == 1);
}

template <int N>
void strides(int64_t (&to)[N], const at::Tensor& t) {
  for (int i = 0; i < N; ++i) to[i] = t.stride(i);
}

void check(int rc) {
  if (rc == KTIR_OK) return;
  PyErr_SetString(rc == KTIR_ERR_UNSUPPORTED ? PyExc_NotImplementedError
                  : rc == KTIR_ERR_ARG       ? PyExc_ValueError
                                             : PyExc_RuntimeError,
                  ktir_last_error());
  throw Failed();
}

PyObject* wrong() { Py_RETURN_NOTIMPLEMENTED; }

// a scale given as a number, or dim ** -0.5
float scale_of(PyObject* o, int64_t dim) {
  if (o == Py_None) return (float)(1.0 / std::sqrt((double)dim));
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Failed();
  return (float)v;
}

bool flag(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Failed();
  return v != 0;
}

// A new tensor, from the allocator without a way through the dispatcher (one token
// appended: 4.1 us a call against 4.6).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, device, c10::nullopt));
}

// a caller's tensor that was written: autograd sees that what it saved of it has changed
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Scratch for calls on one stream, which follow each other and leave its counters at
// zero, so that it is kept between them.  Calls that are being captured share one per
// capture and stream, from the graph's own memory: the graph may be replayed on any
// stream.  Its counters are cleared by a node before the first of them, in every
// replay; the ones after it begin early, as in a stream (32 times append and decode of
// 77 keys: 9.0 us a pair with a clear of the whole, 8.5 MB, in each call, 6.5 without).
at::Tensor workspace_of(Workspaces& w, int dev, cudaStream_t stream, int64_t bytes) {
  if (!capturing()) {
    at::Tensor& t = w.kept[{dev, stream}];
    if (!t.defined() || t.numel() < bytes)
      t = at::zeros({bytes + bytes / 4}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, dev));
    return t;
  }
  cudaStreamCaptureStatus status;
  unsigned long long capture = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(stream, &status, &capture));
  // what other captures had goes back to their graphs
  for (auto it = w.captured.begin(); it != w.captured.end();)
    it = it->second.capture != capture ? w.captured.erase(it) : std::next(it);
  Workspaces::Captured& c = w.captured[{dev, stream}];
  if (!c.t.defined() || c.t.numel() < bytes) {
    c.capture = capture;
    c.t = fresh({bytes}, at::kByte, at::Device(at::kCUDA, dev));
    C10_CUDA_CHECK(cudaMemsetAsync(static_cast<char*>(c.t.data_ptr()) + w.parts, 0, bytes - w.parts, stream));
  }
  return c.t;
}

// out (given, or new) of q's shape
bool output(const Arg& out, const at::Tensor& q, at::Tensor& o) {
  if (out) {
    if (!vectors(*out, q, 3) || !out->sizes().equals(q.sizes())) return false;
    o = *out;
  } else {
    o = fresh(q.sizes(), q.scalar_type(), q.device());
  }
  return true;
}

PyObject* result(PyObject* given, const at::Tensor& o, const at::Tensor& lse) {
  PyObject* r = given != Py_None ? Py_NewRef(given) : THPVariable_Wrap(o);
  if (!lse.defined() || !r) return r;
  PyObject* l = THPVariable_Wrap(lse);
  PyObject* pair = l ? PyTuple_Pack(2, r, l) : nullptr;
  Py_DECREF(r);
  Py_XDECREF(l);
  return pair;
}

// k, v, k_cache, v_cache, slots, q, positions, table, interleaved, q_out
PyObject* kv_append(PyObject* const* a) {
  const Arg k(a[0]), v(a[1]), kc(a[2]), vc(a[3]), slots(a[4]), q(a[5], true), pos(a[6], true), table(a[7], true),
      out(a[9], true);
  if (!(k.ok && v.ok && kc.ok && vc.ok && slots.ok && q.ok && pos.ok && table.ok && out.ok)) return wrong();
  const int dt = dtype_of(*k);
  if (dt < 0 || !k->is_cuda() || !vectors(*k, *k, 3) || !vectors(*v, *k, 3) || !vectors(*kc, *k, 4) ||
      !vectors(*vc, *k, 4) || !v->sizes().equals(k->sizes()) || !vc->sizes().equals(kc->sizes()) ||
      kc->size(2) != k->size(1) || kc->size(2) < 1 || kc->size(3) != k->size(2) || !index(*slots, *k, k->size(0)))
    return wrong();
  if ((bool)pos != (bool)table || (out && !q)) return wrong();
  if (table && (!index(*pos, *k, k->size(0)) || table->dim() != 2 || table->scalar_type() != at::kFloat ||
                table->device() != k->device() || table->stride(1) != 1 || differentiated(*table)))
    return wrong();
  at::Tensor o;
  if (q) {
    if (!vectors(*q, *k, 3) || q->size(0) != k->size(0) || q->size(2) != k->size(2)) return wrong();
    if (!output(out, *q, o)) return wrong();
  }
  KtirKvAppendDesc d = {};
  d.tokens = k->size(0);
  d.kv_heads = (int32_t)k->size(1);
  const bool turn_q = q && q->size(1) > 0;        // none to rotate: keys and values are written all the same
  d.heads = turn_q ? (int32_t)q->size(1) : d.kv_heads;
  if (d.tokens > 0) {
    const c10::cuda::CUDAGuard guard(k->device());
    d.k = k->data_ptr();
    d.v = v->data_ptr();
    d.k_cache = kc->data_ptr();
    d.v_cache = vc->data_ptr();
    d.slots = slots->data_ptr<int32_t>();
    d.status = status_of(k->get_device());
    strides(d.k_stride, *k);
    strides(d.v_stride, *v);
    strides(d.kc_stride, *kc);
    strides(d.vc_stride, *vc);
    d.num_pages = kc->size(0);
    d.page_size = kc->size(1);
    if (turn_q) {
      d.q = q->data_ptr();
      d.q_out = o.data_ptr();
      strides(d.q_stride, *q);
      strides(d.qo_stride, o);
    }
    if (table) {
      d.positions = pos->data_ptr<int32_t>();
      d.table = table->data_ptr<float>();
      d.table_rows = table->size(0);
      d.table_stride = table->stride(0);
      d.rot = (int32_t)table->size(1);
    }
    d.dim = (int32_t)k->size(2);
    d.interleaved = flag(a[8]);
    d.dtype = dt;
    check(ktir_kv_append(&d, c10::cuda::getCurrentCUDAStream(k->get_device()).stream()));
    written(*kc);
    written(*vc);
    if (turn_q && out) written(o);
  }
  if (!q) Py_RETURN_NONE;
  return result(a[9], o, at::Tensor());
}

// q, k_cache, v_cache, pages, lengths, scale, out, return_lse
PyObject* paged_decode(PyObject* const* a) {
  const Arg q(a[0]), kc(a[1]), vc(a[2]), pages(a[3]), lengths(a[4]), out(a[6], true);
  if (!(q.ok && kc.ok && vc.ok && pages.ok && lengths.ok && out.ok)) return wrong();
  const int dt = dtype_of(*q);
  if (dt < 0 || !q->is_cuda() || !vectors(*q, *q, 3) || !vectors(*kc, *q, 4) || !vectors(*vc, *q, 4) ||
      !vc->sizes().equals(kc->sizes()) || kc->size(3) != q->size(2) || kc->size(2) < 1 ||
      q->size(1) % kc->size(2) || pages->scalar_type() != at::kInt || pages->device() != q->device() ||
      pages->dim() != 2 || pages->size(0) != q->size(0) || (pages->size(1) > 1 && pages->stride(1) != 1) ||
      !index(*lengths, *q, q->size(0)))
    return wrong();
  at::Tensor o, lse;
  if (!output(out, *q, o)) return wrong();
  if (flag(a[7])) lse = fresh({q->size(0), q->size(1)}, at::kFloat, q->device());
  KtirPagedDecodeDesc d = {};
  d.batch = q->size(0);
  d.heads = (int32_t)q->size(1);
  if (d.batch > 0 && d.heads > 0) {
    const c10::cuda::CUDAGuard guard(q->device());
    const int dev = q->get_device();
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
    d.kv_heads = (int32_t)kc->size(2);
    d.dim = (int32_t)q->size(2);
    const at::Tensor ws =
        workspace_of(g_decode, dev, stream, ktir_paged_decode_workspace(d.batch, d.heads, d.kv_heads, d.dim));
    d.q = q->data_ptr();
    d.k_cache = kc->data_ptr();
    d.v_cache = vc->data_ptr();
    d.out = o.data_ptr();
    if (lse.defined()) d.lse = lse.data_ptr<float>();
    d.pages = pages->data_ptr<int32_t>();
    d.lengths = lengths->data_ptr<int32_t>();
    d.workspace = ws.data_ptr();
    d.workspace_bytes = ws.numel();
    d.status = status_of(dev);
    d.max_pages = pages->size(1);
    d.page_row = pages->stride(0);
    d.num_pages = kc->size(0);
    d.page_size = kc->size(1);
    strides(d.q_stride, *q);
    strides(d.out_stride, o);
    strides(d.kc_stride, *kc);
    strides(d.vc_stride, *vc);
    d.dtype = dt;
    d.scale = scale_of(a[5], q->size(2));
    check(ktir_paged_decode(&d, stream));
    if (out) written(o);
  }
  return result(a[6], o, lse);
}

// q, k, v, offsets, kv_offsets, causal, scale, out, return_lse
PyObject* prompt_attention(PyObject* const* a) {
  const Arg q(a[0]), k(a[1]), v(a[2]), offsets(a[3]), kv_offsets(a[4], true), out(a[7], true);
  if (!(q.ok && k.ok && v.ok && offsets.ok && kv_offsets.ok && out.ok)) return wrong();
  const int dt = dtype_of(*q);
  if (dt < 0 || !q->is_cuda() || !vectors(*q, *q, 3) || !vectors(*k, *q, 3) || !vectors(*v, *q, 3) ||
      !v->sizes().equals(k->sizes()) || k->size(2) != q->size(2) || k->size(1) < 1 || q->size(1) % k->size(1) ||
      offsets->dim() != 1 || offsets->size(0) < 2 || !index(*offsets, *q, offsets->size(0)) ||
      (kv_offsets ? !index(*kv_offsets, *q, offsets->size(0)) : k->size(0) != q->size(0)))
    return wrong();
  at::Tensor o, lse;
  if (!output(out, *q, o)) return wrong();
  if (flag(a[8])) lse = fresh({q->size(0), q->size(1)}, at::kFloat, q->device());
  KtirPromptDesc d = {};
  d.tokens = q->size(0);
  d.heads = (int32_t)q->size(1);
  if (d.tokens > 0 && d.heads > 0) {
    const c10::cuda::CUDAGuard guard(q->device());
    d.q = q->data_ptr();
    d.k = k->data_ptr();
    d.v = v->data_ptr();
    d.out = o.data_ptr();
    if (lse.defined()) d.lse = lse.data_ptr<float>();
    d.offsets = offsets->data_ptr<int32_t>();
    d.kv_offsets = kv_offsets ? kv_offsets->data_ptr<int32_t>() : d.offsets;
    const int dev = q->get_device();
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
    const at::Tensor ws = workspace_of(g_prompt, dev, stream, ktir_prompt_attention_workspace());
    d.workspace = ws.data_ptr();
    d.workspace_bytes = ws.numel();
    d.status = status_of(dev);
    d.batch = offsets->size(0) - 1;
    d.kv_tokens = k->size(0);
    strides(d.q_stride, *q);
    strides(d.k_stride, *k);
    strides(d.v_stride, *v);
    strides(d.out_stride, o);
    d.kv_heads = (int32_t)k->size(1);
    d.dim = (int32_t)q->size(2);
    d.dtype = dt;
    d.scale = scale_of(a[6], q->size(2));
    d.causal = flag(a[5]);
    check(ktir_prompt_attention(&d, stream));
    if (out) written(o);
  }
  return result(a[7], o, lse);
}

// the status word of a device, or None before its first call
PyObject* status(PyObject* const* a) {
  const long dev = PyLong_AsLong(a[0]);
  if (dev == -1 && PyErr_Occurred()) throw Failed();
  if (dev < 0 || dev >= MAX_DEVICES || !g_status[dev].defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(g_status[dev]);
}

// the kept workspaces of a device are given up: the next calls get cleared ones
PyObject* forget(PyObject* const* a) {
  const long dev = PyLong_AsLong(a[0]);
  if (dev == -1 && PyErr_Occurred()) throw Failed();
  for (auto* kept : {&g_decode.kept, &g_prompt.kept})
    for (auto it = kept->begin(); it != kept->end();) it = it->first.first == dev ? kept->erase(it) : std::next(it);
  Py_RETURN_NONE;
}

// no C++ exception leaves a call
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  HANDLE_TH_ERRORS
  try {
    g_forward = c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
                torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
    return F(args);
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject* const*), int N>
PyCFunction method() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>));
}

PyMethodDef g_methods[] = {
    {"kv_append", method<kv_append, 10>(), METH_FASTCALL, nullptr},
    {"paged_decode", method<paged_decode, 8>(), METH_FASTCALL, nullptr},
    {"prompt_attention", method<prompt_attention, 9>(), METH_FASTCALL, nullptr},
    {"status", method<status, 1>(), METH_FASTCALL, nullptr},
    {"forget", method<forget, 1>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&g_module); }
