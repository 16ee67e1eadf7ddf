// The plain form of the hot kernel shims in native code: tensors that need no conversion, no copy and no reshape go from the
// Python call to the C ABI (include/b200_lite_kernels.h) without ctypes and without Tensor attribute lookups in Python.  A
// decode step calls a few dozen shims, and a kernel takes 4 - 20 us: w8a16_matmul took 13.5 us of host time in Python (5 of
// them in ctypes and the launch), here 5.5; skip_rmsnorm 9.6 and 5.2.
//
// Every function returns None for anything else (other dimensions, strides, types or devices, a bias, tensor subclasses,
// wrapped or fake tensors, active torch modes): the Python shim then does what it always did, error messages included.  The
// results are those of the Python path: same kernels, same arguments, outputs without a gradient; exceptions too (torch's own
// translation: an allocation that fails is a torch.OutOfMemoryError, which the graph captures of ModelRunner wait for).
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <unordered_map>

namespace {

using i64 = int64_t;
struct {
  int64_t (*quant_workspace)(int, i64, i64, i64, i64);
  int64_t (*linear_workspace)(i64, i64, i64, int);
  int (*w8a16)(void*, const void*, const void*, int, const void*, const void*, int, i64, i64, i64, i64, i64, i64, i64, i64, i64,
               i64, void*, i64, void*, i64, void*);
  int (*w4a16)(void*, const void*, const void*, const void*, const void*, const void*, int, i64, i64, i64, int, int, i64, i64, i64,
               void*, i64, void*, i64, int, void*);
  int (*linear)(void*, const void*, const void*, const void*, i64, i64, i64, i64, i64, i64, void*, i64, void*, i64, int, void*);
  int (*w8a8)(void*, const void*, const void*, const void*, const void*, const void*, i64, i64, i64, i64, i64, i64, void*, i64,
              void*, i64, int, void*);
  int (*quantize)(void*, void*, const void*, i64, i64, i64, i64, int, void*);
  int (*norm)(void*, const void*, void*, const void*, i64, i64, i64, i64, i64, float, int, void*);
  int (*norm_quant)(void*, void*, const void*, void*, const void*, i64, i64, i64, i64, i64, float, int, void*);
  int (*swiglu)(void*, const void*, const void*, i64, i64, i64, i64, i64, int, void*);
  int64_t (*kv4_row_bytes)(int, int, int);
  int (*kv4_write)(void*, void*, const void*, const void*, const void*, const void*, const void*, const void*, int, void*, i64, i64, i64, i64,
                   int, int, int, int, i64, i64, i64, i64, i64, i64, i64, i64, i64, i64, i64, i64, int, void*);
  int (*kv4_read)(void*, const void*, i64, i64, const void*, int, i64, int, int, int, int, void*);
  int64_t (*kv4_decode_workspace)(i64, int, int, int, int, i64);
  int (*kv4_decode)(void*, const void*, const void*, i64, i64, const void*, i64, i64, i64, i64, const void*, int, const void*, int, i64, int,
                    int, int, int, i64, float, i64, i64, i64, i64, void*, i64, int, void*);
  int64_t (*kv4_prompt_workspace)(i64, i64, int, int, int, int, i64);
  int (*kv4_prompt)(void*, const void*, const void*, i64, i64, const void*, int, const void*, int, const void*, i64, i64, i64, i64, const void*,
                    int, const void*, int, i64, i64, i64, int, int, int, int, i64, float, i64, i64, i64, i64, void*, i64, int, void*);
  int (*slot_maps)(void*, void*, void*, void*, const void*, int, const void*, int, const void*, int, const void*, int, void*, i64, i64, i64,
                   i64, i64, i64, void*);
  int (*weights_written)(void*);
  i64 (*mx4_scale_bytes)(i64, i64);
  int (*mx4_quantize)(void*, void*, const void*, i64, i64, i64, i64, int, void*);
  int (*mx4_dequantize)(void*, const void*, const void*, i64, i64, i64, i64, int, void*);
  int (*mx4_norm)(void*, void*, void*, const void*, const void*, const void*, i64, i64, i64, i64, i64, float, int, void*);
  int (*mx4_matmul)(void*, void*, const void*, const void*, const void*, const void*, const void*, i64, i64, i64, i64, i64, i64, int, int, int,
                    void*);
  i64 (*mx4_takes_16bit)(i64, i64, i64);
  i64 (*mx4_tile_rows)(i64, int, i64);
  i64 (*mx4_max_tiles)(i64, int, int);
  int (*mx4_scatter)(void*, void*, void*, void*, const void*, const void*, int, i64, int, int, int, i64, i64, int, void*);
  int (*mx4_grouped)(void*, void*, const void*, const void*, const void*, const void*, const void*, i64, int, int, i64, i64, int, void*);
  int (*mx4_combine)(void*, const void*, const void*, const void*, const void*, int, i64, int, i64, int, void*);
  const char* (*last_error)();
} abi;
PyObject* py_zeroed = nullptr;      // kernels._common.zeroed_workspace(bytes, device)
PyObject* py_counters = nullptr;    // kernels._common.counters(device)
PyObject* py_mxfp4 = nullptr;       // kernels.quantization.mxfp4.MXFP4

// ---- which calls are plain ----
constexpr c10::DispatchKeySet kPlainKeys({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA, c10::DispatchKey::AutocastCUDA,
                                          c10::DispatchKey::ADInplaceOrView});

// a dense CUDA tensor that is exactly a torch.Tensor (or Parameter); nullptr otherwise
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && (t.key_set().raw_repr() & ~kPlainKeys.raw_repr()) == 0 && t.is_cuda() ? &t : nullptr;
}
// the current device if every tensor is plain and there, and no mode wants to see the call; -1 otherwise.  A missing function
// (a library built from a subset of the sources) counts as not plain: the Python shim names it.
template <class F>
int device_for(F* fn, std::initializer_list<const at::Tensor*> ts) {
  if (!fn || c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled()) return -1;
  for (const at::Tensor* t : ts)
    if (!t) return -1;
  const int device = c10::cuda::current_device();
  for (const at::Tensor* t : ts)
    if (t->get_device() != device) return -1;
  return device;
}
// ctypes lets other threads run while a launch waits for room in its queue; so does this
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};
int half_code(const at::Tensor& t) { return t.scalar_type() == at::kHalf ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : -1; }
// matrix with unit column stride and at least one element
bool matrix(const at::Tensor& t) { return t.dim() == 2 && t.stride(1) == 1 && t.size(0) > 0 && t.size(1) > 0; }
// activation rows as TMA reads them
bool tma_rows(const at::Tensor& t) { return matrix(t) && t.stride(0) % 8 == 0 && (uintptr_t)t.data_ptr() % 16 == 0; }

PyObject* none() { Py_RETURN_NONE; }
PyObject* failed(int rc) {
  PyErr_Format(PyExc_ValueError, "b200lite error %d: %s", rc, abi.last_error());
  return nullptr;
}
void* stream(int device) { return (void*)c10::cuda::getCurrentCUDAStream(device).stream(); }

// The persistent buffers of kernels/_common.py, one per device; asked for again when a call needs more than before.
struct Kept { at::Tensor zeroed, counters; };
std::unordered_map<int, Kept>& kept() {
  static auto* m = new std::unordered_map<int, Kept>;      // outlives the interpreter's module teardown
  return *m;
}
bool fetch(PyObject* fn, PyObject* args, at::Tensor& out) {
  if (!args) return false;
  PyObject* r = PyObject_CallObject(fn, args);
  Py_DECREF(args);
  if (!r) return false;
  const bool ok = THPVariable_Check(r);
  if (ok) out = THPVariable_Unpack(r);
  Py_DECREF(r);
  if (!ok) PyErr_SetString(PyExc_RuntimeError, "buffer is not a tensor");
  return ok;
}
PyObject* device_of(PyObject* tensor) { return PyObject_GetAttrString(tensor, "device"); }
bool need_counters(int device, PyObject* like, Kept& k) {
  if (k.counters.defined()) return true;
  return fetch(py_counters, Py_BuildValue("(N)", device_of(like)), k.counters);
}
bool need_zeroed(i64 bytes, PyObject* like, Kept& k) {
  if (bytes <= 0 || (k.zeroed.defined() && k.zeroed.numel() >= bytes)) return true;
  return fetch(py_zeroed, Py_BuildValue("(LN)", (long long)bytes, device_of(like)), k.zeroed);
}

// workspace of a quantised GEMM, remembered by its sizes (the plan walks over the tiles); bounded
struct Sizes {
  i64 kind, m, n, k, group, device;
  bool operator==(const Sizes& o) const { return kind == o.kind && m == o.m && n == o.n && k == o.k && group == o.group && device == o.device; }
};
struct Hash {
  size_t operator()(const Sizes& s) const {
    size_t h = 1469598103934665603ull;
    for (i64 v : {s.kind, s.m, s.n, s.k, s.group, s.device}) h = (h ^ (size_t)v) * 1099511628211ull;
    return h;
  }
};
i64 quant_workspace(int kind, i64 m, i64 n, i64 k, i64 group, int device) {
  static auto* seen = new std::unordered_map<Sizes, i64, Hash>;
  const Sizes s{kind, m, n, k, group, device};
  auto it = seen->find(s);
  if (it != seen->end()) return it->second;
  if (seen->size() >= 4096) seen->clear();
  return (*seen)[s] = abi.quant_workspace(kind, m, n, k, group);
}

// Torch's translation of exceptions, without the buffer for warnings of HANDLE_TH_ERRORS: nothing here warns.
#define FAST_BEGIN try {
#define FAST_END                                                      \
  }                                                                   \
  catch (...) {                                                       \
    torch::translate_exception_to_python(std::current_exception());   \
    return nullptr;                                                   \
  }
#define ARGS(n) \
  if (count != (n)) { PyErr_SetString(PyExc_TypeError, "wrong number of arguments"); return nullptr; }

// (x, qweight, scales, group_n, group_k) -> y
PyObject* w8a16(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(5)
  FAST_BEGIN
  const at::Tensor *x = plain(a[0]), *q = plain(a[1]), *s = plain(a[2]);
  const int device = device_for(abi.w8a16, {x, q, s});
  if (device < 0 || !PyLong_CheckExact(a[3]) || !PyLong_CheckExact(a[4])) return none();
  const bool fp8 = q->scalar_type() == at::kByte;
  if ((!fp8 && q->scalar_type() != at::kChar) || x->scalar_type() != at::kHalf || s->scalar_type() != at::kFloat) return none();
  if (!tma_rows(*x) || !matrix(*q) || s->dim() != 2 || x->size(1) != q->size(1)) return none();
  const i64 gn = PyLong_AsLongLong(a[3]), gk = PyLong_AsLongLong(a[4]), m = x->size(0), n = q->size(0), k = q->size(1);
  if (PyErr_Occurred()) return nullptr;
  if (gn < 1 || gk < 1 || (gk % 128 != 0 && gk < k)) return none();
  Kept& kp = kept()[device];
  const int kind = fp8 ? 1 : 2;
  const i64 bytes = quant_workspace(kind, m, n, k, gk, device);
  if (!need_zeroed(bytes, a[0], kp) || !need_counters(device, a[0], kp)) return nullptr;
  void* zeroed = bytes > 0 ? kp.zeroed.data_ptr() : nullptr;
  void* tickets = kp.counters.data_ptr();
  const i64 num_tickets = kp.counters.numel();
  at::Tensor y;
  int rc;
  {
    const Unlocked unlocked;
    y = at::empty({m, n}, x->options());
    rc = abi.w8a16(y.data_ptr(), x->data_ptr(), q->data_ptr(), fp8 ? 1 : 0, s->data_ptr(), nullptr, 0, m, n, k, gn, gk,
                   x->stride(0), q->stride(0), s->stride(0), s->stride(1), n, zeroed,
                   bytes, tickets, num_tickets, stream(device));
  }
  return rc ? failed(rc) : THPVariable_Wrap(std::move(y));
  FAST_END
}

// (x, qweight, scales, zeros, n, k, group_size, zeros_foldable, swiglu) -> y
PyObject* w4a16_packed(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(9)
  FAST_BEGIN
  const at::Tensor *x = plain(a[0]), *q = plain(a[1]), *s = plain(a[2]), *z = plain(a[3]);
  const int device = device_for(abi.w4a16, {x, q, s, z});
  if (device < 0) return none();
  for (int i = 4; i < 7; ++i)
    if (!PyLong_CheckExact(a[i])) return none();
  const i64 n = PyLong_AsLongLong(a[4]), k = PyLong_AsLongLong(a[5]), group = PyLong_AsLongLong(a[6]);
  const int fold = PyObject_IsTrue(a[7]), swiglu = PyObject_IsTrue(a[8]);
  if (PyErr_Occurred()) return nullptr;
  if (x->scalar_type() != at::kHalf || !tma_rows(*x) || x->size(1) != k || q->dim() != 2) return none();
  const i64 m = x->size(0), out = swiglu ? n / 2 : n;
  Kept& kp = kept()[device];
  const i64 bytes = quant_workspace(0, m, n, k, group, device);
  if (!need_zeroed(bytes, a[0], kp) || !need_counters(device, a[0], kp)) return nullptr;
  void* zeroed = bytes > 0 ? kp.zeroed.data_ptr() : nullptr;
  void* tickets = kp.counters.data_ptr();
  const i64 num_tickets = kp.counters.numel();
  at::Tensor y;
  int rc;
  {
    const Unlocked unlocked;
    y = at::empty({m, out}, x->options());
    rc = abi.w4a16(y.data_ptr(), x->data_ptr(), q->data_ptr(), s->data_ptr(), z->data_ptr(), nullptr, 0, m, n, k, (int)group,
                   fold, x->stride(0), q->stride(0), out, zeroed, bytes,
                   tickets, num_tickets, swiglu, stream(device));
  }
  return rc ? failed(rc) : THPVariable_Wrap(std::move(y));
  FAST_END
}

// (x, weight) -> y
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(2)
  FAST_BEGIN
  const at::Tensor *x = plain(a[0]), *w = plain(a[1]);
  const int device = device_for(abi.linear, {x, w});
  if (device < 0) return none();
  const int code = half_code(*x);
  if (code < 0 || w->scalar_type() != x->scalar_type() || !tma_rows(*x) || !matrix(*w) || x->size(1) % 8 != 0 || x->size(1) != w->size(1))
    return none();
  const i64 m = x->size(0), n = w->size(0), k = w->size(1), bytes = abi.linear_workspace(m, n, k, 2);
  Kept& kp = kept()[device];
  if (!need_counters(device, a[0], kp)) return nullptr;
  void* tickets = kp.counters.data_ptr();
  const i64 num_tickets = kp.counters.numel();
  at::Tensor y, ws;
  int rc;
  {
    const Unlocked unlocked;
    y = at::empty({m, n}, x->options());
    if (bytes > 0) ws = at::empty({bytes}, x->options().dtype(at::kByte));
    rc = abi.linear(y.data_ptr(), x->data_ptr(), w->data_ptr(), nullptr, m, n, k, x->stride(0), w->stride(0), n,
                    bytes > 0 ? ws.data_ptr() : nullptr, bytes, tickets, num_tickets, code, stream(device));
  }
  return rc ? failed(rc) : THPVariable_Wrap(std::move(y));
  FAST_END
}

// (qa, a_scales, qweight, weight_scales [N] or [N, 1], bfloat16 out) -> y
PyObject* w8a8(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(5)
  FAST_BEGIN
  const at::Tensor *x = plain(a[0]), *sa = plain(a[1]), *w = plain(a[2]), *sw = plain(a[3]);
  const int device = device_for(abi.w8a8, {x, sa, w, sw});
  if (device < 0) return none();
  const int bf16 = PyObject_IsTrue(a[4]);
  if (bf16 < 0) return nullptr;
  if (x->scalar_type() != at::kChar || w->scalar_type() != at::kChar || sa->scalar_type() != at::kFloat || sw->scalar_type() != at::kFloat)
    return none();
  if (!matrix(*x) || !matrix(*w) || x->size(1) != w->size(1) || x->size(1) % 16 != 0 || w->stride(0) % 16 != 0) return none();
  const i64 m = x->size(0), n = w->size(0), k = w->size(1);
  if (!sa->is_contiguous() || !sw->is_contiguous() || sw->dim() > 2 || (sw->dim() == 2 && sw->size(1) != 1)) return none();
  const i64 bytes = abi.linear_workspace(m, n, k, 1);
  Kept& kp = kept()[device];
  if (!need_counters(device, a[0], kp)) return nullptr;
  void* tickets = kp.counters.data_ptr();
  const i64 num_tickets = kp.counters.numel();
  at::Tensor y, ws;
  int rc;
  {
    const Unlocked unlocked;
    y = at::empty({m, n}, x->options().dtype(bf16 ? at::kBFloat16 : at::kHalf));
    if (bytes > 0) ws = at::empty({bytes}, x->options().dtype(at::kByte));
    rc = abi.w8a8(y.data_ptr(), x->data_ptr(), w->data_ptr(), sa->data_ptr(), sw->data_ptr(), nullptr, m, n, k, x->stride(0),
                  w->stride(0), n, bytes > 0 ? ws.data_ptr() : nullptr, bytes, tickets, num_tickets,
                  bf16, stream(device));
  }
  return rc ? failed(rc) : THPVariable_Wrap(std::move(y));
  FAST_END
}

PyObject* pair_of(at::Tensor a, at::Tensor b) {
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(a)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(b)));
  return r;
}

// (a) -> (q, scales)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(1)
  FAST_BEGIN
  const at::Tensor* x = plain(a[0]);
  const int device = device_for(abi.quantize, {x});
  if (device < 0) return none();
  const int code = half_code(*x);
  if (code < 0 || !matrix(*x)) return none();
  const i64 m = x->size(0), k = x->size(1);
  at::Tensor q, s;
  int rc;
  {
    const Unlocked unlocked;
    q = at::empty({m, k}, x->options().dtype(at::kChar));
    s = at::empty({m}, x->options().dtype(at::kFloat));
    rc = abi.quantize(q.data_ptr(), s.data_ptr(), x->data_ptr(), m, k, x->stride(0), k, code, stream(device));
  }
  return rc ? failed(rc) : pair_of(std::move(q), std::move(s));
  FAST_END
}

// rows of the norms: contiguous matrices that the results may alias
bool norm_rows(const at::Tensor& x, PyObject* res, const at::Tensor* r, const at::Tensor& w) {
  if (x.dim() != 2 || x.size(0) == 0 || x.size(1) == 0 || x.requires_grad() || !x.is_contiguous() || half_code(x) < 0) return false;
  if (w.scalar_type() != x.scalar_type() || !w.is_contiguous()) return false;
  if (res == Py_None) return true;
  return r && r->scalar_type() == x.scalar_type() && r->sizes() == x.sizes() && !r->requires_grad() && r->is_contiguous();
}

// (X, residual or None, weight, eps) -> (Y, residual or X)
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(4)
  FAST_BEGIN
  const at::Tensor *x = plain(a[0]), *r = a[1] == Py_None ? nullptr : plain(a[1]), *w = plain(a[2]);
  const int device = r ? device_for(abi.norm, {x, w, r}) : device_for(abi.norm, {x, w});
  if (device < 0 || !PyFloat_CheckExact(a[3]) || !norm_rows(*x, a[1], r, *w)) return none();
  const i64 rows = x->size(0), n = x->size(1);
  at::Tensor y;
  int rc;
  {
    const Unlocked unlocked;
    y = at::empty({rows, n}, x->options());
    rc = abi.norm(y.data_ptr(), x->data_ptr(), r ? r->data_ptr() : nullptr, w->data_ptr(), rows, n, n, n, n,
                  (float)PyFloat_AS_DOUBLE(a[3]), half_code(*x), stream(device));
  }
  if (rc) return failed(rc);
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(y)));
  PyTuple_SET_ITEM(out, 1, Py_NewRef(r ? a[1] : a[0]));
  return out;
  FAST_END
}

// (X, residual or None, weight, eps) -> (q, scales)
PyObject* norm_quant(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(4)
  FAST_BEGIN
  const at::Tensor *x = plain(a[0]), *r = a[1] == Py_None ? nullptr : plain(a[1]), *w = plain(a[2]);
  const int device = r ? device_for(abi.norm_quant, {x, w, r}) : device_for(abi.norm_quant, {x, w});
  if (device < 0 || !PyFloat_CheckExact(a[3]) || !norm_rows(*x, a[1], r, *w)) return none();
  const i64 rows = x->size(0), n = x->size(1);
  if (n % 8 != 0 || n > 16384) return none();
  at::Tensor q, s;
  int rc;
  {
    const Unlocked unlocked;
    q = at::empty({rows, n}, x->options().dtype(at::kChar));
    s = at::empty({rows}, x->options().dtype(at::kFloat));
    rc = abi.norm_quant(q.data_ptr(), s.data_ptr(), x->data_ptr(), r ? r->data_ptr() : nullptr, w->data_ptr(), rows, n, n, n, n,
                        (float)PyFloat_AS_DOUBLE(a[3]), half_code(*x), stream(device));
  }
  return rc ? failed(rc) : pair_of(std::move(q), std::move(s));
  FAST_END
}

// (a, b) -> silu(a) * b
PyObject* swiglu(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(2)
  FAST_BEGIN
  const at::Tensor *g = plain(a[0]), *u = plain(a[1]);
  const int device = device_for(abi.swiglu, {g, u});
  if (device < 0) return none();
  const int code = g->scalar_type() == at::kFloat ? 2 : half_code(*g);
  if (code < 0 || u->scalar_type() != g->scalar_type() || !matrix(*g) || !matrix(*u) || g->sizes() != u->sizes()) return none();
  const i64 rows = g->size(0), n = g->size(1);
  at::Tensor y;
  int rc;
  {
    const Unlocked unlocked;
    y = at::empty({rows, n}, g->options());
    rc = abi.swiglu(y.data_ptr(), g->data_ptr(), u->data_ptr(), rows, n, g->stride(0), u->stride(0), n, code, stream(device));
  }
  return rc ? failed(rc) : THPVariable_Wrap(std::move(y));
  FAST_END
}

// ---- the cache in 4 bits and slot maps (kernels/kv_int4.py, kernels/slot_maps.py) ----
// heads inside token rows, unit stride in a head; at least one element
bool heads3(const at::Tensor& t) { return t.dim() == 3 && t.stride(2) == 1 && t.numel() > 0; }
// bytes of an index vector's elements: 4 or 8; 0 for anything but a contiguous vector of n
int indices(const at::Tensor& t, i64 n) {
  if (t.dim() != 1 || t.size(0) != n || !t.is_contiguous()) return 0;
  return t.scalar_type() == at::kInt ? 4 : t.scalar_type() == at::kLong ? 8 : 0;
}
bool table2(const at::Tensor& t) { return t.dim() == 2 && t.scalar_type() == at::kInt; }
// rows of a 4-bit cache that hold such heads
bool cache4(const at::Tensor& t, i64 heads, i64 d, i64 group) {
  if (t.scalar_type() != at::kByte || t.dim() != 2 || t.stride(1) != 1 || t.size(0) < 2 || t.stride(0) < t.size(1)) return false;
  if (heads < 1 || heads > 65535 || d > 65535 || group < 1 || group > 65535) return false;
  const i64 need = abi.kv4_row_bytes((int)heads, (int)d, (int)group);
  return need > 0 && t.size(1) >= need;
}
// whole numbers from Python; false: one of them is something else
bool numbers(PyObject* const* a, std::initializer_list<int> at, i64* to) {
  for (int i : at) {
    if (!PyLong_CheckExact(a[i])) return false;
    *to = PyLong_AsLongLong(a[i]);
    if (*to == -1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    ++to;
  }
  return true;
}

// (q, k, v, cos, sin, select_index, kv_buffer, batch, seq, group, out_q or None, out_k or None) -> (out_q or q, out_k or k)
PyObject* kv4_rope_write(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(12)
  FAST_BEGIN
  const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]), *c = plain(a[3]), *s = plain(a[4]), *idx = plain(a[5]), *kv = plain(a[6]);
  const at::Tensor *oq = a[10] == Py_None ? q : plain(a[10]), *ok = a[11] == Py_None ? k : plain(a[11]);
  const int device = device_for(abi.kv4_write, {q, k, v, c, s, idx, kv, oq, ok});
  i64 n[3];
  if (device < 0 || !numbers(a, {7, 8, 9}, n)) return none();
  const int code = half_code(*q);
  if (code < 0 || !heads3(*q) || !heads3(*k) || !heads3(*v) || !heads3(*oq) || !heads3(*ok)) return none();
  for (const at::Tensor* t : {k, v, c, s, oq, ok})
    if (t->scalar_type() != q->scalar_type()) return none();
  const i64 tokens = q->size(0), hq = q->size(1), d = q->size(2), hkv = k->size(1);
  if (n[0] < 1 || n[1] < 1 || n[0] > tokens || n[1] > tokens || n[0] * n[1] != tokens || k->size(0) != tokens || k->size(2) != d || v->sizes() != k->sizes() ||
      oq->sizes() != q->sizes() || ok->sizes() != k->sizes())
    return none();
  if (c->dim() != 3 || c->sizes() != s->sizes() || c->strides() != s->strides() || c->stride(2) != 1 || c->size(0) != n[0] || c->size(1) != n[1] ||
      c->size(2) < d / 2)
    return none();
  const int width = indices(*idx, tokens);
  if (!width || !cache4(*kv, hkv, d, n[2])) return none();
  int rc;
  {
    const Unlocked unlocked;
    rc = abi.kv4_write(oq->data_ptr(), ok->data_ptr(), q->data_ptr(), k->data_ptr(), v->data_ptr(), c->data_ptr(), s->data_ptr(), idx->data_ptr(),
                       width, kv->data_ptr(), kv->stride(0), kv->size(0), tokens, n[1], (int)hq, (int)hkv, (int)d, (int)n[2], q->stride(0),
                       q->stride(1), k->stride(0), k->stride(1), v->stride(0), v->stride(1), c->stride(0), c->stride(1), oq->stride(0),
                       oq->stride(1), ok->stride(0), ok->stride(1), code, stream(device));
  }
  if (rc) return failed(rc);
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, Py_NewRef(a[10] == Py_None ? a[0] : a[10]));
  PyTuple_SET_ITEM(out, 1, Py_NewRef(a[11] == Py_None ? a[1] : a[11]));
  return out;
  FAST_END
}

// (kv_buffer, select_index, kv heads, head_dim, dtype, group) -> values
PyObject* kv4_read(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(6)
  FAST_BEGIN
  const at::Tensor *kv = plain(a[0]), *idx = plain(a[1]);
  const int device = device_for(abi.kv4_read, {kv, idx});
  i64 n[3];
  if (device < 0 || !numbers(a, {2, 3, 5}, n) || !THPDtype_Check(a[4])) return none();
  const at::ScalarType type = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
  if ((type != at::kHalf && type != at::kBFloat16) || idx->dim() != 1 || idx->size(0) < 1 || !cache4(*kv, n[0], n[1], n[2])) return none();
  const i64 tokens = idx->size(0);
  const int width = indices(*idx, tokens);
  if (!width) return none();
  at::Tensor out;
  int rc;
  {
    const Unlocked unlocked;
    out = at::empty({tokens, 2 * n[0], n[1]}, kv->options().dtype(type));
    rc = abi.kv4_read(out.data_ptr(), kv->data_ptr(), kv->stride(0), kv->size(0), idx->data_ptr(), width, tokens, (int)n[0], (int)n[1], (int)n[2],
                      half_code(out), stream(device));
  }
  return rc ? failed(rc) : THPVariable_Wrap(std::move(out));
  FAST_END
}

// (q, kv_buffer, scale, table, req_idx, seq_len, max_len, kv heads, group, out or None) -> out
PyObject* kv4_decode(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(10)
  FAST_BEGIN
  const at::Tensor *q = plain(a[0]), *kv = plain(a[1]), *table = plain(a[3]), *req = plain(a[4]), *len = plain(a[5]);
  const at::Tensor* given = a[9] == Py_None ? q : plain(a[9]);
  const int device = device_for(abi.kv4_decode, {q, kv, table, req, len, given});
  i64 n[3];
  if (device < 0 || !PyFloat_CheckExact(a[2]) || !numbers(a, {6, 7, 8}, n)) return none();
  const int code = half_code(*q);
  if (code < 0 || !heads3(*q) || !table2(*table)) return none();
  const i64 batch = q->size(0), hq = q->size(1), d = q->size(2);
  const int rw = indices(*req, batch), lw = indices(*len, batch);
  if (!rw || !lw || !cache4(*kv, n[1], d, n[2]) || hq % n[1] != 0) return none();
  if (given != q && (given->scalar_type() != q->scalar_type() || given->sizes() != q->sizes() || given->stride(2) != 1)) return none();
  const i64 bytes = abi.kv4_decode_workspace(batch, (int)hq, (int)n[1], (int)d, (int)n[2], n[0]);
  at::Tensor out, ws;
  int rc;
  {
    const Unlocked unlocked;
    out = a[9] == Py_None ? at::empty({batch, hq, d}, q->options()) : *given;
    ws = at::empty({bytes > 16 ? bytes : 16}, q->options().dtype(at::kByte));
    rc = abi.kv4_decode(out.data_ptr(), q->data_ptr(), kv->data_ptr(), kv->stride(0), kv->size(0), table->data_ptr(), table->stride(0),
                        table->stride(1), table->size(0), table->size(1), req->data_ptr(), rw, len->data_ptr(), lw, batch, (int)hq, (int)n[1],
                        (int)d, (int)n[2], n[0], (float)PyFloat_AS_DOUBLE(a[2]), q->stride(0), q->stride(1), out.stride(0), out.stride(1), ws.data_ptr(), bytes,
                        code, stream(device));
  }
  if (rc) return failed(rc);
  return a[9] == Py_None ? THPVariable_Wrap(std::move(out)) : Py_NewRef(a[9]);
  FAST_END
}

// (q, kv_buffer, scale, start, new_len, table, req_idx, seq_len, max_new, max_len, kv heads, group, out or None) -> out
PyObject* kv4_prompt(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(13)
  FAST_BEGIN
  const at::Tensor *q = plain(a[0]), *kv = plain(a[1]), *start = plain(a[3]), *fresh = plain(a[4]), *table = plain(a[5]), *req = plain(a[6]),
                   *len = plain(a[7]);
  const at::Tensor* given = a[12] == Py_None ? q : plain(a[12]);
  const int device = device_for(abi.kv4_prompt, {q, kv, start, fresh, table, req, len, given});
  i64 n[4];
  if (device < 0 || !PyFloat_CheckExact(a[2]) || !numbers(a, {8, 9, 10, 11}, n)) return none();
  const int code = half_code(*q);
  if (code < 0 || !heads3(*q) || !table2(*table) || req->dim() != 1 || req->size(0) < 1) return none();
  const i64 tokens = q->size(0), hq = q->size(1), d = q->size(2), batch = req->size(0);
  const int sw = indices(*start, batch), fw = indices(*fresh, batch), rw = indices(*req, batch), lw = indices(*len, batch);
  if (!sw || !fw || !rw || !lw || !cache4(*kv, n[2], d, n[3]) || hq % n[2] != 0) return none();
  if (given != q && (given->scalar_type() != q->scalar_type() || given->sizes() != q->sizes() || given->stride(2) != 1)) return none();
  const i64 bytes = abi.kv4_prompt_workspace(batch, tokens, (int)hq, (int)n[2], (int)d, (int)n[3], n[1]);
  at::Tensor out, ws;
  int rc;
  {
    const Unlocked unlocked;
    out = a[12] == Py_None ? at::empty({tokens, hq, d}, q->options()) : *given;
    ws = at::empty({bytes > 16 ? bytes : 16}, q->options().dtype(at::kByte));
    rc = abi.kv4_prompt(out.data_ptr(), q->data_ptr(), kv->data_ptr(), kv->stride(0), kv->size(0), start->data_ptr(), sw, fresh->data_ptr(), fw,
                        table->data_ptr(), table->stride(0), table->stride(1), table->size(0), table->size(1), req->data_ptr(), rw,
                        len->data_ptr(), lw, batch, tokens, n[0], (int)hq, (int)n[2], (int)d, (int)n[3], n[1], (float)PyFloat_AS_DOUBLE(a[2]),
                        q->stride(0), q->stride(1), out.stride(0), out.stride(1), ws.data_ptr(), bytes, code, stream(device));
  }
  if (rc) return failed(rc);
  return a[12] == Py_None ? THPVariable_Wrap(std::move(out)) : Py_NewRef(a[12]);
  FAST_END
}

// (req_idx, ctx_len, new_len, table, total, rows or None) -> (select_index, position_ids, start, length)
PyObject* slot_maps(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(6)
  FAST_BEGIN
  const at::Tensor *req = plain(a[0]), *ctx = plain(a[1]), *fresh = plain(a[2]), *table = plain(a[3]);
  const at::Tensor* pool = a[5] == Py_None ? table : plain(a[5]);
  const int device = device_for(abi.slot_maps, {req, ctx, fresh, table, pool});
  i64 total;
  if (device < 0 || !numbers(a, {4}, &total) || total < 1 || req->dim() != 1 || req->size(0) < 1 || !table2(*table)) return none();
  const i64 batch = req->size(0);
  const int rw = indices(*req, batch), cw = indices(*ctx, batch), fw = indices(*fresh, batch);
  if (!rw || !cw || !fw) return none();
  int pw = 4;
  if (pool != table && (pool->dim() != 1 || pool->size(0) < total || !(pw = indices(*pool, pool->size(0))))) return none();
  at::Tensor rows, position, start, length;
  int rc;
  {
    const Unlocked unlocked;
    const auto i32 = table->options();
    rows = at::empty({total}, i32);
    position = at::empty({total}, i32.dtype(at::kLong));
    start = at::empty({batch}, i32);
    length = at::empty({batch}, i32);
    rc = abi.slot_maps(rows.data_ptr(), position.data_ptr(), start.data_ptr(), length.data_ptr(), req->data_ptr(), rw, ctx->data_ptr(), cw,
                       fresh->data_ptr(), fw, pool == table ? nullptr : pool->data_ptr(), pw, table->data_ptr(), table->stride(0),
                       table->stride(1), table->size(0), table->size(1), batch, total, stream(device));
  }
  if (rc) return failed(rc);
  PyObject* out = PyTuple_New(4);
  if (!out) return nullptr;
  int i = 0;
  for (at::Tensor* t : {&rows, &position, &start, &length}) PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(std::move(*t)));
  return out;
  FAST_END
}

// ---- microscaled 4-bit operands (kernels/quantization/mxfp4.py) ----
// An MXFP4 (a named tuple) of one matrix or a stack: the tensors as the class describes them.
struct Mx4 { const at::Tensor *codes = nullptr, *scales = nullptr; bool ready = false; i64 lead = 1, rows = 0, k = 0; };
i64 up(i64 n, i64 to) { return (n + to - 1) / to; }
bool mx4(PyObject* o, i64 dims, Mx4& m) {
  if (!PyTuple_Check(o) || PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != 3) return false;
  const at::Tensor *c = plain(PyTuple_GET_ITEM(o, 0)), *s = plain(PyTuple_GET_ITEM(o, 1));
  if (!c || !s || c->scalar_type() != at::kByte || s->scalar_type() != at::kByte || c->dim() != dims || s->dim() != dims + 3) return false;
  if (!c->is_contiguous() || !s->is_contiguous() || c->numel() == 0 || (uintptr_t)c->data_ptr() % 16 || (uintptr_t)s->data_ptr() % 16) return false;
  m.rows = c->size(dims - 2);
  m.k = 2 * c->size(dims - 1);
  m.lead = dims == 3 ? c->size(0) : 1;
  if (m.k % 32 != 0 || (dims == 3 && s->size(0) != m.lead)) return false;
  const i64 want[5] = {up(m.rows, 128), up(m.k, 128), 32, 4, 4};
  for (int i = 0; i < 5; ++i)
    if (s->size(dims - 2 + i) != want[i]) return false;
  m.codes = c;
  m.scales = s;
  m.ready = PyTuple_GET_ITEM(o, 2) == Py_True;
  return true;
}
// rows of activations that the quantiser reads as they are
bool mx4_rows(const at::Tensor& x, bool wide) {
  if (!matrix(x) || x.size(1) % 32 != 0 || (half_code(x) < 0 && !(wide && x.scalar_type() == at::kFloat))) return false;
  return (uintptr_t)x.data_ptr() % 16 == 0 && x.stride(0) >= 0 && x.stride(0) * x.element_size() % 16 == 0;
}
// A contiguous tensor on the current device, which is that of the arguments: at::empty without the dispatcher (0.5 us less each)
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_generic(sizes, c10::cuda::CUDACachingAllocator::get(), c10::DispatchKeySet(c10::DispatchKey::CUDA), type, c10::nullopt);
}
// MXFP4(codes, scales, False), without the class's own constructor
PyObject* mx4_of(at::Tensor codes, at::Tensor scales) {
  PyTypeObject* type = reinterpret_cast<PyTypeObject*>(py_mxfp4);
  PyObject* r = type->tp_alloc(type, 3);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(codes)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(scales)));
  PyTuple_SET_ITEM(r, 2, Py_NewRef(Py_False));
  return r;
}
at::Tensor mx4_tiles(i64 rows, i64 k) { return fresh({up(rows, 128), up(k, 128), 32, 4, 4}, at::kByte); }

// x -> MXFP4
PyObject* mx4_quantize(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(1)
  FAST_BEGIN
  const at::Tensor* x = plain(a[0]);
  const int device = device_for(abi.mx4_quantize, {x});
  if (device < 0 || !mx4_rows(*x, true)) return none();
  const i64 m = x->size(0), k = x->size(1);
  at::Tensor c, s;
  int rc;
  {
    const Unlocked unlocked;
    c = fresh({m, k / 2}, at::kByte);
    s = mx4_tiles(m, k);
    rc = abi.mx4_quantize(c.data_ptr(), s.data_ptr(), x->data_ptr(), 1, m, k, x->stride(0), x->scalar_type() == at::kFloat ? 2 : half_code(*x),
                          stream(device));
  }
  return rc ? failed(rc) : mx4_of(std::move(c), std::move(s));
  FAST_END
}

// (MXFP4, dtype) -> values
PyObject* mx4_dequantize(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(2)
  FAST_BEGIN
  Mx4 q;
  if (!mx4(a[0], 2, q) || !THPDtype_Check(a[1])) return none();
  const int device = device_for(abi.mx4_dequantize, {q.codes, q.scales});
  const at::ScalarType type = reinterpret_cast<THPDtype*>(a[1])->scalar_type;
  if (device < 0 || (type != at::kHalf && type != at::kBFloat16)) return none();
  at::Tensor y;
  int rc;
  {
    const Unlocked unlocked;
    y = fresh({q.rows, q.k}, type);
    rc = abi.mx4_dequantize(y.data_ptr(), q.codes->data_ptr(), q.scales->data_ptr(), 1, q.rows, q.k, q.k / 2, half_code(y), stream(device));
  }
  return rc ? failed(rc) : THPVariable_Wrap(std::move(y));
  FAST_END
}

// (X, residual or None, weight, eps, out_residual or None) -> MXFP4
PyObject* mx4_norm(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(5)
  FAST_BEGIN
  const at::Tensor *x = plain(a[0]), *r = a[1] == Py_None ? nullptr : plain(a[1]), *w = plain(a[2]), *o = a[4] == Py_None ? r : plain(a[4]);
  const int device = a[1] == Py_None ? device_for(abi.mx4_norm, {x, w}) : device_for(abi.mx4_norm, {x, w, r, o});
  if (device < 0 || !PyFloat_CheckExact(a[3]) || (a[1] == Py_None && a[4] != Py_None)) return none();
  const i64 n = x->dim() > 1 ? x->size(-1) : 0;
  if (n == 0 || n % 32 != 0 || n > 16384 || x->numel() == 0 || half_code(*x) < 0 || w->dim() != 1 || w->size(0) != n) return none();
  for (const at::Tensor* t : {x, w, r, o}) {
    if (!t) continue;
    if (t->scalar_type() != x->scalar_type() || !t->is_contiguous() || (uintptr_t)t->data_ptr() % 16) return none();
    if (t != w && t->sizes() != x->sizes()) return none();
  }
  const i64 rows = x->numel() / n;
  at::Tensor c, s;
  int rc;
  {
    const Unlocked unlocked;
    c = fresh({rows, n / 2}, at::kByte);
    s = mx4_tiles(rows, n);
    rc = abi.mx4_norm(c.data_ptr(), s.data_ptr(), o ? o->data_ptr() : nullptr, x->data_ptr(), r ? r->data_ptr() : nullptr, w->data_ptr(), rows, n,
                      n, n, n, (float)PyFloat_AS_DOUBLE(a[3]), half_code(*x), stream(device));
  }
  return rc ? failed(rc) : mx4_of(std::move(c), std::move(s));
  FAST_END
}

// (x or MXFP4, MXFP4, bias or None, swiglu, out_dtype or None) -> y, with swiglu an MXFP4
PyObject* mx4_matmul(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(5)
  FAST_BEGIN
  Mx4 w, q;
  if (!mx4(a[1], 2, w)) return none();
  const bool biased = a[2] != Py_None;
  const at::Tensor *x = plain(a[0]), *bias = biased ? plain(a[2]) : w.codes;      // w.codes: none
  if (!x && !mx4(a[0], 2, q)) return none();
  if (!abi.mx4_quantize || !abi.mx4_scale_bytes || !abi.mx4_takes_16bit) return none();      // of a library that holds another file's functions alone
  const int device = device_for(abi.mx4_matmul, {x ? x : q.codes, x ? x : q.scales, w.codes, w.scales, bias});
  if (device < 0 || (a[4] != Py_None && !THPDtype_Check(a[4])) || !PyBool_Check(a[3])) return none();
  const bool gated = a[3] == Py_True;
  if (x && (!mx4_rows(*x, false) || x->size(1) != w.k)) return none();
  if (!x && q.k != w.k) return none();
  at::ScalarType type = x ? x->scalar_type() : biased ? bias->scalar_type() : at::kHalf;
  if (a[4] != Py_None) {
    const at::ScalarType wanted = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
    if (x && wanted != type) return none();
    type = wanted;
  }
  if (type != at::kHalf && type != at::kBFloat16) return none();
  if (biased && (bias->dim() != 1 || bias->size(0) != w.rows || !bias->is_contiguous() || bias->scalar_type() != type)) return none();
  if (gated && w.rows % 128 != 0) return none();
  const i64 t = x ? x->size(0) : q.rows, n = w.rows, k = w.k;
  const int code = type == at::kHalf ? 0 : 1;
  at::Tensor y, ys, held;
  int rc = 0;
  {
    const Unlocked unlocked;
    const void *xc, *xs;
    void* st = stream(device);
    i64 stride = k / 2;
    if (x && abi.mx4_takes_16bit(t, n, k)) {
      xc = x->data_ptr();
      xs = nullptr;
      stride = t > 1 ? x->stride(0) : k;
    } else if (x) {
      const i64 at = up(t * k / 2, 256) * 256;
      held = fresh({at + abi.mx4_scale_bytes(t, k)}, at::kByte);
      xc = held.data_ptr();
      xs = (const char*)xc + at;
      rc = abi.mx4_quantize((void*)xc, (void*)xs, x->data_ptr(), 1, t, k, x->stride(0), code, st);
    } else {
      xc = q.codes->data_ptr();
      xs = q.scales->data_ptr();
    }
    if (!rc && !w.ready) rc = abi.weights_written(st);
    y = fresh({t, gated ? n / 4 : n}, gated ? at::kByte : type);
    if (gated) ys = mx4_tiles(t, n / 2);
    if (!rc)
      rc = abi.mx4_matmul(y.data_ptr(), gated ? ys.data_ptr() : nullptr, xc, xs, w.codes->data_ptr(), w.scales->data_ptr(),
                          biased ? bias->data_ptr() : nullptr, t, n, k, stride, k / 2, gated ? n / 4 : n, gated ? 1 : 0, 1, code, st);
  }
  if (rc) return failed(rc);
  return gated ? mx4_of(std::move(y), std::move(ys)) : THPVariable_Wrap(std::move(y));
  FAST_END
}

// (hidden_states, w1, w2, topk_weights, topk_ids) -> out
PyObject* mx4_moe(PyObject*, PyObject* const* a, Py_ssize_t count) {
  ARGS(5)
  FAST_BEGIN
  Mx4 w1, w2;
  if (!mx4(a[1], 3, w1) || !mx4(a[2], 3, w2)) return none();
  const at::Tensor *x = plain(a[0]), *weights = plain(a[3]), *ids = plain(a[4]);
  if (!abi.mx4_scatter || !abi.mx4_combine || !abi.mx4_tile_rows || !abi.mx4_max_tiles || !abi.mx4_scale_bytes) return none();
  const int device = device_for(abi.mx4_grouped, {x, weights, ids, w1.codes, w1.scales, w2.codes, w2.scales});
  if (device < 0 || !mx4_rows(*x, false) || x->size(1) != w1.k) return none();
  const i64 tokens = x->size(0), hidden = w1.k, inner = w2.k, experts = w1.lead;
  if (w2.lead != experts || w2.rows != hidden || w1.rows != 2 * inner || inner % 64 != 0 || experts > 4096) return none();
  if (ids->dim() != 2 || ids->size(0) != tokens || ids->size(1) < 1 || ids->size(1) > 65536 || weights->sizes() != ids->sizes() ||
      !ids->is_contiguous() || !weights->is_contiguous())
    return none();
  const int width = ids->scalar_type() == at::kInt ? 4 : ids->scalar_type() == at::kLong ? 8 : 0;
  const bool wide = weights->scalar_type() == at::kFloat;
  if (!width || (!wide && weights->scalar_type() != x->scalar_type())) return none();
  const int top_k = (int)ids->size(1), code = half_code(*x), e = (int)experts;
  const i64 slots = tokens * top_k;
  const int tile = (int)abi.mx4_tile_rows(slots, e, w1.rows);
  const i64 tiles = abi.mx4_max_tiles(slots, tile, e), rows = tiles * tile;
  // one buffer for what lives within the call
  i64 size = 0;
  auto part = [&](i64 n) { const i64 at = size; size += up(n, 256) * 256; return at; };
  const i64 place = part(4 * slots), table = part(4 + 8 * tiles), xc = part(rows * (hidden / 2)), xs = part(abi.mx4_scale_bytes(std::max<i64>(128, tile) * tiles, hidden)),
            ac = part(rows * (inner / 2)), as = part(abi.mx4_scale_bytes(std::max<i64>(128, tile) * tiles, inner)), y = part((tile == 64 ? 4 : 2) * rows * hidden), low = tile == 64 ? 0 : part(2 * rows * hidden);
  at::Tensor out, held;
  int rc = 0;
  {
    const Unlocked unlocked;
    held = fresh({size}, at::kByte);
    out = fresh({tokens, hidden}, x->scalar_type());
    char* p = (char*)held.data_ptr();
    void* st = stream(device);
    rc = abi.mx4_scatter(p + place, p + table, p + xc, p + xs, x->data_ptr(), ids->data_ptr(), width, tokens, top_k, tile, e, hidden, x->stride(0), code, st);
    if (!rc)
      rc = abi.mx4_grouped(p + ac, p + as, p + xc, p + xs, w1.codes->data_ptr(), w1.scales->data_ptr(), p + table, tiles, tile, e, w1.rows, hidden, 1,
                           st);
    if (!rc)
      rc = abi.mx4_grouped(p + y, tile == 64 ? nullptr : p + low, p + ac, p + as, w2.codes->data_ptr(), w2.scales->data_ptr(), p + table, tiles, tile, e, hidden, inner, 0,
                           st);
    if (!rc) rc = abi.mx4_combine(out.data_ptr(), p + y, tile == 64 ? nullptr : p + low, p + place, weights->data_ptr(), wide ? 1 : 0, tokens, top_k, hidden, code, st);
  }
  return rc ? failed(rc) : THPVariable_Wrap(std::move(out));
  FAST_END
}

// (addresses of the C functions in the order of `abi`, zeroed_workspace, counters, MXFP4)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t count) {
  constexpr Py_ssize_t n = sizeof(abi) / sizeof(void*);
  if (count != n + 3 || !PyType_Check(a[n + 2]) || !PyType_IsSubtype((PyTypeObject*)a[n + 2], &PyTuple_Type)) { PyErr_SetString(PyExc_TypeError, "wrong number of arguments"); return nullptr; }
  for (Py_ssize_t i = 0; i < n; ++i) {
    void* p = PyLong_AsVoidPtr(a[i]);      // 0: not in this library
    if (!p && PyErr_Occurred()) return nullptr;
    reinterpret_cast<void**>(&abi)[i] = p;
  }
  py_zeroed = Py_NewRef(a[n]);
  py_counters = Py_NewRef(a[n + 1]);
  py_mxfp4 = Py_NewRef(a[n + 2]);
  Py_RETURN_NONE;
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(init), FAST(w8a16), FAST(w4a16_packed), FAST(linear), FAST(w8a8), FAST(quantize), FAST(norm),
                         FAST(norm_quant), FAST(swiglu), FAST(kv4_rope_write), FAST(kv4_read), FAST(kv4_decode), FAST(kv4_prompt),
                         FAST(slot_maps), FAST(mx4_quantize), FAST(mx4_dequantize), FAST(mx4_norm), FAST(mx4_matmul), FAST(mx4_moe),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__fast() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", BUILT_FOR) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
