// The per-step calls of the Python face in native code: argument checks, output tensors from
// torch's caching allocator, the current stream, the library call.  A lookup of a few hundred keys
// takes less time on the GPU than the same steps took in Python and ctypes (11 us per call, of
// which the library's own part is 3).  Row movement stays in libugache_b200.so; its entry points
// arrive as addresses, so this module links against torch alone.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <optional>

#include "../../include/ugache_b200.h"

namespace {

struct Entry {
  decltype(&ugc_lookup_i64) lookup_i64;
  decltype(&ugc_lookup_u32) lookup_u32;
  decltype(&ugc_lookup_unique) lookup_unique;
  decltype(&ugc_lookup_pool) lookup_pool;
  decltype(&ugc_record) record;
  decltype(&ugc_route_plan_workspace) route_plan_workspace;
  decltype(&ugc_route_plan) route_plan;
  decltype(&ugc_route_dispatch) route_dispatch;
  decltype(&ugc_route_dispatch_grad) route_dispatch_grad;
  decltype(&ugc_route_combine) route_combine;
  decltype(&ugc_route_combine_grad) route_combine_grad;
  decltype(&ugc_adapter_workspace) adapter_workspace;
  decltype(&ugc_adapter_add) adapter_add;
};
Entry g_ugc = {};
PyObject* g_check = nullptr;  // raises for a status other than UGC_OK

PyObject* raise_status(int status) {
  PyObject* r = PyObject_CallFunction(g_check, "i", status);
  if (r) {  // cannot be: a failing status raises
    Py_DECREF(r);
    PyErr_SetString(PyExc_RuntimeError, "ugache_b200: failed");
  }
  return nullptr;
}

// Key tensor of the call and its bytes per key; `on_gpu`: its device decides the stream or where the
// outputs go (else pinned host keys will do).  False with a Python error set.
bool key_tensor(PyObject* o, const at::Tensor** keys, int* key_bytes, bool reject_other, bool on_gpu) {
  if (!THPVariable_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "keys must be a torch tensor");
    return false;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  const at::ScalarType ty = t.scalar_type();
  if (reject_other && ty != at::kLong && ty != at::kInt && ty != at::kUInt32) {
    PyErr_SetString(PyExc_TypeError, "keys must be int64, int32 or uint32");
    return false;
  }
  if (on_gpu && !t.is_cuda()) {
    PyErr_SetString(PyExc_ValueError, "keys must be a CUDA tensor");
    return false;
  }
  *keys = &t;
  *key_bytes = ty == at::kLong ? 8 : 4;
  return true;
}

// The stream argument: an integer, or None for the device's current stream.
bool stream_arg(PyObject* o, at::DeviceIndex dev, void** stream) {
  if (o == Py_None) {
    *stream = c10::cuda::getCurrentCUDAStream(dev).stream();
    return true;
  }
  *stream = PyLong_AsVoidPtr(o);
  return !PyErr_Occurred();
}

bool tensor_or_none(PyObject* o, const char* what, const at::Tensor** t) {
  *t = nullptr;
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a torch tensor", what);
    return false;
  }
  *t = &THPVariable_Unpack(o);
  return true;
}

at::Tensor device_empty(at::IntArrayRef sizes, at::ScalarType ty, at::Device dev) {
  return at::Tensor(at::detail::empty_cuda(sizes, ty, dev, std::nullopt));
}

bool arg_count(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, n);
  return false;
}

// C++ exceptions become the Python ones torch raises for them (by its translation alone: the buffer for
// warnings that torch's own macros set up besides would be made on every call)
#define UGC_PY_TRY try {
#define UGC_PY_END                                                  \
  }                                                                 \
  catch (...) {                                                     \
    torch::translate_exception_to_python(std::current_exception()); \
    return nullptr;                                                 \
  }

// lookup(ctx, replica, row_bytes, keys, out | None, stream | None) -> out
PyObject* fast_lookup(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!arg_count(n_args, 6)) return nullptr;
  UGC_PY_TRY
  ugc_ctx* ctx = static_cast<ugc_ctx*>(PyLong_AsVoidPtr(a[0]));
  const int replica = (int)PyLong_AsLong(a[1]);
  const int64_t row_bytes = PyLong_AsLongLong(a[2]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *keys, *out;
  int kb;
  void* stream;
  if (!key_tensor(a[3], &keys, &kb, true, a[4] == Py_None || a[5] == Py_None) || !tensor_or_none(a[4], "out", &out) ||
      !stream_arg(a[5], keys->device().index(), &stream))
    return nullptr;
  const int64_t n = keys->numel();
  at::Tensor made;
  if (!out) {
    made = device_empty({n, row_bytes}, at::kByte, keys->device());
    out = &made;
  }
  const void* kp = keys->data_ptr();
  void* op = out->data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = kb == 8 ? g_ugc.lookup_i64(ctx, replica, static_cast<const int64_t*>(kp), (size_t)n, op, stream)
               : g_ugc.lookup_u32(ctx, replica, static_cast<const uint32_t*>(kp), (size_t)n, op, stream);
  Py_END_ALLOW_THREADS
  if (rc != UGC_OK) return raise_status(rc);
  if (!made.defined()) return Py_NewRef(a[4]);
  return THPVariable_Wrap(std::move(made));
  UGC_PY_END
}

// lookup_unique(ctx, replica, row_bytes, keys, stream | None) -> (rows, unique_keys, inverse, n_unique)
PyObject* fast_lookup_unique(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!arg_count(n_args, 5)) return nullptr;
  UGC_PY_TRY
  ugc_ctx* ctx = static_cast<ugc_ctx*>(PyLong_AsVoidPtr(a[0]));
  const int replica = (int)PyLong_AsLong(a[1]);
  const int64_t row_bytes = PyLong_AsLongLong(a[2]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor* keys;
  int kb;
  void* stream;
  if (!key_tensor(a[3], &keys, &kb, false, true) || !stream_arg(a[4], keys->device().index(), &stream)) return nullptr;
  const int64_t n = keys->numel();
  const at::Device dev = keys->device();
  at::Tensor rows = device_empty({n, row_bytes}, at::kByte, dev);
  at::Tensor uniq = device_empty({n}, keys->scalar_type(), dev);
  at::Tensor inverse = device_empty({n}, at::kInt, dev);
  at::Tensor n_unique = device_empty({1}, at::kInt, dev);  // the call writes it, whatever n
  void *rp = rows.data_ptr(), *up = uniq.data_ptr();
  int32_t* ip = inverse.data_ptr<int32_t>();
  uint32_t* np = reinterpret_cast<uint32_t*>(n_unique.data_ptr<int32_t>());
  const void* kp = keys->data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ugc.lookup_unique(ctx, replica, kp, kb, (size_t)n, rp, up, ip, np, stream);
  Py_END_ALLOW_THREADS
  if (rc != UGC_OK) return raise_status(rc);
  PyObject* t = PyTuple_New(4);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(rows)));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(uniq)));
  PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(std::move(inverse)));
  PyTuple_SET_ITEM(t, 3, THPVariable_Wrap(std::move(n_unique)));
  return t;
  UGC_PY_END
}

// lookup_pool(ctx, replica, keys, offsets | None, n_bags, bag_size, elem_type, mode, dim, out | None,
//             stream | None) -> out
PyObject* fast_lookup_pool(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!arg_count(n_args, 11)) return nullptr;
  UGC_PY_TRY
  ugc_ctx* ctx = static_cast<ugc_ctx*>(PyLong_AsVoidPtr(a[0]));
  const int replica = (int)PyLong_AsLong(a[1]);
  const int64_t n_bags = PyLong_AsLongLong(a[4]), bag_size = PyLong_AsLongLong(a[5]);
  const int elem = (int)PyLong_AsLong(a[6]), mode = (int)PyLong_AsLong(a[7]);
  const int64_t dim = PyLong_AsLongLong(a[8]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *keys, *offsets, *out;
  int kb;
  void* stream;
  if (!key_tensor(a[2], &keys, &kb, false, a[9] == Py_None || a[10] == Py_None) || !tensor_or_none(a[3], "offsets", &offsets) ||
      !tensor_or_none(a[9], "out", &out) || !stream_arg(a[10], keys->device().index(), &stream))
    return nullptr;
  at::Tensor made;
  if (!out) {
    made = device_empty({n_bags, dim}, at::kFloat, keys->device());
    out = &made;
  }
  const void* kp = keys->data_ptr();
  const int64_t* fp = offsets ? offsets->data_ptr<int64_t>() : nullptr;
  float* op = static_cast<float*>(out->data_ptr());
  const size_t n = (size_t)keys->numel();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ugc.lookup_pool(ctx, replica, kp, kb, n, fp, (size_t)n_bags, (size_t)bag_size, elem, mode, op, stream);
  Py_END_ALLOW_THREADS
  if (rc != UGC_OK) return raise_status(rc);
  if (!made.defined()) return Py_NewRef(a[9]);
  return THPVariable_Wrap(std::move(made));
  UGC_PY_END
}

// record(ctx, replica, keys, stream | None)
PyObject* fast_record(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!arg_count(n_args, 4)) return nullptr;
  UGC_PY_TRY
  ugc_ctx* ctx = static_cast<ugc_ctx*>(PyLong_AsVoidPtr(a[0]));
  const int replica = (int)PyLong_AsLong(a[1]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor* keys;
  int kb;
  void* stream;
  if (!key_tensor(a[2], &keys, &kb, false, a[3] == Py_None) || !stream_arg(a[3], keys->device().index(), &stream)) return nullptr;
  const void* kp = keys->data_ptr();
  const size_t n = (size_t)keys->numel();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ugc.record(ctx, replica, kp, kb, n, stream);
  Py_END_ALLOW_THREADS
  if (rc != UGC_OK) return raise_status(rc);
  Py_RETURN_NONE;
  UGC_PY_END
}

// ---- routing -------------------------------------------------------------------------------

// What the tensors of one call have in common, set by the first that is looked at.
struct Call {
  at::Device dev = at::Device(at::kCPU);
  at::ScalarType ty = at::kFloat;
  bool has_dev = false, has_ty = false;
};

bool bad(PyObject* type, const char* format, const char* name) {
  PyErr_Format(type, format, name);
  return false;
}

bool on_device(Call* c, const at::Tensor& t, const char* name) {
  if (!t.is_cuda()) return bad(PyExc_ValueError, "%s must be a CUDA tensor", name);
  if (t.layout() != at::kStrided) return bad(PyExc_ValueError, "%s must be a dense tensor", name);
  if (!c->has_dev) {
    c->dev = t.device();
    c->has_dev = true;
  } else if (t.device() != c->dev) {
    return bad(PyExc_ValueError, "%s is on another device than the rest of the call", name);
  }
  return true;
}

bool unpack(PyObject* o, const char* name, at::Tensor* t) {
  if (!THPVariable_Check(o)) return bad(PyExc_TypeError, "%s must be a torch tensor", name);
  *t = THPVariable_Unpack(o);
  return true;
}

// The calls record nothing for autograd: a gradient that somebody waits for would be missing without a word.
bool not_recorded(const at::Tensor& t, const char* name) {
  if (!t.requires_grad() || !at::GradMode::is_enabled()) return true;
  return bad(PyExc_ValueError, "%s requires a gradient, which this call does not record: use it inside a torch.autograd.Function or under torch.no_grad()", name);
}

// The caller's own tensor has been written: what autograd saved of it before is no longer there.
void written(PyObject* o) {
  if (o == Py_None) return;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The call's stream, from its stream argument and the device of its first tensor.  A stream that is named
// becomes the current one meanwhile: what the call allocates or copies belongs to it.
struct OnStream {
  void* stream = nullptr;
  std::optional<c10::cuda::CUDAStreamGuard> guard;
  bool enter(PyObject* tensor, const char* name, PyObject* stream_object, Call* c) {
    at::Tensor t;
    if (!unpack(tensor, name, &t) || !on_device(c, t, name) || !stream_arg(stream_object, c->dev.index(), &stream)) return false;
    if (stream_object != Py_None)
      guard.emplace(c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(stream), c->dev.index()));
    return true;
  }
};

// Rows of a matrix: n of them (at least n with `more`; any number for n < 0) of dim elements (any for
// dim < 0).  An input whose rows are not contiguous or overlap is copied, an output refused.
bool rows_arg(PyObject* o, const char* name, Call* c, int64_t n, bool more, int64_t dim, bool output, at::Tensor* t) {
  if (!unpack(o, name, t)) return false;
  if (t->dim() != 2) return bad(PyExc_ValueError, "%s must have two dimensions", name);
  if (!on_device(c, *t, name) || !not_recorded(*t, name)) return false;
  const at::ScalarType ty = t->scalar_type();
  if (ty != at::kFloat && ty != at::kHalf && ty != at::kBFloat16)
    return bad(PyExc_TypeError, "%s must be float32, float16 or bfloat16", name);
  if (!c->has_ty) {
    c->ty = ty;
    c->has_ty = true;
  } else if (ty != c->ty) {
    return bad(PyExc_TypeError, "%s has another type than the other rows", name);
  }
  if (n >= 0 && (more ? t->size(0) < n : t->size(0) != n)) {
    PyErr_Format(PyExc_ValueError, "%s has %lld rows, %s%lld expected", name, (long long)t->size(0), more ? "at least " : "", (long long)n);
    return false;
  }
  if (dim >= 0 && t->size(1) != dim) {
    PyErr_Format(PyExc_ValueError, "%s has rows of %lld elements, %lld expected", name, (long long)t->size(1), (long long)dim);
    return false;
  }
  if (t->size(1) == 0) return bad(PyExc_ValueError, "%s has rows of no elements", name);
  if ((t->size(1) > 1 && t->stride(1) != 1) || (t->size(0) > 1 && t->stride(0) < t->size(1))) {
    if (output) return bad(PyExc_ValueError, "%s must have contiguous rows that do not overlap", name);
    *t = t->contiguous();
  }
  return true;
}

int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

int elem_type(const Call& c) {
  return c.ty == at::kFloat ? UGC_ELEM_F32 : c.ty == at::kHalf ? UGC_ELEM_F16 : UGC_ELEM_BF16;
}

// A plan's array of int32, or fp32 values per choice; dense, so a copy is made of anything else.
bool words_arg(PyObject* o, const char* name, Call* c, at::ScalarType ty, int64_t numel, at::Tensor* t) {
  if (!unpack(o, name, t) || !on_device(c, *t, name) || !not_recorded(*t, name)) return false;
  if (t->scalar_type() != ty) return bad(PyExc_TypeError, ty == at::kInt ? "%s must be int32" : "%s must be float32", name);
  if (numel >= 0 && t->numel() != numel) {
    PyErr_Format(PyExc_ValueError, "%s has %lld elements, %lld expected", name, (long long)t->numel(), (long long)numel);
    return false;
  }
  *t = t->contiguous();
  return true;
}

// Tokens and choices of `position` ([T] or [T, k]); the plan's offsets.
struct PlanArgs {
  at::Tensor offsets, position;
  int64_t tokens = 0, k = 1, n = 0;
};
bool plan_args(PyObject* offsets, PyObject* position, Call* c, PlanArgs* p) {
  if (!words_arg(position, "position", c, at::kInt, -1, &p->position)) return false;
  if (p->position.dim() < 1 || p->position.dim() > 2) return bad(PyExc_ValueError, "%s must have one or two dimensions", "position");
  p->tokens = p->position.size(0);
  p->k = p->position.dim() == 2 ? p->position.size(1) : 1;
  p->n = p->tokens * p->k;
  if (!offsets) return true;
  if (!words_arg(offsets, "offsets", c, at::kInt, -1, &p->offsets)) return false;
  if (p->offsets.dim() != 1 || p->offsets.numel() < 2) return bad(PyExc_ValueError, "%s must have an entry for each group and one more", "offsets");
  return true;
}
const int32_t* routed(const PlanArgs& p) { return p.offsets.data_ptr<int32_t>() + p.offsets.numel() - 1; }

PyObject* pair(at::Tensor a, at::Tensor b) {
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(a)));
  PyTuple_SET_ITEM(t, 1, b.defined() ? THPVariable_Wrap(std::move(b)) : Py_NewRef(Py_None));
  return t;
}

// route_plan(ids, n_groups, stream | None) -> (offsets, order, position)
PyObject* fast_route_plan(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!arg_count(n_args, 3)) return nullptr;
  UGC_PY_TRY
  Call c;
  OnStream on;
  at::Tensor ids;
  if (!on.enter(a[0], "ids", a[2], &c) || !unpack(a[0], "ids", &ids)) return nullptr;
  if (ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt) {
    PyErr_SetString(PyExc_TypeError, "ids must be int64 or int32");
    return nullptr;
  }
  if (ids.dim() < 1 || ids.dim() > 2) {
    PyErr_SetString(PyExc_ValueError, "ids must have one or two dimensions");
    return nullptr;
  }
  const long n_groups = PyLong_AsLong(a[1]);
  if (PyErr_Occurred()) return nullptr;
  ids = ids.contiguous();
  const int64_t tokens = ids.size(0), k = ids.dim() == 2 ? ids.size(1) : 1;
  const int groups = n_groups < 0 ? -1 : (int)std::min(n_groups, 1l << 30);
  size_t bytes = 0;
  int rc = g_ugc.route_plan_workspace((size_t)tokens, (size_t)k, groups, &bytes);
  if (rc != UGC_OK) return raise_status(rc);
  at::Tensor offsets = device_empty({groups + 1}, at::kInt, c.dev);
  at::Tensor order = device_empty({tokens * k}, at::kInt, c.dev);
  at::Tensor position = device_empty(ids.sizes(), at::kInt, c.dev);
  at::Tensor space;
  if (bytes) space = device_empty({(int64_t)bytes}, at::kByte, c.dev);
  const void* ip = ids.data_ptr();
  int32_t *fp = offsets.data_ptr<int32_t>(), *op = order.data_ptr<int32_t>(), *pp = position.data_ptr<int32_t>();
  void* wp = bytes ? space.data_ptr() : nullptr;
  const int id_bytes = ids.scalar_type() == at::kLong ? 8 : 4, dev = c.dev.index();
  Py_BEGIN_ALLOW_THREADS
  rc = g_ugc.route_plan(dev, ip, id_bytes, (size_t)tokens, (size_t)k, groups, fp, op, pp, wp, bytes, on.stream);
  Py_END_ALLOW_THREADS
  if (rc != UGC_OK) return raise_status(rc);
  PyObject* t = PyTuple_New(3);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(offsets)));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(order)));
  PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(std::move(position)));
  return t;
  UGC_PY_END
}

// route_dispatch(x, offsets, position, weights | None, out | None, stream | None) -> out
PyObject* fast_route_dispatch(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!arg_count(n_args, 6)) return nullptr;
  UGC_PY_TRY
  Call c;
  OnStream on;
  PlanArgs p;
  at::Tensor x, w, out;
  if (!on.enter(a[0], "x", a[5], &c) || !plan_args(a[1], a[2], &c, &p) || !rows_arg(a[0], "x", &c, p.tokens, false, -1, false, &x) ||
      (a[3] != Py_None && !words_arg(a[3], "weights", &c, at::kFloat, p.n, &w)) ||
      (a[4] != Py_None && !rows_arg(a[4], "out", &c, p.n, true, x.size(1), true, &out)))
    return nullptr;
  if (!out.defined()) out = device_empty({p.n, x.size(1)}, c.ty, c.dev);
  const void* xp = x.data_ptr();
  const float* wp = w.defined() ? w.data_ptr<float>() : nullptr;
  const int32_t *pp = p.position.data_ptr<int32_t>(), *rp = routed(p);
  void* op = out.data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ugc.route_dispatch(c.dev.index(), elem_type(c), xp, row_stride(x), wp, pp, rp, (size_t)p.tokens, (size_t)p.k,
                            (size_t)x.size(1), op, row_stride(out), on.stream);
  Py_END_ALLOW_THREADS
  if (rc != UGC_OK) return raise_status(rc);
  written(a[4]);
  return THPVariable_Wrap(std::move(out));
  UGC_PY_END
}

// route_dispatch_grad(dout, offsets, position, weights | None, x | None, dx | None, stream | None) -> (dx, dweights | None)
PyObject* fast_route_dispatch_grad(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!arg_count(n_args, 7)) return nullptr;
  UGC_PY_TRY
  Call c;
  OnStream on;
  PlanArgs p;
  at::Tensor dout, w, x, dx, dw;
  if (!on.enter(a[0], "dout", a[6], &c) || !plan_args(a[1], a[2], &c, &p) || !rows_arg(a[0], "dout", &c, p.n, true, -1, false, &dout) ||
      (a[3] != Py_None && !words_arg(a[3], "weights", &c, at::kFloat, p.n, &w)) ||
      (a[4] != Py_None && !rows_arg(a[4], "x", &c, p.tokens, false, dout.size(1), false, &x)) ||
      (a[5] != Py_None && !rows_arg(a[5], "dx", &c, p.tokens, false, dout.size(1), true, &dx)))
    return nullptr;
  if (!dx.defined()) dx = device_empty({p.tokens, dout.size(1)}, c.ty, c.dev);
  if (x.defined()) dw = device_empty(p.position.sizes(), at::kFloat, c.dev);
  const void *gp = dout.data_ptr(), *xp = x.defined() ? x.data_ptr() : nullptr;
  const float* wp = w.defined() ? w.data_ptr<float>() : nullptr;
  const int32_t* pp = p.position.data_ptr<int32_t>();
  void* op = dx.data_ptr();
  float* dp = dw.defined() ? dw.data_ptr<float>() : nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ugc.route_dispatch_grad(c.dev.index(), elem_type(c), gp, row_stride(dout), xp, xp ? row_stride(x) : 0, wp, pp,
                                 (size_t)p.tokens, (size_t)p.k, (size_t)dout.size(1), op, row_stride(dx), dp, on.stream);
  Py_END_ALLOW_THREADS
  if (rc != UGC_OK) return raise_status(rc);
  written(a[5]);
  return pair(std::move(dx), std::move(dw));
  UGC_PY_END
}

// route_combine(rows, offsets, position, weights | None, out | None, stream | None) -> out
PyObject* fast_route_combine(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!arg_count(n_args, 6)) return nullptr;
  UGC_PY_TRY
  Call c;
  OnStream on;
  PlanArgs p;
  at::Tensor rows, w, out;
  if (!on.enter(a[0], "rows", a[5], &c) || !plan_args(a[1], a[2], &c, &p) || !rows_arg(a[0], "rows", &c, p.n, true, -1, false, &rows) ||
      (a[3] != Py_None && !words_arg(a[3], "weights", &c, at::kFloat, p.n, &w)) ||
      (a[4] != Py_None && !rows_arg(a[4], "out", &c, p.tokens, false, rows.size(1), true, &out)))
    return nullptr;
  if (!out.defined()) out = device_empty({p.tokens, rows.size(1)}, c.ty, c.dev);
  const void* ip = rows.data_ptr();
  const float* wp = w.defined() ? w.data_ptr<float>() : nullptr;
  const int32_t* pp = p.position.data_ptr<int32_t>();
  void* op = out.data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ugc.route_combine(c.dev.index(), elem_type(c), ip, row_stride(rows), wp, pp, (size_t)p.tokens, (size_t)p.k,
                           (size_t)rows.size(1), op, row_stride(out), on.stream);
  Py_END_ALLOW_THREADS
  if (rc != UGC_OK) return raise_status(rc);
  written(a[4]);
  return THPVariable_Wrap(std::move(out));
  UGC_PY_END
}

// route_combine_grad(dy, offsets, position, weights | None, rows | None, drows | None, stream | None) -> (drows, dweights | None)
PyObject* fast_route_combine_grad(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!arg_count(n_args, 7)) return nullptr;
  UGC_PY_TRY
  Call c;
  OnStream on;
  PlanArgs p;
  at::Tensor dy, w, rows, drows, dw;
  if (!on.enter(a[0], "dy", a[6], &c) || !plan_args(a[1], a[2], &c, &p) || !rows_arg(a[0], "dy", &c, p.tokens, false, -1, false, &dy) ||
      (a[3] != Py_None && !words_arg(a[3], "weights", &c, at::kFloat, p.n, &w)) ||
      (a[4] != Py_None && !rows_arg(a[4], "rows", &c, p.n, true, dy.size(1), false, &rows)) ||
      (a[5] != Py_None && !rows_arg(a[5], "drows", &c, p.n, true, dy.size(1), true, &drows)))
    return nullptr;
  if (!drows.defined()) drows = device_empty({p.n, dy.size(1)}, c.ty, c.dev);
  if (rows.defined()) dw = device_empty(p.position.sizes(), at::kFloat, c.dev);
  const void *gp = dy.data_ptr(), *ip = rows.defined() ? rows.data_ptr() : nullptr;
  const float* wp = w.defined() ? w.data_ptr<float>() : nullptr;
  const int32_t *pp = p.position.data_ptr<int32_t>(), *rp = routed(p);
  void* op = drows.data_ptr();
  float* dp = dw.defined() ? dw.data_ptr<float>() : nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ugc.route_combine_grad(c.dev.index(), elem_type(c), gp, row_stride(dy), ip, ip ? row_stride(rows) : 0, wp, pp, rp,
                                (size_t)p.tokens, (size_t)p.k, (size_t)dy.size(1), op, row_stride(drows), dp, on.stream);
  Py_END_ALLOW_THREADS
  if (rc != UGC_OK) return raise_status(rc);
  written(a[5]);
  return pair(std::move(drows), std::move(dw));
  UGC_PY_END
}

// Adapter matrices [G, r, d]: the inner two dimensions dense, adapters any distance apart.
bool adapters_arg(PyObject* o, const char* name, Call* c, at::Tensor* t) {
  if (!unpack(o, name, t)) return false;
  if (t->dim() != 3) return bad(PyExc_ValueError, "%s must have three dimensions", name);
  if (!on_device(c, *t, name) || !not_recorded(*t, name)) return false;
  if (t->scalar_type() != c->ty) return bad(PyExc_TypeError, "%s has another type than base", name);
  const int64_t d = t->size(2);
  if ((d > 1 && t->stride(2) != 1) || (t->size(1) > 1 && t->stride(1) != d) ||
      (t->size(0) > 1 && t->stride(0) < t->size(1) * d))
    *t = t->contiguous();
  return true;
}

// adapter_add(base, x, down, up, offsets, order, scale | None, out | None, stream | None) -> out
PyObject* fast_adapter_add(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!arg_count(n_args, 9)) return nullptr;
  UGC_PY_TRY
  Call c;
  OnStream on;
  at::Tensor base, x, down, up, offsets, order, scale, out;
  if (!on.enter(a[0], "base", a[8], &c) || !rows_arg(a[0], "base", &c, -1, false, -1, false, &base) || !rows_arg(a[1], "x", &c, base.size(0), false, -1, false, &x) ||
      !adapters_arg(a[2], "down", &c, &down) || !adapters_arg(a[3], "up", &c, &up))
    return nullptr;
  const int64_t tokens = base.size(0), groups = down.size(0), rank = down.size(1), dim = x.size(1), out_dim = base.size(1);
  if (down.size(2) != dim || up.size(0) != groups || up.size(1) != out_dim || up.size(2) != rank) {
    PyErr_SetString(PyExc_ValueError, "down must be [adapters, rank, x's row], up [adapters, base's row, rank]");
    return nullptr;
  }
  if (!words_arg(a[4], "offsets", &c, at::kInt, groups + 1, &offsets) || !words_arg(a[5], "order", &c, at::kInt, tokens, &order) ||
      (a[6] != Py_None && !words_arg(a[6], "scale", &c, at::kFloat, groups, &scale)) ||
      (a[7] != Py_None && !rows_arg(a[7], "out", &c, tokens, false, out_dim, true, &out)))
    return nullptr;
  const int n_groups = (int)std::min(groups, (int64_t)1 << 30);
  size_t bytes = 0;
  int rc = g_ugc.adapter_workspace((size_t)tokens, n_groups, (size_t)rank, (size_t)dim, (size_t)out_dim, &bytes);
  if (rc != UGC_OK) return raise_status(rc);
  at::Tensor space;
  if (bytes) space = device_empty({(int64_t)bytes}, at::kByte, c.dev);
  void* wp = bytes ? space.data_ptr() : nullptr;
  if (!out.defined()) out = device_empty({tokens, out_dim}, c.ty, c.dev);
  const void *bp = base.data_ptr(), *xp = x.data_ptr(), *dp = down.data_ptr(), *upp = up.data_ptr();
  const float* sp = scale.defined() ? scale.data_ptr<float>() : nullptr;
  const int32_t *fp = offsets.data_ptr<int32_t>(), *rp = order.data_ptr<int32_t>();
  void* op = out.data_ptr();
  const int64_t ds = groups > 1 ? down.stride(0) : rank * dim, us = groups > 1 ? up.stride(0) : rank * out_dim;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ugc.adapter_add(c.dev.index(), elem_type(c), bp, row_stride(base), xp, row_stride(x), dp, ds, upp, us, sp, fp, rp,
                         (size_t)tokens, n_groups, (size_t)rank, (size_t)dim, (size_t)out_dim,
                         op, row_stride(out), wp, bytes, on.stream);
  Py_END_ALLOW_THREADS
  if (rc != UGC_OK) return raise_status(rc);
  written(a[7]);
  return THPVariable_Wrap(std::move(out));
  UGC_PY_END
}

// bind(check, {entry point name: address})
PyObject* fast_bind(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!arg_count(n_args, 2)) return nullptr;
  auto address = [&](const char* name, auto* slot) {
    PyObject* v = PyDict_GetItemString(a[1], name);
    void* p = v ? PyLong_AsVoidPtr(v) : nullptr;
    if (!p && !PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "%s", name);
    *slot = reinterpret_cast<std::remove_pointer_t<decltype(slot)>>(p);
    return p != nullptr;
  };
  if (!address("ugc_lookup_i64", &g_ugc.lookup_i64) || !address("ugc_lookup_u32", &g_ugc.lookup_u32) ||
      !address("ugc_lookup_unique", &g_ugc.lookup_unique) || !address("ugc_lookup_pool", &g_ugc.lookup_pool) ||
      !address("ugc_record", &g_ugc.record) || !address("ugc_route_plan_workspace", &g_ugc.route_plan_workspace) ||
      !address("ugc_route_plan", &g_ugc.route_plan) || !address("ugc_route_dispatch", &g_ugc.route_dispatch) ||
      !address("ugc_route_dispatch_grad", &g_ugc.route_dispatch_grad) ||
      !address("ugc_route_combine", &g_ugc.route_combine) ||
      !address("ugc_route_combine_grad", &g_ugc.route_combine_grad) ||
      !address("ugc_adapter_workspace", &g_ugc.adapter_workspace) || !address("ugc_adapter_add", &g_ugc.adapter_add))
    return nullptr;
  Py_XDECREF(g_check);
  g_check = Py_NewRef(a[0]);
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fast_bind)), METH_FASTCALL, nullptr},
    {"lookup", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fast_lookup)), METH_FASTCALL, nullptr},
    {"lookup_unique", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fast_lookup_unique)), METH_FASTCALL, nullptr},
    {"lookup_pool", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fast_lookup_pool)), METH_FASTCALL, nullptr},
    {"record", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fast_record)), METH_FASTCALL, nullptr},
    {"route_plan", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fast_route_plan)), METH_FASTCALL, nullptr},
    {"route_dispatch", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fast_route_dispatch)), METH_FASTCALL, nullptr},
    {"route_dispatch_grad", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fast_route_dispatch_grad)), METH_FASTCALL, nullptr},
    {"route_combine", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fast_route_combine)), METH_FASTCALL, nullptr},
    {"route_combine_grad", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fast_route_combine_grad)), METH_FASTCALL, nullptr},
    {"adapter_add", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fast_adapter_add)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast() {
  PyObject* m = PyModule_Create(&kModule);
  if (m && PyModule_AddStringConstant(m, "built_for", UGC_BUILT_FOR) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
