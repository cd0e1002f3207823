// The builtins called with torch tensors, in native code: what DeviceBuiltins and DeviceExecutor do per
// call - check the tensors, find their pointers and torch's current stream, call the C ABI - without
// the interpreter.  Through ctypes a call spent 3 to 5 us on that beside 2 us for the launch itself; here it
// is about 0.3 us, 0.1 of it for the interpreter's lock.
//
// Every function returns True when it has launched.  Anything out of the ordinary - an argument that is no
// contiguous float32 CUDA tensor, sizes that do not agree, a status other than 0 - makes it return
// False without an exception, and the caller takes its checked Python path, which raises, or launches what it can read and
// write within its tensors.  That goes for what torch throws as well (a tensor without storage, as tracing makes them, has
// no data pointer): a C++ exception must not reach the interpreter, where it would end the process.
//
// The C ABI is called without the interpreter's lock, as through ctypes: a launch waits when the GPU's queue is full,
// which may take until another thread has launched what the kernels at its head wait for.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <polar_b200.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <vector>

namespace {

// The tensors of one call: contiguous float32 on one CUDA device.
class Call {
public:
  Call(PyObject* const* args, Py_ssize_t given, Py_ssize_t expected) : args_(args), ok_(given == expected) {}
  const at::Tensor* tensor(int i) {
    if (!ok_) return nullptr;
    if (!THPVariable_Check(args_[i])) {
      ok_ = false;
      return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(args_[i]);
    if (!t.defined() || !t.is_cuda() || t.scalar_type() != at::kFloat || !t.is_contiguous() ||
        (device_ >= 0 && t.get_device() != device_)) {
      ok_ = false;
      return nullptr;
    }
    device_ = t.get_device();
    return &t;
  }
  // None: no tensor, which is no reason to decline.
  const at::Tensor* tensor_or_none(int i) { return ok_ && args_[i] == Py_None ? nullptr : tensor(i); }
  // A matrix whose rows may lie further apart than they are long.
  const at::Tensor* matrix(int i, uint64_t* pitch) {
    const at::Tensor* t = any(args_[i]);
    if (!t) return nullptr;
    ok_ = t->scalar_type() == at::kFloat && t->dim() == 2 && (t->size(1) <= 1 || t->stride(1) == 1) &&
          (t->size(0) <= 1 || t->stride(0) >= t->size(1));
    if (!ok_) return nullptr;
    *pitch = (uint64_t)(t->size(0) <= 1 ? t->size(1) : t->stride(0));
    return t;
  }
  // Ids: whole numbers in fp32, 32 or 64 bits.
  const at::Tensor* ids(int i, int* type) {
    const at::Tensor* t = ok_ && args_[i] == Py_None ? nullptr : any(args_[i]);
    if (!t) return nullptr;
    const auto s = t->scalar_type();
    ok_ = t->is_contiguous() && (s == at::kFloat || s == at::kInt || s == at::kLong);
    *type = s == at::kFloat ? POLAR_B200_IDS_F32 : s == at::kInt ? POLAR_B200_IDS_I32 : POLAR_B200_IDS_I64;
    return ok_ ? t : nullptr;
  }
  // An element of a list: contiguous, of `size` bytes each.
  const at::Tensor* element(PyObject* o, size_t size) {
    const at::Tensor* t = any(o);
    if (!t) return nullptr;
    ok_ = t->is_contiguous() && (size == 4 ? t->scalar_type() == at::kFloat
                                           : t->scalar_type() == at::kFloat8_e4m3fn || t->scalar_type() == at::kByte);
    return ok_ ? t : nullptr;
  }
  float scalar(int i) {
    if (!ok_) return 0.f;
    const double v = PyFloat_AsDouble(args_[i]);
    if (v == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      ok_ = false;
    }
    return (float)v;
  }
  uint64_t whole(int i) {
    if (!ok_) return 0;
    const long long v = PyLong_AsLongLong(args_[i]);
    if (v < 0) {                                           // negative, or not a whole number
      PyErr_Clear();
      ok_ = false;
      return 0;
    }
    return (uint64_t)v;
  }
  void require(bool condition) { ok_ = ok_ && condition; }
  bool ok() const { return ok_; }
  void* stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device_).stream(); }

private:
  // A tensor on the call's device.
  const at::Tensor* any(PyObject* o) {
    if (!ok_) return nullptr;
    ok_ = THPVariable_Check(o);
    if (!ok_) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    ok_ = t.defined() && t.is_cuda() && (device_ < 0 || t.get_device() == device_);
    if (!ok_) return nullptr;
    device_ = t.get_device();
    return &t;
  }
  PyObject* const* args_;
  bool ok_;
  int device_ = -1;
};

// Runs f without the interpreter's lock.  What f needs of Python objects is looked up before.
template <class F>
auto unlocked(F f) {
  PyThreadState* state = PyEval_SaveThread();
  auto r = f();
  PyEval_RestoreThread(state);
  return r;
}

float* data(const at::Tensor* t) { return static_cast<float*>(t->data_ptr()); }
uint64_t numel(const at::Tensor* t) { return (uint64_t)t->numel(); }
float* data_or_null(const at::Tensor* t) { return t ? data(t) : nullptr; }
bool has(const at::Tensor* t, uint64_t n) { return !t || numel(t) == n; }
PyObject* answer(bool launched) { return PyBool_FromLong(launched); }
template <class F, class... A>
PyObject* launched(F f, A... args) {
  return answer(unlocked([&] { return f(args...); }) == 0);
}

using Function = PyObject* (*)(PyObject*, PyObject* const*, Py_ssize_t);
template <Function F>
PyObject* declining(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(self, args, n);
  } catch (const std::exception&) {
    return answer(false);
  }
}
template <Function F>
PyObject* raising(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(self, args, n);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

#define BUILTIN(name) PyObject* name(PyObject*, PyObject* const* args, Py_ssize_t n)

BUILTIN(ffill) {
  Call c(args, n, 2);
  const float v = c.scalar(0);
  const at::Tensor* out = c.tensor(1);
  return c.ok() ? launched(polar_b200_ffill, v, data(out), numel(out), c.stream()) : answer(false);
}
BUILTIN(fadd) {
  Call c(args, n, 5);
  const at::Tensor* a = c.tensor(0);
  const float sa = c.scalar(1);
  const at::Tensor* b = c.tensor(2);
  const float sb = c.scalar(3);
  const at::Tensor* out = c.tensor(4);
  if (c.ok()) c.require(numel(a) == numel(out) && numel(b) == numel(out));
  return c.ok() ? launched(polar_b200_fadd, data(a), sa, data(b), sb, data(out), numel(out), c.stream()) : answer(false);
}
template <int (*F)(const float*, float*, uint64_t, void*)>
BUILTIN(unary) {
  Call c(args, n, 2);
  const at::Tensor *a = c.tensor(0), *out = c.tensor(1);
  if (c.ok()) c.require(numel(a) == numel(out));
  return c.ok() ? launched(F, data(a), data(out), numel(out), c.stream()) : answer(false);
}
template <int (*F)(const float*, const float*, float*, uint64_t, void*)>
BUILTIN(binary) {
  Call c(args, n, 3);
  const at::Tensor *a = c.tensor(0), *b = c.tensor(1), *out = c.tensor(2);
  if (c.ok()) c.require(numel(a) == numel(out) && numel(b) == numel(out));
  return c.ok() ? launched(F, data(a), data(b), data(out), numel(out), c.stream()) : answer(false);
}
BUILTIN(fmulconcat) {
  Call c(args, n, 3);
  const at::Tensor *g = c.tensor(0), *l = c.tensor(1), *out = c.tensor(2);
  if (c.ok()) c.require(numel(g) >= 1 && numel(l) == numel(out));
  return c.ok() ? launched(polar_b200_fmulconcat, data(g), data(l), data(out), numel(out), c.stream()) : answer(false);
}
BUILTIN(fsoftmax) {
  Call c(args, n, 2);
  const at::Tensor *a = c.tensor(0), *out = c.tensor(1);
  if (c.ok()) c.require(numel(a) == numel(out));
  return c.ok() ? launched(polar_b200_fsoftmax, data(a), data(out), numel(out), nullptr, 0, c.stream()) : answer(false);
}
BUILTIN(fpool) {
  Call c(args, n, 6);
  const at::Tensor* a = c.tensor(0);
  const uint64_t wh = c.whole(1), ww = c.whole(2), sh = c.whole(3), sw = c.whole(4);
  const at::Tensor* out = c.tensor(5);
  if (c.ok()) c.require(a->dim() == 2);
  if (!c.ok()) return answer(false);
  const uint64_t h = (uint64_t)a->size(0), w = (uint64_t)a->size(1);
  if (wh && ww && sh && sw && wh <= h && ww <= w && numel(out) < ((h - wh) / sh + 1) * ((w - ww) / sw + 1)) return answer(false);
  return launched(polar_b200_fpool, data(a), h, w, wh, ww, sh, sw, data(out), c.stream());
}
BUILTIN(fconv2d) {
  Call c(args, n, 3);
  const at::Tensor *a = c.tensor(0), *k = c.tensor(1), *out = c.tensor(2);
  if (c.ok()) c.require(a->dim() == 2 && k->dim() == 2);
  if (!c.ok()) return answer(false);
  const int64_t oh = a->size(0) - k->size(0) + 1, ow = a->size(1) - k->size(1) + 1;
  if (oh > 0 && ow > 0 && out->numel() < oh * ow) return answer(false);
  return launched(polar_b200_fconv2d, data(a), (uint64_t)a->size(0), (uint64_t)a->size(1), data(k), (uint64_t)k->size(0),
                  (uint64_t)k->size(1), data(out), c.stream());
}
BUILTIN(ftranspose) {
  Call c(args, n, 2);
  const at::Tensor *a = c.tensor(0), *out = c.tensor(1);
  if (c.ok()) c.require(a->dim() == 2 && numel(a) <= numel(out));
  if (!c.ok()) return answer(false);
  return launched(polar_b200_ftranspose, data(a), (uint64_t)a->size(0), (uint64_t)a->size(1), data(out), c.stream());
}
BUILTIN(fmatmul) {
  Call c(args, n, 5);
  const uint64_t tl = c.whole(0), tr = c.whole(1);
  const at::Tensor *l = c.tensor(2), *r = c.tensor(3), *out = c.tensor(4);
  if (c.ok()) c.require(tl <= 1 && tr <= 1 && l->dim() == 2 && r->dim() == 2 && out->dim() == 2);
  if (!c.ok()) return answer(false);
  const int64_t m = l->size(tl ? 1 : 0), k = l->size(tl ? 0 : 1), cols = r->size(tr ? 0 : 1);
  if (r->size(tr ? 1 : 0) != k || out->size(0) != m || out->size(1) != cols) return answer(false);
  return launched(polar_b200_fmatmul, (int)tl, (int)tr, (uint64_t)m, (uint64_t)cols, (uint64_t)k, data(l), data(r), data(out),
                  nullptr, 0, c.stream());
}

// flayernorm(x, gamma or None, beta or None, eps, out, mean or None, rstd or None)
BUILTIN(flayernorm) {
  Call c(args, n, 7);
  const at::Tensor *x = c.tensor(0), *gamma = c.tensor_or_none(1), *beta = c.tensor_or_none(2);
  const float eps = c.scalar(3);
  const at::Tensor *out = c.tensor(4), *mean = c.tensor_or_none(5), *rstd = c.tensor_or_none(6);
  if (c.ok()) c.require(x->dim() >= 1 && x->size(-1) > 0);
  if (!c.ok()) return answer(false);
  const uint64_t cols = (uint64_t)x->size(-1), rows = numel(x) / cols;
  if (numel(out) != numel(x) || !has(gamma, cols) || !has(beta, cols) || !has(mean, rows) || !has(rstd, rows)) return answer(false);
  return launched(polar_b200_flayernorm, data(x), data_or_null(gamma), data_or_null(beta), eps, rows, cols, data(out), data_or_null(mean),
                  data_or_null(rstd), c.stream());
}
// flayernorm_grad(gradient, x, gamma or None, mean, rstd, dx, dgamma or None, dbeta or None)
BUILTIN(flayernorm_grad) {
  Call c(args, n, 8);
  const at::Tensor *g = c.tensor(0), *x = c.tensor(1), *gamma = c.tensor_or_none(2), *mean = c.tensor(3), *rstd = c.tensor(4);
  const at::Tensor *dx = c.tensor(5), *dgamma = c.tensor_or_none(6), *dbeta = c.tensor_or_none(7);
  if (c.ok()) c.require(x->dim() >= 1 && x->size(-1) > 0);
  if (!c.ok()) return answer(false);
  const uint64_t cols = (uint64_t)x->size(-1), rows = numel(x) / cols;
  if (numel(g) != numel(x) || numel(dx) != numel(x) || !has(gamma, cols) || !has(mean, rows) || !has(rstd, rows) || !has(dgamma, cols) ||
      !has(dbeta, cols))
    return answer(false);
  return launched(polar_b200_flayernorm_grad, data(g), data(x), data_or_null(gamma), data(mean), data(rstd), rows, cols, data(dx),
                  data_or_null(dgamma), data_or_null(dbeta), nullptr, 0, c.stream());
}
// flogprob(logits, ids or None, logprob or None, entropy or None, logsumexp or None, top_ids or None, top_logprob or None)
BUILTIN(flogprob) {
  Call c(args, n, 7);
  uint64_t pitch = 0;
  int type = POLAR_B200_IDS_I64, top_type = -1;
  const at::Tensor *x = c.matrix(0, &pitch), *ids = c.ids(1, &type), *lp = c.tensor_or_none(2), *entropy = c.tensor_or_none(3),
                   *lse = c.tensor_or_none(4), *top_ids = c.ids(5, &top_type), *top_lp = c.tensor_or_none(6);
  if (!c.ok()) return answer(false);
  const uint64_t rows = (uint64_t)x->size(0), classes = (uint64_t)x->size(1);
  if (!has(ids, rows) || !has(lp, rows) || !has(entropy, rows) || !has(lse, rows) || (lp && !ids) || (top_ids && ids && top_type != type))
    return answer(false);
  if (top_ids && !ids) type = top_type;
  for (const at::Tensor* t : {top_ids, top_lp})
    if (t && (t->dim() != 2 || (uint64_t)t->size(0) != rows)) return answer(false);
  if (top_ids && top_lp && top_ids->size(1) != top_lp->size(1)) return answer(false);
  const uint64_t top = top_ids ? (uint64_t)top_ids->size(1) : top_lp ? (uint64_t)top_lp->size(1) : 0;
  return launched(polar_b200_flogprob, data(x), rows, classes, pitch, ids ? ids->data_ptr() : nullptr, type, data_or_null(lp),
                  data_or_null(entropy), data_or_null(lse), top, top_ids ? top_ids->data_ptr() : nullptr, data_or_null(top_lp), c.stream());
}
// flogprob_grad(logits, ids, logsumexp, entropy or None, g_logprob, g_entropy or None, dlogits)
BUILTIN(flogprob_grad) {
  Call c(args, n, 7);
  uint64_t pitch = 0, dpitch = 0;
  int type = POLAR_B200_IDS_I64;
  const at::Tensor *x = c.matrix(0, &pitch), *ids = c.ids(1, &type), *lse = c.tensor(2), *entropy = c.tensor_or_none(3), *g = c.tensor(4),
                   *ge = c.tensor_or_none(5), *dx = c.matrix(6, &dpitch);
  if (!c.ok() || !ids) return answer(false);
  const uint64_t rows = (uint64_t)x->size(0), classes = (uint64_t)x->size(1);
  if ((uint64_t)dx->size(0) != rows || (uint64_t)dx->size(1) != classes || !has(ids, rows) || !has(lse, rows) || !has(entropy, rows) ||
      !has(g, rows) || !has(ge, rows))
    return answer(false);
  return launched(polar_b200_flogprob_grad, data(x), rows, classes, pitch, ids->data_ptr(), type, data(lse), data_or_null(entropy), data(g),
                  data_or_null(ge), data(dx), dpitch, c.stream());
}

// A list or tuple, as long as it lives here.
struct Sequence {
  explicit Sequence(PyObject* o) : list(o == Py_None ? nullptr : PySequence_Fast(o, "")) {
    if (!list) PyErr_Clear();
  }
  ~Sequence() { Py_XDECREF(list); }
  Py_ssize_t size() const { return list ? PySequence_Fast_GET_SIZE(list) : -1; }
  PyObject* operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(list, i); }
  PyObject* list;
};
// fadamw(weights, gradients, first, second, first_scales or None, second_scales or None, step, lr, beta1, beta2, eps,
// weight decays, schedule or None): lists of tensors, and one decay for each
BUILTIN(fadamw) {
  Call c(args, n, 13);
  if (!c.ok()) return answer(false);
  const Sequence w(args[0]), g(args[1]), m(args[2]), v(args[3]), ms(args[4]), vs(args[5]), decays(args[11]);
  const Py_ssize_t count = w.size();
  const bool eight = ms.list != nullptr;
  if (count < 0 || g.size() != count || m.size() != count || v.size() != count || decays.size() != count || (vs.list != nullptr) != eight ||
      (eight && (ms.size() != count || vs.size() != count)))
    return answer(false);
  polar_b200_adamw_options o;
  o.step = c.whole(6);
  o.lr = c.scalar(7), o.beta1 = c.scalar(8), o.beta2 = c.scalar(9), o.eps = c.scalar(10);
  std::vector<polar_b200_adamw_tensor> tensors((size_t)count);
  for (Py_ssize_t i = 0; i < count && c.ok(); ++i) {
    polar_b200_adamw_tensor& t = tensors[(size_t)i];
    const at::Tensor *wt = c.element(w[i], 4), *gt = c.element(g[i], 4), *mt = c.element(m[i], eight ? 1 : 4), *vt = c.element(v[i], eight ? 1 : 4);
    const at::Tensor *mst = eight ? c.element(ms[i], 4) : nullptr, *vst = eight ? c.element(vs[i], 4) : nullptr;
    if (!c.ok()) break;
    t.count = numel(wt);
    const uint64_t blocks = (t.count + 127) / 128;
    c.require(numel(gt) == t.count && numel(mt) == t.count && numel(vt) == t.count && has(mst, blocks) && has(vst, blocks));
    t.weights = data(wt), t.gradient = data(gt), t.first = mt->data_ptr(), t.second = vt->data_ptr();
    t.first_scales = data_or_null(mst), t.second_scales = data_or_null(vst);
    const double decay = PyFloat_AsDouble(decays[i]);
    if (decay == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      c.require(false);
    }
    t.weight_decay = (float)decay;
  }
  const at::Tensor* schedule = c.tensor_or_none(12);
  if (c.ok()) c.require(has(schedule, 2));
  if (!c.ok()) return answer(false);
  o.schedule = data_or_null(schedule);
  if (count == 0) return answer(true);
  return launched(polar_b200_fadamw, tensors.data(), (uint64_t)count, &o, c.stream());
}

// A number for every element of a list, or a list of them.
struct Numbers {
  explicit Numbers(PyObject* o) : list(PyFloat_Check(o) || PyLong_Check(o) ? Py_None : o), one(list.list || o == Py_None ? 0.0 : PyFloat_AsDouble(o)) {
    if (PyErr_Occurred()) PyErr_Clear(), bad = true;
  }
  bool fits(Py_ssize_t count) const { return !bad && (!list.list || list.size() == count); }
  bool at(Py_ssize_t i, float* v) const {
    const double d = list.list ? PyFloat_AsDouble(list[i]) : one;
    if (d == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
    *v = (float)d;
    return true;
  }
  Sequence list;
  double one;
  bool bad = false;
};
// fmuon(weights, gradients, momenta, lr, momentum, nesterov, steps, weight decay or decays, scale or scales or None, a, b, c, schedule or None): lists of
// tensors; no scale: the root of rows / cols where that is above 1.  Its workspace comes from torch's allocator, which keeps it: it is too large for the library's own pool to.
BUILTIN(fmuon) {
  Call c(args, n, 13);
  if (!c.ok()) return answer(false);
  const Sequence w(args[0]), g(args[1]), m(args[2]);
  const Numbers decays(args[7]), scales(args[8]);
  const bool by_shape = args[8] == Py_None;
  const Py_ssize_t count = w.size();
  if (count < 0 || g.size() != count || m.size() != count || args[7] == Py_None || !decays.fits(count) || !scales.fits(count)) return answer(false);
  polar_b200_muon_options o;
  o.lr = c.scalar(3), o.momentum = c.scalar(4), o.nesterov = c.whole(5) != 0;
  const uint64_t steps = c.whole(6);
  o.steps = (uint32_t)std::min<uint64_t>(steps, 1000);
  o.a = c.scalar(9), o.b = c.scalar(10), o.c = c.scalar(11);
  std::vector<polar_b200_muon_tensor> tensors((size_t)count);
  const at::Tensor* some = nullptr;
  for (Py_ssize_t i = 0; i < count && c.ok(); ++i) {
    polar_b200_muon_tensor& t = tensors[(size_t)i];
    const at::Tensor *wt = c.element(w[i], 4), *gt = c.element(g[i], 4), *mt = c.element(m[i], 4);
    if (!c.ok()) break;
    c.require(wt->dim() >= 2);
    for (const at::Tensor* x : {gt, mt})                   // matrices of the same shape, however many dimensions count them
      c.require(c.ok() && x->dim() >= 2 && x->size(-1) == wt->size(-1) && x->size(-2) == wt->size(-2) && numel(x) == numel(wt));
    if (!c.ok()) break;
    t.weights = data(wt), t.gradient = data(gt), t.momentum = data(mt);
    t.rows = (uint64_t)wt->size(-2), t.cols = (uint64_t)wt->size(-1);
    t.matrices = t.rows && t.cols ? numel(wt) / (t.rows * t.cols) : 0;
    c.require(decays.at(i, &t.weight_decay) && scales.at(i, &t.scale));
    if (by_shape) t.scale = (float)std::sqrt(std::max(1.0, (double)t.rows / (double)std::max<uint64_t>(t.cols, 1)));
    some = wt;
  }
  const at::Tensor* schedule = c.tensor_or_none(12);
  if (c.ok()) c.require(has(schedule, 2));
  if (!c.ok()) return answer(false);
  o.schedule = data_or_null(schedule);
  if (count == 0) return answer(true);
  const uint64_t need = polar_b200_fmuon_workspace_bytes(tensors.data(), (uint64_t)count);
  at::Tensor workspace;
  if (need) workspace = at::empty({(int64_t)need}, at::TensorOptions().dtype(at::kByte).device(some->device()));
  return launched(polar_b200_fmuon, tensors.data(), (uint64_t)count, &o, need ? workspace.data_ptr() : nullptr, need, c.stream());
}
// The ids and offsets of packed sequences, of one type.
bool packed(Call& c, int i, int* type, const at::Tensor** ids, const at::Tensor** offsets) {
  int other = -1;
  *ids = c.ids(i, type), *offsets = c.ids(i + 1, &other);
  return c.ok() && *ids && *offsets && other == *type && numel(*offsets) >= 1;
}
// fpolicy_loss(logprob, old_logprob, reference or None, entropy or None, advantage, ids, offsets, advantage_per_token, clip_low, clip_high,
// kl_weight, entropy_weight, count, by_sequence, loss, g_logprob or None, g_entropy or None)
BUILTIN(fpolicy_loss) {
  Call c(args, n, 17);
  int type = POLAR_B200_IDS_I64;
  const at::Tensor *lp = c.tensor(0), *old = c.tensor(1), *ref = c.tensor_or_none(2), *entropy = c.tensor_or_none(3), *advantage = c.tensor(4);
  const at::Tensor *ids, *offsets;
  if (!packed(c, 5, &type, &ids, &offsets)) return answer(false);
  polar_b200_policy_options o;
  const bool per_token = c.whole(7) != 0;
  o.clip_low = c.scalar(8), o.clip_high = c.scalar(9), o.kl_weight = c.scalar(10), o.entropy_weight = c.scalar(11), o.count = c.scalar(12);
  o.by_sequence = c.whole(13) != 0;
  const at::Tensor *loss = c.tensor(14), *g = c.tensor_or_none(15), *ge = c.tensor_or_none(16);
  if (!c.ok()) return answer(false);
  const uint64_t tokens = numel(ids), sequences = numel(offsets) - 1;
  for (const at::Tensor* t : {lp, old, ref, entropy, g, ge})
    if (!has(t, tokens)) return answer(false);
  if (numel(advantage) != (per_token ? tokens : sequences) || numel(loss) != 5 || (ge && !entropy)) return answer(false);
  const polar_b200_policy_batch b = {data(lp), data(old), data_or_null(ref), data_or_null(entropy), data(advantage), ids->data_ptr(),
                                     offsets->data_ptr(), type, per_token, tokens, sequences};
  return launched(polar_b200_fpolicy_loss, &b, &o, data(loss), data_or_null(g), data_or_null(ge), nullptr, 0, c.stream());
}
// fpreference_loss(logprob, reference or None, ids, offsets, beta, smoothing, margin, count, average, loss, rewards or None, g_logprob or None)
BUILTIN(fpreference_loss) {
  Call c(args, n, 12);
  int type = POLAR_B200_IDS_I64;
  const at::Tensor *lp = c.tensor(0), *ref = c.tensor_or_none(1), *ids, *offsets;
  if (!packed(c, 2, &type, &ids, &offsets)) return answer(false);
  polar_b200_preference_options o;
  o.beta = c.scalar(4), o.smoothing = c.scalar(5), o.margin = c.scalar(6), o.count = c.scalar(7), o.average = c.whole(8) != 0;
  const at::Tensor *loss = c.tensor(9), *rewards = c.tensor_or_none(10), *g = c.tensor_or_none(11);
  if (!c.ok()) return answer(false);
  const uint64_t tokens = numel(ids), sequences = numel(offsets) - 1;
  if (sequences % 2 || !has(lp, tokens) || !has(ref, tokens) || !has(g, tokens) || !has(rewards, sequences) || numel(loss) != 3) return answer(false);
  return launched(polar_b200_fpreference_loss, data(lp), data_or_null(ref), ids->data_ptr(), offsets->data_ptr(), type, tokens, sequences / 2, &o,
                  data(loss), data_or_null(rewards), data_or_null(g), nullptr, 0, c.stream());
}

// A program's operations as Python has them: a list of (native name, address of the argument structs, their count).
bool operations(PyObject* list, std::vector<polar_b200_op>* ops) {
  if (!PyList_Check(list)) {
    PyErr_SetString(PyExc_TypeError, "expected a list of (name, address, count)");
    return false;
  }
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
    const char* name;
    unsigned long long address, count;
    if (!PyArg_ParseTuple(PyList_GET_ITEM(list, i), "yKK", &name, &address, &count)) return false;
    ops->push_back({name, reinterpret_cast<const polar_b200_arg*>(address), count});
  }
  return true;
}
// workspace_bytes(operations): what the most demanding one asks for; fmuon builtins in a row, which share their launches, ask together, but for
// no more than 3 GiB, beyond which they are done in groups.
BUILTIN(workspace_bytes) {
  std::vector<polar_b200_op> ops;
  if (n != 1 || !operations(args[0], &ops)) return nullptr;
  uint64_t need = 0, row = 0;
  for (const polar_b200_op& o : ops) {
    const uint64_t one = polar_b200_launch_workspace_bytes(o.name, o.args, o.argc);
    row = std::strcmp(o.name, "fmuon") ? 0 : std::min<uint64_t>(row + one, 3ull << 30);
    need = std::max<uint64_t>({need, one, row});
  }
  return PyLong_FromUnsignedLongLong(need);
}
// create_program(operations, workspace address, its bytes): (status, handle).
BUILTIN(create_program) {
  std::vector<polar_b200_op> ops;
  if (n != 3 || !operations(args[0], &ops)) return nullptr;
  void* workspace = PyLong_AsVoidPtr(args[1]);
  const uint64_t bytes = PyLong_AsUnsignedLongLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  void* program = nullptr;
  const int status = polar_b200_program_create(ops.data(), ops.size(), workspace, bytes, &program);
  return Py_BuildValue("iK", status, (unsigned long long)(uintptr_t)program);
}
// run_program(handle, device index): one pass of a polar_b200_program on the device's current stream; the status.
BUILTIN(run_program) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "run_program(handle, device)");
    return nullptr;
  }
  void* handle = PyLong_AsVoidPtr(args[0]);
  const long device = PyLong_AsLong(args[1]);
  if (PyErr_Occurred()) return nullptr;
  void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  return PyLong_FromLong(unlocked([&] { return polar_b200_program_run(handle, stream); }));
}

#define ENTRY(name, ...) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(__VA_ARGS__)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    ENTRY("ffill", declining<ffill>),
    ENTRY("fcopy", declining<unary<polar_b200_fcopy>>),
    ENTRY("fadd", declining<fadd>),
    ENTRY("fmul", declining<binary<polar_b200_fmul>>),
    ENTRY("fdivide", declining<binary<polar_b200_fdivide>>),
    ENTRY("fsigmoid", declining<unary<polar_b200_fsigmoid>>),
    ENTRY("fsigmoid_unclamped", declining<unary<polar_b200_fsigmoid_unclamped>>),
    ENTRY("flogloss", declining<binary<polar_b200_flogloss>>),
    ENTRY("fmulconcat", declining<fmulconcat>),
    ENTRY("frelu", declining<unary<polar_b200_frelu>>),
    ENTRY("fsoftmax", declining<fsoftmax>),
    ENTRY("fpool", declining<fpool>),
    ENTRY("fconv2d", declining<fconv2d>),
    ENTRY("ftranspose", declining<ftranspose>),
    ENTRY("fmatmul", declining<fmatmul>),
    ENTRY("flayernorm", declining<flayernorm>),
    ENTRY("flayernorm_grad", declining<flayernorm_grad>),
    ENTRY("flogprob", declining<flogprob>),
    ENTRY("flogprob_grad", declining<flogprob_grad>),
    ENTRY("fadamw", declining<fadamw>),
    ENTRY("fmuon", declining<fmuon>),
    ENTRY("fpolicy_loss", declining<fpolicy_loss>),
    ENTRY("fpreference_loss", declining<fpreference_loss>),
    ENTRY("workspace_bytes", raising<workspace_bytes>),
    ENTRY("create_program", raising<create_program>),
    ENTRY("run_program", raising<run_program>),
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "polar_b200_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_polar_b200_torch(void) { return PyModule_Create(&module); }
