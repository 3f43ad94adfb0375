// The short calls' way from Python without its cost: a call whose tensors the kernel takes
// as they are (types, shapes, strides, alignment, one device, the current one) is checked,
// allocated and launched here, in 4 to 10 us (by the call and the box) where the Python wrapper
// and ctypes take 9 to 18.  Anything else returns None: the wrapper's own checks then say what is wrong, or copy.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/hip/HIPFunctions.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <exception>
#include <tuple>

#include "../../include/gdn_mi355x.h"

namespace {

using at::IntArrayRef;
using at::ScalarType;
using at::Tensor;

constexpr ScalarType kBf16 = ScalarType::BFloat16, kF32 = ScalarType::Float, kFp8 = ScalarType::Float8_e4m3fn;
constexpr int64_t kNodes = 64, kGroup = 128;

PyObject* check_status = nullptr;  // raises for a status that is not 0

bool aligned(const Tensor& t, int64_t bytes = 16) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0; }

// A call's tensors: all on one device, as the kernels take them.
struct Taken {
  bool ok = true;
  int dev = -1;

  void need(bool condition) { ok = ok && condition; }

  // dim < 0: any
  const Tensor& tensor(const Tensor& t, ScalarType type, int64_t dim) {
    static const Tensor none;
    if (!ok || !t.is_cuda() || t.scalar_type() != type || t.layout() != at::kStrided || (dim >= 0 && t.dim() != dim)) {
      ok = false;
      return none;
    }
    const int d = t.get_device();
    need(dev < 0 || dev == d);
    dev = d;
    return ok ? t : none;
  }
  const Tensor& tensor(PyObject* o, ScalarType type, int64_t dim) {
    static const Tensor none;
    if (ok && THPVariable_CheckExact(o)) return tensor(THPVariable_Unpack(o), type, dim);
    ok = false;
    return none;
  }
  // [B, T, C] or [B, T, H, D] rows that the kernels read in 16-byte pieces (o: a tensor, or Python's)
  template <class O>
  const Tensor& rows(const O& o, IntArrayRef shape) {
    const Tensor& t = tensor(o, kBf16, static_cast<int64_t>(shape.size()));
    if (!ok) return t;
    const IntArrayRef st = t.strides();
    const bool heads = shape.size() == 4;
    const int64_t width = heads ? shape[2] * shape[3] : shape[2];
    need(t.sizes() == shape && st.back() == 1 && (!heads || st[2] == shape[3] || shape[2] == 1) && width <= st[1] &&
         st[1] < (1 << 24) && st[0] % 8 == 0 && st[1] % 8 == 0 && aligned(t));
    return t;
  }
  template <class O>
  const Tensor& dense(const O& o, ScalarType type, IntArrayRef shape, int64_t align) {
    const Tensor& t = tensor(o, type, static_cast<int64_t>(shape.size()));
    if (ok) need(t.sizes() == shape && t.is_contiguous() && aligned(t, align));
    return t;
  }
  const Tensor& ids(PyObject* o, int64_t B) { return dense(o, ScalarType::Long, {B}, 8); }
  // parents of T nodes and their stride per sequence
  const Tensor& parents(PyObject* o, int64_t B, int64_t T, int64_t& stride) {
    const Tensor& t = tensor(o, ScalarType::Int, -1);
    if (!ok) return t;
    stride = t.dim() == 2 ? T : 0;
    need(T >= 1 && T <= kNodes && t.is_contiguous() &&
         (t.dim() == 2 ? t.size(0) == B && t.size(1) == T : t.dim() == 1 && t.size(0) == T));
    return t;
  }
  const Tensor& state_pool(PyObject* o, int64_t Hv, int64_t D) {
    const Tensor& t = tensor(o, kF32, 4);
    if (ok)
      need(t.size(1) == Hv && t.size(2) == D && t.size(3) == D && t.stride(1) == D * D && t.stride(2) == D &&
           t.stride(3) == 1);
    return t;
  }
  const Tensor& conv_pool(PyObject* o, int64_t C) {
    const Tensor& t = tensor(o, kBf16, 3);
    if (ok) need(t.size(1) == C && t.size(2) == 3 && t.stride(2) == 1);
    return t;
  }
  // a tuple of n, or NULL for None
  PyObject* pending(PyObject* o, Py_ssize_t n) {
    if (o == Py_None) return nullptr;
    need(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == n);
    return ok ? o : nullptr;
  }
  bool here() {
    need(dev >= 0);
    if (ok) need(c10::hip::current_device() == dev);
    return ok;
  }
  void* stream() const { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev).stream(); }
};

template <class T>
T* ptr(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
uint16_t* bf(const Tensor& t) { return static_cast<uint16_t*>(t.data_ptr()); }

// NULL with Python's exception set, for a status that is not 0
bool failed(const char* name, int status) {
  if (status == GDN_OK) return false;
  PyObject* r = PyObject_CallFunction(check_status, "si", name, status);
  if (r) {
    Py_DECREF(r);
    PyErr_Format(PyExc_RuntimeError, "%s: status %d", name, status);
  }
  return true;
}

// What a call of one function gives: its C++ exceptions become what torch makes of them in Python
// (no memory: torch.OutOfMemoryError).
template <class F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F&& f) {
  if (n != want) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    return f();
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

PyObject* none() { Py_RETURN_NONE; }

// x, conv_pool, ids, weight, parents, pending: the conv's arguments.
struct Conv {
  Taken t;
  int64_t B = 0, T = 0, C = 0, p_b = 0, lp_b = 0, last_T = 0;
  const Tensor *x = nullptr, *pool = nullptr, *ids = nullptr, *w = nullptr, *par = nullptr;
  const Tensor *lx = nullptr, *lpar = nullptr, *acc = nullptr;

  bool take(PyObject* const* a) {
    x = &t.tensor(a[0], kBf16, 3);
    if (!t.ok) return false;
    B = x->size(0), T = x->size(1), C = x->size(2);
    t.rows(a[0], {B, T, C});
    pool = &t.conv_pool(a[1], C);
    ids = &t.ids(a[2], B);
    w = &t.tensor(a[3], kBf16, -1);
    par = &t.parents(a[4], B, T, p_b);
    if (!t.ok || w->numel() != 4 * C || w->dim() == 0 || w->size(-1) != 4 || !w->is_contiguous() || !aligned(*w) || C % 8)
      return false;
    if (PyObject* p = t.pending(a[5], 3)) {
      lx = &t.tensor(PyTuple_GET_ITEM(p, 0), kBf16, 3);
      if (!t.ok) return false;
      last_T = lx->size(1);
      t.rows(PyTuple_GET_ITEM(p, 0), {B, last_T, C});
      lpar = &t.parents(PyTuple_GET_ITEM(p, 1), B, last_T, lp_b);
      acc = &t.ids(PyTuple_GET_ITEM(p, 2), B);
    }
    return t.ok;
  }
  int call(const Tensor& y, void* stream) const {
    return gdn_conv_tree(
        bf(*x), x->stride(0), x->stride(1), bf(*pool), pool->stride(0), pool->stride(1), pool->size(0),
        ptr<int64_t>(*ids), bf(*w), ptr<int32_t>(*par), p_b, lx ? bf(*lx) : nullptr, lx ? lx->stride(0) : 0,
        lx ? lx->stride(1) : 0, lpar ? ptr<int32_t>(*lpar) : nullptr, lp_b, acc ? ptr<int64_t>(*acc) : nullptr,
        static_cast<int>(last_T), bf(y), static_cast<int>(B), static_cast<int>(T), static_cast<int>(C), stream);
  }
};

// (x, conv_pool, ids, weight, parents, pending) -> y
PyObject* conv_tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> PyObject* {
    Conv c;
    if (!c.take(a) || !c.t.here()) return none();
    Tensor y = at::empty({c.B, c.T, c.C}, c.x->options());
    return failed("gdn_conv_tree", c.call(y, c.t.stream())) ? nullptr : THPVariable_Wrap(std::move(y));
  });
}

// What the two forms of the rule share: q, k, v, the pool, ids, parents and the pending step.
struct Rule {
  Taken t;
  int64_t B = 0, T = 0, Hk = 0, Hv = 0, D = 0, p_b = 0, lp_b = 0, last_T = 0;
  const Tensor *q = nullptr, *k = nullptr, *v = nullptr, *pool = nullptr, *ids = nullptr, *par = nullptr;
  const Tensor *lk = nullptr, *lg = nullptr, *lu = nullptr, *lpar = nullptr, *acc = nullptr;

  template <class O>
  bool take(const O& oq, const O& ok_, const O& ov, PyObject* opool, PyObject* oids, PyObject* opar, PyObject* opending) {
    k = &t.tensor(ok_, kBf16, 4);
    v = &t.tensor(ov, kBf16, 4);
    if (!t.ok) return false;
    B = k->size(0), T = k->size(1), Hk = k->size(2), D = k->size(3), Hv = v->size(2);
    if (Hk == 0 || Hv % Hk) return false;
    q = &t.rows(oq, {B, T, Hk, D});
    t.rows(ok_, {B, T, Hk, D});
    t.rows(ov, {B, T, Hv, D});
    pool = &t.state_pool(opool, Hv, D);
    ids = &t.ids(oids, B);
    par = &t.parents(opar, B, T, p_b);
    if (PyObject* p = t.pending(opending, 5)) {
      lk = &t.tensor(PyTuple_GET_ITEM(p, 0), kBf16, 4);
      if (!t.ok) return false;
      last_T = lk->size(1);
      t.rows(PyTuple_GET_ITEM(p, 0), {B, last_T, Hk, D});
      lg = &t.dense(PyTuple_GET_ITEM(p, 1), kF32, {B, last_T, Hv}, 16);
      lu = &t.dense(PyTuple_GET_ITEM(p, 2), kF32, {B, last_T, Hv, D}, 16);
      lpar = &t.parents(PyTuple_GET_ITEM(p, 3), B, last_T, lp_b);
      acc = &t.ids(PyTuple_GET_ITEM(p, 4), B);
    }
    return t.ok;
  }
  template <class Entry, class... Gates, class... Out>
  int call(Entry entry, const std::tuple<Gates...>& gates, const std::tuple<Out...>& out, void* stream) const {
    return std::apply(entry, std::tuple_cat(
        std::make_tuple(bf(*q), q->stride(0), q->stride(1), bf(*k), k->stride(0), k->stride(1), bf(*v), v->stride(0),
                        v->stride(1)),
        gates,
        std::make_tuple(ptr<float>(*pool), pool->stride(0), pool->size(0), ptr<int64_t>(*ids), ptr<int32_t>(*par), p_b,
                        lk ? bf(*lk) : nullptr, lk ? lk->stride(0) : int64_t{0}, lk ? lk->stride(1) : int64_t{0},
                        lg ? ptr<float>(*lg) : nullptr, lu ? ptr<float>(*lu) : nullptr,
                        lpar ? ptr<int32_t>(*lpar) : nullptr, lp_b, acc ? ptr<int64_t>(*acc) : nullptr,
                        static_cast<int>(last_T)),
        out,
        std::make_tuple(static_cast<int>(B), static_cast<int>(T), static_cast<int>(Hk), static_cast<int>(Hv),
                        static_cast<int>(D), static_cast<float>(std::pow(static_cast<double>(D), -0.5)), stream)));
  }
};

// The rule alone: its other arguments g, beta, s_pool, ids, parents, pending, and its outputs.
struct Plain {
  Rule r;
  const Tensor *g = nullptr, *beta = nullptr;
  Tensor o, u;

  template <class O>
  bool take(const O& q, const O& k, const O& v, PyObject* const* a) {
    if (!r.take(q, k, v, a[2], a[3], a[4], a[5])) return false;
    g = &r.t.dense(a[0], kF32, {r.B, r.T, r.Hv}, 16);
    beta = &r.t.dense(a[1], kBf16, {r.B, r.T, r.Hv}, 2);
    return r.t.ok;
  }
  void allocate() {
    o = at::empty({r.B, r.T, r.Hv, r.D}, r.v->options());
    u = at::empty({r.B, r.T, r.Hv, r.D}, g->options());
  }
  int call(void* stream) const {
    return r.call(gdn_rule_tree, std::make_tuple(ptr<float>(*g), bf(*beta)), std::make_tuple(bf(o), ptr<float>(u)), stream);
  }
};

// (q, k, v, g, beta, s_pool, ids, parents, pending) -> (o, u)
PyObject* rule_tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    Plain p;
    if (!p.take(a[0], a[1], a[2], a + 3) || !p.r.t.here()) return none();
    p.allocate();
    if (failed("gdn_rule_tree", p.call(p.r.t.stream()))) return nullptr;
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(p.o)), THPVariable_Wrap(std::move(p.u)));
  });
}

// The rule with the layer's gates and norm: its other arguments b, a, a_log, dt_bias, z, norm_weight,
// s_pool, ids, parents, eps, pending, fp8, and its outputs.
struct Layer {
  Rule r;
  bool fp8 = false;
  float eps = 0.0f;
  ScalarType param = kBf16;
  const Tensor *b = nullptr, *ga = nullptr, *a_log = nullptr, *dt = nullptr, *z = nullptr, *w = nullptr;
  Tensor y, scale, u, g;

  template <class O>
  bool take(const O& q, const O& k, const O& v, PyObject* const* a) {
    if (!PyFloat_CheckExact(a[9]) || !PyBool_Check(a[11]) || !r.take(q, k, v, a[6], a[7], a[8], a[10])) return false;
    fp8 = a[11] == Py_True;
    eps = static_cast<float>(PyFloat_AS_DOUBLE(a[9]));
    b = &r.t.dense(a[0], kBf16, {r.B, r.T, r.Hv}, 2);
    ga = &r.t.dense(a[1], kBf16, {r.B, r.T, r.Hv}, 2);
    if (!r.t.ok || !THPVariable_CheckExact(a[2])) return false;
    param = THPVariable_Unpack(a[2]).scalar_type();
    a_log = &r.t.dense(a[2], param, {r.Hv}, 2);
    dt = &r.t.dense(a[3], param, {r.Hv}, 2);
    z = &r.t.rows(a[4], {r.B, r.T, r.Hv * r.D});
    w = &r.t.dense(a[5], kBf16, {r.D}, 16);
    return r.t.ok && (param == kBf16 || param == kF32) && (!fp8 || r.D == kGroup);
  }
  void allocate() {
    const auto f32 = r.pool->options();
    y = at::empty({r.B, r.T, r.Hv, r.D}, r.v->options().dtype(fp8 ? kFp8 : kBf16));
    if (fp8) scale = at::empty_strided({r.B * r.T, r.Hv}, {1, r.B * r.T}, f32);
    u = at::empty({r.B, r.T, r.Hv, r.D}, f32);
    g = at::empty({r.B, r.T, r.Hv}, f32);
  }
  int call(void* stream) const {
    return r.call(
        gdn_rule_tree_layer,
        std::make_tuple(bf(*b), bf(*ga), a_log->data_ptr(), dt->data_ptr(), param == kF32 ? 1 : 0),
        std::make_tuple(bf(*z), z->stride(0), z->stride(1), bf(*w), eps, fp8 ? nullptr : bf(y),
                        fp8 ? ptr<uint8_t>(y) : nullptr, fp8 ? ptr<float>(scale) : nullptr, ptr<float>(u),
                        ptr<float>(g)),
        stream);
  }
  PyObject* given_scale() { return fp8 ? THPVariable_Wrap(std::move(scale)) : none(); }
};

// (q, k, v, b, a, a_log, dt_bias, z, norm_weight, s_pool, ids, parents, eps, pending, fp8)
// -> (y, scale or None, u, g)
PyObject* rule_tree_layer(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 15, [&]() -> PyObject* {
    Layer l;
    if (!l.take(a[0], a[1], a[2], a + 3) || !l.r.t.here()) return none();
    l.allocate();
    if (failed("gdn_rule_tree_layer", l.call(l.r.t.stream()))) return nullptr;
    PyObject* scale = l.given_scale();
    return Py_BuildValue("(NNNN)", THPVariable_Wrap(std::move(l.y)), scale, THPVariable_Wrap(std::move(l.u)),
                         THPVariable_Wrap(std::move(l.g)));
  });
}

// The gated norm in e4m3 of [..., H, D] rows.
struct Norm {
  Taken t;
  int64_t H = 0, D = 0, tokens = 0;
  float eps = 0.0f;
  const Tensor *x = nullptr, *z = nullptr, *w = nullptr;
  Tensor y, scale;

  // z may have the rows' H D columns in one dimension
  bool take(const Tensor& rows, PyObject* oz, PyObject* ow, PyObject* oeps) {
    x = &t.tensor(rows, kBf16, -1);
    if (!t.ok || x->dim() < 2 || !x->is_contiguous() || !aligned(*x) || x->numel() == 0 || !PyFloat_CheckExact(oeps))
      return false;
    eps = static_cast<float>(PyFloat_AS_DOUBLE(oeps));
    H = x->size(-2), D = x->size(-1), tokens = x->numel() / (H * D);
    z = &t.tensor(oz, kBf16, -1);
    if (!t.ok || !z->is_contiguous() || !aligned(*z)) return false;
    at::DimVector flat(x->sizes().begin(), x->sizes().end() - 1);
    flat.back() = H * D;
    t.need(z->sizes() == x->sizes() || z->sizes() == IntArrayRef(flat));
    w = &t.dense(ow, kBf16, {D}, 16);
    return t.ok && H * D % kGroup == 0;
  }
  void allocate() {
    y = at::empty(x->sizes(), x->options().dtype(kFp8));
    scale = at::empty_strided({tokens, H * D / kGroup}, {1, tokens}, x->options().dtype(kF32));
  }
  int call(void* stream) const {
    return gdn_rmsnorm_gated_fp8(bf(*x), H * D, bf(*z), H * D, bf(*w), ptr<uint8_t>(y), ptr<float>(scale), 1, tokens,
                                 tokens, static_cast<int>(H), static_cast<int>(D), eps, stream);
  }
};

// The conv's output and its views q, k, v, for Hk key heads of D.
struct Parts {
  Tensor y, q, k, v;

  // false: no such heads
  bool allocate(const Conv& c, PyObject* heads, PyObject* dim) {
    if (!PyLong_CheckExact(heads) || !PyLong_CheckExact(dim)) return false;
    const int64_t Hk = PyLong_AsLongLong(heads), D = PyLong_AsLongLong(dim);
    if (Hk < 1 || D < 1 || Hk >= 1 << 20 || D >= 1 << 20 || c.C <= 2 * Hk * D || c.C % D) {
      PyErr_Clear();
      return false;
    }
    y = at::empty({c.B, c.T, c.C}, c.x->options());
    const int64_t Hv = c.C / D - 2 * Hk;
    q = y.as_strided({c.B, c.T, Hk, D}, {c.T * c.C, c.C, D, 1}, 0);
    k = y.as_strided({c.B, c.T, Hk, D}, {c.T * c.C, c.C, D, 1}, Hk * D);
    v = y.as_strided({c.B, c.T, Hv, D}, {c.T * c.C, c.C, D, 1}, 2 * Hk * D);
    return true;
  }
};

// Conv and rule of a verify step.  All of it is checked, and everything allocated, before the
// first launch: the conv moves its pool on where a step is pending.
// (conv_tree's six, Hk, D, rule_tree_layer's last twelve) -> (y, scale or None, k, u, g)
PyObject* verify_tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 20, [&]() -> PyObject* {
    Conv c;
    Parts p;
    Layer l;
    if (!c.take(a) || !p.allocate(c, a[6], a[7]) || !l.take(p.q, p.k, p.v, a + 8)) return none();
    if (c.pool->size(0) != l.r.pool->size(0) || !c.t.here() || !l.r.t.here()) return none();
    l.allocate();
    void* stream = c.t.stream();
    if (failed("gdn_rule_tree_layer", l.call(GDN_CHECK_ONLY)) || failed("gdn_conv_tree", c.call(p.y, stream)) ||
        failed("gdn_rule_tree_layer", l.call(stream)))
      return nullptr;
    PyObject* scale = l.given_scale();
    return Py_BuildValue("(NNNNN)", THPVariable_Wrap(std::move(l.y)), scale, THPVariable_Wrap(std::move(p.k)),
                         THPVariable_Wrap(std::move(l.u)), THPVariable_Wrap(std::move(l.g)));
  });
}

// The same with the rule alone and the norm in e4m3 behind it.
// (conv_tree's six, Hk, D, rule_tree's last six, z, norm_weight, eps) -> (y, scale, k, u)
PyObject* verify_tree_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 17, [&]() -> PyObject* {
    Conv c;
    Parts p;
    Plain r;
    Norm m;
    if (!c.take(a) || !p.allocate(c, a[6], a[7]) || !r.take(p.q, p.k, p.v, a + 8)) return none();
    r.allocate();
    if (c.pool->size(0) != r.r.pool->size(0) || !m.take(r.o, a[14], a[15], a[16]) || !c.t.here() || !r.r.t.here() ||
        !m.t.here())
      return none();
    m.allocate();
    void* stream = c.t.stream();
    if (failed("gdn_rule_tree", r.call(GDN_CHECK_ONLY)) || failed("gdn_rmsnorm_gated_fp8", m.call(GDN_CHECK_ONLY)) ||
        failed("gdn_conv_tree", c.call(p.y, stream)) || failed("gdn_rule_tree", r.call(stream)) ||
        failed("gdn_rmsnorm_gated_fp8", m.call(stream)))
      return nullptr;
    return Py_BuildValue("(NNNN)", THPVariable_Wrap(std::move(m.y)), THPVariable_Wrap(std::move(m.scale)),
                         THPVariable_Wrap(std::move(p.k)), THPVariable_Wrap(std::move(r.u)));
  });
}

// (s_pool, conv_pool, ids, parents, accepted, x, k, g, u) -> True
PyObject* commit_tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    Taken t;
    const Tensor& k = t.tensor(a[6], kBf16, 4);
    const Tensor& u = t.tensor(a[8], kF32, 4);
    const Tensor& x = t.tensor(a[5], kBf16, 3);
    if (!t.ok) return none();
    const int64_t B = k.size(0), T = k.size(1), Hk = k.size(2), D = k.size(3), Hv = u.size(2), C = x.size(2);
    if (Hk == 0 || Hv % Hk) return none();
    int64_t p_b = 0;
    t.rows(a[5], {B, T, C});
    t.rows(a[6], {B, T, Hk, D});
    const Tensor& g = t.dense(a[7], kF32, {B, T, Hv}, 16);
    t.dense(a[8], kF32, {B, T, Hv, D}, 16);
    const Tensor& pool = t.state_pool(a[0], Hv, D);
    const Tensor& cpool = t.conv_pool(a[1], C);
    const Tensor& ids = t.ids(a[2], B);
    const Tensor& par = t.parents(a[3], B, T, p_b);
    const Tensor& acc = t.ids(a[4], B);
    if (!t.ok || pool.size(0) != cpool.size(0) || !t.here()) return none();
    const int status = gdn_commit_tree(
        ptr<float>(pool), pool.stride(0), bf(cpool), cpool.stride(0), cpool.stride(1), pool.size(0), ptr<int64_t>(ids),
        ptr<int32_t>(par), p_b, ptr<int64_t>(acc), bf(x), x.stride(0), x.stride(1), bf(k), k.stride(0), k.stride(1),
        ptr<float>(g), ptr<float>(u), static_cast<int>(B), static_cast<int>(T), static_cast<int>(Hk),
        static_cast<int>(Hv), static_cast<int>(D), static_cast<int>(C), t.stream());
    if (failed("gdn_commit_tree", status)) return nullptr;
    Py_RETURN_TRUE;
  });
}

// (x, weight, weight_scale, x_scale or None) -> y
PyObject* linear_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    Taken t;
    const bool ready = a[3] != Py_None;
    const Tensor& w = t.tensor(a[1], kFp8, 2);
    const Tensor& x = t.tensor(a[0], ready ? kFp8 : kBf16, -1);
    const Tensor& ws = t.tensor(a[2], kF32, 2);
    if (!t.ok || x.dim() < 2) return none();
    const int64_t N = w.size(0), K = w.size(1), G = K / kGroup;
    if (K == 0 || K % kGroup || x.size(-1) != K || N == 0 || x.numel() == 0) return none();
    const int64_t M = x.numel() / K;
    t.need(w.stride(1) == 1 && w.stride(0) % 16 == 0 && w.stride(0) >= K && aligned(w) && x.is_contiguous() && aligned(x) &&
           ws.size(0) == (N + kGroup - 1) / kGroup && ws.size(1) == G && (G == 1 || ws.stride(1) == 1) &&
           (N <= kGroup || ws.stride(0) >= G) && M < (int64_t{1} << 31) && N < (int64_t{1} << 31));
    const Tensor* xs = nullptr;
    if (t.ok && ready) {
      xs = &t.tensor(a[3], kF32, 2);
      if (t.ok) t.need(xs->size(0) == M && xs->size(1) == G);
    }
    if (!t.here()) return none();
    const int m = static_cast<int>(M), nn = static_cast<int>(N), kk = static_cast<int>(K);
    int64_t bytes = ready ? 0 : gdn_gemm_fp8_workspace_size(m, nn, kk, 1);
    Tensor work;
    if (bytes > 0) work = at::empty({bytes}, x.options().dtype(ScalarType::Byte));
    at::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = N;
    Tensor y = at::empty(shape, x.options().dtype(kBf16));
    uint16_t* c = bf(y);
    const int status = gdn_gemm_fp8(
        x.data_ptr(), ready ? 0 : 1, K, xs ? ptr<float>(*xs) : nullptr, xs ? xs->stride(0) : 0, xs ? xs->stride(1) : 0,
        ptr<uint8_t>(w), w.stride(0), ptr<float>(ws), N > kGroup ? ws.stride(0) : G, nullptr, 0, 0, m, nn, kk, 1, &c, &N,
        &nn, bytes > 0 ? work.data_ptr() : nullptr, bytes, t.stream());
    return failed("gdn_gemm_fp8", status) ? nullptr : THPVariable_Wrap(std::move(y));
  });
}

// (hidden_states, gate, weight, eps) -> (y, scale)
PyObject* norm_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    Norm m;
    if (!THPVariable_CheckExact(a[0]) || !m.take(THPVariable_Unpack(a[0]), a[1], a[2], a[3]) ||
        m.z->dim() != m.x->dim() || !m.t.here())
      return none();
    m.allocate();
    if (failed("gdn_rmsnorm_gated_fp8", m.call(m.t.stream()))) return nullptr;
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(m.y)), THPVariable_Wrap(std::move(m.scale)));
  });
}

// (x, residual or None, weight, eps, post_weight or None, gate or None, gate_sigmoid, scale, offset, bf16, fp8)
// -> (y or None, y8 or None, scales or None, r)
PyObject* add_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    Taken t;
    const Tensor& x = t.tensor(a[0], kBf16, -1);
    if (!t.ok || x.dim() < 1 || !x.is_contiguous() || x.numel() == 0 || !PyFloat_CheckExact(a[3]) || !PyBool_Check(a[6]) ||
        !PyFloat_CheckExact(a[7]) || !PyFloat_CheckExact(a[8]) || !PyBool_Check(a[9]) || !PyBool_Check(a[10]) ||
        !THPVariable_CheckExact(a[2]))
      return none();
    const int64_t H = x.size(-1), M = x.numel() / H;
    const bool want = a[9] == Py_True, fp8 = a[10] == Py_True;
    const double scale = PyFloat_AS_DOUBLE(a[7]);
    const ScalarType wt = THPVariable_Unpack(a[2]).scalar_type();
    t.need((wt == kBf16 || wt == kF32) && H <= 16384 && M < (int64_t{1} << 31) && (!fp8 || H % kGroup == 0));
    const int64_t align = fp8 ? 16 : 2;
    const Tensor& w = t.dense(a[2], wt, {H}, align);
    t.need(aligned(x, align));
    const Tensor* post = a[4] == Py_None ? nullptr : &t.dense(a[4], wt, {H}, align);
    const Tensor* res = nullptr;
    ScalarType rt = kBf16;
    if (a[1] != Py_None) {
      if (!THPVariable_CheckExact(a[1])) return none();
      rt = THPVariable_Unpack(a[1]).scalar_type();
      t.need(rt == kBf16 || rt == kF32);
      res = &t.dense(a[1], rt, x.sizes(), align);
    }
    const Tensor* gate = nullptr;
    int64_t g_row = 0, g_col = 0;
    if (a[5] != Py_None && t.ok) {
      if (!THPVariable_CheckExact(a[5])) return none();
      const ScalarType gt = THPVariable_Unpack(a[5]).scalar_type();
      t.need(gt == kBf16 || gt == kF32);
      gate = &t.tensor(a[5], gt, -1);
      if (!t.ok || !gate->is_contiguous()) return none();
      at::DimVector rows(x.sizes().begin(), x.sizes().end());
      rows.back() = 1;
      if (H > 1 && gate->sizes() == IntArrayRef(rows)) g_row = 1;
      else if (gate->sizes() == x.sizes()) g_row = H, g_col = 1;
      else if (gate->dim() == 1 && gate->size(0) == H) g_col = 1;
      else return none();
      t.need(g_col == 0 || aligned(*gate, align));
    }
    if (!t.here()) return none();
    const bool same = !res && !post && !gate && scale == 1.0;  // r is x
    Tensor r = same ? x : at::empty(x.sizes(), x.options().dtype(rt));
    Tensor y, y8, ys;
    if (want) y = at::empty(x.sizes(), x.options());
    if (fp8) {
      y8 = at::empty(x.sizes(), x.options().dtype(kFp8));
      ys = at::empty_strided({M, H / kGroup}, {1, M}, x.options().dtype(kF32));
    }
    const int status = gdn_add_rms_norm(
        bf(x), H, res ? res->data_ptr() : nullptr, H, rt == kF32 ? 1 : 0, w.data_ptr(), post ? post->data_ptr() : nullptr,
        wt == kF32 ? 1 : 0, static_cast<float>(PyFloat_AS_DOUBLE(a[8])), gate ? gate->data_ptr() : nullptr,
        gate && gate->scalar_type() == kF32 ? 1 : 0, g_row, g_col, a[6] == Py_True ? 1 : 0, static_cast<float>(scale),
        static_cast<float>(PyFloat_AS_DOUBLE(a[3])), same ? nullptr : r.data_ptr(), want ? bf(y) : nullptr,
        fp8 ? ptr<uint8_t>(y8) : nullptr, fp8 ? ptr<float>(ys) : nullptr, 1, M, M, static_cast<int>(H), t.stream());
    if (failed("gdn_add_rms_norm", status)) return nullptr;
    auto given = [](bool is, Tensor& v) { return is ? THPVariable_Wrap(std::move(v)) : none(); };
    PyObject *oy = given(want, y), *o8 = given(fp8, y8), *os = given(fp8, ys);
    PyObject* o = same ? (Py_INCREF(a[0]), a[0]) : THPVariable_Wrap(std::move(r));
    return Py_BuildValue("(NNNN)", oy, o8, os, o);
  });
}

// The adapters of a product with N columns and its parts.
struct Adapters {
  int64_t S = 0, P = 0, R = 0;
  int n = 0, end[4] = {};
  int64_t width[4] = {};
  const Tensor *a = nullptr, *b = nullptr, *scale = nullptr, *ids = nullptr;
  Tensor work, parts[4];
  int64_t M = 0;

  // arguments lora_a, lora_b, lora_scale, ids; widths: a list, or None for one part
  bool take(Taken& t, PyObject* const* o, PyObject* widths, int64_t rows, int64_t N, int64_t K, IntArrayRef lead) {
    M = rows;
    if (widths == Py_None) {
      n = 1, width[0] = N, end[0] = static_cast<int>(N);
    } else {
      if (!PyList_CheckExact(widths) || PyList_GET_SIZE(widths) < 1 || PyList_GET_SIZE(widths) > 4) return false;
      int64_t sum = 0;
      for (n = 0; n < PyList_GET_SIZE(widths); ++n) {
        PyObject* w = PyList_GET_ITEM(widths, n);
        if (!PyLong_CheckExact(w)) return false;
        width[n] = PyLong_AsLongLong(w);
        if (width[n] <= 0 || width[n] > N - sum) {
          PyErr_Clear();
          return false;
        }
        sum += width[n];
        end[n] = static_cast<int>(sum);
        if (n + 1 < PyList_GET_SIZE(widths) && sum % 16) return false;
      }
      if (sum != N) return false;
    }
    a = &t.tensor(o[0], kBf16, 3);
    b = &t.tensor(o[1], kBf16, 3);
    if (!t.ok) return false;
    S = b->size(0), R = b->size(2), P = n;
    t.need(S > 0 && R >= 8 && R <= 256 && R % 8 == 0 && b->size(1) == N && a->size(0) == S && a->size(1) == P * R &&
           a->size(2) == K && S < (int64_t{1} << 31));
    for (const Tensor* v : {a, b})
      t.need(v->stride(2) == 1 && v->stride(1) == v->size(2) && aligned(*v) &&
             (S == 1 || (v->stride(0) % 8 == 0 && v->stride(0) >= v->size(1) * v->size(2))));
    scale = &t.dense(o[2], kF32, {S}, 4);
    ids = &t.tensor(o[3], ScalarType::Int, -1);
    if (!t.ok) return false;
    t.need(ids->is_contiguous() && ((ids->dim() == 1 && ids->size(0) == M) || ids->sizes() == lead));
    return t.ok;
  }
  uint16_t* v() const { return static_cast<uint16_t*>(work.data_ptr()); }
  int64_t ldv() const { return 2 * P * R; }
  int32_t* groups() const { return reinterpret_cast<int32_t*>(v() + M * ldv()); }
  void allocate(const Tensor& x, IntArrayRef lead) {
    work = at::empty({M * ldv() * 2 + (M + 15) / 16 * 4 + (M <= GDN_LORA_SORT ? 8 * M : 0)}, x.options().dtype(ScalarType::Byte));
    for (int i = 0; i < n; ++i) {
      at::DimVector shape(lead.begin(), lead.end());
      shape.push_back(width[i]);
      parts[i] = at::empty(shape, x.options().dtype(kBf16));
    }
  }
  // x8, s8: x in e4m3 too, and its scales
  int shrink(const Tensor& x, const Tensor* xs, int64_t K, void* stream, uint8_t* x8 = nullptr, float* s8 = nullptr) const {
    return gdn_lora_shrink(x.data_ptr(), xs ? 0 : 1, K, xs ? ptr<float>(*xs) : nullptr, xs ? xs->stride(0) : 0,
                           xs ? xs->stride(1) : 0, bf(*a), a->stride(0), ptr<float>(*scale), ptr<int32_t>(*ids),
                           static_cast<int>(S), static_cast<int>(P), static_cast<int>(R), static_cast<int>(M),
                           static_cast<int>(K), v(), ldv(), groups(), x8, K, s8, 1, M, stream);
  }
  PyObject* given(PyObject* widths) {
    if (widths == Py_None) return THPVariable_Wrap(std::move(parts[0]));
    PyObject* list = PyList_New(n);
    if (!list) return nullptr;
    for (int i = 0; i < n; ++i) PyList_SET_ITEM(list, i, THPVariable_Wrap(std::move(parts[i])));
    return list;
  }
};

// (x, weight, lora_a, lora_b, lora_scale, ids, widths or None) -> y, or the list of its parts
PyObject* linear_lora(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    Taken t;
    const Tensor& x = t.tensor(a[0], kBf16, -1);
    const Tensor& w = t.tensor(a[1], kBf16, 2);
    if (!t.ok || x.dim() < 2 || x.numel() == 0) return none();
    const int64_t N = w.size(0), K = w.size(1);
    if (N == 0 || K == 0 || K % 64 || x.size(-1) != K) return none();
    const int64_t M = x.numel() / K;
    const IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
    t.need(x.is_contiguous() && aligned(x) && w.stride(1) == 1 && w.stride(0) % 8 == 0 && w.stride(0) >= K && aligned(w) &&
           M < (int64_t{1} << 31) && N < (int64_t{1} << 31));
    Adapters l;
    if (!t.ok || !l.take(t, a + 2, a[6], M, N, K, lead) || !t.here()) return none();
    l.allocate(x, lead);
    uint16_t* c[4];
    for (int i = 0; i < l.n; ++i) c[i] = bf(l.parts[i]);
    void* stream = t.stream();
    if (failed("gdn_lora_shrink", l.shrink(x, nullptr, K, stream))) return nullptr;
    const int status = gdn_gemm_bf16_lora(
        bf(x), K, bf(w), w.stride(0), static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), l.n, c, l.width, l.end,
        nullptr, nullptr, nullptr, nullptr, 0, 0, 0, l.v(), l.ldv(), l.groups(), bf(*l.b), l.b->stride(0),
        ptr<int32_t>(*l.ids), static_cast<int>(l.S), static_cast<int>(l.R), l.n, l.end, stream);
    return failed("gdn_gemm_bf16_lora", status) ? nullptr : l.given(a[6]);
  });
}

// (x, weight, weight_scale, lora_a, lora_b, lora_scale, ids, x_scale or None, widths or None) -> the same
PyObject* linear_fp8_lora(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    Taken t;
    const bool ready = a[7] != Py_None;
    const Tensor& x = t.tensor(a[0], ready ? kFp8 : kBf16, -1);
    const Tensor& w = t.tensor(a[1], kFp8, 2);
    if (!t.ok || x.dim() < 2 || x.numel() == 0) return none();
    const int64_t N = w.size(0), K = w.size(1), G = K / kGroup;
    if (N == 0 || K == 0 || K % kGroup || x.size(-1) != K) return none();
    const int64_t M = x.numel() / K;
    const IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
    t.need(x.is_contiguous() && aligned(x) && w.stride(1) == 1 && w.stride(0) % 16 == 0 && w.stride(0) >= K && aligned(w) &&
           M < (int64_t{1} << 31) && N < (int64_t{1} << 31));
    const Tensor& ws = t.dense(a[2], kF32, {(N + kGroup - 1) / kGroup, G}, 4);
    const Tensor* xs = nullptr;
    if (t.ok && ready) {
      xs = &t.tensor(a[7], kF32, 2);
      if (t.ok) t.need(xs->size(0) == M && xs->size(1) == G);
    }
    Adapters l;
    if (!t.ok || !l.take(t, a + 3, a[8], M, N, K, lead) || !t.here()) return none();
    l.allocate(x, lead);
    uint16_t* c[4];
    for (int i = 0; i < l.n; ++i) c[i] = bf(l.parts[i]);
    void* stream = t.stream();
    Tensor x8, made;
    if (!ready) {
      x8 = at::empty({M, K}, x.options().dtype(kFp8));
      made = at::empty_strided({M, G}, {1, M}, x.options().dtype(kF32));
    }
    const int shrunk = ready ? l.shrink(x, xs, K, stream) : l.shrink(x, nullptr, K, stream, ptr<uint8_t>(x8), ptr<float>(made));
    if (failed("gdn_lora_shrink", shrunk)) return nullptr;
    if (!ready) xs = &made;
    const int status = gdn_gemm_fp8_lora(
        ptr<uint8_t>(ready ? x : x8), K, ptr<float>(*xs), xs->stride(0), xs->stride(1), ptr<uint8_t>(w), w.stride(0),
        ptr<float>(ws), G, static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), l.n, c, l.width, l.end, l.v(),
        l.ldv(), l.groups(), bf(*l.b), l.b->stride(0), ptr<int32_t>(*l.ids), static_cast<int>(l.S), static_cast<int>(l.R),
        l.n, l.end, stream);
    return failed("gdn_gemm_fp8_lora", status) ? nullptr : l.given(a[8]);
  });
}

// (check): check(name, status) raises
PyObject* set_check(PyObject*, PyObject* check) {
  Py_INCREF(check);
  Py_XSETREF(check_status, check);
  Py_RETURN_NONE;
}

#define GDN_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"conv_tree", GDN_FAST(conv_tree)},
                         {"rule_tree", GDN_FAST(rule_tree)},
                         {"rule_tree_layer", GDN_FAST(rule_tree_layer)},
                         {"verify_tree", GDN_FAST(verify_tree)},
                         {"verify_tree_norm", GDN_FAST(verify_tree_norm)},
                         {"commit_tree", GDN_FAST(commit_tree)},
                         {"linear_fp8", GDN_FAST(linear_fp8)},
                         {"norm_fp8", GDN_FAST(norm_fp8)},
                         {"add_norm", GDN_FAST(add_norm)},
                         {"linear_lora", GDN_FAST(linear_lora)},
                         {"linear_fp8_lora", GDN_FAST(linear_fp8_lora)},
                         {"set_check", set_check, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "gdn_quick_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_gdn_quick_calls() {
  PyObject* m = PyModule_Create(&module);
  // (of the header that the calls above were compiled with)
  if (m && PyModule_AddIntConstant(m, "ABI_VERSION", GDN_ABI_VERSION) != 0) Py_CLEAR(m);
  return m;
}
