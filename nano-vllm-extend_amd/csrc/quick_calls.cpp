// The short calls' way from Python without its cost: a call whose tensors the kernel takes
// as they are (types, shapes, strides, alignment, one device, the current one) is checked,
// allocated and launched here, in about 5 us where the Python wrapper and ctypes take 9 to
// 14.  Anything else returns None: the wrapper's own checks then say what is wrong, or copy.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/hip/HIPFunctions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
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
  const Tensor& tensor(PyObject* o, ScalarType type, int64_t dim) {
    static const Tensor none;
    if (!ok || !THPVariable_CheckExact(o)) {
      ok = false;
      return none;
    }
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.scalar_type() != type || t.layout() != at::kStrided || (dim >= 0 && t.dim() != dim)) {
      ok = false;
      return none;
    }
    const int d = t.get_device();
    need(dev < 0 || dev == d);
    dev = d;
    return ok ? t : none;
  }
  // [B, T, C] or [B, T, H, D] rows that the kernels read in 16-byte pieces
  const Tensor& rows(PyObject* o, IntArrayRef shape) {
    const Tensor& t = tensor(o, kBf16, static_cast<int64_t>(shape.size()));
    if (!ok) return t;
    const IntArrayRef st = t.strides();
    const bool heads = shape.size() == 4;
    const int64_t width = heads ? shape[2] * shape[3] : shape[2];
    need(t.sizes() == shape && st.back() == 1 && (!heads || st[2] == shape[3] || shape[2] == 1) && width <= st[1] &&
         st[1] < (1 << 24) && st[0] % 8 == 0 && st[1] % 8 == 0 && aligned(t));
    return t;
  }
  const Tensor& dense(PyObject* o, ScalarType type, IntArrayRef shape, int64_t align) {
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

// What a call of one function gives: its C++ exceptions become Python's.
template <class F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F&& f) {
  if (n != want) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    return f();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyObject* none() { Py_RETURN_NONE; }

// (x, conv_pool, ids, weight, parents, pending) -> y
PyObject* conv_tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> PyObject* {
    Taken t;
    const Tensor& x = t.tensor(a[0], kBf16, 3);
    if (!t.ok) return none();
    const int64_t B = x.size(0), T = x.size(1), C = x.size(2);
    int64_t p_b = 0, lp_b = 0, last_T = 0;
    t.rows(a[0], {B, T, C});
    const Tensor& pool = t.conv_pool(a[1], C);
    const Tensor& ids = t.ids(a[2], B);
    const Tensor& w = t.tensor(a[3], kBf16, -1);
    const Tensor& par = t.parents(a[4], B, T, p_b);
    if (!t.ok || w.numel() != 4 * C || w.dim() == 0 || w.size(-1) != 4 || !w.is_contiguous() || C % 8) return none();
    const Tensor *lx = nullptr, *lpar = nullptr, *acc = nullptr;
    if (PyObject* p = t.pending(a[5], 3)) {
      lx = &t.tensor(PyTuple_GET_ITEM(p, 0), kBf16, 3);
      if (!t.ok) return none();
      last_T = lx->size(1);
      t.rows(PyTuple_GET_ITEM(p, 0), {B, last_T, C});
      lpar = &t.parents(PyTuple_GET_ITEM(p, 1), B, last_T, lp_b);
      acc = &t.ids(PyTuple_GET_ITEM(p, 2), B);
    }
    if (!t.here()) return none();
    Tensor y = at::empty({B, T, C}, x.options());
    const int status = gdn_conv_tree(
        bf(x), x.stride(0), x.stride(1), bf(pool), pool.stride(0), pool.stride(1), pool.size(0), ptr<int64_t>(ids), bf(w),
        ptr<int32_t>(par), p_b, lx ? bf(*lx) : nullptr, lx ? lx->stride(0) : 0, lx ? lx->stride(1) : 0,
        lpar ? ptr<int32_t>(*lpar) : nullptr, lp_b, acc ? ptr<int64_t>(*acc) : nullptr, static_cast<int>(last_T), bf(y),
        static_cast<int>(B), static_cast<int>(T), static_cast<int>(C), t.stream());
    return failed("gdn_conv_tree", status) ? nullptr : THPVariable_Wrap(std::move(y));
  });
}

// What the two forms of the rule share: q, k, v, the pool, ids, parents and the pending step.
struct Rule {
  Taken t;
  int64_t B = 0, T = 0, Hk = 0, Hv = 0, D = 0, p_b = 0, lp_b = 0, last_T = 0;
  const Tensor *q = nullptr, *k = nullptr, *v = nullptr, *pool = nullptr, *ids = nullptr, *par = nullptr;
  const Tensor *lk = nullptr, *lg = nullptr, *lu = nullptr, *lpar = nullptr, *acc = nullptr;

  bool take(PyObject* oq, PyObject* ok_, PyObject* ov, PyObject* opool, PyObject* oids, PyObject* opar,
            PyObject* opending) {
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
  int call(Entry entry, const std::tuple<Gates...>& gates, const std::tuple<Out...>& out) const {
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
                        static_cast<int>(D), static_cast<float>(std::pow(static_cast<double>(D), -0.5)), t.stream())));
  }
};

// (q, k, v, g, beta, s_pool, ids, parents, pending) -> (o, u)
PyObject* rule_tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    Rule r;
    if (!r.take(a[0], a[1], a[2], a[5], a[6], a[7], a[8])) return none();
    const Tensor& g = r.t.dense(a[3], kF32, {r.B, r.T, r.Hv}, 16);
    const Tensor& beta = r.t.dense(a[4], kBf16, {r.B, r.T, r.Hv}, 2);
    if (!r.t.here()) return none();
    Tensor o = at::empty({r.B, r.T, r.Hv, r.D}, r.v->options()), u = at::empty({r.B, r.T, r.Hv, r.D}, g.options());
    const int status = r.call(gdn_rule_tree, std::make_tuple(ptr<float>(g), bf(beta)),
                              std::make_tuple(bf(o), ptr<float>(u)));
    if (failed("gdn_rule_tree", status)) return nullptr;
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(o)), THPVariable_Wrap(std::move(u)));
  });
}

// (q, k, v, b, a, a_log, dt_bias, z, norm_weight, s_pool, ids, parents, eps, pending, fp8)
// -> (y, scale or None, u, g)
PyObject* rule_tree_layer(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 15, [&]() -> PyObject* {
    Rule r;
    if (!PyFloat_CheckExact(a[12]) || !PyBool_Check(a[14]) ||
        !r.take(a[0], a[1], a[2], a[9], a[10], a[11], a[13]))
      return none();
    const bool fp8 = a[14] == Py_True;
    const Tensor& b = r.t.dense(a[3], kBf16, {r.B, r.T, r.Hv}, 2);
    const Tensor& ga = r.t.dense(a[4], kBf16, {r.B, r.T, r.Hv}, 2);
    if (!r.t.ok || !THPVariable_CheckExact(a[5])) return none();
    const ScalarType param = THPVariable_Unpack(a[5]).scalar_type();
    const Tensor& a_log = r.t.dense(a[5], param, {r.Hv}, 2);
    const Tensor& dt = r.t.dense(a[6], param, {r.Hv}, 2);
    const Tensor& z = r.t.rows(a[7], {r.B, r.T, r.Hv * r.D});
    const Tensor& w = r.t.dense(a[8], kBf16, {r.D}, 16);
    if ((param != kBf16 && param != kF32) || (fp8 && r.D != kGroup) || !r.t.here()) return none();
    const auto f32 = r.pool->options();
    Tensor y = at::empty({r.B, r.T, r.Hv, r.D}, r.v->options().dtype(fp8 ? kFp8 : kBf16)), scale;
    if (fp8) scale = at::empty_strided({r.B * r.T, r.Hv}, {1, r.B * r.T}, f32);
    Tensor u = at::empty({r.B, r.T, r.Hv, r.D}, f32), g = at::empty({r.B, r.T, r.Hv}, f32);
    const int status = r.call(
        gdn_rule_tree_layer, std::make_tuple(bf(b), bf(ga), a_log.data_ptr(), dt.data_ptr(), param == kF32 ? 1 : 0),
        std::make_tuple(bf(z), z.stride(0), z.stride(1), bf(w), static_cast<float>(PyFloat_AS_DOUBLE(a[12])),
                        fp8 ? nullptr : bf(y), fp8 ? ptr<uint8_t>(y) : nullptr, fp8 ? ptr<float>(scale) : nullptr,
                        ptr<float>(u), ptr<float>(g)));
    if (failed("gdn_rule_tree_layer", status)) return nullptr;
    PyObject* s = fp8 ? THPVariable_Wrap(std::move(scale)) : none();
    return Py_BuildValue("(NNNN)", THPVariable_Wrap(std::move(y)), s, THPVariable_Wrap(std::move(u)),
                         THPVariable_Wrap(std::move(g)));
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
    Taken t;
    const Tensor& x = t.tensor(a[0], kBf16, -1);
    if (!t.ok || x.dim() < 2 || !x.is_contiguous() || !aligned(x) || x.numel() == 0 || !PyFloat_CheckExact(a[3]))
      return none();
    const int64_t H = x.size(-2), D = x.size(-1), tokens = x.numel() / (H * D), G = H * D / kGroup;
    const Tensor& z = t.dense(a[1], kBf16, x.sizes(), 16);
    const Tensor& w = t.dense(a[2], kBf16, {D}, 16);
    if (H * D % kGroup || !t.here()) return none();
    Tensor y = at::empty(x.sizes(), x.options().dtype(kFp8));
    Tensor scale = at::empty_strided({tokens, G}, {1, tokens}, x.options().dtype(kF32));
    const int status = gdn_rmsnorm_gated_fp8(bf(x), H * D, bf(z), H * D, bf(w), ptr<uint8_t>(y), ptr<float>(scale), 1,
                                             tokens, tokens, static_cast<int>(H), static_cast<int>(D),
                                             static_cast<float>(PyFloat_AS_DOUBLE(a[3])), t.stream());
    if (failed("gdn_rmsnorm_gated_fp8", status)) return nullptr;
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(y)), THPVariable_Wrap(std::move(scale)));
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
                         {"commit_tree", GDN_FAST(commit_tree)},
                         {"linear_fp8", GDN_FAST(linear_fp8)},
                         {"norm_fp8", GDN_FAST(norm_fp8)},
                         {"set_check", set_check, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "gdn_quick_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_gdn_quick_calls() { return PyModule_Create(&module); }
