// Host side of the operators on rows and of the optimizer step: what would be Python between a call and its kernels - allocation, the
// choice of kernels, autograd's nodes, tables of addresses.  The kernels themselves are reached through the C ABI's function pointers
// (bind), argument checks stay in Python.  Why native: a norm's or a product's kernels run for 5 to 50 us, autograd in Python around
// them for 110, and reading 350 tensors' addresses in Python takes 190 us beside an optimizer step of 20.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <algorithm>
#include <cstdint>
#include <utility>
#include <vector>
#include "../../include/selfc_hip.h"

namespace {

struct Seq {                       // a list or tuple, borrowed items
  PyObject* fast = nullptr;
  explicit Seq(PyObject* o) { if (o && o != Py_None) fast = PySequence_Fast(o, "expected a list of tensors"); }
  ~Seq() { Py_XDECREF(fast); }
  Py_ssize_t size() const { return fast ? PySequence_Fast_GET_SIZE(fast) : 0; }
  PyObject* item(Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(fast, i); }
};

bool fits(const at::Tensor& t, const at::Tensor& like) {
  return t.layout() == at::kStrided && t.scalar_type() == like.scalar_type() && t.device() == like.device() && t.is_contiguous();
}

// table(params or None, grads, steps or None, address of [len(grads)][4] uint64) -> (tensors with a gradient, their and the others' blocks of
// 256 values), or None where not everything is of one type on one device, contiguous and of equal shapes (the caller looks closer)
PyObject* table(PyObject*, PyObject* args) {
  PyObject *p_, *g_, *s_;
  unsigned long long address;
  if (!PyArg_ParseTuple(args, "OOOK", &p_, &g_, &s_, &address)) return nullptr;
  try {
    Seq ps(p_), gs(g_), ss(s_);
    if (PyErr_Occurred()) return nullptr;
    const Py_ssize_t n = gs.size();
    if ((ps.fast && ps.size() != n) || (ss.fast && ss.size() != n)) Py_RETURN_NONE;
    auto* const rows = reinterpret_cast<std::uint64_t*>(address);
    at::Tensor first;
    long long live = 0, blocks = 0;
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* const go = gs.item(i);
      const bool some = go != Py_None;
      if (some && !THPVariable_Check(go)) Py_RETURN_NONE;
      PyObject* const po = ps.fast ? ps.item(i) : go;
      std::uint64_t* const row = rows + 4 * i;
      row[0] = row[1] = row[2] = row[3] = 0;
      if (po == Py_None) {
        if (ps.fast) Py_RETURN_NONE;
        continue;
      }
      if (!THPVariable_Check(po)) Py_RETURN_NONE;
      const at::Tensor& p = THPVariable_Unpack(po);
      if (!first.defined()) first = p;
      if (!fits(p, first)) Py_RETURN_NONE;
      row[3] = static_cast<std::uint64_t>(p.numel());
      blocks += (p.numel() + 255) / 256;
      if (ps.fast) row[0] = reinterpret_cast<std::uint64_t>(p.data_ptr());
      if (some) {
        const at::Tensor& g = THPVariable_Unpack(go);
        if (!fits(g, first) || !g.sizes().equals(p.sizes())) Py_RETURN_NONE;
        row[1] = reinterpret_cast<std::uint64_t>(g.data_ptr());
        ++live;
      }
      if (ss.fast) {
        if (!THPVariable_Check(ss.item(i))) Py_RETURN_NONE;
        const at::Tensor& s = THPVariable_Unpack(ss.item(i));
        if (s.scalar_type() != at::kFloat || s.device() != first.device() || s.numel() != 1) Py_RETURN_NONE;
        row[2] = reinterpret_cast<std::uint64_t>(s.data_ptr());
      }
    }
    if (ps.fast && live > 1) {                 // each tensor is written by a workgroup of its own
      std::vector<std::pair<std::uint64_t, std::uint64_t>> at;
      at.reserve(live);
      for (Py_ssize_t i = 0; i < n; ++i)
        if (rows[4 * i + 1] && rows[4 * i + 3]) at.emplace_back(rows[4 * i], rows[4 * i] + rows[4 * i + 3] * first.element_size());
      std::sort(at.begin(), at.end());
      for (std::size_t i = 1; i < at.size(); ++i)
        if (at[i].first < at[i - 1].second) throw std::runtime_error("selfc_amd: two of the tensors share memory (one is in the list twice, or they overlap)");
    }
    return Py_BuildValue("LL", live, blocks);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// written(params, grads): the parameters that have a gradient were written in place (autograd's and the weight caches' version counters)
PyObject* written(PyObject*, PyObject* args) {
  PyObject *p_, *g_;
  if (!PyArg_ParseTuple(args, "OO", &p_, &g_)) return nullptr;
  try {
    Seq ps(p_), gs(g_);
    if (PyErr_Occurred()) return nullptr;
    for (Py_ssize_t i = 0; i < gs.size() && i < ps.size(); ++i)
      if (gs.item(i) != Py_None && THPVariable_Check(ps.item(i))) {
        const at::Tensor& p = THPVariable_Unpack(ps.item(i));
        if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
      }
    Py_RETURN_NONE;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// ---- the kernels' library --------------------------------------------------------------------------------------------------
#define ENTRIES(X)                                                                                                                    \
  X(selfc_rmsnorm) X(selfc_rmsnorm_bwd) X(selfc_rmsnorm_bwd_floats) X(selfc_linear_ws_floats) X(selfc_pack_rows) X(selfc_linear_any_layout) X(selfc_linear)       \
  X(selfc_linear_dz_floats) X(selfc_linear_dz) X(selfc_linear_dw_floats) X(selfc_linear_dx) X(selfc_linear_dw) X(selfc_linear_rows_ok) \
  X(selfc_linear_rows) X(selfc_linear_rows_bwd)
struct Api {
#define X(f) decltype(&::f) f = nullptr;
  ENTRIES(X)
#undef X
} api;

// bind({name: address}): once, from the loaded library
PyObject* bind(PyObject*, PyObject* map) {
#define X(f)                                                                        \
  {                                                                                 \
    PyObject* const a = PyDict_GetItemString(map, #f);                              \
    if (!a) { PyErr_SetString(PyExc_KeyError, #f); return nullptr; }                \
    api.f = reinterpret_cast<decltype(&::f)>(PyLong_AsUnsignedLongLong(a));         \
  }
  ENTRIES(X)
#undef X
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

void check(const int rc, const char* what) {
  if (rc == SELFC_OK) return;
  if (rc == SELFC_EINVAL) throw std::runtime_error(std::string(what) + ": SELFC_EINVAL - shape/argument not covered by the HIP kernels");
  throw std::runtime_error(std::string(what) + ": HIP runtime error " + std::to_string(-(rc + 1000)));
}

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

int code(const at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : 3; }
size_t pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* floats(const Tensor& t) { return static_cast<float*>(ptr(t)); }
Tensor empty(const Tensor& like, at::IntArrayRef shape, const at::ScalarType t) { return at::empty(shape, like.options().dtype(t).requires_grad(false)); }
Tensor work(const Tensor& like, const size_t n) { return n ? empty(like, {(int64_t)n}, at::kFloat) : Tensor(); }
int64_t up8(const int64_t n) { return (n + 7) / 8 * 8; }

// a matrix whose rows are contiguous and do not overlap
Tensor rows_of(const Tensor& t) {
  if ((t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1))) return t.contiguous();
  return t;
}
// can the tiled product read it as it is: 16-byte aligned rows of whole 16-byte pieces
bool whole(const Tensor& t) {
  const int64_t per = 16 / t.element_size();
  return reinterpret_cast<std::uintptr_t>(t.data_ptr()) % 16 == 0 && t.size(1) % per == 0 && pitch(t) % per == 0 && pitch(t) < (1u << 21);
}
Tensor pieces(const Tensor& t, void* const stream) {
  if (whole(t)) return t;
  const int64_t per = 16 / t.element_size(), ldd = (t.size(1) + per - 1) / per * per;
  const Tensor out = empty(t, {t.size(0), ldd}, t.scalar_type());
  check(api.selfc_pack_rows(t.data_ptr(), pitch(t), out.data_ptr(), t.size(0), (int)t.size(1), (int)ldd, (int)t.element_size(), stream), "selfc_pack_rows");
  return out;
}

// create_graph=True: the gradients here have none of their own
void first_only() {
  if (at::GradMode::is_enabled()) throw std::runtime_error("selfc_amd: no second derivatives (create_graph=True)");
}

// forward-mode derivatives: the kernels make none, so an input that carries a tangent must not pass as a plain one
void no_tangents(const std::initializer_list<PyObject*> inputs) {
  for (PyObject* const o : inputs)
    if (o != Py_None && THPVariable_Unpack(o)._fw_grad(0).defined()) throw std::runtime_error("selfc_amd: no forward-mode derivatives (an input is a dual tensor)");
}

// ---- norm ----------------------------------------------------------------------------------------------------------------------
struct NormOut { Tensor y, scale, h; };
NormOut run_norm(const Tensor& x, const Tensor& r, const Tensor& w, const double eps, const bool q8, void* const stream) {
  const int64_t rows = x.size(0), cols = x.size(1);
  NormOut o;
  o.y = empty(x, {rows, cols}, q8 ? at::kFloat8_e4m3fn : x.scalar_type());
  if (q8) o.scale = empty(x, {rows}, at::kFloat);
  if (r.defined()) o.h = empty(x, {rows, cols}, x.scalar_type());
  if (rows)
    check(api.selfc_rmsnorm(x.data_ptr(), pitch(x), ptr(r), r.defined() ? pitch(r) : 0, w.data_ptr(), w.scalar_type() == at::kFloat, ptr(o.h), o.y.data_ptr(),
                            floats(o.scale), rows, (int)cols, code(x.scalar_type()), (float)eps, stream), "selfc_rmsnorm");
  return o;
}

// the gradient needs h and the weight only: the row's statistic is recomputed
struct NormFn : torch::autograd::Function<NormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& r, const Tensor& w, const double eps, const int64_t stream) {
    const NormOut o = run_norm(x, r.value_or(Tensor()), w, eps, false, reinterpret_cast<void*>(stream));
    ctx->set_materialize_grads(false);
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["res"] = r.has_value();
    ctx->save_for_backward({o.h.defined() ? o.h : x, w});
    return o.h.defined() ? variable_list{o.y, o.h} : variable_list{o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_only();
    const auto saved = ctx->get_saved_variables();
    const Tensor h = saved[0], w = saved[1];
    const bool res = ctx->saved_data["res"].toBool();
    const bool to_x = ctx->needs_input_grad(0), to_r = res && ctx->needs_input_grad(1), to_w = ctx->needs_input_grad(res ? 2 : 1);
    Tensor dy = g[0], dh = res ? g[1] : Tensor(), dx, dw;
    if (!dy.defined()) {                   // only h was used
      dx = dh;
    } else {
      const int64_t rows = h.size(0), cols = h.size(1);
      dy = dy.contiguous();
      if (dh.defined()) dh = dh.contiguous();
      if (to_x || to_r) dx = empty(h, {rows, cols}, h.scalar_type());
      if (to_w) dw = empty(w, {cols}, w.scalar_type());
      if (rows) {
        const Tensor part = to_w ? work(h, api.selfc_rmsnorm_bwd_floats(rows, (int)cols)) : Tensor();
        check(api.selfc_rmsnorm_bwd(h.data_ptr(), pitch(h), w.data_ptr(), w.scalar_type() == at::kFloat, dy.data_ptr(), ptr(dh), ptr(dx), ptr(dw), floats(part),
                                    rows, (int)cols, code(h.scalar_type()), (float)ctx->saved_data["eps"].toDouble(),
                                    reinterpret_cast<void*>(ctx->saved_data["stream"].toInt())), "selfc_rmsnorm_bwd");
      } else if (to_w) {
        dw.zero_();
      }
    }
    return {to_x ? dx : Tensor(), to_r ? dx : Tensor(), dw, Tensor(), Tensor()};
  }
};

// ---- product -------------------------------------------------------------------------------------------------------------------
// Layers whose weight the rows' kernel holds in shared memory.  It reads any layout, so it takes all rows that would have to be laid out
// first; of the others those whose number pays for every workgroup's copy of the weight: in f16, here and in tiles, 64 x 64 with 2,000 rows
// 4.8 us, 5.1; 128 x 128 with 20,000 8.1, 7.2 and with 50,000 10.4, 11.9; 256 x 256 with 100,000 47.5, 40.2 and with 200,000 71.9, 76.4 (and their
// gradients likewise)
bool narrow(const Tensor& x, const Tensor& w) {
  const int64_t n = w.size(0), k = w.size(1);
  if (n > 256 || k > 256 || !api.selfc_linear_rows_ok((int)n, (int)k)) return false;
  return !whole(x) || !whole(w) || n * k <= 4096 || x.size(0) >= 2 * n * k;
}

// room for the activation's derivative: a bit per value of ReLU and LeakyReLU, 16 bits of the others
Tensor kept(const Tensor& like, const int64_t rows, const int64_t n, const int act) {
  return act == 1 || act == 2 ? empty(like, {rows, up8(n) / 8}, at::kByte) : empty(like, {rows, up8(n)}, at::kShort);
}
struct LinearOut { Tensor y, slope, xp; };          // xp: x as dW's product reads it
// one launch, any layout of x and the weight
LinearOut run_rows(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r, const int act, const bool want_slope, const bool want_xp, void* const stream) {
  const int64_t rows = x.size(0), k = x.size(1), n = w.size(0);
  LinearOut o;
  o.y = empty(x, {rows, n}, x.scalar_type());
  if (want_slope) o.slope = kept(x, rows, n, act);
  const bool as_is = !want_xp || whole(x);
  if (want_xp) o.xp = as_is ? x : empty(x, {rows, up8(k)}, x.scalar_type());
  if (rows)
    check(api.selfc_linear_rows(x.data_ptr(), pitch(x), w.data_ptr(), pitch(w), ptr(b), act, ptr(r), r.defined() ? pitch(r) : 0, o.y.data_ptr(), ptr(o.slope),
                                as_is ? nullptr : o.xp.data_ptr(), rows, (int)n, (int)k, code(x.scalar_type()), stream), "selfc_linear_rows");
  return o;
}
LinearOut run_tiles(const Tensor& x, const Tensor& w, const Tensor& xs, const Tensor& ws, const Tensor& b, const Tensor& r, const int act, const at::ScalarType out,
                    const bool want_slope, const bool grad, void* const stream, Tensor& wp) {
  const int64_t rows = x.size(0), n = w.size(0), es = x.element_size();
  // (the backward pass reads whole pieces)
  const bool lies = !grad && api.selfc_linear_any_layout(rows, (int)x.size(1), (int)es) && !(whole(x) && whole(w));
  const int64_t k = lies ? x.size(1) : (x.size(1) * es + 15) / 16 * 16 / es;
  LinearOut o;
  o.y = empty(x, {rows, n}, out);
  if (want_slope) o.slope = kept(x, rows, n, act);
  o.xp = lies ? x : pieces(x, stream);
  wp = lies ? w : pieces(w, stream);
  if (rows) {
    const Tensor part = work(x, api.selfc_linear_ws_floats(rows, (int)n, (int)k, (int)es));
    check(api.selfc_linear(o.xp.data_ptr(), pitch(o.xp), wp.data_ptr(), pitch(wp), floats(xs), floats(ws), ptr(b), act, ptr(r), r.defined() ? pitch(r) : 0,
                           o.y.data_ptr(), ptr(o.slope), floats(part), rows, (int)n, (int)k, code(x.scalar_type()), code(out), stream), "selfc_linear");
  }
  return o;
}

// kept for the backward pass: x as the kernels read it, the weight, and the activation's derivative
struct LinearFn : torch::autograd::Function<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& r, const int64_t act, const int64_t stream) {
    const bool to_x = x.requires_grad(), to_w = w.requires_grad(), to_b = b && b->requires_grad();
    void* const s = reinterpret_cast<void*>(stream);
    const bool slope = act != 0 && (to_x || to_w || to_b), small = narrow(x, w);
    Tensor wp = w;
    const LinearOut o = small ? run_rows(x, w, b.value_or(Tensor()), r.value_or(Tensor()), (int)act, slope, to_w, s)
                              : run_tiles(x, w, Tensor(), Tensor(), b.value_or(Tensor()), r.value_or(Tensor()), (int)act, x.scalar_type(), slope, true, s, wp);
    ctx->saved_data["dims"] = std::vector<int64_t>{x.size(0), w.size(0), x.size(1), (int64_t)small, stream, b ? 1 : 0, r ? 1 : 0, act};
    ctx->save_for_backward({to_w ? o.xp : Tensor(), to_x ? wp : Tensor(), o.slope});
    return o.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_only();
    const auto saved = ctx->get_saved_variables();
    const Tensor xp = saved[0], wp = saved[1], slope = saved[2];
    const auto d = ctx->saved_data["dims"].toIntVector();
    const int64_t rows = d[0], n = d[1], k = d[2], up = up8(n);
    const bool small = d[3];
    void* const s = reinterpret_cast<void*>(d[4]);
    const bool to_x = ctx->needs_input_grad(0), to_w = ctx->needs_input_grad(1), to_b = d[5] && ctx->needs_input_grad(2), to_r = d[6] && ctx->needs_input_grad(2 + d[5]);
    const Tensor& dy = grads[0];
    const at::ScalarType t = dy.scalar_type();
    const int c = code(t);
    Tensor dx, dw, db;
    if (to_x) dx = empty(dy, {rows, k}, t);
    if (to_w) dw = empty(dy, {n, k}, t);
    if (to_b) db = empty(dy, {n}, t);
    if (rows == 0) {
      if (to_w) dw.zero_();
      if (to_b) db.zero_();
      return {dx, dw, db, to_r ? dy : Tensor(), Tensor(), Tensor()};
    }
    const Tensor g = rows_of(dy);
    // dz as an operand: dy itself where no activation changes it and the products can read it
    const bool as_is = !slope.defined() && whole(g), rows_kernel = to_x && small, make = !as_is && (to_w || (to_x && !rows_kernel));
    const Tensor dz = make ? empty(dy, {rows, up}, t) : g;
    if (rows_kernel)
      check(api.selfc_linear_rows_bwd(g.data_ptr(), pitch(g), ptr(slope), (int)d[7], wp.data_ptr(), pitch(wp), dx.data_ptr(), make ? dz.data_ptr() : nullptr, rows, (int)n,
                                      (int)k, c, s), "selfc_linear_rows_bwd");
    const bool alone = to_b && !to_w;       // with dW, db comes out of that product
    if (alone || (make && !rows_kernel)) {
      const Tensor part = alone ? work(dy, api.selfc_linear_dz_floats(rows, (int)n)) : Tensor();
      check(api.selfc_linear_dz(g.data_ptr(), pitch(g), ptr(slope), (int)d[7], make && !rows_kernel ? dz.data_ptr() : nullptr, up, alone ? db.data_ptr() : nullptr, floats(part),
                                rows, (int)n, c, s), "selfc_linear_dz");
    }
    if (to_x && !rows_kernel) {
      const Tensor part = work(dy, api.selfc_linear_ws_floats(rows, (int)k, (int)n, 2));
      check(api.selfc_linear_dx(dz.data_ptr(), pitch(dz), wp.data_ptr(), pitch(wp), dx.data_ptr(), floats(part), rows, (int)n, (int)k, c, s), "selfc_linear_dx");
    }
    if (to_w) {
      const Tensor part = work(dy, api.selfc_linear_dw_floats(rows, (int)n, (int)k));
      check(api.selfc_linear_dw(dz.data_ptr(), pitch(dz), xp.data_ptr(), pitch(xp), dw.data_ptr(), ptr(db), floats(part), rows, (int)n, (int)k, c, s), "selfc_linear_dw");
    }
    return {dx, dw, db, to_r ? dy : Tensor(), Tensor(), Tensor()};
  }
};

// ---- Python's side -------------------------------------------------------------------------------------------------------------
Tensor tensor(PyObject* o) { return o == Py_None ? Tensor() : THPVariable_Unpack(o); }
OptTensor maybe(PyObject* o) { return o == Py_None ? OptTensor() : OptTensor(THPVariable_Unpack(o)); }
PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// norm(x, r or None, w, eps, q8, grad, stream) -> (y, scale or None, h or None)
PyObject* norm(PyObject*, PyObject* args) {
  PyObject *x, *r, *w;
  double eps;
  int q8, grad;
  unsigned long long stream;
  if (!PyArg_ParseTuple(args, "OOOdppK", &x, &r, &w, &eps, &q8, &grad, &stream)) return nullptr;
  return guarded([&]() -> PyObject* {
    no_tangents({x, r, w});
    NormOut o;
    if (grad) {
      const variable_list v = NormFn::apply(THPVariable_Unpack(x), maybe(r), THPVariable_Unpack(w), eps, (int64_t)stream);
      o.y = v[0];
      if (v.size() > 1) o.h = v[1];
    } else {
      o = run_norm(THPVariable_Unpack(x), tensor(r), THPVariable_Unpack(w), eps, q8, reinterpret_cast<void*>(stream));
    }
    return Py_BuildValue("NNN", wrap(o.y), wrap(o.scale), wrap(o.h));
  });
}

// linear(x, w, b or None, r or None, act, grad, stream) -> y
PyObject* linear(PyObject*, PyObject* args) {
  PyObject *x_, *w_, *b, *r;
  int act, grad;
  unsigned long long stream;
  if (!PyArg_ParseTuple(args, "OOOOipK", &x_, &w_, &b, &r, &act, &grad, &stream)) return nullptr;
  return guarded([&]() -> PyObject* {
    no_tangents({x_, w_, b, r});
    const Tensor &x = THPVariable_Unpack(x_), &w = THPVariable_Unpack(w_);
    if (grad) return wrap(LinearFn::apply(x, w, maybe(b), maybe(r), (int64_t)act, (int64_t)stream));
    void* const s = reinterpret_cast<void*>(stream);
    if (narrow(x, w)) return wrap(run_rows(x, w, tensor(b), tensor(r), act, false, false, s).y);
    Tensor wp;
    return wrap(run_tiles(x, w, Tensor(), Tensor(), tensor(b), tensor(r), act, x.scalar_type(), false, false, s, wp).y);
  });
}

// linear_q8(x, x_scale, w, w_scale, b or None, r or None, act, type of the output as in the C ABI, stream) -> y
PyObject* linear_q8(PyObject*, PyObject* args) {
  PyObject *x, *xs, *w, *ws, *b, *r;
  int act, out;
  unsigned long long stream;
  if (!PyArg_ParseTuple(args, "OOOOOOiiK", &x, &xs, &w, &ws, &b, &r, &act, &out, &stream)) return nullptr;
  return guarded([&]() -> PyObject* {
    no_tangents({x, xs, w, ws, b, r});
    Tensor wp;
    const at::ScalarType t = out == 0 ? at::kFloat : out == 1 ? at::kBFloat16 : at::kHalf;
    return wrap(run_tiles(THPVariable_Unpack(x), THPVariable_Unpack(w), THPVariable_Unpack(xs), THPVariable_Unpack(ws), tensor(b), tensor(r), act, t, false, false,
                          reinterpret_cast<void*>(stream), wp).y);
  });
}

PyMethodDef methods[] = {{"table", table, METH_VARARGS, nullptr},   {"written", written, METH_VARARGS, nullptr}, {"bind", bind, METH_O, nullptr},
                         {"norm", norm, METH_VARARGS, nullptr},     {"linear", linear, METH_VARARGS, nullptr},   {"linear_q8", linear_q8, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
