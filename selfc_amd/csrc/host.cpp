// Host side of the optimizer step: the table of addresses and sizes that selfc_adamw_step takes, read from Python's tensors in one pass.
// (In Python the same checks and reads are seven passes over the lists: 190 us for the 350 tensors of the large rescaling network, more
// than ten times what the GPU needs for the step.)
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/python_variable.h>
#include <cstdint>

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

PyMethodDef methods[] = {{"table", table, METH_VARARGS, nullptr}, {"written", written, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
