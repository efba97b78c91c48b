// Python module `_direct`: the calls of serving_calls.h without the operator dispatcher in between, for the smallest
// launches (a single token's call takes the GPU 4 to 9 us; through torch.ops the host needs 8 to 10 us for it).

#include <Python.h>

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "serving_calls.h"

namespace {

const at::Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a torch.Tensor");
  return THPVariable_Unpack(o);
}

std::optional<at::Tensor> maybe_tensor(PyObject* o, const char* name) {
  if (o == Py_None) return std::nullopt;
  return tensor(o, name);
}

int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}

c10::SmallVector<int64_t, 16> integers(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(PyTuple_Check(o), name, " must be a tuple");
  c10::SmallVector<int64_t, 16> out;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(o); ++i) out.push_back(integer(PyTuple_GET_ITEM(o, i)));
  return out;
}

// A tuple of two tensors (None for an undefined one) and, where `flag` is given, a truth value.
PyObject* tuple_of(const at::Tensor& a, const at::Tensor& b, const bool* flag = nullptr) {
  PyObject* out = PyTuple_New(flag != nullptr ? 3 : 2);
  if (out == nullptr) throw python_error();
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(a));
  if (b.defined()) {
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(b));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(out, 1, Py_None);
  }
  if (flag != nullptr) PyTuple_SET_ITEM(out, 2, PyBool_FromLong(*flag ? 1 : 0));
  return out;
}

// q, k, v, k_prefix, v_prefix, table, plan, scale, return_lse, out
PyObject* attention_planned(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 10, "attention_planned takes 10 arguments");
  const auto [o, lse, captured] = b200attn_torch::attention_planned(
      tensor(a[0], "q"), tensor(a[1], "k"), tensor(a[2], "v"), maybe_tensor(a[3], "k_prefix"),
      maybe_tensor(a[4], "v_prefix"), tensor(a[5], "table"), integers(a[6], "plan"), real(a[7]), truth(a[8]),
      maybe_tensor(a[9], "out"));
  return tuple_of(o, lse, &captured);
  END_HANDLE_TH_ERRORS
}

// q, k, positions, inv_freq, sections, q_weight, k_weight, eps, interleaved, q_out, k_out
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 11, "qk_norm_rope takes 11 arguments");
  const auto [qo, ko] = b200attn_torch::qk_norm_rope(
      tensor(a[0], "q"), maybe_tensor(a[1], "k"), tensor(a[2], "positions"), tensor(a[3], "inv_freq"),
      integers(a[4], "sections"), maybe_tensor(a[5], "q_weight"), maybe_tensor(a[6], "k_weight"), real(a[7]), truth(a[8]),
      maybe_tensor(a[9], "out of q"), maybe_tensor(a[10], "out of k"));
  return tuple_of(qo, ko);
  END_HANDLE_TH_ERRORS
}

// The rules on where an output may lie, for tensors of any device.
PyObject* may_overlap(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 2, "may_overlap takes 2 arguments");
  return PyBool_FromLong(b200attn_torch::may_overlap(tensor(a[0], "a"), tensor(a[1], "b")) ? 1 : 0);
  END_HANDLE_TH_ERRORS
}

PyObject* same_place(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 2, "same_place takes 2 arguments");
  return PyBool_FromLong(b200attn_torch::same_place(tensor(a[0], "a"), tensor(a[1], "b")) ? 1 : 0);
  END_HANDLE_TH_ERRORS
}

PyObject* dense_apart(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 1, "dense_apart takes 1 argument");
  return PyBool_FromLong(b200attn_torch::dense_apart(tensor(a[0], "t")) ? 1 : 0);
  END_HANDLE_TH_ERRORS
}

// out, the input that it may be, another input
PyObject* check_place(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 3, "check_place takes 3 arguments");
  b200attn_torch::check_place("out", tensor(a[0], "out"), "q", &tensor(a[1], "q"), {{"k", &tensor(a[2], "k")}});
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* free_tables(PyObject*, PyObject*) {
  HANDLE_TH_ERRORS
  b200attn_torch::free_tables();
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"free_tables", &free_tables, METH_NOARGS, nullptr},
    {"may_overlap", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&may_overlap)), METH_FASTCALL, nullptr},
    {"same_place", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&same_place)), METH_FASTCALL, nullptr},
    {"dense_apart", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&dense_apart)), METH_FASTCALL, nullptr},
    {"check_place", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&check_place)), METH_FASTCALL, nullptr},
    {"attention_planned", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&attention_planned)), METH_FASTCALL, nullptr},
    {"qk_norm_rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&qk_norm_rope)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_direct", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__direct() { return PyModule_Create(&module); }
