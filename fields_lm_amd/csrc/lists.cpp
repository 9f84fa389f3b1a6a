// lists.cpp — what the optimizer's calls read of a Python list of tensors, in one pass and without a Python
// object per attribute. A step reads some twenty attributes of each of a model's hundreds of tensors: through
// Python's accessors that is 1.2 us a tensor, more than the kernels take for most models.
//
// read(tensors, device_index, dtypes, addresses, counts, codes, expected, block) -> None, or (index, what is wrong)
//   tensors: a list or tuple; dtypes: the torch dtypes taken, in the order of their codes; addresses, counts (int64)
//   and codes (int32): host addresses of arrays that hold len(tensors) words, 0 for not wanted; expected: the same of
//   the counts that the tensors must have, in blocks of `block` values (rounded up).
// same_shapes(a, b) -> the index of the first pair that differs, or -1.
// repeats(addresses, counts, n) -> whether two of the n addresses with a count that is not 0 are equal (counts 0: any).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <vector>

namespace {

// Items of a list or tuple, borrowed.
struct Items {
  PyObject** at = nullptr;
  Py_ssize_t n = 0;
  bool of(PyObject* o) {
    if (!PyList_Check(o) && !PyTuple_Check(o)) {
      PyErr_SetString(PyExc_TypeError, "a list or tuple is wanted");
      return false;
    }
    at = PySequence_Fast_ITEMS(o);
    n = PySequence_Fast_GET_SIZE(o);
    return true;
  }
};

PyObject* wrong(Py_ssize_t i, const char* what) { return Py_BuildValue("(ns)", i, what); }

PyObject* read(PyObject*, PyObject* args) {
  PyObject *list, *types;
  long long device, addresses, counts, codes, expected, block;
  Items items, taken;
  if (!PyArg_ParseTuple(args, "OLOLLLLL", &list, &device, &types, &addresses, &counts, &codes, &expected,
                        &block) || !items.of(list) ||
      !taken.of(types))
    return nullptr;
  at::ScalarType wanted[8];
  if (block < 1) return PyErr_Format(PyExc_ValueError, "a block has 1 value or more");
  if (taken.n > 8) return PyErr_Format(PyExc_ValueError, "at most 8 types");
  for (Py_ssize_t k = 0; k < taken.n; ++k) {
    if (!THPDtype_Check(taken.at[k])) return PyErr_Format(PyExc_TypeError, "a dtype is wanted");
    wanted[k] = reinterpret_cast<THPDtype*>(taken.at[k])->scalar_type;
  }
  try {
    for (Py_ssize_t i = 0; i < items.n; ++i) {
      if (!THPVariable_Check(items.at[i])) return wrong(i, "tensor");
      const at::Tensor& t = THPVariable_Unpack(items.at[i]);
      Py_ssize_t code = 0;
      while (code < taken.n && wanted[code] != t.scalar_type()) ++code;
      if (code == taken.n) return wrong(i, "dtype");
      if (t.layout() != at::kStrided || t.is_neg()) return wrong(i, "layout");
      if (!t.device().is_cuda() || t.device().index() != device) return wrong(i, "device");
      if (!t.is_contiguous()) return wrong(i, "contiguous");
      if (expected && t.numel() != (reinterpret_cast<const int64_t*>(expected)[i] + block - 1) / block) return wrong(i, "count");
      if (addresses) reinterpret_cast<int64_t*>(addresses)[i] = reinterpret_cast<int64_t>(t.data_ptr());
      if (counts) reinterpret_cast<int64_t*>(counts)[i] = t.numel();
      if (codes) reinterpret_cast<int32_t*>(codes)[i] = (int32_t)code;
    }
  } catch (const std::exception& e) {  // a tensor without memory of its own (a wrapper of some transform)
    return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
  }
  Py_RETURN_NONE;
}

PyObject* same_shapes(PyObject*, PyObject* args) {
  PyObject *first, *second;
  Items a, b;
  if (!PyArg_ParseTuple(args, "OO", &first, &second) || !a.of(first) || !b.of(second)) return nullptr;
  try {
    for (Py_ssize_t i = 0; i < a.n; ++i) {
      if (i >= b.n || !THPVariable_Check(a.at[i]) || !THPVariable_Check(b.at[i]) ||
          THPVariable_Unpack(a.at[i]).sizes() != THPVariable_Unpack(b.at[i]).sizes())
        return PyLong_FromSsize_t(i);
    }
  } catch (const std::exception& e) {
    return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
  }
  return PyLong_FromSsize_t(a.n == b.n ? -1 : a.n);
}

PyObject* repeats(PyObject*, PyObject* args) {
  long long addresses, counts, n;
  if (!PyArg_ParseTuple(args, "LLL", &addresses, &counts, &n)) return nullptr;
  try {
    std::vector<int64_t> at;
    for (long long i = 0; i < n; ++i)
      if (!counts || reinterpret_cast<const int64_t*>(counts)[i]) at.push_back(reinterpret_cast<const int64_t*>(addresses)[i]);
    std::sort(at.begin(), at.end());
    return PyBool_FromLong(std::adjacent_find(at.begin(), at.end()) != at.end());
  } catch (const std::exception& e) {
    return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
  }
}

PyMethodDef methods[] = {{"read", read, METH_VARARGS, "addresses, counts and types of a list of tensors"},
                         {"same_shapes", same_shapes, METH_VARARGS, "first pair of unequal shapes"},
                         {"repeats", repeats, METH_VARARGS, "whether an address occurs twice"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_lists", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__lists() { return PyModule_Create(&module); }
