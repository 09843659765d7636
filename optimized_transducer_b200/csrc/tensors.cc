// CPython helper of the Python layer: reads the pointers, sizes and types of a list of
// tensors in one call.  clip_grad_norm_ is handed hundreds of tensors per step, and asking
// each for its pointer, count, type, device and layout from Python takes about 0.3 us per
// tensor, several times what the kernels need (600 tensors, 90 million bfloat16 elements:
// 0.4 ms on the host, 0.1 ms on the device).  libot_b200.so itself knows nothing of torch.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <vector>

#include "../../include/ot_b200.h"

namespace {

// Element type as the library's flags say it; -1 for a type it does not take.
int type_flag(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return 0;
    case at::kDouble: return OT_B200_FP64;
    case at::kBFloat16: return OT_B200_BF16;
    case at::kHalf: return OT_B200_FP16;
    default: return -1;
  }
}

template <typename T> PyObject *as_bytes(const std::vector<T> &v) {
  return PyBytes_FromStringAndSize(reinterpret_cast<const char *>(v.data()), (Py_ssize_t)(v.size() * sizeof(T)));
}

// describe(list) -> (pointers, counts, type flags, device, index, why): three bytes objects
// with one 64-, 64- and 32-bit entry per tensor, and the CUDA device all are on; or, at the
// first tensor that will not do, None four times, its index and "tensor" / "layout" /
// "type" / "cpu" / "device".  "Dense" means one stretch of memory, each element once.
PyObject *describe(PyObject *, PyObject *list) {
  PyObject *seq = PySequence_Fast(list, "expected a sequence of tensors");
  if (seq == nullptr) return nullptr;
  PyObject *result = nullptr;
  try {
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    PyObject **items = PySequence_Fast_ITEMS(seq);
    std::vector<int64_t> pointers((size_t)n), counts((size_t)n);
    std::vector<int32_t> types((size_t)n);
    int device = -1;
    const char *why = nullptr;
    Py_ssize_t i = 0;
    for (; i < n; ++i) {
      if (!THPVariable_Check(items[i])) { why = "tensor"; break; }
      const at::Tensor &t = THPVariable_Unpack(items[i]);
      if (t.layout() != at::kStrided) { why = "layout"; break; }
      if (!t.is_cuda()) { why = "cpu"; break; }
      if (i == 0) device = (int)t.get_device();
      if ((int)t.get_device() != device) { why = "device"; break; }
      const int flag = type_flag(t.scalar_type());
      if (flag < 0) { why = "type"; break; }
      if (!t.is_contiguous() && !t.is_non_overlapping_and_dense()) { why = "layout"; break; }
      pointers[(size_t)i] = (int64_t)reinterpret_cast<uintptr_t>(t.numel() > 0 ? t.data_ptr() : nullptr);
      counts[(size_t)i] = t.numel();
      types[(size_t)i] = flag;
    }
    if (why != nullptr)
      result = Py_BuildValue("(OOOOns)", Py_None, Py_None, Py_None, Py_None, i, why);
    else
      result = Py_BuildValue("(NNNins)", as_bytes(pointers), as_bytes(counts), as_bytes(types), device, n, "");
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  Py_DECREF(seq);
  return result;
}

// alike(a, b): the index of the first pair of tensors whose shapes differ, or whose strides
// do where one of the two is not contiguous; -1 when there is none.
PyObject *alike(PyObject *, PyObject *args) {
  PyObject *a = nullptr, *b = nullptr;
  if (!PyArg_ParseTuple(args, "O!O!", &PyList_Type, &a, &PyList_Type, &b)) return nullptr;
  try {
    const Py_ssize_t n = PyList_GET_SIZE(a) < PyList_GET_SIZE(b) ? PyList_GET_SIZE(a) : PyList_GET_SIZE(b);
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject *x = PyList_GET_ITEM(a, i), *y = PyList_GET_ITEM(b, i);
      if (!THPVariable_Check(x) || !THPVariable_Check(y)) return PyLong_FromSsize_t(i);
      const at::Tensor &s = THPVariable_Unpack(x), &t = THPVariable_Unpack(y);
      if (s.layout() != at::kStrided || t.layout() != at::kStrided || s.sizes() != t.sizes() ||
          (s.strides() != t.strides() && !(s.is_contiguous() && t.is_contiguous())))
        return PyLong_FromSsize_t(i);
    }
    return PyLong_FromLong(-1);
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// written(list): the tensors' version counters move on, as after any write that autograd
// has to know of (inference tensors have none).
PyObject *written(PyObject *, PyObject *list) {
  PyObject *seq = PySequence_Fast(list, "expected a sequence of tensors");
  if (seq == nullptr) return nullptr;
  try {
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq); ++i) {
      const at::Tensor &t = THPVariable_Unpack(PySequence_Fast_GET_ITEM(seq, i));
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  Py_DECREF(seq);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"describe", describe, METH_O, "pointers, counts and types of a list of tensors"},
                         {"alike", alike, METH_VARARGS, "whether two lists of tensors have the same shapes"},
                         {"written", written, METH_O, "moves the tensors' version counters on"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) { return PyModule_Create(&module); }
