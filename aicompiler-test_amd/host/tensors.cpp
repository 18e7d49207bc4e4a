// The Python wrappers' checks of tensors, next to torch's own objects: what five
// methods a tensor would ask takes one call here (1.2 to 0.4 us a tensor, and most of
// the time of a call that ends sooner than its arguments are checked).
#include <Python.h>

#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <exception>

namespace {

// Whether a kernel on `device` can read t as `count` adjacent elements of `type`.
bool readable(const at::Tensor& t, long device, at::ScalarType type, int64_t count) {
  return t.layout() == at::kStrided && t.get_device() == device &&
         t.scalar_type() == type && t.is_contiguous() && t.numel() >= count;
}

PyObject* wrong(const char* what) {
  PyErr_SetString(PyExc_TypeError, what);
  return nullptr;
}

// address(tensor, device, dtype, count): its address, or False where it is not readable.
PyObject* address(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4 || !THPVariable_Check(args[0]) || !THPDtype_Check(args[2]))
    return wrong("address(tensor, device, dtype, count)");
  const long device = PyLong_AsLong(args[1]);
  const long long count = PyLong_AsLongLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  try {
    const at::Tensor& t = THPVariable_Unpack(args[0]);
    if (!readable(t, device, reinterpret_cast<THPDtype*>(args[2])->scalar_type, count))
      Py_RETURN_FALSE;
    return PyLong_FromVoidPtr(t.data_ptr());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// addresses(list of tensors, device, dtype, buffer of 64-bit words): their addresses into
// the buffer; the least number of elements, or False where one is not readable.
PyObject* addresses(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4 || !PyList_Check(args[0]) || !THPDtype_Check(args[2]))
    return wrong("addresses(list, device, dtype, buffer)");
  const long device = PyLong_AsLong(args[1]);
  if (PyErr_Occurred()) return nullptr;
  Py_buffer words;
  if (PyObject_GetBuffer(args[3], &words, PyBUF_WRITABLE) != 0) return nullptr;
  const Py_ssize_t count = PyList_GET_SIZE(args[0]);
  PyObject* result = nullptr;
  if (words.len < count * (Py_ssize_t)sizeof(uint64_t)) {
    wrong("addresses(): the buffer is too small");
  } else {
    try {
      const at::ScalarType type = reinterpret_cast<THPDtype*>(args[2])->scalar_type;
      int64_t least = INT64_MAX;
      Py_ssize_t i = 0;
      for (; i < count; ++i) {
        PyObject* item = PyList_GET_ITEM(args[0], i);
        if (!THPVariable_Check(item)) break;
        const at::Tensor& t = THPVariable_Unpack(item);
        if (!readable(t, device, type, 0)) break;
        least = std::min(least, t.numel());
        static_cast<uint64_t*>(words.buf)[i] = reinterpret_cast<uint64_t>(t.data_ptr());
      }
      result = i < count ? PyBool_FromLong(0) : PyLong_FromLongLong(least);
    } catch (const std::exception& e) {
      PyErr_SetString(PyExc_RuntimeError, e.what());
    }
  }
  PyBuffer_Release(&words);
  return result;
}

PyMethodDef methods[] = {
    {"address", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(address)),
     METH_FASTCALL, nullptr},
    {"addresses", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(addresses)),
     METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tmc_tensors", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tmc_tensors() { return PyModule_Create(&module); }
