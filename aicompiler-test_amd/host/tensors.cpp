// The Python wrappers' checks of tensors, next to torch's own objects: what five
// methods a tensor would ask takes one call here, or one for a whole call of the library
// (the wrapper of tmc_tree_rope_append: 12 us with methods, 7 with a call a tensor, 3 so,
// beside the launch; most of the time of a kernel that ends sooner).
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

// call(function, device, arguments ...): the result of a function of the library that takes
// integers and pointers, 64 bits each, and returns an int.  A pointer's argument is a tensor
// or None and is followed by the dtype and the number of elements that it must have; where
// the tensor is not readable, nothing is called and the result is -1 for the first such
// argument, -2 for the second and so on.
constexpr int kMostWords = 24;
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n < 2) return wrong("call(function, device, ...)");
  void* function = PyLong_AsVoidPtr(args[0]);
  const long device = PyLong_AsLong(args[1]);
  if (PyErr_Occurred()) return nullptr;
  if (!function) return wrong("call(): no function");
  int64_t words[kMostWords] = {};
  int count = 0, pointers = 0;
  try {
    for (Py_ssize_t i = 2; i < n; ++count) {
      if (count == kMostWords) return wrong("call(): too many arguments");
      const bool tensor = THPVariable_Check(args[i]);
      if (!tensor && PyIndex_Check(args[i])) {
        words[count] = PyNumber_AsSsize_t(args[i++], PyExc_OverflowError);
        if (words[count] == -1 && PyErr_Occurred()) return nullptr;
        continue;
      }
      ++pointers;
      if (i + 2 >= n || !THPDtype_Check(args[i + 1]))
        return wrong("call(): a tensor, its dtype and its number of elements");
      const long long elements = PyLong_AsLongLong(args[i + 2]);
      if (PyErr_Occurred()) return nullptr;
      if (args[i] != Py_None) {
        if (!tensor) return wrong("call(): neither an integer nor a tensor");
        const at::Tensor& t = THPVariable_Unpack(args[i]);
        if (!readable(t, device, reinterpret_cast<THPDtype*>(args[i + 1])->scalar_type, elements))
          return PyLong_FromLong(-pointers);
        words[count] = reinterpret_cast<int64_t>(t.data_ptr());
      }
      i += 3;
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  // The x86-64 System V convention passes integers and pointers alike, an int in the low half
  // of its word, and the caller takes back words that the function does not look at.  That the
  // words are the function's own is the caller's to check (_check_words() of the wrappers,
  // against the declared types, which the tests compare with the header).
#if !defined(__x86_64__) || !defined(__linux__)
#error "call() relies on the x86-64 System V convention"
#endif
  using Function = int (*)(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                           int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                           int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t);
  const int64_t* w = words;
  int result;
  Py_BEGIN_ALLOW_THREADS
  result = reinterpret_cast<Function>(function)(
      w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7], w[8], w[9], w[10], w[11], w[12], w[13], w[14],
      w[15], w[16], w[17], w[18], w[19], w[20], w[21], w[22], w[23]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(result);
}

PyMethodDef methods[] = {
    {"address", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(address)),
     METH_FASTCALL, nullptr},
    {"addresses", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(addresses)),
     METH_FASTCALL, nullptr},
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call)), METH_FASTCALL,
     nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tmc_tensors", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tmc_tensors() { return PyModule_Create(&module); }
