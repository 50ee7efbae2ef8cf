// Descriptors of a call's tensors, read where they are: pack() of
// nanovllm_amd/_lib.py asks every tensor for six attributes through Python, 0.47 us
// a tensor and half of a small call's host time; this takes the same fields from
// the tensors themselves (13 tensors: 0.3 us and not 6.5).
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>

#include "nvdsa.h"

namespace {

int32_t dtype_code(at::ScalarType type) {
  switch (type) {
    case at::kInt:
      return NVDSA_INT32;
    case at::kHalf:
      return NVDSA_FLOAT16;
    case at::kBFloat16:
      return NVDSA_BFLOAT16;
    case at::kFloat:
      return NVDSA_FLOAT32;
    case at::kFloat8_e4m3fn:
      return NVDSA_FLOAT8_E4M3;
    default:
      return -1;
  }
}

// (buffer, addresses) as pack() returns them; None where an argument is neither a
// tensor with memory nor None: pack() then goes on by itself.
PyObject* pack(PyObject*, PyObject* const* args, Py_ssize_t count) {
  PyObject* buffer = PyBytes_FromStringAndSize(nullptr, count * static_cast<Py_ssize_t>(sizeof(nvdsa_tensor)));
  PyObject* places = buffer ? PyList_New(count) : nullptr;
  if (places == nullptr) {
    Py_XDECREF(buffer);
    return nullptr;
  }
  char* const base = PyBytes_AS_STRING(buffer);
  bool known = true;
  try {
    for (Py_ssize_t i = 0; i < count && known; ++i) {
      char* const place = base + i * sizeof(nvdsa_tensor);
      nvdsa_tensor item;
      std::memset(&item, 0, sizeof(item));
      PyObject* at = Py_None;
      if (args[i] != Py_None) {
        if (!THPVariable_Check(args[i])) {
          known = false;
          break;
        }
        const at::Tensor& t = THPVariable_Unpack(args[i]);
        if (!t.defined() || !(t.is_cuda() || t.is_cpu())) {
          known = false;
          break;
        }
        const auto sizes = t.sizes();
        item.data = t.data_ptr();
        item.dtype = dtype_code(t.scalar_type());
        item.ndim = sizes.size() <= 4 ? static_cast<int32_t>(sizes.size()) : 5;
        for (size_t d = 0; d < sizes.size() && d < 4; ++d) item.shape[d] = sizes[d];
        item.contiguous = t.is_contiguous() ? 1 : 0;
        item.device = t.is_cuda() ? static_cast<int32_t>(t.get_device()) : (t.is_pinned() ? NVDSA_HOST_MAPPED_DEVICE : -2);
        at = PyLong_FromVoidPtr(place);
      } else {
        Py_INCREF(at);
      }
      if (at == nullptr) {
        Py_DECREF(places);
        Py_DECREF(buffer);
        return nullptr;
      }
      std::memcpy(place, &item, sizeof(item));
      PyList_SET_ITEM(places, i, at);
    }
  } catch (...) {
    PyErr_Clear();   // (a subclass whose sizes are Python's leaves its error set)
    known = false;   // (no memory of its own, symbolic sizes: pack() says so)
  }
  if (!known) {
    Py_DECREF(places);
    Py_DECREF(buffer);
    Py_RETURN_NONE;
  }
  PyObject* both = PyTuple_Pack(2, buffer, places);
  Py_DECREF(places);
  Py_DECREF(buffer);
  return both;
}

PyMethodDef methods[] = {
    {"pack", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(pack)), METH_FASTCALL, "Descriptors of device tensors."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_pack", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// (torch_version: of the headers that `pack` was compiled against; the tensors' fields
// lie where they say, so that the module is of use with that version alone.)
PyMODINIT_FUNC PyInit__tensor_pack() {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", NVDSA_TORCH_VERSION) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
