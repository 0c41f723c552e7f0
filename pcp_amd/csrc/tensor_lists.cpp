// Python lists of torch tensors as the host arrays that the C entry points take (pcp_amd._tensors).
//
// A model has hundreds of gradients, and asking each of them for its address, size, type, contiguity and device from
// Python costs about 0.4 us a tensor and list: 26 tensors in two lists took 20 us of a 32 us call. Here it is
// 8 ns a tensor. No GPU call is made.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <exception>

namespace {

// Element types in the order of pcp_dtype (include/pcp_grpo.h); -1 for others.
int32_t type_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return 0;
    case at::kBFloat16: return 1;
    case at::kFloat: return 2;
    case at::kDouble: return 3;
    case at::kInt: return 4;
    case at::kLong: return 5;
    case at::kBool:
    case at::kByte: return 6;
    default: return -1;
  }
}

// describe(tensors) -> (addresses, counts, types, contiguous, device): int64, int64, int32 and uint8 arrays as bytes, and
// the device index that all share (-1: the CPU, -2: several, -3: there is no tensor). An entry may be
// None: address 0, count -1, type -1, contiguous.
PyObject* describe(PyObject*, PyObject* arg) {
  PyObject* seq = PySequence_Fast(arg, "a list or tuple of tensors is wanted");
  if (!seq) return nullptr;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  PyObject* out[4] = {PyBytes_FromStringAndSize(nullptr, n * 8), PyBytes_FromStringAndSize(nullptr, n * 8),
                      PyBytes_FromStringAndSize(nullptr, n * 4), PyBytes_FromStringAndSize(nullptr, n)};
  bool fine = out[0] && out[1] && out[2] && out[3];
  int64_t device = -3;
  if (fine) {
    auto* at_ = reinterpret_cast<int64_t*>(PyBytes_AS_STRING(out[0]));
    auto* counts = reinterpret_cast<int64_t*>(PyBytes_AS_STRING(out[1]));
    auto* types = reinterpret_cast<int32_t*>(PyBytes_AS_STRING(out[2]));
    auto* contiguous = reinterpret_cast<uint8_t*>(PyBytes_AS_STRING(out[3]));
    try {
      for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* const o = PySequence_Fast_GET_ITEM(seq, i);
        if (o == Py_None) {
          at_[i] = 0;
          counts[i] = -1;
          types[i] = -1;
          contiguous[i] = 1;
          continue;
        }
        if (!THPVariable_Check(o)) {
          PyErr_Format(PyExc_TypeError, "entry %zd is no tensor", i);
          fine = false;
          break;
        }
        const at::Tensor& t = THPVariable_Unpack(o);
        at_[i] = reinterpret_cast<int64_t>(t.data_ptr());
        counts[i] = t.numel();
        types[i] = type_code(t.scalar_type());
        contiguous[i] = t.is_contiguous();
        const int64_t d = t.is_cuda() ? t.get_device() : -1;
        device = device == -3 || device == d ? d : -2;
      }
    } catch (const std::exception& e) {
      PyErr_SetString(PyExc_RuntimeError, e.what());
      fine = false;
    }
  }
  Py_DECREF(seq);
  PyObject* result = fine ? Py_BuildValue("OOOOL", out[0], out[1], out[2], out[3], static_cast<long long>(device)) : nullptr;
  for (PyObject* o : out) Py_XDECREF(o);
  return result;
}

// fit(tensors, sizes...) -> whether every tensor of a list (None among them) has those sizes.
PyObject* fit(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  constexpr Py_ssize_t kMost = 8;
  if (n_args < 1 || n_args - 1 > kMost) {
    PyErr_SetString(PyExc_TypeError, "fit(tensors, sizes...) of at most 8 dimensions");
    return nullptr;
  }
  int64_t sizes[kMost];
  for (Py_ssize_t i = 1; i < n_args; ++i) {
    sizes[i - 1] = PyLong_AsLongLong(args[i]);
    if (sizes[i - 1] == -1 && PyErr_Occurred()) return nullptr;
  }
  PyObject* seq = PySequence_Fast(args[0], "a list or tuple of tensors is wanted");
  if (!seq) return nullptr;
  bool fits = true, fine = true;
  try {
    for (Py_ssize_t i = 0; fits && i < PySequence_Fast_GET_SIZE(seq); ++i) {
      PyObject* const o = PySequence_Fast_GET_ITEM(seq, i);
      if (o == Py_None) continue;
      if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "entry %zd is no tensor", i);
        fine = false;
        break;
      }
      fits = THPVariable_Unpack(o).sizes() == at::IntArrayRef(sizes, n_args - 1);
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    fine = false;
  }
  Py_DECREF(seq);
  return fine ? PyBool_FromLong(fits) : nullptr;
}

PyMethodDef methods[] = {
    {"describe", describe, METH_O, "describe(tensors) -> (addresses, counts, types, contiguous, device)"},
    {"fit", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fit)), METH_FASTCALL, "fit(tensors, sizes...) -> bool"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", "Lists of tensors as host arrays.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&module); }
