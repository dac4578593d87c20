// Addresses of many parameters and their gradients in one call from Python (hi2_amd/optim.py): a few
// nanoseconds a tensor, where attributes read from Python take a tenth of a microsecond each.
#include <torch/csrc/autograd/python_variable.h>

namespace {

// addresses(params, sizes, dtype, device, out_params, out_grads) -> indices of the gradients that
// are not contiguous.  sizes: address of int64 elements, one a parameter; dtype: 0 float32, 1
// float16, 2 bfloat16; out_params, out_grads: addresses of uint64 arrays to fill (a parameter
// without a gradient gets 0).  Raises RuntimeError where a tensor is not what it was.
PyObject* addresses(PyObject*, PyObject* args) {
  PyObject* params;
  unsigned long long sizes, out_params, out_grads;
  int dtype, device;
  if (!PyArg_ParseTuple(args, "O!KiiKK", &PyList_Type, &params, &sizes, &dtype, &device,
                        &out_params, &out_grads))
    return nullptr;
  static const at::ScalarType types[3] = {at::kFloat, at::kHalf, at::kBFloat16};
  if (dtype < 0 || dtype > 2) {
    PyErr_Format(PyExc_ValueError, "dtype %d", dtype);
    return nullptr;
  }
  const int64_t* n = reinterpret_cast<const int64_t*>(sizes);
  uint64_t* to_p = reinterpret_cast<uint64_t*>(out_params);
  uint64_t* to_g = reinterpret_cast<uint64_t*>(out_grads);
  PyObject* odd = PyList_New(0);
  if (!odd) return nullptr;
  auto fail = [&](const char* why, Py_ssize_t i) -> PyObject* {
    Py_DECREF(odd);
    PyErr_Format(PyExc_RuntimeError, "AdamW: %s (parameter %zd)", why, i);
    return nullptr;
  };
  try {
    const Py_ssize_t count = PyList_GET_SIZE(params);
    for (Py_ssize_t i = 0; i < count; ++i) {
      PyObject* o = PyList_GET_ITEM(params, i);
      if (!THPVariable_Check(o)) return fail("not a tensor", i);
      const at::Tensor& p = THPVariable_Unpack(o);
      auto same = [&](const at::Tensor& t) {
        return t.layout() == at::kStrided && t.scalar_type() == types[dtype] &&
               t.numel() == n[i] && t.is_cuda() && t.get_device() == device;
      };
      if (!same(p)) return fail("a parameter's type, size or device changed after construction", i);
      if (!p.is_contiguous()) return fail("a parameter is no longer contiguous", i);
      to_p[i] = reinterpret_cast<uint64_t>(p.data_ptr());
      const at::Tensor& g = p.grad();
      to_g[i] = 0;
      if (!g.defined()) continue;
      if (!same(g)) return fail("a gradient is sparse or has not its parameter's type and size", i);
      if (g.is_contiguous()) {
        to_g[i] = reinterpret_cast<uint64_t>(g.data_ptr());
      } else {
        PyObject* at = PyLong_FromSsize_t(i);
        const int rc = at ? PyList_Append(odd, at) : -1;
        Py_XDECREF(at);
        if (rc) {
          Py_DECREF(odd);
          return nullptr;
        }
      }
    }
  } catch (const std::exception& e) {
    Py_DECREF(odd);
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  return odd;
}

PyMethodDef methods[] = {{"addresses", addresses, METH_VARARGS, "Tensors' addresses."},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) { return PyModule_Create(&module); }
