// What Python would be too slow for.  Addresses of many parameters and their gradients in one call
// (hi2_amd/optim.py): a few nanoseconds a tensor, where attributes read from Python take a tenth of a
// microsecond each.  And the gated activation's place in the autograd graph (hi2_amd/experts.py): a
// backward written in Python hands the interpreter's lock from thread to thread and back, which took
// 41 of the 90 us of a small forward and backward (torch's product of two tensors: 49).
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/hi2x.h"

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

// stepped(params, grads): autograd's version counters of the parameters whose gradients' addresses in
// `grads` (of uint64 elements, one a parameter) are not 0 count the write that a step was to them.
PyObject* stepped(PyObject*, PyObject* args) {
  PyObject* params;
  unsigned long long grads;
  if (!PyArg_ParseTuple(args, "O!K", &PyList_Type, &params, &grads)) return nullptr;
  const uint64_t* g = reinterpret_cast<const uint64_t*>(grads);
  HANDLE_TH_ERRORS
  const Py_ssize_t count = PyList_GET_SIZE(params);
  for (Py_ssize_t i = 0; i < count; ++i) {
    PyObject* o = PyList_GET_ITEM(params, i);
    if (!THPVariable_Check(o)) {
      PyErr_Format(PyExc_RuntimeError, "AdamW: not a tensor (parameter %zd)", i);
      return nullptr;
    }
    const at::Tensor& p = THPVariable_Unpack(o);
    if (g[i] && !p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// The entries of libhi2x.so, by address (the library is loaded by Python, once).
decltype(&hi2x_gated) gated_entry;
decltype(&hi2x_gated_backward) gated_backward_entry;
decltype(&hi2x_last_error) last_error_entry;

PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long f, b, e;
  if (!PyArg_ParseTuple(args, "KKK", &f, &b, &e)) return nullptr;
  gated_entry = reinterpret_cast<decltype(gated_entry)>(f);
  gated_backward_entry = reinterpret_cast<decltype(gated_backward_entry)>(b);
  last_error_entry = reinterpret_cast<decltype(last_error_entry)>(e);
  Py_RETURN_NONE;
}

int type_of(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kHalf ? 1 : 2;
}
int64_t pitch(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
void* stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}
// Rows as the kernels take them.
at::Tensor rows_of(const at::Tensor& t) {
  return (t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1))
             ? t.contiguous()
             : t;
}
void check(int rc) {
  if (rc != HI2X_OK) throw std::runtime_error(last_error_entry());
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Gated : torch::autograd::Function<Gated> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& gate, const at::Tensor& up,
                            int64_t act) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({gate, up});
    ctx->saved_data["act"] = act;
    const c10::DeviceGuard guard(gate.device());
    at::Tensor out = at::empty({gate.size(0), gate.size(1)}, gate.options());
    if (out.numel())
      check(gated_entry(gate.data_ptr(), pitch(gate), up.data_ptr(), pitch(up), gate.size(0),
                        gate.size(1), type_of(gate), (int)act, out.data_ptr(), gate.size(1),
                        stream_of(gate)));
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor()};
    variable_list both(2);
    {
      const at::AutoGradMode off(false);
      const variable_list saved = ctx->get_saved_variables();
      // (saved tensors' hooks may give them back in other strides than they were saved with)
      const at::Tensor gate = rows_of(saved[0]), up = rows_of(saved[1]), grad = rows_of(grads[0]);
      const c10::DeviceGuard guard(gate.device());
      for (at::Tensor& d : both) d = at::empty({gate.size(0), gate.size(1)}, gate.options());
      if (both[0].numel())
        check(gated_backward_entry(grad.data_ptr(), pitch(grad), gate.data_ptr(), pitch(gate),
                                   up.data_ptr(), pitch(up), gate.size(0), gate.size(1),
                                   type_of(gate), (int)ctx->saved_data["act"].toInt(),
                                   both[0].data_ptr(), gate.size(1), both[1].data_ptr(),
                                   gate.size(1), stream_of(gate)));
    }
    if (at::GradMode::is_enabled()) {  // once: a second derivative is refused where it is asked for
      for (at::Tensor& d : both) d.set_requires_grad(true);
      both = (*std::make_shared<torch::autograd::DelayedError>(
          "gated: trying to differentiate twice a function that is differentiable once", 2))(
          std::move(both));
    }
    return {both[0], both[1], at::Tensor()};
  }
};

// gated(gate, up, act) -> act(gate) * up, of two matrices that the kernels take as they lie
PyObject* gated(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *gate, *up;
  int act;
  if (!PyArg_ParseTuple(args, "OOi", &gate, &up, &act)) return nullptr;
  if (!THPVariable_Check(gate) || !THPVariable_Check(up)) {
    PyErr_SetString(PyExc_TypeError, "gated: not a tensor");
    return nullptr;
  }
  if (!gated_entry) {
    PyErr_SetString(PyExc_RuntimeError, "gated: bind() first");
    return nullptr;
  }
  const at::Tensor g = THPVariable_Unpack(gate), u = THPVariable_Unpack(up);
  at::Tensor out;
  {
    const pybind11::gil_scoped_release unlocked;
    out = Gated::apply(g, u, (int64_t)act);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"addresses", addresses, METH_VARARGS, "Tensors' addresses."},
                         {"stepped", stepped, METH_VARARGS, "Count a step's writes."},
                         {"bind", bind, METH_VARARGS, "The library's entries."},
                         {"gated", gated, METH_VARARGS, "The gated activation, differentiable."},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) { return PyModule_Create(&module); }
