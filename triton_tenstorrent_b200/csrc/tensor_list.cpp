// The per-tensor host work of an optimiser step, in one walk over the lists of Python tensors.  A query from Python costs 50 to 100 ns and a step asks ten of them
// for each parameter and its gradient (145 pairs: 107 us for a kernel of 6 us), here a few ns.
//
// Compiled against torch's headers into an extension module of its own next to the C-ABI library, which knows nothing of torch.
#include <torch/csrc/autograd/python_variable.h>

#include <exception>

#include "b200k.h"

namespace {

bool usable(const at::Tensor& t, c10::ScalarType type, c10::DeviceIndex device, const int64_t* dims, int64_t ndim) {
  if (!t.defined() || t.scalar_type() != type || t.layout() != c10::kStrided || !t.is_cuda() || t.get_device() != device || t.dim() != ndim) return false;
  const auto sizes = t.sizes();
  for (int64_t k = 0; k < ndim; ++k)
    if (sizes[k] != dims[k]) return false;
  return t.is_contiguous();
}

// fill_rows(params, grads, count, shapes, table, columns, device, type) -> -1, or whether the gradients are fp32
//
// params   list of `count` tensors; grads: list of as many, or None for the parameters' .grad
// shapes   address of int64s: for each of the `count` tensors its number of dimensions and they
// table    address of int64 [count][columns]: column 0 takes a parameter's address, column 1 its gradient's
// type     of all parameters, as a B200K_DTYPE_*; the gradients are all of this type or all fp32
//
// -1: something is not the usual case (every gradient there, strided, contiguous, on `device`, of the expected shape and type); nothing may be
// concluded from the table then, and the caller goes through the list with its own checks and messages.
PyObject* fill_rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 8) {
    PyErr_SetString(PyExc_TypeError, "fill_rows: 8 arguments expected");
    return nullptr;
  }
  PyObject *params = args[0], *grads = args[1];
  const Py_ssize_t n = PyLong_AsSsize_t(args[2]);
  const auto* shape = static_cast<const int64_t*>(PyLong_AsVoidPtr(args[3]));
  auto* table = static_cast<int64_t*>(PyLong_AsVoidPtr(args[4]));
  const int64_t columns = PyLong_AsLongLong(args[5]);
  const auto device = static_cast<c10::DeviceIndex>(PyLong_AsLong(args[6]));
  const long code = PyLong_AsLong(args[7]);
  if (PyErr_Occurred()) return nullptr;
  if (code < B200K_DTYPE_F32 || code > B200K_DTYPE_F16) return PyLong_FromLong(-1);
  const auto type = code == B200K_DTYPE_F32 ? c10::kFloat : code == B200K_DTYPE_BF16 ? c10::kBFloat16 : c10::kHalf;
  if (!PyList_CheckExact(params) || (grads != Py_None && !PyList_CheckExact(grads))) return PyLong_FromLong(-1);
  if (n < 1 || PyList_GET_SIZE(params) != n || (grads != Py_None && PyList_GET_SIZE(grads) != n)) return PyLong_FromLong(-1);
  try {
    c10::ScalarType gtype = type;
    for (Py_ssize_t i = 0; i < n; ++i) {
      const int64_t ndim = *shape++;
      PyObject* item = PyList_GET_ITEM(params, i);
      if (!THPVariable_Check(item)) return PyLong_FromLong(-1);
      const at::Tensor& p = THPVariable_Unpack(item);
      at::Tensor g;
      if (grads == Py_None) {
        g = p.grad();
      } else {
        PyObject* other = PyList_GET_ITEM(grads, i);
        if (!THPVariable_Check(other)) return PyLong_FromLong(-1);
        g = THPVariable_Unpack(other);
      }
      if (i == 0 && g.defined() && g.scalar_type() == c10::kFloat) gtype = c10::kFloat;
      if (!usable(p, type, device, shape, ndim) || !usable(g, gtype, device, shape, ndim)) return PyLong_FromLong(-1);
      table[i * columns] = reinterpret_cast<int64_t>(p.data_ptr());
      table[i * columns + 1] = reinterpret_cast<int64_t>(g.data_ptr());
      shape += ndim;
    }
    return PyLong_FromLong(gtype == c10::kFloat ? 1 : 0);
  } catch (const std::exception&) {      // a tensor without memory of its own, say
    return PyLong_FromLong(-1);
  } catch (...) {
    return PyLong_FromLong(-1);
  }
}

PyMethodDef methods[] = {{"fill_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fill_rows)), METH_FASTCALL, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_list", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_list() { return PyModule_Create(&module); }
