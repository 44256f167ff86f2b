// Host side of the many-tensor operators: reads the addresses of a parameter list and of its gradients straight from the tensors.
//
// A Python loop over `p.data_ptr(), p.grad, p.grad.data_ptr()` and the checks costs ~0.6 us per tensor; for the 144 tensors of the smallest
// network that is several times the kernel's own run time.
#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>
#include <Python.h>
#include <cstdint>
#include <exception>

namespace {

struct Expected {            // the host copy of one record of the optimizer's tensor table
  int64_t n, off;
  int32_t group, dt;
};

int code_of(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1; }

// same element order in memory: equal strides wherever a dimension has more than one element
bool same_order(const at::Tensor& a, const at::Tensor& b) {
  const auto sa = a.strides(), sb = b.strides(), n = a.sizes();
  for (size_t i = 0; i < n.size(); ++i)
    if (n[i] != 1 && sa[i] != sb[i]) return false;
  return true;
}

// gather(params, expected, device, out) -> (tensors with a gradient, None or [indices whose gradient lies in another element order])
// expected: address of Expected[len(params)]; out: address of {parameter, gradient} pairs, gradient 0 where there is none.
PyObject* gather(PyObject*, PyObject* args) {
  PyObject* list;
  unsigned long long expected_at, out_at;
  int device;
  if (!PyArg_ParseTuple(args, "O!KiK", &PyList_Type, &list, &expected_at, &device, &out_at)) return nullptr;
  const Expected* want = reinterpret_cast<const Expected*>(expected_at);
  uint64_t* out = reinterpret_cast<uint64_t*>(out_at);
  PyObject* other = nullptr;
  try {
    const Py_ssize_t count = PyList_GET_SIZE(list);
    Py_ssize_t grads = 0;
    for (Py_ssize_t i = 0; i < count; ++i) {
      PyObject* o = PyList_GET_ITEM(list, i);
      const char* wrong = nullptr;
      if (!THPVariable_Check(o)) wrong = "is not a tensor";
      else {
        const at::Tensor& p = THPVariable_Unpack(o);
        if (p.layout() != at::kStrided || !p.device().is_cuda() || p.device().index() != device) wrong = "has left the optimizer's device";
        else if (p.numel() != want[i].n || code_of(p.scalar_type()) != want[i].dt) wrong = "has another size or type than when the optimizer first ran";
        else if (!p.is_non_overlapping_and_dense()) wrong = "is not dense in memory";
        else {
          const at::Tensor& g = p.grad();
          out[2 * i] = reinterpret_cast<uint64_t>(p.data_ptr());
          out[2 * i + 1] = 0;
          if (g.defined()) {
            if (g.layout() != at::kStrided) wrong = "has a sparse gradient";
            else if (g.device() != p.device() || g.scalar_type() != p.scalar_type() || g.sizes() != p.sizes()) wrong = "has a gradient of another device, type or shape";
            else {
              ++grads;
              p.unsafeGetTensorImpl()->bump_version();      // the kernel writes it behind autograd's back: a stale saved tensor has to be noticed
              if (same_order(p, g)) out[2 * i + 1] = reinterpret_cast<uint64_t>(g.data_ptr());
              else {
                if (!other && !(other = PyList_New(0))) return nullptr;
                PyObject* k = PyLong_FromSsize_t(i);
                const int err = k ? PyList_Append(other, k) : -1;
                Py_XDECREF(k);
                if (err) { Py_DECREF(other); return nullptr; }
              }
            }
          }
        }
      }
      if (wrong) {
        Py_XDECREF(other);
        return PyErr_Format(PyExc_ValueError, "parameter %zd %s", i, wrong);
      }
    }
    return other ? Py_BuildValue("nN", grads, other) : Py_BuildValue("nO", grads, Py_None);
  } catch (const std::exception& e) {
    Py_XDECREF(other);
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {{"gather", gather, METH_VARARGS, "addresses of parameters and gradients"}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_tensors", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host_tensors() { return PyModule_Create(&module); }
