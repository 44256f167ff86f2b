// Host side of the many-tensor operators and of the int8 layer.
//
// The former read the addresses of a parameter list and of its gradients straight from the tensors: a Python loop over `p.data_ptr(), p.grad, p.grad.data_ptr()` and the checks costs ~0.6 us per tensor; for the 144 tensors of the smallest
// network that is several times the kernel's own run time.
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/library.h>
#include <Python.h>
#include <cstdint>
#include <exception>
#include <optional>
#include <tuple>
#include <vector>
#include "../../include/mpmae_hip.h"

namespace {

int code_of(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1; }

// same element order in memory: equal strides wherever a dimension has more than one element, and the memory holds the values themselves (no negated view)
bool same_order(const at::Tensor& a, const at::Tensor& b) {
  if (b.is_neg()) return false;
  const auto sa = a.strides(), sb = b.strides(), n = a.sizes();
  for (size_t i = 0; i < n.size(); ++i)
    if (n[i] != 1 && sa[i] != sb[i]) return false;
  return true;
}

// what decides the order of a dense tensor's elements in memory
uint64_t order_of(const at::Tensor& t) {
  uint64_t h = 1469598103934665603ull;
  const auto n = t.sizes(), s = t.strides();
  for (size_t i = 0; i < n.size(); ++i)
    if (n[i] != 1) h = ((h ^ (uint64_t)n[i]) * 1099511628211ull ^ (uint64_t)s[i]) * 1099511628211ull;
  return h | 1;
}

// gather(params, table, device, out, orders, update) -> (tensors with a gradient, whether a parameter has moved, None or [indices whose gradient lies in another element order])
// table: address of the host copy of MpmaeAdamwTensor[len(params)], whose parameter addresses are brought up to date; device: index of the GPU, -1 for host
// memory; out: address of the gradients' addresses, 0 where there is none; orders: address of one word per parameter, 0 before the first call, that holds it to
// its element order (its moments lie in the same); update: the parameters with a gradient are about to be written.
// The whole list is looked over first: a refusal leaves the table, the orders and the parameters' versions as they were, so that the call after it still sees what
// has moved.
PyObject* gather(PyObject*, PyObject* args) {
  PyObject* list;
  unsigned long long expected_at, out_at, orders_at;
  int device, update;
  if (!PyArg_ParseTuple(args, "O!KiKKp", &PyList_Type, &list, &expected_at, &device, &out_at, &orders_at, &update)) return nullptr;
  MpmaeAdamwTensor* want = reinterpret_cast<MpmaeAdamwTensor*>(expected_at);
  uint64_t* out = reinterpret_cast<uint64_t*>(out_at);
  uint64_t* orders = reinterpret_cast<uint64_t*>(orders_at);
  PyObject* other = nullptr;
  try {
    const Py_ssize_t count = PyList_GET_SIZE(list);
    const c10::Device home(device >= 0 ? c10::DeviceType::CUDA : c10::DeviceType::CPU, (c10::DeviceIndex)device);
    struct Seen { c10::TensorImpl* p; void *at, *grad; uint64_t order; };
    static thread_local std::vector<Seen> seen;
    seen.assign(count, Seen{});
    Py_ssize_t grads = 0;
    for (Py_ssize_t i = 0; i < count; ++i) {
      PyObject* o = PyList_GET_ITEM(list, i);
      const char* wrong = nullptr;
      if (!THPVariable_Check(o)) wrong = "is not a tensor";
      else {
        const at::Tensor& p = THPVariable_Unpack(o);
        Seen& s = seen[i];
        if (p.layout() != at::kStrided || p.device() != home) wrong = "has left the optimizer's device";
        else if (p.numel() != want[i].n || code_of(p.scalar_type()) != want[i].dt) wrong = "has another size or type than when the optimizer first ran";
        else if (!p.is_non_overlapping_and_dense() || p.is_neg()) wrong = "is not dense in memory";
        else if (p.is_inference()) wrong = "was made in inference mode: it has no version to count";
        else if (s.order = order_of(p); orders[i] && orders[i] != s.order) wrong = "has its elements in another order than when the optimizer first ran";
        else {
          s.at = p.data_ptr();      // (throws where there is no memory behind it)
          if (const at::Tensor& g = p.grad(); g.defined()) {
            if (g.layout() != at::kStrided) wrong = "has a sparse gradient";
            else if (g.device() != home || g.scalar_type() != p.scalar_type() || g.sizes() != p.sizes()) wrong = "has a gradient of another device, type or shape";
            else {
              ++grads;
              s.p = p.unsafeGetTensorImpl();
              void* const at = g.data_ptr();
              if (same_order(p, g)) s.grad = at;
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
    // nothing fails from here on
    bool moved = false;
    for (Py_ssize_t i = 0; i < count; ++i) {
      const Seen& s = seen[i];
      moved |= want[i].p != s.at;
      want[i].p = s.at;
      orders[i] = s.order;
      out[i] = reinterpret_cast<uint64_t>(s.grad);
      if (update && s.p) s.p->bump_version();      // the kernel writes it behind autograd's back: a stale saved tensor has to be noticed
    }
    PyObject* const flag = moved ? Py_True : Py_False;
    return other ? Py_BuildValue("nON", grads, flag, other) : Py_BuildValue("nOO", grads, flag, Py_None);
  } catch (const std::exception& e) {
    Py_XDECREF(other);
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// same_lists(param_groups, params, counts) -> whether the groups' lists, one after the other, hold these very parameters, counts[g] of them in group g
PyObject* same_lists(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 3 || !PyList_Check(args[0]) || !PyList_Check(args[1]) || !PyList_Check(args[2]))
    return PyErr_Format(PyExc_TypeError, "same_lists(param_groups, params, counts): three lists");
  const Py_ssize_t ngroups = PyList_GET_SIZE(args[0]), total = PyList_GET_SIZE(args[1]);
  if (ngroups != PyList_GET_SIZE(args[2])) Py_RETURN_FALSE;
  Py_ssize_t at = 0;
  for (Py_ssize_t g = 0; g < ngroups; ++g) {
    PyObject* const group = PyList_GET_ITEM(args[0], g);
    PyObject* const list = PyDict_Check(group) ? PyDict_GetItemString(group, "params") : nullptr;      // (borrowed)
    if (!list || !PyList_Check(list)) Py_RETURN_FALSE;
    const Py_ssize_t n = PyList_GET_SIZE(list);
    const long want = PyLong_AsLong(PyList_GET_ITEM(args[2], g));
    if (want == -1 && PyErr_Occurred()) return nullptr;
    if (n != want || at + n > total) Py_RETURN_FALSE;
    for (Py_ssize_t i = 0; i < n; ++i)
      if (PyList_GET_ITEM(list, i) != PyList_GET_ITEM(args[1], at + i)) Py_RETURN_FALSE;
    at += n;
  }
  return PyBool_FromLong(at == total);
}

using AdamwEntry = int (*)(const MpmaeAdamwArgs*, const void* const*, const double*, int, mpmae_stream_t);
AdamwEntry adamw_entry = nullptr;          // of libmpmae_hip.so, from bind()

// adamw(address of MpmaeAdamwArgs, address of the gradients' addresses, param_groups, device) -> 2 * hipError + whether the stream is being captured. The settings of
// the groups, the stream and the launches of a step: through ctypes they take as long again as the launches.
PyObject* adamw(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 4 || !PyList_Check(args[2])) return PyErr_Format(PyExc_TypeError, "adamw(args, grads, param_groups, device)");
  const auto* const a = static_cast<const MpmaeAdamwArgs*>(PyLong_AsVoidPtr(args[0]));
  const auto* const grads = static_cast<const void* const*>(PyLong_AsVoidPtr(args[1]));
  const long device = PyLong_AsLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  static PyObject* const keys[4] = {PyUnicode_InternFromString("lr"), PyUnicode_InternFromString("betas"), PyUnicode_InternFromString("eps"),
                                    PyUnicode_InternFromString("weight_decay")};
  const Py_ssize_t ngroups = PyList_GET_SIZE(args[2]);
  std::vector<double> groups(5 * ngroups);
  for (Py_ssize_t g = 0; g < ngroups; ++g) {
    PyObject* const group = PyList_GET_ITEM(args[2], g);
    double* out = groups.data() + 5 * g;
    const auto number = [&](PyObject* x) { *out = PyFloat_AsDouble(x); return *out++ != -1.0 || !PyErr_Occurred(); };
    for (int i = 0; i < 4; ++i) {
      PyObject* const x = PyDict_Check(group) ? PyDict_GetItemWithError(group, keys[i]) : nullptr;      // (borrowed)
      if (!x) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_KeyError, "a parameter group has no %U", keys[i]);
      if (i == 0 && THPVariable_Check(x)) return PyErr_Format(PyExc_ValueError, "lr is a number: a tensor would have to be read back on every step");
      if (i != 1) {
        if (!number(x)) return nullptr;
        continue;
      }
      const THPObjectPtr two(PySequence_Fast(x, "betas are two numbers"));
      if (!two) return nullptr;
      if (PySequence_Fast_GET_SIZE(two.get()) != 2) return PyErr_Format(PyExc_ValueError, "betas are two numbers: %R", x);
      for (int j = 0; j < 2; ++j) if (!number(PySequence_Fast_GET_ITEM(two.get(), j))) return nullptr;
    }
  }
  TORCH_CHECK(adamw_entry, "the kernels are not loaded");
  c10::OptionalDeviceGuard guard(c10::Device(c10::DeviceType::CUDA, (c10::DeviceIndex)device));
  const hipStream_t stream = c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream();
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &status) != hipSuccess) (void)hipGetLastError();
  const int err = adamw_entry(a, grads, groups.data(), (int)ngroups, stream);
  return PyLong_FromLong(2l * err + (status != hipStreamCaptureStatusNone));
  END_HANDLE_TH_ERRORS
}

// ---- the int8 linear layer and its quantiser, as operators of torch's dispatcher (mpmae::linear_int8, mpmae::quantize_int8): a trace, a dispatch mode or a
// functional transform sees the call. What they allocate is filled by this library, behind the dispatcher's back, so nothing above may take it for the result.
using LinearEntry = int (*)(int, const MpmaeI8Args*, mpmae_stream_t);
using PartBytes = long long (*)(int, int, int);
using QuantEntry = int (*)(int, const void*, long long, int, int, int8_t*, int, float*, mpmae_stream_t);
LinearEntry linear_entry = nullptr;          // of libmpmae_hip.so, from bind()
PartBytes part_bytes = nullptr;
QuantEntry quant_entry = nullptr;

PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long linear, part, quant, adamw;
  if (!PyArg_ParseTuple(args, "KKKK", &linear, &part, &quant, &adamw)) return nullptr;
  adamw_entry = reinterpret_cast<AdamwEntry>(adamw);
  linear_entry = reinterpret_cast<LinearEntry>(linear);
  part_bytes = reinterpret_cast<PartBytes>(part);
  quant_entry = reinterpret_cast<QuantEntry>(quant);
  Py_RETURN_NONE;
}

// rows of k elements that lie next to each other
at::Tensor rows_of(const at::Tensor& x, int64_t k) {
  if (x.dim() == 2 && (x.stride(1) == 1 || k == 1)) return x;
  const at::Tensor r = x.reshape({-1, k});
  return r.stride(1) == 1 || k == 1 ? r : r.contiguous();
}
mpmae_stream_t stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
constexpr int64_t row_bytes(int64_t k) { return (k + 127) / 128 * 128; }

std::tuple<at::Tensor, at::Tensor> quantize_gpu(const at::Tensor& w) {
  const int dt = code_of(w.scalar_type());
  TORCH_CHECK_VALUE(w.dim() == 2 && w.numel() > 0 && w.size(1) <= 131071 && w.size(0) <= INT32_MAX && dt >= 0 && w.layout() == at::kStrided,
                    "a weight is a dense matrix [N, K] of fp32, bf16 or fp16, K at most 131071");
  TORCH_CHECK_VALUE(w.device().is_cuda(), "this layer runs on the GPU only: the weight is on ", w.device());
  TORCH_CHECK(quant_entry, "the kernels are not loaded: mmearth_train_amd.int8.load_ops()");
  const int64_t n = w.size(0), k = w.size(1);
  c10::OptionalDeviceGuard guard(w.device());
  const at::Tensor r = rows_of(w, k);
  at::Tensor q = at::empty({n, row_bytes(k)}, w.options().dtype(at::kChar)), scale = at::empty({n}, w.options().dtype(at::kFloat));
  const int err = quant_entry(dt, r.data_ptr(), r.stride(0), (int)n, (int)k, static_cast<int8_t*>(q.data_ptr()), (int)q.size(1), static_cast<float*>(scale.data_ptr()), stream_of(w));
  TORCH_CHECK(!err, "quant_i8 failed with hipError ", err);
  return {q, scale};
}

std::tuple<at::Tensor, at::Tensor> quantize_meta(const at::Tensor& w) {
  TORCH_CHECK_VALUE(w.dim() == 2, "a weight is a matrix [N, K]");
  const c10::SymInt n = w.sym_size(0), kp = (w.sym_size(1) + 127) / 128 * 128;
  return {at::empty_symint({n, kp}, w.options().dtype(at::kChar)), at::empty_symint({n}, w.options().dtype(at::kFloat))};
}

// y = x W^T + bias: checks, output, workspace and launch (in Python they take 11 us, longer than the kernel for a single row)
at::Tensor linear_gpu(const at::Tensor& x, const at::Tensor& q, const at::Tensor& scale, const std::optional<at::Tensor>& bias, int64_t k) {
  const int dt = code_of(x.scalar_type());
  TORCH_CHECK_VALUE(dt >= 0 && x.layout() == at::kStrided, "inputs are dense fp32, bf16 or fp16 tensors, not ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == k, "inputs end in ", k, " elements, the weight's");
  TORCH_CHECK_VALUE(x.device() == q.device() && x.device().is_cuda(), "the input is on ", x.device(), ", the weight on ", q.device());
  const auto plain = [&](const at::Tensor& t, at::ScalarType type, int64_t numel) {
    return t.device() == q.device() && t.scalar_type() == type && t.is_contiguous() && t.numel() == numel;
  };
  TORCH_CHECK_VALUE(q.dim() == 2 && q.scalar_type() == at::kChar && q.is_contiguous() && q.size(0) >= 1 && k >= 1 && q.size(1) == row_bytes(k) &&
                        plain(scale, at::kFloat, q.size(0)) && (!bias || plain(*bias, at::kFloat, q.size(0))) && !(reinterpret_cast<uintptr_t>(q.data_ptr()) & 15),
                    "a weight is what quantize_weight makes: int8 rows of K rounded up to a multiple of 128, fp32 scales and bias, contiguous");
  TORCH_CHECK(linear_entry, "the kernels are not loaded: mmearth_train_amd.int8.load_ops()");
  const int64_t n = q.size(0), kp = q.size(1);
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  c10::OptionalDeviceGuard guard(x.device());
  at::Tensor y = at::empty(shape, x.options());
  if (!y.numel()) return y;
  const at::Tensor r = rows_of(x, k);
  const int64_t m = r.size(0);
  TORCH_CHECK_VALUE(m <= INT32_MAX && n <= INT32_MAX, "more than 2^31 - 1 rows");
  const int64_t codes = m * (kp + 4), part_at = (codes + 15) / 16 * 16;
  const at::Tensor ws = at::empty({part_at + part_bytes((int)m, (int)n, (int)k)}, x.options().dtype(at::kByte));
  char* at = static_cast<char*>(ws.data_ptr());
  MpmaeI8Args a{};
  a.x = r.data_ptr(); a.q = reinterpret_cast<int8_t*>(at); a.sx = reinterpret_cast<float*>(at + m * kp);
  a.w = static_cast<const int8_t*>(q.data_ptr()); a.sw = static_cast<const float*>(scale.data_ptr());
  a.bias = bias ? static_cast<const float*>(bias->data_ptr()) : nullptr;
  a.y = y.data_ptr(); a.part = reinterpret_cast<int*>(at + part_at);
  a.ldx = r.stride(0); a.ldy = n; a.M = (int)m; a.N = (int)n; a.K = (int)k; a.ldq = (int)kp; a.ldw = (int)kp;
  const int err = linear_entry(dt, &a, stream_of(x));
  TORCH_CHECK(!err, "linear_i8 failed with hipError ", err);
  return y;
}

at::Tensor linear_meta(const at::Tensor& x, const at::Tensor& q, const at::Tensor&, const std::optional<at::Tensor>&, int64_t k) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.sym_size(-1) == k, "inputs end in ", k, " elements, the weight's");
  c10::SymDimVector shape(x.sym_sizes().begin(), x.sym_sizes().end());
  shape.back() = q.sym_size(0);
  return at::empty_symint(shape, x.options());
}

using Linear = at::Tensor(const at::Tensor&, const at::Tensor&, const at::Tensor&, const std::optional<at::Tensor>&, int64_t);
at::Tensor call_linear(const at::Tensor& x, const at::Tensor& q, const at::Tensor& scale, const std::optional<at::Tensor>& bias, int64_t k) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("mpmae::linear_int8", "").typed<Linear>();
  return op.call(x, q, scale, bias, k);
}

// no backward pass and no tangent: an input that needs either is refused
at::Tensor linear_autograd(const at::Tensor& x, const at::Tensor& q, const at::Tensor& scale, const std::optional<at::Tensor>& bias, int64_t k) {
  const bool forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const at::Tensor* t : {&x, &scale, bias ? &*bias : &x}) {
    TORCH_CHECK(!(t->requires_grad() && at::GradMode::is_enabled()), "linear_int8 has no backward pass: call it under torch.no_grad()");
    TORCH_CHECK(!(forward && t->_fw_grad(0).defined()), "linear_int8 has no derivative: an input is a dual tensor of forward-mode differentiation");
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return call_linear(x, q, scale, bias, k);
}

// linear_i8(x, q, scale, bias or None, k) -> y
PyObject* linear_i8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !THPVariable_Check(args[2]) || (args[3] != Py_None && !THPVariable_Check(args[3])))
    return PyErr_Format(PyExc_TypeError, "linear_i8(x, q, scale, bias, k)");
  const long long k = PyLong_AsLongLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  return THPVariable_Wrap(call_linear(THPVariable_Unpack(args[0]), THPVariable_Unpack(args[1]), THPVariable_Unpack(args[2]),
                                      args[3] == Py_None ? std::optional<at::Tensor>() : std::optional<at::Tensor>(THPVariable_Unpack(args[3])), k));
  END_HANDLE_TH_ERRORS
}

TORCH_LIBRARY(mpmae, m) {
  m.def("linear_int8(Tensor x, Tensor q, Tensor scale, Tensor? bias, int k) -> Tensor");
  m.def("quantize_int8(Tensor weight) -> (Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(mpmae, CUDA, m) {
  m.impl("linear_int8", linear_gpu);
  m.impl("quantize_int8", quantize_gpu);
}
TORCH_LIBRARY_IMPL(mpmae, CPU, m) {      // (their refusals)
  m.impl("linear_int8", linear_gpu);
  m.impl("quantize_int8", quantize_gpu);
}
TORCH_LIBRARY_IMPL(mpmae, Meta, m) {
  m.impl("linear_int8", linear_meta);
  m.impl("quantize_int8", quantize_meta);
}
TORCH_LIBRARY_IMPL(mpmae, Autograd, m) { m.impl("linear_int8", linear_autograd); }

PyMethodDef methods[] = {{"gather", gather, METH_VARARGS, "addresses of parameters and gradients"},
                         {"same_lists", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(same_lists)), METH_FASTCALL, "whether parameter lists are still the same"},
                         {"linear_i8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(linear_i8)), METH_FASTCALL, "int8 linear layer"},
                         {"adamw", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(adamw)), METH_FASTCALL, "one step"},
                         {"bind", bind, METH_VARARGS, "entry points of the kernel library"}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_tensors", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host_tensors() { return PyModule_Create(&module); }
