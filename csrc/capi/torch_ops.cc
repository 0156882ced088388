// The 8-bit operators' calls on torch tensors without the interpreter in between: checks, result allocation and launch of
// the plain case - contiguous CUDA tensors of the right types and shapes on the current device, new results.  For
// everything else (strided operands, destinations, other devices, gradients, traces, wrong arguments, a failed launch) the
// functions return None and the Python operators go their general way, which also words the errors.  A call costs 3.3 to
// 4.3 us this way (two hosts), 2.8 of them the launch itself, instead of 8 to 13.
//
// Accessors of torch's tensors are compiled in, so the module serves the torch that it was built for, which `built_for`
// names (the build passes TCA_TORCH); the loader leaves it alone under any other.
//
// The launchers come as addresses: libtca_hip.so is loaded by its own loader.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <iterator>
#include <limits>
#include <type_traits>

#include "kernels.h"

namespace py = pybind11;

namespace {

// called through their declarations: a launcher whose arguments change does not compile here until its call does
decltype(&tca_int8_quantize_launch) g_quantize;
decltype(&tca_int8_rms_norm_launch) g_norm;
decltype(&tca_int8_dequantize_launch) g_dequantize;
decltype(&tca_int8_linear_launch) g_linear;
decltype(&tca_int8_linear_workspace_bytes) g_workspace;

// element type codes of the kernels, -1: another type
int Code(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kHalf ? 1 : t == at::kBFloat16 ? 2 : -1;
}
at::ScalarType Type(long code) { return code == 0 ? at::kFloat : code == 1 ? at::kHalf : at::kBFloat16; }

constexpr long long kMostWidth = 1ll << 29, kMostK = 131071;

// Whether something records this thread's operations: torch.jit.trace, or make_fx, at either of its levels.
bool Traced() {
  return at::tracer::impl::is_dispatch_enabled() ||
         c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value() ||
         c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
}

// A plain operand: a contiguous tensor on the current CUDA device that needs no gradient and has no tangent, in a call that
// nothing traces.  `device` is set by the first operand (-1 before it): without a GPU there is no current device to ask for.
struct Operand {
  const at::Tensor* t = nullptr;
  bool Take(PyObject* o, int& device) {
    if (!THPVariable_CheckExact(o)) return false;
    t = &THPVariable_Unpack(o);
    if (!t->is_cuda() || t->layout() != at::kStrided || !t->is_contiguous() || t->requires_grad() || t->is_conj() || t->is_neg() ||
        t->_fw_grad(0).defined())
      return false;
    if (device < 0) {
      if (Traced()) return false;
      device = t->device().index();
      return c10::hip::current_device() == device;
    }
    return t->device().index() == device;
  }
  const at::Tensor& operator*() const { return *t; }
  const at::Tensor* operator->() const { return t; }
};

void* CurrentStream(int device) { return c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(device)).stream(); }

// a new tensor on that device, past torch's dispatcher (0.2 us less)
at::Tensor New(at::IntArrayRef shape, at::ScalarType type, int device) {
  return at::Tensor(at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device)), std::nullopt));
}

#define NOT_PLAIN Py_RETURN_NONE

// a tuple of the results, or null where one could not be made
template <typename... Results>
PyObject* Tuple(Results&&... results) {
  const py::object made[] = {py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(results)))...};
  PyObject* tuple = PyTuple_New(sizeof...(results));
  for (Py_ssize_t i = 0; tuple && i < static_cast<Py_ssize_t>(sizeof...(results)); ++i) {
    if (!made[i]) {
      Py_CLEAR(tuple);
      break;
    }
    PyTuple_SET_ITEM(tuple, i, py::object(made[i]).release().ptr());
  }
  return tuple;
}

// (x, gated) -> (q, scale)
PyObject* Quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2) NOT_PLAIN;
  int device = -1;
  const bool gated = args[1] == Py_True;
  Operand x;
  if (!x.Take(args[0], device)) NOT_PLAIN;
  const int code = Code(x->scalar_type());
  const auto sizes = x->sizes();
  if (code < 0 || sizes.empty() || sizes.back() < 1 || sizes.back() > kMostWidth || (gated && sizes.back() % 2)) NOT_PLAIN;
  const long long width = gated ? sizes.back() / 2 : sizes.back();
  at::DimVector shape(sizes.begin(), sizes.end());
  shape.back() = width;
  at::Tensor q = New(shape, at::kChar, device);
  at::Tensor scale = New(sizes.slice(0, sizes.size() - 1), at::kFloat, device);
  const long long rows = scale.numel();
  if (rows && g_quantize(x->const_data_ptr(), q.mutable_data_ptr(), scale.mutable_data_ptr(), code, gated, rows, width,
                         sizes.back(), width, CurrentStream(device)))
    NOT_PLAIN;
  return Tuple(q, scale);
  END_HANDLE_TH_ERRORS
}

// (x, weight, residual or None, eps) -> (q, scale) or (q, scale, sum)
PyObject* Norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) NOT_PLAIN;
  int device = -1;
  const bool with_residual = args[2] != Py_None;
  Operand x, weight, residual;
  if (!x.Take(args[0], device) || !weight.Take(args[1], device) || (with_residual && !residual.Take(args[2], device)) ||
      !PyFloat_CheckExact(args[3]))
    NOT_PLAIN;
  const double eps = PyFloat_AS_DOUBLE(args[3]);
  const int code = Code(x->scalar_type());
  const auto sizes = x->sizes();
  if (code < 0 || sizes.empty() || sizes.back() < 1 || sizes.back() > kMostWidth || weight->dim() != 1 ||
      weight->size(0) != sizes.back() || (weight->scalar_type() != at::kFloat && weight->scalar_type() != x->scalar_type()) ||
      !(eps > 0 && eps < std::numeric_limits<double>::infinity()) ||
      (with_residual && (residual->scalar_type() != x->scalar_type() || residual->sizes() != sizes)))
    NOT_PLAIN;
  const long long width = sizes.back();
  at::Tensor q = New(sizes, at::kChar, device);
  at::Tensor scale = New(sizes.slice(0, sizes.size() - 1), at::kFloat, device);
  at::Tensor sum;
  if (with_residual) sum = New(sizes, x->scalar_type(), device);
  const long long rows = scale.numel();
  if (rows && g_norm(x->const_data_ptr(), with_residual ? residual->const_data_ptr() : nullptr, weight->const_data_ptr(),
                     q.mutable_data_ptr(), scale.mutable_data_ptr(), with_residual ? sum.mutable_data_ptr() : nullptr, code,
                     weight->scalar_type() == at::kFloat, eps, rows, width, width, with_residual ? width : 0, width,
                     with_residual ? width : 0, CurrentStream(device)))
    NOT_PLAIN;
  return with_residual ? Tuple(q, scale, sum) : Tuple(q, scale);
  END_HANDLE_TH_ERRORS
}

// 8-bit rows with their scales
bool Quantized(const Operand& q, const Operand& scale) {
  const auto sizes = q->sizes();
  return q->scalar_type() == at::kChar && scale->scalar_type() == at::kFloat && !sizes.empty() &&
         scale->sizes() == sizes.slice(0, sizes.size() - 1);
}

// (q, scale, code) -> values
PyObject* Dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) NOT_PLAIN;
  int device = -1;
  Operand q, scale;
  if (!q.Take(args[0], device) || !scale.Take(args[1], device) || !Quantized(q, scale)) NOT_PLAIN;
  const long code = PyLong_AsLong(args[2]);
  const long long width = q->sizes().back(), rows = scale->numel();
  if (width < 1 || width > kMostWidth) NOT_PLAIN;
  at::Tensor out = New(q->sizes(), Type(code), device);
  if (rows && g_dequantize(q->const_data_ptr(), scale->const_data_ptr(), out.mutable_data_ptr(), static_cast<int>(code), rows,
                           width, width, width, CurrentStream(device)))
    NOT_PLAIN;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (x, x_scale, weight, weight_scale, bias or None, residual or None, code) -> y
PyObject* Linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) NOT_PLAIN;
  int device = -1;
  Operand x, x_scale, weight, weight_scale, bias, residual;
  const bool with_bias = args[4] != Py_None, with_residual = args[5] != Py_None;
  if (!x.Take(args[0], device) || !x_scale.Take(args[1], device) || !weight.Take(args[2], device) ||
      !weight_scale.Take(args[3], device) || (with_bias && !bias.Take(args[4], device)) ||
      (with_residual && !residual.Take(args[5], device)) || !Quantized(x, x_scale) || !Quantized(weight, weight_scale))
    NOT_PLAIN;
  const long code = PyLong_AsLong(args[6]);
  const auto sizes = x->sizes();
  const long long k = sizes.back(), tokens = x_scale->numel();
  if (weight->dim() != 2 || weight->size(1) != k || k < 1 || k > kMostK) NOT_PLAIN;
  const long long outputs = weight->size(0);
  at::DimVector shape(sizes.begin(), sizes.end());
  shape.back() = outputs;
  const at::ScalarType type = Type(code);
  if (with_bias && (bias->scalar_type() != type || bias->dim() != 1 || bias->size(0) != outputs)) NOT_PLAIN;
  if (with_residual && (residual->scalar_type() != type || residual->sizes() != at::IntArrayRef(shape))) NOT_PLAIN;
  at::Tensor out = New(shape, type, device);
  if (tokens && outputs) {
    const void *xp = x->const_data_ptr(), *wp = weight->const_data_ptr();
    at::Tensor workspace;
    if (((reinterpret_cast<uintptr_t>(xp) | reinterpret_cast<uintptr_t>(wp) | k) & 15) != 0) {
      const long long bytes = g_workspace(xp, wp, tokens, outputs, k, k, k);
      if (bytes) workspace = New({bytes}, at::kChar, device);
    }
    if (g_linear(xp, x_scale->const_data_ptr(), wp, weight_scale->const_data_ptr(), with_bias ? bias->const_data_ptr() : nullptr,
                 with_residual ? residual->const_data_ptr() : nullptr, out.mutable_data_ptr(), static_cast<int>(code), tokens,
                 outputs, k, k, k, with_residual ? outputs : 0, outputs,
                 workspace.defined() ? workspace.mutable_data_ptr() : nullptr, CurrentStream(device)))
      NOT_PLAIN;
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// the launchers that are called here, as `launchers` names them, and where `use` puts their addresses
template <auto& kFunction>
void Set(unsigned long long address) {
  kFunction = reinterpret_cast<std::remove_reference_t<decltype(kFunction)>>(address);
}
struct Launcher {
  const char* name;
  void (*set)(unsigned long long);
};
constexpr Launcher kLaunchers[] = {{"tca_int8_quantize_launch", Set<g_quantize>},
                                   {"tca_int8_rms_norm_launch", Set<g_norm>},
                                   {"tca_int8_dequantize_launch", Set<g_dequantize>},
                                   {"tca_int8_linear_launch", Set<g_linear>},
                                   {"tca_int8_linear_workspace_bytes", Set<g_workspace>}};

// the launchers' addresses, in that order
PyObject* Use(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != static_cast<Py_ssize_t>(std::size(kLaunchers))) {
    PyErr_SetString(PyExc_TypeError, "an address for each of the launchers");
    return nullptr;
  }
  unsigned long long addresses[std::size(kLaunchers)];
  for (Py_ssize_t i = 0; i < n; ++i) {
    addresses[i] = PyLong_AsUnsignedLongLong(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  for (Py_ssize_t i = 0; i < n; ++i) kLaunchers[i].set(addresses[i]);
  Py_RETURN_NONE;
}

PyCFunction Fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef kMethods[] = {{"use", Fast(Use), METH_FASTCALL, nullptr},
                          {"quantize", Fast(Quantize), METH_FASTCALL, nullptr},
                          {"rms_norm", Fast(Norm), METH_FASTCALL, nullptr},
                          {"dequantize", Fast(Dequantize), METH_FASTCALL, nullptr},
                          {"linear", Fast(Linear), METH_FASTCALL, nullptr},
                          {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_tca_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tca_torch() {
  PyObject* module = PyModule_Create(&kModule);
  PyObject* names = PyTuple_New(std::size(kLaunchers));
  for (size_t i = 0; names && i < std::size(kLaunchers); ++i) {
    PyObject* name = PyUnicode_FromString(kLaunchers[i].name);
    if (!name) Py_CLEAR(names);
    else PyTuple_SET_ITEM(names, i, name);
  }
  if (module && names && PyModule_AddStringConstant(module, "built_for", TCA_TORCH) == 0 &&
      PyModule_AddObject(module, "launchers", names) == 0)
    return module;  // names belongs to it now
  Py_XDECREF(names);
  Py_XDECREF(module);
  return nullptr;
}
