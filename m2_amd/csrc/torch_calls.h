// What the CPython extensions share that call libm2_amd.so for a module's operators (answer_calls.cpp, causal_calls.cpp): errors, streams, checks of arguments.
#pragma once
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>

#include "../../include/m2_amd.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

decltype(&m2_last_error) last_error;      // of libm2_amd.so, which m2_amd/_lib.py has loaded

template <typename F>
void set(F& f, uintptr_t address) { f = reinterpret_cast<F>(address); }

void check(int rc) { TORCH_CHECK(rc == M2_OK, "libm2_amd error ", rc, ": ", last_error()); }

void* current_stream() { return c10::hip::getCurrentHIPStream().stream(); }

void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

int type_of(const char* name, const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), name, ": must live on the GPU (m2_amd has no CPU path); got device ", t.device());
  TORCH_CHECK_TYPE(t.layout() == at::kStrided, name, ": must be strided, got ", t.layout());
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, name, ": must be float32 or bfloat16, got ", t.scalar_type());
  return t.scalar_type() == at::kFloat ? M2_DTYPE_F32 : M2_DTYPE_BF16;
}

// The values one behind the other.
Tensor dense(const Tensor& t) { return t.defined() ? (t.is_neg() ? t.resolve_neg() : t).contiguous() : t; }

// Arguments come by position, without pybind's conversions (1.1 us a call).
const Tensor& tensor(const char* name, PyObject* o) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, ": expected a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
optional<Tensor> tensor_or_none(const char* name, PyObject* o) { return o == Py_None ? std::nullopt : optional<Tensor>(tensor(name, o)); }
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

// Refuses what a kernel that is given a tensor's memory would answer wrongly: tensors that are no plain ones, transforms of functions (vmap, jvp, ...), traces,
// forward-mode gradients, and (unless grad_ok) gradients.
const Tensor& values(const char* name, PyObject* o, bool grad_ok) {
  TORCH_CHECK_TYPE(THPVariable_CheckExact(o), name, ": expected a plain tensor, got ", Py_TYPE(o)->tp_name);
  const Tensor& t = THPVariable_Unpack(o);
  TORCH_CHECK(!c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) && !torch::jit::tracer::isTracing() && !t._fw_grad(0).defined(), name,
              ": function transforms, traces and forward-mode gradients are not supported");
  TORCH_CHECK(grad_ok || !t.requires_grad() || !at::GradMode::is_enabled(), name,
              ": this operator has no gradient; call it under torch.no_grad() or on a detached tensor");
  return t;
}

PyObject* object_of(Tensor t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(t));
}

}  // namespace
