// What the torch sides of the library's calls share: which tensors they take, and when torch is being watched.
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/autograd/python_variable.h>

namespace xnq_torch {

inline int xnq_dtype(at::ScalarType t) { // F32 0, F16 1, BF16 30: the ggml ids
  return t == at::kFloat ? 0 : (t == at::kHalf ? 1 : (t == at::kBFloat16 ? 30 : -1));
}
// an ordinary dense CUDA tensor: no subclass, no wrapper of a transform
inline bool plain(PyObject *o) {
  if (!THPVariable_CheckExact(o)) return false;
  constexpr c10::DispatchKeySet allowed({c10::DispatchKey::CUDA, c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::AutogradCUDA, c10::DispatchKey::AutocastCUDA});
  const c10::DispatchKeySet ks = THPVariable_Unpack(o).key_set();
  return (ks.raw_repr() & ~allowed.raw_repr()) == 0 && ks.has(c10::DispatchKey::CUDA);
}
// Something of torch looks at operators or replaces them: a function or dispatch mode, a transform of torch.func (whatever tensors it has wrapped), a tracer.
inline bool observed() {
  constexpr c10::DispatchKeySet ordinary({c10::DispatchKey::BackendSelect, c10::DispatchKey::ADInplaceOrView});
  return (c10::impl::tls_local_dispatch_key_set().included_.raw_repr() & ~ordinary.raw_repr()) != 0 || c10::impl::TorchDispatchModeTLS::any_modes_set() ||
         at::impl::torch_function_mode_enabled();
}
// a tensor on the current device (what empty_cuda does behind its look for the device)
inline at::Tensor empty_here(at::IntArrayRef shape, at::ScalarType t) {
  return at::Tensor(at::detail::empty_generic(shape, c10::cuda::CUDACachingAllocator::get(), c10::DispatchKeySet(c10::DispatchKey::CUDA), t, std::nullopt));
}
struct RelaxedCapture { // (a graph that another thread is capturing does not mind what this one allocates or frees)
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  RelaxedCapture() { (void)cudaThreadExchangeStreamCaptureMode(&mode); }
  ~RelaxedCapture() { (void)cudaThreadExchangeStreamCaptureMode(&mode); }
};

// torch_kv_cache.cpp
PyObject *kv_cache(PyObject *, PyObject *);
PyObject *kv_bind(PyObject *, PyObject *);
PyObject *kv_store(PyObject *, PyObject *const *, Py_ssize_t);
PyObject *kv_rope_store(PyObject *, PyObject *const *, Py_ssize_t);
PyObject *kv_load(PyObject *, PyObject *const *, Py_ssize_t);
PyObject *kv_attend(PyObject *, PyObject *const *, Py_ssize_t);
PyObject *kv_reserve(PyObject *, PyObject *const *, Py_ssize_t);
PyObject *kv_plan(PyObject *, PyObject *const *, Py_ssize_t);
PyObject *kv_keep(PyObject *, PyObject *const *, Py_ssize_t);
PyObject *kv_plan_handle(PyObject *, PyObject *);
PyObject *kv_plan_view(PyObject *, PyObject *);

} // namespace xnq_torch
