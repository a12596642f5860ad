// mi_torch_plain.hpp -- which torch tensors the native calls take: shared by
// the units of the _torch_call extension.
#pragma once
#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <Python.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

namespace mi_torch {

// A dense contiguous tensor on a HIP device that nothing intercepts: an exact Tensor or
// Parameter whose dispatch keys are the device's own, autograd's and
// autocast's (no conjugate or negative view, no functorch, Python or sparse
// key).
inline const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  static const uint64_t allowed =
      (c10::DispatchKeySet(c10::DispatchKey::CUDA) | c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) |
       c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView) | c10::autocast_dispatch_keyset).raw_repr();
  if (!t.defined() || (t.key_set().raw_repr() & ~allowed) != 0) return nullptr;
  if (!t.is_cuda() || !t.is_contiguous()) return nullptr;
  return &t;
}
inline const at::Tensor* plain(PyObject* o, at::ScalarType dtype) {
  const at::Tensor* t = plain(o);
  return t && t->scalar_type() == dtype ? t : nullptr;
}

// No mode or transform is active on this thread.
inline bool no_mode() {
  if (at::impl::torch_function_mode_enabled() || c10::impl::dispatch_mode_enabled()) return false;
  static const uint64_t allowed = (c10::default_included_set | c10::autocast_dispatch_keyset).raw_repr();
  return (c10::impl::tls_local_dispatch_key_set().included_.raw_repr() & ~allowed) == 0;
}

inline bool disjoint(const at::Tensor& out, const at::Tensor& in) {
  const uintptr_t o = (uintptr_t)out.data_ptr(), i = (uintptr_t)in.data_ptr();
  return o + out.nbytes() <= i || i + in.nbytes() <= o;
}

}  // namespace mi_torch
