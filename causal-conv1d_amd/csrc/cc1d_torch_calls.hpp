// What the direct calls from Python share (see causal_conv1d.cpp: "direct calls from Python").
#pragma once

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/impl/LocalDispatchKeySet.h>

#include <optional>

#include "cc1d_torch.hpp"

// The direct calls of mixer.cpp, ended by an entry without a name.
PyMethodDef *mixer_direct_calls();

namespace {

inline bool plain(PyObject *o) { return THPVariable_CheckExact(o); }
inline bool plain_or_none(PyObject *o) { return o == Py_None || plain(o); }
inline std::optional<at::Tensor> optional_tensor(PyObject *o) {
    return o == Py_None ? std::optional<at::Tensor>() : std::optional<at::Tensor>(THPVariable_Unpack(o));
}
inline bool generic_path_needed() {
    return at::impl::torch_function_mode_enabled() || torch::jit::tracer::isTracing();
}

template <typename F>
auto typed_op(const char *name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

#define NOT_IMPLEMENTED() do { Py_INCREF(Py_NotImplemented); return Py_NotImplemented; } while (0)

inline bool functorch_active() {
    return c10::impl::tls_local_dispatch_key_set().included_.has(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}
// What only the Python function answers for: functorch transforms and forward-mode gradients, which it refuses in its own words.
inline bool python_graph_needed(const std::optional<at::Tensor> &t) { return t.has_value() && (t->has_names() || t->_fw_grad(0).defined()); }

}  // namespace
