// race_torch.h -- what the C++ calls share (race_torch.cpp: the attention operators,
// layers_torch.cpp: the operators around them).
#pragma once
#include <dlfcn.h>
#include <torch/extension.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <string>

#include "../../include/race_attention.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

extern PyObject *race_error;  // _lib.RaceError

// of layers_torch.cpp: its functions of the library, and its Python entries
void bind_layers(void *library, const std::string &path);
void add_layers(py::module_ &m);

// A call that these functions do not take, or whose status is an error.
struct NotTaken {};

// Raise RaceError where Python code cannot be fallen back to (the engine's thread).
[[noreturn]] inline void raise_race_error(const char *what, int rc, const char *text) {
    const std::string msg = std::string(what) + " failed (" + std::to_string(rc) + "): " + text;
    py::gil_scoped_acquire gil;
    PyErr_SetString(race_error, msg.c_str());
    python_error e;
    e.persist();
    throw e;
}

inline void *stream_of(const Tensor &x) { return (void *)c10::hip::getCurrentHIPStream(x.device().index()).stream(); }

// a plain strided CUDA tensor of the current device: no wrapper of a transform, a mode or a subclass
inline bool plain(const Tensor &x) {
    return x.defined() && x.is_cuda() && x.layout() == at::kStrided && x.unsafeGetTensorImpl()->has_storage() &&
           !x.unsafeGetTensorImpl()->is_python_dispatch() && !x.is_conj() && !x.is_neg() &&
           !x._fw_grad(/*level=*/0).defined();  // forward-mode AD: refused by the Python Functions
}
// torch.Tensor or torch.nn.Parameter itself (THPVariable_CheckExact takes both), no other subclass
inline bool is_tensor(py::handle o) { return THPVariable_CheckExact(o.ptr()); }

inline void *ptr(const Tensor &x) { return x.data_ptr(); }
inline float *fptr(const Tensor &x) { return x.defined() ? static_cast<float *>(x.data_ptr()) : nullptr; }

inline Tensor bytes(size_t n, const Tensor &like) {
    return at::empty({(int64_t)(n < 16 ? 16 : n)}, like.options().dtype(at::kByte));
}
inline Tensor fp32(at::IntArrayRef shape, const Tensor &like) { return at::empty(shape, like.options().dtype(at::kFloat)); }

// whether calls are recorded or redirected: Python's paths then take them
inline bool redirected() {
    return torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::any_modes_set();
}
