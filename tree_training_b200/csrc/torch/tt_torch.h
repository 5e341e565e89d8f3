// What the torch bindings share: errors, argument checks, the stream of a call.
#pragma once

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <array>
#include <atomic>
#include <optional>
#include <string>

#include "../../../include/tree_training_b200.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

namespace tt_torch {

// ---- errors and arguments ------------------------------------------------------

// A status of the library other than TT_OK; becomes the package's TTError.
struct Failure : std::runtime_error {
  std::string fn;
  int code;
  Failure(const char* f, int c)
      : std::runtime_error(std::string(f) + " failed: " + tt_status_string(c) + " (status " +
                           std::to_string(c) + ")"),
        fn(f), code(c) {}
};

inline void check_status(const char* fn, int code) {
  if (code != TT_OK) throw Failure(fn, code);
}

[[noreturn]] inline void type_error(const std::string& s) { throw py::type_error(s); }
[[noreturn]] inline void value_error(const std::string& s) { throw py::value_error(s); }

inline int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TT_F32;
    case at::kBFloat16: return TT_BF16;
    case at::kHalf: return TT_F16;
    default: return -1;
  }
}

inline void need_cuda(const char* op, const char* name, const Tensor& t, const Tensor& first) {
  if (!t.defined()) return;
  if (!t.is_cuda())
    throw std::runtime_error(std::string(op) + ": " + name + " must be a CUDA tensor (no CPU path)");
  if (t.device() != first.device())
    throw std::runtime_error(std::string(op) + ": " + name + " is on " + t.device().str() +
                             ", other tensors on " + first.device().str());
}

inline void need_int(const char* op, const char* what, const Tensor& t) {
  if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)
    type_error(std::string(op) + ": int64/int32 " + what + " required");
}

// The C ABI's sizes have 32 bits: larger ones are refused, not cut off.
inline void need_size(const char* op, const char* what, int64_t n) {
  if (n > 0x7fffffff)
    value_error(std::string(op) + ": " + what + " of " + std::to_string(n) +
                " is over the limit of 2^31 - 1");
}

// There are no forward-mode derivatives: a result without its tangent would be
// wrong without a word.  (A tangent counts with gradients turned off, too.)
inline void no_tangent(const char* op, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined())
      throw std::runtime_error(std::string(op) + ": forward-mode derivatives are not supported");
}

inline bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// [rows, D] with unit last stride and rows that do not overlap (else a copy, as of
// tensors whose sign is kept beside their memory).
inline Tensor rows2d(const Tensor& t) {
  if (t.is_neg()) return t.resolve_neg().contiguous();
  if (t.stride(1) == 1 && (t.stride(0) >= t.size(1) || t.size(0) <= 1)) return t;
  return t.contiguous();
}

inline const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
inline void* out(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline int64_t row_stride(const Tensor& t) { return t.defined() ? t.stride(0) : 0; }

inline Tensor empty(at::IntArrayRef sizes, const Tensor& like, at::ScalarType type) {
  return at::empty(sizes, like.options().dtype(type).memory_format(at::MemoryFormat::Contiguous)
                              .requires_grad(false));
}

// The device and stream of a call.
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(const Tensor& t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

// The device's status word, which check_device_status reads: asked for once.
inline std::array<std::atomic<int32_t*>, 64> status_words;

inline int32_t* status_of(const Tensor& t) {
  const int i = t.device().index();
  TORCH_CHECK(i >= 0 && i < (int)status_words.size(), "device index out of range");
  int32_t* p = status_words[i].load(std::memory_order_acquire);
  if (!p) {
    py::gil_scoped_acquire gil;
    py::object word = py::module_::import("tree_training_b200.attention")
                          .attr("_status_word")(py::cast(t.device()));
    p = word.cast<Tensor>().data_ptr<int32_t>();
    status_words[i].store(p, std::memory_order_release);
  }
  return p;
}

// Gradients that are differentiated again (create_graph) raise there.
inline variable_list once(const char* op, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(op) + ": its gradients cannot be differentiated again", 1);
  for (auto& g : grads) {
    if (!g.defined()) continue;
    variable_list one{g.detach().requires_grad_(true)};
    g = (*error)(std::move(one))[0];
  }
  return grads;
}

}  // namespace tt_torch
