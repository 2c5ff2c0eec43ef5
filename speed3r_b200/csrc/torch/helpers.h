// What the operators' files share: argument checks, allocation, and the rules of differentiation that every operator follows.
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/CUDAEvent.h>
#include <ATen/cuda/CachingHostAllocator.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <cmath>
#include <tuple>
#include <vector>

#include "../../../include/speed3r_b200.h"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void need(const Tensor& t, const char* name, at::ScalarType dtype = at::kBFloat16, bool contiguous = true) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor: the speed3r_b200 kernels have no CPU path");
  TORCH_CHECK(t.scalar_type() == dtype, name, " must be ", dtype, ", got ", t.scalar_type());
  TORCH_CHECK(!contiguous || t.is_contiguous(), name, " must be contiguous");
}

// Sizes that are divided by: a division by zero ends the process in C++, where Python raised.
template <typename... N>
void need_positive(const char* what, N... n) {
  TORCH_CHECK(((n > 0) && ...), what, ": block, window and stride must be positive");
}

void check(int rc, const char* what) {
  if (rc == 0) return;
  char msg[512];
  s3r_last_error(msg, sizeof(msg));
  TORCH_CHECK(false, what, " failed with code ", rc, ": ", msg);
}

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
const int32_t* i32(const Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }
int32_t* i32m(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }
float* f32(const Tensor& t) { return static_cast<float*>(t.data_ptr()); }
// Through the dispatcher an empty tensor takes twice as long (1.4 us), and a small call is made of such times.
Tensor fresh(at::IntArrayRef shape, const Tensor& like, at::ScalarType dtype) {
  if (like.is_cuda()) return at::detail::empty_cuda(shape, dtype, like.device(), c10::nullopt);
  return at::empty(shape, like.options().dtype(dtype));
}
// contiguous, whatever the strides of `t` (at::empty_like would keep a permuted layout)
Tensor fresh_like(const Tensor& t) { return fresh(t.sizes(), t, t.scalar_type()); }
// The same values at a multiple of 16 bytes: a contiguous view may begin anywhere in its storage (a slice, a flattened
// parameter buffer), and the kernels load vectors.
Tensor aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(); }
optional<Tensor> aligned(const optional<Tensor>& t) { return t.has_value() ? optional<Tensor>(aligned(*t)) : t; }
Tensor none(const Tensor& like) { return at::empty({0}, like.options()); }

// Forward-mode derivatives are refused, in every operator and whether a gradient is wanted or not: past the nodes, the base
// operators would drop a tangent without a word.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const optional<Tensor>& t) { return t.has_value() && has_tangent(*t); }
bool has_tangent(at::TensorList list) {
  for (const Tensor& t : list)
    if (has_tangent(t)) return true;
  return false;
}
template <typename... T>
void no_tangents(const T&... t) {
  if (!torch::autograd::ForwardADLevel::try_get_by_idx(0)) return;       // there are none; looking at each tensor of a list takes a lock each
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(t) || ...), "speed3r_b200: forward mode AD is not implemented for the operators of this package");
}
template <typename... T>
bool wants_grad(const T&... t) {
  no_tangents(t...);
  return at::GradMode::is_enabled() && (t.requires_grad() || ...);
}

// A backward of a node.  It runs without recording; where its result is to be differentiated again (create_graph), the result
// raises when that is tried: no operator here has a second derivative, and without this one would be missing silently.
template <typename F>
variable_list once(const variable_list& incoming, F&& backward) {
  const bool again = at::GradMode::is_enabled();
  variable_list g;
  {
    at::NoGradGuard no_grad;
    g = backward();
  }
  if (!again) return g;
  // the error stands between the result and all it depends on: the node's own inputs and the incoming gradients
  torch::autograd::edge_list edges = torch::autograd::collect_next_edges(incoming);
  if (const auto node = torch::autograd::get_current_node()) edges.insert(edges.end(), node->next_edges().begin(), node->next_edges().end());
  const auto error = std::make_shared<torch::autograd::Error>("the backward of speed3r_b200 operators cannot be differentiated again",
                                                              std::move(edges));
  for (Tensor& t : g)
    if (t.defined()) {
      t = t.detach();
      torch::autograd::set_history(t, error);
    }
  return g;
}

// a tensor with memory, not one of those that a tracer runs the backward on
bool plain(const Tensor& t) {
  return t.is_cuda() && !t.key_set().has(c10::DispatchKey::Python) && !t.key_set().has(c10::DispatchKey::Functionalize) &&
         !c10::impl::dispatch_mode_enabled();
}

// Calls a base operator through the dispatcher (shape functions, tracers and modes see it).
#define S3R_DISPATCHED(fn)                                                                              \
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("speed3r_b200::" #fn, "").typed<decltype(fn)>(); \
  return op.call

}  // namespace
