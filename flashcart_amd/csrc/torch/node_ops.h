// What the PyTorch operators over the node-wise C entry points share: the entry points, checks of arguments, dispatch.
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/library.h>

#include "../../../include/flashcart_hip.h"

namespace fct {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
  decltype(&fc_status_string) status_string;
  decltype(&fc_embedding_fwd) embedding_fwd;
  decltype(&fc_embedding_bwd_workspace) embedding_bwd_workspace;
  decltype(&fc_embedding_bwd) embedding_bwd;
  decltype(&fc_dropout_add) dropout_add;
  decltype(&fc_ffn_saved) ffn_saved;
  decltype(&fc_ffn_fwd_workspace) ffn_fwd_workspace;
  decltype(&fc_ffn_fwd) ffn_fwd;
  decltype(&fc_ffn_bwd_workspace) ffn_bwd_workspace;
  decltype(&fc_ffn_bwd) ffn_bwd;
  decltype(&fc_node_dense_saved) node_dense_saved;
  decltype(&fc_node_dense_fwd_workspace) node_dense_fwd_workspace;
  decltype(&fc_node_dense_fwd) node_dense_fwd;
  decltype(&fc_node_dense_bwd_workspace) node_dense_bwd_workspace;
  decltype(&fc_node_dense_bwd) node_dense_bwd;
  decltype(&fc_quantized_dense_workspace) quantized_dense_workspace;
  decltype(&fc_quantized_dense) quantized_dense;
  decltype(&fc_row_norm_fwd) row_norm_fwd;
  decltype(&fc_row_norm_quantize) row_norm_quantize;
  decltype(&fc_row_norm_bwd_workspace) row_norm_bwd_workspace;
  decltype(&fc_row_norm_bwd) row_norm_bwd;
};
extern Api api;

inline void check(int64_t status, const char* what) {
  TORCH_CHECK(status == 0, what, " failed: ", api.status_string((int)status), " (status ", status, ")");
}

inline int32_t code_of(const char* name, const Tensor& t) {
  const auto type = t.scalar_type();
  TORCH_CHECK_TYPE(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf, "`", name,
                   "` must be float32, bfloat16 or float16, got ", type, ".");
  return type == at::kFloat ? FC_F32 : type == at::kBFloat16 ? FC_BF16 : FC_F16;
}

// The tensor, checked, as contiguous memory on the device of `first`.
inline Tensor take(const char* name, const Tensor& t, at::ScalarType type, const Tensor& first) {
  TORCH_CHECK(t.is_cuda(), "flashcart_amd runs its kernels on ROCm devices only; `", name, "` is on ", t.device(),
              ". Move the model and inputs to a GPU (model.to('cuda')).");
  TORCH_CHECK_TYPE(t.scalar_type() == type, "`", name, "` must be ", type, ", got ", t.scalar_type(), ".");
  TORCH_CHECK(t.device() == first.device(), "`", name, "` is on ", t.device(), ", the other arguments are on ",
              first.device(), ".");
  return t.contiguous();
}
inline Tensor take_ids(const Tensor& ids, const Tensor& first) {
  return take("ids", ids.scalar_type() == at::kInt ? ids.to(at::kLong) : ids, at::kLong, first);
}

inline void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

inline Tensor bytes(const Tensor& like, int64_t size, const char* what) {
  if (size < 0) check(-size, what);
  return at::empty({size}, like.options().dtype(at::kByte));
}

// Whether a call with these inputs goes through its autograd formula: where autograd records it, and where an input carries
// a forward-mode tangent (in either grad mode), which the formula refuses; below it the tangent would be lost.
inline bool records(std::initializer_list<const Tensor*> inputs) {
  const bool grad = at::GradMode::is_enabled();
  for (const Tensor* t : inputs)
    if (t->defined() && ((grad && t->requires_grad()) || t->_fw_grad(/*level=*/0).defined())) return true;
  return false;
}

// An operator called through the dispatcher: differentiable, or what is below autograd (a kernel, or what stands in for one
// under tracing and fake tensors) where the caller has excluded autograd.
template <class F>
auto dispatched(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
#define FCT_DISPATCHED(name, ...) \
  static const auto op = dispatched<decltype(name)>("flashcart::" #name); \
  return op.call(__VA_ARGS__)

inline int32_t aligned(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if ((uintptr_t)t->const_data_ptr() & 15) return 0;
  return 1;
}

}  // namespace fct
