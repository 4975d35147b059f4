// train_ops_common.h -- what the PyTorch operators of the training step share:
// checks, allocation, and the autograd nodes' helpers.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <cstdlib>
#include <optional>

#include "muon_train_sm100.h"

namespace muon_train_ops {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// Of a launch on the current device.  With MUON_POLAR_DEBUG_SYNC set (read on
// every call) it also synchronises, and raises if a wait of a kernel ran out.
inline void CheckStatus(int rc, const char* who) {
  TORCH_CHECK(rc == MUON_POLAR_OK, who, " failed, status=", rc,
              ", detail=", muon_polar_status_string(rc));
  if (std::getenv("MUON_POLAR_DEBUG_SYNC") == nullptr) return;
  uint32_t flags = 0;
  const int read = muon_train_read_device_status(c10::cuda::current_device(), &flags, /*clear=*/1);
  TORCH_CHECK(read == MUON_POLAR_OK, who, " failed, status=", read,
              ", detail=", muon_polar_status_string(read));
  TORCH_CHECK(flags == 0, who, " gave up on a bounded wait, status word=", flags);
}

inline int Dtype(const Tensor& t, const char* who, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return MUON_TRAIN_F32;
    case at::kBFloat16: return MUON_TRAIN_BF16;
    case at::kHalf: return MUON_TRAIN_F16;
    default: TORCH_CHECK_TYPE(false, who, ": ", name, " must be float32, bfloat16 or float16, got ",
                              t.scalar_type());
  }
}

inline void CheckCuda(const Tensor& t, const char* who, const char* name) {
  TORCH_CHECK_VALUE(t.device().is_cuda(), who, ": ", name, " must be a CUDA tensor, got ", t.device());
}
inline void CheckDevice(const Tensor& t, const Tensor& like, const char* who, const char* name) {
  TORCH_CHECK_VALUE(t.device() == like.device(), who, ": ", name, " must be on ", like.device(),
                    ", got ", t.device());
}

// An uninitialised contiguous CUDA tensor, without the dispatcher's way there:
// small calls are bound by the host.
inline Tensor Empty(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt));
}

inline void* Ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline const Tensor& Given(const OptTensor& t) {
  static const Tensor none;
  return t.has_value() && t->defined() ? *t : none;
}
inline void* Stream(const Tensor& t) {
  return static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

// Tangents are not carried on, nor is a gradient of a gradient computed: say
// so instead of returning a result that autograd would take for a constant.
inline void NoTangents(std::initializer_list<const Tensor*> inputs, const char* who) {
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), who,
                                ": forward-mode differentiation (jvp) is not supported");
}
inline void NoSecondOrder(const variable_list& grads, const char* who) {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), who,
                              ": the gradient cannot be differentiated again (create_graph=True)");
  for (const Tensor& g : grads) NoTangents({&g}, who);
}

inline at::IntArrayRef Lead(const Tensor& t) { return t.sizes().slice(0, t.dim() - 1); }

template <typename Fn>
auto Op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Fn>();
}

// Whether autograd records a call: otherwise it goes to the kernels directly.
inline bool Recorded(std::initializer_list<const Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : inputs)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// A node of the graph whose next edges are `inputs`, in order.
template <typename N, typename... Inputs>
std::shared_ptr<N> MakeNode(const Inputs&... inputs) {
  auto node = std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return node;
}

inline OptTensor Optional(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// Clips `grads` in place, or into `out` where it is not empty; their norm goes to
// `norm` (one fp32 element).  By pointers: to copy a tensor that Python holds
// counts its object's references too.  block_ops.cpp
using TensorPointers = c10::ArrayRef<const Tensor*>;
void clip_gradients(TensorPointers grads, TensorPointers out, double max_norm, bool largest, const Tensor& norm);

}  // namespace muon_train_ops
