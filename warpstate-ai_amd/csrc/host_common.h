// What the C++ operators share (csrc/host_ops.cpp, csrc/host_layer.cpp).
#pragma once

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>

#include "../../include/warpstate_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
typedef std::tuple<Tensor, Tensor, Tensor, Tensor> FourTensors;
typedef std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> FiveTensors;

constexpr int64_t kBlock = 128;

inline void check(int status, const char* name) {
  TORCH_CHECK(status == 0, name, " failed (status ", status, "): ", ws_last_error());
}
inline void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
inline int64_t up(int64_t n, int64_t unit) { return (n + unit - 1) / unit * unit; }
inline int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }
inline int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
inline void* ptr(const Tensor& t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }
inline Tensor bytes(const Tensor& like, at::IntArrayRef sizes) { return at::empty(sizes, like.options().dtype(at::kByte)); }
inline Tensor floats(const Tensor& like, at::IntArrayRef sizes) { return at::empty(sizes, like.options().dtype(at::kFloat)); }

template <class Signature>
c10::TypedOperatorHandle<Signature> find(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}
// The operator below autograd.
template <class Op, class... Args>
auto below(const Op& op, Args&&... args) {
  at::AutoDispatchBelowAutograd guard;
  return op.call(std::forward<Args>(args)...);
}
// Whether a call with these inputs records a node.
template <class... Inputs>
bool records(const Inputs&... inputs) {
  return at::GradMode::is_enabled() && (inputs.requires_grad() || ...);
}
template <class... Inputs>
void refuse_tangents(const char* name, const Inputs&... inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(inputs._fw_grad(/*level=*/0).defined() || ...), name,
                              " has no forward-mode derivative");
}

}  // namespace
