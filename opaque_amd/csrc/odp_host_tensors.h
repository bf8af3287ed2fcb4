// What the host helpers' operator calls share: types, streams, rows, and what
// autograd may and may not do with their nodes.  No device code.
#pragma once

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <memory>
#include <string>

#include "../../include/opaque_dp.h"

namespace odp_host {

inline int code_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return ODP_DTYPE_F32;
    case at::kBFloat16: return ODP_DTYPE_BF16;
    case at::kHalf: return ODP_DTYPE_F16;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t.scalar_type());
  }
}

inline odp_stream_t stream_of(const at::Tensor& t) {
  return reinterpret_cast<odp_stream_t>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream());
}

inline at::Tensor bytes_on(const at::Tensor& t, int64_t n) { return at::empty({n}, t.options().dtype(at::kByte)); }
inline int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// What the memory holds is the tensor's values (a view of a conjugate's imaginary part has theirs negated).
inline at::Tensor plain(const at::Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// Rows with unit column stride and a pitch of at least the width, copied if laid out otherwise.
inline at::Tensor pitched(const at::Tensor& given) {
  const at::Tensor t = plain(given);
  at::Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  if ((r.stride(1) != 1 && r.size(1) > 1) || r.stride(0) < r.size(1)) r = r.clone(at::MemoryFormat::Contiguous);
  return r;
}

// The same as the kernels take them; a contiguous tensor of any dimensions as it
// is, without the 1.5 us of a view.
struct Rows {
  at::Tensor held;
  const void* at = nullptr;
  int64_t n = 0, width = 0, pitch = 0;
  Rows() = default;
  explicit Rows(const at::Tensor& t) : width(t.size(-1)) {
    const bool whole = t.is_contiguous() && !t.is_neg();
    held = whole ? t : pitched(t);
    n = t.numel() / width;
    pitch = whole ? width : held.stride(0);
    at = held.data_ptr();
  }
};

// A tangent on an input would be dropped without a word: the kernels read values.
inline void no_tangent(const at::Tensor& t, const char* who) {
  TORCH_CHECK(!t._fw_grad(0).defined(), who, " have no forward-mode derivative");
}

// Gradients that is_grads_batched brings are a batch without an address.
inline constexpr c10::DispatchKeySet kBatched{c10::DispatchKey::Batched, c10::DispatchKey::FuncTorchBatched};
inline void no_batch(at::TensorList gs, const char* who) {
  for (const at::Tensor& g : gs)
    TORCH_CHECK(!g.defined() || !g.key_set().has_any(kBatched), who,
                " take no gradients batched by is_grads_batched (or vectorize=True): torch.func's transforms run");
}

// Ties a first derivative to what it depends on, so that asking for a second
// one is an error instead of zero: to the gradients gs it came from and, with
// `inputs`, to the inputs of the node whose backward pass calls this (by
// their edges: their values need not be kept).
inline at::Tensor first_only(at::TensorList gs, at::Tensor d, bool inputs, const char* who) {
  if (!d.defined() || !at::GradMode::is_enabled()) return d;
  torch::autograd::edge_list on;
  if (inputs)
    for (const auto& e : torch::autograd::get_current_node()->next_edges())
      if (e.is_valid()) on.push_back(e);
  for (const at::Tensor& g : gs)
    if (g.defined() && g.requires_grad()) on.push_back(torch::autograd::impl::gradient_edge(g));
  if (on.empty()) return d;
  const auto error = std::make_shared<torch::autograd::Error>(std::string(who) + " have no second derivative",
                                                              std::move(on));
  d = d.detach();
  torch::autograd::set_history(d, error);
  return d;
}

// What comes back from autograd is what was saved, wherever its hooks had it
// meanwhile: the kernels take addresses.
inline void as_saved(const at::Tensor& t, const at::Tensor& like, at::ScalarType type, at::IntArrayRef shape,
                     const char* who) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == type && t.sizes() == shape, who,
              ": a saved tensor came back as ", t.scalar_type(), " ", t.sizes(), " on ", t.device(), ", not as ", type,
              " ", shape, " on ", like.device());
}
inline at::Tensor whole(const at::Tensor& t, const at::Tensor& like, at::ScalarType type, at::IntArrayRef shape,
                        const char* who) {
  as_saved(t, like, type, shape, who);
  return t.contiguous();
}

}  // namespace odp_host
