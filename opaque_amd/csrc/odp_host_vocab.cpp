// The vocabulary operators' calls outside torch.func, on the host: arguments
// to addresses, workspaces, and the autograd nodes.  No device code; the work
// is the C entry points of libopaque_dp.so, bound by address.
//
// The same calls in Python cost 100 us (a lookup and its gradient) to 180 us
// (a loss and its gradients) of host time, most of it in the backward pass,
// whose thread takes the interpreter lock; small batches are bound by that.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <atomic>
#include <memory>
#include <string>
#include <unordered_map>

#include "../../include/opaque_dp.h"

namespace py = pybind11;

namespace {

// The bound entry points.
struct Abi {
  decltype(&odp_last_error) last_error = nullptr;
  decltype(&odp_embed_rows) embed_rows = nullptr;
  decltype(&odp_token_sort_scratch) token_sort_scratch = nullptr;
  decltype(&odp_token_sort) token_sort = nullptr;
  decltype(&odp_embed_sum_scratch) embed_sum_scratch = nullptr;
  decltype(&odp_embed_grad) embed_grad = nullptr;
  decltype(&odp_xent_rows) xent_rows = nullptr;
  decltype(&odp_xent_stats_scratch) xent_stats_scratch = nullptr;
  decltype(&odp_xent_kept) xent_kept = nullptr;
  decltype(&odp_xent_losses) xent_losses = nullptr;
  decltype(&odp_xent_reduce) xent_reduce = nullptr;
  decltype(&odp_xent_pitch) xent_pitch = nullptr;
  decltype(&odp_xent_dlogits) xent_dlogits = nullptr;
  decltype(&odp_xent_dx_scratch) xent_dx_scratch = nullptr;
  decltype(&odp_xent_dx) xent_dx = nullptr;
  decltype(&odp_xent_dx_rows) xent_dx_rows = nullptr;
  decltype(&odp_xent_dw_scratch) xent_dw_scratch = nullptr;
  decltype(&odp_xent_dw) xent_dw = nullptr;
};
Abi abi;

void bind(const std::unordered_map<std::string, uintptr_t>& at) {
  Abi b;
#define ODP_BIND(name) b.name = reinterpret_cast<decltype(b.name)>(at.at("odp_" #name))
  ODP_BIND(last_error);
  ODP_BIND(embed_rows);
  ODP_BIND(token_sort_scratch);
  ODP_BIND(token_sort);
  ODP_BIND(embed_sum_scratch);
  ODP_BIND(embed_grad);
  ODP_BIND(xent_rows);
  ODP_BIND(xent_stats_scratch);
  ODP_BIND(xent_kept);
  ODP_BIND(xent_losses);
  ODP_BIND(xent_reduce);
  ODP_BIND(xent_pitch);
  ODP_BIND(xent_dlogits);
  ODP_BIND(xent_dx_scratch);
  ODP_BIND(xent_dx);
  ODP_BIND(xent_dx_rows);
  ODP_BIND(xent_dw_scratch);
  ODP_BIND(xent_dw);
#undef ODP_BIND
  abi = b;
}

void check(int rc, const char* what) { TORCH_CHECK(rc == ODP_OK, what, " failed with status ", rc, ": ", abi.last_error()); }

int code_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return ODP_DTYPE_F32;
    case at::kBFloat16: return ODP_DTYPE_BF16;
    case at::kHalf: return ODP_DTYPE_F16;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t.scalar_type());
  }
}

odp_stream_t stream_of(const at::Tensor& t) {
  return reinterpret_cast<odp_stream_t>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream());
}

at::Tensor bytes_on(const at::Tensor& t, int64_t n) { return at::empty({n}, t.options().dtype(at::kByte)); }
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// Rows with unit column stride and a pitch of at least the width, copied if laid out otherwise.
at::Tensor pitched(const at::Tensor& t) {
  at::Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  if ((r.stride(1) != 1 && r.size(1) > 1) || r.stride(0) < r.size(1)) r = r.clone(at::MemoryFormat::Contiguous);
  return r;
}

// A tangent on an input would be dropped without a word: the kernels read values.
void no_tangent(const at::Tensor& t) {
  TORCH_CHECK(!t._fw_grad(0).defined(), "the vocabulary operators have no forward-mode derivative");
}

// Ties a first derivative to what it depends on, so that asking for a second
// one is an error instead of zero: to the gradient g it came from and, with
// `inputs`, to the inputs of the node whose backward pass calls this (by
// their edges: their values need not be kept).
at::Tensor first_only(const at::Tensor& g, at::Tensor d, bool inputs) {
  if (!d.defined() || !at::GradMode::is_enabled()) return d;
  torch::autograd::edge_list on;
  if (inputs)
    for (const auto& e : torch::autograd::get_current_node()->next_edges())
      if (e.is_valid()) on.push_back(e);
  if (g.requires_grad()) on.push_back(torch::autograd::impl::gradient_edge(g));
  if (on.empty()) return d;
  const auto error = std::make_shared<torch::autograd::Error>(
      "the vocabulary operators have no second derivative", std::move(on));
  d = d.detach();
  torch::autograd::set_history(d, error);
  return d;
}

// What comes back from autograd is what was saved, wherever its hooks had it
// meanwhile: the kernels take addresses.
void as_saved(const at::Tensor& t, const at::Tensor& like, at::ScalarType type, at::IntArrayRef shape) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == type && t.sizes() == shape,
              "vocabulary operators: a saved tensor came back as ", t.scalar_type(), " ", t.sizes(), " on ", t.device(),
              ", not as ", type, " ", shape, " on ", like.device());
}
at::Tensor whole(const at::Tensor& t, const at::Tensor& like, at::ScalarType type, at::IntArrayRef shape) {
  as_saved(t, like, type, shape);
  return t.contiguous();
}

// ---------------------------------------------------------------------------
// Embedding
// ---------------------------------------------------------------------------

at::Tensor embed_rows(const at::Tensor& tokens, const at::Tensor& weight, double scale) {
  const c10::OptionalDeviceGuard guard(weight.device());
  const at::Tensor w = pitched(weight), y = tokens.contiguous();
  std::vector<int64_t> shape(tokens.sizes().vec());
  shape.push_back(w.size(1));
  at::Tensor out = at::empty(shape, w.options());
  check(abi.embed_rows(stream_of(w), code_of(w), y.data_ptr(), (int)y.element_size(), y.numel(), w.data_ptr(),
                       w.stride(0), w.size(0), w.size(1), (float)scale, out.data_ptr()),
        "odp_embed_rows");
  return out;
}

struct Embed : torch::autograd::Function<Embed> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& tokens, const at::Tensor& weight,
                            double scale, int64_t padding) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["tokens"] = tokens.sizes().vec();
    ctx->saved_data["wide"] = tokens.scalar_type() == at::kLong;
    return embed_rows(tokens, weight, scale);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    if (!ctx->needs_input_grad(1) || !grads[0].defined()) return {{}, {}, {}, {}};
    at::Tensor dw;
    {
      at::NoGradGuard no_grad;
      const c10::OptionalDeviceGuard guard(grads[0].device());
      const at::Tensor g = pitched(grads[0]);
      const at::Tensor y = whole(ctx->get_saved_variables()[0], g, ctx->saved_data["wide"].toBool() ? at::kLong : at::kInt,
                                 ctx->saved_data["tokens"].toIntVector());
      const int64_t n = y.numel(), width = g.size(1), vocab = ctx->saved_data["vocab"].toInt();
      const int dt = code_of(g);
      dw = at::empty({vocab, width}, g.options());
      const int64_t scratch = up16(std::max(abi.token_sort_scratch(n, vocab), abi.embed_sum_scratch(dt, n, width, 0)));
      const at::Tensor work = bytes_on(g, scratch + 8 * n);
      char* at = (char*)work.data_ptr();
      uint32_t* keys = (uint32_t*)(at + scratch);
      const odp_stream_t s = stream_of(g);
      check(abi.token_sort(s, y.data_ptr(), (int)y.element_size(), n, vocab, ctx->saved_data["padding"].toInt(),
                           nullptr, nullptr, 0, at, keys, keys + n, nullptr, dw.data_ptr(), (int64_t)dw.nbytes()),
            "odp_token_sort");
      check(abi.embed_grad(s, dt, g.data_ptr(), g.stride(0), n, width, keys, keys + n, vocab,
                           (float)ctx->saved_data["scale"].toDouble(), at, dw.data_ptr()),
            "odp_embed_grad");
    }
    return {{}, first_only(grads[0], dw, false), {}, {}};
  }
};

at::Tensor embedding(const at::Tensor& tokens, const at::Tensor& weight, double scale, int64_t padding) {
  py::gil_scoped_release nogil;
  no_tangent(weight);
  if (at::GradMode::is_enabled() && weight.requires_grad()) return Embed::apply(tokens, weight, scale, padding);
  return embed_rows(tokens, weight, scale);
}

// ---------------------------------------------------------------------------
// Linear cross entropy
// ---------------------------------------------------------------------------

// The head with rows on the 16-byte grid, less than ODP_XENT_WIDE apart: itself, or a copy padded with zero columns.
at::Tensor head_rows(const at::Tensor& weight) {
  at::Tensor w = pitched(weight);
  const int64_t per = 16 / w.element_size();
  if (w.size(1) % per == 0 && w.stride(0) % per == 0 && w.stride(0) < ODP_XENT_WIDE &&
      reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0)
    return w;
  at::Tensor wide = at::zeros({w.size(0), (w.size(1) + per - 1) / per * per}, w.options());
  wide.narrow(1, 0, w.size(1)).copy_(w);
  return wide;
}

// The packed rows of a call (odp_xent_rows) and what its backward needs.
struct Packed {
  at::Tensor w, xc, ids, losses, stat, logits;  // logits: where they are kept
  int64_t n, cols, width, vocab;
  int dt;
  int32_t* count() const { return (int32_t*)ids.data_ptr(); }
  float* counted() const { return (float*)count() + 1; }
  int32_t* act() const { return count() + 2; }
  int32_t* tgt() const { return act() + std::max<int64_t>(n, 1); }
  int32_t* where() const { return tgt() + std::max<int64_t>(n, 1); }
  float* kept() const { return logits.defined() ? (float*)logits.data_ptr() : nullptr; }
  int64_t kept_pitch() const { return abi.xent_pitch(dt, vocab); }
};

// Kept logits of `bytes` bytes, or an undefined tensor where those of all
// losses that live would pass `most` together.
std::atomic<int64_t> kept_bytes{0};
at::Tensor keep_logits(at::IntArrayRef shape, const at::TensorOptions& options, int64_t bytes, int64_t most) {
  const int64_t before = kept_bytes.fetch_add(bytes);
  const auto share = std::shared_ptr<void>(nullptr, [bytes](void*) { kept_bytes.fetch_sub(bytes); });
  if (before > most - bytes) return {};
  const at::Tensor own = at::empty(shape, options);
  return at::for_blob(own.data_ptr(), shape)
      .deleter([own, share](void*) {})
      .options(options)
      .target_device(own.device())
      .make_tensor();
}

// The rows' statistics go to stat_out.  keep_bytes: up to which the logits of
// all live losses are kept for their backward passes.
Packed xent_forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& target,
                    const at::Tensor& stat_out, double softcap, int64_t ignore, int64_t keep_bytes) {
  Packed p;
  p.w = head_rows(weight);
  const at::Tensor rows = pitched(x), y = target.contiguous();
  p.n = y.numel();
  p.cols = rows.size(1);
  p.width = p.w.size(1);
  p.vocab = p.w.size(0);
  p.dt = code_of(rows);
  const int64_t room = std::max<int64_t>(p.n, 1);
  p.xc = at::empty({room, p.width}, rows.options());
  p.ids = at::empty({3 * room + 2}, rows.options().dtype(at::kInt));
  p.losses = at::empty(target.sizes(), rows.options().dtype(at::kFloat));
  p.stat = stat_out;
  float* losses = (float*)p.losses.data_ptr();
  float* stat = (float*)p.stat.data_ptr();
  const odp_stream_t s = stream_of(rows);
  check(abi.xent_rows(s, p.dt, rows.data_ptr(), rows.stride(0), p.n, p.cols, p.width, y.data_ptr(),
                      (int)y.element_size(), p.vocab, ignore, 0, p.xc.data_ptr(), p.act(), p.tgt(), p.where(),
                      p.count(), losses, stat),
        "odp_xent_rows");
  const int64_t kept = abi.xent_kept(p.dt, p.n, p.width, p.vocab);
  if (kept > 0 && kept <= keep_bytes)
    p.logits = keep_logits({p.n, p.kept_pitch()}, p.losses.options(), kept, keep_bytes);
  const at::Tensor work = bytes_on(rows, abi.xent_stats_scratch(p.dt, p.n, p.vocab));
  check(abi.xent_losses(s, p.dt, p.xc.data_ptr(), p.n, p.width, p.act(), p.tgt(), p.count(), p.w.data_ptr(),
                        p.w.stride(0), p.vocab, (float)softcap, work.data_ptr(), losses, stat, p.kept(), p.kept_pitch()),
        "odp_xent_losses");
  return p;
}

// reduction: 0 none, 1 sum, 2 mean.
at::Tensor xent_result(const Packed& p, int64_t reduction) {
  if (reduction == 0) return p.losses;
  at::Tensor out = at::empty({}, p.losses.options());
  check(abi.xent_reduce(stream_of(p.xc), (const float*)p.losses.data_ptr(), p.n, reduction == 2 ? p.counted() : nullptr,
                        (float*)out.data_ptr()),
        "odp_xent_reduce");
  return out;
}

struct Xent : torch::autograd::Function<Xent> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                            const at::Tensor& target, const at::Tensor& stat, double softcap, int64_t ignore,
                            int64_t reduction, int64_t piece_bytes, int64_t keep_bytes) {
    const c10::OptionalDeviceGuard guard(x.device());
    const Packed p = xent_forward(x, weight, target, stat, softcap, ignore, keep_bytes);
    // Saved as autograd's own are: a later change of the head in place is an error (where it was not copied), hooks
    // see every tensor, and all go when the backward pass is through.
    ctx->save_for_backward({p.w, p.xc, p.ids, p.stat, p.logits});
    auto& d = ctx->saved_data;
    d["n"] = p.n;
    d["dt"] = (int64_t)p.dt;
    d["vocab"] = p.vocab;
    d["width"] = p.width;
    d["cols"] = p.cols;
    d["softcap"] = softcap;
    d["mean"] = reduction == 2;
    d["piece_bytes"] = piece_bytes;
    d["x_shape"] = x.sizes().vec();
    return xent_result(p, reduction);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    at::Tensor dx, dw;
    if (!grads[0].defined()) return {{}, {}, {}, {}, {}, {}, {}, {}, {}};
    const torch::autograd::variable_list saved = ctx->get_saved_variables();
    {
      at::NoGradGuard no_grad;
      const c10::OptionalDeviceGuard guard(grads[0].device());
      auto& sd = ctx->saved_data;
      Packed p;
      p.n = sd["n"].toInt();
      p.cols = sd["cols"].toInt();
      p.width = sd["width"].toInt();
      p.vocab = sd["vocab"].toInt();
      p.dt = (int)sd["dt"].toInt();
      const at::ScalarType type = p.dt == ODP_DTYPE_F32 ? at::kFloat : at::kBFloat16;
      const int64_t room = std::max<int64_t>(p.n, 1);
      as_saved(saved[0], grads[0], type, {p.vocab, p.width});
      p.w = head_rows(saved[0]);
      p.xc = whole(saved[1], grads[0], type, {room, p.width});
      p.ids = whole(saved[2], grads[0], at::kInt, {3 * room + 2});
      p.stat = whole(saved[3].reshape({-1}), grads[0], at::kFloat, {p.n * ODP_XENT_STAT});
      if (saved[4].defined()) p.logits = whole(saved[4], grads[0], at::kFloat, {p.n, p.kept_pitch()});
      const float softcap = (float)sd["softcap"].toDouble();
      const at::Tensor g = grads[0].contiguous();
      const int stride = g.dim() > 0 ? 1 : 0;
      const float* over = sd["mean"].toBool() ? p.counted() : nullptr;
      const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
      const int64_t es = p.xc.element_size(), edge = abi.xent_pitch(p.dt, 1);
      const int64_t fit = std::min(sd["piece_bytes"].toInt() / (room * es) / edge * edge,
                                   ODP_XENT_PIECE - edge);
      const int64_t pieces = (p.vocab + std::max(fit, edge) - 1) / std::max(fit, edge);
      const int64_t piece = std::min(p.vocab, ((p.vocab + pieces - 1) / pieces + edge - 1) / edge * edge);
      const at::Tensor d = at::empty({room, abi.xent_pitch(p.dt, piece)}, p.xc.options());
      at::Tensor sums;
      if (need_x) {
        dx = at::empty(sd["x_shape"].toIntVector(), p.xc.options());
        sums = bytes_on(p.xc, abi.xent_dx_scratch(p.dt, p.n, p.width));
      }
      if (need_w) dw = at::empty({p.vocab, p.width}, p.xc.options());
      const at::Tensor rest = at::empty({room}, p.stat.options());
      const odp_stream_t s = stream_of(p.xc);
      for (int64_t v0 = 0; v0 < p.vocab; v0 += piece) {
        const int64_t vc = std::min(piece, p.vocab - v0), ldd = abi.xent_pitch(p.dt, vc);
        check(abi.xent_dlogits(s, p.dt, p.xc.data_ptr(), p.n, p.width, p.act(), p.tgt(), p.count(), p.w.data_ptr(),
                               p.w.stride(0), p.vocab, softcap, v0, vc, (const float*)p.stat.data_ptr(),
                               (const float*)g.data_ptr(), stride, over, p.kept(), p.kept_pitch(), d.data_ptr(), ldd,
                               (float*)rest.data_ptr()),
              "odp_xent_dlogits");
        if (need_x)
          check(abi.xent_dx(s, p.dt, p.n, p.width, p.count(), p.w.data_ptr(), p.w.stride(0), p.vocab, v0, vc, piece,
                            d.data_ptr(), ldd, sums.data_ptr()),
                "odp_xent_dx");
        if (need_w) {
          const int64_t split = abi.xent_dw_scratch(p.dt, p.n, vc, p.width);
          const at::Tensor slots = split > 0 ? bytes_on(p.xc, split) : at::Tensor();
          check(abi.xent_dw(s, p.dt, p.xc.data_ptr(), p.n, p.width, p.count(), vc, d.data_ptr(), ldd,
                            split > 0 ? slots.data_ptr() : nullptr, (char*)dw.data_ptr() + v0 * p.width * es, p.width),
                "odp_xent_dw");
        }
      }
      if (need_x)
        check(abi.xent_dx_rows(s, p.dt, p.n, p.cols, p.width, p.count(), p.where(), p.tgt(), p.w.data_ptr(),
                               p.w.stride(0), piece, sums.data_ptr(), (const float*)rest.data_ptr(), dx.data_ptr()),
              "odp_xent_dx_rows");
      if (need_w && p.cols != p.width) dw = dw.narrow(1, 0, p.cols).contiguous();
    }
    return {first_only(grads[0], dx, true), first_only(grads[0], dw, true), {}, {}, {}, {}, {}, {}, {}};
  }
};

at::Tensor xent(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& target, const at::Tensor& stat,
                double softcap, int64_t ignore, int64_t reduction, int64_t piece_bytes, int64_t keep_bytes) {
  no_tangent(x);
  no_tangent(weight);
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad()))
    return Xent::apply(x, weight, target, stat, softcap, ignore, reduction, piece_bytes, keep_bytes);
  const c10::OptionalDeviceGuard guard(x.device());
  return xent_result(xent_forward(x, weight, target, stat, softcap, ignore, 0), reduction);
}

at::Tensor stat_of(const at::Tensor& x, const at::Tensor& target) {
  std::vector<int64_t> shape(target.sizes().vec());
  shape.push_back(ODP_XENT_STAT);
  return at::empty(shape, x.options().dtype(at::kFloat).requires_grad(false));
}

at::Tensor cross_entropy(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& target, double softcap,
                         int64_t ignore, int64_t reduction, int64_t piece_bytes, int64_t keep_bytes) {
  py::gil_scoped_release nogil;
  return xent(x, weight, target, stat_of(x, target), softcap, ignore, reduction, piece_bytes, keep_bytes);
}

// The token losses and their rows' statistics, which have no gradient.
std::pair<at::Tensor, at::Tensor> token_losses(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& target,
                                               double softcap, int64_t ignore, int64_t piece_bytes,
                                               int64_t keep_bytes) {
  py::gil_scoped_release nogil;
  const at::Tensor stat = stat_of(x, target);
  return {xent(x, weight, target, stat, softcap, ignore, 0, piece_bytes, keep_bytes), stat};
}

}  // namespace

void add_vocabulary(py::module_& m) {
  m.def("bind", &bind, py::arg("entry_points"));
  m.def("embedding", &embedding, py::arg("tokens"), py::arg("weight"), py::arg("scale"), py::arg("padding"));
  m.def("cross_entropy", &cross_entropy, py::arg("x"), py::arg("weight"), py::arg("target"), py::arg("softcap"),
        py::arg("ignore"), py::arg("reduction"), py::arg("piece_bytes"), py::arg("keep_bytes"));
  m.def("token_losses", &token_losses, py::arg("x"), py::arg("weight"), py::arg("target"), py::arg("softcap"),
        py::arg("ignore"), py::arg("piece_bytes"), py::arg("keep_bytes"));
}
