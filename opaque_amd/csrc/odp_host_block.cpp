// The calls of the operators around a block's linears (the root-mean-square
// norm, routing) and of the tree norm outside torch.func, on the host:
// arguments to addresses, workspaces, and the autograd nodes.  No device code;
// the work is the C entry points of libopaque_dp.so, bound by address.
#include <map>
#include <unordered_map>

#include "odp_host_tensors.h"

namespace py = pybind11;

namespace {

using odp_host::bytes_on;
using odp_host::code_of;
using odp_host::pitched;
using odp_host::stream_of;

struct Abi {
  decltype(&odp_last_error) last_error = nullptr;
  decltype(&odp_rms_norm) rms_norm = nullptr;
  decltype(&odp_rms_norm_grad_scratch) rms_norm_grad_scratch = nullptr;
  decltype(&odp_rms_norm_grad) rms_norm_grad = nullptr;
  decltype(&odp_route) route = nullptr;
  decltype(&odp_route_grad) route_grad = nullptr;
  decltype(&odp_tree_norm_scratch) tree_norm_scratch = nullptr;
  decltype(&odp_tree_norm) tree_norm = nullptr;
};
Abi abi;

void bind(const std::unordered_map<std::string, uintptr_t>& at) {
  Abi b;
#define ODP_BIND(name) b.name = reinterpret_cast<decltype(b.name)>(at.at("odp_" #name))
  ODP_BIND(last_error);
  ODP_BIND(rms_norm);
  ODP_BIND(rms_norm_grad_scratch);
  ODP_BIND(rms_norm_grad);
  ODP_BIND(route);
  ODP_BIND(route_grad);
  ODP_BIND(tree_norm_scratch);
  ODP_BIND(tree_norm);
#undef ODP_BIND
  abi = b;
}

void check(int rc, const char* what) { TORCH_CHECK(rc == ODP_OK, what, " failed with status ", rc, ": ", abi.last_error()); }

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<at::Tensor>;

bool wants_grad(const Maybe& t) { return t.has_value() && t->requires_grad(); }

// ---------------------------------------------------------------------------
// Root-mean-square norm
// ---------------------------------------------------------------------------

constexpr const char* kNorms = "the norm operators";

// Gains [width] (one for all rows) or [gains][width] (one for each group of rows).
struct Gain {
  at::Tensor t;  // held while the launch is made
  const void* at = nullptr;
  int64_t pitch = 0, count = 1;
  int dt;
  Gain(const Maybe& w, int rows_dt) : dt(rows_dt) {
    if (!w.has_value()) return;
    t = *w;
    dt = code_of(t);
    if (t.dim() == 1) {
      t = t.contiguous();
    } else {
      count = t.size(0);
      if (t.stride(0) != 0 || (t.stride(1) != 1 && t.size(1) > 1)) t = pitched(t), pitch = t.stride(0);
    }
    at = t.data_ptr();
  }
};

struct Normed {
  at::Tensor y, h, rstd, scales;
};

// quant: 0 none, 1 a scale per row, 2 per 128 columns.
Normed norm_forward(const at::Tensor& x, const Maybe& residual, const Maybe& weight, double eps, double offset,
                    bool keep, int64_t quant) {
  const c10::OptionalDeviceGuard guard(x.device());
  const at::Tensor rows = pitched(x), r = residual.has_value() ? pitched(*residual) : at::Tensor();
  const int dt = code_of(rows), ht = r.defined() ? code_of(r) : dt;
  const int64_t n = rows.size(0), width = rows.size(1);
  const Gain g(weight, dt);
  Normed out;
  out.y = at::empty(x.sizes(), quant ? rows.options().dtype(at::kFloat8_e4m3fn) : rows.options());
  if (r.defined()) out.h = at::empty(x.sizes(), r.options());
  const auto f32 = rows.options().dtype(at::kFloat);
  std::vector<int64_t> shape(x.sizes().vec());
  shape.pop_back();
  if (keep) out.rstd = at::empty(shape, f32);
  if (quant) {
    if (quant == 2) shape.push_back((width + 127) / 128);
    out.scales = at::empty(shape, f32);
  }
  check(abi.rms_norm(stream_of(rows), dt, ht, g.dt, rows.data_ptr(), rows.stride(0), r.defined() ? r.data_ptr() : nullptr,
                     r.defined() ? r.stride(0) : 0, n, width, g.at, g.pitch, g.count, (float)eps, (float)offset,
                     (int)quant, out.y.data_ptr(), r.defined() ? out.h.data_ptr() : nullptr,
                     keep ? (float*)out.rstd.data_ptr() : nullptr, quant ? (float*)out.scales.data_ptr() : nullptr),
        "odp_rms_norm");
  return out;
}

struct Norm : torch::autograd::Function<Norm> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const Maybe& residual, const Maybe& weight,
                               double eps, double offset) {
    Normed o = norm_forward(x, residual, weight, eps, offset, true, 0);
    const at::Tensor& h = residual.has_value() ? o.h : x;
    ctx->save_for_backward({h, o.rstd, weight.has_value() ? *weight : at::Tensor()});
    ctx->set_materialize_grads(false);
    auto& d = ctx->saved_data;
    d["residual"] = residual.has_value();
    d["weight"] = weight.has_value();
    d["offset"] = offset;
    d["shape"] = x.sizes().vec();
    d["x"] = (int64_t)x.scalar_type();
    d["h"] = (int64_t)h.scalar_type();
    if (weight.has_value()) {
      d["w"] = (int64_t)weight->scalar_type();
      d["w_shape"] = weight->sizes().vec();
    }
    ctx->mark_non_differentiable({o.rstd});
    return residual.has_value() ? variable_list{o.y, o.rstd, o.h} : variable_list{o.y, o.rstd};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    auto& sd = ctx->saved_data;
    const bool has_r = sd["residual"].toBool(), has_w = sd["weight"].toBool();
    const at::Tensor gh0 = has_r ? grads[2] : at::Tensor();
    if (!grads[0].defined() && !gh0.defined()) return {{}, {}, {}, {}, {}};
    const variable_list saved = ctx->get_saved_variables();
    const bool need_x = ctx->needs_input_grad(0), need_r = has_r && ctx->needs_input_grad(1);
    const bool need_w = has_w && ctx->needs_input_grad(has_r ? 2 : 1);
    at::Tensor dx, dr, dw;
    {
      at::NoGradGuard no_grad;
      const at::Tensor& like = grads[0].defined() ? grads[0] : gh0;
      const c10::OptionalDeviceGuard guard(like.device());
      const auto shape = sd["shape"].toIntVector();
      const auto xt = (at::ScalarType)sd["x"].toInt(), ht = (at::ScalarType)sd["h"].toInt();
      odp_host::as_saved(saved[0], like, ht, shape, kNorms);
      const at::Tensor h = pitched(saved[0]);
      const int64_t n = h.size(0), width = h.size(1);
      const at::Tensor rstd = odp_host::whole(saved[1].reshape({-1}), like, at::kFloat, {n}, kNorms);
      Maybe w;
      if (has_w) {
        odp_host::as_saved(saved[2], like, (at::ScalarType)sd["w"].toInt(), sd["w_shape"].toIntVector(), kNorms);
        w = saved[2];
      }
      const Gain g(w, code_of(at::empty({0}, h.options().dtype(xt))));
      const at::Tensor gy = grads[0].defined() ? pitched(grads[0]) : at::zeros({n, width}, h.options().dtype(xt));
      const at::Tensor gh = gh0.defined() ? pitched(gh0) : at::Tensor();
      const bool same = xt == ht;
      if (need_x || need_r) dx = at::empty(shape, gy.options());
      if (need_r && !same) dr = at::empty(shape, h.options());
      if (need_w) {
        dw = n > 0 ? at::empty(w->sizes(), w->options()) : at::zeros(w->sizes(), w->options());
      }
      const int64_t words = need_w ? abi.rms_norm_grad_scratch(n, width, g.count) : 0;
      const at::Tensor work = words > 0 ? bytes_on(h, words) : at::Tensor();
      check(abi.rms_norm_grad(stream_of(h), code_of(gy), code_of(h), g.dt, h.data_ptr(), h.stride(0),
                              (const float*)rstd.data_ptr(), gy.data_ptr(), gy.stride(0),
                              gh.defined() ? gh.data_ptr() : nullptr, gh.defined() ? gh.stride(0) : 0, n, width, g.at,
                              g.pitch, g.count, (float)sd["offset"].toDouble(),
                              work.defined() ? work.data_ptr() : nullptr, dx.defined() ? dx.data_ptr() : nullptr,
                              dr.defined() ? dr.data_ptr() : nullptr, dw.defined() ? dw.data_ptr() : nullptr),
            "odp_rms_norm_grad");
      if (need_r && same) dr = dx;
      if (!need_x) dx = at::Tensor();
    }
    dw = odp_host::first_only(grads, dw, true, kNorms);
    const bool shared = dx.defined() && dr.defined() && dx.is_same(dr);
    dx = odp_host::first_only(grads, dx, true, kNorms);
    dr = shared ? dx : odp_host::first_only(grads, dr, true, kNorms);
    return {dx, dr, dw, {}, {}};
  }
};

// (y, 1 / sqrt(..)) or, with a residual, (y, 1 / sqrt(..), the sum); without `keep` the second may be undefined.
variable_list normed(const at::Tensor& x, const Maybe& residual, const Maybe& weight, double eps, double offset,
                     bool keep) {
  odp_host::no_tangent(x, kNorms);
  if (residual.has_value()) odp_host::no_tangent(*residual, kNorms);
  if (weight.has_value()) odp_host::no_tangent(*weight, kNorms);
  if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(residual) || wants_grad(weight)))
    return Norm::apply(x, residual, weight, eps, offset);
  const Normed o = norm_forward(x, residual, weight, eps, offset, keep, 0);
  return residual.has_value() ? variable_list{o.y, o.rstd, o.h} : variable_list{o.y, o.rstd};
}

// (y,) or, with a residual, (y, the sum).
variable_list rms_norm(const at::Tensor& x, const Maybe& residual, const Maybe& weight, double eps, double offset) {
  py::gil_scoped_release nogil;
  variable_list out = normed(x, residual, weight, eps, offset, false);
  out.erase(out.begin() + 1);
  return out;
}

// With what the backward pass takes of the rows: for a rule of torch.func, which may have transforms above it.
variable_list rms_norm_kept(const at::Tensor& x, const Maybe& residual, const Maybe& weight, double eps,
                            double offset) {
  py::gil_scoped_release nogil;
  return normed(x, residual, weight, eps, offset, true);
}

// (q, scales) or, with a residual, (q, scales, the sum).
variable_list rms_norm_quantized(const at::Tensor& x, const Maybe& residual, const Maybe& weight, double eps,
                                 double offset, int64_t quant) {
  py::gil_scoped_release nogil;
  at::NoGradGuard no_grad;
  const Normed o = norm_forward(x, residual, weight, eps, offset, false, quant);
  return residual.has_value() ? variable_list{o.y, o.scales, o.h} : variable_list{o.y, o.scales};
}

// ---------------------------------------------------------------------------
// Routing
// ---------------------------------------------------------------------------

constexpr const char* kRoutes = "the routing operator";

struct Options {
  bool sigmoid;
  int64_t groups, top_groups, best, top_k;
  bool renorm;
  double scale;
};

std::pair<at::Tensor, at::Tensor> route_forward(const at::Tensor& z, const Maybe& bias, const Options& o) {
  const c10::OptionalDeviceGuard guard(z.device());
  const at::Tensor rows = pitched(z), b = bias.has_value() ? bias->contiguous() : at::Tensor();
  std::vector<int64_t> shape(z.sizes().vec());
  shape.back() = o.top_k;
  const at::Tensor index = at::empty(shape, rows.options().dtype(at::kLong));
  const at::Tensor weights = at::empty(shape, rows.options().dtype(at::kFloat));
  check(abi.route(stream_of(rows), code_of(rows), rows.data_ptr(), rows.stride(0), rows.size(0), rows.size(1),
                  (int)o.sigmoid, b.defined() ? (const float*)b.data_ptr() : nullptr,
                  b.defined() && b.dim() == 2 ? b.size(0) : 1, o.groups, o.top_groups, (int)o.best, o.top_k,
                  (int)o.renorm, (float)o.scale, (int64_t*)index.data_ptr(), (float*)weights.data_ptr()),
        "odp_route");
  return {index, weights};
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& z, const Maybe& bias, const Options& o) {
    const auto out = route_forward(z, bias, o);
    ctx->mark_non_differentiable({out.first});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({z, out.first});
    auto& d = ctx->saved_data;
    d["sigmoid"] = o.sigmoid;
    d["renorm"] = o.renorm;
    d["scale"] = o.scale;
    d["top_k"] = o.top_k;
    d["type"] = (int64_t)z.scalar_type();
    d["shape"] = z.sizes().vec();
    return {out.first, out.second};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[1].defined() || !ctx->needs_input_grad(0)) return {{}, {}, {}};
    at::Tensor dz;
    {
      at::NoGradGuard no_grad;
      const at::Tensor& gw = grads[1];
      const c10::OptionalDeviceGuard guard(gw.device());
      auto& sd = ctx->saved_data;
      auto shape = sd["shape"].toIntVector();
      const variable_list saved = ctx->get_saved_variables();
      odp_host::as_saved(saved[0], gw, (at::ScalarType)sd["type"].toInt(), shape, kRoutes);
      const at::Tensor rows = pitched(saved[0]);
      const int64_t top_k = sd["top_k"].toInt();
      dz = at::empty(shape, rows.options());
      shape.back() = top_k;
      const at::Tensor index = odp_host::whole(saved[1], gw, at::kLong, shape, kRoutes);
      const at::Tensor g = gw.contiguous();
      check(abi.route_grad(stream_of(rows), code_of(rows), rows.data_ptr(), rows.stride(0), rows.size(0), rows.size(1),
                           (int)sd["sigmoid"].toBool(), top_k, (int)sd["renorm"].toBool(), (float)sd["scale"].toDouble(),
                           (const int64_t*)index.data_ptr(), (const float*)g.data_ptr(), top_k, dz.data_ptr()),
            "odp_route_grad");
    }
    return {odp_host::first_only(grads, dz, true, kRoutes), {}, {}};
  }
};

std::pair<at::Tensor, at::Tensor> route(const at::Tensor& z, const Maybe& bias, bool sigmoid, int64_t groups,
                                        int64_t top_groups, int64_t best, int64_t top_k, bool renorm, double scale) {
  py::gil_scoped_release nogil;
  odp_host::no_tangent(z, kRoutes);
  const Options o{sigmoid, groups, top_groups, best, top_k, renorm, scale};
  if (at::GradMode::is_enabled() && z.requires_grad()) {
    const variable_list out = Route::apply(z, bias, o);
    return {out[0], out[1]};
  }
  return route_forward(z, bias, o);
}

// ---------------------------------------------------------------------------
// Norm of a tree
// ---------------------------------------------------------------------------

int tree_code(const at::Tensor& t) { return t.scalar_type() == at::kDouble ? ODP_DTYPE_F64 : code_of(t); }

// The leaves scaled (with `clip`; else none) and their norm.  The scaled ones
// lie in one buffer per type, with the leaves' own strides where those leave no
// gaps.
std::pair<std::vector<at::Tensor>, at::Tensor> tree_norm(const std::vector<at::Tensor>& leaves, bool clip,
                                                         double max_norm, bool wide) {
  py::gil_scoped_release nogil;
  at::NoGradGuard no_grad;
  const c10::OptionalDeviceGuard guard(leaves.at(0).device());
  constexpr int64_t kAlign = 64;
  std::vector<at::Tensor> src(leaves.size()), out;
  std::map<at::ScalarType, std::pair<int64_t, at::Tensor>> buffers;
  std::vector<int64_t> at_(leaves.size()), table(leaves.size() * ODP_TN_FIELDS);
  for (size_t i = 0; i < leaves.size(); ++i) {
    const at::Tensor& t = leaves[i];
    src[i] = t.is_non_overlapping_and_dense() ? t : t.contiguous();
    auto& b = buffers[t.scalar_type()];
    at_[i] = b.first;
    b.first += (t.numel() + kAlign - 1) / kAlign * kAlign;
  }
  if (clip)
    for (auto& b : buffers) b.second.second = at::empty({b.second.first}, leaves[0].options().dtype(b.first));
  for (size_t i = 0; i < leaves.size(); ++i) {
    const at::Tensor& t = src[i];
    int64_t* row = table.data() + i * ODP_TN_FIELDS;
    row[ODP_TN_SRC] = reinterpret_cast<int64_t>(t.const_data_ptr());
    row[ODP_TN_N] = t.numel();
    row[ODP_TN_DTYPE] = tree_code(t);
    row[ODP_TN_DST] = 0;
    if (!clip) continue;
    const at::Tensor& b = buffers[t.scalar_type()].second;
    // A tensor over its buffer's storage, made directly (no dispatch, no view record: the leaves are outputs).
    at::Tensor o = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(b.storage()), b.key_set(), b.dtype());
    o.unsafeGetTensorImpl()->set_sizes_and_strides(t.sizes(), t.strides(), at_[i]);
    row[ODP_TN_DST] = reinterpret_cast<int64_t>(b.data_ptr()) + at_[i] * (int64_t)b.element_size();
    out.push_back(std::move(o));
  }
  const at::Tensor norm = at::empty({}, leaves[0].options().dtype(wide ? at::kDouble : at::kFloat));
  const at::Tensor work = bytes_on(leaves[0], abi.tree_norm_scratch((int64_t)leaves.size()));
  check(abi.tree_norm(stream_of(leaves[0]), table.data(), (int64_t)leaves.size(), (int)clip, max_norm, (int)wide,
                      work.data_ptr(), norm.data_ptr()),
        "odp_tree_norm");
  return {out, norm};
}

}  // namespace

void add_block(py::module_& m) {
  m.def("bind_block", &bind, py::arg("entry_points"));
  m.def("rms_norm", &rms_norm, py::arg("x"), py::arg("residual"), py::arg("weight"), py::arg("eps"), py::arg("offset"));
  m.def("rms_norm_kept", &rms_norm_kept, py::arg("x"), py::arg("residual"), py::arg("weight"), py::arg("eps"),
        py::arg("offset"));
  m.def("rms_norm_quantized", &rms_norm_quantized, py::arg("x"), py::arg("residual"), py::arg("weight"),
        py::arg("eps"), py::arg("offset"), py::arg("quant"));
  m.def("route", &route, py::arg("z"), py::arg("bias"), py::arg("sigmoid"), py::arg("groups"), py::arg("top_groups"),
        py::arg("best"), py::arg("top_k"), py::arg("renorm"), py::arg("scale"));
  m.def("tree_norm", &tree_norm, py::arg("leaves"), py::arg("clip"), py::arg("max_norm"), py::arg("wide"));
}
