// The calls of the operators around a block's linears (the root-mean-square
// norm, routing) and of the tree norm outside torch.func, on the host:
// arguments to addresses, workspaces, and the autograd nodes.  No device code;
// the work is the C entry points of libopaque_dp.so, bound by address.
#include <algorithm>
#include <map>
#include <unordered_map>

#include "odp_host_tensors.h"

namespace py = pybind11;

namespace {

using odp_host::bytes_on;
using odp_host::code_of;
using odp_host::pitched;
using odp_host::Rows;
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

using torch::autograd::SavedVariable;
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
    t = odp_host::plain(*w);
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

void no_tangents(const at::Tensor& x, const Maybe& residual, const Maybe& weight) {
  odp_host::no_tangent(x, kNorms);
  if (residual.has_value()) odp_host::no_tangent(*residual, kNorms);
  if (weight.has_value()) odp_host::no_tangent(*weight, kNorms);
}

// quant: 0 none, 1 a scale per row, 2 per 128 columns.
Normed norm_forward(const at::Tensor& x, const Maybe& residual, const Maybe& weight, double eps, double offset,
                    bool keep, int64_t quant) {
  const c10::OptionalDeviceGuard guard(x.device());
  const Rows rows(x), r = residual.has_value() ? Rows(*residual) : Rows();
  const int dt = code_of(x), ht = residual.has_value() ? code_of(*residual) : dt;
  const int64_t n = rows.n, width = rows.width;
  const Gain g(weight, dt);
  Normed out;
  const bool with = residual.has_value();
  out.y = at::empty(x.sizes(), quant ? x.options().dtype(at::kFloat8_e4m3fn) : x.options());
  if (with) out.h = at::empty(x.sizes(), residual->options());
  const auto f32 = x.options().dtype(at::kFloat);
  if (keep) out.rstd = at::empty(x.sizes().slice(0, x.dim() - 1), f32);
  if (quant) {
    std::vector<int64_t> shape(x.sizes().vec());
    shape.pop_back();
    if (quant == 2) shape.push_back((width + 127) / 128);
    out.scales = at::empty(shape, f32);
  }
  check(abi.rms_norm(stream_of(x), dt, ht, g.dt, rows.at, rows.pitch, r.at, r.pitch, n, width, g.at, g.pitch, g.count,
                     (float)eps, (float)offset, (int)quant, out.y.data_ptr(), with ? out.h.data_ptr() : nullptr,
                     keep ? (float*)out.rstd.data_ptr() : nullptr, quant ? (float*)out.scales.data_ptr() : nullptr),
        "odp_rms_norm");
  return out;
}

// Nodes of their own, with their fields as they are: torch's wrapper for
// custom functions keeps them in a map by name, which takes 8 us of a call.
struct NormNode final : torch::autograd::Node {
  SavedVariable h, rstd, w;
  bool has_r = false, has_w = false;
  double offset = 0.0;
  at::ScalarType xt, ht, wt;
  std::vector<int64_t> shape, w_shape;

  std::string name() const override { return "RmsNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    h.reset_data();
    rstd.reset_data();
    w.reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const at::Tensor& gy0 = grads[0];
    const at::Tensor gh0 = has_r ? grads[1] : at::Tensor();
    if (!gy0.defined() && !gh0.defined()) return variable_list(3);
    odp_host::no_batch(grads, kNorms);
    const at::Tensor h_ = h.unpack(has_r ? shared_from_this() : nullptr), rstd_ = rstd.unpack();
    const at::Tensor w_ = has_w ? w.unpack() : at::Tensor();
    const bool need_x = task_should_compute_output(0), need_r = task_should_compute_output(1);
    const bool need_w = task_should_compute_output(2);
    at::Tensor dx, dr, dw;
    {
      at::NoGradGuard no_grad;
      const at::Tensor& like = gy0.defined() ? gy0 : gh0;
      const c10::OptionalDeviceGuard guard(like.device());
      odp_host::as_saved(h_, like, ht, shape, kNorms);
      const Rows rows(h_);
      const int64_t n = rows.n, width = rows.width;
      odp_host::as_saved(rstd_, like, at::kFloat, at::IntArrayRef(shape).slice(0, shape.size() - 1), kNorms);
      const at::Tensor stat = rstd_.contiguous();
      if (has_w) odp_host::as_saved(w_, like, wt, w_shape, kNorms);
      const auto options = h_.options().dtype(xt);
      const Rows gy(gy0.defined() ? gy0 : at::zeros(shape, options)), gh = gh0.defined() ? Rows(gh0) : Rows();
      const Gain g(has_w ? Maybe(w_) : Maybe(), code_of(gy.held));
      const bool same = xt == ht;
      if (need_x || need_r) dx = at::empty(shape, options);
      if (need_r && !same) dr = at::empty(shape, h_.options());
      if (need_w) dw = n > 0 ? at::empty(w_shape, w_.options()) : at::zeros(w_shape, w_.options());
      const int64_t words = need_w ? abi.rms_norm_grad_scratch(n, width, g.count) : 0;
      const at::Tensor work = words > 0 ? bytes_on(h_, words) : at::Tensor();
      const auto at = [](const at::Tensor& t, const void* p, int64_t items) {
        return p == nullptr ? nullptr : (char*)const_cast<void*>(p) + items * (int64_t)t.element_size();
      };
      const auto out = [&](const at::Tensor& t, int64_t items) { return t.defined() ? at(t, t.data_ptr(), items) : nullptr; };
      // More gains than a call takes go in parts of about one size, each with enough of them to need no scratch;
      // an empty batch may have none.
      const int64_t parts = (g.count + ODP_NORM_GRAD_GAINS - 1) / ODP_NORM_GRAD_GAINS;
      const int64_t most = n > 0 ? (g.count + parts - 1) / parts : 0, each = n > 0 ? n / g.count : 0;
      for (int64_t i = 0; n > 0 && i < g.count; i += most) {
        const int64_t gains = std::min(most, g.count - i), row = i * each;
        check(abi.rms_norm_grad(stream_of(h_), code_of(gy.held), code_of(h_), g.dt, at(h_, rows.at, row * rows.pitch),
                                rows.pitch, (const float*)stat.data_ptr() + row, at(gy.held, gy.at, row * gy.pitch),
                                gy.pitch, at(h_, gh.at, row * gh.pitch), gh.pitch, gains * each, width,
                                at(g.t, g.at, i * g.pitch), g.pitch, gains, (float)offset,
                                work.defined() ? work.data_ptr() : nullptr, out(dx, row * width), out(dr, row * width),
                                out(dw, i * width)),
              "odp_rms_norm_grad");
      }
      if (need_r && same) dr = dx;
      if (!need_x) dx = at::Tensor();
    }
    dw = odp_host::first_only(grads, dw, true, kNorms);
    const bool shared = dx.defined() && dr.defined() && dx.is_same(dr);
    dx = odp_host::first_only(grads, dx, true, kNorms);
    dr = shared ? dx : odp_host::first_only(grads, dr, true, kNorms);
    return {dx, dr, dw};
  }
};

// (y, 1 / sqrt(..)) or, with a residual, (y, 1 / sqrt(..), the sum); without `keep` the second may be undefined.
variable_list normed(const at::Tensor& x, const Maybe& residual, const Maybe& weight, double eps, double offset,
                     bool keep) {
  no_tangents(x, residual, weight);
  bool grad = true;
  if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(residual) || wants_grad(weight)))
    keep = true;
  else
    grad = false;
  Normed o;
  {
    at::NoGradGuard no_grad;
    o = norm_forward(x, residual, weight, eps, offset, keep, 0);
  }
  if (grad) {
    const bool has_r = residual.has_value(), has_w = weight.has_value();
    const at::Tensor none, &r = has_r ? *residual : none, &w = has_w ? *weight : none;
    auto node = std::shared_ptr<NormNode>(new NormNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, r, w));
    torch::autograd::set_history(o.y, node);
    if (has_r) torch::autograd::set_history(o.h, node);
    node->h = SavedVariable(has_r ? o.h : x, has_r);
    node->rstd = SavedVariable(o.rstd, false);
    if (has_w) node->w = SavedVariable(w, false);
    node->has_r = has_r;
    node->has_w = has_w;
    node->offset = offset;
    node->xt = x.scalar_type();
    node->ht = has_r ? r.scalar_type() : node->xt;
    node->shape = x.sizes().vec();
    if (has_w) node->wt = w.scalar_type(), node->w_shape = w.sizes().vec();
  }
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
  no_tangents(x, residual, weight);
  const Normed o = norm_forward(x, residual, weight, eps, offset, false, quant);
  return residual.has_value() ? variable_list{o.y, o.scales, o.h} : variable_list{o.y, o.scales};
}

// ---------------------------------------------------------------------------
// Routing
// ---------------------------------------------------------------------------

constexpr const char* kRoutes = "the routing operators";

struct Options {
  bool sigmoid;
  int64_t groups, top_groups, best, top_k;
  bool renorm;
  double scale;
};

std::pair<at::Tensor, at::Tensor> route_forward(const at::Tensor& z, const Maybe& bias, const Options& o) {
  const c10::OptionalDeviceGuard guard(z.device());
  const Rows rows(z);
  const at::Tensor b = bias.has_value() ? odp_host::plain(*bias).contiguous() : at::Tensor();
  std::vector<int64_t> shape(z.sizes().vec());
  shape.back() = o.top_k;
  const at::Tensor index = at::empty(shape, z.options().dtype(at::kLong));
  const at::Tensor weights = at::empty(shape, z.options().dtype(at::kFloat));
  check(abi.route(stream_of(z), code_of(z), rows.at, rows.pitch, rows.n, rows.width, (int)o.sigmoid,
                  b.defined() ? (const float*)b.data_ptr() : nullptr, b.defined() && b.dim() == 2 ? b.size(0) : 1,
                  o.groups, o.top_groups, (int)o.best, o.top_k, (int)o.renorm, (float)o.scale,
                  (int64_t*)index.data_ptr(), (float*)weights.data_ptr()),
        "odp_route");
  return {index, weights};
}

struct RouteNode final : torch::autograd::Node {
  SavedVariable z, index;
  Options o;
  at::ScalarType type;
  std::vector<int64_t> shape;

  std::string name() const override { return "RouteBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    z.reset_data();
    index.reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const at::Tensor& gw = grads[0];
    if (!gw.defined() || !task_should_compute_output(0)) return variable_list(1);
    odp_host::no_batch(grads, kRoutes);
    const at::Tensor z_ = z.unpack(), index_ = index.unpack();
    at::Tensor dz;
    {
      at::NoGradGuard no_grad;
      const c10::OptionalDeviceGuard guard(gw.device());
      odp_host::as_saved(z_, gw, type, shape, kRoutes);
      const Rows rows(z_);
      std::vector<int64_t> chosen(shape);
      chosen.back() = o.top_k;
      const at::Tensor at_ = odp_host::whole(index_, gw, at::kLong, chosen, kRoutes);
      const at::Tensor g = odp_host::plain(gw).contiguous();
      dz = at::empty(shape, z_.options());
      check(abi.route_grad(stream_of(z_), code_of(z_), rows.at, rows.pitch, rows.n, rows.width, (int)o.sigmoid, o.top_k,
                           (int)o.renorm, (float)o.scale, (const int64_t*)at_.data_ptr(), (const float*)g.data_ptr(),
                           o.top_k, dz.data_ptr()),
            "odp_route_grad");
    }
    return {odp_host::first_only(grads, dz, true, kRoutes)};
  }
};

std::pair<at::Tensor, at::Tensor> route(const at::Tensor& z, const Maybe& bias, bool sigmoid, int64_t groups,
                                        int64_t top_groups, int64_t best, int64_t top_k, bool renorm, double scale) {
  py::gil_scoped_release nogil;
  odp_host::no_tangent(z, kRoutes);
  const Options o{sigmoid, groups, top_groups, best, top_k, renorm, scale};
  std::pair<at::Tensor, at::Tensor> out;
  {
    at::NoGradGuard no_grad;
    out = route_forward(z, bias, o);
  }
  if (at::GradMode::is_enabled() && z.requires_grad()) {
    auto node = std::shared_ptr<RouteNode>(new RouteNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(z));
    torch::autograd::set_history(out.second, node);
    node->z = SavedVariable(z, false);
    node->index = SavedVariable(out.first, false);
    node->o = o;
    node->type = z.scalar_type();
    node->shape = z.sizes().vec();
  }
  return out;
}

// ---------------------------------------------------------------------------
// Norm of a tree
// ---------------------------------------------------------------------------

int tree_code(const at::Tensor& t) { return t.scalar_type() == at::kDouble ? ODP_DTYPE_F64 : code_of(t); }

// The leaves scaled (with `clip`; else none) and their norm.  The scaled ones
// lie in one buffer per type, with the leaves' own strides where those leave no
// gaps.
std::pair<std::vector<at::Tensor>, at::Tensor> tree_norm(const std::vector<at::Tensor>& leaves, bool clip,
                                                         double max_norm, const std::string& who) {
  py::gil_scoped_release nogil;
  at::NoGradGuard no_grad;
  bool wide = false;
  for (const at::Tensor& t : leaves) {
    const auto type = t.scalar_type();
    TORCH_CHECK_TYPE(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf || type == at::kDouble, who,
                     " supports float32, bfloat16, float16 and float64 leaves, got ", type);
    TORCH_CHECK(t.is_cuda() && t.device() == leaves[0].device(), who,
                " runs on the GPU: its leaves must be CUDA tensors of one device");
    odp_host::no_tangent(t, "the tree norm's operators");
    wide = wide || type == at::kDouble;
  }
  const c10::OptionalDeviceGuard guard(leaves.at(0).device());
  constexpr int64_t kAlign = 64;
  std::vector<at::Tensor> src(leaves.size()), out;
  std::map<at::ScalarType, std::pair<int64_t, at::Tensor>> buffers;
  std::vector<int64_t> at_(leaves.size()), table(leaves.size() * ODP_TN_FIELDS);
  for (size_t i = 0; i < leaves.size(); ++i) {
    const at::Tensor t = odp_host::plain(leaves[i]);
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
  m.def("tree_norm", &tree_norm, py::arg("leaves"), py::arg("clip"), py::arg("max_norm"), py::arg("name"));
}
