// Operators of the `supa` namespace: what a transformer does between its
// matrix products and before its optimizer step.  They have no aten schema;
// torch.supa.residual_norm, rotary_embedding(_) and clip_grad_norm_ call them
// (torch_supa/supa/transformer.py).  Arguments are checked here; the device
// work is the C ABI's, on the tensors' device and its current stream, with
// workspaces from the caching allocator.
//
// Every call goes through the dispatcher below autograd, forward and backward, so
// that dispatch modes see it and tensors that wrap others (fake tensors, those of
// function transforms) reach a kernel that knows them; Meta kernels give the
// results' shapes.
#include <ATen/MemoryOverlap.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

#include "common.h"

namespace supa {
namespace {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = std::optional<at::Tensor>;

bool is_float16_or_32(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
bool given(const OptTensor& t) { return t.has_value() && t->defined(); }
OptTensor maybe(const at::Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
const void* ptr(const OptTensor& t) { return given(t) ? t->data_ptr() : nullptr; }

// Values of forward-mode differentiation would be dropped without a word.
void check_no_tangent(const char* op, std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), op,
                                ": no forward-mode derivative");
}
const at::Tensor& tensor(const OptTensor& t) {
  static const at::Tensor none;
  return given(t) ? *t : none;
}

// The operator of this schema name, called through the dispatcher.
template <typename F> c10::TypedOperatorHandle<F> find_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").template typed<F>();
}

// Meta tensors stand for supa ones.
bool is_supa(const at::Tensor& t) { return t.device().type() == kSupa || t.is_meta(); }
at::Tensor empty_beside(const at::Tensor& t, c10::IntArrayRef sizes, at::ScalarType dtype) {
  return t.is_meta() ? at::empty(sizes, t.options().dtype(dtype)) : empty_supa(sizes, dtype, t.device().index());
}

void check_on(const char* op, const char* name, const at::Tensor& t, const at::Tensor& like) {
  TORCH_CHECK(t.device() == like.device(), op, ": ", name, " is on ", t.device(), ", expected ", like.device());
}

// ------------------------------------------------------------ residual_norm
// x or residual as rows at one distance, elements contiguous; a copy where a
// view has no such form.
struct Rows {
  at::Tensor t;
  int64_t stride;
};
Rows rows_of(const at::Tensor& t) {
  const int64_t nd = t.dim(), width = t.size(-1);
  bool ok = width == 1 || t.stride(-1) == 1;
  int64_t stride = width, next = -1;  // next: the distance of a step in the dim before
  for (int64_t i = nd - 2; i >= 0 && ok; --i) {
    if (t.size(i) == 1) continue;
    if (next < 0) stride = t.stride(i);
    else ok = t.stride(i) == next;
    next = t.stride(i) * t.size(i);
  }
  if (!ok) return {t.contiguous(), width};
  return {t, stride};
}

struct NormArgs {
  double scale, eps;
  int64_t post, norm, period;
};

// The consecutive rows that share a row of the gate: the gate's leading dims are
// x's first ones, and 1 (or nothing) from there on.
int64_t gate_period(const at::Tensor& gate, const at::Tensor& x) {
  const int64_t nd = x.dim(), shift = nd - gate.dim();
  bool ok = gate.dim() >= 1 && shift >= 0 && gate.size(-1) == x.size(-1);
  int64_t period = 1;
  bool shared = false;  // walking back from the last leading dim: no longer shared
  for (int64_t i = nd - 2; i >= 0 && ok; --i) {
    const int64_t g = i >= shift ? gate.size(i - shift) : 1;
    if (x.size(i) == 1 && g == 1) continue;
    if (g == 1 && !shared) period *= x.size(i);
    else if (g == x.size(i)) shared = true;
    else ok = false;
  }
  TORCH_CHECK(ok, "residual_norm: a gate of shape ", gate.sizes(), " does not fit x of shape ", x.sizes(),
              ": its last dim is x's, its leading dims are x's first ones and then 1");
  return period;
}

// What a call has beside x and residual.
struct NormParams {
  OptTensor gate, post_weight, post_bias, weight, bias;
};

// Sizes, types, norms and parameters, forward and backward; `like` has x's shape.
void check_norm(const char* op, const at::Tensor& like, at::ScalarType dtype, at::ScalarType residual_dtype, NormArgs& a,
                const NormParams& p) {
  TORCH_CHECK(is_float16_or_32(dtype), op, ": expected float32, bfloat16 or float16, got x of ", dtype);
  TORCH_CHECK(like.dim() >= 1, op, ": expected x with a last dim to normalise, got a scalar");
  TORCH_CHECK(residual_dtype == dtype || residual_dtype == at::kFloat, op, ": expected residual of x's dtype (", dtype,
              ") or float32, got ", residual_dtype);
  const int64_t width = like.size(-1);
  TORCH_CHECK(width >= 1 && width <= SUPA_AMD_RESIDUAL_NORM_MAX_WIDTH, op, ": the last dim holds ", width,
              " elements, expected 1 to ", SUPA_AMD_RESIDUAL_NORM_MAX_WIDTH);
  TORCH_CHECK(like.numel() / width < (int64_t(1) << 31), op, ": expected fewer than 2^31 rows");
  TORCH_CHECK(std::isfinite(a.eps) && a.eps >= 0, op, ": expected eps >= 0, got ", a.eps);
  for (int64_t n : {a.post, a.norm})
    TORCH_CHECK(n >= SUPA_AMD_NORM_NONE && n <= SUPA_AMD_NORM_LAYER, op, ": no norm has number ", n);
  std::optional<at::ScalarType> param;
  const auto check_param = [&](const char* name, const OptTensor& t) {
    if (!given(t)) return;
    check_on(op, name, *t, like);
    const at::ScalarType s = t->scalar_type();
    TORCH_CHECK(s == dtype || s == at::kFloat, op, ": expected ", name, " of x's dtype (", dtype, ") or float32, got ", s);
    TORCH_CHECK(!param || *param == s, op, ": gate, weights and biases are of one dtype, got ", *param, " and ", s);
    param = s;
  };
  const auto check_vector = [&](const char* name, const OptTensor& t, bool allowed, const char* when) {
    if (!given(t)) return;
    TORCH_CHECK(allowed, op, ": ", name, " is given ", when);
    TORCH_CHECK(t->dim() == 1 && t->size(0) == width, op, ": expected ", name, " of shape [", width, "], got ",
                t->sizes());
    check_param(name, t);
  };
  check_vector("post_weight", p.post_weight, a.post != SUPA_AMD_NORM_NONE, "without a post norm");
  check_vector("post_bias", p.post_bias, a.post == SUPA_AMD_NORM_LAYER, "with a post norm that is not a layer norm");
  check_vector("weight", p.weight, a.norm != SUPA_AMD_NORM_NONE, "without a norm");
  check_vector("bias", p.bias, a.norm == SUPA_AMD_NORM_LAYER, "with a norm that is not a layer norm");
  check_param("gate", p.gate);
  a.period = given(p.gate) ? gate_period(*p.gate, like) : 1;
}

void check_residual_norm(const at::Tensor& x, const at::Tensor& residual, NormArgs& a, const NormParams& p) {
  constexpr const char* op = "residual_norm";
  TORCH_CHECK(is_supa(x), op, ": expected supa tensors, got x on ", x.device());
  check_on(op, "residual", residual, x);
  TORCH_CHECK(x.sizes() == residual.sizes(), op, ": x is of shape ", x.sizes(), ", residual of ", residual.sizes());
  check_norm(op, x, x.scalar_type(), residual.scalar_type(), a, p);
}

OptTensor contiguous(const OptTensor& t) { return given(t) ? OptTensor(t->contiguous()) : std::nullopt; }

NormParams contiguous(const NormParams& p) {
  return {contiguous(p.gate), contiguous(p.post_weight), contiguous(p.post_bias), contiguous(p.weight),
          contiguous(p.bias)};
}

supa_amd_residual_norm_desc norm_desc(int64_t rows, int64_t width, at::ScalarType dtype, at::ScalarType residual_dtype,
                                      const NormArgs& a, const NormParams& p) {
  supa_amd_residual_norm_desc d{};
  d.width = width;
  d.rows = rows;
  d.x_stride = d.residual_stride = width;
  d.gate_period = a.period;
  d.dtype = dtype_code(dtype);
  d.residual_dtype = dtype_code(residual_dtype);
  d.param_dtype = d.dtype;
  for (const OptTensor* t : {&p.gate, &p.post_weight, &p.post_bias, &p.weight, &p.bias})
    if (given(*t)) d.param_dtype = dtype_code((*t)->scalar_type());
  d.post_norm = (int32_t)a.post;
  d.norm = (int32_t)a.norm;
  d.residual_scale = a.scale;
  d.eps = a.eps;
  d.gate = ptr(p.gate);
  d.post_weight = ptr(p.post_weight);
  d.post_bias = ptr(p.post_bias);
  d.weight = ptr(p.weight);
  d.bias = ptr(p.bias);
  return d;
}

// Outputs of a forward call: h, y (undefined without a norm), the rows' statistics
// (if wanted and there is a norm).
using NormResult = std::tuple<at::Tensor, at::Tensor, at::Tensor>;
NormResult norm_outputs(const at::Tensor& x, const at::Tensor& residual, const NormArgs& a, bool want_stats) {
  const int64_t rows[] = {x.numel() / x.size(-1), 4};
  at::Tensor h = empty_beside(x, x.sizes(), residual.scalar_type()), y, stats;
  if (a.norm != SUPA_AMD_NORM_NONE) y = empty_beside(x, x.sizes(), x.scalar_type());
  if (want_stats && (a.post != SUPA_AMD_NORM_NONE || a.norm != SUPA_AMD_NORM_NONE))
    stats = empty_beside(x, rows, at::kFloat);
  return {h, y, stats};
}

NormResult norm_forward(const at::Tensor& x, const at::Tensor& residual, NormArgs a, const NormParams& params,
                        bool want_stats) {
  check_residual_norm(x, residual, a, params);
  const c10::DeviceGuard guard(x.device());
  const NormResult r = norm_outputs(x, residual, a, want_stats);
  const auto& [h, y, stats] = r;
  if (x.numel() == 0) return r;
  const Rows xr = rows_of(x), rr = rows_of(residual);
  const NormParams p = contiguous(params);
  supa_amd_residual_norm_desc d =
      norm_desc(x.numel() / x.size(-1), x.size(-1), x.scalar_type(), residual.scalar_type(), a, p);
  d.x = xr.t.data_ptr();
  d.x_stride = xr.stride;
  d.residual = rr.t.data_ptr();
  d.residual_stride = rr.stride;
  check_status(supa_amd_residual_norm_forward(&d, h.data_ptr(), y.defined() ? y.data_ptr() : nullptr,
                                              stats.defined() ? stats.data_ptr<float>() : nullptr,
                                              current_stream(x.device().index())),
               "residual_norm");
  return r;
}

#define SUPA_NORM_PARAMS                                                                                             \
  const at::Tensor &x, const at::Tensor &residual, const OptTensor &gate, double scale, int64_t post,                \
      const OptTensor &post_weight, const OptTensor &post_bias, int64_t norm, const OptTensor &weight,               \
      const OptTensor &bias, double eps

std::tuple<at::Tensor, at::Tensor> residual_norm(SUPA_NORM_PARAMS) {
  auto [h, y, stats] = norm_forward(x, residual, {scale, eps, post, norm, 1},
                                    {gate, post_weight, post_bias, weight, bias}, false);
  return {h, y};
}
NormResult residual_norm_forward(SUPA_NORM_PARAMS) {
  return norm_forward(x, residual, {scale, eps, post, norm, 1}, {gate, post_weight, post_bias, weight, bias}, true);
}

std::tuple<at::Tensor, at::Tensor> residual_norm_meta(SUPA_NORM_PARAMS) {
  NormArgs a{scale, eps, post, norm, 1};
  check_residual_norm(x, residual, a, {gate, post_weight, post_bias, weight, bias});
  auto [h, y, stats] = norm_outputs(x, residual, a, false);
  return {h, y};
}
NormResult residual_norm_forward_meta(SUPA_NORM_PARAMS) {
  NormArgs a{scale, eps, post, norm, 1};
  check_residual_norm(x, residual, a, {gate, post_weight, post_bias, weight, bias});
  return norm_outputs(x, residual, a, true);
}

// The inputs' places among the gradients.
enum NormInput { kX, kResidual, kGate, kPostWeight, kPostBias, kWeight, kBias, kNormInputs };
using NormGrads = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

// What the backward reads: the gradients of h and y (one of them at least), x and
// residual or, in their place, h; the forward's statistics; its other arguments.
#define SUPA_NORM_BACKWARD_PARAMS                                                                                    \
  const OptTensor &grad_h, const OptTensor &grad_y, const OptTensor &x, const OptTensor &residual,                   \
      const OptTensor &h, const OptTensor &stats, const OptTensor &gate, double scale, int64_t post,                 \
      const OptTensor &post_weight, const OptTensor &post_bias, int64_t norm, const OptTensor &weight,               \
      const OptTensor &bias, double eps, at::ScalarType dtype, at::ScalarType residual_dtype,                        \
      std::array<bool, 7> wanted

// Checks the arguments and allocates the gradients that are wanted.
std::array<at::Tensor, kNormInputs> norm_grads(SUPA_NORM_BACKWARD_PARAMS, NormArgs& a) {
  constexpr const char* op = "residual_norm (backward)";
  TORCH_CHECK(given(grad_h) || given(grad_y), op, ": expected a gradient of h or y");
  const at::Tensor& like = given(grad_h) ? *grad_h : *grad_y;
  TORCH_CHECK(is_supa(like), op, ": expected supa tensors, got a gradient on ", like.device());
  check_norm(op, like, dtype, residual_dtype, a, {gate, post_weight, post_bias, weight, bias});
  const int64_t rows[] = {like.numel() / like.size(-1), 4};
  const auto check = [&](const char* name, const OptTensor& t, at::ScalarType type, c10::IntArrayRef sizes) {
    if (!given(t)) return;
    check_on(op, name, *t, like);
    TORCH_CHECK(t->scalar_type() == type && t->sizes() == sizes, op, ": expected ", name, " of ", type, " and shape ",
                sizes, ", got ", t->scalar_type(), " of ", t->sizes());
  };
  check("grad_h", grad_h, residual_dtype, like.sizes());
  check("grad_y", grad_y, dtype, like.sizes());
  check("x", x, dtype, like.sizes());
  check("residual", residual, residual_dtype, like.sizes());
  check("h", h, residual_dtype, like.sizes());
  check("stats", stats, at::kFloat, rows);
  const OptTensor* params[] = {&gate, &post_weight, &post_bias, &weight, &bias};
  std::array<at::Tensor, kNormInputs> out;
  if (wanted[kX]) out[kX] = empty_beside(like, like.sizes(), dtype);
  if (wanted[kResidual]) out[kResidual] = empty_beside(like, like.sizes(), residual_dtype);
  for (int i = kGate; i < kNormInputs; ++i)
    if (const OptTensor& p = *params[i - kGate]; wanted[i] && given(p))
      out[i] = empty_beside(like, p->sizes(), p->scalar_type());
  return out;
}

NormGrads residual_norm_backward(SUPA_NORM_BACKWARD_PARAMS) {
  NormArgs a{scale, eps, post, norm, 1};
  const at::Tensor& like = given(grad_h) ? *grad_h : tensor(grad_y);
  const c10::OptionalDeviceGuard guard(like.defined() ? std::optional(like.device()) : std::nullopt);
  auto out = norm_grads(grad_h, grad_y, x, residual, h, stats, gate, scale, post, post_weight, post_bias, norm, weight,
                        bias, eps, dtype, residual_dtype, wanted, a);
  if (like.numel() == 0) {
    for (auto& t : out)
      if (t.defined()) t.zero_();
    return std::tuple_cat(out);
  }
  const OptTensor gh = contiguous(grad_h), gy = contiguous(grad_y), hc = contiguous(h), st = contiguous(stats);
  const NormParams p = contiguous(NormParams{gate, post_weight, post_bias, weight, bias});
  supa_amd_residual_norm_desc d = norm_desc(like.numel() / like.size(-1), like.size(-1), dtype, residual_dtype, a, p);
  Rows xr{}, rr{};  // hold copies until the launch
  if (given(x)) {
    xr = rows_of(*x);
    d.x = xr.t.data_ptr();
    d.x_stride = xr.stride;
  }
  if (given(residual)) {
    rr = rows_of(*residual);
    d.residual = rr.t.data_ptr();
    d.residual_stride = rr.stride;
  }
  const int64_t ws_bytes = supa_amd_residual_norm_backward_workspace_bytes(&d);
  TORCH_CHECK(ws_bytes >= 0, "residual_norm: ", supa_amd_status_string((int)ws_bytes));
  const auto dev = like.device().index();
  const at::Tensor ws = empty_supa({ws_bytes}, at::kByte, dev);
  const auto data = [&](int i) -> void* { return out[i].defined() ? out[i].data_ptr() : nullptr; };
  check_status(supa_amd_residual_norm_backward(&d, ptr(hc), ptr(gh), ptr(gy), static_cast<const float*>(ptr(st)), data(kX),
                                               data(kResidual), data(kGate), data(kPostWeight), data(kPostBias),
                                               data(kWeight), data(kBias), ws.data_ptr(), ws_bytes, current_stream(dev)),
               "residual_norm (backward)");
  return std::tuple_cat(out);
}
NormGrads residual_norm_backward_meta(SUPA_NORM_BACKWARD_PARAMS) {
  NormArgs a{scale, eps, post, norm, 1};
  return std::tuple_cat(norm_grads(grad_h, grad_y, x, residual, h, stats, gate, scale, post, post_weight, post_bias, norm,
                                   weight, bias, eps, dtype, residual_dtype, wanted, a));
}

// A node of its own, with plain fields, instead of a custom Function: the small
// calls of training are bound by the host, and it takes 6 us off a pass.  x and
// residual are saved for the backward, which forms h from them again; without
// post norm and gate h alone is enough where it is float32.  A 16-bit h, once rounded,
// is off by half a step of its own, which a layer norm magnifies by mean / deviation
// of the row ([3, 11, 520] bf16, mean 8, deviation 0.25: gradients off by 6 half steps
// of theirs); forming it again costs a read ([8192, 4096] bf16, RMS norm, both ways:
// 118 us, from the rounded h 107; [16384, 8192] 452, 397).
struct ResidualNormBackward final : public torch::autograd::Node {
  std::string name() const override { return "ResidualNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    residual.reset_data();
    h.reset_data();
    stats.reset_data();
    for (SavedVariable& p : params) p.reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "residual_norm: the gradient has no gradient of its own (create_graph)");
    variable_list out(kNormInputs);
    const OptTensor gh = maybe(grads[0]), gy = grads.size() > 1 ? maybe(grads[1]) : std::nullopt;
    if (!gh && !gy) return out;
    std::lock_guard<std::mutex> lock(mutex_);
    const c10::Device device = gh ? gh->device() : gy->device();
    // hooks on saved tensors (offloading, recomputation) may give them back otherwise; other strides do no harm
    const auto back = [&](const SavedVariable& v, std::optional<at::ScalarType> dtype, c10::IntArrayRef sizes) {
      const at::Tensor t = v.unpack(shared_from_this());
      TORCH_CHECK(!t.defined() || (t.device() == device && t.scalar_type() == dtype && t.sizes() == sizes),
                  "residual_norm: a saved tensor came back as ", t.scalar_type(), " of shape ", t.sizes(), " on ",
                  t.device(), ", expected shape ", sizes, " on ", device);
      return maybe(t);
    };
    const int64_t width[] = {shape.back()}, rows[] = {stats_rows, 4};
    const OptTensor xt = back(x, dtype, shape), rt = back(residual, residual_dtype, shape),
                    ht = back(h, residual_dtype, shape), st = back(stats, at::kFloat, rows);
    OptTensor p[kNormInputs];
    std::array<bool, 7> wanted;
    for (int i = 0; i < kNormInputs; ++i) {
      wanted[i] = task_should_compute_output(i);
      if (i >= kGate) p[i] = back(params[i], param_dtype, i == kGate ? c10::IntArrayRef(gate_shape) : c10::IntArrayRef(width));
    }
    static const auto op = find_op<decltype(residual_norm_backward)>("supa::_residual_norm_backward");
    const at::AutoDispatchBelowAutograd below;
    std::tie(out[kX], out[kResidual], out[kGate], out[kPostWeight], out[kPostBias], out[kWeight], out[kBias]) =
        op.call(gh, gy, xt, rt, ht, st, p[kGate], scale, post, p[kPostWeight], p[kPostBias], norm, p[kWeight], p[kBias],
                eps, dtype, residual_dtype, wanted);
    return out;
  }

  SavedVariable x, residual, h, stats, params[kNormInputs];
  at::ScalarType dtype, residual_dtype;
  std::optional<at::ScalarType> param_dtype;
  double scale, eps;
  int64_t post, norm, stats_rows;
  std::vector<int64_t> shape, gate_shape;
};

std::tuple<at::Tensor, at::Tensor> residual_norm_autograd(c10::DispatchKeySet ks, SUPA_NORM_PARAMS) {
  check_no_tangent("residual_norm", {&x, &residual, &tensor(gate), &tensor(post_weight), &tensor(post_bias),
                                     &tensor(weight), &tensor(bias)});
  const OptTensor* params[] = {&gate, &post_weight, &post_bias, &weight, &bias};
  bool needs = x.requires_grad() || residual.requires_grad();
  for (const OptTensor* t : params) needs = needs || (given(*t) && (*t)->requires_grad());
  if (!needs || !at::GradMode::is_enabled()) {
    static const auto op = find_op<decltype(residual_norm)>("supa::residual_norm");
    const at::AutoDispatchBelowAutograd below;
    return op.redispatch(ks & c10::after_autograd_keyset, x, residual, gate, scale, post, post_weight, post_bias, norm,
                         weight, bias, eps);
  }
  NormArgs a{scale, eps, post, norm, 1};
  check_residual_norm(x, residual, a, {gate, post_weight, post_bias, weight, bias});
  auto node = std::shared_ptr<ResidualNormBackward>(new ResidualNormBackward(), torch::autograd::deleteNode);
  const auto edge = [](const OptTensor& t) {
    return given(t) ? torch::autograd::impl::gradient_edge(*t) : torch::autograd::Edge();
  };
  node->set_next_edges({torch::autograd::impl::gradient_edge(x), torch::autograd::impl::gradient_edge(residual),
                        edge(gate), edge(post_weight), edge(post_bias), edge(weight), edge(bias)});
  at::Tensor xr, rr, h, y, stats;
  OptTensor g;
  {
    static const auto op = find_op<decltype(residual_norm_forward)>("supa::_residual_norm_forward");
    const at::AutoDispatchBelowAutograd below;
    xr = rows_of(x).t;  // a copy is made once, for both ways
    rr = rows_of(residual).t;
    g = contiguous(gate);
    std::tie(h, y, stats) = op.call(xr, rr, g, scale, post, post_weight, post_bias, norm, weight, bias, eps);
  }
  node->dtype = x.scalar_type();
  node->residual_dtype = residual.scalar_type();
  node->scale = scale;
  node->eps = eps;
  node->post = post;
  node->norm = norm;
  node->shape = x.sizes().vec();
  node->stats_rows = x.numel() / x.size(-1);
  const bool from_h = !given(gate) && post == SUPA_AMD_NORM_NONE &&
                      (norm == SUPA_AMD_NORM_NONE || residual.scalar_type() == at::kFloat);
  const bool needs_h = norm != SUPA_AMD_NORM_NONE;
  if (!from_h) node->x = SavedVariable(xr, false);
  if (!from_h && needs_h) node->residual = SavedVariable(rr, false);
  if (stats.defined()) node->stats = SavedVariable(stats, false);
  for (int i = kGate; i < kNormInputs; ++i) {
    const OptTensor& p = i == kGate ? g : *params[i - kGate];
    if (!given(p)) continue;
    node->params[i] = SavedVariable(*p, false);
    node->param_dtype = p->scalar_type();
  }
  if (given(gate)) node->gate_shape = gate->sizes().vec();
  torch::autograd::set_history(h, node);
  if (y.defined()) torch::autograd::set_history(y, node);
  if (from_h && needs_h) node->h = SavedVariable(h, true);
  return {h, y};
}

// --------------------------------------------------------- rotary_embedding
struct RotaryArgs {
  at::Tensor frequencies;  // contiguous float64
  OptTensor positions;
  int64_t offset;
  bool interleaved;
  double scale;
  bool inverse;
};

// [seq, heads, dim] or [batch, seq, heads, dim].
struct RotaryShape {
  int64_t batch, seq, heads, dim;
};
RotaryShape rotary_shape(const char* op, const char* name, const at::Tensor& t) {
  TORCH_CHECK(t.dim() == 3 || t.dim() == 4, op, ": expected ", name,
              " of shape [seq, heads, dim] or [batch, seq, heads, dim], got ", t.sizes());
  return {t.dim() == 4 ? t.size(0) : 1, t.size(-3), t.size(-2), t.size(-1)};
}

RotaryArgs check_rotary(const char* op, const at::Tensor& q, const OptTensor& k, const at::Tensor& frequencies,
                        const OptTensor& positions, int64_t offset, bool interleaved, double scale, bool inverse) {
  TORCH_CHECK(is_supa(q), op, ": expected supa tensors, got q on ", q.device());
  TORCH_CHECK(is_float16_or_32(q.scalar_type()), op, ": expected float32, bfloat16 or float16, got q of ",
              q.scalar_type());
  const RotaryShape s = rotary_shape(op, "q", q);
  if (given(k)) {
    check_on(op, "k", *k, q);
    TORCH_CHECK(k->scalar_type() == q.scalar_type(), op, ": q is of ", q.scalar_type(), ", k of ", k->scalar_type());
    const RotaryShape r = rotary_shape(op, "k", *k);
    TORCH_CHECK(k->dim() == q.dim() && r.batch == s.batch && r.seq == s.seq && r.dim == s.dim, op,
                ": q and k differ in more than their heads: ", q.sizes(), " and ", k->sizes());
  }
  check_on(op, "frequencies", frequencies, q);
  TORCH_CHECK(frequencies.dim() == 1 && at::isFloatingType(frequencies.scalar_type()), op,
              ": expected frequencies as a vector of floats, got ", frequencies.scalar_type(), " of shape ",
              frequencies.sizes());
  const int64_t rotary = 2 * frequencies.size(0);
  TORCH_CHECK(rotary >= 2 && rotary <= s.dim && rotary <= 1024, op, ": ", frequencies.size(0),
              " frequencies rotate ", rotary, " elements of a head; expected 2 to ", std::min<int64_t>(s.dim, 1024));
  TORCH_CHECK(!frequencies.requires_grad(), op, ": frequencies have no gradient");
  TORCH_CHECK(std::isfinite(scale), op, ": expected a finite scale, got ", scale);
  if (given(positions)) {
    check_on(op, "positions", *positions, q);
    TORCH_CHECK(positions->scalar_type() == at::kLong || positions->scalar_type() == at::kInt, op,
                ": expected int64 or int32 positions, got ", positions->scalar_type());
    const bool ok = (positions->dim() == 1 && positions->size(0) == s.seq) ||
                    (positions->dim() == 2 && q.dim() == 4 && positions->size(1) == s.seq &&
                     (positions->size(0) == s.batch || positions->size(0) == 1));
    TORCH_CHECK(ok, op, ": expected positions of shape [", s.seq, "]", q.dim() == 4 ? " or [batch, seq]" : "",
                ", got ", positions->sizes());
  }
  TORCH_CHECK(s.batch * s.seq < (int64_t(1) << 31), op, ": expected fewer than 2^31 tokens");
  TORCH_CHECK(s.dim < (int64_t(1) << 24), op, ": expected heads of fewer than 2^24 elements, got ", s.dim);
  // frequencies of another type are widened, not formed anew
  return {frequencies.to(at::kDouble).contiguous(), positions, offset, interleaved, scale, inverse};
}

supa_amd_rotary_tensor rotary_tensor(const at::Tensor& in, const at::Tensor& out) {
  TORCH_INTERNAL_ASSERT(in.stride(-1) == 1 && out.stride(-1) == 1);
  supa_amd_rotary_tensor t{};
  t.in = in.data_ptr();
  t.out = out.data_ptr();
  t.heads = in.size(-2);
  for (int i = 0; i < 3; ++i) {
    const int64_t dim = in.dim() - 4 + i;
    t.in_strides[i] = dim < 0 ? 0 : in.stride(dim);
    t.out_strides[i] = dim < 0 ? 0 : out.stride(dim);
  }
  return t;
}

void launch_rotary(const char* op, const at::Tensor& q, const at::Tensor& q_out, const at::Tensor& k,
                   const at::Tensor& k_out, const RotaryArgs& a) {
  const RotaryShape s = rotary_shape(op, "q", q);
  supa_amd_rotary_desc d{};
  d.batch = s.batch;
  d.seq = s.seq;
  d.dim = s.dim;
  d.rotary = 2 * a.frequencies.size(0);
  d.dtype = dtype_code(q.scalar_type());
  d.layout = a.interleaved ? SUPA_AMD_ROTARY_INTERLEAVED : SUPA_AMD_ROTARY_HALF;
  d.inverse = a.inverse;
  d.position_dtype = SUPA_AMD_I64;
  d.scale = a.scale;
  d.frequencies = a.frequencies.data_ptr<double>();
  d.offset = a.offset;
  if (given(a.positions)) {
    const at::Tensor& p = *a.positions;
    d.positions = p.data_ptr();
    d.position_dtype = dtype_code(p.scalar_type());
    d.position_strides[0] = p.dim() == 2 && p.size(0) > 1 ? p.stride(0) : 0;
    d.position_strides[1] = p.stride(-1);
  }
  if (q.numel() > 0) d.q = rotary_tensor(q, q_out);
  if (k.defined() && k.numel() > 0) d.k = rotary_tensor(k, k_out);
  if (!d.q.in && !d.k.in) return;
  check_status(supa_amd_rotary(&d, current_stream(q.device().index())), op);
}

at::Tensor heads_contiguous(const at::Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

// An output in t's order of dims.  Of windows that slide over each other the strides
// do not say which dim is innermost, and empty_like may take another than the last.
at::Tensor rotated_like(const at::Tensor& t) {
  const at::Tensor out = at::empty_like(t);
  return out.stride(-1) == 1 ? out : at::empty_like(t, at::MemoryFormat::Contiguous);
}

std::tuple<at::Tensor, at::Tensor> rotary_embedding(const at::Tensor& q, const OptTensor& k,
                                                    const at::Tensor& frequencies, const OptTensor& positions,
                                                    int64_t offset, bool interleaved, double scale, bool inverse) {
  constexpr const char* op = "rotary_embedding";
  const c10::OptionalDeviceGuard guard(q.device());
  const RotaryArgs a = check_rotary(op, q, k, frequencies, positions, offset, interleaved, scale, inverse);
  const at::Tensor qi = heads_contiguous(q), ki = given(k) ? heads_contiguous(*k) : at::Tensor();
  const at::Tensor qo = rotated_like(qi), ko = ki.defined() ? rotated_like(ki) : at::Tensor();
  if (!q.is_meta()) launch_rotary(op, qi, qo, ki, ko, a);
  return {qo, ko};
}

// A step through memory, in bytes, and how often the one and the other tensor take it.
struct Step {
  int64_t stride, one, other;
};
using Steps = c10::SmallVector<Step, 8>;

// The steps of a tensor and, if there is one, of another, from long to short; a
// step that both take is one step, one that a tensor takes in two dims is two.
Steps steps_of(const at::Tensor& one, const at::Tensor& other = {}) {
  Steps steps;
  const auto add = [&](const at::Tensor& t, int64_t Step::* times) {
    for (int64_t i = 0; i < t.dim(); ++i) {
      if (t.size(i) == 1) continue;
      const int64_t stride = t.stride(i) * (int64_t)t.element_size();
      auto at = std::find_if(steps.begin(), steps.end(), [&](const Step& s) { return s.stride == stride && s.*times == 0; });
      if (at == steps.end()) at = steps.insert(at, {stride, 0, 0});
      (*at).*times = t.size(i) - 1;
    }
  };
  add(one, &Step::one);
  if (other.defined()) add(other, &Step::other);
  std::sort(steps.begin(), steps.end(), [](const Step& a, const Step& b) { return a.stride > b.stride; });
  return steps;
}

// Whether blocks of `block` bytes, one at every combination of the first n steps
// (the one tensor's), keep apart: each step goes past all that the smaller ones reach.
bool apart(const Steps& steps, size_t n, int64_t block) {
  for (size_t i = n; i-- > 0;) {
    if (steps[i].stride < block) return false;
    block += steps[i].one * steps[i].stride;
  }
  return true;
}

// Whether two tensors share no memory, of any types and shapes: over their smaller
// steps (or none, or all) each fills a block, the other's beside the one's, and
// their larger steps, which both may take, lead from one such pair of blocks to the
// next (q and k of a packed projection, token by token or sample by sample; the
// columns of a matrix).
bool beside(const at::Tensor& a, const at::Tensor& b) {
  const bool ordered = a.data_ptr() <= b.data_ptr();
  const at::Tensor &one = ordered ? a : b, &other = ordered ? b : a;
  const int64_t distance = static_cast<const char*>(other.data_ptr()) - static_cast<const char*>(one.data_ptr());
  const Steps steps = steps_of(one, other);
  int64_t first = (int64_t)one.element_size(), second = (int64_t)other.element_size();  // the blocks' bytes
  for (size_t outer = steps.size();; --outer) {
    // the other's first block lies so many steps ahead, and `gap` behind the one's block there
    int64_t gap = distance;
    Steps joint(steps.begin(), steps.begin() + outer);
    for (Step& s : joint) {
      if (s.stride == 0) return false;
      const int64_t ahead = gap / s.stride;
      gap -= ahead * s.stride;
      s.one = std::max(s.one, s.other + ahead);
    }
    if (first <= gap && apart(joint, outer, gap + second)) return true;
    if (outer == 0) return false;
    first += steps[outer - 1].one * steps[outer - 1].stride;
    second += steps[outer - 1].other * steps[outer - 1].stride;
  }
}

void rotary_embedding_(at::Tensor& q, const OptTensor& k, const at::Tensor& frequencies, const OptTensor& positions,
                       int64_t offset, bool interleaved, double scale, bool inverse) {
  constexpr const char* op = "rotary_embedding_";
  const c10::OptionalDeviceGuard guard(q.device());
  const RotaryArgs a = check_rotary(op, q, k, frequencies, positions, offset, interleaved, scale, inverse);
  for (const at::Tensor* t : {(const at::Tensor*)&q, given(k) ? &*k : nullptr}) {
    if (!t || t->numel() == 0) continue;
    TORCH_CHECK(t->stride(-1) == 1, op, ": expected heads whose elements are contiguous");
    const Steps steps = steps_of(*t);
    TORCH_CHECK(apart(steps, steps.size(), (int64_t)t->element_size()), op,
                ": expected a tensor whose heads do not overlap in memory");
  }
  if (q.is_meta()) return;
  if (given(k) && q.numel() > 0 && k->numel() > 0)
    TORCH_CHECK(beside(q, *k), op, ": q and k overlap in memory");
  launch_rotary(op, q, q, given(k) ? *k : at::Tensor(), given(k) ? *k : at::Tensor(), a);
}

c10::TypedOperatorHandle<decltype(rotary_embedding)> rotary_op() {
  static const auto op = find_op<decltype(rotary_embedding)>("supa::rotary_embedding");
  return op;
}

// The rotation back, by the same operator, which has a gradient of its own.
struct RotaryEmbeddingBackward final : public torch::autograd::Node {
  std::string name() const override { return "RotaryEmbeddingBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    frequencies.reset_data();
    positions.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    variable_list out(2);
    const at::Tensor gq = task_should_compute_output(0) ? grads[0] : at::Tensor();
    const at::Tensor gk = grads.size() > 1 && task_should_compute_output(1) ? grads[1] : at::Tensor();
    if (!gq.defined() && !gk.defined()) return out;
    std::lock_guard<std::mutex> lock(mutex_);
    const bool both = gq.defined() && gk.defined();
    const at::Tensor& first = gq.defined() ? gq : gk;
    const OptTensor second = both ? OptTensor(gk) : std::nullopt;
    const at::Tensor f = frequencies.unpack();
    const OptTensor p = maybe(positions.unpack());
    auto [a, b] = rotary_op().call(first, second, f, p, offset, interleaved, scale, !inverse);
    if (gq.defined()) out[0] = a;
    if (gk.defined()) out[1] = both ? b : a;
    return out;
  }

  SavedVariable frequencies, positions;
  int64_t offset;
  bool interleaved, inverse;
  double scale;
};

std::tuple<at::Tensor, at::Tensor> rotary_embedding_autograd(c10::DispatchKeySet ks, const at::Tensor& q,
                                                             const OptTensor& k, const at::Tensor& frequencies,
                                                             const OptTensor& positions, int64_t offset,
                                                             bool interleaved, double scale, bool inverse) {
  check_no_tangent("rotary_embedding", {&q, &tensor(k), &frequencies});
  const bool needs = q.requires_grad() || (given(k) && k->requires_grad());
  TORCH_CHECK(!frequencies.requires_grad(), "rotary_embedding: frequencies have no gradient");
  const auto forward = [&] {
    const at::AutoDispatchBelowAutograd below;
    return rotary_op().redispatch(ks & c10::after_autograd_keyset, q, k, frequencies, positions, offset, interleaved,
                                  scale, inverse);
  };
  if (!needs || !at::GradMode::is_enabled()) return forward();
  auto node = std::shared_ptr<RotaryEmbeddingBackward>(new RotaryEmbeddingBackward(), torch::autograd::deleteNode);
  torch::autograd::edge_list edges{torch::autograd::impl::gradient_edge(q)};
  if (given(k)) edges.push_back(torch::autograd::impl::gradient_edge(*k));
  else edges.emplace_back();
  node->set_next_edges(std::move(edges));
  node->offset = offset;
  node->interleaved = interleaved;
  node->inverse = inverse;
  node->scale = scale;
  auto [qo, ko] = forward();
  node->frequencies = SavedVariable(frequencies, false);
  if (given(positions)) node->positions = SavedVariable(*positions, false);
  torch::autograd::set_history(qo, node);
  if (ko.defined()) torch::autograd::set_history(ko, node);
  return {qo, ko};
}

c10::TypedOperatorHandle<decltype(rotary_embedding_)> rotary_op_() {
  static const auto op = find_op<decltype(rotary_embedding_)>("supa::rotary_embedding_");
  return op;
}

void rotary_embedding_autograd_(c10::DispatchKeySet ks, at::Tensor& q, const OptTensor& k, const at::Tensor& frequencies,
                                const OptTensor& positions, int64_t offset, bool interleaved, double scale,
                                bool inverse) {
  TORCH_CHECK(!at::GradMode::is_enabled() || !(q.requires_grad() || (given(k) && k->requires_grad())),
              "rotary_embedding_: the call in place has no gradient; use rotary_embedding");
  check_no_tangent("rotary_embedding_", {&q, &tensor(k), &frequencies});
  const at::AutoDispatchBelowAutograd below;
  rotary_op_().redispatch(ks & c10::after_autograd_keyset, q, k, frequencies, positions, offset, interleaved, scale,
                          inverse);
}

// A tensor that was written has a new version, in inference mode too (where autograd's
// kernels are left out, this key's are not).
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void rotary_embedding_versions_(c10::DispatchKeySet ks, at::Tensor& q, const OptTensor& k,
                                const at::Tensor& frequencies, const OptTensor& positions, int64_t offset,
                                bool interleaved, double scale, bool inverse) {
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    rotary_op_().redispatch(ks & c10::after_ADInplaceOrView_keyset, q, k, frequencies, positions, offset, interleaved,
                            scale, inverse);
  }
  written(q);
  if (given(k)) written(*k);
}

// ----------------------------------------------------------- clip_grad_norm_
// Checks the arguments; the norm's type.
at::ScalarType check_clip(const char* op, at::TensorList grads, double max_norm, double ord) {
  TORCH_CHECK(!grads.empty(), op, ": expected at least one tensor");
  TORCH_CHECK(max_norm >= 0, op, ": expected max_norm >= 0, got ", max_norm);
  TORCH_CHECK(ord == 1.0 || ord == 2.0 || ord == HUGE_VAL, op, ": expected the norm 1, 2 or inf, got ", ord);
  const c10::Device device = grads[0].device();
  at::ScalarType norm_type = at::kFloat;
  for (const at::Tensor& g : grads) {
    TORCH_CHECK(is_supa(g) && g.layout() == at::kStrided, op, ": expected dense supa tensors, got one of layout ",
                g.layout(), " on ", g.device());
    TORCH_CHECK(g.device() == device, op, ": the tensors are on ", device, " and ", g.device(), ", expected one device");
    const at::ScalarType t = g.scalar_type();
    TORCH_CHECK(is_float16_or_32(t) || t == at::kDouble, op, ": expected floating tensors, got one of ", t);
    if (t == at::kDouble) norm_type = at::kDouble;
  }
  return norm_type;
}

at::Tensor clip_grad_norm_meta_(at::TensorList grads, double max_norm, double ord, bool /*error_if_nonfinite*/) {
  const at::ScalarType norm_type = check_clip("clip_grad_norm_", grads, max_norm, ord);
  return empty_beside(grads[0], {}, norm_type);
}

at::Tensor clip_grad_norm_(at::TensorList grads, double max_norm, double ord, bool error_if_nonfinite) {
  constexpr const char* op = "clip_grad_norm_";
  const at::ScalarType norm_type = check_clip(op, grads, max_norm, ord);
  const c10::Device device = grads[0].device();
  const size_t n = grads.size();
  std::vector<at::Tensor> copies;         // of tensors that are not dense, in the list's order
  std::vector<void*> p(n);
  std::vector<int64_t> numel(n);
  std::vector<int32_t> dtypes(n);
  // the memory from a tensor's first element to behind its last, and the tensor
  std::vector<std::tuple<const char*, const char*, size_t>> spans;
  spans.reserve(n);
  const c10::DeviceGuard guard(device);
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor& g = grads[i];
    at::Tensor x = g;
    if (!g.is_non_overlapping_and_dense()) {
      at::assert_no_internal_overlap(g);
      x = g.contiguous();
      copies.push_back(x);
    }
    if (g.numel() > 0) {
      int64_t last = 0;
      for (int64_t d = 0; d < g.dim(); ++d) last += (g.size(d) - 1) * g.stride(d);
      const char* at = static_cast<const char*>(g.data_ptr());
      spans.emplace_back(at, at + (last + 1) * (int64_t)g.element_size(), i);
    }
    p[i] = x.data_ptr();
    numel[i] = x.numel();
    dtypes[i] = dtype_code(g.scalar_type());
  }
  // two that reach over each other have to lie beside each other, as the columns of a matrix do
  std::sort(spans.begin(), spans.end());
  for (size_t i = 0; i < spans.size(); ++i) {
    const auto& [at, end, one] = spans[i];
    for (size_t j = i + 1; j < spans.size() && std::get<0>(spans[j]) < end; ++j) {
      TORCH_CHECK(beside(grads[one], grads[std::get<2>(spans[j])]), op, ": two of the tensors share memory");
    }
  }
  const auto dev = device.index();
  const int64_t ws_bytes = supa_amd_grad_norm_workspace_bytes((int32_t)n, numel.data(), dtypes.data());
  TORCH_CHECK(ws_bytes >= 0, op, ": ", supa_amd_status_string((int)ws_bytes));
  const at::Tensor ws = empty_supa({ws_bytes}, at::kByte, dev);
  at::Tensor norm = empty_supa({}, norm_type, dev);
  const hipStream_t st = current_stream(dev);
  if (error_if_nonfinite) {  // reads the norm back before anything is scaled
    check_status(supa_amd_grad_norm((int32_t)n, p.data(), numel.data(), dtypes.data(), ord, norm.data_ptr(),
                                    dtype_code(norm_type), ws.data_ptr(), ws_bytes, st),
                 op);
    const double v = norm.item().toDouble();
    TORCH_CHECK(std::isfinite(v), "The total norm of order ", ord, " for gradients from `parameters` is non-finite, so "
                "it cannot be clipped. To disable this error and scale the gradients by the non-finite norm anyway, "
                "set `error_if_nonfinite=False`");
    check_status(supa_amd_grad_scale((int32_t)n, p.data(), numel.data(), dtypes.data(), max_norm, ws.data_ptr(),
                                     ws_bytes, st),
                 op);
  } else {
    check_status(supa_amd_clip_grad_norm((int32_t)n, p.data(), numel.data(), dtypes.data(), ord, max_norm,
                                         norm.data_ptr(), dtype_code(norm_type), ws.data_ptr(), ws_bytes, st),
                 op);
  }
  size_t c = 0;
  for (size_t i = 0; i < n && c < copies.size(); ++i) {
    if (grads[i].is_non_overlapping_and_dense()) continue;
    grads[i].copy_(copies[c++]);
  }
  return norm;
}

c10::TypedOperatorHandle<decltype(clip_grad_norm_)> clip_op() {
  static const auto op = find_op<decltype(clip_grad_norm_)>("supa::clip_grad_norm_");
  return op;
}

at::Tensor clip_grad_norm_autograd_(c10::DispatchKeySet ks, at::TensorList grads, double max_norm, double ord,
                                    bool error_if_nonfinite) {
  const at::AutoDispatchBelowAutograd below;  // the scaling is no part of a graph, as under no_grad
  return clip_op().redispatch(ks & c10::after_autograd_keyset, grads, max_norm, ord, error_if_nonfinite);
}

at::Tensor clip_grad_norm_versions_(c10::DispatchKeySet ks, at::TensorList grads, double max_norm, double ord,
                                    bool error_if_nonfinite) {
  at::Tensor norm;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    norm = clip_op().redispatch(ks & c10::after_ADInplaceOrView_keyset, grads, max_norm, ord, error_if_nonfinite);
  }
  for (const at::Tensor& g : grads) written(g);
  return norm;
}

}  // namespace
}  // namespace supa

TORCH_LIBRARY(supa, m) {
  m.def(
      "residual_norm(Tensor x, Tensor residual, Tensor? gate, float residual_scale, int post_norm, Tensor? post_weight, "
      "Tensor? post_bias, int norm, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor)");
  // its parts for training: the rows' statistics beside h and y; the gradients of the seven tensors
  m.def(
      "_residual_norm_forward(Tensor x, Tensor residual, Tensor? gate, float residual_scale, int post_norm, Tensor? "
      "post_weight, Tensor? post_bias, int norm, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor, Tensor)");
  m.def(
      "_residual_norm_backward(Tensor? grad_h, Tensor? grad_y, Tensor? x, Tensor? residual, Tensor? h, Tensor? stats, "
      "Tensor? gate, float residual_scale, int post_norm, Tensor? post_weight, Tensor? post_bias, int norm, Tensor? weight, "
      "Tensor? bias, float eps, ScalarType dtype, ScalarType residual_dtype, bool[7] output_mask) -> "
      "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "rotary_embedding(Tensor q, Tensor? k, Tensor frequencies, Tensor? positions, int offset, bool interleaved, "
      "float scale, bool inverse) -> (Tensor, Tensor)");
  m.def(
      "rotary_embedding_(Tensor(a!) q, Tensor(b!)? k, Tensor frequencies, Tensor? positions, int offset, "
      "bool interleaved, float scale, bool inverse) -> ()");
  m.def("clip_grad_norm_(Tensor(a!)[] grads, float max_norm, float ord, bool error_if_nonfinite) -> Tensor");
}

TORCH_LIBRARY_IMPL(supa, PrivateUse1, m) {
  using namespace supa;
  m.impl("residual_norm", TORCH_FN(residual_norm));
  m.impl("_residual_norm_forward", TORCH_FN(residual_norm_forward));
  m.impl("_residual_norm_backward", TORCH_FN(residual_norm_backward));
  m.impl("rotary_embedding", TORCH_FN(rotary_embedding));
  m.impl("rotary_embedding_", TORCH_FN(rotary_embedding_));
  m.impl("clip_grad_norm_", TORCH_FN(clip_grad_norm_));
}

TORCH_LIBRARY_IMPL(supa, Meta, m) {
  using namespace supa;
  m.impl("residual_norm", TORCH_FN(residual_norm_meta));
  m.impl("_residual_norm_forward", TORCH_FN(residual_norm_forward_meta));
  m.impl("_residual_norm_backward", TORCH_FN(residual_norm_backward_meta));
  m.impl("rotary_embedding", TORCH_FN(rotary_embedding));
  m.impl("rotary_embedding_", TORCH_FN(rotary_embedding_));
  m.impl("clip_grad_norm_", TORCH_FN(clip_grad_norm_meta_));
}

namespace supa {
namespace {
void autograd_kernels(torch::Library& m) {
  m.impl("residual_norm", TORCH_FN(residual_norm_autograd));
  m.impl("rotary_embedding", TORCH_FN(rotary_embedding_autograd));
  m.impl("rotary_embedding_", TORCH_FN(rotary_embedding_autograd_));
  m.impl("clip_grad_norm_", TORCH_FN(clip_grad_norm_autograd_));
}
}  // namespace
}  // namespace supa
TORCH_LIBRARY_IMPL(supa, AutogradPrivateUse1, m) { supa::autograd_kernels(m); }
TORCH_LIBRARY_IMPL(supa, ADInplaceOrView, m) {
  using namespace supa;
  m.impl("rotary_embedding_", TORCH_FN(rotary_embedding_versions_));
  m.impl("clip_grad_norm_", TORCH_FN(clip_grad_norm_versions_));
}
TORCH_LIBRARY_IMPL(supa, Autograd, m) { supa::autograd_kernels(m); }  // meta tensors, and wrappers of any
