// Operators of the `supa` namespace on rows of logits, beside the losses: distillation
// from a teacher's top logits, the balance loss of a router, and what a server does
// to logits before it draws from them.  torch.supa.distillation_loss,
// router_balance_loss and adjust_logits(_) call them (torch_supa/supa/logits.py).
// Arguments are checked here; the device work is the C ABI's, on the tensors'
// device and its current stream, with workspaces from the caching allocator.
//
// Every call goes through the dispatcher below autograd, forward and backward, and has a Meta kernel,
// as the operators of a transformer do.
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include <cmath>
#include <tuple>
#include <vector>

#include "supa_ops.h"

namespace supa {
namespace {

bool is_index(at::ScalarType t) { return t == at::kLong || t == at::kInt; }

void check_reduction(const char* op, int64_t reduction) {
  TORCH_CHECK(reduction == SUPA_AMD_REDUCTION_NONE || reduction == SUPA_AMD_REDUCTION_MEAN ||
                  reduction == SUPA_AMD_REDUCTION_SUM,
              op, ": no reduction has number ", reduction);
}

// A gradient is the operator's own only where autograd will not ask for its gradient.
void check_once(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, ": the gradient has no gradient of its own (create_graph)");
}

// ------------------------------------------------------- distillation_loss
// Logits as rows at up to two distances, elements contiguous: row r lies at
// (r / inner) stride[0] + (r % inner) stride[1]; a copy where a view has no such form.
struct LogitRows {
  at::Tensor t;
  int64_t inner, stride[2];
};
LogitRows logit_rows(const at::Tensor& t) {
  const int64_t vocab = t.size(-1);
  bool ok = vocab == 1 || t.stride(-1) == 1;
  int64_t size[2] = {1, 1}, stride[2] = {0, 0};  // inner, outer
  int level = 0;
  for (int64_t i = t.dim() - 2; i >= 0 && ok; --i) {
    if (t.size(i) == 1) continue;
    if (size[level] > 1 && t.stride(i) != stride[level] * size[level]) ++level;
    if (level > 1) {
      ok = false;
    } else if (size[level] == 1) {
      stride[level] = t.stride(i);
      size[level] = t.size(i);
    } else {
      size[level] *= t.size(i);
    }
  }
  if (!ok) return {t.contiguous(), std::max<int64_t>(1, t.numel() / vocab), {0, vocab}};
  return {t, std::max<int64_t>(1, size[0]), {stride[1], stride[0]}};
}

// Rows of another tensor of the logits' leading dims, split into outer and inner ones as the
// logits' are; `width` elements each, contiguous (has_row: in a last dim of its own).  A copy where a view
// has no such form.
LogitRows rows_beside(const at::Tensor& t, int64_t inner, bool has_row) {
  const int64_t leading = t.dim() - (has_row ? 1 : 0), width = has_row ? t.size(-1) : 1;
  bool ok = !has_row || width == 1 || t.stride(-1) == 1;
  int64_t size[2] = {1, 1}, stride[2] = {0, 0};  // inner, outer
  for (int64_t i = leading - 1; i >= 0 && ok; --i) {
    if (t.size(i) == 1) continue;
    const int level = size[0] == inner ? 1 : 0;
    if (size[level] == 1) stride[level] = t.stride(i);
    else ok = t.stride(i) == stride[level] * size[level];
    size[level] *= t.size(i);
  }
  if (!ok || (size[0] != inner && t.numel() > 0)) return {t.contiguous(), inner, {inner * width, width}};
  return {t, inner, {stride[1], stride[0]}};
}

void check_distill_logits(const char* op, const at::Tensor& logits, double temperature, int64_t reduction) {
  TORCH_CHECK(is_supa(logits), op, ": expected supa tensors, got logits on ", logits.device());
  TORCH_CHECK(is_float16_or_32(logits.scalar_type()), op, ": expected float32, bfloat16 or float16, got logits of ",
              logits.scalar_type());
  TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1 && logits.size(-1) < (int64_t(1) << 31), op,
              ": expected logits with a last dim of 1 to 2^31 - 1 tokens, got shape ", logits.sizes());
  TORCH_CHECK(logits.numel() / logits.size(-1) < (int64_t(1) << 31), op, ": expected fewer than 2^31 rows");
  TORCH_CHECK(temperature >= 1e-30 && temperature <= 1e30, op, ": expected a temperature of 1e-30 to 1e30, got ", temperature);
  check_reduction(op, reduction);
}

void check_distill(const at::Tensor& logits, const at::Tensor& indices, const at::Tensor& teacher,
                   const OptTensor& teacher_lse, double temperature, int64_t reduction) {
  constexpr const char* op = "distillation_loss";
  check_distill_logits(op, logits, temperature, reduction);
  check_on(op, "indices", indices, logits);
  TORCH_CHECK(is_index(indices.scalar_type()), op, ": expected int64 or int32 indices, got ", indices.scalar_type());
  TORCH_CHECK(indices.dim() == logits.dim() && indices.sizes().slice(0, logits.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
              op, ": indices of shape ", indices.sizes(), " do not fit logits of shape ", logits.sizes(),
              ": they differ in the last dim alone");
  TORCH_CHECK(indices.size(-1) >= 1 && indices.size(-1) <= SUPA_AMD_DISTILL_MAX_ENTRIES, op, ": expected 1 to ",
              SUPA_AMD_DISTILL_MAX_ENTRIES, " tokens a row, got ", indices.size(-1));
  check_on(op, "teacher_logits", teacher, logits);
  TORCH_CHECK(is_float16_or_32(teacher.scalar_type()), op, ": expected teacher_logits of float32, bfloat16 or float16, got ",
              teacher.scalar_type());
  TORCH_CHECK(teacher.sizes() == indices.sizes(), op, ": indices are of shape ", indices.sizes(),
              ", teacher_logits of ", teacher.sizes());
  if (given(teacher_lse)) {
    check_on(op, "teacher_lse", *teacher_lse, logits);
    TORCH_CHECK(at::isFloatingType(teacher_lse->scalar_type()) &&
                    teacher_lse->sizes() == logits.sizes().slice(0, logits.dim() - 1),
                op, ": expected teacher_lse as floats of shape ", logits.sizes().slice(0, logits.dim() - 1), ", got ",
                teacher_lse->scalar_type(), " of shape ", teacher_lse->sizes());
  }
}

supa_amd_distill_desc distill_desc(const LogitRows& x, int64_t entries, double temperature, int64_t reduction) {
  supa_amd_distill_desc d{};
  d.vocab = x.t.size(-1);
  d.rows = x.t.numel() / d.vocab;
  d.entries = entries;
  d.inner = x.inner;
  d.logits_strides[0] = x.stride[0];
  d.logits_strides[1] = x.stride[1];
  d.dtype = dtype_code(x.t.scalar_type());
  d.teacher_dtype = SUPA_AMD_F32;
  d.index_dtype = SUPA_AMD_I64;
  d.reduction = (int32_t)reduction;
  d.temperature = temperature;
  d.logits = x.t.data_ptr();
  return d;
}

// loss, count (undefined without a reduction), the rows' statistics, the pairs as the backward reads them (if wanted).
using DistillResult = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;
DistillResult distill_outputs(const at::Tensor& logits, const at::Tensor& indices, int64_t reduction, bool want_pairs) {
  const auto leading = logits.sizes().slice(0, logits.dim() - 1);
  const int64_t stats[] = {logits.numel() / logits.size(-1), 8};
  const bool none = reduction == SUPA_AMD_REDUCTION_NONE;
  std::vector<int64_t> pairs = indices.sizes().vec();
  pairs.push_back(2);
  return {empty_beside(logits, none ? leading : c10::IntArrayRef(), at::kFloat),
          none ? at::Tensor() : empty_beside(logits, {}, at::kFloat), empty_beside(logits, stats, at::kFloat),
          want_pairs ? empty_beside(logits, pairs, at::kInt) : at::Tensor()};
}

#define SUPA_DISTILL_PARAMS                                                                                     \
  const at::Tensor &logits, const at::Tensor &indices, const at::Tensor &teacher, const OptTensor &teacher_lse, \
      double temperature, int64_t reduction

DistillResult distill_run(SUPA_DISTILL_PARAMS, bool want_pairs) {
  check_distill(logits, indices, teacher, teacher_lse, temperature, reduction);
  const c10::DeviceGuard guard(logits.device());
  const DistillResult r = distill_outputs(logits, indices, reduction, want_pairs);
  const auto& [loss, count, stats, pairs] = r;
  const LogitRows x = logit_rows(logits);
  const LogitRows ids = rows_beside(indices, x.inner, true), t = rows_beside(teacher, x.inner, true);
  supa_amd_distill_desc d = distill_desc(x, indices.size(-1), temperature, reduction);
  d.index_dtype = dtype_code(indices.scalar_type());
  d.indices = ids.t.data_ptr();
  d.teacher_dtype = dtype_code(teacher.scalar_type());
  d.teacher = t.t.data_ptr();
  LogitRows lse{};
  const bool lse64 = given(teacher_lse) && teacher_lse->scalar_type() == at::kDouble;
  if (given(teacher_lse)) lse = rows_beside(lse64 ? *teacher_lse : teacher_lse->to(at::kFloat), x.inner, false);
  for (int i = 0; i < 2; ++i) {
    d.indices_strides[i] = ids.stride[i];
    d.teacher_strides[i] = t.stride[i];
    d.lse_strides[i] = lse.stride[i];
  }
  // an empty tensor has no address, and says "given" all the same: there are no rows then
  if (lse.t.defined() && !lse64) d.teacher_lse = lse.t.data_ptr<float>();
  const auto dev = logits.device().index();
  const int64_t ws_bytes = supa_amd_distill_workspace_bytes(&d);
  TORCH_CHECK(ws_bytes >= 0, "distillation_loss: ", supa_amd_status_string((int)ws_bytes));
  const at::Tensor ws = empty_supa({ws_bytes}, at::kByte, dev);
  float* const counts = count.defined() ? count.data_ptr<float>() : nullptr;
  void* const kept = pairs.defined() ? pairs.data_ptr() : nullptr;
  check_status(lse64 ? supa_amd_distill_forward_lse64(&d, lse.t.data_ptr<double>(), loss.data_ptr<float>(), counts,
                                                      stats.data_ptr<float>(), kept, ws.data_ptr(), ws_bytes,
                                                      stream_error_flag(dev), current_stream(dev))
                     : supa_amd_distill_forward(&d, loss.data_ptr<float>(), counts, stats.data_ptr<float>(), kept,
                                                ws.data_ptr(), ws_bytes, stream_error_flag(dev), current_stream(dev)),
               "distillation_loss");
  return r;
}

at::Tensor distillation_loss(SUPA_DISTILL_PARAMS) {
  return std::get<0>(distill_run(logits, indices, teacher, teacher_lse, temperature, reduction, false));
}
DistillResult distillation_loss_forward(SUPA_DISTILL_PARAMS) {
  return distill_run(logits, indices, teacher, teacher_lse, temperature, reduction, true);
}
at::Tensor distillation_loss_meta(SUPA_DISTILL_PARAMS) {
  check_distill(logits, indices, teacher, teacher_lse, temperature, reduction);
  return std::get<0>(distill_outputs(logits, indices, reduction, false));
}
DistillResult distillation_loss_forward_meta(SUPA_DISTILL_PARAMS) {
  check_distill(logits, indices, teacher, teacher_lse, temperature, reduction);
  return distill_outputs(logits, indices, reduction, true);
}

#define SUPA_DISTILL_BACKWARD_PARAMS                                                                             \
  const at::Tensor &grad_loss, const at::Tensor &logits, const OptTensor &count, const at::Tensor &stats,        \
      const at::Tensor &pairs, double temperature, int64_t reduction

at::Tensor distill_grad(SUPA_DISTILL_BACKWARD_PARAMS) {
  constexpr const char* op = "distillation_loss (backward)";
  check_distill_logits(op, logits, temperature, reduction);
  const int64_t rows[] = {logits.numel() / logits.size(-1), 8};
  const bool none = reduction == SUPA_AMD_REDUCTION_NONE;
  const auto check = [&](const char* name, const at::Tensor& t, c10::IntArrayRef sizes) {
    check_on(op, name, t, logits);
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.sizes() == sizes, op, ": expected ", name, " of Float and shape ", sizes,
                ", got ", t.scalar_type(), " of ", t.sizes());
  };
  check("grad_loss", grad_loss, none ? logits.sizes().slice(0, logits.dim() - 1) : c10::IntArrayRef());
  check("stats", stats, rows);
  check_on(op, "pairs", pairs, logits);
  TORCH_CHECK(pairs.scalar_type() == at::kInt && pairs.dim() == logits.dim() + 1 && pairs.size(-1) == 2 &&
                  pairs.sizes().slice(0, logits.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
              op, ": pairs of ", pairs.scalar_type(), " and shape ", pairs.sizes(), " do not fit logits of shape ", logits.sizes());
  TORCH_CHECK(none || given(count), op, ": expected the count of the rows");
  if (!none) check("count", *count, {});
  return empty_beside(logits, logits.sizes(), logits.scalar_type());
}
at::Tensor distillation_loss_backward(SUPA_DISTILL_BACKWARD_PARAMS) {
  const c10::OptionalDeviceGuard guard(logits.device());
  const at::Tensor grad = distill_grad(grad_loss, logits, count, stats, pairs, temperature, reduction);
  if (logits.numel() == 0) return grad;
  const LogitRows x = logit_rows(logits);
  const at::Tensor g = grad_loss.contiguous(), st = stats.contiguous(), p = pairs.contiguous();
  const supa_amd_distill_desc d = distill_desc(x, p.size(-2), temperature, reduction);
  check_status(supa_amd_distill_backward(&d, g.data_ptr<float>(), static_cast<const float*>(ptr(count)),
                                         st.data_ptr<float>(), p.data_ptr(), grad.data_ptr(),
                                         current_stream(logits.device().index())),
               "distillation_loss (backward)");
  return grad;
}
at::Tensor distillation_loss_backward_meta(SUPA_DISTILL_BACKWARD_PARAMS) {
  return distill_grad(grad_loss, logits, count, stats, pairs, temperature, reduction);
}

// What a node takes back from its saved tensors: hooks on them (offloading, recomputation) may give back others.
void check_back(const char* op, const at::Tensor& t, const c10::Device& device) {
  TORCH_CHECK(t.defined() && t.device() == device, op, ": a saved tensor came back on ",
              t.defined() ? t.device() : c10::Device(at::kCPU), ", expected ", device);
}

struct DistillationLossBackward final : public torch::autograd::Node {
  std::string name() const override { return "DistillationLossBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&logits, &count, &stats, &pairs}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    check_once("distillation_loss");
    variable_list out(1);
    if (!grads[0].defined() || !task_should_compute_output(0)) return out;
    std::lock_guard<std::mutex> lock(mutex_);
    const at::Tensor x = logits.unpack(shared_from_this()), c = count.unpack(shared_from_this()),
                     s = stats.unpack(shared_from_this()), p = pairs.unpack(shared_from_this());
    for (const at::Tensor* t : {&x, &s, &p}) check_back("distillation_loss", *t, grads[0].device());
    static const auto op = find_op<decltype(distillation_loss_backward)>("supa::_distillation_loss_backward");
    const at::AutoDispatchBelowAutograd below;
    out[0] = op.call(grads[0], x, maybe(c), s, p, temperature, reduction);
    return out;
  }
  SavedVariable logits, count, stats, pairs;
  double temperature;
  int64_t reduction;
};

at::Tensor distillation_loss_autograd(c10::DispatchKeySet ks, SUPA_DISTILL_PARAMS) {
  check_no_tangent("distillation_loss", {&logits, &teacher, &tensor(teacher_lse)});
  if (at::GradMode::is_enabled())
    TORCH_CHECK(!teacher.requires_grad() && !(given(teacher_lse) && teacher_lse->requires_grad()),
                "distillation_loss: the teacher has no gradient; detach teacher_logits and teacher_lse");
  if (!logits.requires_grad() || !at::GradMode::is_enabled()) {
    static const auto op = find_op<decltype(distillation_loss)>("supa::distillation_loss");
    const at::AutoDispatchBelowAutograd below;
    return op.redispatch(ks & c10::after_autograd_keyset, logits, indices, teacher, teacher_lse, temperature, reduction);
  }
  check_distill(logits, indices, teacher, teacher_lse, temperature, reduction);
  auto node = std::shared_ptr<DistillationLossBackward>(new DistillationLossBackward(), torch::autograd::deleteNode);
  node->set_next_edges({torch::autograd::impl::gradient_edge(logits)});
  node->temperature = temperature;
  node->reduction = reduction;
  at::Tensor x, loss, count, stats, pairs;
  {
    static const auto op = find_op<decltype(distillation_loss_forward)>("supa::_distillation_loss_forward");
    const at::AutoDispatchBelowAutograd below;
    x = logit_rows(logits).t;  // a copy is made once, for both ways
    std::tie(loss, count, stats, pairs) = op.call(x, indices, teacher, teacher_lse, temperature, reduction);
  }
  node->logits = SavedVariable(x, false);
  if (count.defined()) node->count = SavedVariable(count, false);
  node->stats = SavedVariable(stats, false);
  node->pairs = SavedVariable(pairs, false);
  torch::autograd::set_history(loss, node);
  return loss;
}

// ----------------------------------------------------- router_balance_loss
// The logits as [sequences, tokens, experts].
struct BalanceShape {
  int64_t sequences, tokens, experts;
};
BalanceShape check_balance_sizes(const char* op, const at::Tensor& logits, const OptTensor& mask, int64_t k, int64_t scores,
                                 bool per_sequence) {
  TORCH_CHECK(is_supa(logits), op, ": expected supa tensors, got logits on ", logits.device());
  TORCH_CHECK(is_float16_or_32(logits.scalar_type()), op, ": expected float32, bfloat16 or float16, got logits of ",
              logits.scalar_type());
  TORCH_CHECK(logits.dim() >= (per_sequence ? 2 : 1), op, ": expected logits of shape ",
              per_sequence ? "[..., tokens, experts]" : "[..., experts]", ", got ", logits.sizes());
  const int64_t experts = logits.size(-1);
  TORCH_CHECK(experts >= 1 && experts <= 1024, op, ": expected 1 to 1024 experts, got ", experts);
  TORCH_CHECK(k >= 1 && k <= experts, op, ": expected 1 to ", experts, " choices a token, got ", k);
  const int64_t rows = logits.numel() / experts;
  TORCH_CHECK(rows < (int64_t(1) << 31), op, ": expected fewer than 2^31 tokens");
  TORCH_CHECK(scores == SUPA_AMD_SCORES_SOFTMAX || scores == SUPA_AMD_SCORES_SIGMOID, op, ": no scores have number ", scores);
  if (given(mask)) {
    check_on(op, "mask", *mask, logits);
    TORCH_CHECK(mask->scalar_type() == at::kBool && mask->sizes() == logits.sizes().slice(0, logits.dim() - 1), op,
                ": expected mask as bools of shape ", logits.sizes().slice(0, logits.dim() - 1), ", got ",
                mask->scalar_type(), " of shape ", mask->sizes());
  }
  if (!per_sequence) return {1, rows, experts};
  int64_t sequences = 1;
  for (int64_t i = 0; i < logits.dim() - 2; ++i) sequences *= logits.size(i);
  return {sequences, logits.size(-2), experts};
}
BalanceShape check_balance(const at::Tensor& logits, const at::Tensor& chosen, const OptTensor& mask, int64_t scores,
                           bool per_sequence) {
  constexpr const char* op = "router_balance_loss";
  TORCH_CHECK(chosen.dim() >= 1, op, ": expected experts of shape [..., k], got a scalar");
  const BalanceShape s = check_balance_sizes(op, logits, mask, chosen.size(-1), scores, per_sequence);
  check_on(op, "experts", chosen, logits);
  TORCH_CHECK(is_index(chosen.scalar_type()), op, ": expected int64 or int32 experts, got ", chosen.scalar_type());
  TORCH_CHECK(chosen.dim() == logits.dim() && chosen.sizes().slice(0, logits.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
              op, ": experts of shape ", chosen.sizes(), " do not fit logits of shape ", logits.sizes(),
              ": they differ in the last dim alone");
  return s;
}

supa_amd_balance_desc balance_desc(const BalanceShape& s, const at::Tensor& logits, const OptTensor& mask, int64_t k,
                                   int64_t scores) {
  supa_amd_balance_desc d{};
  d.sequences = s.sequences;
  d.tokens = s.tokens;
  d.experts = s.experts;
  d.k = k;
  d.dtype = dtype_code(logits.scalar_type());
  d.index_dtype = SUPA_AMD_I64;
  d.scores = (int32_t)scores;
  d.logits = logits.data_ptr();
  d.mask = ptr(mask);
  return d;
}

// loss, counts, and for the backward the experts' loads and the sequences' scales.
using BalanceResult = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;
BalanceResult balance_outputs(const at::Tensor& logits, const BalanceShape& s, bool per_sequence) {
  std::vector<int64_t> counts;
  if (per_sequence) counts = logits.sizes().slice(0, logits.dim() - 2).vec();
  counts.push_back(s.experts);
  return {empty_beside(logits, {}, at::kFloat), empty_beside(logits, counts, at::kLong),
          empty_beside(logits, counts, at::kFloat), empty_beside(logits, {s.sequences + 1}, at::kFloat)};
}

#define SUPA_BALANCE_PARAMS \
  const at::Tensor &logits, const at::Tensor &chosen, const OptTensor &mask, int64_t scores, bool per_sequence

BalanceResult router_balance_loss_forward(SUPA_BALANCE_PARAMS) {
  const BalanceShape s = check_balance(logits, chosen, mask, scores, per_sequence);
  const c10::DeviceGuard guard(logits.device());
  const BalanceResult r = balance_outputs(logits, s, per_sequence);
  const auto& [loss, counts, load, scale] = r;
  if (s.sequences == 0) {
    loss.zero_();
    return r;
  }
  const at::Tensor x = logits.contiguous(), ids = chosen.contiguous();
  const OptTensor m = contiguous(mask);
  supa_amd_balance_desc d = balance_desc(s, x, m, ids.size(-1), scores);
  d.index_dtype = dtype_code(ids.scalar_type());
  d.chosen = ids.data_ptr();
  const auto dev = logits.device().index();
  const int64_t ws_bytes = supa_amd_balance_workspace_bytes(&d);
  TORCH_CHECK(ws_bytes >= 0, "router_balance_loss: ", supa_amd_status_string((int)ws_bytes));
  const at::Tensor ws = empty_supa({ws_bytes}, at::kByte, dev);
  check_status(supa_amd_balance_forward(&d, loss.data_ptr<float>(), counts.data_ptr<int64_t>(), load.data_ptr<float>(),
                                        scale.data_ptr<float>(), ws.data_ptr(), ws_bytes, stream_error_flag(dev),
                                        current_stream(dev)),
               "router_balance_loss");
  return r;
}
std::tuple<at::Tensor, at::Tensor> router_balance_loss(SUPA_BALANCE_PARAMS) {
  auto [loss, counts, load, scale] = router_balance_loss_forward(logits, chosen, mask, scores, per_sequence);
  return {loss, counts};
}
BalanceResult router_balance_loss_forward_meta(SUPA_BALANCE_PARAMS) {
  return balance_outputs(logits, check_balance(logits, chosen, mask, scores, per_sequence), per_sequence);
}
std::tuple<at::Tensor, at::Tensor> router_balance_loss_meta(SUPA_BALANCE_PARAMS) {
  auto [loss, counts, load, scale] = router_balance_loss_forward_meta(logits, chosen, mask, scores, per_sequence);
  return {loss, counts};
}

#define SUPA_BALANCE_BACKWARD_PARAMS                                                                                 \
  const at::Tensor &grad_loss, const at::Tensor &logits, const OptTensor &mask, const at::Tensor &load,              \
      const at::Tensor &scale, int64_t k, int64_t scores, bool per_sequence

at::Tensor balance_grad(SUPA_BALANCE_BACKWARD_PARAMS) {
  constexpr const char* op = "router_balance_loss (backward)";
  const BalanceShape s = check_balance_sizes(op, logits, mask, k, scores, per_sequence);
  const auto check = [&](const char* name, const at::Tensor& t, int64_t n) {
    check_on(op, name, t, logits);
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.numel() == n, op, ": expected ", name, " as ", n, " floats, got ",
                t.scalar_type(), " of ", t.sizes());
  };
  check("grad_loss", grad_loss, 1);
  check("load", load, s.sequences * s.experts);
  check("scale", scale, s.sequences + 1);
  return empty_beside(logits, logits.sizes(), logits.scalar_type());
}
at::Tensor router_balance_loss_backward(SUPA_BALANCE_BACKWARD_PARAMS) {
  const c10::OptionalDeviceGuard guard(logits.device());
  const at::Tensor grad = balance_grad(grad_loss, logits, mask, load, scale, k, scores, per_sequence);
  if (logits.numel() == 0) return grad;
  const at::Tensor x = logits.contiguous(), g = grad_loss.contiguous(), l = load.contiguous(), sc = scale.contiguous();
  const OptTensor m = contiguous(mask);
  const BalanceShape s = check_balance_sizes("router_balance_loss", logits, mask, k, scores, per_sequence);
  const supa_amd_balance_desc d = balance_desc(s, x, m, k, scores);
  check_status(supa_amd_balance_backward(&d, g.data_ptr<float>(), l.data_ptr<float>(), sc.data_ptr<float>(),
                                         grad.data_ptr(), current_stream(logits.device().index())),
               "router_balance_loss (backward)");
  return grad;
}
at::Tensor router_balance_loss_backward_meta(SUPA_BALANCE_BACKWARD_PARAMS) {
  return balance_grad(grad_loss, logits, mask, load, scale, k, scores, per_sequence);
}

struct RouterBalanceLossBackward final : public torch::autograd::Node {
  std::string name() const override { return "RouterBalanceLossBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&logits, &mask, &load, &scale}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    check_once("router_balance_loss");
    variable_list out(1);
    if (!grads[0].defined() || !task_should_compute_output(0)) return out;
    std::lock_guard<std::mutex> lock(mutex_);
    const at::Tensor x = logits.unpack(shared_from_this()), m = mask.unpack(shared_from_this()),
                     l = load.unpack(shared_from_this()), s = scale.unpack(shared_from_this());
    for (const at::Tensor* t : {&x, &l, &s}) check_back("router_balance_loss", *t, grads[0].device());
    static const auto op = find_op<decltype(router_balance_loss_backward)>("supa::_router_balance_loss_backward");
    const at::AutoDispatchBelowAutograd below;
    out[0] = op.call(grads[0], x, maybe(m), l, s, k, scores, per_sequence);
    return out;
  }
  SavedVariable logits, mask, load, scale;
  int64_t k, scores;
  bool per_sequence;
};

std::tuple<at::Tensor, at::Tensor> router_balance_loss_autograd(c10::DispatchKeySet ks, SUPA_BALANCE_PARAMS) {
  check_no_tangent("router_balance_loss", {&logits});
  if (!logits.requires_grad() || !at::GradMode::is_enabled()) {
    static const auto op = find_op<decltype(router_balance_loss)>("supa::router_balance_loss");
    const at::AutoDispatchBelowAutograd below;
    return op.redispatch(ks & c10::after_autograd_keyset, logits, chosen, mask, scores, per_sequence);
  }
  check_balance(logits, chosen, mask, scores, per_sequence);
  auto node = std::shared_ptr<RouterBalanceLossBackward>(new RouterBalanceLossBackward(), torch::autograd::deleteNode);
  node->set_next_edges({torch::autograd::impl::gradient_edge(logits)});
  node->k = chosen.size(-1);
  node->scores = scores;
  node->per_sequence = per_sequence;
  at::Tensor x, loss, counts, load, scale;
  OptTensor m;
  {
    static const auto op = find_op<decltype(router_balance_loss_forward)>("supa::_router_balance_loss_forward");
    const at::AutoDispatchBelowAutograd below;
    x = logits.contiguous();  // a copy is made once, for both ways
    m = contiguous(mask);
    std::tie(loss, counts, load, scale) = op.call(x, chosen, m, scores, per_sequence);
  }
  node->logits = SavedVariable(x, false);
  if (given(m)) node->mask = SavedVariable(*m, false);
  node->load = SavedVariable(load, false);
  node->scale = SavedVariable(scale, false);
  torch::autograd::set_history(loss, node);
  return {loss, counts};
}

// ----------------------------------------------------------- adjust_logits
// A parameter of each row: a tensor, or a number for all of them.
#define SUPA_ADJUST_PARAMS                                                                                        \
  const OptTensor &tokens, const OptTensor &lengths, const OptTensor &prompt_lengths, const OptTensor &repetition, \
      double repetition_value, const OptTensor &presence, double presence_value, const OptTensor &frequency,      \
      double frequency_value, const OptTensor &bias_tokens, const OptTensor &bias, const OptTensor &allowed
#define SUPA_ADJUST_ARGS                                                                                       \
  tokens, lengths, prompt_lengths, repetition, repetition_value, presence, presence_value, frequency,          \
      frequency_value, bias_tokens, bias, allowed

void check_adjust(const char* op, const at::Tensor& logits, SUPA_ADJUST_PARAMS) {
  TORCH_CHECK(is_supa(logits), op, ": expected supa tensors, got logits on ", logits.device());
  TORCH_CHECK(is_float16_or_32(logits.scalar_type()), op, ": expected float32, bfloat16 or float16, got logits of ",
              logits.scalar_type());
  TORCH_CHECK((logits.dim() == 1 || logits.dim() == 2) && logits.size(-1) >= 1, op,
              ": expected logits of shape [vocab] or [rows, vocab], got ", logits.sizes());
  TORCH_CHECK(logits.size(-1) < (int64_t(1) << 29), op, ": expected fewer than 2^29 tokens, got ", logits.size(-1));
  const bool batch = logits.dim() == 2;
  const int64_t rows = batch ? logits.size(0) : 1;
  TORCH_CHECK(rows < (int64_t(1) << 31), op, ": expected fewer than 2^31 rows");
  // a row of values for each row of logits; `shared`: or one for all
  const auto check_rows = [&](const char* name, const OptTensor& t, bool shared) {
    if (!given(t)) return;
    check_on(op, name, *t, logits);
    TORCH_CHECK((t->dim() == 2 && batch && t->size(0) == rows) || (t->dim() == 1 && (shared || !batch)), op,
                ": expected ", name, " of shape ", batch ? "[rows, n]" : "[n]", shared && batch ? " or [n]" : "",
                ", got ", t->sizes(), " for logits of shape ", logits.sizes());
  };
  const auto check_value = [&](const char* name, const OptTensor& t, bool index) {
    if (!given(t)) return;
    check_on(op, name, *t, logits);
    TORCH_CHECK(index ? is_index(t->scalar_type()) : t->scalar_type() == at::kFloat, op, ": expected ", name, " of ",
                index ? "int64 or int32" : "float32", ", got ", t->scalar_type());
    TORCH_CHECK(t->dim() == (batch ? 1 : 0) && t->numel() == rows, op, ": expected ", name, " of shape [",
                batch ? std::to_string(rows) : "", "], got ", t->sizes());
  };
  check_rows("tokens", tokens, false);
  if (given(tokens)) {
    TORCH_CHECK(is_index(tokens->scalar_type()), op, ": expected int64 or int32 tokens, got ", tokens->scalar_type());
    TORCH_CHECK(tokens->size(-1) < (int64_t(1) << 31), op, ": expected a history of fewer than 2^31 tokens");
  }
  check_value("lengths", lengths, true);
  check_value("prompt_lengths", prompt_lengths, true);
  check_value("repetition", repetition, false);
  check_value("presence", presence, false);
  check_value("frequency", frequency, false);
  // as float32, which the kernel takes them in
  TORCH_CHECK(std::isfinite((float)repetition_value) && (float)repetition_value > 0, op, ": expected repetition > 0, got ", repetition_value);
  TORCH_CHECK(std::isfinite((float)presence_value) && std::isfinite((float)frequency_value), op, ": expected finite penalties, got ",
              presence_value, " and ", frequency_value);
  const bool penalties = given(repetition) || given(presence) || given(frequency) || repetition_value != 1.0 ||
                         presence_value != 0.0 || frequency_value != 0.0;
  TORCH_CHECK(given(tokens) || !(penalties || given(lengths) || given(prompt_lengths)), op,
              ": penalties and lengths need the tokens of the history");
  TORCH_CHECK(given(bias_tokens) == given(bias), op, ": bias_tokens and bias are given together");
  if (given(bias)) {
    check_rows("bias_tokens", bias_tokens, true);
    check_rows("bias", bias, true);
    TORCH_CHECK(is_index(bias_tokens->scalar_type()) && bias->scalar_type() == at::kFloat, op,
                ": expected int64 or int32 bias_tokens and a float32 bias, got ", bias_tokens->scalar_type(), " and ",
                bias->scalar_type());
    TORCH_CHECK(bias_tokens->size(-1) == bias->size(-1) && bias->size(-1) < (int64_t(1) << 30), op, ": bias_tokens hold ",
                bias_tokens->size(-1), " tokens a row, bias ", bias->size(-1), " values");
  }
  if (given(allowed)) {
    check_rows("allowed", allowed, true);
    const int64_t words = (logits.size(-1) + 31) / 32;
    TORCH_CHECK(allowed->scalar_type() == at::kInt && allowed->size(-1) >= words, op,
                ": expected allowed as int32 words of 32 tokens, at least ", words, " a row, got ", allowed->scalar_type(),
                " of shape ", allowed->sizes());
  }
}

// Rows whose elements are contiguous.
at::Tensor row_contiguous(const OptTensor& t) {
  if (!given(t)) return {};
  return t->size(-1) <= 1 || t->stride(-1) == 1 ? *t : t->contiguous();
}
int64_t row_stride(const at::Tensor& t) { return t.defined() && t.dim() == 2 && t.size(0) > 1 ? t.stride(0) : 0; }

void launch_adjust(const char* op, const at::Tensor& in, const at::Tensor& out, SUPA_ADJUST_PARAMS) {
  if (in.numel() == 0) return;
  const at::Tensor tok = row_contiguous(tokens), bt = row_contiguous(bias_tokens), b = row_contiguous(bias),
                   mask = row_contiguous(allowed);
  const OptTensor len = contiguous(lengths), prompt = contiguous(prompt_lengths), rep = contiguous(repetition),
                  pres = contiguous(presence), freq = contiguous(frequency);
  supa_amd_adjust_desc d{};
  d.rows = in.dim() == 2 ? in.size(0) : 1;
  d.vocab = in.size(-1);
  d.dtype = dtype_code(in.scalar_type());
  d.in = in.data_ptr();
  d.out = out.data_ptr();
  d.in_stride = row_stride(in);
  d.out_stride = row_stride(out);
  d.repetition_value = repetition_value;
  d.presence_value = presence_value;
  d.frequency_value = frequency_value;
  if (tok.defined() && tok.numel() > 0) {
    d.history = tok.size(-1);
    d.tokens = tok.data_ptr();
    d.tokens_stride = row_stride(tok);
    d.token_dtype = dtype_code(tok.scalar_type());
    const auto values = [](const OptTensor& t) { return static_cast<const float*>(ptr(t)); };
    d.repetition = values(rep);
    d.presence = values(pres);
    d.frequency = values(freq);
    d.lengths = ptr(len);
    d.prompt_lengths = ptr(prompt);
    if (given(len)) d.length_dtype = dtype_code(len->scalar_type());
    if (given(prompt)) d.prompt_dtype = dtype_code(prompt->scalar_type());
  }
  if (b.defined() && b.size(-1) > 0) {
    d.biases = b.size(-1);
    d.bias_tokens = bt.data_ptr();
    d.bias_token_dtype = dtype_code(bt.scalar_type());
    d.bias = b.data_ptr<float>();
    d.bias_tokens_stride = row_stride(bt);
    d.bias_stride = row_stride(b);
  }
  if (mask.defined()) {
    d.allowed = static_cast<const uint32_t*>(mask.data_ptr());
    d.allowed_stride = row_stride(mask);
  }
  check_status(supa_amd_adjust_logits(&d, current_stream(in.device().index())), op);
}

at::Tensor adjust_logits(const at::Tensor& logits, SUPA_ADJUST_PARAMS) {
  constexpr const char* op = "adjust_logits";
  check_adjust(op, logits, SUPA_ADJUST_ARGS);
  const c10::OptionalDeviceGuard guard(logits.device());
  const at::Tensor out = empty_beside(logits, logits.sizes(), logits.scalar_type());
  if (!logits.is_meta()) launch_adjust(op, row_contiguous(logits), out, SUPA_ADJUST_ARGS);
  return out;
}

void adjust_logits_(at::Tensor& logits, SUPA_ADJUST_PARAMS) {
  constexpr const char* op = "adjust_logits_";
  check_adjust(op, logits, SUPA_ADJUST_ARGS);
  const c10::OptionalDeviceGuard guard(logits.device());
  if (logits.numel() == 0) return;
  TORCH_CHECK(logits.size(-1) == 1 || logits.stride(-1) == 1, op, ": expected rows whose elements are contiguous");
  const Steps steps = steps_of(logits);
  TORCH_CHECK(apart(steps, steps.size(), (int64_t)logits.element_size()), op, ": expected logits whose rows do not overlap in memory");
  if (logits.is_meta()) return;
  for (const OptTensor* t : {&tokens, &lengths, &prompt_lengths, &repetition, &presence, &frequency, &bias_tokens, &bias, &allowed})
    if (given(*t) && (*t)->numel() > 0 && (*t)->storage().is_alias_of(logits.storage()))
      TORCH_CHECK(beside(logits, **t), op, ": another argument shares memory with the logits");
  launch_adjust(op, logits, logits, SUPA_ADJUST_ARGS);
}

void check_adjust_gradients(const char* op, const at::Tensor& logits, SUPA_ADJUST_PARAMS) {
  check_no_tangent(op, {&logits, &tensor(repetition), &tensor(presence), &tensor(frequency), &tensor(bias)});
  if (!at::GradMode::is_enabled()) return;
  bool needs = logits.requires_grad();
  for (const OptTensor* t : {&repetition, &presence, &frequency, &bias}) needs = needs || (given(*t) && (*t)->requires_grad());
  TORCH_CHECK(!needs, op, ": no gradient; call it under torch.no_grad() or on detached tensors");
}

at::Tensor adjust_logits_autograd(c10::DispatchKeySet ks, const at::Tensor& logits, SUPA_ADJUST_PARAMS) {
  check_adjust_gradients("adjust_logits", logits, SUPA_ADJUST_ARGS);
  static const auto op = find_op<decltype(adjust_logits)>("supa::adjust_logits");
  const at::AutoDispatchBelowAutograd below;
  return op.redispatch(ks & c10::after_autograd_keyset, logits, SUPA_ADJUST_ARGS);
}

c10::TypedOperatorHandle<decltype(adjust_logits_)> adjust_op_() {
  static const auto op = find_op<decltype(adjust_logits_)>("supa::adjust_logits_");
  return op;
}
void adjust_logits_autograd_(c10::DispatchKeySet ks, at::Tensor& logits, SUPA_ADJUST_PARAMS) {
  check_adjust_gradients("adjust_logits_", logits, SUPA_ADJUST_ARGS);
  const at::AutoDispatchBelowAutograd below;
  adjust_op_().redispatch(ks & c10::after_autograd_keyset, logits, SUPA_ADJUST_ARGS);
}
void adjust_logits_versions_(c10::DispatchKeySet ks, at::Tensor& logits, SUPA_ADJUST_PARAMS) {
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    adjust_op_().redispatch(ks & c10::after_ADInplaceOrView_keyset, logits, SUPA_ADJUST_ARGS);
  }
  written(logits);
}

}  // namespace
}  // namespace supa

TORCH_LIBRARY_FRAGMENT(supa, m) {
  m.def(
      "distillation_loss(Tensor logits, Tensor indices, Tensor teacher_logits, Tensor? teacher_lse, float temperature, "
      "int reduction) -> Tensor");
  // its parts for training: the count, the rows' statistics and the pairs beside the loss
  m.def(
      "_distillation_loss_forward(Tensor logits, Tensor indices, Tensor teacher_logits, Tensor? teacher_lse, float "
      "temperature, int reduction) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "_distillation_loss_backward(Tensor grad_loss, Tensor logits, Tensor? count, Tensor stats, Tensor pairs, "
      "float temperature, int reduction) -> Tensor");
  m.def(
      "router_balance_loss(Tensor logits, Tensor experts, Tensor? mask, int scores, bool per_sequence) -> (Tensor, Tensor)");
  m.def(
      "_router_balance_loss_forward(Tensor logits, Tensor experts, Tensor? mask, int scores, bool per_sequence) -> "
      "(Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "_router_balance_loss_backward(Tensor grad_loss, Tensor logits, Tensor? mask, Tensor load, Tensor scale, int k, "
      "int scores, bool per_sequence) -> Tensor");
#define SUPA_ADJUST_SCHEMA                                                                                        \
  "Tensor? tokens, Tensor? lengths, Tensor? prompt_lengths, Tensor? repetition, float repetition_value, Tensor? " \
  "presence, float presence_value, Tensor? frequency, float frequency_value, Tensor? bias_tokens, Tensor? bias, " \
  "Tensor? allowed)"
  m.def("adjust_logits(Tensor logits, " SUPA_ADJUST_SCHEMA " -> Tensor");
  m.def("adjust_logits_(Tensor(a!) logits, " SUPA_ADJUST_SCHEMA " -> ()");
}

TORCH_LIBRARY_IMPL(supa, PrivateUse1, m) {
  using namespace supa;
  m.impl("distillation_loss", TORCH_FN(distillation_loss));
  m.impl("_distillation_loss_forward", TORCH_FN(distillation_loss_forward));
  m.impl("_distillation_loss_backward", TORCH_FN(distillation_loss_backward));
  m.impl("router_balance_loss", TORCH_FN(router_balance_loss));
  m.impl("_router_balance_loss_forward", TORCH_FN(router_balance_loss_forward));
  m.impl("_router_balance_loss_backward", TORCH_FN(router_balance_loss_backward));
  m.impl("adjust_logits", TORCH_FN(adjust_logits));
  m.impl("adjust_logits_", TORCH_FN(adjust_logits_));
}

TORCH_LIBRARY_IMPL(supa, Meta, m) {
  using namespace supa;
  m.impl("distillation_loss", TORCH_FN(distillation_loss_meta));
  m.impl("_distillation_loss_forward", TORCH_FN(distillation_loss_forward_meta));
  m.impl("_distillation_loss_backward", TORCH_FN(distillation_loss_backward_meta));
  m.impl("router_balance_loss", TORCH_FN(router_balance_loss_meta));
  m.impl("_router_balance_loss_forward", TORCH_FN(router_balance_loss_forward_meta));
  m.impl("_router_balance_loss_backward", TORCH_FN(router_balance_loss_backward_meta));
  m.impl("adjust_logits", TORCH_FN(adjust_logits));
  m.impl("adjust_logits_", TORCH_FN(adjust_logits_));
}

namespace supa {
namespace {
void logit_autograd_kernels(torch::Library& m) {
  m.impl("distillation_loss", TORCH_FN(distillation_loss_autograd));
  m.impl("router_balance_loss", TORCH_FN(router_balance_loss_autograd));
  m.impl("adjust_logits", TORCH_FN(adjust_logits_autograd));
  m.impl("adjust_logits_", TORCH_FN(adjust_logits_autograd_));
}
}  // namespace
}  // namespace supa
TORCH_LIBRARY_IMPL(supa, AutogradPrivateUse1, m) { supa::logit_autograd_kernels(m); }
TORCH_LIBRARY_IMPL(supa, Autograd, m) { supa::logit_autograd_kernels(m); }  // meta tensors, and wrappers of any
TORCH_LIBRARY_IMPL(supa, ADInplaceOrView, m) { m.impl("adjust_logits_", TORCH_FN(supa::adjust_logits_versions_)); }
