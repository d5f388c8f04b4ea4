// C entry points of the gated residual with the norms around it; its kernels
// are residual_norm.h's, compiled for each type in residual_norm_*.hip.
#include "residual_norm.h"

namespace sa {

#define SA_RN_EXTERN(T, R)                                                                                       \
  extern template int rn_forward_t<T, R>(const supa_amd_residual_norm_desc*, const RnArgs&, void*, void*, float*, \
                                         hipStream_t);                                                          \
  extern template int rn_backward_t<T, R>(const supa_amd_residual_norm_desc*, const RnArgs&, const RnPlan&,      \
                                          const RnGrads&, int, void*, void*, void*, void*, void*, hipStream_t);
SA_RN_EXTERN(float, float)
SA_RN_EXTERN(bf16, bf16)
SA_RN_EXTERN(bf16, float)
SA_RN_EXTERN(f16, f16)
SA_RN_EXTERN(f16, float)
#undef SA_RN_EXTERN

struct RnFns {
  decltype(&rn_forward_t<float, float>) forward;
  decltype(&rn_backward_t<float, float>) backward;
};
template <typename F> int rn_with(const supa_amd_residual_norm_desc& d, F&& go) {
  const bool wide = d.residual_dtype == SUPA_AMD_F32;
  switch (d.dtype) {
    case SUPA_AMD_F32: return go(RnFns{rn_forward_t<float, float>, rn_backward_t<float, float>});
    case SUPA_AMD_BF16:
      return wide ? go(RnFns{rn_forward_t<bf16, float>, rn_backward_t<bf16, float>})
                  : go(RnFns{rn_forward_t<bf16, bf16>, rn_backward_t<bf16, bf16>});
    default:
      return wide ? go(RnFns{rn_forward_t<f16, float>, rn_backward_t<f16, float>})
                  : go(RnFns{rn_forward_t<f16, f16>, rn_backward_t<f16, f16>});
  }
}

}  // namespace sa

using namespace sa;

extern "C" {

int supa_amd_residual_norm_forward(const supa_amd_residual_norm_desc* d, void* h, void* y, float* stats, void* stream) {
  const int rc = rn_check(d);
  if (rc) return rc;
  if (d->rows == 0) return SUPA_AMD_OK;
  if (!d->x || !d->residual || !h || (d->norm != SUPA_AMD_NORM_NONE) != (y != nullptr)) return SUPA_AMD_EINVAL;
  if (!aligned(stats, 16)) return SUPA_AMD_EINVAL;
  const RnArgs a = rn_args(*d);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return rn_with(*d, [&](auto fns) { return fns.forward(d, a, h, y, stats, st); });
}

int64_t supa_amd_residual_norm_backward_workspace_bytes(const supa_amd_residual_norm_desc* d) {
  const int rc = rn_check(d);
  if (rc) return rc;
  if (d->rows == 0) return 0;
  return (int64_t)rn_plan(*d).parts * 5 * d->width * 4;
}

int supa_amd_residual_norm_backward(const supa_amd_residual_norm_desc* d, const void* h, const void* grad_h,
                                    const void* grad_y, const float* stats, void* grad_x, void* grad_residual,
                                    void* grad_gate, void* grad_post_weight, void* grad_post_bias, void* grad_weight,
                                    void* grad_bias, void* workspace, int64_t ws_bytes, void* stream) {
  const int rc = rn_check(d);
  if (rc) return rc;
  if (d->rows == 0) return SUPA_AMD_EINVAL;  // the caller's zeros
  const bool post = d->post_norm != SUPA_AMD_NORM_NONE, norm = d->norm != SUPA_AMD_NORM_NONE;
  if ((post || d->gate) && h) return SUPA_AMD_EINVAL;
  if ((post || grad_gate || (norm && !h)) && !d->x) return SUPA_AMD_EINVAL;
  if (norm && !h && !d->residual) return SUPA_AMD_EINVAL;
  if (((post || norm) && !stats) || !aligned(stats, 16) || !aligned(workspace, 4)) return SUPA_AMD_EINVAL;
  if ((!d->gate && grad_gate) || (!post && (grad_post_weight || grad_post_bias)) || (!norm && (grad_weight || grad_bias)))
    return SUPA_AMD_EINVAL;
  if ((d->post_norm != SUPA_AMD_NORM_LAYER && grad_post_bias) || (d->norm != SUPA_AMD_NORM_LAYER && grad_bias))
    return SUPA_AMD_EINVAL;
  const int64_t need = supa_amd_residual_norm_backward_workspace_bytes(d);
  if (!workspace || ws_bytes < need) return SUPA_AMD_EWORKSPACE;
  const RnArgs a = rn_args(*d);
  const RnPlan p = rn_plan(*d);
  RnGrads o{};
  o.h = h;
  o.gh = grad_h;
  o.gy = norm ? grad_y : nullptr;
  o.stats = reinterpret_cast<const float4*>(stats);
  o.gx = grad_x;
  o.gres = grad_residual;
  o.ggate = grad_gate;
  o.part = static_cast<float*>(workspace);
  o.section = p.section;
  o.sections = p.sections;
  o.first = p.first;
  o.step = p.step;
  o.span = p.span;
  o.cuts = p.cuts;
  o.per = p.per;
  o.want_gate = !grad_gate ? 0 : p.elementwise ? 2 : 1;
  o.want_pw = grad_post_weight != nullptr;
  o.want_pb = grad_post_bias != nullptr;
  o.want_w = grad_weight != nullptr;
  o.want_b = grad_bias != nullptr;
  const int gate_sums = o.want_gate == 1 && p.cuts > 1 ? 1 : 0;
  o.sums = gate_sums + o.want_pw + o.want_pb + o.want_w + o.want_b;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return rn_with(*d, [&](auto fns) {
    return fns.backward(d, a, p, o, gate_sums, grad_gate, grad_post_weight, grad_post_bias, grad_weight, grad_bias, st);
  });
}

}  // extern "C"
