// residual_norm.h for bfloat16, with a residual of bfloat16 or float32.
#include "residual_norm.h"

namespace sa {

template int rn_forward_t<bf16, bf16>(const supa_amd_residual_norm_desc*, const RnArgs&, void*, void*, float*, hipStream_t);
template int rn_backward_t<bf16, bf16>(const supa_amd_residual_norm_desc*, const RnArgs&, const RnPlan&, const RnGrads&, int,
                                     void*, void*, void*, void*, void*, hipStream_t);
template int rn_forward_t<bf16, float>(const supa_amd_residual_norm_desc*, const RnArgs&, void*, void*, float*, hipStream_t);
template int rn_backward_t<bf16, float>(const supa_amd_residual_norm_desc*, const RnArgs&, const RnPlan&, const RnGrads&, int,
                                     void*, void*, void*, void*, void*, hipStream_t);

}  // namespace sa
