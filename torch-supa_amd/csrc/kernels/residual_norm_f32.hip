// residual_norm.h for float32.
#include "residual_norm.h"

namespace sa {

template int rn_forward_t<float, float>(const supa_amd_residual_norm_desc*, const RnArgs&, void*, void*, float*, hipStream_t);
template int rn_backward_t<float, float>(const supa_amd_residual_norm_desc*, const RnArgs&, const RnPlan&, const RnGrads&, int,
                                     void*, void*, void*, void*, void*, hipStream_t);

}  // namespace sa
