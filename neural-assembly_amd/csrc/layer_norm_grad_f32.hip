// layer_norm_grad_f32.hip -- the backward pass of layer norm and its join, f32 rows.
#include "layer_norm_grad_impl.hpp"

namespace nh {

template int launch_ln_grad<float, LN_PLAIN>(const LnGradArgs<float> &, float *, float *);
template int launch_ln_grad<float, LN_ADD>(const LnGradArgs<float> &, float *, float *);
template int launch_ln_grad<float, LN_DROP>(const LnGradArgs<float> &, float *, float *);

}  // namespace nh
