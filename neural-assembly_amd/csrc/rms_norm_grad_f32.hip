// rms_norm_grad_f32.hip -- the backward pass of RMS norm, f32 rows.
#include "rms_norm_grad_impl.hpp"

namespace nh {

template int launch_rms_grad<float>(const RmsGradArgs<float> &, float *);

}  // namespace nh
