// rms_norm_grad_f64.hip -- the backward pass of RMS norm, f64 rows.
#include "rms_norm_grad_impl.hpp"

namespace nh {

template int launch_rms_grad<double>(const RmsGradArgs<double> &, double *);

}  // namespace nh
