// layer_norm_grad_f64.hip -- the backward pass of layer norm and its join, f64 rows.
#include "layer_norm_grad_impl.hpp"

namespace nh {

template int launch_ln_grad<double, LN_PLAIN>(const LnGradArgs<double> &, double *, double *);
template int launch_ln_grad<double, LN_ADD>(const LnGradArgs<double> &, double *, double *);
template int launch_ln_grad<double, LN_DROP>(const LnGradArgs<double> &, double *, double *);

}  // namespace nh
