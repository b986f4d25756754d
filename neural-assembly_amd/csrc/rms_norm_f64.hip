// rms_norm_f64.hip -- the forward pass of RMS norm and rows to 8 bits for f64 rows.
#include "rms_norm_impl.hpp"

namespace nh {

template int launch_rms<double, false, RMS_VALUES>(const RmsArgs<double> &);
template int launch_rms<double, true, RMS_VALUES>(const RmsArgs<double> &);
template int launch_rms<double, false, RMS_CODES>(const RmsArgs<double> &);
template int launch_rms<double, true, RMS_CODES>(const RmsArgs<double> &);
template int launch_rms<double, false, ROW_CODES>(const RmsArgs<double> &);

}  // namespace nh
