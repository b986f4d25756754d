// rms_norm_f32.hip -- the forward pass of RMS norm and rows to 8 bits for f32 rows.
#include "rms_norm_impl.hpp"

namespace nh {

template int launch_rms<float, false, RMS_VALUES>(const RmsArgs<float> &);
template int launch_rms<float, true, RMS_VALUES>(const RmsArgs<float> &);
template int launch_rms<float, false, RMS_CODES>(const RmsArgs<float> &);
template int launch_rms<float, true, RMS_CODES>(const RmsArgs<float> &);
template int launch_rms<float, false, ROW_CODES>(const RmsArgs<float> &);

}  // namespace nh
