// rms_norm.hpp -- what the forward (rms_norm.hip) and the backward pass (rms_norm_grad.hip) of
// RMS norm share.
#pragma once

#include "layer_norm.hpp"
#include "quant_rows.hpp"

namespace nh {

// 1 / sqrt of the mean square; NaN where the sum of squares is not finite.
NH_DEV double rms_rstd(double sum, double inv_c, double eps)
{
    const double r = rsqrt_d(sum * inv_c + eps);
    return sum < __builtin_inf() ? r : __builtin_nan("");
}

template <typename T>
struct RmsGradArgs {
    const T *dy, *h, *gamma, *rstd, *dh;  // gamma, dh: may be null
    T *dx;                                // may be null
    T *part;                              // [blocks][cols] partial sums of dgamma, or null
    int64_t rows, cols;
};

// dgamma: may be null.  Defined for both types.
template <typename T>
int launch_rms_grad(const RmsGradArgs<T> &a, T *dgamma);

}  // namespace nh
