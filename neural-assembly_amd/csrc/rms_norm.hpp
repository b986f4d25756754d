// rms_norm.hpp -- what the forward (rms_norm_impl.hpp) and the backward pass
// (rms_norm_grad_impl.hpp) of RMS norm share.
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

enum { RMS_VALUES = 0, RMS_CODES = 1, ROW_CODES = 2 };

template <typename T>
struct RmsArgs {
    const T *x, *res, *gamma;  // res: where it is added; gamma: may be null
    T *h, *y, *rstd, *scale;   // h, rstd: may be null; y: values; scale: codes
    int8_t *codes;
    int64_t stride, rows, cols;
    double inv_c, eps;
};

// Defined for both types, every output, ADD where rows are joined.
template <typename T, bool ADD, int OUT>
int launch_rms(const RmsArgs<T> &a);

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
