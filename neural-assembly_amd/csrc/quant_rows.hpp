// quant_rows.hpp -- a row's values in 8 bits with one scale: code = 127 w / a rounded to
// the nearest whole number, halves away from zero, a = max |w| over the row, scale = a / 127.
#pragma once

#include "common.hpp"

namespace nh {

// max of |w| over values of which one may be NaN: NaN then.
NH_DEV double amax_comb(double a, double b) { return b > a || b != b ? b : a; }

// The codes of a row whose largest |w| is a.  w / a is taken as w * (127 / a); where that lies
// next to a half the quotient is compared with it exactly (254 |w| against (2 b - 1) a, each
// product with its rounding error), so codes depend on the row's values alone and ties are
// ties.  T = double: rows whose products would leave the range are scaled by a power of two.
template <typename T>
struct RowCodes {
    double a, inv, up;
    bool live;  // finite and not all zero
    NH_DEV explicit RowCodes(double a0) : a(a0), inv(0.0), up(1.0)
    {
        live = a0 > 0.0 && a0 < __builtin_inf();
        if (!live) return;
        if constexpr (sizeof(T) == 8) {
            up = a0 < 0x1p-900 ? 0x1p200 : (a0 > 0x1p900 ? 0x1p-200 : 1.0);
            a = a0 * up;
        }
        inv = 127.0 / a;
    }
    NH_DEV int code(double w) const
    {
        if constexpr (sizeof(T) == 8) w *= up;
        const double m = __builtin_fabs(w), s = m * inv + 0.5;
        double f = __builtin_floor(s);
        const double d = s - f;
        if (__builtin_fabs(d - 0.5) > 0.5 - 1e-9) {
            const double b = __builtin_rint(s), c = b + b - 1.0;
            const double p = 254.0 * m, q = c * a;
            const double over = (p - q) + (__builtin_fma(254.0, m, -p) - __builtin_fma(c, a, -q));
            f = over >= 0.0 ? b : b - 1.0;
        }
        const int i = int(f);
        return live ? (w < 0.0 ? -i : i) : 0;
    }
    // scale of codes that stand for w * by
    NH_DEV T scale(double a0, double by) const
    {
        if (!(a0 < __builtin_inf())) return T(__builtin_nan(""));
        return T(a / 127.0 * by / up);
    }
};

}  // namespace nh
