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
// ties.  f32 rows take the quotient in float first (within 3 units of 2^-24 of it: of |w| rounded
// to float, of the factor, of the product: 2.3e-5 steps) and only what falls within 5e-5 of a half,
// one value in ten thousand, in double (rows to 8 bits f32 [16384, 4096] 74 -> 66 us, bound by
// double's conversions before).  T = double: rows whose products would leave the range are
// scaled by a power of two.
template <typename T>
struct RowCodes {
    double a, inv, up;
    float inv_f;  // 0: not in float
    bool live;    // finite and not all zero
    NH_DEV explicit RowCodes(double a0) : a(a0), inv(0.0), up(1.0), inv_f(0.0f)
    {
        live = a0 > 0.0 && a0 < __builtin_inf();
        if (!live) return;
        if constexpr (sizeof(T) == 8) {
            up = a0 < 0x1p-900 ? 0x1p200 : (a0 > 0x1p900 ? 0x1p-200 : 1.0);
            a = a0 * up;
        }
        inv = 127.0 / a;
        if (sizeof(T) == 4 && a0 > 0x1p-90 && a0 < 0x1p120) inv_f = float(inv);
    }
    // floor(127 |w| / a + 1/2), m = |w|.
    NH_DEV int whole(double m) const
    {
        if constexpr (sizeof(T) == 8) m *= up;
        const double s = m * inv + 0.5;
        double f = __builtin_floor(s);
        const double d = s - f;
        if (__builtin_fabs(d - 0.5) > 0.5 - 1e-9) {
            const double b = __builtin_rint(s), c = b + b - 1.0;
            const double p = 254.0 * m, q = c * a;
            const double over = (p - q) + (__builtin_fma(254.0, m, -p) - __builtin_fma(c, a, -q));
            f = over >= 0.0 ? b : b - 1.0;
        }
        return int(f);
    }
    // The code of w = h g.
    NH_DEV int code(T h, T g) const
    {
        if constexpr (sizeof(T) == 4) {
            if (inv_f > 0.0f) {  // the same for the row
                const float w = h * g, s = __builtin_fmaf(__builtin_fabsf(w), inv_f, 0.5f), f = __builtin_floorf(s);
                int i = int(f);
                if (__builtin_fabsf(s - f - 0.5f) > 0.5f - 5e-5f) i = whole(__builtin_fabs(double(h) * double(g)));
                return w < 0.0f ? -i : i;
            }
        }
        const double w = double(h) * double(g);
        const int i = whole(__builtin_fabs(w));
        return live ? (w < 0.0 ? -i : i) : 0;
    }
    // scale of codes that stand for w * by.  A row of zeros has 0, also where `by` is infinite (the norm
    // of one with eps = 0).
    NH_DEV T scale(double a0, double by) const
    {
        if (!(a0 < __builtin_inf())) return T(__builtin_nan(""));
        if (a0 == 0.0 && by == by) return T(0);
        return T(a / 127.0 * by / up);
    }
};

}  // namespace nh
