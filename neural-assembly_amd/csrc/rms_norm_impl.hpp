// rms_norm_impl.hpp -- the forward pass of RMS norm with its output as values or as 8-bit codes,
// and rows to 8 bits (formulas: rms_norm.hip), compiled for each type by rms_norm_f32.hip and
// rms_norm_f64.hip.
#pragma once

#include "rms_norm.hpp"

namespace nh {

// Codes of W values side by side, as one store.
template <int W>
NH_DEV void store_codes(int8_t *p, const int (&c)[W])
{
    if constexpr (W == 1) {
        *p = int8_t(c[0]);
    } else {
        typedef int8_t B __attribute__((ext_vector_type(W), aligned(1)));
        B b;
#pragma unroll
        for (int j = 0; j < W; j++) b[j] = int8_t(c[j]);
        *reinterpret_cast<B *>(p) = b;
    }
}

// Maximum over a block, NaN where one value is.
template <int NT>
NH_DEV double group_amax(double v, double *lds)
{
    const auto comb = [](double a, double b) { return amax_comb(a, b); };
    return RowGrp<NT>::across(RowGrp<NT>::part(v, comb), lds, comb);
}

// How a group's lanes hold a row: NT lanes, VPT vectors each, the first F of them whole.
// kAhead: two rows, one in flight while the other is worked on; the resident blocks go by the loads
// that suit the memory, about 48 KB a CU in flight, and more where rows are read alone (rows to 8
// bits f32 [16384, 4096] 65.6 us with 3 waves a SIMD, 56.8 with 5, 61.7 with 8; [8192, 8192] 74.8
// with 2, 59.6 with 3).  kParams: gamma is loaded before the row's sums, not behind them.
template <typename T, int NT, int VPT, bool ADD, int OUT>
struct RmsPlan {
    static constexpr int NB = NT < 256 ? 256 : NT, RPB = NB / NT;
    static constexpr bool kAhead = !ADD && NT < 1024;
    static constexpr bool kParams = kAhead || (VPT <= 4 && NT < 1024);
    static constexpr int F = NT < 1024 || VPT <= 4 ? VPT - 1 : VPT / 2;
    static constexpr int kWaves = !kAhead ? (NT == 1024 ? 4 : 1)
                                  : OUT == ROW_CODES ? (VPT >= 5 ? 3 : VPT >= 3 ? 5 : 8)
                                                     : (VPT >= 5 ? 2 : VPT >= 3 ? 3 : VPT == 2 ? 5 : 8);
    static constexpr int kPerCu = kWaves * 256 / NB;  // resident blocks
};

// Groups of NT lanes walk the rows, r = group, group + groups, ...: a row is read once, its
// square sum and its largest |w| taken from the registers by one exchange.  Bound by HBM: f32
// [16384, 4096] 85 us, with the residual 175, and to 8 bits 131 (a copy of as many bytes 83, 176,
// 140); [65536, 1000] 92, 177, 132 (84, 171, 136); [4096, 16384] 94, 190, 152 (86, 176, 140).  f64
// [8192, 4096] with the residual 175 (a copy 176), to 8 bits 138 (136), and to 8 bits alone 63 (47; the
// vector units: codes of f64 rows are made in double).
template <typename T, int NT, int VPT, bool ADD, int OUT, bool PAST>
__global__ __launch_bounds__((RmsPlan<T, NT, VPT, ADD, OUT>::NB), (RmsPlan<T, NT, VPT, ADD, OUT>::kWaves)) void k_rms_rows(
    RmsArgs<T> a, int64_t r_base)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    using G = RowGrp<NT>;
    using S = RowStream<T, PAST>;
    using Plan = RmsPlan<T, NT, VPT, ADD, OUT>;
    constexpr int VN = Vec16<T>::n, RPB = Plan::RPB;
    constexpr bool SUM = OUT != ROW_CODES, MAX = OUT != RMS_VALUES;
    __shared__ double lds_q[2][G::kWaves], lds_m[2][G::kWaves];
    const int lane = threadIdx.x % NT, sub = RPB == 1 ? 0 : threadIdx.x / NT;
    const int64_t cols = a.cols;
    const RowCut<T> cut(cols);
    const auto in_row = [&](int k) { return k < Plan::F || lane + k * NT < cut.ncv; };
    const bool has_t = lane < cut.rem;
    const auto param = [&](int k) {
        V v;
#pragma unroll
        for (int j = 0; j < VN; j++) v[j] = T(1);
        if (SUM && a.gamma && in_row(k)) v = *(reinterpret_cast<const U *>(a.gamma) + lane + k * NT);
        return v;
    };
    constexpr bool kParams = SUM && Plan::kParams;
    V g[kParams ? VPT : 1];
    if constexpr (kParams) {
#pragma unroll
        for (int k = 0; k < VPT; k++) g[k] = param(k);
    }
    const T gt = SUM && a.gamma && has_t ? a.gamma[cut.sc(lane)] : T(1);
    struct Row {
        V x[VPT], res[ADD ? VPT : 1];
        T xt, rest;
    };
    const auto load = [&](Row &w, int64_t r) {
        const int64_t at = r * cols;
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) w.x[k] = S::load(reinterpret_cast<const U *>(a.x + at) + lane + k * NT);
        w.xt = has_t ? a.x[at + cut.sc(lane)] : T(0);
        if constexpr (ADD) {
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (in_row(k)) w.res[k] = S::load(reinterpret_cast<const U *>(a.res + at) + lane + k * NT);
            w.rest = has_t ? a.res[at + cut.sc(lane)] : T(0);
        }
    };
    const auto work = [&](Row &w, int64_t r, int odd) {
        const int64_t at = r * cols;
        if constexpr (ADD) {
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (in_row(k)) {
#pragma unroll
                    for (int j = 0; j < VN; j++) w.x[k][j] = w.res[k][j] + w.x[k][j];
                    if (a.h) S::store(w.x[k], reinterpret_cast<U *>(a.h + at) + lane + k * NT);
                }
            if (has_t) {
                w.xt = w.rest + w.xt;
                if (a.h) a.h[at + cut.sc(lane)] = w.xt;
            }
        }
        double q = 0.0, m = 0.0;
        constexpr bool FMAX = OUT == ROW_CODES && sizeof(T) == 4;  // the values themselves: their maximum in float
        float mf = 0.0f;
        bool odd_value = false;  // NaN, which the maximum passes over
        const auto gamma = [&](int k) {
            if constexpr (kParams) {
                hide(g[k]);
                return g[k];
            } else {
                return param(k);
            }
        };
        const auto take = [&](T h, T gv) {
            if constexpr (SUM) q = __builtin_fma(double(h), double(h), q);
            if constexpr (FMAX) {
                mf = __builtin_fmaxf(mf, __builtin_fabsf(h));
                odd_value |= h != h;
            } else if constexpr (MAX) {
                m = amax_comb(m, __builtin_fabs(double(h) * double(gv)));
            }
        };
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) {
                V gk;
                if constexpr (MAX) gk = gamma(k);
#pragma unroll
                for (int j = 0; j < VN; j++) take(w.x[k][j], MAX ? gk[j] : T(1));
            }
        if (has_t) take(w.xt, gt);
        if constexpr (FMAX) m = odd_value ? __builtin_nan("") : double(mf);
        const auto add = [](double x, double y) { return x + y; };
        const auto most = [](double x, double y) { return amax_comb(x, y); };
        if constexpr (SUM) q = G::part(q, add);
        if constexpr (MAX) m = G::part(m, most);
        if constexpr (G::kWaves > 1) {
            if ((threadIdx.x & 63) == 0) {
                if constexpr (SUM) lds_q[odd][threadIdx.x >> 6] = q;
                if constexpr (MAX) lds_m[odd][threadIdx.x >> 6] = m;
            }
            __syncthreads();
            if constexpr (SUM) q = lds_q[odd][0];
            if constexpr (MAX) m = lds_m[odd][0];
#pragma unroll
            for (int i = 1; i < G::kWaves; i++) {
                if constexpr (SUM) q += lds_q[odd][i];
                if constexpr (MAX) m = amax_comb(m, lds_m[odd][i]);
            }
        }
        const double rstd = SUM ? rms_rstd(q, a.inv_c, a.eps) : 1.0;
        const RowCodes<T> codes(MAX ? m : 0.0);
        if (lane == 0) {
            if (SUM && a.rstd) a.rstd[r] = T(rstd);
            if (MAX) a.scale[r] = codes.scale(m, rstd);
        }
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) {
                hide(w.x[k]);
                const V gk = gamma(k);
                if constexpr (MAX) {
                    int c[VN];
#pragma unroll
                    for (int j = 0; j < VN; j++) c[j] = codes.code(w.x[k][j], gk[j]);
                    store_codes<VN>(a.codes + r * a.stride + int64_t(lane + k * NT) * VN, c);
                } else {
                    V o;
#pragma unroll
                    for (int j = 0; j < VN; j++) o[j] = T(double(w.x[k][j]) * rstd * double(gk[j]));
                    S::store(o, reinterpret_cast<U *>(a.y + at) + lane + k * NT);
                }
            }
        if (has_t) {
            if constexpr (MAX) {
                const int c[1] = {codes.code(w.xt, gt)};
                store_codes<1>(a.codes + r * a.stride + cut.sc(lane), c);
            } else {
                a.y[at + cut.sc(lane)] = T(double(w.xt) * rstd * double(gt));
            }
        }
    };
    int64_t r = r_base + int64_t(blockIdx.x) * RPB + sub;
    Row w;
    if (r >= a.rows) return;  // uniform per group; a block of one row has one
    load(w, r);
    if constexpr (Plan::kAhead) {
        const int64_t step = int64_t(gridDim.x) * RPB;
        Row next;
        for (int odd = 0; r < a.rows; r += step, odd ^= 1) {
            if (r + step < a.rows) load(next, r + step);
            work(w, r, odd);
            w = next;
        }
    } else {
        work(w, r, 0);
    }
}

// Rows wider than a block's registers: two walks of a block, h, its square sum and its
// largest |w|, then the outputs (f32 [670, 100000] 148 us, with the residual 302, where a copy of
// the tensors once takes 85 and 175).
template <typename T, bool ADD, int OUT>
__global__ __launch_bounds__(kLnWide) void k_rms_wide(RmsArgs<T> a, int64_t r_base)
{
    using G = RowGrp<kLnWide>;
    __shared__ double lds_q[G::kWaves], lds_a[G::kWaves];
    const int64_t r = r_base + blockIdx.x, cols = a.cols, at = r * cols;
    const auto load = [&](auto w, int64_t c) {
        constexpr int W = decltype(w)::value;
        struct {
            Pack<T, W> x, res, g;
        } v;
        v.x = Pack<T, W>::load(a.x + at + c);
        if constexpr (ADD) v.res = Pack<T, W>::load(a.res + at + c);
#pragma unroll
        for (int j = 0; j < W; j++) v.g.v[j] = T(1);
        if (OUT != ROW_CODES && a.gamma) v.g = Pack<T, W>::load(a.gamma + c);
        return v;
    };
    const auto join = [&](const auto &v, int j) {
        if constexpr (ADD) return T(v.res.v[j] + v.x.v[j]);
        else return v.x.v[j];
    };
    double q = 0.0, m = 0.0;
    walk_row<T>(cols, load, [&](auto w, int64_t, const auto &v) {
        constexpr int W = decltype(w)::value;
#pragma unroll
        for (int j = 0; j < W; j++) {
            const double h = double(join(v, j));
            if constexpr (OUT != ROW_CODES) q = __builtin_fma(h, h, q);
            if constexpr (OUT != RMS_VALUES) m = amax_comb(m, __builtin_fabs(h * double(v.g.v[j])));
        }
    });
    double rstd = 1.0;
    if constexpr (OUT != ROW_CODES) rstd = rms_rstd(G::sum(q, lds_q), a.inv_c, a.eps);
    if constexpr (OUT != RMS_VALUES) m = group_amax<kLnWide>(m, lds_a);
    const RowCodes<T> codes(OUT != RMS_VALUES ? m : 0.0);
    if (threadIdx.x == 0) {
        if (OUT != ROW_CODES && a.rstd) a.rstd[r] = T(rstd);
        if (OUT != RMS_VALUES) a.scale[r] = codes.scale(m, rstd);
    }
    walk_row<T>(cols, load, [&](auto w, int64_t c, const auto &v) {
        constexpr int W = decltype(w)::value;
        Pack<T, W> h, o;
        int b[W];
#pragma unroll
        for (int j = 0; j < W; j++) {
            h.v[j] = join(v, j);
            if constexpr (OUT == RMS_VALUES) o.v[j] = T(double(h.v[j]) * rstd * double(v.g.v[j]));
            else b[j] = codes.code(h.v[j], v.g.v[j]);
        }
        if (ADD && a.h) h.store(a.h + at + c);
        if constexpr (OUT == RMS_VALUES) o.store(a.y + at + c);
        else store_codes<W>(a.codes + r * a.stride + c, b);
    });
}

template <typename T, bool ADD, int OUT, int NT, int VPT>
static void launch_rms_rows(const RmsArgs<T> &a)
{
    using Plan = RmsPlan<T, NT, VPT, ADD, OUT>;
    with_stream<T, NT>(a.cols, [&](auto past) {
        const auto launch = [&](unsigned g, int64_t base) {
            NH_LAUNCH((k_rms_rows<T, NT, VPT, ADD, OUT, decltype(past)::value>), dim3(g), dim3(Plan::NB), 0, stream(), a,
                      base);
        };
        if constexpr (Plan::kAhead) {
            const int64_t most = int64_t(num_cus()) * Plan::kPerCu, need = ceil_div(a.rows, int64_t(Plan::RPB));
            launch(unsigned(need < most ? need : most), 0);
        } else {
            for_row_launches(a.rows, Plan::RPB, Plan::NB, launch);
        }
    });
}

// The fewest of LO to HI vectors per lane of NT that hold the row.
template <typename T, bool ADD, int OUT, int NT, int LO, int HI>
static void launch_rms_exact(const RmsArgs<T> &a, int64_t ncv)
{
    if constexpr (LO < HI) {
        if (ncv > NT * LO) return launch_rms_exact<T, ADD, OUT, NT, LO + 1, HI>(a, ncv);
    }
    launch_rms_rows<T, ADD, OUT, NT, LO>(a);
}

// The fewest lanes whose registers hold the row, by its width alone (layer norm's rule: the
// sums over the lanes and what a row costs once are spread over the most values).
template <typename T, bool ADD, int OUT>
int launch_rms(const RmsArgs<T> &a)
{
    const int64_t ncv = a.cols / Vec16<T>::n;
    if (ncv <= 4) launch_rms_rows<T, ADD, OUT, 4, 1>(a);
    else if (ncv <= 8 * 4) launch_rms_exact<T, ADD, OUT, 8, 1, 4>(a, ncv);
    else if (ncv <= 16 * 4) launch_rms_exact<T, ADD, OUT, 16, 3, 4>(a, ncv);
    else if (ncv <= 32 * 4) launch_rms_exact<T, ADD, OUT, 32, 3, 4>(a, ncv);
    else if (ncv <= 64 * 4) launch_rms_exact<T, ADD, OUT, 64, 3, 4>(a, ncv);
    else if (ncv <= 256 * 8) launch_rms_exact<T, ADD, OUT, 256, 2, 8>(a, ncv);
    else if (ncv <= 1024 * 4) launch_rms_exact<T, ADD, OUT, 1024, 3, 4>(a, ncv);
    else if (ncv <= 1024 * 8) launch_rms_rows<T, ADD, OUT, 1024, 8>(a);
    else if (ncv <= 1024 * 16) launch_rms_rows<T, ADD, OUT, 1024, 16>(a);
    else
        for_row_launches(a.rows, 1, kLnWide, [&](unsigned g, int64_t base) {
            NH_LAUNCH((k_rms_wide<T, ADD, OUT>), dim3(g), dim3(kLnWide), 0, stream(), a, base);
        });
    return check_launch();
}

}  // namespace nh
