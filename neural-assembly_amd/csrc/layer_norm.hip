// layer_norm.hip -- layer norm over the last dimension, forward and backward,
// alone and joined with the residual add and the counter-based dropout before
// it (the end of a transformer's sublayer).
//
//   forward:  h = x, or residual + dropout(x) (two roundings, as the two calls);
//             mean = sum h / C; var = sum (h - mean)^2 / C; rstd = 1 / sqrt(var + eps);
//             y = (h - mean) rstd gamma + beta
//   backward, from the saved mean and rstd: xh = (h - mean) rstd; w = dy gamma;
//             d = rstd (w - mean_c(w) - xh mean_c(w xh)) [+ dh, the gradient that
//             reaches h besides]; dresidual = d, dx = dropout's map of d;
//             dgamma = sum_rows dy xh; dbeta = sum_rows dy
//
// Everything between the loads and the stores is in double, f32 rows rounded once
// per output; mean and rstd are stored in the rows' type (the mean's rounding
// moves xh by what half an ulp of an input of the mean's size would).  The
// variance is taken from the centred values, which are still in registers.
//
// A row is held by one group of lanes, part of a wave to a block of 1024, at any
// width and alignment (RowCut), so each tensor is read once and written once.
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "philox.hpp"
#include "row_group.hpp"

namespace nh {

enum { LN_PLAIN = 0, LN_ADD = 1, LN_DROP = 2 };

// Hides where v's values came from, in place: or the compiler keeps the doubles that an
// earlier pass over the row made of them (two or more registers per value, and
// spills) instead of converting again.
template <typename V>
NH_DEV void hide(V &v)
{
    asm("" : "+v"(v));
}

// s / n from inv = 1 / n: the quotient corrected by its remainder, so that a row of one
// value has exactly that mean (its sum is exact in double).  The remainder of an
// infinity is NaN: it stays as it is.
NH_DEV double over(double s, int64_t n, double inv)
{
    const double m = s * inv, c = __builtin_fma(__builtin_fma(-m, double(n), s), inv, m);
    return c == c ? c : m;
}

// 1 / sqrt(v) from the hardware's estimate y and one third-order step: with e = 1 - v y^2,
// y (1 + e / 2 + 3 e^2 / 8).  0, infinity and NaN take the estimate.
NH_DEV double rsqrt_d(double v)
{
    const double y = __builtin_amdgcn_rsq(v);
    const double e = __builtin_fma(-(v * y), y, 1.0);
    const double r = __builtin_fma(y * e, __builtin_fma(e, 0.375, 0.5), y);
    return v > 0.0 && v < __builtin_inf() ? r : y;
}

// ---- keep bits of a row's vectors ----------------------------------------------------------

// Keep bits of the elements of a row that a lane holds.  Where the row's width is
// a multiple of 8, groups do not cross rows and the lanes that share one make
// its bits in turn (mask_of); elsewhere the group of lanes makes all the row's
// bits, a byte per group, in LDS.
template <typename T, int NT, int VPT>
struct RowKeep {
    static constexpr int VN = Vec16<T>::n, P = kGroupLanes<T>;
    static constexpr int kBytes = NT * VPT * VN / 8 + 4;  // (lds) groups that a row can touch, and one byte more
    uint32_t m[VPT];  // vector k: element j at bit j / 2 + 16 (j % 2)
    uint32_t tail;    // the scalar's, bit 0

    NH_DEV void make(int64_t r, int64_t cols, const RowCut<T> &cut, int lane, const DropKey &key, uint8_t *lds)
    {
        tail = 0;
        if ((cols & 7) == 0) {
            const int64_t v0 = r * (cols / VN) + lane;
#pragma unroll
            for (int k0 = 0; k0 < VPT; k0 += P) {
                const uint32_t own = keep_mask(uint64_t(v0 + (k0 + (lane & (P - 1))) * NT) / P, key);
                m[k0] = mask_of<T, 0>(own, lane);
                if (k0 + 1 < VPT) m[k0 + 1] = mask_of<T, 1>(own, lane);
                if constexpr (P == 4) {
                    if (k0 + 2 < VPT) m[k0 + 2] = mask_of<T, 2>(own, lane);
                    if (k0 + 3 < VPT) m[k0 + 3] = mask_of<T, 3>(own, lane);
                }
            }
            return;
        }
        const uint64_t first = uint64_t(r) * uint64_t(cols), g0 = first / 8;
        const int o = int(first % 8), groups = int((o + cols + 7) / 8);
        for (int q = lane; q < groups; q += NT) lds[q] = uint8_t(keep_in_order(keep_mask(g0 + q, key)));
        if constexpr (NT <= 64) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        } else {
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            const int at = o + (lane + k * NT) * VN, b = at >> 3 < groups ? at >> 3 : 0;
            const uint32_t s = (uint32_t(lds[b]) | uint32_t(lds[b + 1]) << 8) >> (at & 7);  // element j at bit j
            if constexpr (VN == 4) m[k] = (s & 1u) | (s & 4u) >> 1 | (s & 2u) << 15 | (s & 8u) << 14;
            else m[k] = (s & 1u) | (s & 2u) << 15;
        }
        if (lane < cut.rem) {
            const int at = o + int(cut.sc(lane));
            tail = uint32_t(lds[at >> 3]) >> (at & 7);
        }
    }
    NH_DEV static constexpr int bit(int j) { return (j >> 1) + 16 * (j & 1); }
};

// ---- forward -------------------------------------------------------------------------------

template <typename T>
struct LnArgs {
    const T *x, *res, *gamma, *beta;  // res: joined forms; gamma, beta: may be null
    T *h, *y, *mean, *rstd;           // h, mean, rstd: may be null
    int64_t rows, cols;
    double eps;
    DropArgs drop;
};

// One row per group of NT lanes, VPT vectors per lane, the first F of them whole, and
// one scalar.  Bound by HBM while enough rows are in flight.
template <typename T, int NT, int VPT, int F, int MODE>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void k_ln_rows(LnArgs<T> a, int64_t r_base)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    using G = RowGrp<NT>;
    using K = RowKeep<T, NT, VPT>;
    constexpr int VN = Vec16<T>::n;
    constexpr int RPB = NT < 256 ? 256 / NT : 1;
    __shared__ double lds_s[G::kWaves], lds_q[G::kWaves];
    __shared__ uint8_t lds_keep[MODE == LN_DROP ? RPB : 1][MODE == LN_DROP ? K::kBytes : 1];
    const int lane = threadIdx.x % NT, sub = threadIdx.x / NT;
    const int64_t r = r_base + int64_t(blockIdx.x) * RPB + sub;
    if (RPB > 1 && r >= a.rows) return;  // uniform per group; a block of one row has one
    const int64_t cols = a.cols;
    const RowCut<T> cut(cols);
    const auto in_row = [&](int k) { return k < F || lane + k * NT < cut.ncv; };
    const bool has_t = lane < cut.rem;
    const int64_t at = r * cols;
    V v[VPT];
    T vt = T(0);
#pragma unroll
    for (int k = 0; k < VPT; k++)
        if (in_row(k)) v[k] = __builtin_nontemporal_load(reinterpret_cast<const U *>(a.x + at) + lane + k * NT);
    if (has_t) vt = a.x[at + cut.sc(lane)];
    if constexpr (MODE != LN_PLAIN) {
        V w[VPT];
        T wt = T(0);
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) w[k] = __builtin_nontemporal_load(reinterpret_cast<const U *>(a.res + at) + lane + k * NT);
        if (has_t) wt = a.res[at + cut.sc(lane)];
        if constexpr (MODE == LN_DROP) {
            const DropKey key(a.drop);
            const T scale = T(a.drop.scale);
            K keep;
            keep.make(r, cols, cut, lane, key, lds_keep[sub]);
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (in_row(k)) {
#pragma unroll
                    for (int j = 0; j < VN; j++) v[k][j] = w[k][j] + dropped<T>(v[k][j], scale, keep.m[k], K::bit(j));
                }
            vt = wt + dropped<T>(vt, scale, keep.tail, 0);
        } else {
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (in_row(k)) {
#pragma unroll
                    for (int j = 0; j < VN; j++) v[k][j] = w[k][j] + v[k][j];
                }
            vt = wt + vt;
        }
        if (a.h) {
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (in_row(k)) __builtin_nontemporal_store(v[k], reinterpret_cast<U *>(a.h + at) + lane + k * NT);
            if (has_t) a.h[at + cut.sc(lane)] = vt;
        }
    }
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < VPT; k++)
        if (in_row(k)) {
#pragma unroll
            for (int j = 0; j < VN; j++) s += double(v[k][j]);
        }
    if (has_t) s += double(vt);
    const double inv_c = 1.0 / double(cols);
    const double mean = over(G::sum(s, lds_s), cols, inv_c);
    double q = 0.0;
#pragma unroll
    for (int k = 0; k < VPT; k++)
        if (in_row(k)) {
            hide(v[k]);
#pragma unroll
            for (int j = 0; j < VN; j++) {
                const double d = double(v[k][j]) - mean;
                q = __builtin_fma(d, d, q);
            }
        }
    if (has_t) {
        const double d = double(vt) - mean;
        q = __builtin_fma(d, d, q);
    }
    const double rstd = rsqrt_d(G::sum(q, lds_q) * inv_c + a.eps);
    if (lane == 0) {
        if (a.mean) a.mean[r] = T(mean);
        if (a.rstd) a.rstd[r] = T(rstd);
    }
    const auto out = [&](T xv, T g, T b) {
        return T(__builtin_fma((double(xv) - mean) * rstd, double(g), double(b)));
    };
#pragma unroll
    for (int k = 0; k < VPT; k++)
        if (in_row(k)) {
            V g, b, o;
#pragma unroll
            for (int j = 0; j < VN; j++) {
                g[j] = T(1);
                b[j] = T(0);
            }
            if (a.gamma) g = *(reinterpret_cast<const U *>(a.gamma) + lane + k * NT);
            if (a.beta) b = *(reinterpret_cast<const U *>(a.beta) + lane + k * NT);
            hide(v[k]);
#pragma unroll
            for (int j = 0; j < VN; j++) o[j] = out(v[k][j], g[j], b[j]);
            __builtin_nontemporal_store(o, reinterpret_cast<U *>(a.y + at) + lane + k * NT);
        }
    if (has_t) {
        const int64_t c = cut.sc(lane);
        a.y[at + c] = out(vt, a.gamma ? a.gamma[c] : T(1), a.beta ? a.beta[c] : T(0));
    }
}

// Rows wider than a block's registers, in three walks of a block of 1024 lanes: h
// and its sum, the centred squares, y.
constexpr int kLnWide = 1024;

template <typename T, int MODE>
NH_DEV T ln_value(const LnArgs<T> &a, int64_t i, const DropKey &key, T scale)
{
    if constexpr (MODE == LN_PLAIN) return a.x[i];
    else if constexpr (MODE == LN_ADD) return a.res[i] + a.x[i];
    else
        return a.res[i] + dropped<T>(a.x[i], scale, keep_in_order(keep_mask(uint64_t(i) / 8, key)), int(i % 8));
}

template <typename T, int MODE>
__global__ __launch_bounds__(kLnWide) void k_ln_wide(LnArgs<T> a, int64_t r_base)
{
    using G = RowGrp<kLnWide>;
    __shared__ double lds_s[G::kWaves], lds_q[G::kWaves];
    const DropKey key(a.drop);
    const T scale = T(a.drop.scale);
    const int64_t r = r_base + blockIdx.x, cols = a.cols, at = r * cols;
    double s = 0.0, q = 0.0;
    for (int64_t c = threadIdx.x; c < cols; c += kLnWide) {
        const T v = ln_value<T, MODE>(a, at + c, key, scale);
        if (MODE != LN_PLAIN && a.h) a.h[at + c] = v;
        s += double(v);
    }
    const double mean = G::sum(s, lds_s) / double(cols);
    const auto value = [&](int64_t c) {
        return MODE != LN_PLAIN && a.h ? a.h[at + c] : ln_value<T, MODE>(a, at + c, key, scale);
    };
    for (int64_t c = threadIdx.x; c < cols; c += kLnWide) {
        const double d = double(value(c)) - mean;
        q = __builtin_fma(d, d, q);
    }
    const double rstd = 1.0 / sqrt(G::sum(q, lds_q) / double(cols) + a.eps);
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[r] = T(mean);
        if (a.rstd) a.rstd[r] = T(rstd);
    }
    for (int64_t c = threadIdx.x; c < cols; c += kLnWide) {
        const T v = value(c);
        const double g = a.gamma ? double(a.gamma[c]) : 1.0, b = a.beta ? double(a.beta[c]) : 0.0;
        a.y[at + c] = T(__builtin_fma((double(v) - mean) * rstd, g, b));
    }
}

template <typename T, int MODE, int NT, int VPT, int F = VPT - 1>
static void launch_ln_rows(const LnArgs<T> &a)
{
    for_row_launches(a.rows, NT < 256 ? 256 / NT : 1, [&](unsigned g, int64_t base) {
        NH_LAUNCH((k_ln_rows<T, NT, VPT, F, MODE>), dim3(g), dim3(NT < 256 ? 256 : NT), 0, stream(), a, base);
    });
}

// The fewest of LO to 4 vectors per lane of NT that hold the row.
template <typename T, int MODE, int NT, int LO>
static void launch_ln_exact(const LnArgs<T> &a, int64_t ncv)
{
    if constexpr (LO < 4) {
        if (ncv > NT * LO) return launch_ln_exact<T, MODE, NT, LO + 1>(a, ncv);
    }
    launch_ln_rows<T, MODE, NT, LO>(a);
}

template <typename T, int MODE>
static int launch_ln(const LnArgs<T> &a)
{
    const int64_t ncv = a.cols / Vec16<T>::n;
    if (ncv <= 4 * 4) launch_ln_exact<T, MODE, 4, 1>(a, ncv);
    else if (ncv <= 16 * 4) launch_ln_exact<T, MODE, 16, 2>(a, ncv);
    else if (ncv <= 64 * 4) launch_ln_exact<T, MODE, 64, 2>(a, ncv);
    else if (ncv <= 256 * 4) launch_ln_exact<T, MODE, 256, 2>(a, ncv);
    else if (ncv <= 512 * 4) launch_ln_exact<T, MODE, 512, 3>(a, ncv);
    else if (ncv <= 1024 * 4) launch_ln_exact<T, MODE, 1024, 3>(a, ncv);
    else if (ncv <= 1024 * 8) launch_ln_rows<T, MODE, 1024, 8, 4>(a);
    else if (ncv <= 1024 * 16) launch_ln_rows<T, MODE, 1024, 16, 8>(a);
    else
        for_row_launches(a.rows, 1, [&](unsigned g, int64_t base) {
            NH_LAUNCH((k_ln_wide<T, MODE>), dim3(g), dim3(kLnWide), 0, stream(), a, base);
        });
    return check_launch();
}

// ---- backward ------------------------------------------------------------------------------

template <typename T>
struct LnGradArgs {
    const T *dy, *h, *gamma, *mean, *rstd, *dh;  // gamma, dh: may be null
    T *dx, *dres;                                // either may be null
    T *part;                                     // [blocks][2][cols] partial sums of dgamma and dbeta, or null
    int64_t rows, cols;
    DropArgs drop;
};

// How a group's lanes hold a row of the backward pass, and how many groups a CU
// holds.  NT lanes, VPT vectors each.  Up to 4 vectors: gamma and the sums of dgamma and dbeta
// (in double) in registers.  5 to 8: the sums in LDS, in the rows' type (128 KB at
// most), gamma from the L2 for each row.  More: no sums (k_ln_cols takes them).
template <typename T, int NT, int VPT>
struct LnGradPlan {
    static constexpr int NB = NT < 256 ? 256 : NT, RPB = NB / NT;
    static constexpr bool kRegs = VPT <= 4;
    static constexpr int F = VPT <= 8 ? VPT - 1 : VPT / 2;  // vectors that are whole
    static constexpr int kWaves = VPT >= 3 || NT >= 512 ? 2 : 3;  // per SIMD
    static constexpr int kPerCu = kWaves * 256 / NB;              // resident blocks
};

// Groups of NT lanes walk the rows, r = group, group + groups, ...: each tensor
// read once, the next row's loads issued before this one is worked on, the row's
// two sums by one exchange (LDS slots alternate between rows, so one barrier a row
// is enough), and each lane's columns of dgamma and dbeta summed over the rows (SUMS).
// The block's groups fold theirs through LDS and the block leaves one row of
// partials, in the rows' type (the rounding of one of some hundred terms of a sum that is
// itself rounded so).  `block` of `blocks`.
template <typename T, int NT, int VPT, int MODE, bool SUMS>
NH_DEV void ln_grad_rows(const LnGradArgs<T> &a, int64_t block, int64_t blocks)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    using G = RowGrp<NT>;
    using K = RowKeep<T, NT, VPT>;
    using Plan = LnGradPlan<T, NT, VPT>;
    constexpr int VN = Vec16<T>::n, RPB = Plan::RPB;
    constexpr bool LS = SUMS && !Plan::kRegs, RS = SUMS && Plan::kRegs;
    __shared__ double lds_s[2][G::kWaves], lds_q[2][G::kWaves];
    __shared__ uint8_t lds_keep[2][MODE == LN_DROP ? RPB : 1][MODE == LN_DROP ? K::kBytes : 1];
    __shared__ V lds_g[LS ? VPT : 1][LS ? NT : 1], lds_b[LS ? VPT : 1][LS ? NT : 1];
    const int lane = threadIdx.x % NT, sub = threadIdx.x / NT;
    const int64_t cols = a.cols;
    const RowCut<T> cut(cols);
    const auto in_row = [&](int k) { return k < Plan::F || lane + k * NT < cut.ncv; };
    const bool has_t = lane < cut.rem;
    const double inv_c = 1.0 / double(cols);
    V g[Plan::kRegs ? VPT : 1];
    const auto gamma = [&](int k) {
        V v;
#pragma unroll
        for (int j = 0; j < VN; j++) v[j] = T(1);
        if (a.gamma && in_row(k)) v = *(reinterpret_cast<const U *>(a.gamma) + lane + k * NT);
        return v;
    };
    if constexpr (Plan::kRegs) {
#pragma unroll
        for (int k = 0; k < VPT; k++) g[k] = gamma(k);
    }
    T gt = T(1);
    if (a.gamma && has_t) gt = a.gamma[cut.sc(lane)];
    double sg[RS ? VPT : 1][VN], sb[RS ? VPT : 1][VN], sgt = 0.0, sbt = 0.0;
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        if constexpr (RS) {
#pragma unroll
            for (int j = 0; j < VN; j++) sg[k][j] = sb[k][j] = 0.0;
        } else if constexpr (LS) {
            V z;
#pragma unroll
            for (int j = 0; j < VN; j++) z[j] = T(0);
            lds_g[k][lane] = lds_b[k][lane] = z;  // a lane's own slots
        }
    }
    const DropKey key(a.drop);
    const T scale = T(a.drop.scale);
    struct Row {
        V x[VPT], dy[VPT];
        T xt, dyt, mean, rstd;
    };
    const auto load = [&](Row &w, int64_t r) {
        const int64_t at = r * cols;
        w.mean = a.mean[r];
        w.rstd = a.rstd[r];
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) w.x[k] = __builtin_nontemporal_load(reinterpret_cast<const U *>(a.h + at) + lane + k * NT);
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) w.dy[k] = __builtin_nontemporal_load(reinterpret_cast<const U *>(a.dy + at) + lane + k * NT);
        if (has_t) {
            w.xt = a.h[at + cut.sc(lane)];
            w.dyt = a.dy[at + cut.sc(lane)];
        }
    };
    const int64_t step = blocks * RPB;
    int64_t r = block * RPB + sub;
    Row w, next;
    if (r < a.rows) load(w, r);
    for (int odd = 0; r < a.rows; r += step, odd ^= 1) {
        const int64_t at = r * cols;
        constexpr bool kEarly = MODE != LN_PLAIN && VPT <= 8;  // dh fits beside x and dy
        V dh[kEarly ? VPT : 1];
        T dht = T(0);
        if constexpr (MODE != LN_PLAIN) {
            if (a.dh) {
#pragma unroll
                for (int k = 0; k < (kEarly ? VPT : 0); k++)
                    if (in_row(k))
                        dh[k] = __builtin_nontemporal_load(reinterpret_cast<const U *>(a.dh + at) + lane + k * NT);
                if (has_t) dht = a.dh[at + cut.sc(lane)];
            }
        }
        if (VPT <= 8 && r + step < a.rows) load(next, r + step);
        const double mean = double(w.mean), rstd = double(w.rstd);
        K keep;
        if constexpr (MODE == LN_DROP) keep.make(r, cols, cut, lane, key, lds_keep[odd][sub]);
        double s = 0.0, q = 0.0;
        const auto sums = [&](T xv, T dyv, T gv, double &ag, double &ab) {
            const double d = double(dyv), xh = (double(xv) - mean) * rstd, wv = d * double(gv);
            s += wv;
            q = __builtin_fma(wv, xh, q);
            ag = __builtin_fma(d, xh, ag);
            ab += d;
        };
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) {
                V gk, vg, vb;
                if constexpr (Plan::kRegs) gk = g[k];
                else gk = gamma(k);
                if constexpr (LS) {
                    vg = lds_g[k][lane];
                    vb = lds_b[k][lane];
                }
#pragma unroll
                for (int j = 0; j < VN; j++) {
                    if constexpr (LS) {
                        double ag = double(vg[j]), ab = double(vb[j]);
                        sums(w.x[k][j], w.dy[k][j], gk[j], ag, ab);
                        vg[j] = T(ag);
                        vb[j] = T(ab);
                    } else {
                        sums(w.x[k][j], w.dy[k][j], gk[j], sg[RS ? k : 0][j], sb[RS ? k : 0][j]);
                    }
                }
                if constexpr (RS) {
                    // taken here: the compiler would put them off past the stores, with
                    // their operands' doubles kept until then
#pragma unroll
                    for (int j = 0; j < VN; j++) asm volatile("" : "+v"(sg[k][j]), "+v"(sb[k][j]));
                }
                if constexpr (LS) {
                    lds_g[k][lane] = vg;
                    lds_b[k][lane] = vb;
                    asm volatile("" : "+v"(s), "+v"(q) : : "memory");  // one vector's terms in registers at a time
                }
            }
        if (has_t) sums(w.xt, w.dyt, gt, sgt, sbt);
        // both sums over the row by one exchange
        const auto add = [](double p, double t) { return p + t; };
        s = G::part(s, add);
        q = G::part(q, add);
        if constexpr (G::kWaves > 1) {
            if ((threadIdx.x & 63) == 0) {
                lds_s[odd][threadIdx.x >> 6] = s;
                lds_q[odd][threadIdx.x >> 6] = q;
            }
            __syncthreads();
            s = lds_s[odd][0];
            q = lds_q[odd][0];
#pragma unroll
            for (int i = 1; i < G::kWaves; i++) {
                s += lds_s[odd][i];
                q += lds_q[odd][i];
            }
        }
        const double c1 = s * inv_c, c2 = q * inv_c;
        const auto grad = [&](T xv, T dyv, T gv) {
            const double xh = (double(xv) - mean) * rstd, wv = double(dyv) * double(gv);
            return T(rstd * (__builtin_fma(-xh, c2, wv - c1)));
        };
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if ((MODE != LN_PLAIN || a.dx) && in_row(k)) {
                hide(w.x[k]);
                hide(w.dy[k]);
                V o, gk;
                if constexpr (Plan::kRegs) {
                    hide(g[k]);
                    gk = g[k];
                } else {
                    gk = gamma(k);
                }
#pragma unroll
                for (int j = 0; j < VN; j++) o[j] = grad(w.x[k][j], w.dy[k][j], gk[j]);
                if constexpr (MODE != LN_PLAIN) {
                    if (a.dh) {
                        V d;
                        if constexpr (kEarly) d = dh[k];
                        else d = __builtin_nontemporal_load(reinterpret_cast<const U *>(a.dh + at) + lane + k * NT);
#pragma unroll
                        for (int j = 0; j < VN; j++) o[j] = o[j] + d[j];
                    }
                    if (a.dres) __builtin_nontemporal_store(o, reinterpret_cast<U *>(a.dres + at) + lane + k * NT);
                }
                if constexpr (MODE == LN_DROP) {
#pragma unroll
                    for (int j = 0; j < VN; j++) o[j] = dropped<T>(o[j], scale, keep.m[k], K::bit(j));
                }
                if (MODE == LN_PLAIN || a.dx)
                    __builtin_nontemporal_store(o, reinterpret_cast<U *>(a.dx + at) + lane + k * NT);
            }
        if (has_t) {
            const int64_t i = at + cut.sc(lane);
            T o = grad(w.xt, w.dyt, gt);
            if constexpr (MODE != LN_PLAIN) {
                if (a.dh) o = o + dht;
                if (a.dres) a.dres[i] = o;
            }
            if constexpr (MODE == LN_DROP) o = dropped<T>(o, scale, keep.tail, 0);
            if (a.dx) a.dx[i] = o;
        }
        if constexpr (VPT <= 8) w = next;
        else if (r + step < a.rows) load(w, r + step);  // no registers for two rows
    }
    if constexpr (SUMS) {
        T *pg = a.part + block * 2 * cols, *pb = pg + cols;
        if constexpr (RPB == 1) {
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (in_row(k)) {
                    V og, ob;
                    if constexpr (LS) {
                        og = lds_g[k][lane];
                        ob = lds_b[k][lane];
                    } else {
#pragma unroll
                        for (int j = 0; j < VN; j++) {
                            og[j] = T(sg[k][j]);
                            ob[j] = T(sb[k][j]);
                        }
                    }
                    *(reinterpret_cast<U *>(pg) + lane + k * NT) = og;
                    *(reinterpret_cast<U *>(pb) + lane + k * NT) = ob;
                }
            if (has_t) {
                pg[cut.sc(lane)] = T(sgt);
                pb[cut.sc(lane)] = T(sbt);
            }
        } else {
            // fold the block's groups, one vector slot at a time
            __shared__ double fold[2 * VN][256];
            const auto across = [&](auto n_c, const double *vg, const double *vb, int64_t c0, bool mine) {
                constexpr int n = decltype(n_c)::value;
                __syncthreads();
#pragma unroll
                for (int j = 0; j < n; j++) {
                    fold[j][threadIdx.x] = vg[j];
                    fold[n + j][threadIdx.x] = vb[j];
                }
                __syncthreads();
                for (int e = threadIdx.x; e < 2 * n * NT; e += 256) {
                    const int l = e % NT, j = e / NT;
                    double t = fold[j][l];
                    for (int i = 1; i < RPB; i++) t += fold[j][l + i * NT];
                    fold[j][l] = t;
                }
                __syncthreads();
                if (sub == 0 && mine) {
                    for (int j = 0; j < n; j++) {
                        pg[c0 + j] = T(fold[j][lane]);
                        pb[c0 + j] = T(fold[n + j][lane]);
                    }
                }
            };
#pragma unroll
            for (int k = 0; k < VPT; k++)
                across(std::integral_constant<int, VN>{}, sg[k], sb[k], int64_t(lane + k * NT) * VN, in_row(k));
            if (cut.rem) across(std::integral_constant<int, 1>{}, &sgt, &sbt, cut.sc(lane), has_t);
        }
    }
}

template <typename T, int NT, int VPT, int MODE, bool SUMS>
__global__ __launch_bounds__((LnGradPlan<T, NT, VPT>::NB), (LnGradPlan<T, NT, VPT>::kWaves)) void k_ln_grad(
    LnGradArgs<T> a)
{
    ln_grad_rows<T, NT, VPT, MODE, SUMS>(a, blockIdx.x, gridDim.x);
}

// Sums of few rows, without partials: 16 columns a block of NB lanes, the rows
// by NB / 16 streams of 8 rows in flight, folded in LDS.
template <typename T, int NB>
NH_DEV void ln_few_cols(const LnGradArgs<T> &a, int64_t block, T *dgamma, T *dbeta)
{
    constexpr int S = NB / 16, UN = 8;
    __shared__ double sh[2][S][16];
    const int cl = threadIdx.x & 15, st = threadIdx.x >> 4;
    const int64_t cols = a.cols, c = block * 16 + cl;
    double g = 0.0, b = 0.0;
    if (c < cols)
        for (int64_t r = st; r < a.rows; r += S * UN) {
            T dy[UN], x[UN], m[UN], rs[UN];
#pragma unroll
            for (int u = 0; u < UN; u++)
                if (r + u * S < a.rows) {
                    const int64_t q = r + u * S;
                    dy[u] = a.dy[q * cols + c];
                    x[u] = a.h[q * cols + c];
                    m[u] = a.mean[q];
                    rs[u] = a.rstd[q];
                }
#pragma unroll
            for (int u = 0; u < UN; u++)
                if (r + u * S < a.rows) {
                    const double d = double(dy[u]);
                    g = __builtin_fma(d, (double(x[u]) - double(m[u])) * double(rs[u]), g);
                    b += d;
                }
        }
    sh[0][st][cl] = g;
    sh[1][st][cl] = b;
    __syncthreads();
    if (st < 2 && c < cols) {
        double t = sh[st][0][cl];
        for (int i = 1; i < S; i++) t += sh[st][i][cl];
        T *out = st ? dbeta : dgamma;
        if (out) out[c] = T(t);
    }
}

// The backward pass of few rows in one launch: blocks 0 .. nrows - 1 take the rows,
// the others columns (which read x and dy again, from the caches).  Either
// part may be absent.
template <typename T, int NT, int VPT, int MODE>
__global__ __launch_bounds__((LnGradPlan<T, NT, VPT>::NB)) void k_ln_grad_few(LnGradArgs<T> a, int nrows, T *dgamma,
                                                                             T *dbeta)
{
    if (int(blockIdx.x) < nrows) ln_grad_rows<T, NT, VPT, MODE, false>(a, blockIdx.x, nrows);
    else ln_few_cols<T, LnGradPlan<T, NT, VPT>::NB>(a, int64_t(blockIdx.x) - nrows, dgamma, dbeta);
}

// Column sums of the partials: [n][2 cols] -> dgamma, dbeta.  A block of 16
// waves takes 64 columns, the waves the partials in turn, eight in flight each.
template <typename T>
__global__ __launch_bounds__(1024) void k_ln_fold(const T *__restrict__ part, int64_t n, int64_t cols,
                                                  T *__restrict__ dgamma, T *__restrict__ dbeta)
{
    constexpr int UN = 8;
    __shared__ double sh[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = int64_t(blockIdx.x) * 64 + lane;
    double s = 0.0;
    if (c < 2 * cols) {
        const T *p = part + c;
        int64_t i = w;
        for (; i + 16 * (UN - 1) < n; i += 16 * UN) {
            T v[UN];
#pragma unroll
            for (int u = 0; u < UN; u++) v[u] = p[(i + 16 * u) * 2 * cols];
#pragma unroll
            for (int u = 0; u < UN; u++) s += double(v[u]);
        }
        T v[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) v[u] = i + 16 * u < n ? p[(i + 16 * u) * 2 * cols] : T(0);
#pragma unroll
        for (int u = 0; u < UN; u++) s += double(v[u]);
    }
    sh[w][lane] = s;
    __syncthreads();
    if (w == 0 && c < 2 * cols) {
        for (int i = 1; i < 16; i++) s += sh[i][lane];
        T *out = c < cols ? dgamma : dbeta;
        if (out) out[c < cols ? c : c - cols] = T(s);
    }
}

// Rows wider than a block's registers: the row's sums, then the outputs, reading
// every tensor again, element by element.
template <typename T, int MODE>
__global__ __launch_bounds__(kLnWide) void k_ln_grad_wide(LnGradArgs<T> a, int64_t r_base)
{
    using G = RowGrp<kLnWide>;
    __shared__ double lds_s[G::kWaves], lds_q[G::kWaves];
    const DropKey key(a.drop);
    const T scale = T(a.drop.scale);
    const int64_t r = r_base + blockIdx.x, cols = a.cols, at = r * cols;
    const double mean = double(a.mean[r]), rstd = double(a.rstd[r]);
    double s = 0.0, q = 0.0;
    for (int64_t c = threadIdx.x; c < cols; c += kLnWide) {
        const double xh = (double(a.h[at + c]) - mean) * rstd;
        const double w = double(a.dy[at + c]) * (a.gamma ? double(a.gamma[c]) : 1.0);
        s += w;
        q = __builtin_fma(w, xh, q);
    }
    const double c1 = G::sum(s, lds_s) / double(cols), c2 = G::sum(q, lds_q) / double(cols);
    for (int64_t c = threadIdx.x; c < cols; c += kLnWide) {
        const int64_t i = at + c;
        const double xh = (double(a.h[i]) - mean) * rstd;
        const double w = double(a.dy[i]) * (a.gamma ? double(a.gamma[c]) : 1.0);
        T o = T(rstd * __builtin_fma(-xh, c2, w - c1));
        if constexpr (MODE != LN_PLAIN) {
            if (a.dh) o = o + a.dh[i];
            if (a.dres) a.dres[i] = o;
        }
        if constexpr (MODE == LN_DROP)
            o = dropped<T>(o, scale, keep_in_order(keep_mask(uint64_t(i) / 8, key)), int(i % 8));
        if (a.dx) a.dx[i] = o;
    }
}

// Column sums beside a row pass that cannot hold them: 64 lanes of VN columns a block, the
// rows of its chunk by 8 waves, four in flight each.
template <typename T>
__global__ __launch_bounds__(512) void k_ln_cols(LnGradArgs<T> a, int64_t chunk)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, W = 8, UN = 4;
    __shared__ double sh[W][2 * VN][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t cols = a.cols, c = (int64_t(blockIdx.x) * 64 + lane) * VN;
    const int64_t r0 = int64_t(blockIdx.y) * chunk, r1 = r0 + chunk < a.rows ? r0 + chunk : a.rows;
    const bool whole = c + VN <= cols;
    double s[2 * VN];
#pragma unroll
    for (int j = 0; j < 2 * VN; j++) s[j] = 0.0;
    for (int64_t r = r0 + w; r < r1; r += W * UN) {
        V x[UN], dy[UN];
#pragma unroll
        for (int u = 0; u < UN; u++)
            if (r + u * W < r1) {
                const int64_t at = (r + u * W) * cols + c;
                if (whole) {
                    x[u] = *reinterpret_cast<const U *>(a.h + at);
                    dy[u] = *reinterpret_cast<const U *>(a.dy + at);
                } else {
#pragma unroll
                    for (int j = 0; j < VN; j++) {
                        x[u][j] = c + j < cols ? a.h[at + j] : T(0);
                        dy[u][j] = c + j < cols ? a.dy[at + j] : T(0);
                    }
                }
            }
#pragma unroll
        for (int u = 0; u < UN; u++)
            if (r + u * W < r1) {
                const double mean = double(a.mean[r + u * W]), rstd = double(a.rstd[r + u * W]);
#pragma unroll
                for (int j = 0; j < VN; j++) {
                    const double d = double(dy[u][j]);
                    s[j] = __builtin_fma(d, (double(x[u][j]) - mean) * rstd, s[j]);
                    s[VN + j] += d;
                }
            }
    }
#pragma unroll
    for (int j = 0; j < 2 * VN; j++) sh[w][j][lane] = s[j];
    __syncthreads();
    // wave w folds columns' sum w of each lane (2 VN <= W)
    if (w < 2 * VN && c + w % VN < cols) {
        double t = sh[0][w][lane];
        for (int i = 1; i < W; i++) t += sh[i][w][lane];
        a.part[(int64_t(blockIdx.y) * 2 + w / VN) * cols + c + w % VN] = T(t);
    }
}

// Device memory for the partials of one call.  A call that is being captured
// has a block of its own, which stays with the graph (it is not given back:
// the graph may be replayed whenever, beside any other); otherwise the block
// returns to the cache once the launches that use it are enqueued.
struct Partials {
    void *p = nullptr;
    bool keep = false;
    int open(size_t bytes)
    {
        keep = stream_recording();
        p = keep ? dev_alloc_own(bytes) : dev_alloc(bytes);
        return p ? NEURAL_OK : set_error(NEURAL_ERR_OUT_OF_MEMORY);
    }
    ~Partials()
    {
        if (p && !keep) dev_free(p);
    }
};

// Column sums by k_ln_cols and a fold.
template <typename T>
static int launch_ln_cols(LnGradArgs<T> a, T *dgamma, T *dbeta)
{
    const int64_t gx = ceil_div(a.cols, 64 * Vec16<T>::n);
    int64_t chunks = ceil_div(int64_t(num_cus()) * 2, gx);
    const int64_t most = ceil_div(a.rows, 32);
    chunks = chunks < most ? chunks : most;
    const int64_t chunk = ceil_div(a.rows, chunks);
    chunks = ceil_div(a.rows, chunk);
    Partials part;
    NH_TRY(part.open(size_t(chunks) * 2 * size_t(a.cols) * sizeof(T)));
    a.part = static_cast<T *>(part.p);
    NH_LAUNCH((k_ln_cols<T>), dim3(unsigned(gx), unsigned(chunks)), dim3(512), 0, stream(), a, chunk);
    NH_LAUNCH((k_ln_fold<T>), dim3(unsigned(ceil_div(2 * a.cols, 64))), dim3(1024), 0, stream(), a.part, chunks, a.cols,
              dgamma, dbeta);
    return check_launch();
}

// Few rows: what the one launch of k_ln_grad_few is for.  By the shape alone, so that equal
// rows give equal sums whatever else a call asks for.
constexpr int64_t kFewRows = 512, kFewValues = int64_t(1) << 20;
static bool few_rows(int64_t rows, int64_t cols) { return rows <= kFewRows && rows * cols <= kFewValues; }

template <typename T, int MODE, int NT, int VPT>
static int launch_ln_grad_rows(const LnGradArgs<T> &a0, T *dgamma, T *dbeta)
{
    using Plan = LnGradPlan<T, NT, VPT>;
    LnGradArgs<T> a = a0;
    const bool sums = dgamma || dbeta, rows = a.dx || a.dres;
    const int64_t need = ceil_div(a.rows, int64_t(Plan::RPB));
    if (few_rows(a.rows, a.cols)) {
        const auto few = [&](int64_t nr, int64_t nc) {
            NH_LAUNCH((k_ln_grad_few<T, NT, VPT, MODE>), dim3(unsigned(nr + nc)), dim3(Plan::NB), 0, stream(), a, int(nr),
                      dgamma, dbeta);
        };
        const int64_t nr = rows ? need : 0, nc = sums ? ceil_div(a.cols, 16) : 0;
        // the columns read what an output in place writes over: they go first then
        const bool over = a.dx == a.h || a.dx == a.dy || a.dres == a.h || a.dres == a.dy;
        if (rows && sums && over) {
            few(0, nc);
            few(nr, 0);
        } else {
            few(nr, nc);
        }
        return check_launch();
    }
    // as many blocks as the CUs hold at once, no more than rows
    const int64_t most = int64_t(num_cus()) * Plan::kPerCu;
    const int64_t nb = need < most ? need : most;
    if constexpr (VPT <= 8) {
        if (sums) {
            Partials part;
            NH_TRY(part.open(size_t(nb) * 2 * size_t(a.cols) * sizeof(T)));
            a.part = static_cast<T *>(part.p);
            NH_LAUNCH((k_ln_grad<T, NT, VPT, MODE, true>), dim3(unsigned(nb)), dim3(Plan::NB), 0, stream(), a);
            NH_LAUNCH((k_ln_fold<T>), dim3(unsigned(ceil_div(2 * a.cols, 64))), dim3(1024), 0, stream(), a.part, nb,
                      a.cols, dgamma, dbeta);
            return check_launch();
        }
    } else if (sums) {
        NH_TRY(launch_ln_cols(a, dgamma, dbeta));
    }
    if (rows) NH_LAUNCH((k_ln_grad<T, NT, VPT, MODE, false>), dim3(unsigned(nb)), dim3(Plan::NB), 0, stream(), a);
    return check_launch();
}

// The fewest of LO to HI vectors per lane of NT that hold the row.
template <typename T, int MODE, int NT, int LO, int HI>
static int launch_ln_grad_exact(const LnGradArgs<T> &a, int64_t ncv, T *dgamma, T *dbeta)
{
    if constexpr (LO < HI) {
        if (ncv > NT * LO) return launch_ln_grad_exact<T, MODE, NT, LO + 1, HI>(a, ncv, dgamma, dbeta);
    }
    return launch_ln_grad_rows<T, MODE, NT, LO>(a, dgamma, dbeta);
}

template <typename T, int MODE>
static int launch_ln_grad(const LnGradArgs<T> &a, T *dgamma, T *dbeta)
{
    const int64_t ncv = a.cols / Vec16<T>::n;
    if (ncv <= 4 * 4) return launch_ln_grad_exact<T, MODE, 4, 1, 4>(a, ncv, dgamma, dbeta);
    if (ncv <= 16 * 4) return launch_ln_grad_exact<T, MODE, 16, 2, 4>(a, ncv, dgamma, dbeta);
    if (ncv <= 64 * 4) return launch_ln_grad_exact<T, MODE, 64, 2, 4>(a, ncv, dgamma, dbeta);
    if (ncv <= 256 * 4) return launch_ln_grad_exact<T, MODE, 256, 2, 4>(a, ncv, dgamma, dbeta);
    if (ncv <= 512 * 8) return launch_ln_grad_exact<T, MODE, 512, 3, 8>(a, ncv, dgamma, dbeta);
    if (ncv <= 512 * 16) return launch_ln_grad_rows<T, MODE, 512, 16>(a, dgamma, dbeta);
    // the columns first: the row pass may write over what they read
    if (dgamma || dbeta) NH_TRY(launch_ln_cols(a, dgamma, dbeta));
    if (a.dx || a.dres)
        for_row_launches(a.rows, 1, [&](unsigned g, int64_t base) {
            NH_LAUNCH((k_ln_grad_wide<T, MODE>), dim3(g), dim3(kLnWide), 0, stream(), a, base);
        });
    return check_launch();
}

// ---- arguments -----------------------------------------------------------------------------

// A call's tensors, checked before anything runs: rows of the last dimension
// of `like`, in its type.  Optional tensors may be null.
struct LnCall {
    const NeuralTensor *like;
    int64_t rows = 0, cols = 0;

    int open(const NeuralTensor *t)
    {
        like = t;
        NH_TRY(check_tensor(t));
        if (t->ndim < 1) return set_error(NEURAL_ERR_DIM_MISMATCH);
        cols = t->shape[t->ndim - 1];
        rows = cols > 0 ? numel(t) / cols : 0;
        return is_contiguous(t) ? NEURAL_OK : set_error(NEURAL_ERR_INVALID_ARGUMENT);
    }
    int type(const NeuralTensor *t) const
    {
        NH_TRY(check_tensor(t));
        return t->dtype == like->dtype ? NEURAL_OK : set_error(NEURAL_ERR_DTYPE_MISMATCH);
    }
    // the shape of `like`
    int same(const NeuralTensor *t) const
    {
        if (!t) return NEURAL_OK;
        NH_TRY(type(t));
        if (t->ndim != like->ndim) return set_error(NEURAL_ERR_SHAPE_MISMATCH);
        for (int64_t i = 0; i < t->ndim; i++)
            if (t->shape[i] != like->shape[i]) return set_error(NEURAL_ERR_SHAPE_MISMATCH);
        return is_contiguous(t) ? NEURAL_OK : set_error(NEURAL_ERR_INVALID_ARGUMENT);
    }
    // n values (one per row or per column)
    int vec(const NeuralTensor *t, int64_t n) const
    {
        if (!t) return NEURAL_OK;
        NH_TRY(type(t));
        if (numel(t) != n) return set_error(NEURAL_ERR_SHAPE_MISMATCH);
        return is_contiguous(t) ? NEURAL_OK : set_error(NEURAL_ERR_INVALID_ARGUMENT);
    }
};

// Outputs share no bytes with each other or with an input, except that an output
// may be one of the first `in_place` inputs itself (tensors of the rows' shape).
static int check_apart(std::initializer_list<NeuralTensor *> outs, std::initializer_list<const NeuralTensor *> ins,
                       size_t in_place)
{
    for (auto o = outs.begin(); o != outs.end(); ++o) {
        if (!*o) continue;
        for (auto p = o + 1; p != outs.end(); ++p)
            if (tensors_may_overlap(*o, *p)) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
        size_t k = 0;
        for (const NeuralTensor *i : ins) {
            const bool itself = k++ < in_place && i && i->data == (*o)->data && numel(i) == numel(*o);
            if (!itself && tensors_may_overlap(*o, i)) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
        }
    }
    return NEURAL_OK;
}

template <typename T>
static int read_t(const NeuralTensor *t, const T *&p)
{
    const void *v = nullptr;
    if (t) NH_TRY(dev_read(t, &v));
    p = static_cast<const T *>(v);
    return NEURAL_OK;
}
template <typename T>
static int write_t(NeuralTensor *t, T *&p)
{
    void *v = nullptr;
    if (t) NH_TRY(dev_write(t, &v, true));
    p = static_cast<T *>(v);
    return NEURAL_OK;
}
static int written(std::initializer_list<NeuralTensor *> outs)
{
    for (NeuralTensor *t : outs)
        if (t) NH_TRY(dev_written(t));
    return set_error(NEURAL_OK);
}

struct LnTensors {
    NeuralTensor *out, *hidden;
    const NeuralTensor *in, *residual, *gamma, *beta;
    NeuralTensor *mean, *rstd;
};

template <typename T>
static int ln_run(const LnTensors &t, const LnCall &c, double eps, const DropArgs &drop, int mode)
{
    LnArgs<T> a{};
    a.rows = c.rows;
    a.cols = c.cols;
    a.eps = eps;
    a.drop = drop;
    NH_TRY(read_t(t.in, a.x));
    NH_TRY(read_t(t.residual, a.res));
    NH_TRY(read_t(t.gamma, a.gamma));
    NH_TRY(read_t(t.beta, a.beta));
    NH_TRY(write_t(t.out, a.y));
    NH_TRY(write_t(t.hidden, a.h));
    NH_TRY(write_t(t.mean, a.mean));
    NH_TRY(write_t(t.rstd, a.rstd));
    if (mode == LN_PLAIN) NH_TRY((launch_ln<T, LN_PLAIN>(a)));
    else if (mode == LN_ADD) NH_TRY((launch_ln<T, LN_ADD>(a)));
    else NH_TRY((launch_ln<T, LN_DROP>(a)));
    return written({t.out, t.hidden, t.mean, t.rstd});
}

static int ln_forward(const LnTensors &t, double p, const NeuralDropoutKey *key, double eps, bool joined)
{
    NH_TRY(ensure_init());
    if (!t.out || !t.in || (joined && !t.residual)) return set_error(NEURAL_ERR_NULL_POINTER);
    LnCall c;
    NH_TRY(c.open(t.in));
    NH_TRY(c.same(t.out));
    NH_TRY(c.same(t.hidden));
    NH_TRY(c.same(t.residual));
    NH_TRY(c.vec(t.gamma, c.cols));
    NH_TRY(c.vec(t.beta, c.cols));
    NH_TRY(c.vec(t.mean, c.rows));
    NH_TRY(c.vec(t.rstd, c.rows));
    if (!(eps >= 0.0 && eps < __builtin_inf())) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    NH_TRY(check_apart({t.out, t.hidden, t.mean, t.rstd}, {t.in, t.residual, t.gamma, t.beta}, 2));
    DropArgs drop{};
    if (joined && p != 0.0) NH_TRY(drop_args(p, key, drop));
    if (numel(t.in) == 0) return set_error(NEURAL_OK);
    const int mode = !joined ? LN_PLAIN : (p == 0.0 ? LN_ADD : LN_DROP);
    return t.in->dtype == NEURAL_DTYPE_FLOAT32 ? ln_run<float>(t, c, eps, drop, mode)
                                               : ln_run<double>(t, c, eps, drop, mode);
}

struct LnGradTensors {
    NeuralTensor *dx, *dres, *dgamma, *dbeta;
    const NeuralTensor *dy, *dh, *h, *gamma, *mean, *rstd;
};

template <typename T>
static int ln_grad_run(const LnGradTensors &t, const LnCall &c, const DropArgs &drop, int mode)
{
    LnGradArgs<T> a{};
    a.rows = c.rows;
    a.cols = c.cols;
    a.drop = drop;
    NH_TRY(read_t(t.dy, a.dy));
    NH_TRY(read_t(t.dh, a.dh));
    NH_TRY(read_t(t.h, a.h));
    NH_TRY(read_t(t.gamma, a.gamma));
    NH_TRY(read_t(t.mean, a.mean));
    NH_TRY(read_t(t.rstd, a.rstd));
    NH_TRY(write_t(t.dx, a.dx));
    NH_TRY(write_t(t.dres, a.dres));
    T *dgamma = nullptr, *dbeta = nullptr;
    NH_TRY(write_t(t.dgamma, dgamma));
    NH_TRY(write_t(t.dbeta, dbeta));
    if (mode == LN_PLAIN) NH_TRY((launch_ln_grad<T, LN_PLAIN>(a, dgamma, dbeta)));
    else if (mode == LN_ADD) NH_TRY((launch_ln_grad<T, LN_ADD>(a, dgamma, dbeta)));
    else NH_TRY((launch_ln_grad<T, LN_DROP>(a, dgamma, dbeta)));
    return written({t.dx, t.dres, t.dgamma, t.dbeta});
}

static int ln_backward(const LnGradTensors &t, double p, const NeuralDropoutKey *key, bool joined)
{
    NH_TRY(ensure_init());
    if (!t.dy || !t.h || !t.mean || !t.rstd || (!t.dx && !t.dres && !t.dgamma && !t.dbeta))
        return set_error(NEURAL_ERR_NULL_POINTER);
    LnCall c;
    NH_TRY(c.open(t.h));
    NH_TRY(c.same(t.dy));
    NH_TRY(c.same(t.dh));
    NH_TRY(c.same(t.dx));
    NH_TRY(c.same(t.dres));
    NH_TRY(c.vec(t.gamma, c.cols));
    NH_TRY(c.vec(t.mean, c.rows));
    NH_TRY(c.vec(t.rstd, c.rows));
    NH_TRY(c.vec(t.dgamma, c.cols));
    NH_TRY(c.vec(t.dbeta, c.cols));
    NH_TRY(check_apart({t.dx, t.dres, t.dgamma, t.dbeta}, {t.dy, t.h, t.dh, t.gamma, t.mean, t.rstd}, 3));
    DropArgs drop{};
    if (joined && p != 0.0) NH_TRY(drop_args(p, key, drop));
    if (numel(t.h) == 0) {  // sums over no rows
        if (t.dgamma) NH_TRY(neural_tensor_fill(t.dgamma, 0.0));
        if (t.dbeta) NH_TRY(neural_tensor_fill(t.dbeta, 0.0));
        return set_error(NEURAL_OK);
    }
    const int mode = !joined ? LN_PLAIN : (p == 0.0 ? LN_ADD : LN_DROP);
    return t.h->dtype == NEURAL_DTYPE_FLOAT32 ? ln_grad_run<float>(t, c, drop, mode)
                                              : ln_grad_run<double>(t, c, drop, mode);
}

}  // namespace nh

using namespace nh;

extern "C" {

int neural_layer_norm_forward(NeuralTensor *out, const NeuralTensor *in, const NeuralTensor *gamma,
                              const NeuralTensor *beta, double eps, NeuralTensor *mean, NeuralTensor *rstd)
{
    return ln_forward({out, nullptr, in, nullptr, gamma, beta, mean, rstd}, 0.0, nullptr, eps, false);
}

int neural_layer_norm_backward(NeuralTensor *grad_in, NeuralTensor *grad_gamma, NeuralTensor *grad_beta,
                               const NeuralTensor *grad_out, const NeuralTensor *in, const NeuralTensor *gamma,
                               const NeuralTensor *mean, const NeuralTensor *rstd)
{
    return ln_backward({grad_in, nullptr, grad_gamma, grad_beta, grad_out, nullptr, in, gamma, mean, rstd}, 0.0,
                       nullptr, false);
}

int neural_dropout_add_layer_norm_forward(NeuralTensor *out, NeuralTensor *hidden, const NeuralTensor *in,
                                          const NeuralTensor *residual, const NeuralTensor *gamma,
                                          const NeuralTensor *beta, double p, const NeuralDropoutKey *key, double eps,
                                          NeuralTensor *mean, NeuralTensor *rstd)
{
    return ln_forward({out, hidden, in, residual, gamma, beta, mean, rstd}, p, key, eps, true);
}

int neural_dropout_add_layer_norm_backward(NeuralTensor *grad_in, NeuralTensor *grad_residual,
                                           NeuralTensor *grad_gamma, NeuralTensor *grad_beta,
                                           const NeuralTensor *grad_out, const NeuralTensor *grad_hidden,
                                           const NeuralTensor *hidden, const NeuralTensor *gamma,
                                           const NeuralTensor *mean, const NeuralTensor *rstd, double p,
                                           const NeuralDropoutKey *key)
{
    return ln_backward({grad_in, grad_residual, grad_gamma, grad_beta, grad_out, grad_hidden, hidden, gamma, mean, rstd},
                       p, key, true);
}

}  // extern "C"
