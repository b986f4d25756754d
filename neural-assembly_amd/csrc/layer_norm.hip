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
// Everything between the loads and the stores is in double, f32 rows rounded once per
// output (dgamma and dbeta once more for what each block leaves of them); mean and rstd
// are stored in the rows' type (the mean's rounding moves xh by what half an ulp of an
// input of the mean's size would).  The variance is taken from the centred values, which
// are still in registers.
//
// A row is held by one group of lanes, part of a wave to a block of 1024, at any
// width and alignment (RowCut), so each tensor is read once and written once.
#include <cmath>
#include <initializer_list>

#include "layer_norm.hpp"

namespace nh {

// ---- forward -------------------------------------------------------------------------------

template <typename T>
struct LnArgs {
    const T *x, *res, *gamma, *beta;  // res: joined forms; gamma, beta: may be null
    T *h, *y, *mean, *rstd;           // h, mean, rstd: may be null
    int64_t rows, cols;
    double inv_c, eps;
    DropArgs drop;
};

// How a group's lanes hold a row: NT lanes, VPT vectors each, the first F of them whole.
// kAhead: two rows, one in flight while the other is worked on.
// Then a CU holds about 12 vectors a lane and SIMD of rows in flight (48 KB); more
// or fewer wait longer: f32 [8192, 4096] (4 vectors) 45.7 us with 3 waves a SIMD, 47.4 with
// 4, and 50.7 with a row per block; [16384, 2048] (2 vectors) 46.9 with 5, 48.0 with 6,
// 49.2 with 3.  The joined forms, with two loads for a value and two stores, want the
// most blocks instead.
template <typename T, int NT, int VPT, int MODE>
struct LnPlan {
    static constexpr int NB = NT < 256 ? 256 : NT, RPB = NB / NT;
    static constexpr bool kAhead = MODE == LN_PLAIN && NT < 1024;
    // gamma and beta are loaded before the row's sums, not behind them: joined f32 [64, 4096]
    // 4.5 -> 4.1 us, [8192, 4096] 93.0 -> 89.5 (with dropout 93.0, 92.4; [4096, 1024], from the
    // caches, 12.5 -> 13.4: 96 registers instead of 64)
    static constexpr bool kParams = kAhead || (VPT <= 4 && NT < 1024);
    static constexpr int F = NT < 1024 || VPT <= 4 ? VPT - 1 : VPT / 2;
    static constexpr int kWaves = !kAhead ? (NT == 1024 ? 4 : 1) : VPT >= 5 ? 2 : VPT >= 3 ? 3 : VPT == 2 ? 5 : 8;
    static constexpr int kPerCu = kWaves * 256 / NB;  // resident blocks
};

// Groups of NT lanes walk the rows, r = group, group + groups, ...: a row is read
// once, its mean and then its variance taken from the registers.  Bound by HBM.
template <typename T, int NT, int VPT, int MODE, bool PAST>
__global__ __launch_bounds__((LnPlan<T, NT, VPT, MODE>::NB), (LnPlan<T, NT, VPT, MODE>::kWaves)) void k_ln_rows(
    LnArgs<T> a, int64_t r_base)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    using G = RowGrp<NT>;
    using K = RowKeep<T, NT, VPT>;
    using S = RowStream<T, PAST>;
    using Plan = LnPlan<T, NT, VPT, MODE>;
    constexpr int VN = Vec16<T>::n, RPB = Plan::RPB;
    __shared__ double lds_s[2][G::kWaves], lds_q[2][G::kWaves];
    __shared__ uint8_t lds_keep[2][MODE == LN_DROP ? RPB : 1][MODE == LN_DROP ? K::kBytes : 1];
    const int lane = threadIdx.x % NT, sub = threadIdx.x / NT;
    const int64_t cols = a.cols;
    const RowCut<T> cut(cols);
    const auto in_row = [&](int k) { return k < Plan::F || lane + k * NT < cut.ncv; };
    const bool has_t = lane < cut.rem;
    const auto param = [&](const T *p, int k, T none) {
        V v;
#pragma unroll
        for (int j = 0; j < VN; j++) v[j] = none;
        if (p && in_row(k)) v = *(reinterpret_cast<const U *>(p) + lane + k * NT);
        return v;
    };
    V g[Plan::kParams ? VPT : 1], b[Plan::kParams ? VPT : 1];
    if constexpr (Plan::kParams) {
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            g[k] = param(a.gamma, k, T(1));
            b[k] = param(a.beta, k, T(0));
        }
    }
    const T gt = a.gamma && has_t ? a.gamma[cut.sc(lane)] : T(1), bt = a.beta && has_t ? a.beta[cut.sc(lane)] : T(0);
    const double inv_c = a.inv_c;
    const DropKey key(a.drop);
    const T scale = T(a.drop.scale);
    struct Row {
        V x[VPT], res[MODE == LN_PLAIN ? 1 : VPT];
        T xt, rest;
    };
    const auto load = [&](Row &w, int64_t r) {
        const int64_t at = r * cols;
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) w.x[k] = S::load(reinterpret_cast<const U *>(a.x + at) + lane + k * NT);
        w.xt = has_t ? a.x[at + cut.sc(lane)] : T(0);
        if constexpr (MODE != LN_PLAIN) {
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (in_row(k)) w.res[k] = S::load(reinterpret_cast<const U *>(a.res + at) + lane + k * NT);
            w.rest = has_t ? a.res[at + cut.sc(lane)] : T(0);
        }
    };
    const auto work = [&](Row &w, int64_t r, int odd) {
        const int64_t at = r * cols;
        if constexpr (MODE != LN_PLAIN) {
            if constexpr (MODE == LN_DROP) {
                K keep;
                keep.make(r, cols, cut, lane, key, lds_keep[odd][sub]);
#pragma unroll
                for (int k = 0; k < VPT; k++)
                    if (in_row(k)) {
#pragma unroll
                        for (int j = 0; j < VN; j++)
                            w.x[k][j] = w.res[k][j] + dropped<T>(w.x[k][j], scale, keep.m[k], K::bit(j));
                    }
                w.xt = w.rest + dropped<T>(w.xt, scale, keep.tail, 0);
            } else {
#pragma unroll
                for (int k = 0; k < VPT; k++)
                    if (in_row(k)) {
#pragma unroll
                        for (int j = 0; j < VN; j++) w.x[k][j] = w.res[k][j] + w.x[k][j];
                    }
                w.xt = w.rest + w.xt;
            }
            if (a.h) {
#pragma unroll
                for (int k = 0; k < VPT; k++)
                    if (in_row(k)) S::store(w.x[k], reinterpret_cast<U *>(a.h + at) + lane + k * NT);
                if (has_t) a.h[at + cut.sc(lane)] = w.xt;
            }
        }
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) {
#pragma unroll
                for (int j = 0; j < VN; j++) s += double(w.x[k][j]);
            }
        if (has_t) s += double(w.xt);
        const double mean = over(G::sum(s, lds_s[odd]), cols, inv_c);
        double q = 0.0;
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) {
                hide(w.x[k]);
#pragma unroll
                for (int j = 0; j < VN; j++) {
                    const double d = double(w.x[k][j]) - mean;
                    q = __builtin_fma(d, d, q);
                }
            }
        if (has_t) {
            const double d = double(w.xt) - mean;
            q = __builtin_fma(d, d, q);
        }
        const double rstd = rsqrt_d(G::sum(q, lds_q[odd]) * inv_c + a.eps);
        if (lane == 0) {
            if (a.mean) a.mean[r] = T(mean);
            if (a.rstd) a.rstd[r] = T(rstd);
        }
        const auto out = [&](T xv, T gv, T bv) {
            return T(__builtin_fma((double(xv) - mean) * rstd, double(gv), double(bv)));
        };
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) {
                hide(w.x[k]);
                V gk, bk, o;
                if constexpr (Plan::kParams) {
                    hide(g[k]);
                    hide(b[k]);
                    gk = g[k];
                    bk = b[k];
                } else {
                    gk = param(a.gamma, k, T(1));
                    bk = param(a.beta, k, T(0));
                }
#pragma unroll
                for (int j = 0; j < VN; j++) o[j] = out(w.x[k][j], gk[j], bk[j]);
                S::store(o, reinterpret_cast<U *>(a.y + at) + lane + k * NT);
            }
        if (has_t) a.y[at + cut.sc(lane)] = out(w.xt, gt, bt);
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

// Rows wider than a block's registers, in three walks of a block: h and its sum, the
// centred squares, y.  How much of the row the caches keep between the walks bounds it
// (f32 [335, 100000] 100 us, 177 us joined with dropout and h stored; a copy of the same
// bytes 43 and 86; element by element it took 178 and 410, and f32 [127, 262147] 390, now
// 132).
template <typename T, int MODE>
__global__ __launch_bounds__(kLnWide) void k_ln_wide(LnArgs<T> a, int64_t r_base)
{
    using G = RowGrp<kLnWide>;
    __shared__ double lds_s[G::kWaves], lds_q[G::kWaves];
    const DropKey key(a.drop);
    const T scale = T(a.drop.scale);
    const int64_t r = r_base + blockIdx.x, cols = a.cols, at = r * cols;
    const auto load_in = [&](auto w, int64_t c) {
        constexpr int W = decltype(w)::value;
        struct {
            Pack<T, W> x, res;
        } v;
        v.x = Pack<T, W>::load(a.x + at + c);
        if constexpr (MODE != LN_PLAIN) v.res = Pack<T, W>::load(a.res + at + c);
        return v;
    };
    const auto join = [&](auto w, int64_t c, const auto &v) {  // h's values
        constexpr int W = decltype(w)::value;
        Pack<T, W> h = v.x;
        if constexpr (MODE != LN_PLAIN) {
            const uint32_t m = MODE == LN_DROP ? keep_at<W>(at + c, key) : 0;
#pragma unroll
            for (int j = 0; j < W; j++)
                h.v[j] = v.res.v[j] + (MODE == LN_DROP ? dropped<T>(h.v[j], scale, m, j) : h.v[j]);
        }
        return h;
    };
    // h once more, from where it was stored or made again
    const auto again = [&](auto use) {
        if (MODE != LN_PLAIN && a.h)
            walk_row<T>(cols, [&](auto w, int64_t c) { return Pack<T, decltype(w)::value>::load(a.h + at + c); }, use);
        else
            walk_row<T>(cols, load_in, [&](auto w, int64_t c, const auto &v) { use(w, c, join(w, c, v)); });
    };
    double s = 0.0, q = 0.0;
    walk_row<T>(cols, load_in, [&](auto w, int64_t c, const auto &v) {
        constexpr int W = decltype(w)::value;
        const Pack<T, W> h = join(w, c, v);
        if (MODE != LN_PLAIN && a.h) h.store(a.h + at + c);
#pragma unroll
        for (int j = 0; j < W; j++) s += double(h.v[j]);
    });
    const double mean = over(G::sum(s, lds_s), cols, a.inv_c);
    again([&](auto w, int64_t, const auto &h) {
#pragma unroll
        for (int j = 0; j < decltype(w)::value; j++) {
            const double d = double(h.v[j]) - mean;
            q = __builtin_fma(d, d, q);
        }
    });
    const double rstd = rsqrt_d(G::sum(q, lds_q) * a.inv_c + a.eps);
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[r] = T(mean);
        if (a.rstd) a.rstd[r] = T(rstd);
    }
    again([&](auto w, int64_t c, const auto &h) {
        constexpr int W = decltype(w)::value;
        Pack<T, W> g, b, o;
        if (a.gamma) g = Pack<T, W>::load(a.gamma + c);
        if (a.beta) b = Pack<T, W>::load(a.beta + c);
#pragma unroll
        for (int j = 0; j < W; j++)
            o.v[j] = T(__builtin_fma((double(h.v[j]) - mean) * rstd, a.gamma ? double(g.v[j]) : 1.0,
                                     a.beta ? double(b.v[j]) : 0.0));
        o.store(a.y + at + c);
    });
}

template <typename T, int MODE, int NT, int VPT>
static void launch_ln_rows(const LnArgs<T> &a)
{
    using Plan = LnPlan<T, NT, VPT, MODE>;
    with_stream<T, NT>(a.cols, [&](auto past) {
        const auto launch = [&](unsigned g, int64_t base) {
            NH_LAUNCH((k_ln_rows<T, NT, VPT, MODE, decltype(past)::value>), dim3(g), dim3(Plan::NB), 0, stream(), a, base);
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
template <typename T, int MODE, int NT, int LO, int HI>
static void launch_ln_exact(const LnArgs<T> &a, int64_t ncv)
{
    if constexpr (LO < HI) {
        if (ncv > NT * LO) return launch_ln_exact<T, MODE, NT, LO + 1, HI>(a, ncv);
    }
    launch_ln_rows<T, MODE, NT, LO>(a);
}

// The fewest lanes whose registers hold the row, so that the sums over them and what a row
// costs once are spread over the most values; from 8193 f32 values a block of 1024, which
// answers a single row sooner.  (All forms go by the width alone, and alike: equal rows have
// equal statistics.)
template <typename T, int MODE>
static int launch_ln(const LnArgs<T> &a)
{
    const int64_t ncv = a.cols / Vec16<T>::n;
    if (ncv <= 4) launch_ln_rows<T, MODE, 4, 1>(a);
    else if (ncv <= 8 * 4) launch_ln_exact<T, MODE, 8, 1, 4>(a, ncv);
    else if (ncv <= 16 * 4) launch_ln_exact<T, MODE, 16, 3, 4>(a, ncv);
    else if (ncv <= 32 * 4) launch_ln_exact<T, MODE, 32, 3, 4>(a, ncv);
    else if (ncv <= 64 * 4) launch_ln_exact<T, MODE, 64, 3, 4>(a, ncv);
    else if (ncv <= 256 * 8) launch_ln_exact<T, MODE, 256, 2, 8>(a, ncv);
    else if (ncv <= 1024 * 4) launch_ln_exact<T, MODE, 1024, 3, 4>(a, ncv);
    else if (ncv <= 1024 * 8) launch_ln_rows<T, MODE, 1024, 8>(a);
    else if (ncv <= 1024 * 16) launch_ln_rows<T, MODE, 1024, 16>(a);
    else
        for_row_launches(a.rows, 1, kLnWide, [&](unsigned g, int64_t base) {
            NH_LAUNCH((k_ln_wide<T, MODE>), dim3(g), dim3(kLnWide), 0, stream(), a, base);
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

// Outputs share no bytes with each other or with an input, except that one of the first
// kRowOuts outputs may be one of the first `row_ins` inputs itself: those are the tensors
// of the rows' shape.  (Of one row, or one column, the others have as many values: the
// column sums are written beside the rows that are still read.)
constexpr ptrdiff_t kRowOuts = 2;
static int check_apart(std::initializer_list<NeuralTensor *> outs, std::initializer_list<const NeuralTensor *> ins,
                       size_t row_ins)
{
    for (auto o = outs.begin(); o != outs.end(); ++o) {
        if (!*o) continue;
        const size_t in_place = o - outs.begin() < kRowOuts ? row_ins : 0;
        for (auto p = o + 1; p != outs.end(); ++p)
            if (tensors_may_overlap(*o, *p)) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
        size_t k = 0;
        for (const NeuralTensor *i : ins) {
            const bool itself = k++ < in_place && i && (i->data == (*o)->data || i->dev == (*o)->dev) &&
                                numel(i) == numel(*o);
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
    a.inv_c = 1.0 / double(c.cols);
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
