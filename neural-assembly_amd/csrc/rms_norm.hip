// rms_norm.hip -- root-mean-square norm over the last dimension with the residual's
// addition before it, its output as values or as 8-bit codes with a scale per row, and rows
// to 8 bits without a norm.
//
//   h = x, or residual + x (rounded); rstd = 1 / sqrt(sum h^2 / C + eps)
//   values: y = h rstd gamma
//   codes:  w = h gamma, a = max |w|, code = 127 w / a (rstd cancels), scale = a rstd / 127
//   rows to 8 bits: w = x, scale = a / 127
//
// Sums and maxima are in double, and so is everything between the loads and the stores:
// f32 values round once per output (w is exact in double for f32 rows), and codes are
// decided exactly (quant_rows.hpp).
#include <cmath>

#include "rms_norm.hpp"
#include "row_call.hpp"

namespace nh {

enum { RMS_VALUES = 0, RMS_CODES = 1, ROW_CODES = 2 };

template <typename T>
struct RmsArgs {
    const T *x, *res, *gamma;  // res: where it is added; gamma: may be null
    T *h, *y, *rstd, *scale;   // h, rstd: may be null; y: values; scale: codes
    int8_t *codes;
    int64_t stride, rows, cols;
    double inv_c, eps;
};

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

// A block of kLnWide lanes walks a row of any width twice: h, its square sum and its largest
// |w|, then the outputs.
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
            const double hv = double(h.v[j]), g = double(v.g.v[j]);
            if constexpr (OUT == RMS_VALUES) o.v[j] = T(hv * rstd * g);
            else b[j] = codes.code(hv * g);
        }
        if (ADD && a.h) h.store(a.h + at + c);
        if constexpr (OUT == RMS_VALUES) o.store(a.y + at + c);
        else store_codes<W>(a.codes + r * a.stride + c, b);
    });
}

template <typename T, bool ADD, int OUT>
static int launch_rms(const RmsArgs<T> &a)
{
    for_row_launches(a.rows, 1, kLnWide, [&](unsigned g, int64_t base) {
        NH_LAUNCH((k_rms_wide<T, ADD, OUT>), dim3(g), dim3(kLnWide), 0, stream(), a, base);
    });
    return check_launch();
}

// ---- arguments -----------------------------------------------------------------------------

struct RmsTensors {
    NeuralTensor *out, *hidden;
    const NeuralTensor *in, *residual, *gamma;
    NeuralTensor *rstd, *scale;
    int8_t *codes;
    int64_t stride;
};

template <typename T>
static int rms_run(const RmsTensors &t, const RowCall &c, double eps, int out, Staged &codes)
{
    RmsArgs<T> a{};
    a.rows = c.rows;
    a.cols = c.cols;
    a.inv_c = 1.0 / double(c.cols);
    a.eps = eps;
    a.codes = static_cast<int8_t *>(codes.dev);
    a.stride = t.stride;
    NH_TRY(read_t(t.in, a.x));
    NH_TRY(read_t(t.residual, a.res));
    NH_TRY(read_t(t.gamma, a.gamma));
    NH_TRY(write_t(t.out, a.y));
    NH_TRY(write_t(t.hidden, a.h));
    NH_TRY(write_t(t.rstd, a.rstd));
    NH_TRY(write_t(t.scale, a.scale));
    if (out == ROW_CODES) NH_TRY((launch_rms<T, false, ROW_CODES>(a)));
    else if (out == RMS_CODES)
        NH_TRY((t.residual ? launch_rms<T, true, RMS_CODES>(a) : launch_rms<T, false, RMS_CODES>(a)));
    else NH_TRY((t.residual ? launch_rms<T, true, RMS_VALUES>(a) : launch_rms<T, false, RMS_VALUES>(a)));
    if (out != RMS_VALUES) NH_TRY(codes.finish(true));
    return written({t.out, t.hidden, t.rstd, t.scale});
}

static int rms_forward(const RmsTensors &t, double eps, int out)
{
    NH_TRY(ensure_init());
    if (!t.in || (out == RMS_VALUES ? !t.out : !t.codes || !t.scale)) return set_error(NEURAL_ERR_NULL_POINTER);
    RowCall c;
    NH_TRY(c.open(t.in));
    NH_TRY(c.same(t.out));
    NH_TRY(c.same(t.hidden));
    NH_TRY(c.same(t.residual));
    NH_TRY(c.vec(t.gamma, c.cols));
    NH_TRY(c.vec(t.rstd, c.rows));
    NH_TRY(c.vec(t.scale, c.rows));
    if (!(eps >= 0.0 && eps < __builtin_inf())) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    if (t.hidden && !t.residual) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    NH_TRY(check_apart({t.out, t.hidden, t.rstd, t.scale}, {t.in, t.residual, t.gamma}, 2));
    if (out != RMS_VALUES && t.stride < c.cols) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    if (numel(t.in) == 0) return set_error(NEURAL_OK);
    Staged codes;
    if (out != RMS_VALUES) {
        if (t.stride > int64_t(kMaxRawCount / uint64_t(c.rows))) return set_error(NEURAL_ERR_TENSOR_TOO_LARGE);
        const size_t bytes = size_t(c.rows) * size_t(t.stride);
        for (const NeuralTensor *u : {static_cast<const NeuralTensor *>(t.hidden), static_cast<const NeuralTensor *>(t.scale),
                                      t.in, t.residual, t.gamma})
            if (raw_may_overlap(t.codes, bytes, u)) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
        // (host memory between the rows comes back as it was)
        NH_TRY(codes.open(t.codes, bytes, t.stride > c.cols));
    }
    return t.in->dtype == NEURAL_DTYPE_FLOAT32 ? rms_run<float>(t, c, eps, out, codes)
                                               : rms_run<double>(t, c, eps, out, codes);
}

struct RmsGradTensors {
    NeuralTensor *dx, *dgamma;
    const NeuralTensor *dy, *dh, *h, *gamma, *rstd;
};

template <typename T>
static int rms_grad_run(const RmsGradTensors &t, const RowCall &c)
{
    RmsGradArgs<T> a{};
    a.rows = c.rows;
    a.cols = c.cols;
    NH_TRY(read_t(t.dy, a.dy));
    NH_TRY(read_t(t.dh, a.dh));
    NH_TRY(read_t(t.h, a.h));
    NH_TRY(read_t(t.gamma, a.gamma));
    NH_TRY(read_t(t.rstd, a.rstd));
    NH_TRY(write_t(t.dx, a.dx));
    T *dgamma = nullptr;
    NH_TRY(write_t(t.dgamma, dgamma));
    NH_TRY(launch_rms_grad<T>(a, dgamma));
    return written({t.dx, t.dgamma});
}

static int rms_backward(const RmsGradTensors &t)
{
    NH_TRY(ensure_init());
    if (!t.dy || !t.h || !t.rstd || (!t.dx && !t.dgamma)) return set_error(NEURAL_ERR_NULL_POINTER);
    RowCall c;
    NH_TRY(c.open(t.h));
    NH_TRY(c.same(t.dy));
    NH_TRY(c.same(t.dh));
    NH_TRY(c.same(t.dx));
    NH_TRY(c.vec(t.gamma, c.cols));
    NH_TRY(c.vec(t.rstd, c.rows));
    NH_TRY(c.vec(t.dgamma, c.cols));
    NH_TRY(check_apart({t.dx, nullptr, t.dgamma}, {t.dy, t.h, t.dh, t.gamma, t.rstd}, 3));
    if (numel(t.h) == 0) {  // a sum over no rows
        if (t.dgamma) NH_TRY(neural_tensor_fill(t.dgamma, 0.0));
        return set_error(NEURAL_OK);
    }
    return t.h->dtype == NEURAL_DTYPE_FLOAT32 ? rms_grad_run<float>(t, c) : rms_grad_run<double>(t, c);
}

}  // namespace nh

using namespace nh;

extern "C" {

int neural_rms_norm_forward(NeuralTensor *out, NeuralTensor *hidden, const NeuralTensor *in,
                            const NeuralTensor *residual, const NeuralTensor *gamma, double eps, NeuralTensor *rstd)
{
    return rms_forward({out, hidden, in, residual, gamma, rstd, nullptr, nullptr, 0}, eps, RMS_VALUES);
}

int neural_rms_norm_backward(NeuralTensor *grad_in, NeuralTensor *grad_gamma, const NeuralTensor *grad_out,
                             const NeuralTensor *grad_hidden, const NeuralTensor *hidden, const NeuralTensor *gamma,
                             const NeuralTensor *rstd)
{
    return rms_backward({grad_in, grad_gamma, grad_out, grad_hidden, hidden, gamma, rstd});
}

int neural_rms_norm_forward_q8(int8_t *codes, int64_t stride, NeuralTensor *scale, NeuralTensor *hidden,
                               const NeuralTensor *in, const NeuralTensor *residual, const NeuralTensor *gamma,
                               double eps)
{
    return rms_forward({nullptr, hidden, in, residual, gamma, nullptr, scale, codes, stride}, eps, RMS_CODES);
}

int neural_quantize_rows(int8_t *codes, int64_t stride, NeuralTensor *scale, const NeuralTensor *in)
{
    return rms_forward({nullptr, nullptr, in, nullptr, nullptr, nullptr, scale, codes, stride}, 0.0, ROW_CODES);
}

}  // extern "C"
