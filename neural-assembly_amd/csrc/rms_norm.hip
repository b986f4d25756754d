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
        NH_TRY(open_raw(codes, t.codes, bytes, t.stride > c.cols));
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
