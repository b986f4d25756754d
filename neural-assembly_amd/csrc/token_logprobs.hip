// token_logprobs.hip -- log probabilities of given tokens, entropy and top alternatives of
// rows of logits, and their gradient.
//
//   z = x / temperature; with m = max x and d = x - m: s = sum exp(d / T), t = sum exp(d / T) d / T;
//   lse = m / T + log s; logprob = (x_t - m) / T - log s; entropy = log s - t / s
//   gradient: (g (1_t - p) - e p (log p + H)) / T, p = exp(z - lse)
//
// s and t are summed in double: where one token has nearly all the probability, logprob and
// entropy are as small as the rest of s, which a sum in float would round away beside 1.
#include <cmath>

#include "row_call.hpp"
#include "row_group.hpp"

namespace nh {

constexpr int kLpMaxTop = 64;

// An alternative: a larger value comes first, of equal ones the lower index.  i < 0: none.
template <typename T>
struct LpKey {
    T v;
    int i;
    NH_DEV static LpKey none() { return {-__builtin_inff(), -1}; }
    NH_DEV bool before(const LpKey &o) const
    {
        return i >= 0 && (o.i < 0 || v > o.v || (v == o.v && i < o.i));
    }
};

template <typename T>
struct LpArgs {
    const T *x;
    const int64_t *tokens;  // or null
    T *logprob, *entropy, *lse, *top_lp;  // any may be null
    int64_t *top_ids;                     // or null
    int64_t rows, cols;
    int k;
    double inv_t;
};

// A row per block, read for its maximum, for its sums, and for each alternative.
template <typename T>
__global__ __launch_bounds__(256) void k_lp_row(LpArgs<T> a, int64_t r_base)
{
    using G = RowGrp<256>;
    __shared__ double lds_m[4], lds_s[4], lds_t[4];
    __shared__ T lds_v[4];
    __shared__ int lds_i[4];
    const int64_t r = r_base + blockIdx.x, cols = a.cols;
    const T *x = a.x + r * cols;
    const int64_t tok = a.tokens ? a.tokens[r] : 0;
    const bool first = threadIdx.x == 0;
    if (tok < 0) {
        if (first) {
            if (a.logprob) a.logprob[r] = T(0);
            if (a.entropy) a.entropy[r] = T(0);
            if (a.lse) a.lse[r] = T(0);
        }
        for (int q = threadIdx.x; q < a.k; q += 256) {
            if (a.top_ids) a.top_ids[r * a.k + q] = -1;
            if (a.top_lp) a.top_lp[r * a.k + q] = -T(__builtin_inf());
        }
        return;
    }
    double m = -__builtin_inf();
    for (int64_t c = threadIdx.x; c < cols; c += 256) m = __builtin_fmax(m, double(x[c]));
    m = G::max(m, lds_m);
    const double m0 = m == -__builtin_inf() ? 0.0 : m;
    double s = 0.0, t = 0.0;
    for (int64_t c = threadIdx.x; c < cols; c += 256) {
        const double d = (double(x[c]) - m0) * a.inv_t;
        const double e = exp(d);
        s += e;
        t += d < -2000.0 ? 0.0 : e * d;
    }
    s = G::sum(s, lds_s);
    t = G::sum(t, lds_t);
    const double ls = log(s);  // -inf where every logit is masked, NaN with a NaN or an infinity
    if (first) {
        if (a.logprob) {
            double lp = __builtin_nan("");
            if (tok < cols) lp = s == 0.0 ? -__builtin_inf() : (double(x[tok]) - m0) * a.inv_t - ls;
            a.logprob[r] = T(lp);
        }
        if (a.entropy) a.entropy[r] = T(s == 0.0 ? 0.0 : ls - t / s);
        if (a.lse) a.lse[r] = T(m0 * a.inv_t + ls);
    }
    LpKey<T> last = LpKey<T>::none();
    for (int q = 0; q < a.k; q++) {
        LpKey<T> best = LpKey<T>::none();
        for (int64_t c = threadIdx.x; c < cols; c += 256) {
            const LpKey<T> k{x[c], int(c)};
            if (k.v > -T(__builtin_inf()) && (q == 0 || last.before(k)) && k.before(best)) best = k;
        }
        for (int off = 32; off >= 1; off >>= 1) {
            const LpKey<T> o{__shfl_xor(best.v, off, 64), __shfl_xor(best.i, off, 64)};
            if (o.before(best)) best = o;
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            lds_v[threadIdx.x >> 6] = best.v;
            lds_i[threadIdx.x >> 6] = best.i;
        }
        __syncthreads();
        for (int w = 0; w < 4; w++) {
            const LpKey<T> o{lds_v[w], lds_i[w]};
            if (o.before(best)) best = o;
        }
        last = best;
        const bool ok = s == s;
        if (first) {
            if (a.top_ids) a.top_ids[r * a.k + q] = ok ? int64_t(best.i) : -1;
            if (a.top_lp)
                a.top_lp[r * a.k + q] = !ok ? T(__builtin_nan(""))
                                        : best.i < 0 ? -T(__builtin_inf())
                                                     : T((double(best.v) - m0) * a.inv_t - ls);
        }
        if (best.i < 0) {
            for (int u = q + 1 + threadIdx.x; u < a.k; u += 256) {
                if (a.top_ids) a.top_ids[r * a.k + u] = -1;
                if (a.top_lp) a.top_lp[r * a.k + u] = ok ? -T(__builtin_inf()) : T(__builtin_nan(""));
            }
            break;
        }
    }
}

template <typename T>
struct LpGradArgs {
    const T *x, *g, *e, *lse, *entropy;  // g, e, entropy: may be null
    const int64_t *tokens;               // or null
    T *dx;
    int64_t rows, cols;
    double inv_t;
};

template <typename T>
__global__ __launch_bounds__(256) void k_lp_grad_row(LpGradArgs<T> a, int64_t r_base)
{
    const int64_t r = r_base + blockIdx.x, cols = a.cols;
    const T *x = a.x + r * cols;
    T *dx = a.dx + r * cols;
    const int64_t tok = a.tokens ? a.tokens[r] : -2;
    const double lse = double(a.lse[r]);
    if ((a.tokens && tok < 0) || lse == -__builtin_inf()) {
        for (int64_t c = threadIdx.x; c < cols; c += 256) dx[c] = T(0);
        return;
    }
    double g = a.g ? double(a.g[r]) : 0.0;
    if (a.g && tok >= cols) g = __builtin_nan("");
    const double e = a.e ? double(a.e[r]) : 0.0, h = a.e ? double(a.entropy[r]) : 0.0;
    for (int64_t c = threadIdx.x; c < cols; c += 256) {
        const double lp = double(x[c]) * a.inv_t - lse, p = exp(lp);
        double v = g * ((c == tok ? 1.0 : 0.0) - p);
        if (a.e && !(p == 0.0)) v -= e * p * (lp + h);
        dx[c] = T(v * a.inv_t);
    }
}

template <typename T>
static int launch_lp(const LpArgs<T> &a)
{
    for_row_launches(a.rows, 1, 256, [&](unsigned g, int64_t base) {
        NH_LAUNCH((k_lp_row<T>), dim3(g), dim3(256), 0, stream(), a, base);
    });
    return check_launch();
}

template <typename T>
static int launch_lp_grad(const LpGradArgs<T> &a)
{
    for_row_launches(a.rows, 1, 256, [&](unsigned g, int64_t base) {
        NH_LAUNCH((k_lp_grad_row<T>), dim3(g), dim3(256), 0, stream(), a, base);
    });
    return check_launch();
}

// ---- arguments -----------------------------------------------------------------------------

struct LpTensors {
    NeuralTensor *logprob, *entropy, *lse;
    int64_t *top_ids;
    NeuralTensor *top_lp;
    int64_t k;
    const NeuralTensor *logits;
    const int64_t *tokens;
};

static bool lp_temperature(double t) { return t > 0.0 && t < __builtin_inf() && 1.0 / t < __builtin_inf(); }

template <typename T>
static int lp_run(const LpTensors &t, const RowCall &c, double temperature, const Staged &tokens, const Staged &ids)
{
    LpArgs<T> a{};
    a.rows = c.rows;
    a.cols = c.cols;
    a.k = int(t.k);
    a.inv_t = 1.0 / temperature;
    a.tokens = static_cast<const int64_t *>(tokens.dev);
    a.top_ids = static_cast<int64_t *>(ids.dev);
    NH_TRY(read_t(t.logits, a.x));
    NH_TRY(write_t(t.logprob, a.logprob));
    NH_TRY(write_t(t.entropy, a.entropy));
    NH_TRY(write_t(t.lse, a.lse));
    NH_TRY(write_t(t.k ? t.top_lp : nullptr, a.top_lp));
    NH_TRY(launch_lp<T>(a));
    return written({t.logprob, t.entropy, t.lse, t.k ? t.top_lp : nullptr});
}

static int lp_forward(LpTensors t, double temperature)
{
    NH_TRY(ensure_init());
    if (!t.logits || (t.logprob && !t.tokens)) return set_error(NEURAL_ERR_NULL_POINTER);
    if (t.k < 0 || t.k > kLpMaxTop) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    if (t.k == 0) {
        t.top_ids = nullptr;
        t.top_lp = nullptr;
    }
    if (!t.logprob && !t.entropy && !t.lse && !t.top_ids && !t.top_lp) return set_error(NEURAL_ERR_NULL_POINTER);
    if (!t.top_ids && !t.top_lp) t.k = 0;
    RowCall c;
    NH_TRY(c.open(t.logits));
    NH_TRY(c.vec(t.logprob, c.rows));
    NH_TRY(c.vec(t.entropy, c.rows));
    NH_TRY(c.vec(t.lse, c.rows));
    NH_TRY(c.vec(t.top_lp, c.rows * t.k));
    if (!lp_temperature(temperature)) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    if (c.cols >= int64_t(1) << 31) return set_error(NEURAL_ERR_TENSOR_TOO_LARGE);
    NH_TRY(check_apart({t.logprob, t.entropy, t.lse, t.top_lp}, {t.logits}, 0));
    if (numel(t.logits) == 0) return set_error(NEURAL_OK);
    const size_t tok_bytes = size_t(c.rows) * 8, id_bytes = size_t(c.rows) * size_t(t.k) * 8;
    for (const NeuralTensor *u : {t.logprob, t.entropy, t.lse, t.top_lp, const_cast<NeuralTensor *>(t.logits)})
        if (raw_may_overlap(t.top_ids, id_bytes, u) || (u != t.logits && raw_may_overlap(t.tokens, tok_bytes, u)))
            return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    if (raws_may_overlap(t.top_ids, id_bytes, t.tokens, tok_bytes)) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    Staged tokens, ids;
    if (t.tokens) NH_TRY(tokens.open(t.tokens, tok_bytes, true));
    if (t.top_ids) NH_TRY(ids.open(t.top_ids, id_bytes, false));
    NH_TRY((t.logits->dtype == NEURAL_DTYPE_FLOAT32 ? lp_run<float>(t, c, temperature, tokens, ids)
                                                    : lp_run<double>(t, c, temperature, tokens, ids)));
    if (t.top_ids) NH_TRY(ids.finish(true));
    if (t.tokens) NH_TRY(tokens.finish(false));
    return set_error(NEURAL_OK);
}

struct LpGradTensors {
    NeuralTensor *dx;
    const NeuralTensor *g, *e, *logits;
    const int64_t *tokens;
    const NeuralTensor *lse, *entropy;
};

template <typename T>
static int lp_grad_run(const LpGradTensors &t, const RowCall &c, double temperature, const Staged &tokens)
{
    LpGradArgs<T> a{};
    a.rows = c.rows;
    a.cols = c.cols;
    a.inv_t = 1.0 / temperature;
    a.tokens = static_cast<const int64_t *>(tokens.dev);
    NH_TRY(read_t(t.logits, a.x));
    NH_TRY(read_t(t.g, a.g));
    NH_TRY(read_t(t.e, a.e));
    NH_TRY(read_t(t.lse, a.lse));
    NH_TRY(read_t(t.entropy, a.entropy));
    NH_TRY(write_t(t.dx, a.dx));
    NH_TRY(launch_lp_grad<T>(a));
    return written({t.dx});
}

static int lp_backward(const LpGradTensors &t, double temperature)
{
    NH_TRY(ensure_init());
    if (!t.dx || !t.logits || !t.lse || (!t.g && !t.e) || (t.g && !t.tokens) || (t.e && !t.entropy))
        return set_error(NEURAL_ERR_NULL_POINTER);
    RowCall c;
    NH_TRY(c.open(t.logits));
    NH_TRY(c.same(t.dx));
    NH_TRY(c.vec(t.g, c.rows));
    NH_TRY(c.vec(t.e, c.rows));
    NH_TRY(c.vec(t.lse, c.rows));
    NH_TRY(c.vec(t.entropy, c.rows));
    if (!lp_temperature(temperature)) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    if (c.cols >= int64_t(1) << 31) return set_error(NEURAL_ERR_TENSOR_TOO_LARGE);
    NH_TRY(check_apart({t.dx}, {t.logits, t.g, t.e, t.lse, t.entropy}, 1));
    if (numel(t.logits) == 0) return set_error(NEURAL_OK);
    const size_t tok_bytes = size_t(c.rows) * 8;
    if (raw_may_overlap(t.tokens, tok_bytes, t.dx)) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    Staged tokens;
    if (t.tokens) NH_TRY(tokens.open(t.tokens, tok_bytes, true));
    NH_TRY((t.logits->dtype == NEURAL_DTYPE_FLOAT32 ? lp_grad_run<float>(t, c, temperature, tokens)
                                                    : lp_grad_run<double>(t, c, temperature, tokens)));
    if (t.tokens) NH_TRY(tokens.finish(false));
    return set_error(NEURAL_OK);
}

}  // namespace nh

using namespace nh;

extern "C" {

int neural_token_logprobs_forward(NeuralTensor *logprob, NeuralTensor *entropy, NeuralTensor *lse, int64_t *top_ids,
                                  NeuralTensor *top_logprobs, int64_t k, const NeuralTensor *logits,
                                  const int64_t *tokens, double temperature)
{
    return lp_forward({logprob, entropy, lse, top_ids, top_logprobs, k, logits, tokens}, temperature);
}

int neural_token_logprobs_backward(NeuralTensor *grad_logits, const NeuralTensor *g, const NeuralTensor *e,
                                   const NeuralTensor *logits, const int64_t *tokens, const NeuralTensor *lse,
                                   const NeuralTensor *entropy, double temperature)
{
    return lp_backward({grad_logits, g, e, logits, tokens, lse, entropy}, temperature);
}

}  // extern "C"
