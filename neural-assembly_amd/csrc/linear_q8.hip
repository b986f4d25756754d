// linear_q8.hip -- the product of rows in 8 bits with 8-bit weights by output channel:
//   out[m, n] = act(scale[m] wscale[n] sum_k A[m, k] W[n, k] + bias[n]) + residual[m, n]
// The sum is exact in int32 (k <= 131071: |sum| <= k 2^14 < 2^31).  Its scaling and the bias
// are in double and rounded once to the dtype; the activation works on that value as the
// elementwise activations do, and the residual is added to its result: two more roundings in
// f32, each half a unit of values that the f32 elementwise calls would leave as well.
#include <cmath>

#include "act_fns.hpp"
#include "row_call.hpp"

namespace nh {

template <typename T>
struct LinArgs {
    const int8_t *a, *w;
    int64_t lda, ldw;
    const T *sa, *sw, *bias, *res;  // bias, res: may be null
    T *out;
    int64_t m, n, k;
    int act;
    double alpha;
};

// The activation of one value, by neural_bias_add_act's functors.
NH_DEV float act_of(float z, int act, double alpha)
{
    switch (act) {
    case NEURAL_ACT_RELU: return FnReluAct{}(z);
    case NEURAL_ACT_SIGMOID: return ActFn<ASigmoid>{}(z);
    case NEURAL_ACT_TANH: return TanhF32Fn{}(z);
    case NEURAL_ACT_GELU: return HeadTailFn<GeluF32>{}(z);
    case NEURAL_ACT_LEAKY_RELU: return ActFn<ALeaky>{ALeaky{alpha}}(z);
    case NEURAL_ACT_ELU: return HeadTailFn<EluF32>{EluF32{alpha}}(z);
    case NEURAL_ACT_SELU: return HeadTailFn<SeluF32>{}(z);
    case NEURAL_ACT_SWISH: return HeadTailFn<SwishF32>{}(z);
    case NEURAL_ACT_MISH: return HeadTailFn<MishF32>{}(z);
    case NEURAL_ACT_HARDSWISH: return HardswishF32Fn{}(z);
    case NEURAL_ACT_SOFTPLUS: return HeadTailFn<SoftplusF32>{}(z);
    case NEURAL_ACT_HARDTANH: return ActFn<AHardtanh>{}(z);
    default: return z;
    }
}
NH_DEV double act_of(double z, int act, double alpha)
{
    switch (act) {
    case NEURAL_ACT_RELU: return FnReluAct{}(z);
    case NEURAL_ACT_SIGMOID: return ActFn<ASigmoid>{}(z);
    case NEURAL_ACT_TANH: return ActFn<ATanh>{}(z);
    case NEURAL_ACT_GELU: return ActFn<AGelu>{}(z);
    case NEURAL_ACT_LEAKY_RELU: return ActFn<ALeaky>{ALeaky{alpha}}(z);
    case NEURAL_ACT_ELU: return ActFn<AElu>{AElu{alpha}}(z);
    case NEURAL_ACT_SELU: return ActFn<ASelu>{}(z);
    case NEURAL_ACT_SWISH: return ActFn<ASwish>{}(z);
    case NEURAL_ACT_MISH: return ActFn<AMish>{}(z);
    case NEURAL_ACT_HARDSWISH: return ActFn<AHardswish>{}(z);
    case NEURAL_ACT_SOFTPLUS: return ActFn<ASoftplus>{}(z);
    case NEURAL_ACT_HARDTANH: return ActFn<AHardtanh>{}(z);
    default: return z;
    }
}

// scale * sum + bias, rounded to the dtype.
template <typename T>
NH_DEV T lin_value(int acc, T sa, T sw, T bias)
{
    return T(double(acc) * (double(sa) * double(sw)) + double(bias));
}

// 64 x 64 results a block, 4 x 4 a lane, from tiles of 64 codes in LDS, byte by byte.
template <typename T>
__global__ __launch_bounds__(256) void k_lin_tile(LinArgs<T> g, int64_t nbx, int64_t b_base)
{
    __shared__ int sa[64][17], sw[64][17];
    const int tid = threadIdx.x;
    const int64_t b = b_base + blockIdx.x, m0 = b / nbx * 64, n0 = b % nbx * 64;
    const int ty = tid / 16, tx = tid % 16;
    int acc[4][4] = {};
    for (int64_t k0 = 0; k0 < g.k; k0 += 64) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = ty + 16 * i;
            const int64_t k = k0 + 4 * tx;
            uint32_t va = 0, vw = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (m0 + r < g.m && k + e < g.k) va |= uint32_t(uint8_t(g.a[(m0 + r) * g.lda + k + e])) << (8 * e);
                if (n0 + r < g.n && k + e < g.k) vw |= uint32_t(uint8_t(g.w[(n0 + r) * g.ldw + k + e])) << (8 * e);
            }
            sa[r][tx] = int(va);
            sw[r][tx] = int(vw);
        }
        __syncthreads();
#pragma unroll 4
        for (int q = 0; q < 16; q++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    acc[i][j] = __builtin_amdgcn_sdot4(sa[ty + 16 * i][q], sw[tx + 16 * j][q], acc[i][j], false);
        __syncthreads();
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m >= g.m || n >= g.n) continue;
            T z = act_of(lin_value<T>(acc[i][j], g.sa[m], g.sw[n], g.bias ? g.bias[n] : T(0)), g.act, g.alpha);
            if (g.res) z = z + g.res[m * g.n + n];
            g.out[m * g.n + n] = z;
        }
}

template <typename T>
static int launch_linear(const LinArgs<T> &g)
{
    const int64_t nbx = ceil_div(g.n, 64);
    for_row_launches(nbx * ceil_div(g.m, 64), 1, 256, [&](unsigned blocks, int64_t base) {
        NH_LAUNCH((k_lin_tile<T>), dim3(blocks), dim3(256), 0, stream(), g, nbx, base);
    });
    return check_launch();
}

// ---- arguments -----------------------------------------------------------------------------

struct LinTensors {
    NeuralTensor *out;
    const NeuralTensor *scale, *w_scale, *bias, *residual;
    const int8_t *codes, *w_codes;
    int64_t stride, w_stride, k;
    int act;
    double alpha;
};

constexpr int64_t kLinMaxK = 131071;

template <typename T>
static int lin_run(const LinTensors &t, const RowCall &c, const Staged &a, const Staged &w)
{
    LinArgs<T> g{};
    g.a = static_cast<const int8_t *>(a.dev);
    g.w = static_cast<const int8_t *>(w.dev);
    g.lda = t.stride;
    g.ldw = t.w_stride;
    g.m = c.rows;
    g.n = c.cols;
    g.k = t.k;
    g.act = t.act;
    g.alpha = t.alpha;
    NH_TRY(read_t(t.scale, g.sa));
    NH_TRY(read_t(t.w_scale, g.sw));
    NH_TRY(read_t(t.bias, g.bias));
    NH_TRY(read_t(t.residual, g.res));
    NH_TRY(write_t(t.out, g.out));
    NH_TRY(launch_linear<T>(g));
    return written({t.out});
}

static int linear_q8(const LinTensors &t)
{
    NH_TRY(ensure_init());
    if (!t.out || !t.scale || !t.w_scale || !t.codes || !t.w_codes) return set_error(NEURAL_ERR_NULL_POINTER);
    RowCall c;
    NH_TRY(c.open(t.out));
    NH_TRY(c.same(t.residual));
    NH_TRY(c.vec(t.scale, c.rows));
    NH_TRY(c.vec(t.w_scale, c.cols));
    NH_TRY(c.vec(t.bias, c.cols));
    if (t.k < 1 || t.stride < t.k || t.w_stride < t.k || t.act < NEURAL_ACT_NONE || t.act > NEURAL_ACT_HARDTANH)
        return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    if (t.k > kLinMaxK) return set_error(NEURAL_ERR_TENSOR_TOO_LARGE);
    NH_TRY(check_apart({t.out}, {t.residual, t.scale, t.w_scale, t.bias}, 1));
    if (numel(t.out) == 0) return set_error(NEURAL_OK);
    if (t.stride > int64_t(kMaxRawCount / uint64_t(c.rows)) || t.w_stride > int64_t(kMaxRawCount / uint64_t(c.cols)))
        return set_error(NEURAL_ERR_TENSOR_TOO_LARGE);
    const size_t a_bytes = size_t(c.rows - 1) * size_t(t.stride) + size_t(t.k);
    const size_t w_bytes = size_t(c.cols - 1) * size_t(t.w_stride) + size_t(t.k);
    if (raw_may_overlap(t.codes, a_bytes, t.out) || raw_may_overlap(t.w_codes, w_bytes, t.out))
        return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    Staged a, w;
    NH_TRY(a.open(t.codes, a_bytes, true));
    NH_TRY(w.open(t.w_codes, w_bytes, true));
    NH_TRY((t.out->dtype == NEURAL_DTYPE_FLOAT32 ? lin_run<float>(t, c, a, w) : lin_run<double>(t, c, a, w)));
    NH_TRY(a.finish(false));
    NH_TRY(w.finish(false));
    return set_error(NEURAL_OK);
}

}  // namespace nh

extern "C" int neural_linear_q8(NeuralTensor *out, const int8_t *codes, int64_t stride, const NeuralTensor *scale,
                                const int8_t *w_codes, int64_t w_stride, const NeuralTensor *w_scale, int64_t k,
                                const NeuralTensor *bias, int act, double alpha, const NeuralTensor *residual)
{
    return nh::linear_q8({out, scale, w_scale, bias, residual, codes, w_codes, stride, w_stride, k, act, alpha});
}
