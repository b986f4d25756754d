// activations.hip -- the ten tensor-level activations plus sigmoid.
//
// Formulas are those of activations_c.c:124-158 (and node_sigmoid,
// activations.asm:352-413): each element is widened to double, the formula is
// evaluated in double, and f32 tensors store one final rounding to float
// (activations_c.c:71-77).
//
// The piecewise-linear ones (leaky_relu, hardswish, hardtanh) and the exp-based
// ones (elu, selu, swish, sigmoid) evaluate the reference expression as
// written (f32 tensors: in float where the reference's double rounding is
// invisible at 1e-5, see the *F32 functors).  tanh, gelu, mish and softplus are evaluated by closed forms built
// on one double exp, which costs a fifth to a third of the device library's
// double tanh / log on gfx950 (measured ~141 and ~70 FP64 instructions per
// element for tanh and log, ~18 for exp), while keeping the two roundings of
// the reference that decide its low-order result:
//
//   u = 1.0 + exp(x)   (softplus, mish): for x << 0, u - 1 is exp(x) quantized to
//                       multiples of 2^-52; the closed forms take t = u - 1 (exact)
//                       so the result carries the reference's quantization;
//   1.0 + tanh(z)       (gelu, z << 0): tanh(z) rounds to a multiple of 2^-53 in
//                       [-1, -0.5], so 1 + tanh(z) is that multiple; it is
//                       rebuilt as rint(eps * 2^53) * 2^-53 from eps = 1 - |tanh z|
//                       computed to a few ulp (a few 2^-53 steps at most).
//
// Everything else matches the reference's value to ~1e-14 relative or better
// (libm differences aside), far inside the 1e-5 (f32) / 1e-12 + 1e-15 (f64) bars.
// f32 tensors use the float-output paths below.
#include <cmath>

#include "act_fns.hpp"
#include "ew_impl.hpp"

namespace nh {

template <class A, class F32>
static int act2(void *out, const void *in, F32 f32, A a = A{})
{
    if (!out || !in) return set_error(NEURAL_ERR_NULL_POINTER);
    ActFn<A> f64{a};
    return run_unary(static_cast<NeuralTensor *>(out), static_cast<const NeuralTensor *>(in), f32, f64);
}

template <class A>
static int act(void *out, const void *in, A a = A{})
{
    return act2<A>(out, in, ActFn<A>{a}, a);
}

static int act_gelu_impl(void *out, const void *in) { return act2<AGelu>(out, in, HeadTailFn<GeluF32>{}); }
static int act_swish_impl(void *out, const void *in) { return act2<ASwish>(out, in, HeadTailFn<SwishF32>{}); }
static int act_mish_impl(void *out, const void *in) { return act2<AMish>(out, in, HeadTailFn<MishF32>{}); }
static int act_softplus_impl(void *out, const void *in) { return act2<ASoftplus>(out, in, HeadTailFn<SoftplusF32>{}); }
static int act_tanh_impl(void *out, const void *in) { return act2<ATanh>(out, in, TanhF32Fn{}); }
static int act_elu_impl(void *out, const void *in, double alpha)
{
    return act2<AElu>(out, in, HeadTailFn<EluF32>{EluF32{alpha}}, AElu{alpha});
}
static int act_selu_impl(void *out, const void *in) { return act2<ASelu>(out, in, HeadTailFn<SeluF32>{}); }

// Bias add then activation, one pass: y = act(x + b) with x + b rounded in
// the tensor's dtype first (nn_layers.asm:472-539 then activations_c.c), so
// the result equals neural_bias_add followed by the activation bit for bit.
template <class F32, class F64>
struct OpAddAct {
    using F32T = F32;
    F32 f32;
    F64 f64;
    NH_DEV float operator()(float x, float b) const { return f32(x + b); }
    NH_DEV double operator()(double x, double b) const { return f64(x + b); }
};
template <class F32, class F64>
OpAddAct<F32, F64> add_act(F32 f32, F64 f64) { return {f32, f64}; }

static int bias_add_act(NeuralTensor *out, const NeuralTensor *x, const NeuralTensor *bias, int act, double alpha)
{
    if (!out || !x || !bias) return set_error(NEURAL_ERR_NULL_POINTER);
    if (bias->ndim < 1 || x->ndim < 1 || numel(bias) != x->shape[x->ndim - 1])
        return set_error(NEURAL_ERR_SHAPE_MISMATCH);
    if (out->ndim != x->ndim) return set_error(NEURAL_ERR_SHAPE_MISMATCH);
    for (int64_t i = 0; i < x->ndim; i++)
        if (out->shape[i] != x->shape[i]) return set_error(NEURAL_ERR_SHAPE_MISMATCH);
    switch (act) {
    case NEURAL_ACT_NONE: return binary_api(out, x, bias, add_act(FnIdentity{}, FnIdentity{}));
    case NEURAL_ACT_RELU: return binary_api(out, x, bias, add_act(FnReluAct{}, FnReluAct{}));
    case NEURAL_ACT_SIGMOID: return binary_api(out, x, bias, add_act(ActFn<ASigmoid>{}, ActFn<ASigmoid>{}));
    case NEURAL_ACT_TANH: return binary_api(out, x, bias, add_act(TanhF32Fn{}, ActFn<ATanh>{}));
    case NEURAL_ACT_GELU: return binary_api(out, x, bias, add_act(HeadTailFn<GeluF32>{}, ActFn<AGelu>{}));
    case NEURAL_ACT_LEAKY_RELU:
        return binary_api(out, x, bias, add_act(ActFn<ALeaky>{ALeaky{alpha}}, ActFn<ALeaky>{ALeaky{alpha}}));
    case NEURAL_ACT_ELU:
        return binary_api(out, x, bias, add_act(HeadTailFn<EluF32>{EluF32{alpha}}, ActFn<AElu>{AElu{alpha}}));
    case NEURAL_ACT_SELU: return binary_api(out, x, bias, add_act(HeadTailFn<SeluF32>{}, ActFn<ASelu>{}));
    case NEURAL_ACT_SWISH: return binary_api(out, x, bias, add_act(HeadTailFn<SwishF32>{}, ActFn<ASwish>{}));
    case NEURAL_ACT_MISH: return binary_api(out, x, bias, add_act(HeadTailFn<MishF32>{}, ActFn<AMish>{}));
    case NEURAL_ACT_HARDSWISH: return binary_api(out, x, bias, add_act(HardswishF32Fn{}, ActFn<AHardswish>{}));
    case NEURAL_ACT_SOFTPLUS:
        return binary_api(out, x, bias, add_act(HeadTailFn<SoftplusF32>{}, ActFn<ASoftplus>{}));
    case NEURAL_ACT_HARDTANH: return binary_api(out, x, bias, add_act(ActFn<AHardtanh>{}, ActFn<AHardtanh>{}));
    default: return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    }
}

}  // namespace nh

using namespace nh;

extern "C" {

int act_tanh(void *out, const void *in) { return act_tanh_impl(out, in); }
int act_gelu(void *out, const void *in) { return act_gelu_impl(out, in); }
int act_leaky_relu(void *out, const void *in, double alpha) { return act<ALeaky>(out, in, ALeaky{alpha}); }
int act_elu(void *out, const void *in, double alpha) { return act_elu_impl(out, in, alpha); }
int act_selu(void *out, const void *in) { return act_selu_impl(out, in); }
int act_swish(void *out, const void *in) { return act_swish_impl(out, in); }
int act_mish(void *out, const void *in) { return act_mish_impl(out, in); }
int act_hardswish(void *out, const void *in) { return act2<AHardswish>(out, in, HardswishF32Fn{}); }
int act_softplus(void *out, const void *in) { return act_softplus_impl(out, in); }
int act_hardtanh(void *out, const void *in) { return act<AHardtanh>(out, in); }

// Tensor-typed aliases of the header's neural_* activations
// (neural_api.h:387-486).
int neural_sigmoid(NeuralTensor *out, const NeuralTensor *in) { return act<ASigmoid>(out, in); }
int neural_tanh(NeuralTensor *out, const NeuralTensor *in) { return act_tanh_impl(out, in); }
int neural_gelu(NeuralTensor *out, const NeuralTensor *in) { return act_gelu_impl(out, in); }
int neural_leaky_relu(NeuralTensor *out, const NeuralTensor *in, double alpha) { return act<ALeaky>(out, in, ALeaky{alpha}); }
int neural_elu(NeuralTensor *out, const NeuralTensor *in, double alpha) { return act_elu_impl(out, in, alpha); }
int neural_selu(NeuralTensor *out, const NeuralTensor *in) { return act_selu_impl(out, in); }
int neural_swish(NeuralTensor *out, const NeuralTensor *in) { return act_swish_impl(out, in); }
int neural_mish(NeuralTensor *out, const NeuralTensor *in) { return act_mish_impl(out, in); }
int neural_hardswish(NeuralTensor *out, const NeuralTensor *in) { return act2<AHardswish>(out, in, HardswishF32Fn{}); }
int neural_softplus(NeuralTensor *out, const NeuralTensor *in) { return act_softplus_impl(out, in); }
int neural_hardtanh(NeuralTensor *out, const NeuralTensor *in) { return act<AHardtanh>(out, in); }

int neural_bias_add_act(NeuralTensor *out, const NeuralTensor *x, const NeuralTensor *bias, int act, double alpha)
{
    return bias_add_act(out, x, bias, act, alpha);
}

}  // extern "C"
