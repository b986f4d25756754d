// counter_dropout.hip -- inverted dropout whose mask is a function of the
// element's index, a seed and an offset (philox.hpp), forward and backward: no
// mask is stored and no state is kept between calls.
//
// out = keep ? x * scale : +0 with scale = 1 / (1 - p) rounded to the type; the
// backward pass is the same map of the gradient.  What bounds it: HBM, one read
// and one write.
#include <cmath>

#include "philox.hpp"

namespace nh {

int drop_args(double p, const NeuralDropoutKey *key, DropArgs &a)
{
    if (!key) return set_error(NEURAL_ERR_NULL_POINTER);
    if (!(p >= 0.0 && p <= 1.0)) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    if (reinterpret_cast<uintptr_t>(key) & 7) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    a.dev = nullptr;
    a.seed = a.offset = 0;
    if (is_device_ptr(key)) {
        a.dev = reinterpret_cast<const uint64_t *>(key);
    } else {
        a.seed = key->seed;
        a.offset = key->offset;
    }
    const uint64_t thr = uint64_t(std::nearbyint(p * 4294967296.0));
    a.t = uint32_t(thr >> 16);
    a.tlow = uint32_t(thr & 0xFFFFu);
    a.scale = p < 1.0 ? 1.0 / (1.0 - p) : 0.0;
    return NEURAL_OK;
}

constexpr int kCdBlock = 256;

// A block takes P vectors per lane, kCdBlock apart (P lanes share a group, so
// each makes the bits of one), all loaded before the ten rounds.  Bound by HBM: f32
// [16384, 4096] 85.0 us, 6.3 TB/s (the library's copy 89); f64 [16384, 4096] 178, 6.0 TB/s.
template <typename T>
__global__ __launch_bounds__(kCdBlock) void k_counter_dropout(const T *x, T *y, int64_t n, DropArgs a)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, P = kGroupLanes<T>;
    const DropKey key(a);
    const T scale = T(a.scale);
    const int lane = threadIdx.x;
    const int64_t nv = n / VN, tile = int64_t(kCdBlock) * P;
    const U *xv = reinterpret_cast<const U *>(x);
    U *yv = reinterpret_cast<U *>(y);
    for (int64_t base = int64_t(blockIdx.x) * tile; base < nv; base += int64_t(gridDim.x) * tile) {
        const int64_t q = base + lane;
        V v[P];
#pragma unroll
        for (int k = 0; k < P; k++)
            if (q + k * kCdBlock < nv) v[k] = __builtin_nontemporal_load(xv + q + k * kCdBlock);
        const uint32_t own = keep_mask(uint64_t(q + int64_t(lane & (P - 1)) * kCdBlock) / P, key);
        uint32_t m[P];
        m[0] = mask_of<T, 0>(own, lane);
        m[1] = mask_of<T, 1>(own, lane);
        if constexpr (P == 4) {
            m[2] = mask_of<T, 2>(own, lane);
            m[3] = mask_of<T, 3>(own, lane);
        }
#pragma unroll
        for (int k = 0; k < P; k++)
            if (q + k * kCdBlock < nv) {
                V o;
#pragma unroll
                for (int j = 0; j < VN; j++) o[j] = dropped<T>(v[k][j], scale, m[k], (j >> 1) + 16 * (j & 1));
                __builtin_nontemporal_store(o, yv + q + k * kCdBlock);
            }
    }
    // the values past the vectors
    if (blockIdx.x == 0 && nv * VN + lane < n) {
        const int64_t i = nv * VN + lane;
        y[i] = dropped<T>(x[i], scale, keep_in_order(keep_mask(uint64_t(i) / 8, key)), int(i % 8));
    }
}

template <typename T>
static int launch_counter_dropout(const T *x, T *y, int64_t n, const DropArgs &a)
{
    int64_t g = ceil_div(n / Vec16<T>::n, int64_t(kCdBlock) * kGroupLanes<T>);
    g = g < 1 ? 1 : (g < kMaxGridBlocks ? g : kMaxGridBlocks);
    NH_LAUNCH((k_counter_dropout<T>), dim3(unsigned(g)), dim3(kCdBlock), 0, stream(), x, y, n, a);
    return check_launch();
}

static int counter_dropout_api(NeuralTensor *out, const NeuralTensor *in, double p, const NeuralDropoutKey *key)
{
    NH_TRY(ensure_init());
    if (!out || !in) return set_error(NEURAL_ERR_NULL_POINTER);
    NH_TRY(check_tensor(in));
    NH_TRY(check_tensor(out));
    if (in->dtype != out->dtype) return set_error(NEURAL_ERR_DTYPE_MISMATCH);
    const int64_t n = numel(in);
    if (numel(out) != n) return set_error(NEURAL_ERR_SHAPE_MISMATCH);
    if (!is_contiguous(in) || !is_contiguous(out)) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    if (tensors_may_overlap(out, in) && out->data != in->data && out->dev != in->dev)
        return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    DropArgs a;
    NH_TRY(drop_args(p, key, a));
    if (n == 0) return set_error(NEURAL_OK);
    const void *src = nullptr;
    void *dst = nullptr;
    NH_TRY(dev_read(in, &src));
    NH_TRY(dev_write(out, &dst, true));
    if (in->dtype == NEURAL_DTYPE_FLOAT32)
        NH_TRY(launch_counter_dropout(static_cast<const float *>(src), static_cast<float *>(dst), n, a));
    else
        NH_TRY(launch_counter_dropout(static_cast<const double *>(src), static_cast<double *>(dst), n, a));
    NH_TRY(dev_written(out));
    return set_error(NEURAL_OK);
}

}  // namespace nh

extern "C" {

int neural_counter_dropout_forward(NeuralTensor *out, const NeuralTensor *in, double p, const NeuralDropoutKey *key)
{
    return nh::counter_dropout_api(out, in, p, key);
}

int neural_counter_dropout_backward(NeuralTensor *grad_in, const NeuralTensor *grad_out, double p,
                                    const NeuralDropoutKey *key)
{
    return nh::counter_dropout_api(grad_in, grad_out, p, key);
}

}  // extern "C"
