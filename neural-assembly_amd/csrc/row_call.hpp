// row_call.hpp -- what the entry points that work on rows of tensors share: checks of
// their arguments, and device memory for the partial results of one call.
#pragma once

#include <initializer_list>

#include "common.hpp"

namespace nh {

// A call's tensors, checked before anything runs: rows of the last dimension
// of `like`, in its type.  Optional tensors may be null.
struct RowCall {
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
inline int check_apart(std::initializer_list<NeuralTensor *> outs, std::initializer_list<const NeuralTensor *> ins,
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
int read_t(const NeuralTensor *t, const T *&p)
{
    const void *v = nullptr;
    if (t) NH_TRY(dev_read(t, &v));
    p = static_cast<const T *>(v);
    return NEURAL_OK;
}
template <typename T>
int write_t(NeuralTensor *t, T *&p)
{
    void *v = nullptr;
    if (t) NH_TRY(dev_write(t, &v, true));
    p = static_cast<T *>(v);
    return NEURAL_OK;
}
inline int written(std::initializer_list<NeuralTensor *> outs)
{
    for (NeuralTensor *t : outs)
        if (t) NH_TRY(dev_written(t));
    return set_error(NEURAL_OK);
}

// A call's buffer that is no tensor, in host or device memory.  Host memory is copied now, which
// a captured call cannot do again when it is replayed: it is refused before anything is recorded.
inline int open_raw(Staged &s, const void *p, size_t bytes, bool upload)
{
    if (!is_device_ptr(p) && stream_recording()) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    return s.open(p, bytes, upload);
}

// Device memory for the partials of one call.  A call that is being captured
// has the graph's (which may be replayed whenever, beside any other); otherwise
// the block returns to the cache once the launches that use it are enqueued.
struct Partials {
    void *p = nullptr;
    bool keep = false;
    int open(size_t bytes)
    {
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        if (const hipError_t e = hipStreamIsCapturing(stream(), &status)) {  // nothing is launched then
            (void)hipGetLastError();
            return hip_fail(e);
        }
        keep = status != hipStreamCaptureStatusNone;
        if (keep) return graph_alloc(bytes, &p);
        p = dev_alloc(bytes);
        return p ? NEURAL_OK : set_error(NEURAL_ERR_OUT_OF_MEMORY);
    }
    ~Partials()
    {
        if (p && !keep) dev_free(p);
    }
};

}  // namespace nh
