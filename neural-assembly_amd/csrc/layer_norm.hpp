// layer_norm.hpp -- what the forward (layer_norm.hip) and the backward pass
// (layer_norm_grad_impl.hpp) of layer norm share: the modes, rounding helpers and the keep bits
// of a row's values.
#pragma once

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

// How a group's vectors of a row are read and written: past the caches (NT, each
// byte is used once), except where one access of a wave leaves parts of 64-byte
// blocks to the next, which then are fetched, and written, twice: f32 [838860, 40] 114 us ->
// 59.5, [335544, 100] 61.0 -> 55.5, [86037, 390] 60.9 -> 54.0 (rows of whole blocks the
// other way, when both were measured: [349525, 96] 49.8, 52.2 through the caches, [83886, 400]
// 47.8, 51.8; now 47.1 and 49.5).
template <typename T, bool PAST>
struct RowStream {
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    NH_DEV static V load(const U *p)
    {
        if constexpr (PAST) return __builtin_nontemporal_load(p);
        else return *p;
    }
    NH_DEV static void store(const V &v, U *p)
    {
        if constexpr (PAST) __builtin_nontemporal_store(v, p);
        else *p = v;
    }
};

// run(std::bool_constant<PAST>) for groups of NT lanes.
template <typename T, int NT, typename R>
auto with_stream(int64_t cols, R run)
{
    if constexpr (NT >= 64) {
        return run(std::true_type{});
    } else {
        if (cols * int64_t(sizeof(T)) % 64 == 0) return run(std::true_type{});
        return run(std::false_type{});
    }
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

// ---- the backward pass's arguments ---------------------------------------------------------

template <typename T>
struct LnGradArgs {
    const T *dy, *h, *gamma, *mean, *rstd, *dh;  // gamma, dh: may be null
    T *dx, *dres;                                // either may be null
    T *part;                                     // [blocks][2][cols] partial sums of dgamma and dbeta, or null
    int64_t rows, cols;
    DropArgs drop;
};

// dgamma, dbeta: may be null.  Defined for both types and all modes.
template <typename T, int MODE>
int launch_ln_grad(const LnGradArgs<T> &a, T *dgamma, T *dbeta);

// ---- rows wider than a group's registers -------------------------------------------------

constexpr int kLnWide = 1024;  // lanes of their blocks

// W values side by side: a 16-byte access at the element's own alignment, or one element.
template <typename T, int W>
struct Pack {
    T v[W];
    NH_DEV static Pack load(const T *p)
    {
        Pack r;
        if constexpr (W == 1) {
            r.v[0] = *p;
        } else {
            const typename VecU<T>::type u = *reinterpret_cast<const typename VecU<T>::type *>(p);
#pragma unroll
            for (int j = 0; j < W; j++) r.v[j] = u[j];
        }
        return r;
    }
    NH_DEV void store(T *p) const
    {
        if constexpr (W == 1) {
            *p = v[0];
        } else {
            typename Vec16<T>::type u;
#pragma unroll
            for (int j = 0; j < W; j++) u[j] = v[j];
            *reinterpret_cast<typename VecU<T>::type *>(p) = u;
        }
    }
};

// The row's columns by a block of kLnWide lanes, four vectors in flight each, then the
// values past the vectors: use(width, first column, load(width, first column)).
template <typename T, typename L, typename F>
NH_DEV void walk_row(int64_t cols, L load, F use)
{
    constexpr int VN = Vec16<T>::n, UN = 4;
    using W = std::integral_constant<int, VN>;
    const int64_t ncv = cols / VN;
    for (int64_t q = threadIdx.x; q < ncv; q += UN * kLnWide) {
        decltype(load(W{}, q)) v[UN];
#pragma unroll
        for (int u = 0; u < UN; u++)
            if (q + u * kLnWide < ncv) v[u] = load(W{}, (q + u * kLnWide) * VN);
#pragma unroll
        for (int u = 0; u < UN; u++)
            if (q + u * kLnWide < ncv) use(W{}, (q + u * kLnWide) * VN, v[u]);
    }
    const int64_t c = ncv * VN + threadIdx.x;
    if (c < cols) use(std::integral_constant<int, 1>{}, c, load(std::integral_constant<int, 1>{}, c));
}

// Keep bits of the W elements from flat index i, element j at bit j.
template <int W>
NH_DEV uint32_t keep_at(int64_t i, const DropKey &key)
{
    const int o = int(i & 7);
    uint32_t m = keep_in_order(keep_mask(uint64_t(i) / 8, key)) >> o;
    if (o + W > 8) m |= keep_in_order(keep_mask(uint64_t(i) / 8 + 1, key)) << (8 - o);
    return m;
}

}  // namespace nh
