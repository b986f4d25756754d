// philox.hpp -- the counter-based random numbers of the dropout whose mask is
// never stored: any element's draw from its index, a key and an offset alone.
//
// Generator: Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", 2011): ten rounds of
//   (c0, c1, c2, c3) <- (hi(M1 c2) ^ c1 ^ k0, lo(M1 c2), hi(M0 c0) ^ c3 ^ k1, lo(M0 c0))
// with the key raised by (W0, W1) after each.  The key is the 64-bit seed, the
// counter a 64-bit block number and the 64-bit offset.
//
// Element i of the flat tensor is place e = i % 8 of group g = i / 8.  Half e
// (16 bits, low half of a word first) of block 2 g is the upper and of block
// 2 g + 1 the lower half of its 32-bit draw r; it is dropped where r < thr =
// round(p 2^32).  The upper half alone decides unless it equals thr >> 16, so
// the second block is made only by lanes that hold such an element (one in 8192
// groups): eight draws of 32 bits for the ten rounds of one block.  (Both blocks always:
// f32 [4096, 1024], which the caches hold, 8.0 us instead of 7.2; [16384, 4096] the same
// 85, bound by HBM with vector issue in 11% of the cycles.)
#pragma once

#include "common.hpp"

namespace nh {

// A call's dropout: how to draw and what a kept element is multiplied by.
struct DropArgs {
    uint64_t seed, offset;
    const uint64_t *dev;  // {seed, offset} in device memory instead, or null
    uint32_t t, tlow;     // thr >> 16 (up to 65536: p = 1) and its low 16 bits
    double scale;         // 1 / (1 - p)
};

// The same with the key's words in registers, made once per kernel.
struct DropKey {
    uint32_t k0, k1, o0, o1, t, tlow;
    NH_DEV explicit DropKey(const DropArgs &a) : t(a.t), tlow(a.tlow)
    {
        const uint64_t s = a.dev ? a.dev[0] : a.seed, o = a.dev ? a.dev[1] : a.offset;
        k0 = uint32_t(s);
        k1 = uint32_t(s >> 32);
        o0 = uint32_t(o);
        o1 = uint32_t(o >> 32);
    }
};

NH_DEV uint4 philox(uint64_t block, const DropKey &d)
{
    uint32_t c0 = uint32_t(block), c1 = uint32_t(block >> 32), c2 = d.o0, c3 = d.o1, k0 = d.k0, k1 = d.k1;
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const uint64_t p0 = uint64_t(0xD2511F53u) * c0, p1 = uint64_t(0xCD9E8D57u) * c2;
        c0 = uint32_t(p1 >> 32) ^ c1 ^ k0;
        c1 = uint32_t(p1);
        c2 = uint32_t(p0 >> 32) ^ c3 ^ k1;
        c3 = uint32_t(p0);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
NH_DEV u16x2 as_u16x2(uint32_t v) { return __builtin_bit_cast(u16x2, v); }
NH_DEV uint32_t as_u32(u16x2 v) { return __builtin_bit_cast(uint32_t, v); }

// The keep bits of group g: element e at bit e / 2 + 16 (e % 2), that is word by
// word as packed 16-bit arithmetic leaves them (a saturated difference and a
// minimum per word instead of a comparison per element).
NH_DEV uint32_t keep_mask(uint64_t g, const DropKey &d)
{
    const uint4 w4 = philox(2 * g, d);
    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
    const u16x2 one = {1, 1};
    uint32_t m = 0;
    if (d.t > 0xFFFFu) return 0;  // p = 1: uniform
    const u16x2 tt = {uint16_t(d.t), uint16_t(d.t)};
    if (d.tlow == 0) {  // uniform: kept where the upper half >= t, no lower half needed
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const u16x2 below = __builtin_elementwise_sub_sat(tt, as_u16x2(w[q]));
            m |= as_u32(__builtin_elementwise_min(below, one)) << q;
        }
        return m ^ 0x000F000Fu;
    }
    u16x2 near = {0xFFFF, 0xFFFF};
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const u16x2 above = __builtin_elementwise_sub_sat(as_u16x2(w[q]), tt);
        m |= as_u32(__builtin_elementwise_min(above, one)) << q;
        near = __builtin_elementwise_min(near, as_u16x2(w[q] ^ as_u32(tt)));
    }
    if (near[0] == 0 || near[1] == 0) {  // rare
        const uint4 v4 = philox(2 * g + 1, d);
        const uint32_t v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if ((w[q] & 0xFFFFu) == d.t && (v[q] & 0xFFFFu) >= d.tlow) m |= 1u << q;
            if ((w[q] >> 16) == d.t && (v[q] >> 16) >= d.tlow) m |= 0x10000u << q;
        }
    }
    return m;
}

// keep_mask's bits in the order of the elements, bits 0 to 7.
NH_DEV uint32_t keep_in_order(uint32_t m)
{
    const auto spread = [](uint32_t v) {  // bits 0..3 to 0, 2, 4, 6
        v = (v | (v << 2)) & 0x33u;
        return (v | (v << 1)) & 0x55u;
    };
    return spread(m & 0xFu) | (spread((m >> 16) & 0xFu) << 1);
}

// kept ? x * scale : +0 for the element whose keep bit is bit b of m: the
// product's bits masked, so that what x holds (NaN, infinity) does not matter
// where it is dropped.
template <typename T>
NH_DEV T dropped(T x, T scale, uint32_t m, int b)
{
    const T v = x * scale;
    const int32_t keep = int32_t(m << (31 - b)) >> 31;
    if constexpr (sizeof(T) == 4) {
        return __int_as_float(__float_as_int(v) & keep);
    } else {
        return __longlong_as_double(__double_as_longlong(v) & (long long)keep);
    }
}

// Lanes that hold the 16-byte vectors of one group side by side (2 for f32, 4
// for f64) make one group's bits each, for their vectors k = 0, 1, ... in turn,
// and read each other's: mask_of<T, k % P>(own bits) are those of vector k,
// shifted so that element j of the vector is at bit j / 2 + 16 (j % 2).
template <typename T> constexpr int kGroupLanes = 8 / Vec16<T>::n;
template <typename T, int K>
NH_DEV uint32_t mask_of(uint32_t own, int lane)
{
    static_assert(K < kGroupLanes<T>, "");
    if constexpr (sizeof(T) == 4) {
        constexpr int ctrl = K | (K << 2) | ((2 + K) << 4) | ((2 + K) << 6);
        return uint32_t(dpp_i<ctrl>(int(own))) >> (2 * (lane & 1));
    } else {
        constexpr int ctrl = K | (K << 2) | (K << 4) | (K << 6);
        return uint32_t(dpp_i<ctrl>(int(own))) >> (lane & 3);
    }
}

// Argument checks and the call's DropArgs: p in [0, 1]; key: host or device
// memory, two 64-bit words.
int drop_args(double p, const NeuralDropoutKey *key, DropArgs &a);

}  // namespace nh
