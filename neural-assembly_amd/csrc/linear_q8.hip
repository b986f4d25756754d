// linear_q8.hip -- the product of rows in 8 bits with 8-bit weights by output channel:
//   out[m, n] = act(scale[m] wscale[n] sum_k A[m, k] W[n, k] + bias[n]) + residual[m, n]
// The sum is exact in int32 (k <= 131071: |sum| <= k 2^14 < 2^31).  Its scaling and the bias
// are in double and rounded once to the dtype; the activation works on that value as the
// elementwise activations do, and the residual is added to its result: two more roundings in
// f32, each half a unit of values that the f32 elementwise calls would leave as well.
#include <cmath>
#include <type_traits>

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
    bool cut;  // k ends inside a unit of 16 bytes of A's rows, and other bytes follow it
};

// The activation of N values, by neural_bias_add_act's functors: the branch is taken once.
template <typename T, int N>
NH_DEV void act_all(T (&z)[N], int act, double alpha)
{
    const auto each = [&](auto f) {
#pragma unroll
        for (int e = 0; e < N; e++) z[e] = f(z[e]);
    };
    constexpr bool F32 = sizeof(T) == 4;
    switch (act) {
    case NEURAL_ACT_NONE: break;
    case NEURAL_ACT_RELU: each(FnReluAct{}); break;
    case NEURAL_ACT_SIGMOID: each(ActFn<ASigmoid>{}); break;
    case NEURAL_ACT_TANH: each(std::conditional_t<F32, TanhF32Fn, ActFn<ATanh>>{}); break;
    case NEURAL_ACT_GELU: each(std::conditional_t<F32, HeadTailFn<GeluF32>, ActFn<AGelu>>{}); break;
    case NEURAL_ACT_LEAKY_RELU: each(ActFn<ALeaky>{ALeaky{alpha}}); break;
    case NEURAL_ACT_ELU:
        if constexpr (F32) each(HeadTailFn<EluF32>{EluF32{alpha}});
        else each(ActFn<AElu>{AElu{alpha}});
        break;
    case NEURAL_ACT_SELU: each(std::conditional_t<F32, HeadTailFn<SeluF32>, ActFn<ASelu>>{}); break;
    case NEURAL_ACT_SWISH: each(std::conditional_t<F32, HeadTailFn<SwishF32>, ActFn<ASwish>>{}); break;
    case NEURAL_ACT_MISH: each(std::conditional_t<F32, HeadTailFn<MishF32>, ActFn<AMish>>{}); break;
    case NEURAL_ACT_HARDSWISH: each(std::conditional_t<F32, HardswishF32Fn, ActFn<AHardswish>>{}); break;
    case NEURAL_ACT_SOFTPLUS: each(std::conditional_t<F32, HeadTailFn<SoftplusF32>, ActFn<ASoftplus>>{}); break;
    default: each(ActFn<AHardtanh>{}); break;
    }
}

// scale * sum + bias, rounded to the dtype.
template <typename T>
NH_DEV T lin_value(int acc, T sa, T sw, T bias)
{
    return T(double(acc) * (double(sa) * double(sw)) + double(bias));
}

typedef int i32x16 __attribute__((ext_vector_type(16)));

// ---- operands --------------------------------------------------------------------------------

constexpr int64_t kLinMaxLd = int64_t(1) << 22;  // 256 rows of it stay in a 32-bit offset

// Rows of codes copied to rows of `ldd` bytes (a multiple of 16) at an aligned address, the bytes
// past k zero.  A wave takes 64 units of 16 bytes of a row.
struct LinPad {
    const int8_t *src;
    int8_t *dst;
    int64_t ld, rows;  // rows 0: nothing to copy
};
__global__ __launch_bounds__(256) void k_lin_pad(LinPad a, LinPad w, int ldd, int k)
{
    typedef int W __attribute__((ext_vector_type(4), aligned(1)));
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t parts = (ldd / 16 + 63) / 64;
    const int64_t first = a.rows * parts, end = first + w.rows * parts;
    for (int64_t t0 = int64_t(blockIdx.x) * 4 + wave; t0 < end; t0 += int64_t(gridDim.x) * 4) {
        const bool of_a = t0 < first;
        const LinPad &p = of_a ? a : w;
        const uint64_t t = t0 - (of_a ? 0 : first);
        const int64_t r = t >> 32 ? t / parts : uint32_t(t) / parts;
        const int at = 16 * (64 * int(t - r * parts) + lane);
        if (at >= ldd) continue;
        const int8_t *src = p.src + r * p.ld + at;
        i32x4 v;
        if (at + 16 <= k) {
            v = *reinterpret_cast<const W *>(src);
        } else {
            int8_t b[16];
#pragma unroll
            for (int q = 0; q < 16; q++) b[q] = at + q < k ? src[q] : int8_t(0);
            __builtin_memcpy(&v, b, 16);
        }
        *reinterpret_cast<i32x4 *>(p.dst + r * ldd + at) = v;
    }
}

// 16 codes of a row from place k (a multiple of 16) on, zeros past the row's end: what is loaded, and
// what that makes.  A row at a multiple of 4 bytes is loaded as it lies.  Of others (BYTES) the
// words that its bytes lie in are loaded, and shifted: loads of 16 bytes from odd addresses take
// several times as long (16 x 4097 -> 4096 18.6 us, by words 10.7).  No word is loaded of which
// no byte is the row's.
template <bool BYTES>
struct LinUnit {
    i32x4 v;
    int last, shift;  // BYTES: the fifth word, and where in the first one the row's bytes begin
    NH_DEV void load(const int8_t *row, int64_t k, int64_t end)
    {
        typedef int W __attribute__((ext_vector_type(4), aligned(4)));
        shift = BYTES ? int(reinterpret_cast<uintptr_t>(row) & 3) : 0;
        v = i32x4{0, 0, 0, 0};
        last = 0;
        if (k + 16 <= end) {
            const int *p = reinterpret_cast<const int *>(row + k - shift);
            v = *reinterpret_cast<const W *>(p);
            if constexpr (BYTES) last = p[shift ? 4 : 3];
        } else if (k < end) {
            int8_t b[16];
#pragma unroll
            for (int q = 0; q < 16; q++) b[q] = k + q < end ? row[k + q] : int8_t(0);
            __builtin_memcpy(&v, b, 16);
            shift = 0;
        }
    }
    NH_DEV i32x4 codes() const
    {
        if constexpr (!BYTES) return v;
        i32x4 r;
#pragma unroll
        for (int q = 0; q < 4; q++)
            r[q] = int(__builtin_amdgcn_alignbyte(uint32_t(q < 3 ? v[q < 3 ? q + 1 : 3] : last), uint32_t(v[q]), shift));
        return r;
    }
};

// What lanes fetch in the place of units past the rows' end.
__device__ const int g_lin_zero[4] = {0, 0, 0, 0};

// 16 bytes per lane from memory straight into LDS: lane l's to `lds` + 16 l (lds: the same for the
// wave, in bytes).  Two forms of the address: a uniform base and 32 bits per lane, or 64 bits.
// The counter that the compiler keeps of loads in flight does not know these; the waits are
// written out where their data is read.
NH_DEV void lds_load(uint32_t lds, uint32_t at, const int8_t *base)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(at), "s"(base) : "memory");
}
NH_DEV void lds_load(uint32_t lds, const void *p)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(p) : "memory");
}
// At most `N` of this wave's loads still in flight and its LDS reads done; then the block's.
template <int N>
NH_DEV void wait_and_meet()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// ---- the product by matrix instructions -------------------------------------------------------

// WM x WN waves, each TM x TN tiles of 32 x 32 results; slices of 16 KU codes of the block's rows
// of A and W pass through ST buffers in LDS.
template <int WM_, int WN_, int TM_, int TN_, int KU_, int ST_, int PER_SIMD_>
struct LinShape {
    static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, KU = KU_, ST = ST_, PER_SIMD = PER_SIMD_;
    static constexpr int NW = WM * WN, NT = 64 * NW, BM = 32 * WM * TM, BN = 32 * WN * TN;
    static constexpr int kSlice = 16 * KU, kStage = (BM + BN) * kSlice;  // bytes of a row, of a buffer
    static constexpr int kRows = 64 / KU, kLoads = (BM + BN) / kRows / NW;  // rows a load (1 KB), loads per wave
    static constexpr int kOut = 32 * TN + 4;                             // the epilogue's rows of a wave
    static_assert(BM % (kRows * NW) == 0 && BN % (kRows * NW) == 0, "whole loads per wave");
    static constexpr int kLoadsA = BM / kRows / NW;
    // (of larger tiles the registers for it would spill; 256 x 256 as it is has 16 bytes of scratch a lane)
    static constexpr bool kCut = TM * TN == 1;
};

// Tile of block `h` of nbm x nbn: the hardware deals blocks to the 8 XCDs in turn, each with its own
// L2, so each XCD gets consecutive numbers, and those go through groups of G rows of tiles,
// column by column, so that the blocks of an XCD share few panels of A and W.
NH_DEV void lin_tile(int64_t h, int64_t nbm, int64_t nbn, int64_t &bm, int64_t &bn)
{
    constexpr int64_t G = 8;
    const int64_t nb = nbm * nbn, x = h & 7, q = nb >> 3, rest = nb & 7;
    const int64_t L = x * q + (x < rest ? x : rest) + (h >> 3);
    const int64_t gsz = G * nbn, g = L / gsz, r = L - g * gsz, first = g * G;
    const int64_t rows = nbm - first < G ? nbm - first : G;
    bm = first + r % rows;
    bn = r / rows;
}

// Where few tiles meet a long depth, LIN_PART blocks sum a part of it each and leave their
// registers, and LIN_JOIN blocks add those up and end as LIN_WHOLE ones do.
enum { LIN_WHOLE = 0, LIN_PART = 1, LIN_JOIN = 2 };

// (A's rows are the second operand: a lane's results are of one row of A and, four at a time,
// consecutive columns.)
// What bounds it, at 8192 x 4096 -> 16384 on 256 x 256 tiles (541 us, 2.03 POP/s): of a tile's 124
// thousand cycles (64 us) 101 are the main loop's, in which the matrix units are busy 65% of the time;
// then all CUs store a tile at once, at the memory's rate, with the scaling beside it.  The cycles are
// the same for codes of zeros, at 2.38 GHz and 456 us: with real ones the power leaves 1.95 GHz.  gelu
// adds 6 us, in vector issue.  The stores straight from the registers, 32 bytes of a row at a time,
// took 818 us in all.
template <typename T, typename S, int MODE>
__global__ __launch_bounds__(S::NT, S::PER_SIMD) void k_lin_mfma(LinArgs<T> g, int64_t nbm, int64_t nbn, int64_t b_base,
                                                                  i32x4 *parts, int splits)
{
    constexpr int TM = S::TM, TN = S::TN, ST = S::ST, KU = S::KU, BM = S::BM, BN = S::BN, C = KU / 2;
    static_assert(S::NW * 32 * S::kOut * int(sizeof(T)) <= ST * S::kStage, "the epilogue's rows fit the buffers");
    __shared__ __attribute__((aligned(1024))) int8_t smem[ST * S::kStage];
    __shared__ T par_a[BM], par_w[BN], par_b[BN];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int64_t bm, bn;
    const int split = MODE == LIN_PART ? int(blockIdx.x) % splits : 0;
    const int64_t tile = b_base + (MODE == LIN_PART ? int(blockIdx.x) / splits : int(blockIdx.x));
    lin_tile(tile, nbm, nbn, bm, bn);
    const int64_t m0 = bm * BM, n0 = bn * BN;
    const int wr = 32 * TM * (w / S::WN), wc = 32 * TN * (w % S::WN);
    const int frow = lane & 31, hi = lane >> 5;
    const auto scales = [&] {
        for (int i = threadIdx.x; i < BM; i += S::NT) par_a[i] = m0 + i < g.m ? g.sa[m0 + i] : T(0);
        for (int i = threadIdx.x; i < BN; i += S::NT) {
            par_w[i] = n0 + i < g.n ? g.sw[n0 + i] : T(0);
            par_b[i] = g.bias && n0 + i < g.n ? g.bias[n0 + i] : T(0);
        }
    };
    i32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = i32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    // the block's registers of a part: 16 bytes a lane side by side
    const auto at_part = [&](int p, int q) {
        return parts + (((tile - b_base) * splits + p) * S::NW + w) * int64_t(TM * TN * 4 * 64) + q * 64 + lane;
    };
    if constexpr (MODE == LIN_JOIN) {
        scales();
#pragma unroll 1
        for (int p = 0; p < splits; p++)
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const i32x4 c = *at_part(p, (i * TN + j) * 4 + v);
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[i][j][4 * v + e] += c[e];
                    }
        __syncthreads();
    } else {
        // LDS rows of KU units of 16 bytes; unit u of row r lies at u ^ swz(r), so that the sixteen
        // lanes of a 16-byte read that go at once cover the 64 banks once.  A load puts lane l's
        // unit at place l % KU of row l / KU: it fetches the unit that belongs there.
        const auto swz = [](int r) { return KU == 4 ? r >> 2 & 3 : r >> 1 & 7; };
        const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) int8_t *)smem));
        uint32_t at[S::kLoads];
        int unit[S::kLoads];
#pragma unroll
        for (int q = 0; q < S::kLoads; q++) {
            const bool of_a = q < S::kLoadsA;
            const int r = (w + (of_a ? q : q - S::kLoadsA) * S::NW) * S::kRows + lane / KU;
            const int64_t last = of_a ? g.m - 1 - m0 : g.n - 1 - n0;
            unit[q] = (lane % KU) ^ swz(r);
            at[q] = uint32_t((r < last ? r : last) * (of_a ? g.lda : g.ldw) + 16 * unit[q]);
        }
        const int8_t *pa = g.a + m0 * g.lda, *pw = g.w + n0 * g.ldw;
        const int all = int((g.k + S::kSlice - 1) / S::kSlice), whole = int(g.k / S::kSlice), units = int((g.k + 15) / 16);
        const int begin = MODE == LIN_PART ? all * split / splits : 0;
        const int steps = MODE == LIN_PART ? all * (split + 1) / splits : all;
        // past the end: a slice again, so that the count of loads stays
        const int past = S::kCut && steps - begin > 1 ? steps - 2 : steps - 1;
        const auto issue = [&](int s, int buf) {
            s = s < steps ? s : past;
            const uint32_t lds = lds0 + buf * S::kStage;
            const int8_t *sa = pa + int64_t(s) * S::kSlice, *sw = pw + int64_t(s) * S::kSlice;
            if (s < whole) {
#pragma unroll
                for (int q = 0; q < S::kLoads; q++) lds_load(lds + 1024 * (w + q * S::NW), at[q], q < S::kLoadsA ? sa : sw);
                return;
            }
            // Where k ends inside a unit of A's rows in place, they go through registers, which
            // leave out what lies behind it (W's is then multiplied by zeros).  All loads before
            // have then ended.
            const bool inside = S::kCut && g.cut;
            if (inside) {
#pragma unroll
                for (int q = 0; q < S::kLoadsA; q++) {
                    LinUnit<false> u;
                    u.load(sa + at[q] - 16 * unit[q], 16 * unit[q], g.k - int64_t(s) * S::kSlice);
                    *reinterpret_cast<i32x4 *>(smem + buf * S::kStage + 1024 * (w + q * S::NW) + 16 * lane) = u.codes();
                }
                asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
            }
#pragma unroll
            for (int q = 0; q < S::kLoads; q++) {
                if (inside && q < S::kLoadsA) continue;
                const int8_t *p = (q < S::kLoadsA ? sa : sw) + at[q];
                lds_load(lds + 1024 * (w + q * S::NW),
                         KU * s + unit[q] < units ? static_cast<const void *>(p) : g_lin_zero);
            }
        };
        const int fsw = swz(frow);
        i32x4 fa[2][TM], fw[2][TN];
        const auto read = [&](int buf, int c) {
            const int8_t *p = smem + buf * S::kStage + frow * S::kSlice + (((2 * c + hi) ^ fsw) * 16);
#pragma unroll
            for (int i = 0; i < TM; i++) fa[c & 1][i] = *reinterpret_cast<const i32x4 *>(p + (wr + 32 * i) * S::kSlice);
#pragma unroll
            for (int j = 0; j < TN; j++) fw[c & 1][j] = *reinterpret_cast<const i32x4 *>(p + (BM + wc + 32 * j) * S::kSlice);
        };
        const auto multiply = [&](int c) {
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[c & 1][j], fa[c & 1][i], acc[i][j], 0, 0, 0);
        };
#pragma unroll
        for (int s = 0; s < ST; s++) issue(begin + s, s);
        if constexpr (MODE == LIN_WHOLE) scales();
        wait_and_meet<0>();
        read(0, 0);
        int cur = 0;
        for (int s = begin; s < steps; s++) {
            // Slice s, its first chunk of 32 codes in registers already.
#pragma unroll
            for (int c = 0; c + 1 < C; c++) {
                read(cur, c + 1);
                __builtin_amdgcn_sched_barrier(0);
                multiply(c);
                __builtin_amdgcn_sched_barrier(0);
            }
            // Slice s + 1 is there, and every wave has read all of slice s: its buffer is free.
            wait_and_meet<S::kLoads *(ST - 2)>();
            const int next = cur + 1 == ST ? 0 : cur + 1;
            read(next, 0);
            issue(s + ST, cur);
            __builtin_amdgcn_sched_barrier(0);
            multiply(C - 1);
            __builtin_amdgcn_sched_barrier(0);
            cur = next;
        }
        wait_and_meet<0>();
    }
    if constexpr (MODE == LIN_PART) {
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int v = 0; v < 4; v++)
                    *at_part(split, (i * TN + j) * 4 + v) =
                        i32x4{acc[i][j][4 * v], acc[i][j][4 * v + 1], acc[i][j][4 * v + 2], acc[i][j][4 * v + 3]};
        return;
    }

    // The epilogue: a wave's results go through its own part of LDS, 32 rows at a time, so that a
    // lane has four columns side by side.  Result v of lane l is column 8 (v / 4) + 4 (l / 32) + v %
    // 4, row l % 32 of its tile.  Sums lie there as their bits (f32) or as doubles.
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, Q = 4 / VN, CL = 8 * TN, RPI = 64 / CL, NI = 32 / RPI;  // lanes per row, rows at once
    T *rows = reinterpret_cast<T *>(smem) + w * 32 * S::kOut;
    const int cl = lane % CL, rl = lane / CL;
    const int64_t n = n0 + wc + 4 * cl;
    T sw[4], bias[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        sw[e] = par_w[wc + 4 * cl + e];
        bias[e] = par_b[wc + 4 * cl + e];
    }
    constexpr int UA = TM * TN == 1 ? 4 : TM * TN <= 4 ? 2 : 1;  // rows of a turn, as registers allow
    const bool full = n + 4 <= g.n, act = g.act != NEURAL_ACT_NONE;
    const auto sums = [&](int r, int (&c)[4]) {
        const T *p = rows + r * S::kOut + 4 * cl;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (sizeof(T) == 4) c[e] = __float_as_int(p[e]);
            else c[e] = int(p[e]);
        }
    };
#pragma unroll 1
    for (int i = 0; i < TM; i++) {
        const int64_t mi = m0 + wr + 32 * i;
        V res[NI][Q];
        if (g.res && full) {
#pragma unroll
            for (int u = 0; u < NI; u++)
                if (mi + rl + u * RPI < g.m) {
#pragma unroll
                    for (int q = 0; q < Q; q++)
                        res[u][q] = *(reinterpret_cast<const U *>(g.res + (mi + rl + u * RPI) * g.n + n) + q);
                }
        }
        const auto dump = [&](const i32x16 (&t)[TN]) {
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    T x;
                    if constexpr (sizeof(T) == 4) x = __int_as_float(t[j][v]);
                    else x = double(t[j][v]);
                    rows[frow * S::kOut + 32 * j + 8 * (v / 4) + 4 * hi + v % 4] = x;
                }
        };
        if (i == 0) dump(acc[0]);
        if constexpr (TM > 1) if (i == 1) dump(acc[1]);
        if constexpr (TM > 2) if (i == 2) dump(acc[2]);
        if constexpr (TM > 3) if (i == 3) dump(acc[3]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const auto value = [&](int r, T (&z)[4]) {
            int c[4];
            sums(r, c);
            const T sa = par_a[wr + 32 * i + r];
#pragma unroll
            for (int e = 0; e < 4; e++) z[e] = lin_value<T>(c[e], sa, sw[e], bias[e]);
        };
        const auto store = [&](int64_t m, const T (&z)[4]) {
            const int64_t o = m * g.n + n;
            if (m < g.m && full) {
#pragma unroll
                for (int q = 0; q < Q; q++) {
                    V y;
#pragma unroll
                    for (int e = 0; e < VN; e++) y[e] = z[q * VN + e];
                    __builtin_nontemporal_store(y, reinterpret_cast<U *>(g.out + o) + q);
                }
            } else if (m < g.m) {
                for (int e = 0; e < 4; e++)
                    if (n + e < g.n) g.out[o + e] = z[e];
            }
        };
        if (act) {  // one copy of the activations' code, so a loop
#pragma unroll 1
            for (int r = rl; r < 32; r += UA * RPI) {
                T z[UA][4], zz[4 * UA];
#pragma unroll
                for (int q = 0; q < UA; q++) value(r + q * RPI, z[q]);
#pragma unroll
                for (int q = 0; q < 4 * UA; q++) zz[q] = z[q / 4][q % 4];
                act_all(zz, g.act, g.alpha);
#pragma unroll
                for (int q = 0; q < 4 * UA; q++) z[q / 4][q % 4] = zz[q];
#pragma unroll
                for (int q = 0; q < UA; q++) {
                    if (!g.res) {
                        store(mi + r + q * RPI, z[q]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) rows[(r + q * RPI) * S::kOut + 4 * cl + e] = z[q][e];
                    }
                }
            }
        }
        if (!act || g.res) {
#pragma unroll
            for (int u = 0; u < NI; u++) {
                const int r = rl + u * RPI;
                const int64_t m = mi + r;
                T z[4];
                if (act) {
#pragma unroll
                    for (int e = 0; e < 4; e++) z[e] = rows[r * S::kOut + 4 * cl + e];
                } else {
                    value(r, z);
                }
                if (g.res) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        T y = res[u][e / VN][e % VN];
                        if (!full) y = m < g.m && n + e < g.n ? g.res[m * g.n + n + e] : T(0);
                        z[e] = z[e] + y;
                    }
                }
                store(m, z);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- few rows ------------------------------------------------------------------------------------

// Up to 16 rows, or groups of 16: the weights are read once a group and are what the time goes to.  A
// block takes 16 output channels; its 8 waves share out the depth, each with UN slices of 64 codes in flight from memory
// to registers, and add up in LDS.  Rows and weights may lie at any address.  1 x 4096 -> 4096 5.3
// us (a launch alone 3.5; 64 x 64 tiles 11.2), 16 rows 6.6, 1 x 16384 -> 4096 12.6 (5.3 TB/s; 31).
template <typename T, bool BYTES>
__global__ __launch_bounds__(512) void k_lin_few(LinArgs<T> g, int64_t b_base)
{
    constexpr int W = 8, UN = 8;
    __shared__ i32x4 part[W][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n0 = (b_base + int64_t(blockIdx.x)) * 16;
    const int r = lane & 15, u = lane >> 4, m = 16 * int(blockIdx.y) + r;
    const int8_t *pw = g.w + (n0 + r < g.n ? n0 + r : g.n - 1) * g.ldw, *pa = g.a + (m < g.m ? m : g.m - 1) * g.lda;
    i32x4 acc{0, 0, 0, 0};
    const int64_t slices = (g.k + 63) / 64, s0 = slices * w / W, s1 = slices * (w + 1) / W;
    for (int64_t s = s0; s < s1; s += UN) {
        LinUnit<BYTES> vw[UN], va[UN];
        const bool inside = (s + UN) * 64 <= g.k && s + UN <= s1;  // uniform
#pragma unroll
        for (int q = 0; q < UN; q++) {
            const int64_t k = (s + q) * 64 + 16 * u, end = inside ? INT64_MAX : s + q < s1 ? g.k : 0;
            vw[q].load(pw, k, end);
            va[q].load(pa, k, end);
        }
#pragma unroll
        for (int q = 0; q < UN; q++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(vw[q].codes(), va[q].codes(), acc, 0, 0, 0);
    }
    part[w][lane] = acc;
    __syncthreads();
    // result v of lane l: row l % 16 of the block's, channel 4 (l / 16) + v
    if (w > 0) return;
#pragma unroll
    for (int q = 1; q < W; q++) acc += part[q][lane];
    const int64_t n = n0 + 4 * u;
    if (m < g.m && n < g.n) {
        const T sa = g.sa[m];
        T z[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
            z[e] = n + e < g.n ? lin_value<T>(acc[e], sa, g.sw[n + e], g.bias ? g.bias[n + e] : T(0)) : T(0);
        act_all(z, g.act, g.alpha);
        const int64_t o = m * g.n + n;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (n + e < g.n) g.out[o + e] = g.res ? z[e] + g.res[o + e] : z[e];
    }
}

// ---- the choice --------------------------------------------------------------------------------

// Parts of the depth for few tiles: as many blocks as two a CU, none under 16 slices (2048 codes),
// and at least 3, as the parts' way through memory and the second launch cost some 4 us: 64 x
// 16384 -> 4096 32 us whole, 20 in 8 parts; 64 x 4096 -> 4096 11.6 whole, 12.4 in 4; 64 x 4096 ->
// 16384 14 whole, 18 in 2.
template <typename S>
static int lin_splits(int64_t tiles, int64_t k)
{
    const int64_t want = int64_t(num_cus()) * 2 / tiles, most = ceil_div(k, S::kSlice) / 16;
    const int64_t n = want < most ? want : most;
    return n < 3 ? 1 : int(n);
}

// Rows that all begin at multiples of 4 bytes.
template <typename T>
static bool lin_words(const LinArgs<T> &g)
{
    return ((reinterpret_cast<uintptr_t>(g.a) | reinterpret_cast<uintptr_t>(g.w) | uintptr_t(g.lda) | uintptr_t(g.ldw)) & 3) == 0;
}

// Rows that go straight to LDS, without a copy.
static bool lin_in_place(const int8_t *p, int64_t ld)
{
    return ((reinterpret_cast<uintptr_t>(p) | uintptr_t(ld)) & 15) == 0 && ld < kLinMaxLd;
}

// The product on shape S: copies of what does not go straight to LDS (through registers, as few
// rows do, 577 x 1001 -> 3001 in f64 took 22 us for 17; by words, three slices ahead, 24), long depths
// in parts where S is SMALL.
template <typename T, typename S, bool SMALL>
static int launch_lin_shape(LinArgs<T> g)
{
    const int64_t nbm = ceil_div(g.m, S::BM), nbn = ceil_div(g.n, S::BN), ldd = (g.k + 63) / 64 * 64;
    g.cut = (g.k & 15) != 0 && lin_in_place(g.a, g.lda);
    const size_t ba = lin_in_place(g.a, g.lda) && (S::kCut || !g.cut) ? 0 : size_t(g.m) * size_t(ldd);
    const size_t bw = lin_in_place(g.w, g.ldw) ? 0 : size_t(g.n) * size_t(ldd);
    const int splits = SMALL ? lin_splits<S>(nbm * nbn, g.k) : 1;
    const size_t bp = splits > 1 ? size_t(nbm * nbn) * size_t(splits) * size_t(S::BM * S::BN * 4) : 0;
    Partials block;  // (one: a captured call's blocks share memory)
    if (bp + ba + bw) NH_TRY(block.open(bp + ba + bw));
    int8_t *mem = static_cast<int8_t *>(block.p);
    i32x4 *parts = reinterpret_cast<i32x4 *>(mem);
    if (ba + bw) {
        const LinPad a{g.a, mem + bp, g.lda, ba ? g.m : 0}, w{g.w, mem + bp + ba, g.ldw, bw ? g.n : 0};
        const int64_t need = ceil_div((a.rows + w.rows) * ceil_div(ldd, 1024), 4);
        NH_LAUNCH(k_lin_pad, dim3(unsigned(need < kMaxGridBlocks ? need : kMaxGridBlocks)), dim3(256), 0, stream(), a, w,
                  int(ldd), int(g.k));
        if (ba) {
            g.a = a.dst;
            g.lda = ldd;
        }
        if (bw) {
            g.w = w.dst;
            g.ldw = ldd;
        }
    }
    if constexpr (SMALL) {
        if (splits > 1) {  // (few tiles: one launch each)
            const unsigned tiles = unsigned(nbm * nbn);
            NH_LAUNCH((k_lin_mfma<T, S, LIN_PART>), dim3(tiles * unsigned(splits)), dim3(S::NT), 0, stream(), g, nbm, nbn,
                      int64_t(0), parts, splits);
            NH_LAUNCH((k_lin_mfma<T, S, LIN_JOIN>), dim3(tiles), dim3(S::NT), 0, stream(), g, nbm, nbn, int64_t(0), parts,
                      splits);
            return check_launch();
        }
    }
    for_row_launches(nbm * nbn, 1, S::NT, [&](unsigned blocks, int64_t base) {
        NH_LAUNCH((k_lin_mfma<T, S, LIN_WHOLE>), dim3(blocks), dim3(S::NT), 0, stream(), g, nbm, nbn, base, parts, 1);
    });
    return check_launch();
}

// By the cost of each shape, in us for a depth of 4096 as measured here (no other depth was; in a short
// one the tiles' ends and stores weigh more): the most tiles that fall to one CU at what one costs it
// alone, or all tiles at what they cost when every CU works.  A small
// tile answers sooner where there are few of them, a large one reads less for each product:
// 300 x 4096 -> 4096 15 us on 64 x 64 tiles, 25 on 128 x 128, 54 on 256 x 256; 1024 rows 33, 27,
// 54; 2048 rows 58, 42, 55 and 40 on 128 x 256; 4096 rows 110, 93, 71 on 256 x 256.
struct LinCost {
    double per_cu, fixed, all;  // all: per 64 x 64 of results
};
template <typename S>
static double lin_cost(int64_t m, int64_t n, const LinCost &c)
{
    const int64_t tiles = ceil_div(m, S::BM) * ceil_div(n, S::BN);
    const double alone = c.fixed + c.per_cu * double(ceil_div(tiles, num_cus()));
    const double all = c.all * double(tiles) * double(S::BM * S::BN / 4096) * (256.0 / num_cus());
    return alone > all ? alone : all;
}

template <typename T>
static int launch_linear(const LinArgs<T> &g)
{
    // Up to 16 rows (wider, 64 x 64 tiles stream better what they do not copy: 1 x 4096 -> 16384 15.9
    // us, 13.3 by tiles; 16 rows of 4100 codes -> 16000 22.9 us, 35.5 with a copy of the weights; one of
    // 4097 28.8 and 34.8), and more in groups of 16 where that is still few blocks and spares the copy
    // (64 x 1001 -> 1000 5.8 us, 9.6 with it; 32 x 4097 -> 4096 19.0, 22.7, 64 35.3, 23.3; 64 x 4100 ->
    // 4096 22.0, 23.2; 17 x 16001 -> 1000 24.8, 21.8).
    const int64_t blocks_n = ceil_div(g.n, 16), groups = ceil_div(g.m, 16), cus = num_cus();
    const bool copied = !lin_in_place(g.w, g.ldw);
    if (groups == 1 ? blocks_n <= 2 * cus || copied
                    : copied && g.k <= 8192 && groups * blocks_n <= (lin_words(g) ? 4 : 2) * cus) {
        for_row_launches(blocks_n, 1, 512 * groups, [&](unsigned blocks, int64_t base) {
            const dim3 grid(blocks, unsigned(groups));
            if (lin_words(g)) NH_LAUNCH((k_lin_few<T, false>), grid, dim3(512), 0, stream(), g, base);
            else NH_LAUNCH((k_lin_few<T, true>), grid, dim3(512), 0, stream(), g, base);
        });
        return check_launch();
    }
    using S64 = LinShape<2, 2, 1, 1, 8, 3, 2>;
    if constexpr (sizeof(T) == 8) {  // (its epilogue takes twice the LDS: two shapes)
        using S128 = LinShape<2, 2, 2, 2, 8, 3, 1>;
        return ceil_div(g.m, 128) * ceil_div(g.n, 128) >= 2 * num_cus() ? launch_lin_shape<T, S128, false>(g)
                                                                        : launch_lin_shape<T, S64, true>(g);
    } else {
        using S128x64 = LinShape<2, 2, 2, 1, 8, 3, 2>;
        using S128 = LinShape<2, 2, 2, 2, 8, 2, 2>;
        using S128x256 = LinShape<2, 4, 2, 2, 8, 3, 2>;
        using S256 = LinShape<2, 4, 4, 2, 8, 2, 2>;
        const double cost[] = {lin_cost<S64>(g.m, g.n, {7.0, 4.0, 0.028}), lin_cost<S128x64>(g.m, g.n, {10.0, 8.0, 0.025}),
                               lin_cost<S128>(g.m, g.n, {17.0, 9.0, 0.0205}),
                               lin_cost<S128x256>(g.m, g.n, {34.0, 5.0, 0.0194}),
                               lin_cost<S256>(g.m, g.n, {50.0, 4.0, 0.0173})};
        int best = 0;
        for (int i = 1; i < 5; i++)
            if (cost[i] < cost[best]) best = i;
        switch (best) {
        case 0: return launch_lin_shape<T, S64, true>(g);
        case 1: return launch_lin_shape<T, S128x64, false>(g);
        case 2: return launch_lin_shape<T, S128, false>(g);
        case 3: return launch_lin_shape<T, S128x256, false>(g);
        default: return launch_lin_shape<T, S256, false>(g);
        }
    }
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
    const size_t a_bytes = size_t(c.rows) * size_t(t.stride), w_bytes = size_t(c.cols) * size_t(t.w_stride);
    if (raw_may_overlap(t.codes, a_bytes, t.out) || raw_may_overlap(t.w_codes, w_bytes, t.out))
        return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    Staged a, w;
    NH_TRY(open_raw(a, t.codes, a_bytes, true));
    NH_TRY(open_raw(w, t.w_codes, w_bytes, true));
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
