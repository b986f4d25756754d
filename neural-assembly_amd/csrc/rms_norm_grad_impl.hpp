// rms_norm_grad_impl.hpp -- the backward pass of RMS norm, joined with the residual stream's
// gradient, compiled for each type by rms_norm_grad_f32.hip and rms_norm_grad_f64.hip:
//   xh = h rstd; w = dy gamma; dx = rstd (w - xh mean_c(w xh)) [rounded, + dh];
//   dgamma = sum_rows dy xh
// in double; dx is rounded once (twice with dh), dgamma once more for what each block leaves.
#pragma once

#include <type_traits>

#include "rms_norm.hpp"
#include "row_call.hpp"

namespace nh {

// A row of any width by a block of kLnWide lanes, in two walks: the row's sum, then dx.  What is
// wider than registers hold is read twice, by the column sums once more: f32 [1638, 40000] 321 us
// (a copy of the tensors once 127).
template <typename T>
__global__ __launch_bounds__(kLnWide) void k_rms_grad_wide(RmsGradArgs<T> a, int64_t r_base)
{
    using G = RowGrp<kLnWide>;
    __shared__ double lds_q[G::kWaves];
    const int64_t r = r_base + blockIdx.x, cols = a.cols, at = r * cols;
    const double rstd = double(a.rstd[r]), inv_c = 1.0 / double(cols);
    const auto load = [&](auto w, int64_t c) {
        constexpr int W = decltype(w)::value;
        struct {
            Pack<T, W> x, dy, g;
        } v;
        v.x = Pack<T, W>::load(a.h + at + c);
        v.dy = Pack<T, W>::load(a.dy + at + c);
#pragma unroll
        for (int j = 0; j < W; j++) v.g.v[j] = T(1);
        if (a.gamma) v.g = Pack<T, W>::load(a.gamma + c);
        return v;
    };
    double q = 0.0;
    walk_row<T>(cols, load, [&](auto w, int64_t, const auto &v) {
#pragma unroll
        for (int j = 0; j < decltype(w)::value; j++)
            q = __builtin_fma(double(v.dy.v[j]) * double(v.g.v[j]), double(v.x.v[j]) * rstd, q);
    });
    const double c2 = G::sum(q, lds_q) * inv_c;
    walk_row<T>(cols, load, [&](auto w, int64_t c, const auto &v) {
        constexpr int W = decltype(w)::value;
        Pack<T, W> o;
#pragma unroll
        for (int j = 0; j < W; j++) {
            const double xh = double(v.x.v[j]) * rstd, wv = double(v.dy.v[j]) * double(v.g.v[j]);
            o.v[j] = T(rstd * __builtin_fma(-xh, c2, wv));
        }
        if (a.dh) {
            const Pack<T, W> d = Pack<T, W>::load(a.dh + at + c);
#pragma unroll
            for (int j = 0; j < W; j++) o.v[j] = o.v[j] + d.v[j];
        }
        o.store(a.dx + at + c);
    });
}

// Column sums by chunks of rows: 64 lanes of VN columns a block, the chunk's rows by 8 waves,
// four in flight each; a chunk leaves one row of partials.  b_base: the launch's first block.
template <typename T>
__global__ __launch_bounds__(512) void k_rms_cols(RmsGradArgs<T> a, int64_t chunk, int64_t b_base)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, W = 8, UN = 4;
    __shared__ double sh[W][VN][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t cols = a.cols, c = ((b_base + int64_t(blockIdx.x)) * 64 + lane) * VN;
    const int64_t r0 = int64_t(blockIdx.y) * chunk, r1 = r0 + chunk < a.rows ? r0 + chunk : a.rows;
    const bool whole = c + VN <= cols;
    double s[VN];
#pragma unroll
    for (int j = 0; j < VN; j++) s[j] = 0.0;
    for (int64_t r = r0 + w; r < r1; r += W * UN) {
        V x[UN], dy[UN];
#pragma unroll
        for (int u = 0; u < UN; u++)
            if (r + u * W < r1) {
                const int64_t at = (r + u * W) * cols + c;
                if (whole) {
                    x[u] = *reinterpret_cast<const U *>(a.h + at);
                    dy[u] = *reinterpret_cast<const U *>(a.dy + at);
                } else {
#pragma unroll
                    for (int j = 0; j < VN; j++) {
                        x[u][j] = c + j < cols ? a.h[at + j] : T(0);
                        dy[u][j] = c + j < cols ? a.dy[at + j] : T(0);
                    }
                }
            }
#pragma unroll
        for (int u = 0; u < UN; u++)
            if (r + u * W < r1) {
                const double rstd = double(a.rstd[r + u * W]);
#pragma unroll
                for (int j = 0; j < VN; j++) s[j] = __builtin_fma(double(dy[u][j]), double(x[u][j]) * rstd, s[j]);
            }
    }
#pragma unroll
    for (int j = 0; j < VN; j++) sh[w][j][lane] = s[j];
    __syncthreads();
    // wave w folds the lanes' columns w (VN <= W)
    if (w < VN && c + w < cols) {
        double t = sh[0][w][lane];
        for (int i = 1; i < W; i++) t += sh[i][w][lane];
        a.part[int64_t(blockIdx.y) * cols + c + w] = T(t);
    }
}

// Column sums of the partials: [n][cols] -> dgamma, 32 columns a block of 1024 lanes.
template <typename T>
__global__ __launch_bounds__(1024) void k_rms_fold(const T *__restrict__ part, int64_t n, int64_t cols,
                                                   T *__restrict__ dgamma, int64_t b_base)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, C = 32, L = C / VN, S = 1024 / L, UN = 4, TPC = 1024 / C;
    __shared__ double sh[S][C + 1];  // (read by columns below: no two lanes on a bank)
    const int vl = threadIdx.x % L, st = threadIdx.x / L;
    const int64_t c0 = (b_base + int64_t(blockIdx.x)) * C, c = c0 + vl * VN;
    double s[VN];
#pragma unroll
    for (int j = 0; j < VN; j++) s[j] = 0.0;
    for (int64_t i = st; i < n; i += S * UN) {
        V v[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const T *p = part + (i + u * S) * cols + c;
            if (i + u * S < n) {
                if (c + VN <= cols) {
                    v[u] = *reinterpret_cast<const U *>(p);
                } else {
#pragma unroll
                    for (int j = 0; j < VN; j++) v[u][j] = c + j < cols ? p[j] : T(0);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < UN; u++)
            if (i + u * S < n) {
#pragma unroll
                for (int j = 0; j < VN; j++) s[j] += double(v[u][j]);
            }
    }
#pragma unroll
    for (int j = 0; j < VN; j++) sh[st][vl * VN + j] = s[j];
    __syncthreads();
    // 32 lanes side by side take a column's streams
    const int e = threadIdx.x / TPC, part_of = threadIdx.x % TPC;
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < S / TPC; i++) t += sh[part_of + i * TPC][e];
    t = RowGrp<TPC>::sum(t, nullptr);
    if (part_of == 0 && c0 + e < cols) dgamma[c0 + e] = T(t);
}

template <typename T>
static void launch_rms_fold(const T *part, int64_t n, int64_t cols, T *dgamma)
{
    for_row_launches(ceil_div(cols, 32), 1, 1024, [&](unsigned g, int64_t base) {
        NH_LAUNCH((k_rms_fold<T>), dim3(g), dim3(1024), 0, stream(), part, n, cols, dgamma, base);
    });
}

// Column sums by k_rms_cols and a fold.
template <typename T>
static int launch_rms_cols(RmsGradArgs<T> a, T *dgamma)
{
    const int64_t gx = ceil_div(a.cols, 64 * Vec16<T>::n);
    int64_t chunks = ceil_div(int64_t(num_cus()) * 2, gx);
    const int64_t most = ceil_div(a.rows, 32);
    chunks = chunks < most ? chunks : most;
    const int64_t chunk = ceil_div(a.rows, chunks);
    chunks = ceil_div(a.rows, chunk);
    Partials part;
    NH_TRY(part.open(size_t(chunks) * size_t(a.cols) * sizeof(T)));
    a.part = static_cast<T *>(part.p);
    for_row_launches(gx, 1, 512, [&](unsigned g, int64_t base) {
        NH_LAUNCH((k_rms_cols<T>), dim3(g, unsigned(chunks)), dim3(512), 0, stream(), a, chunk, base);
    });
    launch_rms_fold(a.part, chunks, a.cols, dgamma);
    return check_launch();
}

// How a group's lanes hold a row of the backward pass, and how many groups a CU holds.  NT
// lanes, VPT vectors each.  The sums of dgamma over the rows are in double in registers up to 8
// vectors; gamma is in registers up to 4 vectors, else in LDS (64 KB at most): a load of it for
// each row would wait for the next row's loads, which are older.  16 vectors: no sums (k_rms_cols
// takes them), gamma from the L2.
template <typename T, int NT, int VPT>
struct RmsGradPlan {
    static constexpr int NB = NT < 256 ? 256 : NT, RPB = NB / NT;
    static constexpr bool kGammaRegs = VPT <= 4, kGammaLds = VPT > 4 && VPT <= 8;
    static constexpr int F = VPT <= 8 ? VPT - 1 : VPT / 2;        // vectors that are whole
    static constexpr int kWaves = VPT >= 3 || NT >= 512 ? 2 : 3;  // per SIMD
    static constexpr int kPerCu = kWaves * 256 / NB;              // resident blocks
};

// Groups of NT lanes walk the rows: each tensor read once, the next row's loads issued before this
// one is worked on, the row's sum by one exchange (LDS slots alternate between rows), and each
// lane's columns of dgamma summed over the rows.  The block's groups fold theirs through LDS
// and the block leaves one row of partials, in the rows' type.  `block` of `blocks`.  Bound by HBM:
// f32 [16384, 4096] 134 us (a copy of as many bytes 130), with dh 175 (175); [65536, 1000] 138 and
// 193 (128, 172); [4096, 16384] 150 and 211 (132, 177).  f64 [8192, 4096] 139 and 181 (131, 175), [32768,
// 1000] 146 and 195 (126, 170); [2048, 16384], gamma's sums by k_rms_cols, 228 and 313 (130, 175).
template <typename T, int NT, int VPT, bool DH, bool SUMS, bool PAST>
NH_DEV void rms_grad_rows(const RmsGradArgs<T> &a, int64_t block, int64_t blocks)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    using G = RowGrp<NT>;
    using S = RowStream<T, PAST>;
    using Plan = RmsGradPlan<T, NT, VPT>;
    constexpr int VN = Vec16<T>::n, RPB = Plan::RPB;
    __shared__ double lds_q[2][G::kWaves];
    __shared__ V lds_gamma[Plan::kGammaLds ? VPT : 1][Plan::kGammaLds ? NT : 1];
    const int lane = threadIdx.x % NT, sub = RPB == 1 ? 0 : threadIdx.x / NT;
    const int64_t cols = a.cols;
    const RowCut<T> cut(cols);
    const auto in_row = [&](int k) { return k < Plan::F || lane + k * NT < cut.ncv; };
    const bool has_t = lane < cut.rem;
    const double inv_c = 1.0 / double(cols);
    V g[Plan::kGammaRegs ? VPT : 1];
    const auto gamma = [&](int k) {
        V v;
#pragma unroll
        for (int j = 0; j < VN; j++) v[j] = T(1);
        if (a.gamma && in_row(k)) v = *(reinterpret_cast<const U *>(a.gamma) + lane + k * NT);
        return v;
    };
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        if constexpr (Plan::kGammaRegs) g[k] = gamma(k);
        else if constexpr (Plan::kGammaLds) lds_gamma[k][lane] = gamma(k);  // a lane's own slots
    }
    const auto gamma_of = [&](int k) {
        if constexpr (Plan::kGammaRegs) return g[k];
        else if constexpr (Plan::kGammaLds) return lds_gamma[k][lane];
        else return gamma(k);
    };
    T gt = T(1);
    if (a.gamma && has_t) gt = a.gamma[cut.sc(lane)];
    double sg[SUMS ? VPT : 1][VN], sgt = 0.0;
    if constexpr (SUMS) {
#pragma unroll
        for (int k = 0; k < VPT; k++)
#pragma unroll
            for (int j = 0; j < VN; j++) sg[k][j] = 0.0;
    }
    struct Row {
        V x[VPT], dy[VPT];
        T xt, dyt, rstd;
    };
    const auto load = [&](Row &w, int64_t r) {
        const int64_t at = r * cols;
        w.rstd = a.rstd[r];  // first, since loads return in order and the row's work begins with it
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) w.x[k] = S::load(reinterpret_cast<const U *>(a.h + at) + lane + k * NT);
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) w.dy[k] = S::load(reinterpret_cast<const U *>(a.dy + at) + lane + k * NT);
        if (has_t) {
            w.xt = a.h[at + cut.sc(lane)];
            w.dyt = a.dy[at + cut.sc(lane)];
        }
    };
    const int64_t step = blocks * RPB;
    int64_t r = block * RPB + sub;
    const auto work = [&](Row &w, Row &next, int64_t r, int odd, bool ahead) {
        const int64_t at = r * cols;
        constexpr bool kEarly = DH && VPT <= 6;  // dh fits beside x, dy and the next row's
        V dh[kEarly ? VPT : 1];
        T dht = T(0);
        if constexpr (DH) {
#pragma unroll
            for (int k = 0; k < (kEarly ? VPT : 0); k++)
                if (in_row(k)) dh[k] = S::load(reinterpret_cast<const U *>(a.dh + at) + lane + k * NT);
            if (has_t) dht = a.dh[at + cut.sc(lane)];
        }
        if (ahead && r + step < a.rows) load(next, r + step);
        const double rstd = double(w.rstd);
        double q = 0.0;
        const auto sums = [&](T xv, T dyv, T gv, double &ag) {
            const double d = double(dyv), xh = double(xv) * rstd;
            q = __builtin_fma(d * double(gv), xh, q);
            if constexpr (SUMS) ag = __builtin_fma(d, xh, ag);
        };
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) {
                const V gk = gamma_of(k);
#pragma unroll
                for (int j = 0; j < VN; j++) sums(w.x[k][j], w.dy[k][j], gk[j], sg[SUMS ? k : 0][j]);
                if constexpr (SUMS) {
                    // taken here: the compiler would put them off past the stores, with
                    // their operands' doubles kept until then
#pragma unroll
                    for (int j = 0; j < VN; j++) asm volatile("" : "+v"(sg[k][j]));
                }
            }
        if (has_t) sums(w.xt, w.dyt, gt, sgt);
        q = G::sum(q, lds_q[odd]);
        const double c2 = q * inv_c;
        const auto grad = [&](T xv, T dyv, T gv) {
            return T(rstd * __builtin_fma(-(double(xv) * rstd), c2, double(dyv) * double(gv)));
        };
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (a.dx && in_row(k)) {
                hide(w.x[k]);
                hide(w.dy[k]);
                if constexpr (Plan::kGammaRegs) hide(g[k]);
                const V gk = gamma_of(k);
                V o;
#pragma unroll
                for (int j = 0; j < VN; j++) o[j] = grad(w.x[k][j], w.dy[k][j], gk[j]);
                if constexpr (DH) {
                    V d;
                    if constexpr (kEarly) d = dh[k];
                    else d = S::load(reinterpret_cast<const U *>(a.dh + at) + lane + k * NT);
#pragma unroll
                    for (int j = 0; j < VN; j++) o[j] = o[j] + d[j];
                }
                S::store(o, reinterpret_cast<U *>(a.dx + at) + lane + k * NT);
            }
        if (a.dx && has_t) {
            const T o = grad(w.xt, w.dyt, gt);
            a.dx[at + cut.sc(lane)] = DH ? T(o + dht) : o;
        }
    };
    Row w;
    if (r < a.rows) load(w, r);
    if constexpr (VPT <= 8) {
        Row next;
        for (int odd = 0; r < a.rows; r += step, odd ^= 1) {
            work(w, next, r, odd, true);
            w = next;
        }
    } else {  // no registers for two rows
        for (int odd = 0; r < a.rows; r += step, odd ^= 1) {
            work(w, w, r, odd, false);
            if (r + step < a.rows) load(w, r + step);
        }
    }
    if constexpr (SUMS) {
        T *pg = a.part + block * cols;
        if constexpr (RPB == 1) {
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (in_row(k)) {
                    V o;
#pragma unroll
                    for (int j = 0; j < VN; j++) o[j] = T(sg[k][j]);
                    *(reinterpret_cast<U *>(pg) + lane + k * NT) = o;
                }
            if (has_t) pg[cut.sc(lane)] = T(sgt);
        } else {
            // fold the block's groups, one vector slot at a time
            __shared__ double fold[VN][256];
            const auto across = [&](auto n_c, const double *v, int64_t c0, bool mine) {
                constexpr int n = decltype(n_c)::value;
                __syncthreads();
#pragma unroll
                for (int j = 0; j < n; j++) fold[j][threadIdx.x] = v[j];
                __syncthreads();
                // O sums of RPB values by TPO lanes each, side by side
                constexpr int O = n * NT, TPO = O >= 256 ? 1 : (256 / O > 16 ? 16 : 256 / O);
                for (int e = threadIdx.x / TPO; e < O; e += 256 / TPO) {
                    const int l = e % NT, j = e / NT;
                    double t = 0.0;
                    for (int i = threadIdx.x % TPO; i < RPB; i += TPO) t += fold[j][l + i * NT];
                    if constexpr (TPO >= 2) t += dpp_d<kDppXor1>(t);
                    if constexpr (TPO >= 4) t += dpp_d<kDppXor2>(t);
                    if constexpr (TPO >= 8) t += dpp_d<kDppHalfMirror>(t);
                    if constexpr (TPO >= 16) t += dpp_d<kDppMirror>(t);
                    if (threadIdx.x % TPO == 0) fold[j][l] = t;
                }
                __syncthreads();
                if (sub == 0 && mine) {
                    for (int j = 0; j < n; j++) pg[c0 + j] = T(fold[j][lane]);
                }
            };
#pragma unroll
            for (int k = 0; k < VPT; k++)
                across(std::integral_constant<int, VN>{}, sg[k], int64_t(lane + k * NT) * VN, in_row(k));
            if (cut.rem) across(std::integral_constant<int, 1>{}, &sgt, cut.sc(lane), has_t);
        }
    }
}

template <typename T, int NT, int VPT, bool DH, bool SUMS, bool PAST>
__global__ __launch_bounds__((RmsGradPlan<T, NT, VPT>::NB), (RmsGradPlan<T, NT, VPT>::kWaves)) void k_rms_grad(
    RmsGradArgs<T> a)
{
    rms_grad_rows<T, NT, VPT, DH, SUMS, PAST>(a, blockIdx.x, gridDim.x);
}

// Sums of few rows, without partials: a block of NB lanes takes 128 bytes of columns, a
// vector a lane, the rows by NB / 8 streams, four of them in flight each, folded in LDS.
template <typename T, int NB>
NH_DEV void rms_few_cols(const RmsGradArgs<T> &a, int64_t block, T *dgamma)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, L = 8, S = NB / L, UN = 4, C = L * VN;
    __shared__ double sh[S][C];
    const int vl = threadIdx.x % L, st = threadIdx.x / L;
    const int64_t cols = a.cols, c = block * C + vl * VN;
    const bool whole = c + VN <= cols;
    double g[VN];
#pragma unroll
    for (int j = 0; j < VN; j++) g[j] = 0.0;
    for (int64_t r = st; r < a.rows; r += S * UN) {
        V x[UN], dy[UN];
        T rs[UN];
#pragma unroll
        for (int u = 0; u < UN; u++)
            if (r + u * S < a.rows) {
                const int64_t q = r + u * S, at = q * cols + c;
                rs[u] = a.rstd[q];
                if (whole) {
                    x[u] = *reinterpret_cast<const U *>(a.h + at);
                    dy[u] = *reinterpret_cast<const U *>(a.dy + at);
                } else {
#pragma unroll
                    for (int j = 0; j < VN; j++) {
                        x[u][j] = c + j < cols ? a.h[at + j] : T(0);
                        dy[u][j] = c + j < cols ? a.dy[at + j] : T(0);
                    }
                }
            }
#pragma unroll
        for (int u = 0; u < UN; u++)
            if (r + u * S < a.rows) {
                const double rstd = double(rs[u]);
#pragma unroll
                for (int j = 0; j < VN; j++) g[j] = __builtin_fma(double(dy[u][j]), double(x[u][j]) * rstd, g[j]);
            }
    }
#pragma unroll
    for (int j = 0; j < VN; j++) sh[st][vl * VN + j] = g[j];
    __syncthreads();
    // 8 lanes side by side take an eighth of the streams
    const int e = threadIdx.x / 8, part = threadIdx.x % 8;
    if (e < C) {  // whole waves: C is 32 or 16
        double t = 0.0;
        for (int i = part; i < S; i += 8) t += sh[i][e];
        t = RowGrp<8>::sum(t, nullptr);
        const int64_t at = block * C + e;
        if (part == 0 && at < cols) dgamma[at] = T(t);
    }
}

// The backward pass of few rows in one launch: blocks 0 .. nrows - 1 take the rows,
// the others columns (which read x and dy again, from the caches).  Either part may be absent.
template <typename T, int NT, int VPT, bool DH>
__global__ __launch_bounds__((RmsGradPlan<T, NT, VPT>::NB)) void k_rms_grad_few(RmsGradArgs<T> a, int nrows, T *dgamma)
{
    if (int(blockIdx.x) < nrows) rms_grad_rows<T, NT, VPT, DH, false, false>(a, blockIdx.x, nrows);
    else rms_few_cols<T, RmsGradPlan<T, NT, VPT>::NB>(a, int64_t(blockIdx.x) - nrows, dgamma);
}

// Few rows: what the one launch of k_rms_grad_few is for (f32 [197, 768] 3.4 us, 6.5 by k_rms_grad
// and the fold of its partials; [512, 4096] 7.4, 11.5; [512, 8192] 15.0, 14.9; [2048, 768] 14.4,
// 8.3).  By the shape alone, so that equal rows give equal sums whatever else a call asks for.
inline bool rms_few_rows(int64_t rows, int64_t cols) { return rows <= 512 && rows * cols <= int64_t(1) << 22; }

template <typename T, bool DH, int NT, int VPT>
static int launch_rms_grad_rows(const RmsGradArgs<T> &a0, T *dgamma)
{
    using Plan = RmsGradPlan<T, NT, VPT>;
    RmsGradArgs<T> a = a0;
    const int64_t need = ceil_div(a.rows, int64_t(Plan::RPB));
    if (rms_few_rows(a.rows, a.cols)) {
        const auto few = [&](int64_t nr, int64_t nc) {
            NH_LAUNCH((k_rms_grad_few<T, NT, VPT, DH>), dim3(unsigned(nr + nc)), dim3(Plan::NB), 0, stream(), a, int(nr),
                      dgamma);
        };
        const int64_t nr = a.dx ? need : 0, nc = dgamma ? ceil_div(a.cols, 8 * Vec16<T>::n) : 0;
        // the columns read what an output in place writes over: they go first then
        if (nr && nc && (a.dx == a.h || a.dx == a.dy)) {
            few(0, nc);
            few(nr, 0);
        } else {
            few(nr, nc);
        }
        return check_launch();
    }
    // as many blocks as the CUs hold at once, no more than rows
    const int64_t most = int64_t(num_cus()) * Plan::kPerCu, nb = need < most ? need : most;
    return with_stream<T, NT>(a.cols, [&](auto past) -> int {
        constexpr bool kPast = decltype(past)::value;
        if constexpr (VPT <= 8) {
            if (dgamma) {
                Partials part;
                NH_TRY(part.open(size_t(nb) * size_t(a.cols) * sizeof(T)));
                a.part = static_cast<T *>(part.p);
                NH_LAUNCH((k_rms_grad<T, NT, VPT, DH, true, kPast>), dim3(unsigned(nb)), dim3(Plan::NB), 0, stream(), a);
                launch_rms_fold(a.part, nb, a.cols, dgamma);
                return check_launch();
            }
        } else if (dgamma) {
            NH_TRY(launch_rms_cols(a, dgamma));
        }
        if (a.dx)
            NH_LAUNCH((k_rms_grad<T, NT, VPT, DH, false, kPast>), dim3(unsigned(nb)), dim3(Plan::NB), 0, stream(), a);
        return check_launch();
    });
}

// The fewest of LO to HI vectors per lane of NT that hold the row.
template <typename T, bool DH, int NT, int LO, int HI>
static int launch_rms_grad_exact(const RmsGradArgs<T> &a, int64_t ncv, T *dgamma)
{
    if constexpr (LO < HI) {
        if (ncv > NT * LO) return launch_rms_grad_exact<T, DH, NT, LO + 1, HI>(a, ncv, dgamma);
    }
    return launch_rms_grad_rows<T, DH, NT, LO>(a, dgamma);
}

template <typename T, bool DH>
static int launch_rms_grad_by(const RmsGradArgs<T> &a, T *dgamma)
{
    const int64_t ncv = a.cols / Vec16<T>::n;
    if (ncv <= 4) return launch_rms_grad_rows<T, DH, 4, 1>(a, dgamma);
    if (ncv <= 8 * 4) return launch_rms_grad_exact<T, DH, 8, 1, 4>(a, ncv, dgamma);
    if (ncv <= 16 * 4) return launch_rms_grad_exact<T, DH, 16, 3, 4>(a, ncv, dgamma);
    if (ncv <= 32 * 4) return launch_rms_grad_exact<T, DH, 32, 3, 4>(a, ncv, dgamma);
    if (ncv <= 64 * 4) return launch_rms_grad_exact<T, DH, 64, 3, 4>(a, ncv, dgamma);
    if (ncv <= 256 * 4) return launch_rms_grad_exact<T, DH, 256, 2, 4>(a, ncv, dgamma);
    if (ncv <= 512 * 8) return launch_rms_grad_exact<T, DH, 512, 3, 8>(a, ncv, dgamma);
    if (ncv <= 512 * 16) return launch_rms_grad_rows<T, DH, 512, 16>(a, dgamma);
    // the columns first: the row pass may write over what they read
    if (dgamma) NH_TRY(launch_rms_cols(a, dgamma));
    if (a.dx)
        for_row_launches(a.rows, 1, kLnWide, [&](unsigned g, int64_t base) {
            NH_LAUNCH((k_rms_grad_wide<T>), dim3(g), dim3(kLnWide), 0, stream(), a, base);
        });
    return check_launch();
}

template <typename T>
int launch_rms_grad(const RmsGradArgs<T> &a, T *dgamma)
{
    return a.dh ? launch_rms_grad_by<T, true>(a, dgamma) : launch_rms_grad_by<T, false>(a, dgamma);
}

}  // namespace nh
