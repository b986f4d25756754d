// layer_norm_grad_impl.hpp -- the backward pass of layer norm and of its join with the residual
// add and the counter-based dropout (formulas: layer_norm.hip), compiled for each type by
// layer_norm_grad_f32.hip and layer_norm_grad_f64.hip.
#pragma once

#include <type_traits>

#include "layer_norm.hpp"

namespace nh {

// How a group's lanes hold a row of the backward pass, and how many groups a CU
// holds.  NT lanes, VPT vectors each.  The sums of dgamma and dbeta over the rows are in
// double in every form: up to 4 vectors both in registers, and gamma; 5 to 8 vectors in LDS
// (128 KB at most: f64 rows both, f32 rows dgamma's, with dbeta's in registers), and gamma too
// where it fits beside them, else in registers: a load of it for each row would wait for the next
// row's loads, which are older.  16 vectors: no sums (k_ln_cols takes them), gamma from the L2.
template <typename T, int NT, int VPT>
struct LnGradPlan {
    static constexpr int NB = NT < 256 ? 256 : NT, RPB = NB / NT;
    static constexpr bool kRegs = VPT <= 4;                            // both sums in registers
    static constexpr bool kSplit = !kRegs && VPT <= 8 && sizeof(T) == 4;  // dbeta's in registers, dgamma's in LDS
    static constexpr bool kGammaRegs = VPT <= 4 || VPT == 7 || VPT == 8;
    static constexpr bool kGammaLds = VPT == 5 || VPT == 6;            // 144 KB with the sums
    // Two rows in turn, not copied from one to the other, which waits for the second's
    // loads before the third's are issued: for the one block that a CU holds, where
    // the registers allow it.  f32 [6710, 5000] 86.7 -> 79.8 us, joined 136 -> 130;
    // where other blocks fill the wait it loses ([43690, 768] 71.8, with it 75.8).
    static constexpr bool turns(int mode)
    {
        return NT == 512 && (mode == LN_PLAIN ? VPT <= 8 : VPT <= 6 && VPT != 4);
    }
    static constexpr int F = VPT <= 8 ? VPT - 1 : VPT / 2;  // vectors that are whole
    static constexpr int kWaves = VPT >= 3 || NT >= 512 ? 2 : 3;  // per SIMD
    static constexpr int kPerCu = kWaves * 256 / NB;              // resident blocks
};

// Bound by HBM: three streams (the joined forms five), and for the listed widths within
// 10% of a copy of the same bytes: f32 [16384, 4096] 136 us where the copy takes 134, and 4.9
// for the partials' fold (k_ln_fold); joined 221 and 4.7 (225); [200000, 96] 40.2 and 4.5 (38).
// f64 rows of an odd width, whose accesses straddle one 128-byte line in eight: 40.2 and
// 5.3 at [4096, 2049] (33).
//
// Groups of NT lanes walk the rows, r = group, group + groups, ...: each tensor
// read once, the next row's loads issued before this one is worked on, the row's
// two sums by one exchange (LDS slots alternate between rows, so one barrier a row
// is enough), and each lane's columns of dgamma and dbeta summed over the rows (SUMS).
// The block's groups fold theirs through LDS and the block leaves one row of
// partials, in the rows' type (the rounding of one of some hundred terms of a sum that is
// itself rounded so).  `block` of `blocks`.
//
// f32 rows of 8193 to 16387 values have one block's sums of 256 KB: dgamma's take 128 KB of LDS
// and dbeta's 64 registers a lane, which leaves none for a second row where gamma is in
// registers too (7 and 8 vectors, the joined forms' 6): there a vector of the next row is
// loaded as soon as this row's has been used for the last time, and dh behind the row's sums.
// (Both sums in LDS as floats, rounded every row, and the next row in registers: [2048, 16384]
// 84.5 us, now 85.6, joined 154, now 150; [2396, 14000] 88.2, now 92.0, joined 159, now 151;
// narrower alike; but 80 rows a block lost 11 u in dbeta, now 2 u.)
template <typename T, int NT, int VPT, int MODE, bool SUMS, bool PAST>
NH_DEV void ln_grad_rows(const LnGradArgs<T> &a, int64_t block, int64_t blocks)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    using G = RowGrp<NT>;
    using K = RowKeep<T, NT, VPT>;
    using S = RowStream<T, PAST>;
    using Plan = LnGradPlan<T, NT, VPT>;
    constexpr int VN = Vec16<T>::n, RPB = Plan::RPB;
    using D2 = typename Vec16<double>::type;
    constexpr bool SS = SUMS && Plan::kSplit, RS = SUMS && Plan::kRegs, LS = SUMS && !SS && !RS;
    constexpr bool RB = RS || SS;  // dbeta's sums in registers
    static_assert(!LS || sizeof(T) == 8, "the sums are in double");
    __shared__ double lds_s[2][G::kWaves], lds_q[2][G::kWaves];
    __shared__ uint8_t lds_keep[2][MODE == LN_DROP ? RPB : 1][MODE == LN_DROP ? K::kBytes : 1];
    __shared__ V lds_g[LS ? VPT : 1][LS ? NT : 1], lds_b[LS ? VPT : 1][LS ? NT : 1];
    __shared__ D2 lds_split[SS ? VPT : 1][SS ? VN / 2 : 1][SS ? NT : 1];
    // (a block of one row: a uniform row saves the address registers that SS is short of)
    const int lane = threadIdx.x % NT, sub = RPB == 1 ? 0 : threadIdx.x / NT;
    const int64_t cols = a.cols;
    const RowCut<T> cut(cols);
    const auto in_row = [&](int k) { return k < Plan::F || lane + k * NT < cut.ncv; };
    const bool has_t = lane < cut.rem;
    const double inv_c = 1.0 / double(cols);
    __shared__ V lds_gamma[Plan::kGammaLds ? VPT : 1][Plan::kGammaLds ? NT : 1];
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
    double sg[RS ? VPT : 1][VN], sb[RB ? VPT : 1][VN], sgt = 0.0, sbt = 0.0;
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        if constexpr (RS) {
#pragma unroll
            for (int j = 0; j < VN; j++) sg[k][j] = sb[k][j] = 0.0;
        } else if constexpr (SS) {
#pragma unroll
            for (int j = 0; j < VN; j++) sb[k][j] = 0.0;
#pragma unroll
            for (int i = 0; i < VN / 2; i++) lds_split[k][i][lane] = D2{0.0, 0.0};  // a lane's own slots
        } else if constexpr (LS) {
            V z;
#pragma unroll
            for (int j = 0; j < VN; j++) z[j] = T(0);
            lds_g[k][lane] = lds_b[k][lane] = z;  // a lane's own slots
        }
    }
    const DropKey key(a.drop);
    const T scale = T(a.drop.scale);
    struct Row {
        V x[VPT], dy[VPT];
        T xt, dyt, mean, rstd;
    };
    const auto load_x = [&](Row &w, int64_t at, int k) {
        if (in_row(k)) w.x[k] = S::load(reinterpret_cast<const U *>(a.h + at) + lane + k * NT);
    };
    const auto load_dy = [&](Row &w, int64_t at, int k) {
        if (in_row(k)) w.dy[k] = S::load(reinterpret_cast<const U *>(a.dy + at) + lane + k * NT);
    };
    // first, since loads return in order and the row's work begins with them (behind the row's
    // others: [512, 4096] 9.3 us, 8.9 so)
    const auto load_stats = [&](Row &w, int64_t r) {
        w.mean = a.mean[r];
        w.rstd = a.rstd[r];
    };
    const auto load_tail = [&](Row &w, int64_t at) {
        if (has_t) {
            w.xt = a.h[at + cut.sc(lane)];
            w.dyt = a.dy[at + cut.sc(lane)];
        }
    };
    const auto load = [&](Row &w, int64_t r) {
        const int64_t at = r * cols;
        load_stats(w, r);
#pragma unroll
        for (int k = 0; k < VPT; k++) load_x(w, at, k);
#pragma unroll
        for (int k = 0; k < VPT; k++) load_dy(w, at, k);
        load_tail(w, at);
    };
    const int64_t step = blocks * RPB;
    int64_t r = block * RPB + sub;
    // kReload: no registers for two rows; a vector of the next row is loaded where this row's
    // has been used for the last time.
    constexpr bool kReload = SS && (Plan::kGammaRegs || (MODE != LN_PLAIN && VPT == 6));
    // Work on row r in w; `ahead`: the next row's loads are issued here, into next.
    const auto work = [&](Row &w, Row &next, int64_t r, int odd, bool ahead) {
        const int64_t at = r * cols;
        constexpr bool kEarly = MODE != LN_PLAIN && VPT <= 8;  // dh fits beside x and dy
        V dh[kEarly ? VPT : 1];
        T dht = T(0);
        const auto load_dh = [&] {
            if (!a.dh) return;
#pragma unroll
            for (int k = 0; k < (kEarly ? VPT : 0); k++)
                if (in_row(k)) dh[k] = S::load(reinterpret_cast<const U *>(a.dh + at) + lane + k * NT);
            if (has_t) dht = a.dh[at + cut.sc(lane)];
        };
        if constexpr (MODE != LN_PLAIN && !kReload) load_dh();
        if (ahead && r + step < a.rows) load(next, r + step);
        const double mean = double(w.mean), rstd = double(w.rstd);
        K keep;
        if constexpr (MODE == LN_DROP) keep.make(r, cols, cut, lane, key, lds_keep[odd][sub]);
        double s = 0.0, q = 0.0;
        const auto sums = [&](T xv, T dyv, T gv, double &ag, double &ab) {
            const double d = double(dyv), xh = (double(xv) - mean) * rstd, wv = d * double(gv);
            s += wv;
            q = __builtin_fma(wv, xh, q);
            ag = __builtin_fma(d, xh, ag);
            ab += d;
        };
#pragma unroll
        for (int k = 0; k < VPT; k++)
            if (in_row(k)) {
                const V gk = gamma_of(k);
                V vg, vb;
                D2 vd[SS ? VN / 2 : 1];
                if constexpr (LS) {
                    vg = lds_g[k][lane];
                    vb = lds_b[k][lane];
                } else if constexpr (SS) {
#pragma unroll
                    for (int i = 0; i < VN / 2; i++) vd[i] = lds_split[k][i][lane];
                }
#pragma unroll
                for (int j = 0; j < VN; j++) {
                    if constexpr (LS) {
                        double ag = double(vg[j]), ab = double(vb[j]);
                        sums(w.x[k][j], w.dy[k][j], gk[j], ag, ab);
                        vg[j] = T(ag);
                        vb[j] = T(ab);
                    } else if constexpr (SS) {
                        double ag = vd[j / 2][j % 2];
                        sums(w.x[k][j], w.dy[k][j], gk[j], ag, sb[k][j]);
                        vd[j / 2][j % 2] = ag;
                    } else {
                        sums(w.x[k][j], w.dy[k][j], gk[j], sg[RS ? k : 0][j], sb[RB ? k : 0][j]);
                    }
                }
                if constexpr (RS) {
                    // taken here: the compiler would put them off past the stores, with
                    // their operands' doubles kept until then
#pragma unroll
                    for (int j = 0; j < VN; j++) asm volatile("" : "+v"(sg[k][j]), "+v"(sb[k][j]));
                }
                if constexpr (LS) {
                    lds_g[k][lane] = vg;
                    lds_b[k][lane] = vb;
                    asm volatile("" : "+v"(s), "+v"(q) : : "memory");  // one vector's terms in registers at a time
                }
                if constexpr (SS) {
#pragma unroll
                    for (int i = 0; i < VN / 2; i++) lds_split[k][i][lane] = vd[i];
#pragma unroll
                    for (int j = 0; j < VN; j++) asm volatile("" : "+v"(sb[k][j]));
                    asm volatile("" : "+v"(s), "+v"(q) : : "memory");
                }
            }
        if (has_t) sums(w.xt, w.dyt, gt, sgt, sbt);
        if constexpr (MODE != LN_PLAIN && kReload) load_dh();
        // both sums over the row by one exchange
        const auto add = [](double p, double t) { return p + t; };
        s = G::part(s, add);
        q = G::part(q, add);
        if constexpr (G::kWaves > 1) {
            if ((threadIdx.x & 63) == 0) {
                lds_s[odd][threadIdx.x >> 6] = s;
                lds_q[odd][threadIdx.x >> 6] = q;
            }
            __syncthreads();
            s = lds_s[odd][0];
            q = lds_q[odd][0];
#pragma unroll
            for (int i = 1; i < G::kWaves; i++) {
                s += lds_s[odd][i];
                q += lds_q[odd][i];
            }
        }
        const double c1 = s * inv_c, c2 = q * inv_c;
        const auto grad = [&](T xv, T dyv, T gv) {
            const double xh = (double(xv) - mean) * rstd, wv = double(dyv) * double(gv);
            return T(rstd * (__builtin_fma(-xh, c2, wv - c1)));
        };
        const int64_t after = (r + step) * cols;
        const bool again = kReload && r + step < a.rows;
        if (again) load_stats(w, r + step);
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            if ((MODE != LN_PLAIN || a.dx) && in_row(k)) {
                hide(w.x[k]);
                hide(w.dy[k]);
                if constexpr (Plan::kGammaRegs) hide(g[k]);
                const V gk = gamma_of(k);
                V o;
#pragma unroll
                for (int j = 0; j < VN; j++) o[j] = grad(w.x[k][j], w.dy[k][j], gk[j]);
                if constexpr (MODE != LN_PLAIN) {
                    if (a.dh) {
                        V d;
                        if constexpr (kEarly) d = dh[k];
                        else d = S::load(reinterpret_cast<const U *>(a.dh + at) + lane + k * NT);
#pragma unroll
                        for (int j = 0; j < VN; j++) o[j] = o[j] + d[j];
                    }
                    if (a.dres) S::store(o, reinterpret_cast<U *>(a.dres + at) + lane + k * NT);
                }
                if constexpr (MODE == LN_DROP) {
#pragma unroll
                    for (int j = 0; j < VN; j++) o[j] = dropped<T>(o[j], scale, keep.m[k], K::bit(j));
                }
                if (MODE == LN_PLAIN || a.dx)
                    S::store(o, reinterpret_cast<U *>(a.dx + at) + lane + k * NT);
            }
            if (again) {
                load_x(w, after, k);
                load_dy(w, after, k);
            }
        }
        if (has_t) {
            const int64_t i = at + cut.sc(lane);
            T o = grad(w.xt, w.dyt, gt);
            if constexpr (MODE != LN_PLAIN) {
                if (a.dh) o = o + dht;
                if (a.dres) a.dres[i] = o;
            }
            if constexpr (MODE == LN_DROP) o = dropped<T>(o, scale, keep.tail, 0);
            if (a.dx) a.dx[i] = o;
        }
        if (again) load_tail(w, after);
    };
    Row w;
    if (r < a.rows) load(w, r);
    if constexpr (kReload) {
        for (int odd = 0; r < a.rows; r += step, odd ^= 1) work(w, w, r, odd, false);
    } else if constexpr (Plan::turns(MODE)) {
        Row v;
        while (r < a.rows) {
            work(w, v, r, 0, true);
            r += step;
            if (r >= a.rows) break;
            work(v, w, r, 1, true);
            r += step;
        }
    } else if constexpr (VPT <= 8) {
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
        T *pg = a.part + block * 2 * cols, *pb = pg + cols;
        if constexpr (RPB == 1) {
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (in_row(k)) {
                    V og, ob;
                    if constexpr (LS) {
                        og = lds_g[k][lane];
                        ob = lds_b[k][lane];
                    } else {
#pragma unroll
                        for (int j = 0; j < VN; j++) {
                            og[j] = T(SS ? lds_split[k][SS ? j / 2 : 0][lane][j % 2] : sg[RS ? k : 0][j]);
                            ob[j] = T(sb[k][j]);
                        }
                    }
                    *(reinterpret_cast<U *>(pg) + lane + k * NT) = og;
                    *(reinterpret_cast<U *>(pb) + lane + k * NT) = ob;
                }
            if (has_t) {
                pg[cut.sc(lane)] = T(sgt);
                pb[cut.sc(lane)] = T(sbt);
            }
        } else {
            // fold the block's groups, one vector slot at a time
            __shared__ double fold[2 * VN][256];
            const auto across = [&](auto n_c, const double *vg, const double *vb, int64_t c0, bool mine) {
                constexpr int n = decltype(n_c)::value;
                __syncthreads();
#pragma unroll
                for (int j = 0; j < n; j++) {
                    fold[j][threadIdx.x] = vg[j];
                    fold[n + j][threadIdx.x] = vb[j];
                }
                __syncthreads();
                // O sums of RPB values by TPO lanes each, side by side
                constexpr int O = 2 * n * NT, TPO = O >= 256 ? 1 : (256 / O > 16 ? 16 : 256 / O);
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
                    for (int j = 0; j < n; j++) {
                        pg[c0 + j] = T(fold[j][lane]);
                        pb[c0 + j] = T(fold[n + j][lane]);
                    }
                }
            };
#pragma unroll
            for (int k = 0; k < VPT; k++)
                across(std::integral_constant<int, VN>{}, sg[k], sb[k], int64_t(lane + k * NT) * VN, in_row(k));
            if (cut.rem) across(std::integral_constant<int, 1>{}, &sgt, &sbt, cut.sc(lane), has_t);
        }
    }
}

template <typename T, int NT, int VPT, int MODE, bool SUMS, bool PAST>
__global__ __launch_bounds__((LnGradPlan<T, NT, VPT>::NB), (LnGradPlan<T, NT, VPT>::kWaves)) void k_ln_grad(
    LnGradArgs<T> a)
{
    ln_grad_rows<T, NT, VPT, MODE, SUMS, PAST>(a, blockIdx.x, gridDim.x);
}

// Sums of few rows, without partials: a block of NB lanes takes 128 bytes of columns, a
// vector a lane, the rows by NB / 8 streams, four of them in flight each, folded in LDS.
template <typename T, int NB>
NH_DEV void ln_few_cols(const LnGradArgs<T> &a, int64_t block, T *dgamma, T *dbeta)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, L = 8, S = NB / L, UN = 4, C = L * VN;
    __shared__ double sh[S][2 * C];  // [stream][dgamma of C columns, dbeta of C]
    const int vl = threadIdx.x % L, st = threadIdx.x / L;
    const int64_t cols = a.cols, c = block * C + vl * VN;
    const bool whole = c + VN <= cols;
    double g[VN], b[VN];
#pragma unroll
    for (int j = 0; j < VN; j++) g[j] = b[j] = 0.0;
    for (int64_t r = st; r < a.rows; r += S * UN) {
        V x[UN], dy[UN];
        T m[UN], rs[UN];
#pragma unroll
        for (int u = 0; u < UN; u++)
            if (r + u * S < a.rows) {
                const int64_t q = r + u * S, at = q * cols + c;
                m[u] = a.mean[q];
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
                const double mean = double(m[u]), rstd = double(rs[u]);
#pragma unroll
                for (int j = 0; j < VN; j++) {
                    const double d = double(dy[u][j]);
                    g[j] = __builtin_fma(d, (double(x[u][j]) - mean) * rstd, g[j]);
                    b[j] += d;
                }
            }
    }
#pragma unroll
    for (int j = 0; j < VN; j++) {
        sh[st][vl * VN + j] = g[j];
        sh[st][C + vl * VN + j] = b[j];
    }
    __syncthreads();
    // 4 lanes side by side take a quarter of the streams each
    const int e = threadIdx.x / 4, part = threadIdx.x % 4;
    if (e < 2 * C) {  // whole waves: 2 C is 64 or 32
        double t = 0.0;
        for (int i = part; i < S; i += 4) t += sh[i][e];
        t += dpp_d<kDppXor1>(t);
        t += dpp_d<kDppXor2>(t);
        const int64_t at = block * C + e % C;
        T *out = e < C ? dgamma : dbeta;
        if (part == 0 && out && at < cols) out[at] = T(t);
    }
}

// The backward pass of few rows in one launch: blocks 0 .. nrows - 1 take the rows,
// the others columns (which read x and dy again, from the caches).  Either
// part may be absent.  Bound by latency; against the row pass and a fold of its
// partials (two launches and a round trip): f32 [197, 768] 7.9 -> 3.9 us, [256, 4096] 11.5 ->
// 5.6, [512, 4096] 17.1 -> 10.7, f64 [512, 1024] 13.1 -> 6.9.  From some 1000 rows a column's
// stream of rows is longer than that ([1000, 1000] 11.1, 20).
template <typename T, int NT, int VPT, int MODE>
__global__ __launch_bounds__((LnGradPlan<T, NT, VPT>::NB)) void k_ln_grad_few(LnGradArgs<T> a, int nrows, T *dgamma,
                                                                             T *dbeta)
{
    if (int(blockIdx.x) < nrows) ln_grad_rows<T, NT, VPT, MODE, false, false>(a, blockIdx.x, nrows);
    else ln_few_cols<T, LnGradPlan<T, NT, VPT>::NB>(a, int64_t(blockIdx.x) - nrows, dgamma, dbeta);
}

// Column sums of the partials: [n][2 cols] -> dgamma, dbeta.  A block of 1024 lanes
// takes 32 columns, the partials by 128 (f64 64) streams of four in flight.  f32
// [4096, 1024] in all 15.9 us with 64 columns, 15.3 with 32; f64 [4096, 2049] 45.3 with 32,
// 46.7 with 16.  b_base: the launch's first block, not its first column, which the compiler
// would not know to be even: f64 [15360, 34] joined 10.9 us, 10.35 so.
template <typename T>
__global__ __launch_bounds__(1024) void k_ln_fold(const T *__restrict__ part, int64_t n, int64_t cols,
                                                  T *__restrict__ dgamma, T *__restrict__ dbeta, int64_t b_base)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, C = 32, L = C / VN, S = 1024 / L, UN = 4, TPC = 1024 / C;
    __shared__ double sh[S][C + 1];  // (read by columns below: no two lanes on a bank)
    const int vl = threadIdx.x % L, st = threadIdx.x / L;
    const int64_t width = 2 * cols, c0 = (b_base + int64_t(blockIdx.x)) * C, c = c0 + vl * VN;
    double s[VN];
#pragma unroll
    for (int j = 0; j < VN; j++) s[j] = 0.0;
    for (int64_t i = st; i < n; i += S * UN) {
        V v[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const T *p = part + (i + u * S) * width + c;
            if (i + u * S < n) {
                if (c + VN <= width) {
                    v[u] = *reinterpret_cast<const U *>(p);
                } else {
#pragma unroll
                    for (int j = 0; j < VN; j++) v[u][j] = c + j < width ? p[j] : T(0);
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
    const int64_t at = c0 + e;
    if (part_of == 0 && at < width) {
        T *out = at < cols ? dgamma : dbeta;
        if (out) out[at < cols ? at : at - cols] = T(t);
    }
}

template <typename T>
static void launch_ln_fold(const T *part, int64_t n, int64_t cols, T *dgamma, T *dbeta)
{
    for_row_launches(ceil_div(2 * cols, 32), 1, 1024, [&](unsigned g, int64_t base) {
        NH_LAUNCH((k_ln_fold<T>), dim3(g), dim3(1024), 0, stream(), part, n, cols, dgamma, dbeta, base);
    });
}

// Rows wider than a block's registers: the row's sums, then the outputs, reading
// every tensor again, and the column sums apart (k_ln_cols): three readings bound it
// (f32 [335, 100000] 206 us, 280 us joined; a copy of the least bytes 65 and 109).
template <typename T, int MODE>
__global__ __launch_bounds__(kLnWide) void k_ln_grad_wide(LnGradArgs<T> a, int64_t r_base)
{
    using G = RowGrp<kLnWide>;
    __shared__ double lds_s[G::kWaves], lds_q[G::kWaves];
    const DropKey key(a.drop);
    const T scale = T(a.drop.scale);
    const int64_t r = r_base + blockIdx.x, cols = a.cols, at = r * cols;
    const double mean = double(a.mean[r]), rstd = double(a.rstd[r]), inv_c = 1.0 / double(cols);
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
    double s = 0.0, q = 0.0;
    walk_row<T>(cols, load, [&](auto w, int64_t, const auto &v) {
#pragma unroll
        for (int j = 0; j < decltype(w)::value; j++) {
            const double xh = (double(v.x.v[j]) - mean) * rstd, wv = double(v.dy.v[j]) * double(v.g.v[j]);
            s += wv;
            q = __builtin_fma(wv, xh, q);
        }
    });
    const double c1 = G::sum(s, lds_s) * inv_c, c2 = G::sum(q, lds_q) * inv_c;
    walk_row<T>(cols, load, [&](auto w, int64_t c, const auto &v) {
        constexpr int W = decltype(w)::value;
        Pack<T, W> o;
#pragma unroll
        for (int j = 0; j < W; j++) {
            const double xh = (double(v.x.v[j]) - mean) * rstd, wv = double(v.dy.v[j]) * double(v.g.v[j]);
            o.v[j] = T(rstd * __builtin_fma(-xh, c2, wv - c1));
        }
        if constexpr (MODE != LN_PLAIN) {
            if (a.dh) {
                const Pack<T, W> d = Pack<T, W>::load(a.dh + at + c);
#pragma unroll
                for (int j = 0; j < W; j++) o.v[j] = o.v[j] + d.v[j];
            }
            if (a.dres) o.store(a.dres + at + c);
        }
        if constexpr (MODE == LN_DROP) {
            const uint32_t m = keep_at<W>(at + c, key);
#pragma unroll
            for (int j = 0; j < W; j++) o.v[j] = dropped<T>(o.v[j], scale, m, j);
        }
        if (a.dx) o.store(a.dx + at + c);
    });
}

// Column sums beside a row pass that cannot hold them: 64 lanes of VN columns a block, the
// rows of its chunk by 8 waves, four in flight each.  b_base: as k_ln_fold's.
template <typename T>
__global__ __launch_bounds__(512) void k_ln_cols(LnGradArgs<T> a, int64_t chunk, int64_t b_base)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, W = 8, UN = 4;
    __shared__ double sh[W][2 * VN][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t cols = a.cols, c = ((b_base + int64_t(blockIdx.x)) * 64 + lane) * VN;
    const int64_t r0 = int64_t(blockIdx.y) * chunk, r1 = r0 + chunk < a.rows ? r0 + chunk : a.rows;
    const bool whole = c + VN <= cols;
    double s[2 * VN];
#pragma unroll
    for (int j = 0; j < 2 * VN; j++) s[j] = 0.0;
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
                const double mean = double(a.mean[r + u * W]), rstd = double(a.rstd[r + u * W]);
#pragma unroll
                for (int j = 0; j < VN; j++) {
                    const double d = double(dy[u][j]);
                    s[j] = __builtin_fma(d, (double(x[u][j]) - mean) * rstd, s[j]);
                    s[VN + j] += d;
                }
            }
    }
#pragma unroll
    for (int j = 0; j < 2 * VN; j++) sh[w][j][lane] = s[j];
    __syncthreads();
    // wave w folds columns' sum w of each lane (2 VN <= W)
    if (w < 2 * VN && c + w % VN < cols) {
        double t = sh[0][w][lane];
        for (int i = 1; i < W; i++) t += sh[i][w][lane];
        a.part[(int64_t(blockIdx.y) * 2 + w / VN) * cols + c + w % VN] = T(t);
    }
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

// Column sums by k_ln_cols and a fold.
template <typename T>
static int launch_ln_cols(LnGradArgs<T> a, T *dgamma, T *dbeta)
{
    const int64_t gx = ceil_div(a.cols, 64 * Vec16<T>::n);
    int64_t chunks = ceil_div(int64_t(num_cus()) * 2, gx);
    const int64_t most = ceil_div(a.rows, 32);
    chunks = chunks < most ? chunks : most;
    const int64_t chunk = ceil_div(a.rows, chunks);
    chunks = ceil_div(a.rows, chunk);
    Partials part;
    NH_TRY(part.open(size_t(chunks) * 2 * size_t(a.cols) * sizeof(T)));
    a.part = static_cast<T *>(part.p);
    for_row_launches(gx, 1, 512, [&](unsigned g, int64_t base) {
        NH_LAUNCH((k_ln_cols<T>), dim3(g, unsigned(chunks)), dim3(512), 0, stream(), a, chunk, base);
    });
    launch_ln_fold(a.part, chunks, a.cols, dgamma, dbeta);
    return check_launch();
}

// Few rows: what the one launch of k_ln_grad_few is for.  By the shape alone, so that equal
// rows give equal sums whatever else a call asks for.
constexpr int64_t kFewRows = 512, kFewValues = int64_t(1) << 22;
inline bool few_rows(int64_t rows, int64_t cols) { return rows <= kFewRows && rows * cols <= kFewValues; }

template <typename T, int MODE, int NT, int VPT>
static int launch_ln_grad_rows(const LnGradArgs<T> &a0, T *dgamma, T *dbeta)
{
    using Plan = LnGradPlan<T, NT, VPT>;
    LnGradArgs<T> a = a0;
    const bool sums = dgamma || dbeta, rows = a.dx || a.dres;
    const int64_t need = ceil_div(a.rows, int64_t(Plan::RPB));
    if (few_rows(a.rows, a.cols)) {
        const auto few = [&](int64_t nr, int64_t nc) {
            NH_LAUNCH((k_ln_grad_few<T, NT, VPT, MODE>), dim3(unsigned(nr + nc)), dim3(Plan::NB), 0, stream(), a, int(nr),
                      dgamma, dbeta);
        };
        const int64_t nr = rows ? need : 0, nc = sums ? ceil_div(a.cols, 8 * Vec16<T>::n) : 0;
        // the columns read what an output in place writes over: they go first then
        const bool over = a.dx == a.h || a.dx == a.dy || a.dres == a.h || a.dres == a.dy;
        if (rows && sums && over) {
            few(0, nc);
            few(nr, 0);
        } else {
            few(nr, nc);
        }
        return check_launch();
    }
    // as many blocks as the CUs hold at once, no more than rows
    const int64_t most = int64_t(num_cus()) * Plan::kPerCu;
    const int64_t nb = need < most ? need : most;
    return with_stream<T, NT>(a.cols, [&](auto past) -> int {
        constexpr bool kPast = decltype(past)::value;
        if constexpr (VPT <= 8) {
            if (sums) {
                Partials part;
                NH_TRY(part.open(size_t(nb) * 2 * size_t(a.cols) * sizeof(T)));
                a.part = static_cast<T *>(part.p);
                NH_LAUNCH((k_ln_grad<T, NT, VPT, MODE, true, kPast>), dim3(unsigned(nb)), dim3(Plan::NB), 0, stream(), a);
                launch_ln_fold(a.part, nb, a.cols, dgamma, dbeta);
                return check_launch();
            }
        } else if (sums) {
            NH_TRY(launch_ln_cols(a, dgamma, dbeta));
        }
        if (rows)
            NH_LAUNCH((k_ln_grad<T, NT, VPT, MODE, false, kPast>), dim3(unsigned(nb)), dim3(Plan::NB), 0, stream(), a);
        return check_launch();
    });
}

// The fewest of LO to HI vectors per lane of NT that hold the row.
template <typename T, int MODE, int NT, int LO, int HI>
static int launch_ln_grad_exact(const LnGradArgs<T> &a, int64_t ncv, T *dgamma, T *dbeta)
{
    if constexpr (LO < HI) {
        if (ncv > NT * LO) return launch_ln_grad_exact<T, MODE, NT, LO + 1, HI>(a, ncv, dgamma, dbeta);
    }
    return launch_ln_grad_rows<T, MODE, NT, LO>(a, dgamma, dbeta);
}

template <typename T, int MODE>
int launch_ln_grad(const LnGradArgs<T> &a, T *dgamma, T *dbeta)
{
    const int64_t ncv = a.cols / Vec16<T>::n;
    if (ncv <= 4) return launch_ln_grad_rows<T, MODE, 4, 1>(a, dgamma, dbeta);
    if (ncv <= 8 * 4) return launch_ln_grad_exact<T, MODE, 8, 1, 4>(a, ncv, dgamma, dbeta);
    if (ncv <= 16 * 4) return launch_ln_grad_exact<T, MODE, 16, 3, 4>(a, ncv, dgamma, dbeta);
    if (ncv <= 32 * 4) return launch_ln_grad_exact<T, MODE, 32, 3, 4>(a, ncv, dgamma, dbeta);
    if (ncv <= 64 * 4) return launch_ln_grad_exact<T, MODE, 64, 3, 4>(a, ncv, dgamma, dbeta);
    if (ncv <= 256 * 4) return launch_ln_grad_exact<T, MODE, 256, 2, 4>(a, ncv, dgamma, dbeta);
    if (ncv <= 512 * 8) return launch_ln_grad_exact<T, MODE, 512, 3, 8>(a, ncv, dgamma, dbeta);
    if (ncv <= 512 * 16) return launch_ln_grad_rows<T, MODE, 512, 16>(a, dgamma, dbeta);
    // the columns first: the row pass may write over what they read
    if (dgamma || dbeta) NH_TRY(launch_ln_cols(a, dgamma, dbeta));
    if (a.dx || a.dres)
        for_row_launches(a.rows, 1, kLnWide, [&](unsigned g, int64_t base) {
            NH_LAUNCH((k_ln_grad_wide<T, MODE>), dim3(g), dim3(kLnWide), 0, stream(), a, base);
        });
    return check_launch();
}

}  // namespace nh
