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

// What a part of a row leaves: its largest value m, s = sum exp((x - m) / T) and t = sum
// exp((x - m) / T) (x - m).
struct LpPart {
    double m, s, t;
};

// The sums of two parts by the larger m.  A part without values (m -inf) has s = t = 0, or NaN
// where it holds NaN, which stays.
NH_DEV LpPart lp_join(const LpPart &a, const LpPart &b, double inv_t)
{
    const double none = -__builtin_inf(), m = __builtin_fmax(a.m, b.m);
    const double da = a.m == none ? 0.0 : a.m - m, db = b.m == none ? 0.0 : b.m - m;
    const double fa = a.m == none ? 0.0 : exp(da * inv_t), fb = b.m == none ? 0.0 : exp(db * inv_t);
    return {m, a.s * fa + b.s * fb, fa * (a.t + da * a.s) + fb * (b.t + db * b.s)};
}

// The same over N parts, and over a wave's lanes: one exponential for each.
template <int N>
NH_DEV LpPart lp_join_all(const LpPart (&p)[N], double inv_t)
{
    LpPart r{p[0].m, 0.0, 0.0};
#pragma unroll
    for (int i = 1; i < N; i++) r.m = __builtin_fmax(r.m, p[i].m);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const bool any = p[i].m != -__builtin_inf();
        const double d = any ? p[i].m - r.m : 0.0, f = any ? exp(d * inv_t) : 0.0;
        r.s += p[i].s * f;
        r.t += f * (p[i].t + d * p[i].s);
    }
    return r;
}
NH_DEV LpPart lp_join_wave(const LpPart &p, double inv_t)
{
    const double m = RowGrp<64>::max(p.m, nullptr);
    const bool any = p.m != -__builtin_inf();
    const double d = any ? p.m - m : 0.0, f = any ? exp(d * inv_t) : 0.0;
    return {m, wave_dsum(p.s * f), wave_dsum(f * (p.t + d * p.s))};
}

// A row's results from its sums.
struct LpRow {
    double m, inv_t, s, ls;  // m: 0 where every logit is masked
    NH_DEV LpRow(const LpPart &p, double it) : m(p.m == -__builtin_inf() ? 0.0 : p.m), inv_t(it), s(p.s), ls(log(p.s)) {}
    NH_DEV bool sound() const { return s == s; }
    NH_DEV double logprob(double x) const { return s == 0.0 ? -__builtin_inf() : (x - m) * inv_t - ls; }
    NH_DEV double lse() const { return m * inv_t + ls; }
    NH_DEV double entropy(double t) const { return s == 0.0 ? 0.0 : ls - t * inv_t / s; }
};

template <typename T>
NH_DEV void lp_store(const LpArgs<T> &a, int64_t r, int64_t tok, const LpRow &row, double t)
{
    if (a.logprob) a.logprob[r] = tok < a.cols ? T(row.logprob(double(a.x[r * a.cols + tok]))) : T(__builtin_nan(""));
    if (a.entropy) a.entropy[r] = T(row.entropy(t));
    if (a.lse) a.lse[r] = T(row.lse());
}
template <typename T>
NH_DEV void lp_store_top(const LpArgs<T> &a, int64_t r, int q, const LpKey<T> &k, const LpRow &row)
{
    if (a.top_ids) a.top_ids[r * a.k + q] = row.sound() ? int64_t(k.i) : -1;
    if (a.top_lp)
        a.top_lp[r * a.k + q] = !row.sound() ? T(__builtin_nan("")) : k.i < 0 ? -T(__builtin_inf()) : T(row.logprob(double(k.v)));
}
// A row that is not used, by a group of NT lanes.
template <typename T, int NT>
NH_DEV void lp_unused(const LpArgs<T> &a, int64_t r, int lane)
{
    if (lane == 0) {
        if (a.logprob) a.logprob[r] = T(0);
        if (a.entropy) a.entropy[r] = T(0);
        if (a.lse) a.lse[r] = T(0);
    }
    for (int q = lane; q < a.k; q += NT) {
        if (a.top_ids) a.top_ids[r * a.k + q] = -1;
        if (a.top_lp) a.top_lp[r * a.k + q] = -T(__builtin_inf());
    }
}

// All lanes of a group, a wave or a block of 256.
template <int NT>
NH_DEV void lp_meet()
{
    if constexpr (NT == 64) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}

template <typename T>
NH_DEV LpKey<T> lp_first(const LpKey<T> &a, const LpKey<T> &b) { return b.before(a) ? b : a; }
template <typename T>
NH_DEV LpKey<T> lp_wave_first(LpKey<T> k)
{
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) k = lp_first(k, LpKey<T>{__shfl_xor(k.v, off, 64), __shfl_xor(k.i, off, 64)});
    return k;
}

// LDS of a group that orders alternatives.
template <typename T, int NT>
struct LpOrder {
    static constexpr int kCand = NT == 64 ? 256 : 1024;
    T v[kCand];
    int i[kCand];
    int n;
    T wave_v[4];
    int wave_i[4];
    LpKey<T> out[kLpMaxTop];
};

// The k first of n candidates (n <= kCand, all apart) into o.out: a candidate's place is
// the number of those before it.
template <typename T, int NT>
NH_DEV void lp_rank(LpOrder<T, NT> &o, int n, int k, int lane)
{
    for (int q = lane; q < k; q += NT)
        if (q >= n) o.out[q] = LpKey<T>::none();
    for (int c = lane; c < n; c += NT) {
        const LpKey<T> mine{o.v[c], o.i[c]};
        int place = 0;
        for (int j = 0; j < n; j++) place += LpKey<T>{o.v[j], o.i[j]}.before(mine) ? 1 : 0;
        if (place < k) o.out[place] = mine;
    }
}

// The k first keys by k rounds of the group's best key behind the one found before: for rows
// whose values crowd at the bound (each(f): f(key) for every key of a lane).
template <typename T, int NT, typename E>
NH_DEV void lp_rounds(LpOrder<T, NT> &o, int k, int lane, E each)
{
    LpKey<T> last = LpKey<T>::none();
    for (int q = 0; q < k; q++) {
        LpKey<T> best = LpKey<T>::none();
        if (q == 0 || last.i >= 0)
            each([&](const LpKey<T> &c) {
                if (c.before(best) && (q == 0 || last.before(c))) best = c;
            });
        best = lp_wave_first(best);
        if constexpr (NT > 64) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) {
                o.wave_v[threadIdx.x >> 6] = best.v;
                o.wave_i[threadIdx.x >> 6] = best.i;
            }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NT / 64; w++) best = lp_first(best, LpKey<T>{o.wave_v[w], o.wave_i[w]});
        }
        last = best;
        if (lane == 0) o.out[q] = best;
    }
}

// Where a row is split: its parts' sums and alternatives, [rows][parts] and [rows][parts][k].
template <typename T>
struct LpScratch {
    LpPart *part;
    T *v;
    int *i;
};

// A group of NT lanes (a wave, or a block of 256) holds one of `parts` parts of a row in
// registers, VPT vectors a lane: one read.  Each wave takes its own largest value as the
// reference of its exponentials.  The k first values of the part: with j = k / waves rounded up,
// the j-th largest of a wave's lanes' largest values, and the least of those over the waves, is
// passed by k values at least; what passes it (some 2 k in a random row) is collected and
// ordered by counting.  Bound by HBM where rows are many.
template <typename T, int NT, int VPT>
__global__ __launch_bounds__(256) void k_lp_parts(LpArgs<T> a, LpScratch<T> scratch, int parts, int64_t b_base)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, RPB = 256 / NT, W = NT / 64;
    __shared__ LpPart sh[4];
    __shared__ LpOrder<T, NT> order[RPB];
    const int lane = threadIdx.x % NT, sub = RPB == 1 ? 0 : threadIdx.x / NT;
    const int64_t unit = (b_base + int64_t(blockIdx.x)) * RPB + sub;
    const int64_t r = parts == 1 ? unit : unit / parts;
    const int p = parts == 1 ? 0 : int(unit - r * parts);
    if (RPB > 1 && r >= a.rows) return;
    const int64_t tok = a.tokens ? a.tokens[r] : 0;
    if (tok < 0) {
        if (parts == 1) lp_unused<T, NT>(a, r, lane);
        return;
    }
    // vectors v0 .. v1 of the row, and in the last part the values past them
    const int64_t cols = a.cols, ncv = cols / VN, per = (ncv + parts - 1) / parts;
    const int64_t v0 = p * per < ncv ? p * per : ncv, v1 = v0 + per < ncv ? v0 + per : ncv;
    const int nv = int(v1 - v0), rem = p == parts - 1 ? int(cols - ncv * VN) : 0;
    const T *x = a.x + r * cols;
    const T none = -T(__builtin_inf());
    V v[VPT];
#pragma unroll
    for (int k = 0; k < VPT; k++) {
#pragma unroll
        for (int j = 0; j < VN; j++) v[k][j] = none;
        if (lane + k * NT < nv) v[k] = __builtin_nontemporal_load(reinterpret_cast<const U *>(x) + v0 + lane + k * NT);
    }
    const T vt = lane < rem ? x[ncv * VN + lane] : none;
    const auto each = [&](auto f) {  // f(value, its index in the row), in order of the index
#pragma unroll
        for (int k = 0; k < VPT; k++)
#pragma unroll
            for (int j = 0; j < VN; j++) f(v[k][j], int((v0 + lane + k * NT) * VN + j));
        f(vt, int(ncv * VN + lane));
    };
    T top = none;  // the lane's largest
    each([&](T y, int) { top = sizeof(T) == 4 ? __builtin_fmaxf(top, y) : __builtin_fmax(top, y); });
    const T m = RowGrp<64>::max(top, nullptr);
    LpPart sum{double(m), 0.0, 0.0};
    const T ref = m == none ? T(0) : m;
    if constexpr (sizeof(T) == 4) {
        // exp(d / T) = 2^(d c), c = log2(e) / T in two floats: the product's rounding error and
        // the second part go into the result as a factor 1 + error ln 2.
        const double cd = a.inv_t * 1.4426950408889634;
        const float c = float(cd), c2 = float(cd - double(c)), least = -200.0f / c;  // exp(least / T) = 0
        const auto term = [&](float y, float &e, float &ed) {
            float d = y - ref;
            d = d < least ? least : d;  // (NaN stays)
            const float h = d * c, lo = __builtin_fmaf(d, c2, __builtin_fmaf(d, c, -h));
            e = __builtin_amdgcn_exp2f(h);
            e = __builtin_fmaf(e, lo * 0.693147181f, e);
            ed = e * d;
            sum.s += double(e);
        };
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            float e, q[4];
#pragma unroll
            for (int j = 0; j < 4; j++) term(v[k][j], e, q[j]);
            sum.t += double((q[0] + q[1]) + (q[2] + q[3]));
        }
        if (rem) {  // uniform
            float e, q;
            term(vt, e, q);
            sum.t += double(q);
        }
    } else {
        each([&](T y, int) {
            const double d = y - ref, e = exp(d * a.inv_t);
            sum.s += e;
            sum.t += d * a.inv_t < -2000.0 ? 0.0 : e * d;
        });
    }
    sum.s = wave_dsum(sum.s);
    sum.t = wave_dsum(sum.t);
    LpOrder<T, NT> &o = order[sub];
    if (lane == 0) o.n = 0;
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = sum;
    }
    if (a.k) {
        T left = top, bound = none;
        for (int q = 0; q < (a.k + W - 1) / W; q++) {
            bound = RowGrp<64>::max(left, nullptr);
            const uint64_t who = __ballot(left == bound);
            if (bound == none) break;
            if ((threadIdx.x & 63) == __builtin_ctzll(who)) left = none;
        }
        if (W > 1 && (threadIdx.x & 63) == 0) o.wave_v[threadIdx.x >> 6] = bound;
        lp_meet<NT>();
        if constexpr (W > 1) {
#pragma unroll
            for (int w = 0; w < W; w++) bound = o.wave_v[w] < bound ? o.wave_v[w] : bound;
        }
        const auto passes = [&](T y) { return y >= bound && y > none; };
        int mine = 0;
        each([&](T y, int) { mine += passes(y) ? 1 : 0; });
        int before = mine;  // of the wave's lanes up to this one
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int u = __shfl_up(before, off, 64);
            if (int(threadIdx.x & 63) >= off) before += u;
        }
        int at = 0;
        if ((threadIdx.x & 63) == 63) at = atomicAdd(&o.n, before);
        at = __shfl(at, 63, 64) + before - mine;
        if (mine)
            each([&](T y, int i) {
                if (passes(y)) {
                    if (at < o.kCand) {
                        o.v[at] = y;
                        o.i[at] = i;
                    }
                    at++;
                }
            });
        lp_meet<NT>();
        const int n = o.n;
        if (n <= o.kCand) {
            lp_rank<T, NT>(o, n, a.k, lane);
        } else {
            lp_rounds<T, NT>(o, a.k, lane, [&](auto f) {
                each([&](T y, int i) {
                    if (y > none) f(LpKey<T>{y, i});
                });
            });
        }
    }
    lp_meet<NT>();
    if constexpr (W > 1) sum = lp_join_all(sh, a.inv_t);
    if (parts == 1) {
        const LpRow row(sum, a.inv_t);
        if (lane == 0) lp_store(a, r, tok, row, sum.t);
        for (int q = lane; q < a.k; q += NT) lp_store_top(a, r, q, o.out[q], row);
    } else {
        if (lane == 0) scratch.part[unit] = sum;
        for (int q = lane; q < a.k; q += NT) {
            scratch.v[unit * a.k + q] = o.out[q].v;
            scratch.i[unit * a.k + q] = o.out[q].i;
        }
    }
}

// A row's parts joined, NT lanes a row.  The alternatives: the largest of the parts' k-th
// values is passed by k of all at least.
template <typename T, int NT>
__global__ __launch_bounds__(256) void k_lp_join(LpArgs<T> a, LpScratch<T> scratch, int parts, int64_t b_base)
{
    constexpr int RPB = 256 / NT, W = NT / 64;
    __shared__ LpPart sh[4];
    __shared__ T sh_b[4];
    __shared__ LpOrder<T, NT> order[1];  // (a wave a row: no alternatives)
    const int lane = threadIdx.x % NT, sub = RPB == 1 ? 0 : threadIdx.x / NT;
    const int64_t r = (b_base + int64_t(blockIdx.x)) * RPB + sub;
    if (RPB > 1 && r >= a.rows) return;
    const int64_t tok = a.tokens ? a.tokens[r] : 0;
    if (tok < 0) return lp_unused<T, NT>(a, r, lane);
    const T none = -T(__builtin_inf());
    const LpPart *part = scratch.part + r * parts;
    const T *kv = scratch.v + r * parts * a.k;
    const int *ki = scratch.i + r * parts * a.k;
    LpPart sum{-__builtin_inf(), 0.0, 0.0};
    T bound = none;
    for (int p = lane; p < parts; p += NT) {
        sum = lp_join(sum, part[p], a.inv_t);
        if (a.k) {
            const T b = kv[int64_t(p) * a.k + a.k - 1];
            bound = b > bound ? b : bound;
        }
    }
    sum = lp_join_wave(sum, a.inv_t);
    if constexpr (W > 1) {
        bound = RowGrp<64>::max(bound, nullptr);
        if ((threadIdx.x & 63) == 0) {
            sh[threadIdx.x >> 6] = sum;
            sh_b[threadIdx.x >> 6] = bound;
        }
        if (threadIdx.x == 0) order[0].n = 0;
        __syncthreads();
        sum = lp_join_all(sh, a.inv_t);
        bound = sh_b[0];
#pragma unroll
        for (int w = 1; w < W; w++) bound = sh_b[w] > bound ? sh_b[w] : bound;
    }
    const LpRow row(sum, a.inv_t);
    if (lane == 0) lp_store(a, r, tok, row, sum.t);
    if constexpr (W > 1) {
        if (!a.k) return;
        LpOrder<T, NT> &o = order[0];
        const int64_t n_all = int64_t(parts) * a.k;
        for (int64_t c = lane; c < n_all; c += NT) {
            const LpKey<T> key{kv[c], ki[c]};
            if (key.i >= 0 && key.v >= bound) {
                const int at = atomicAdd(&o.n, 1);  // (any order: they are ordered after)
                if (at < o.kCand) {
                    o.v[at] = key.v;
                    o.i[at] = key.i;
                }
            }
        }
        __syncthreads();
        const int n = o.n;
        if (n <= o.kCand) {
            lp_rank<T, NT>(o, n, a.k, lane);
        } else {
            lp_rounds<T, NT>(o, a.k, lane, [&](auto f) {
                for (int64_t c = lane; c < n_all; c += NT) f(LpKey<T>{kv[c], ki[c]});
            });
        }
        __syncthreads();
        for (int q = lane; q < a.k; q += NT) lp_store_top(a, r, q, o.out[q], row);
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

// What a row's gradient is made of; rows that are not used or have every logit masked: g = e = 0
// and zero.
struct LpGradRow {
    double lse, g, e, h;
    int64_t tok;
    bool zero;
};

template <typename T>
NH_DEV LpGradRow lp_grad_row(const LpGradArgs<T> &a, int64_t r)
{
    LpGradRow w;
    w.tok = a.tokens ? a.tokens[r] : -2;
    w.lse = double(a.lse[r]);
    w.g = a.g ? double(a.g[r]) : 0.0;
    if (a.g && w.tok >= a.cols) w.g = __builtin_nan("");
    w.e = a.e ? double(a.e[r]) : 0.0;
    w.h = a.e ? double(a.entropy[r]) : 0.0;
    w.zero = (a.tokens && w.tok < 0) || w.lse == -__builtin_inf();
    return w;
}

// log p in double, its exponential to f32 accuracy for f32 rows, the terms in double.
template <typename T>
NH_DEV T lp_grad(T x, bool at, const LpGradRow &w, double inv_t)
{
    const double lp = double(x) * inv_t - w.lse;
    double p;
    if constexpr (sizeof(T) == 4) p = double(exp_d2f(lp));
    else p = exp(lp);
    double v = w.g * ((at ? 1.0 : 0.0) - p);
    const double ent = w.e * p * (lp + w.h);
    v -= p == 0.0 ? 0.0 : ent;  // (a masked logit: 0 * -inf)
    return w.zero ? T(0) : T(v * inv_t);
}

// Rows of at least kLpFlat values (and f64 rows of half): the tensor as one run of vectors that
// begin at 128-byte lines of dx, so that stores fill whole lines whatever the rows' width (f32
// [4096, 50257], whose rows start anywhere).  A block's 1024 vectors lie in two rows at most.
constexpr int64_t kLpFlat = 4096;
template <typename T>
__global__ __launch_bounds__(256) void k_lp_grad_flat(LpGradArgs<T> a, int64_t head, int64_t b_base)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, P = 4;
    const int64_t n = a.rows * a.cols, nv = (n - head) / VN, q0 = (b_base + int64_t(blockIdx.x)) * 256 * P;
    const int64_t first = head + q0 * VN, r0 = first / a.cols;  // uniform
    V x[P];
#pragma unroll
    for (int k = 0; k < P; k++) {
        const int64_t q = q0 + threadIdx.x + k * 256;
        if (q < nv) x[k] = __builtin_nontemporal_load(reinterpret_cast<const U *>(a.x + head) + q);
    }
    const LpGradRow w0 = lp_grad_row(a, r0 < a.rows ? r0 : a.rows - 1);
    const LpGradRow w1 = lp_grad_row(a, r0 + 1 < a.rows ? r0 + 1 : a.rows - 1);
    const int64_t off = first - r0 * a.cols;
#pragma unroll
    for (int k = 0; k < P; k++) {
        const int64_t q = q0 + threadIdx.x + k * 256;
        if (q < nv) {
            const int64_t c = off + int64_t(threadIdx.x + k * 256) * VN;
            V o;
#pragma unroll
            for (int j = 0; j < VN; j++) {
                const bool next = c + j >= a.cols;
                const int64_t col = next ? c + j - a.cols : c + j;
                LpGradRow w;
                w.lse = next ? w1.lse : w0.lse;
                w.g = next ? w1.g : w0.g;
                w.e = next ? w1.e : w0.e;
                w.h = next ? w1.h : w0.h;
                w.zero = next ? w1.zero : w0.zero;
                o[j] = lp_grad(x[k][j], col == (next ? w1.tok : w0.tok), w, a.inv_t);
            }
            __builtin_nontemporal_store(o, reinterpret_cast<U *>(a.dx + head) + q);
        }
    }
    // the values before the first vector and past the last
    if (b_base + int64_t(blockIdx.x) == 0 && threadIdx.x < 64) {
        const int64_t tail = head + nv * VN;
        const int64_t i = int64_t(threadIdx.x) < head ? int64_t(threadIdx.x) : tail + threadIdx.x - head;
        if (i < n) {
            const int64_t r = i / a.cols;
            const LpGradRow w = lp_grad_row(a, r);
            a.dx[i] = lp_grad(a.x[i], i - r * a.cols == w.tok, w, a.inv_t);
        }
    }
}

// Narrower rows: NT lanes a row.
template <typename T, int NT>
__global__ __launch_bounds__(256) void k_lp_grad_row(LpGradArgs<T> a, int64_t r_base)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, RPB = 256 / NT;
    const int lane = threadIdx.x % NT, sub = RPB == 1 ? 0 : threadIdx.x / NT;
    const int64_t r = r_base + int64_t(blockIdx.x) * RPB + sub;
    if (RPB > 1 && r >= a.rows) return;
    const LpGradRow w = lp_grad_row(a, r);
    const T *x = a.x + r * a.cols;
    T *dx = a.dx + r * a.cols;
    const int ncv = int(a.cols / VN), rem = int(a.cols % VN);
    for (int q = lane; q < ncv; q += NT) {
        const V v = *(reinterpret_cast<const U *>(x) + q);
        V o;
#pragma unroll
        for (int j = 0; j < VN; j++) o[j] = lp_grad(v[j], int64_t(q) * VN + j == w.tok, w, a.inv_t);
        *(reinterpret_cast<U *>(dx) + q) = o;
    }
    if (lane < rem) {
        const int64_t c = int64_t(ncv) * VN + lane;
        dx[c] = lp_grad(x[c], c == w.tok, w, a.inv_t);
    }
}

template <typename T, int NT, int VPT>
static void launch_lp_parts(const LpArgs<T> &a, const LpScratch<T> &scratch, int parts)
{
    for_row_launches(a.rows * parts, 256 / NT, 256, [&](unsigned g, int64_t base) {
        NH_LAUNCH((k_lp_parts<T, NT, VPT>), dim3(g), dim3(256), 0, stream(), a, scratch, parts, base / (256 / NT));
    });
}

// By the width alone, so that equal rows have equal results in any batch: a wave up to 256
// vectors, a block up to 1024, and as many blocks as it takes beyond, joined by a second launch.
template <typename T>
static int launch_lp(const LpArgs<T> &a)
{
    const int64_t ncv = a.cols / Vec16<T>::n;
    const LpScratch<T> no{};
    if (ncv <= 64) launch_lp_parts<T, 64, 1>(a, no, 1);
    else if (ncv <= 128) launch_lp_parts<T, 64, 2>(a, no, 1);
    else if (ncv <= 256) launch_lp_parts<T, 64, 4>(a, no, 1);
    else if (ncv <= 512) launch_lp_parts<T, 256, 2>(a, no, 1);
    else if (ncv <= 1024) launch_lp_parts<T, 256, 4>(a, no, 1);
    else {
        const int parts = int(ceil_div(ncv, 1024));
        const size_t units = size_t(a.rows) * size_t(parts), keys = units * size_t(a.k);
        Partials block;
        NH_TRY(block.open(units * sizeof(LpPart) + keys * (sizeof(T) + sizeof(int))));
        LpScratch<T> scratch{static_cast<LpPart *>(block.p), nullptr, nullptr};
        scratch.v = reinterpret_cast<T *>(scratch.part + units);
        scratch.i = reinterpret_cast<int *>(scratch.v + keys);
        launch_lp_parts<T, 256, 4>(a, scratch, parts);
        const int rpb = a.k ? 1 : 4;
        for_row_launches(a.rows, rpb, 256, [&](unsigned g, int64_t base) {
            if (a.k) NH_LAUNCH((k_lp_join<T, 256>), dim3(g), dim3(256), 0, stream(), a, scratch, parts, base);
            else NH_LAUNCH((k_lp_join<T, 64>), dim3(g), dim3(256), 0, stream(), a, scratch, parts, base / 4);
        });
        return check_launch();
    }
    return check_launch();
}

template <typename T>
static int launch_lp_grad(const LpGradArgs<T> &a)
{
    if (a.cols * int64_t(sizeof(T)) >= kLpFlat * 4) {
        const int64_t n = a.rows * a.cols, es = int64_t(sizeof(T));
        int64_t head = int64_t(-reinterpret_cast<uintptr_t>(a.dx) & 127) / es;
        head = head < n ? head : n;
        const int64_t blocks = ceil_div((n - head) / Vec16<T>::n, 1024);
        for_row_launches(blocks > 0 ? blocks : 1, 1, 256, [&](unsigned g, int64_t base) {
            NH_LAUNCH((k_lp_grad_flat<T>), dim3(g), dim3(256), 0, stream(), a, head, base);
        });
    } else if (a.cols * int64_t(sizeof(T)) <= 4096) {
        for_row_launches(a.rows, 4, 256, [&](unsigned g, int64_t base) {
            NH_LAUNCH((k_lp_grad_row<T, 64>), dim3(g), dim3(256), 0, stream(), a, base);
        });
    } else {
        for_row_launches(a.rows, 1, 256, [&](unsigned g, int64_t base) {
            NH_LAUNCH((k_lp_grad_row<T, 256>), dim3(g), dim3(256), 0, stream(), a, base);
        });
    }
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
