// token_logprobs.hip -- log probabilities of given tokens, entropy and top alternatives of
// rows of logits, and their gradient.
//
//   z = x / temperature; with m = max x and d = x - m: s = sum exp(d / T), t = sum exp(d / T) d / T;
//   lse = m / T + log s; logprob = (x_t - m) / T - log s; entropy = log s - t / s
//   gradient: (g (1_t - p) - e p (log p + H)) / T, log p = z - lse, or (x - m) / T - log s
//
// s and t are summed in double: where one token has nearly all the probability, logprob and
// entropy are as small as the rest of s, which a sum in float would round away beside 1.
#include <cmath>
#include <limits>
#include <type_traits>

#include "row_call.hpp"
#include "row_group.hpp"

namespace nh {

constexpr int kLpMaxTop = 64;

// An alternative as one key: of two, the larger key comes first, a larger value, of equal ones (0
// and -0 too) the lower index.  A key of zero is none, behind all.
template <typename T> struct LpKey;
template <>
struct LpKey<float> {
    uint64_t k;
    NH_DEV static LpKey none() { return {0}; }
    NH_DEV static LpKey of(float v, int i)
    {
        const int b = __float_as_int(v + 0.0f);
        return {uint64_t(uint32_t(b) ^ (uint32_t(b >> 31) | 0x80000000u)) << 32 | ~uint32_t(i)};
    }
    NH_DEV bool before(const LpKey &o) const { return k > o.k; }
    NH_DEV bool any() const { return k != 0; }
    NH_DEV int index() const { return any() ? int(~uint32_t(k)) : -1; }
    NH_DEV float value() const
    {
        const uint32_t o = uint32_t(k >> 32);
        return any() ? __uint_as_float(o >> 31 ? o ^ 0x80000000u : ~o) : -__builtin_inff();
    }
    NH_DEV LpKey of_lane(int off) const { return {uint64_t(__shfl_xor((long long)(k), off, 64))}; }
};
template <>
struct LpKey<double> {
    uint64_t k;
    uint64_t i;  // ~index, 0 for none
    NH_DEV static LpKey none() { return {0, 0}; }
    NH_DEV static LpKey of(double v, int i)
    {
        const int64_t b = __double_as_longlong(v + 0.0);
        return {uint64_t(b) ^ (uint64_t(b >> 63) | 0x8000000000000000ull), ~uint32_t(i)};
    }
    NH_DEV bool before(const LpKey &o) const { return k > o.k || (k == o.k && i > o.i); }
    NH_DEV bool any() const { return i != 0; }
    NH_DEV int index() const { return any() ? int(~uint32_t(i)) : -1; }
    NH_DEV double value() const
    {
        return any() ? __longlong_as_double(int64_t(k >> 63 ? k ^ 0x8000000000000000ull : ~k)) : -__builtin_inf();
    }
    NH_DEV LpKey of_lane(int off) const
    {
        return {uint64_t(__shfl_xor((long long)(k), off, 64)), uint64_t(__shfl_xor((long long)(i), off, 64))};
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
    bool four;  // lse holds four values a row: lse, m, log s, entropy
    double inv_t;
};

// What a part of a row leaves: its largest value m, s = sum exp((x - m) / T) and t = sum
// exp((x - m) / T) (x - m).
struct LpPart {
    double m, s, t;
};

// A part's t moved by d, times f = exp(d / T).  Where f is 0 nothing of it is left, but d s may lie past
// double's range (logits at its lowest value as masks).  NaN stays.
NH_DEV double lp_moved(const LpPart &p, double d, double f)
{
    return f == 0.0 ? f * p.t : f * (p.t + d * p.s);
}

// The sums of two parts by the larger m.  A part without values (m -inf) has s = t = 0, or NaN
// where it holds NaN, which stays.
NH_DEV LpPart lp_join(const LpPart &a, const LpPart &b, double inv_t)
{
    const double none = -__builtin_inf(), m = __builtin_fmax(a.m, b.m);
    const double da = a.m == none ? 0.0 : a.m - m, db = b.m == none ? 0.0 : b.m - m;
    const double fa = a.m == none ? 0.0 : exp(da * inv_t), fb = b.m == none ? 0.0 : exp(db * inv_t);
    return {m, a.s * fa + b.s * fb, lp_moved(a, da, fa) + lp_moved(b, db, fb)};
}

// The same over a wave's lanes: one exponential for each.
NH_DEV LpPart lp_join_wave(const LpPart &p, double inv_t)
{
    const double m = RowGrp<64>::max(p.m, nullptr);
    const bool any = p.m != -__builtin_inf();
    const double d = any ? p.m - m : 0.0, f = any ? exp(d * inv_t) : 0.0;
    return {m, wave_dsum(p.s * f), wave_dsum(lp_moved(p, d, f))};
}

// A row's results from its sums.
struct LpRow {
    double m, inv_t, s, ls;  // m: 0 where every logit is masked
    NH_DEV static LpRow of(const LpPart &p, double it)
    {
        return {p.m == -__builtin_inf() ? 0.0 : p.m, it, p.s, log(p.s)};
    }
    NH_DEV bool sound() const { return s == s; }
    // (halves: the difference of two f64 logits may pass double's range where that over T does not)
    NH_DEV double logprob(double x) const
    {
        return s == 0.0 ? -__builtin_inf() : (0.5 * x - 0.5 * m) * (2.0 * inv_t) - ls;
    }
    NH_DEV double lse() const { return m * inv_t + ls; }
    NH_DEV double entropy(double t) const { return s == 0.0 ? 0.0 : ls - t * inv_t / s; }
};

template <typename T>
NH_DEV T lp_logit(const LpArgs<T> &a, int64_t r, int64_t tok)
{
    return a.logprob && tok < a.cols ? a.x[r * a.cols + tok] : T(0);
}
template <typename T>
NH_DEV void lp_store(const LpArgs<T> &a, int64_t r, int64_t tok, T logit, const LpRow &row, double t)
{
    if (a.logprob) a.logprob[r] = tok < a.cols ? T(row.logprob(double(logit))) : T(__builtin_nan(""));
    if (a.entropy) a.entropy[r] = T(row.entropy(t));
    if (a.lse && a.four) {
        const T v[4] = {T(row.lse()), T(row.m), T(row.ls), T(row.entropy(t))};
#pragma unroll
        for (int q = 0; q < 4; q++) a.lse[4 * r + q] = v[q];
    } else if (a.lse) {
        a.lse[r] = T(row.lse());
    }
}
template <typename T>
NH_DEV void lp_store_top(const LpArgs<T> &a, int64_t r, int q, const LpKey<T> &k, const LpRow &row)
{
    if (a.top_ids) a.top_ids[r * a.k + q] = row.sound() ? int64_t(k.index()) : -1;
    if (a.top_lp)
        a.top_lp[r * a.k + q] = !row.sound() ? T(__builtin_nan("")) : k.any() ? T(row.logprob(double(k.value()))) : -T(__builtin_inf());
}
// A row that is not used, by a group of NT lanes.
template <typename T, int NT>
NH_DEV void lp_unused(const LpArgs<T> &a, int64_t r, int lane)
{
    if (lane == 0) {
        if (a.logprob) a.logprob[r] = T(0);
        if (a.entropy) a.entropy[r] = T(0);
        if (a.lse)
            for (int q = 0; q < (a.four ? 4 : 1); q++) a.lse[(a.four ? 4 : 1) * r + q] = T(0);
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

// The wave's largest value, NaN passed over, the same in every lane: sixteen lanes by four moves,
// then one of each sixteen.
NH_DEV float lp_wave_top(float v)
{
    v = __builtin_fmaxf(v, dpp_f<kDppXor1>(v));
    v = __builtin_fmaxf(v, dpp_f<kDppXor2>(v));
    v = __builtin_fmaxf(v, dpp_f<kDppHalfMirror>(v));
    v = __builtin_fmaxf(v, dpp_f<kDppMirror>(v));
    const auto of = [&](int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); };
    return __builtin_fmaxf(__builtin_fmaxf(of(0), of(16)), __builtin_fmaxf(of(32), of(48)));
}
NH_DEV double lp_wave_top(double v) { return RowGrp<64>::max(v, nullptr); }

// LDS of a group that orders alternatives: a list of candidates for each of its waves.
template <typename T, int NT>
struct LpOrder {
    static constexpr int W = NT / 64, kCand = 256;
    alignas(16) LpKey<T> key[W][kCand + 2];
    alignas(16) int n[W];
    T wave_v[W];
    LpKey<T> wave_key[W], out[kLpMaxTop];
};

// Whether every wave's candidates fit its list.
template <typename T, int NT>
NH_DEV bool lp_fits(const LpOrder<T, NT> &o)
{
    bool fits = true;
#pragma unroll
    for (int u = 0; u < NT / 64; u++) fits &= o.n[u] <= o.kCand;
    return fits;
}

// The k first of the waves' lists (n[w] <= kCand, all apart) into out: a candidate's place is the
// number of those before it.  Each wave places its own, four lanes to a candidate, which share
// the lists.
template <typename T, int NT>
NH_DEV void lp_rank(LpOrder<T, NT> &o, int k, int lane)
{
    constexpr int W = NT / 64, STEP = W == 1 ? 8 : 2;
    const int w = W == 1 ? 0 : lane >> 6, quad = lane & 3, list = W == 1 ? 0 : quad;
    int total = 0;
#pragma unroll
    for (int u = 0; u < W; u++) total += o.n[u];
    for (int q = total + lane; q < k; q += NT) o.out[q] = LpKey<T>::none();
    const int n = o.n[list], own = o.n[w];
    for (int c0 = 0; c0 < own; c0 += 16) {
        const int c = c0 + ((lane & 63) >> 2);
        const LpKey<T> mine = o.key[w][c < own ? c : own];
        int place = 0;
#pragma unroll 4
        for (int j = W == 1 ? 2 * quad : 0; j < n; j += STEP) {
            struct alignas(16) {
                LpKey<T> k[2];
            } pair;
            pair.k[0] = o.key[list][j];
            pair.k[1] = o.key[list][j + 1];
            place += pair.k[0].before(mine) ? 1 : 0;
            place += pair.k[1].before(mine) ? 1 : 0;
        }
        place += dpp_i<kDppXor1>(place);
        place += dpp_i<kDppXor2>(place);
        if (quad == 0 && c < own && place < k) o.out[place] = mine;
    }
}

// The k first keys by k rounds of the group's best key behind the one found before: for rows
// whose values crowd at the bound (each(f): f(value, index) for every key of a lane).
template <typename T, int NT, typename E>
NH_DEV void lp_rounds(LpOrder<T, NT> &o, int k, int lane, const E &each)
{
    LpKey<T> last = LpKey<T>::none();
    for (int q = 0; q < k; q++) {
        LpKey<T> best = LpKey<T>::none();
        each([&](T v, int i) {
            const LpKey<T> c = LpKey<T>::of(v, i);
            if (v > -T(__builtin_inf()) && (q == 0 || last.before(c)) && c.before(best)) best = c;
        });
        if (q > 0 && !last.any()) best = LpKey<T>::none();
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) {
            const LpKey<T> u = best.of_lane(off);
            if (u.before(best)) best = u;
        }
        if constexpr (NT > 64) {
            __syncthreads();
            if ((lane & 63) == 0) o.wave_key[lane >> 6] = best;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NT / 64; w++)
                if (o.wave_key[w].before(best)) best = o.wave_key[w];
        }
        last = best;
        if (lane == 0) o.out[q] = best;
    }
}

// The k first of a group's keys into o.out.  pop(true) gives the lane's largest value that was not
// taken yet, of those that stand for its keys, pop(false) looks at it.  With j = k / waves rounded
// up, the j-th of them over a wave, and the least of that over the waves, is passed by k keys at
// least; what passes it (some 2 k where values are in no order) each wave collects, lane by lane
// (emit(least, f): f(value, index) for the lane's keys from least on), and it is ordered by counting.
// What bounds it is one wave's latency, some 7 cycles an instruction.
template <typename T, int NT, typename P, typename C, typename E>
NH_DEV void lp_select(LpOrder<T, NT> &o, int k, int lane, P pop, C emit, const E &each)
{
    constexpr int W = NT / 64;
    const int w = W == 1 ? 0 : lane >> 6, wl = lane & 63;
    const T none = -T(__builtin_inf());
    T left = pop(false), bound = none;
    for (int q = 1;; q++) {
        bound = lp_wave_top(left);
        if (q * W >= k || bound == none) break;
        const uint64_t who = __ballot(left == bound);
        if (wl == int(__builtin_ctzll(who))) left = pop(true);
    }
    if constexpr (W > 1) {
        if (wl == 0) o.wave_v[w] = bound;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < W; u++) bound = o.wave_v[u] < bound ? o.wave_v[u] : bound;
    }
    const T least = bound == none ? -std::numeric_limits<T>::max() : bound;
    int own = 0, at = 0, n = 0;  // the lane's, those of the lanes before, the wave's
    each([&](T y, int) { own += y >= least ? 1 : 0; });
    for (int b = 0; __ballot(own >> b); b++) {
        const uint64_t who = __ballot(own >> b & 1);
        at += int(__builtin_amdgcn_mbcnt_hi(uint32_t(who >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(who), 0))) << b;
        n += int(__builtin_popcountll(who)) << b;
    }
    if (n <= o.kCand) emit(least, [&](T y, int i) { o.key[w][at++] = LpKey<T>::of(y, i); });
    if (wl == 0) o.n[w] = n;
    if (wl < 2 && n <= o.kCand) o.key[w][n + wl] = LpKey<T>::none();
    lp_meet<NT>();
    if (lp_fits(o)) lp_rank<T, NT>(o, k, lane);
    else lp_rounds<T, NT>(o, k, lane, each);
    lp_meet<NT>();
}

// What the other waves of a block do meanwhile: they meet as often.  first() runs beside the lists'
// making, then() beside their ordering.
template <typename T, int NT, typename F, typename G>
NH_DEV void lp_beside(const LpOrder<T, NT> &o, int k, const F &first, const G &then)
{
    __syncthreads();  // the bounds
    first();
    __syncthreads();  // the lists
    then();
    if (!lp_fits(o))
        for (int q = 0; q < k; q++) {  // lp_rounds
            __syncthreads();
            __syncthreads();
        }
    __syncthreads();  // the order
}

// Where a row is split: its waves' sums, [rows][parts][4], and its parts' alternatives,
// [rows][parts][k].
template <typename T>
struct LpScratch {
    LpPart *sums;
    LpKey<T> *keys;
};

// Sums alone, alternatives by the waves that sum, or by as many others beside them.
enum { LP_SUMS = 0, LP_TOP = 1, LP_TOP_BESIDE = 2 };
constexpr int lp_lanes(int nt, int mode) { return mode == LP_TOP_BESIDE ? 2 * nt : nt < 256 ? 256 : nt; }

// A row is cut into parts of 256 lanes, `per` vectors at most, VPT a lane, or of a wave where it is
// narrow; a group of NT lanes holds one part in registers: one read.  Each wave takes its own
// largest value as the reference of its exponentials.
// r_base: the launch's first row.  What bounds it where rows are many: the vector units, with HBM
// close behind (f32: about 16 issue slots a value; [4096, 50257] 140 us, a copy's rate 137); with
// alternatives the latency of ordering them (k = 1: 212 us, 20: 256, 64: 383; with four waves a
// SIMD, for which nine registers were spilled, 231, 257 and 347).  f64, an exponential in double a
// value: [2048, 50257] 159 us (a copy's rate 133), k = 20 252.
template <typename T, int NT, int VPT, int MODE>
__global__ __launch_bounds__(lp_lanes(NT, MODE), (MODE == LP_SUMS ? 1 : 3)) void k_lp_parts(
    LpArgs<T> a, LpScratch<T> scratch, int parts, int64_t per, int64_t r_base)
{
    constexpr bool TOP = MODE != LP_SUMS, TWO = MODE == LP_TOP_BESIDE;
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, RPB = 256 / NT, W = NT / 64;
    __shared__ LpPart sh[W];
    __shared__ LpRow row_of;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool sums = !TWO || wave < W, tops = TOP && (!TWO || wave >= W);
    const int lane = threadIdx.x % NT, sub = RPB == 1 ? 0 : threadIdx.x / NT;
    const int rl = RPB > 1 ? int(blockIdx.x) * RPB + sub : int(blockIdx.x / unsigned(parts));
    const int p = RPB > 1 ? 0 : int(blockIdx.x) - rl * parts;
    const int64_t r = r_base + rl;
    if (RPB > 1 && r >= a.rows) return;
    const int64_t tok = a.tokens ? a.tokens[r] : 0;
    if (tok < 0) {
        if (parts == 1 && sums) lp_unused<T, NT>(a, r, lane);
        return;
    }
    // vectors v0 .. of the row, and in the last part the values past them
    const int64_t cols = a.cols, ncv = cols / VN, v0 = p * per < ncv ? p * per : ncv;
    const int nv = int(ncv - v0 < per ? ncv - v0 : per), rem = p == parts - 1 ? int(cols - ncv * VN) : 0;
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
    const int first = int((v0 + lane) * VN);
    const auto each = [&](auto f) {  // f(value, its index in the row)
#pragma unroll
        for (int k = 0; k < VPT; k++)
#pragma unroll
            for (int j = 0; j < VN; j++) f(v[k][j], first + k * NT * VN + j);
        if (rem) f(vt, int(ncv * VN) + lane);
    };
    const auto most = [](T y, T z) {
        if constexpr (sizeof(T) == 4) return __builtin_fmaxf(y, z);
        else return __builtin_fmax(y, z);
    };
    T top = vt, vmax[VPT];  // the lane's largest, and each vector's
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        vmax[k] = v[k][0];
#pragma unroll
        for (int j = 1; j < VN; j++) vmax[k] = most(vmax[k], v[k][j]);
        top = most(top, vmax[k]);
    }
    LpPart sum;
    const auto add = [&] {
        const T m = RowGrp<64>::max(top, nullptr);
        sum = {double(m), 0.0, 0.0};
        const T ref = m == none ? T(0) : m;
        if constexpr (sizeof(T) == 4) {
            // exp(d / T) = 2^(d c), c = log2(e) / T in two floats: the product's rounding error and
            // the second part go into the result as a factor 1 + error ln 2.  Four values are added
            // in float, except where one of them is the largest, whose 1 would swallow the others.
            const double cd = a.inv_t * 1.4426950408889634;
            const float c = float(cd), c2 = float(cd - double(c));
            const float least = float(-200.0 * 0.6931471805599453 / a.inv_t);  // exp(least / T) = 0
            const auto term = [&](float y, float &ed) {
                float d = y - ref;
                d = d < least ? least : d;  // (NaN stays)
                const float h = d * c, lo = __builtin_fmaf(d, c2, __builtin_fmaf(d, c, -h));
                float e = __builtin_amdgcn_exp2f(h);
                e = __builtin_fmaf(e, lo * 0.693147181f, e);
                ed = e * d;
                return e;
            };
#pragma unroll
            for (int k = 0; k < VPT; k++) {
                float e[4], q[4];
#pragma unroll
                for (int j = 0; j < 4; j++) e[j] = term(v[k][j], q[j]);
                sum.t += double((q[0] + q[1]) + (q[2] + q[3]));
                if (__ballot(vmax[k] == m)) sum.s += (double(e[0]) + double(e[1])) + (double(e[2]) + double(e[3]));
                else sum.s += double((e[0] + e[1]) + (e[2] + e[3]));
            }
            if (rem) {  // uniform
                float q;
                sum.s += double(term(vt, q));
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
    };
    if (!TWO) add();
    __shared__ LpOrder<T, NT> order[TOP ? RPB : 1];
    const auto finish = [&] {  // a row of one part, by the first wave that sums
        if constexpr (W > 1) sum = lp_join_wave(lane < W ? sh[lane < W ? lane : 0] : LpPart{-__builtin_inf(), 0.0, 0.0}, a.inv_t);
        const LpRow row = LpRow::of(sum, a.inv_t);
        if (lane == 0) lp_store(a, r, tok, lp_logit(a, r, tok), row, sum.t);
        return row;
    };
    const auto leave = [&] {  // a wave's sums
        if ((threadIdx.x & 63) == 0) (parts == 1 ? sh : scratch.sums + (r * parts + p) * W)[wave % W] = sum;
    };
    if constexpr (TOP) if (tops) {
        // Alternatives of a wave that are many for its lanes: its vectors stand for their values,
        // not its lanes (64 rows of 1000, k = 64: 20 us, by lanes 53, as too much passes the bound;
        // k = 40: 13 both; k = 24: 9.7 and 8.7).
        const bool fine = NT == 64 && a.k > 40;
        T over = top, scalar = vt;
        T over_v[VPT];
#pragma unroll
        for (int k = 0; k < VPT; k++) over_v[k] = vmax[k];
        const auto pop = [&](bool next) {
            if (next) {
                if (fine) {
                    bool gone = false;
#pragma unroll
                    for (int k = 0; k < VPT; k++) {
                        const bool it = !gone && over_v[k] == over;
                        over_v[k] = it ? none : over_v[k];
                        gone |= it;
                    }
                    scalar = gone ? scalar : none;
                    over = scalar;
#pragma unroll
                    for (int k = 0; k < VPT; k++) over = most(over, over_v[k]);
                } else {
                    over = none;
                }
            }
            return over;
        };
        const auto emit = [&](T least, auto f) {
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (vmax[k] >= least) {
#pragma unroll
                    for (int j = 0; j < VN; j++)
                        if (v[k][j] >= least) f(v[k][j], first + k * NT * VN + j);
                }
            if (vt >= least) f(vt, int(ncv * VN) + lane);
        };
        lp_select<T, NT>(order[sub], a.k, lane, pop, emit, each);
    }
    const LpOrder<T, NT> &o = order[TOP ? sub : 0];
    if constexpr (TWO) {
        if (sums)
            lp_beside<T, NT>(
                o, a.k,
                [&] {
                    add();
                    leave();
                },
                [&] {
                    if (parts == 1 && wave == 0) {
                        const LpRow row = finish();
                        if (lane == 0) row_of = row;
                    }
                });
        if (tops && parts == 1)
            for (int q = lane; q < a.k; q += NT) lp_store_top(a, r, q, o.out[q], row_of);
    } else if (W > 1 || parts > 1) {
        leave();
    }
    if (parts > 1) {
        if (tops)
            for (int q = lane; q < a.k; q += NT) scratch.keys[(r * parts + p) * a.k + q] = o.out[q];
        return;
    }
    if constexpr (!TWO) {
        if constexpr (W > 1) __syncthreads();
        if (W > 1 && wave > 0) return;
        const LpRow row = finish();
        if constexpr (TOP)
            for (int q = lane; q < a.k; q += NT) lp_store_top(a, r, q, o.out[q], row);
    }
}

// A row's parts joined: NT lanes a row, a wave where no alternatives are asked for.  What the
// parts left comes from the other dies' caches: all of it is asked for first.
template <typename T, int NT>
__global__ __launch_bounds__(NT == 64 ? 256 : NT + 64) void k_lp_join(LpArgs<T> a, LpScratch<T> scratch, int parts, int64_t b_base)
{
    constexpr int RPB = 256 / NT, HELD = NT == 64 ? 1 : 4;
    const bool tops = NT > 64 && threadIdx.x < NT;  // NT > 64: the last wave joins the sums beside
    const int lane = threadIdx.x % NT, sub = RPB == 1 ? 0 : threadIdx.x / NT;
    const int64_t r = (b_base + int64_t(blockIdx.x)) * RPB + sub;
    if (RPB > 1 && r >= a.rows) return;
    const LpPart empty{-__builtin_inf(), 0.0, 0.0};
    const LpPart *sums = scratch.sums + r * parts * 4;
    LpPart sum = !tops && lane < parts * 4 ? sums[lane] : empty;
    const int64_t n = int64_t(parts) * a.k;
    const LpKey<T> *keys = scratch.keys + r * n;
    const int turn = (lane & 63) * (NT / 64) + lane / 64;  // few keys go to all waves
    LpKey<T> held[HELD];                                  // the first of a lane's keys
    if (tops) {
#pragma unroll
        for (int q = 0; q < HELD; q++) held[q] = turn + q * NT < n ? keys[turn + q * NT] : LpKey<T>::none();
    }
    const int64_t tok = a.tokens ? a.tokens[r] : 0;
    if (tok < 0) {
        if (NT == 64 || tops) lp_unused<T, NT>(a, r, lane);
        return;
    }
    const auto join = [&] {  // one wave, in one order
        const T logit = lp_logit(a, r, tok);
        for (int p = lane + 64; p < parts * 4; p += 64) sum = lp_join(sum, sums[p], a.inv_t);
        sum = lp_join_wave(sum, a.inv_t);
        const LpRow row = LpRow::of(sum, a.inv_t);
        if (lane == 0) lp_store(a, r, tok, logit, row, sum.t);
        return row;
    };
    if constexpr (NT == 64) {
        join();
    } else {
        __shared__ LpRow row_of;
        __shared__ LpOrder<T, NT> o;
        if (!tops) {
            lp_beside<T, NT>(
                o, a.k,
                [&] {
                    const LpRow row = join();
                    if (lane == 0) row_of = row;
                },
                [] {});
            return;
        }
        const auto each = [&](auto f) {
#pragma unroll
            for (int q = 0; q < HELD; q++)
                if (turn + q * NT < n) f(held[q].value(), held[q].index());
            for (int64_t c = turn + HELD * NT; c < n; c += NT) f(keys[c].value(), keys[c].index());
        };
        const T none = -T(__builtin_inf());
        T top = none;  // (a place without a value holds none)
        each([&](T y, int) { top = y > top ? y : top; });
        const auto pop = [&](bool next) {
            if (next) top = none;  // a lane's keys by their largest alone
            return top;
        };
        const auto emit = [&](T least, auto f) {
            each([&](T y, int i) {
                if (y >= least) f(y, i);
            });
        };
        lp_select<T, NT>(o, a.k, lane, pop, emit, each);
        for (int q = lane; q < a.k; q += NT) lp_store_top(a, r, q, o.out[q], row_of);
    }
}

template <typename T>
struct LpGradArgs {
    const T *x, *g, *e, *lse, *entropy;  // g, e, entropy: may be null
    const int64_t *tokens;               // or null
    T *dx;
    int64_t rows, cols;
    bool four;  // lse holds four values a row
    double inv_t;
};

// Where |lse| is below this, log p = x / T - lse from the saved lse: its rounding to f32 leaves at most
// 2^-19 of p.  Beyond it the rounding grows with |lse|, which low temperatures and large logits make as
// large as any number (past f32's range at T = 1e-10): such rows take (x - m) / T - log s, from the four
// values that the forward call left of them, or are summed anew.
constexpr double kLpNear = 64.0;

// What a row's gradient is made of: dx = -p (g + e (log p + H)) / T, and + g / T at the token.
// f32 rows: log2 p = x a + b in double, its exponential to f32's accuracy; f64 rows: log p.  p = 0
// (a masked logit) leaves 0: log p is held above -inf.
template <typename T>
struct LpGradRow {
    static constexpr double L = sizeof(T) == 4 ? 1.4426950408889634 : 1.0;
    double a, b, ref, g, e, h;
    int64_t tok;
    bool zero;  // a row that is not used, or with every logit masked
    bool far;   // lp_far_row's: whether all logits are masked, too, shows there
    NH_DEV LpGradRow(const LpGradArgs<T> &q, int64_t r)
    {
        tok = q.tokens ? q.tokens[r] : -2;
        const T *saved = q.lse + (q.four ? 4 * r : r);
        const double lse = double(saved[0]);
        a = q.inv_t * L;
        b = -lse * L;
        ref = 0.0;
        g = q.g ? double(q.g[r]) * q.inv_t : 0.0;
        if (q.g && tok >= q.cols) g = __builtin_nan("");
        e = q.e ? double(q.e[r]) * q.inv_t : 0.0;
        h = q.e ? double(q.four ? saved[3] : q.entropy[r]) : 0.0;
        zero = q.tokens && tok < 0;
        far = !zero && __builtin_fabs(lse) >= kLpNear;
        if (far && q.four) {
            far = false;
            const double ls = double(saved[2]);
            ref = double(saved[1]);
            b = -ls * L;
            zero = ls == -__builtin_inf();
        }
    }
    // p of its logarithm t (base 2 for f32 rows); lp: log p.
    NH_DEV static double prob(double t, double &lp)
    {
        if constexpr (sizeof(T) == 4) {
            t = t < -300.0 ? -300.0 : t;
            const double n = __builtin_rint(t);
            lp = t * 0.6931471805599453;
            return double(__builtin_ldexpf(__builtin_amdgcn_exp2f(float(t - n)), int(n)));
        } else {
            lp = t < -2000.0 ? -2000.0 : t;
            return exp(lp);
        }
    }
    NH_DEV T operator()(T x, bool at) const
    {
        double lp;
        const double p = prob(__builtin_fma(double(x) - ref, a, b), lp);
        const double v = -p * __builtin_fma(e, lp + h, g);
        return zero ? T(0) : T(at ? v + g : v);
    }
};

// A far row by NT lanes in two walks, UN vectors a lane in flight: its sums, s = sum exp((x - m) / T)
// by the lane's largest logit m so far (factors in double where it rises, so that they add no error),
// then the gradient of log p = (x - m) / T - log s.  One group does the whole row, as dx may be the
// logits.
template <typename T, int NT>
NH_DEV void lp_far_row(const LpGradArgs<T> &q, LpGradRow<T> w, int64_t r, int lane)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    using G = RowGrp<NT>;
    constexpr int VN = Vec16<T>::n, UN = 4;
    __shared__ double lds[2][G::kWaves];
    const U *x = reinterpret_cast<const U *>(q.x + r * q.cols);
    U *dx = reinterpret_cast<U *>(q.dx + r * q.cols);
    const int ncv = int(q.cols / VN), rem = int(q.cols % VN);
    const int64_t c = int64_t(ncv) * VN + lane;  // the value past the vectors
    const T none = -T(__builtin_inf());
    const T xt = lane < rem ? q.x[r * q.cols + c] : none;
    T m = none;
    double s = 0.0, lp;
    for (int k0 = lane; k0 < ncv + NT; k0 += UN * NT) {  // (NT more: a turn at least, for xt)
        V v[UN];
        T top = k0 == lane ? xt : none;
#pragma unroll
        for (int u = 0; u < UN; u++) {
#pragma unroll
            for (int j = 0; j < VN; j++) v[u][j] = none;
            if (k0 + u * NT < ncv) v[u] = x[k0 + u * NT];
        }
#pragma unroll
        for (int u = 0; u < UN; u++)
#pragma unroll
            for (int j = 0; j < VN; j++) top = v[u][j] > top ? v[u][j] : top;
        if (top > m) {
            if (m != none) s *= exp((double(m) - double(top)) * q.inv_t);
            m = top;
        }
        if (m == none) continue;
        const auto term = [&](T y) { s += w.prob((double(y) - double(m)) * w.a, lp); };
#pragma unroll
        for (int u = 0; u < UN; u++)
#pragma unroll
            for (int j = 0; j < VN; j++) term(v[u][j]);
        if (k0 == lane) term(xt);
    }
    if constexpr (NT > 64) __syncthreads();  // (a block may have two such rows)
    const double most = G::max(double(m), lds[0]);
    w.zero = most == -__builtin_inf();
    s = G::sum(m == none ? 0.0 : s * exp((double(m) - most) * q.inv_t), lds[1]);
    w.ref = w.zero ? 0.0 : most;
    w.b = -log(s) * w.L;
    for (int k0 = lane; k0 < ncv; k0 += UN * NT) {
        V v[UN];
#pragma unroll
        for (int u = 0; u < UN; u++)
            if (k0 + u * NT < ncv) v[u] = x[k0 + u * NT];
#pragma unroll
        for (int u = 0; u < UN; u++)
            if (k0 + u * NT < ncv) {
                V o;
#pragma unroll
                for (int j = 0; j < VN; j++) o[j] = w(v[u][j], int64_t(k0 + u * NT) * VN + j == w.tok);
                dx[k0 + u * NT] = o;
            }
    }
    if (lane < rem) q.dx[r * q.cols + c] = w(xt, c == w.tok);
}

// Rows of at least kLpFlat f32 values (f64: half): the tensor as one run of vectors that begin at
// 128-byte lines of dx, so that stores fill whole lines whatever the rows' width (f32 [4096, 50257],
// whose rows start anywhere: 268 us, a copy of as many bytes 276; with all rows far 498, 267 from four
// values; one far row of 131072 70 us and 4.1).  A block's 1024 vectors lie in two rows at most, mostly
// in one: its numbers are the same for the block then, and nothing is read for a row that is not used.
// f64 [2048, 50257] 268 us (a copy 272).
constexpr int64_t kLpFlat = 4096;
template <typename T>
__global__ __launch_bounds__(256) void k_lp_grad_flat(LpGradArgs<T> a, int64_t head, int64_t b_base)
{
    using V = typename Vec16<T>::type;
    using U = typename VecU<T>::type;
    constexpr int VN = Vec16<T>::n, P = 4;
    const int64_t n = a.rows * a.cols, nv = (n - head) / VN, q0 = (b_base + int64_t(blockIdx.x)) * 256 * P;
    const int64_t first = head + q0 * VN, r0 = first / a.cols, off = first - r0 * a.cols;  // uniform
    const U *x = reinterpret_cast<const U *>(a.x + head) + q0;
    U *dx = reinterpret_cast<U *>(a.dx + head) + q0;
    const int left = nv - q0 < 256 * P ? int(nv - q0) : 256 * P, lane = threadIdx.x;
    if (r0 < a.rows) {
        const LpGradRow<T> w0(a, r0);
        const bool one = off + 256 * P * VN <= a.cols;
        if (one && !w0.far) {
            const int64_t at = w0.tok - off;  // the token, from the block's first value
            V v[P];
            if (!w0.zero) {
#pragma unroll
                for (int k = 0; k < P; k++)
                    if (lane + k * 256 < left) v[k] = __builtin_nontemporal_load(x + lane + k * 256);
            }
#pragma unroll
            for (int k = 0; k < P; k++)
                if (lane + k * 256 < left) {
                    V o;
#pragma unroll
                    for (int j = 0; j < VN; j++) o[j] = w0.zero ? T(0) : w0(v[k][j], false);
                    if (at / VN == lane + k * 256 && at >= 0 && !w0.zero) {
#pragma unroll
                        for (int j = 0; j < VN; j++)
                            if (j == at % VN) o[j] = w0(v[k][j], true);
                    }
                    __builtin_nontemporal_store(o, dx + lane + k * 256);
                }
        } else if (!one) {
            const LpGradRow<T> w1(a, r0 + 1 < a.rows ? r0 + 1 : r0);
#pragma unroll
            for (int k = 0; k < P; k++)
                if (lane + k * 256 < left) {
                    const int64_t c = off + int64_t(lane + k * 256) * VN;
                    if (!w0.far && !w1.far) {
                        const V v = __builtin_nontemporal_load(x + lane + k * 256);
                        V o;
#pragma unroll
                        for (int j = 0; j < VN; j++)
                            o[j] = c + j < a.cols ? w0(v[j], c + j == w0.tok) : w1(v[j], c + j - a.cols == w1.tok);
                        __builtin_nontemporal_store(o, dx + lane + k * 256);
                    } else {  // the values of the row that is not far
                        const T *xs = reinterpret_cast<const T *>(x + lane + k * 256);
                        T *dxs = reinterpret_cast<T *>(dx + lane + k * 256);
                        for (int j = 0; j < VN; j++) {
                            const bool second = c + j >= a.cols;
                            if (second ? w1.far : w0.far) continue;
                            dxs[j] = second ? w1(xs[j], c + j - a.cols == w1.tok) : w0(xs[j], c + j == w0.tok);
                        }
                    }
                }
            if (w1.far && r0 + 1 < a.rows) lp_far_row<T, 256>(a, w1, r0 + 1, lane);
        }
        // a far row is the block's in which it begins (row 0: the first's)
        if (w0.far && (off == 0 || first == head)) lp_far_row<T, 256>(a, w0, r0, lane);
    }
    // the values before the first vector and past the last
    if (b_base + int64_t(blockIdx.x) == 0 && threadIdx.x < 64) {
        const int64_t tail = head + nv * VN;
        const int64_t i = int64_t(threadIdx.x) < head ? int64_t(threadIdx.x) : tail + threadIdx.x - head;
        if (i < n) {
            const int64_t r = i / a.cols;
            const LpGradRow<T> w(a, r);
            if (!w.far) a.dx[i] = w(a.x[i], i - r * a.cols == w.tok);
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
    const LpGradRow<T> w(a, r);
    if (w.far) {
        lp_far_row<T, NT>(a, w, r, lane);
        return;
    }
    const T *x = a.x + r * a.cols;
    T *dx = a.dx + r * a.cols;
    const int ncv = int(a.cols / VN), rem = int(a.cols % VN);
    for (int q = lane; q < ncv; q += NT) {
        const V v = *(reinterpret_cast<const U *>(x) + q);
        V o;
#pragma unroll
        for (int j = 0; j < VN; j++) o[j] = w(v[j], int64_t(q) * VN + j == w.tok);
        *(reinterpret_cast<U *>(dx) + q) = o;
    }
    if (lane < rem) {
        const int64_t c = int64_t(ncv) * VN + lane;
        dx[c] = w(x[c], c == w.tok);
    }
}

// Where there are no more blocks than CUs other waves find the alternatives, with the same result
// ([1, 8192], k = 20: 5.8 us, 7.4 by the waves that sum; [64, 32000] 11.8, 13.2); with more the waves
// are missed ([512, 32000] 50 us, 29).
template <typename T, int NT, int VPT>
static void launch_lp_parts(const LpArgs<T> &a, const LpScratch<T> &scratch, int parts, int64_t per)
{
    const int64_t rpb = NT < 256 ? 256 / NT : 1, most = kMaxGridBlocks / 2 / parts * rpb;  // rows a launch
    for (int64_t base = 0; base < a.rows; base += most) {
        const int64_t n = a.rows - base < most ? a.rows - base : most;
        const dim3 grid(unsigned(ceil_div(n, rpb) * parts));
        const auto go = [&](auto kernel, int mode) {
            NH_LAUNCH(kernel, grid, dim3(unsigned(lp_lanes(NT, mode))), 0, stream(), a, scratch, parts, per, base);
        };
        if constexpr (NT > 64) {
            if (a.k && int(grid.x) <= num_cus()) {
                go(k_lp_parts<T, NT, VPT, LP_TOP_BESIDE>, LP_TOP_BESIDE);
                continue;
            }
        }
        if (a.k) go(k_lp_parts<T, NT, VPT, LP_TOP>, LP_TOP);
        else go(k_lp_parts<T, NT, VPT, LP_SUMS>, LP_SUMS);
    }
}

// By the width alone, so that equal rows have equal results in any batch: a wave up to 256
// vectors, 256 lanes up to 2048, and beyond parts of that by blocks of their own, joined by a second
// launch (one block of 1024 for four parts: [64, 32000] with one alternative 22.9 us, where two
// launches then took 13.5; now 9.8).
template <typename T>
static int launch_lp(const LpArgs<T> &a)
{
    const int64_t ncv = a.cols / Vec16<T>::n;
    const LpScratch<T> no{};
    const int parts = int(ceil_div(ncv, 2048));
    const int64_t per = parts ? ceil_div(ncv, parts) : 0;
    if (ncv <= 64) launch_lp_parts<T, 64, 1>(a, no, 1, 64);
    else if (ncv <= 128) launch_lp_parts<T, 64, 2>(a, no, 1, 128);
    else if (ncv <= 256) launch_lp_parts<T, 64, 4>(a, no, 1, 256);
    else if (ncv <= 512) launch_lp_parts<T, 256, 2>(a, no, 1, 512);
    else if (ncv <= 1024) launch_lp_parts<T, 256, 4>(a, no, 1, 1024);
    else if (ncv <= 2048) launch_lp_parts<T, 256, 8>(a, no, 1, 2048);
    else {
        const size_t units = size_t(a.rows) * size_t(parts), keys = units * size_t(a.k);
        Partials block;
        NH_TRY(block.open(units * 4 * sizeof(LpPart) + keys * sizeof(LpKey<T>)));
        LpScratch<T> scratch{static_cast<LpPart *>(block.p), nullptr};
        scratch.keys = reinterpret_cast<LpKey<T> *>(scratch.sums + units * 4);
        launch_lp_parts<T, 256, 8>(a, scratch, parts, per);
        for_row_launches(a.rows, a.k ? 1 : 4, 256 + 64, [&](unsigned g, int64_t base) {
            if (a.k) NH_LAUNCH((k_lp_join<T, 256>), dim3(g), dim3(256 + 64), 0, stream(), a, scratch, parts, base);
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

// (f32 rows have 1 / T and differences of logits times their weight in float)
static bool lp_temperature(double t) { return t >= 1e-10 && t <= 1e10; }

// lse of one value a row, or four.
static bool lp_four(const NeuralTensor *lse, const RowCall &c) { return lse && numel(lse) != c.rows; }
static int lp_check_lse(const NeuralTensor *lse, const RowCall &c)
{
    return c.vec(lse, lse && numel(lse) == 4 * c.rows ? 4 * c.rows : c.rows);
}

template <typename T>
static int lp_run(const LpTensors &t, const RowCall &c, double temperature, const Staged &tokens, const Staged &ids)
{
    LpArgs<T> a{};
    a.rows = c.rows;
    a.cols = c.cols;
    a.k = int(t.k);
    a.four = lp_four(t.lse, c);
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
    NH_TRY(lp_check_lse(t.lse, c));
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
    if (t.tokens) NH_TRY(open_raw(tokens, t.tokens, tok_bytes, true));
    if (t.top_ids) NH_TRY(open_raw(ids, t.top_ids, id_bytes, false));
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
    a.four = lp_four(t.lse, c);
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
    if (!t.dx || !t.logits || !t.lse || (!t.g && !t.e) || (t.g && !t.tokens)) return set_error(NEURAL_ERR_NULL_POINTER);
    RowCall c;
    NH_TRY(c.open(t.logits));
    NH_TRY(c.same(t.dx));
    NH_TRY(c.vec(t.g, c.rows));
    NH_TRY(c.vec(t.e, c.rows));
    NH_TRY(lp_check_lse(t.lse, c));
    NH_TRY(c.vec(t.entropy, c.rows));
    if (t.e && !t.entropy && !lp_four(t.lse, c)) return set_error(NEURAL_ERR_NULL_POINTER);
    if (!lp_temperature(temperature)) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    if (c.cols >= int64_t(1) << 31) return set_error(NEURAL_ERR_TENSOR_TOO_LARGE);
    NH_TRY(check_apart({t.dx}, {t.logits, t.g, t.e, t.lse, t.entropy}, 1));
    if (numel(t.logits) == 0) return set_error(NEURAL_OK);
    const size_t tok_bytes = size_t(c.rows) * 8;
    if (raw_may_overlap(t.tokens, tok_bytes, t.dx)) return set_error(NEURAL_ERR_INVALID_ARGUMENT);
    Staged tokens;
    if (t.tokens) NH_TRY(open_raw(tokens, t.tokens, tok_bytes, true));
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
