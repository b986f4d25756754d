// rms_norm_grad.hip -- the backward pass of RMS norm, joined with the residual stream's
// gradient:
//   xh = h rstd; w = dy gamma; dx = rstd (w - xh mean_c(w xh)) [rounded, + dh];
//   dgamma = sum_rows dy xh
// in double; dx is rounded once (twice with dh), dgamma once more for what each block leaves.
#include "rms_norm.hpp"
#include "row_call.hpp"

namespace nh {

// A row of any width by a block of kLnWide lanes, in two walks: the row's sum, then dx.
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

template <typename T>
int launch_rms_grad(const RmsGradArgs<T> &a, T *dgamma)
{
    // the columns first: the row pass may write over what they read
    if (dgamma) NH_TRY(launch_rms_cols(a, dgamma));
    if (a.dx)
        for_row_launches(a.rows, 1, kLnWide, [&](unsigned g, int64_t base) {
            NH_LAUNCH((k_rms_grad_wide<T>), dim3(g), dim3(kLnWide), 0, stream(), a, base);
        });
    return check_launch();
}

template int launch_rms_grad<float>(const RmsGradArgs<float> &, float *);
template int launch_rms_grad<double>(const RmsGradArgs<double> &, double *);

}  // namespace nh
