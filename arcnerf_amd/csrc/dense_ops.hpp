// DenseOps<T>: one translation unit per element type includes this and instantiates it.
#pragma once

#include "dense.hpp"

namespace arcn {

template <typename T>
static const T *tp(const void *p) {
    return static_cast<const T *>(p);
}

template <typename T>
int DenseOps<T>::fwd(const void *x, int64_t ld_x, const void *w, const void *b, const void *res, int64_t ld_res, void *y, int act, float beta, int64_t rows, int K, int N,
                     hipStream_t st) {
    DenseArgs<T> p = {};
    p.i = {tp<T>(w), nullptr, K, N, K, 0};
    p.j = {tp<T>(x), nullptr, ld_x, rows, K, 0};
    p.bias = tp<T>(b);
    p.res = tp<T>(res);
    p.ld_res = ld_res;
    p.out = static_cast<T *>(y);
    p.ld_out = N;
    p.act = act;
    p.beta = beta;
    p.inv_beta = 1.f / beta;
    if (dense_few(sizeof(T), rows, N)) {
        const dim3 grid((unsigned)ceil_div<int>(N, 16), (unsigned)ceil_div<int64_t>(rows, 32));
        if (rows <= 16) hipLaunchKernelGGL((dense_few_kernel<T, false, 1>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((dense_few_kernel<T, false, 2>), grid, dim3(256), 0, st, p);
        return check_launch("dense_fwd");
    }
    return launch_tiles<T, kDenseFwd>(p, st);
}

template <typename T>
int DenseOps<T>::dx(const void *dz, int64_t ld_dz, const void *w, const void *w2, void *dx, int64_t rows, int N, int K, hipStream_t st) {
    DenseArgs<T> p = {};
    p.i = {tp<T>(w), tp<T>(w2), K, K, N, N / 2};
    p.j = {tp<T>(dz), nullptr, ld_dz, rows, N, 0};
    p.out = static_cast<T *>(dx);
    p.ld_out = K;
    return launch_tiles<T, kDenseDx>(p, st);
}

template <typename T>
int DenseOps<T>::dz_dx(const void *x, int64_t ld_x, const void *w, const void *b, const void *dy, int64_t ld_dy, void *dz, void *dx_, int act, float beta, float *sums,
                       int64_t *n_sums, int64_t rows, int K, int N, hipStream_t st) {
    DenseArgs<T> p = {};
    p.i = {tp<T>(w), nullptr, K, N, K, 0};
    p.j = {tp<T>(x), nullptr, ld_x, rows, K, 0};
    p.bias = tp<T>(b);
    p.res = tp<T>(dy);
    p.ld_res = ld_dy;
    p.out = static_cast<T *>(dz);
    p.ld_out = N;
    p.sums = sums;
    p.act = act;
    p.beta = beta;
    p.inv_beta = 1.f / beta;
    const bool stays = dx_ && dense_stays<T>(rows, K, N);
    if (stays) {
        p.out2 = static_cast<T *>(dx_);
        p.ld_out2 = K;
    }
    if (int rc = stays ? launch_dz_dx<T>(p, st) : launch_tiles<T, kDenseDz>(p, st)) return rc;
    if (sums) *n_sums = p.n_sums;
    return !stays && dx_ ? dx(dz, N, w, nullptr, dx_, rows, N, K, st) : ARCN_OK;
}

template <typename T>
int DenseOps<T>::dw(const void *dz, int64_t ld_dz, const void *x, int64_t ld_x, const float *sums, int64_t n_sums, void *dw, void *db, float *scratch, int64_t rows, int N,
                    int K, hipStream_t st) {
    DenseArgs<T> p = {};
    p.i = {tp<T>(x), nullptr, ld_x, K, rows, 0};
    p.j = {tp<T>(dz), nullptr, ld_dz, N, rows, 0};
    p.partial = scratch;
    p.want_sums = db != nullptr;
    p.sums = const_cast<float *>(sums);      // (read)
    p.n_sums = n_sums;
    p.slabs = dense_dw_slabs(sizeof(T), rows, N, K);
    if (int rc = launch_tiles<T, kDenseDw>(p, st)) return rc;
    const int64_t n = (int64_t)N * K, n_db = db ? N : 0;
    sum_partials<T>(scratch, p.slabs, n, n_db, static_cast<T *>(dw), static_cast<T *>(db), st);
    return check_launch("dense_dw");
}

template <typename T>
int DenseOps<T>::gated_fwd(const void *x, int64_t ld_x, const void *wg, const void *wu, const void *bg, const void *bu, void *h, int act, float beta, int64_t rows, int K,
                           int H, hipStream_t st) {
    DenseArgs<T> p = {};
    p.i = {tp<T>(wg), tp<T>(wu), K, H, K, 0};
    p.j = {tp<T>(x), nullptr, ld_x, rows, K, 0};
    p.bias = tp<T>(bg);
    p.bias2 = tp<T>(bu);
    p.out = static_cast<T *>(h);
    p.ld_out = H;
    p.act = act;
    p.beta = beta;
    p.inv_beta = 1.f / beta;
    if (dense_few(sizeof(T), rows, 2 * (int64_t)H)) {
        const dim3 grid((unsigned)ceil_div<int>(H, 16), (unsigned)ceil_div<int64_t>(rows, 32));
        if (rows <= 16) hipLaunchKernelGGL((dense_few_kernel<T, true, 1>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((dense_few_kernel<T, true, 2>), grid, dim3(256), 0, st, p);
        return check_launch("gated_fwd");
    }
    return launch_tiles<T, kGatedFwd>(p, st);
}

template <typename T>
int DenseOps<T>::gated_bwd(const void *x, int64_t ld_x, const void *wg, const void *wu, const void *bg, const void *bu, const void *dy, int64_t ld_dy, const void *wd,
                           void *dgu, int act, float beta, float *sums, int64_t *n_sums, int64_t rows, int K, int H, int N, hipStream_t st) {
    DenseArgs<T> p = {};
    p.i = {tp<T>(wg), tp<T>(wu), K, H, K, 0};
    p.j = {tp<T>(x), nullptr, ld_x, rows, K, 0};
    p.i2 = {tp<T>(wd), nullptr, H, H, N, 0};
    p.j2 = {tp<T>(dy), nullptr, ld_dy, rows, N, 0};
    p.bias = tp<T>(bg);
    p.bias2 = tp<T>(bu);
    p.out = static_cast<T *>(dgu);
    p.ld_out = 2 * (int64_t)H;
    p.sums = sums;
    p.act = act;
    p.beta = beta;
    p.inv_beta = 1.f / beta;
    if (int rc = launch_tiles<T, kGatedBwd>(p, st)) return rc;
    if (sums) *n_sums = p.n_sums;
    return ARCN_OK;
}

}  // namespace arcn
