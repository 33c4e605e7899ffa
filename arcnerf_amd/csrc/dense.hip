// Entry points of the dense and gated layers (dense.hpp): argument checks and the choice of the element type.
#include "dense.hpp"

namespace arcn {

static bool dense_type(int dtype) { return dtype >= ARCN_DTYPE_F32 && dtype <= ARCN_DTYPE_F16; }
static bool dense_act(int act, float beta) {
    if (act == ARCN_ACT_SOFTPLUS) return beta > 0.f;
    return act == ARCN_ACT_NONE || act == ARCN_ACT_RELU || act == ARCN_ACT_SIGMOID || act == ARCN_ACT_SILU || act == ARCN_ACT_GELU;
}
static bool dense_sizes(int64_t rows, int a, int b) { return rows >= 0 && a >= 1 && b >= 1 && a <= (1 << 24) && b <= (1 << 24); }
// of the backward's products: N may be the two halves of a gated layer side by side
static bool dense_sizes_n(int64_t rows, int K, int N) { return N >= 1 && dense_sizes(rows, K, N - N / 2); }

// where the column sums go: none, or those of a 16-bit layer; no rows yet
static bool dense_sums(int dtype, const float *sums, int64_t sums_floats, int64_t *n_sums, int64_t rows, int64_t N) {
    if (n_sums) *n_sums = 0;
    return !sums || (dtype != ARCN_DTYPE_F32 && n_sums && sums_floats >= dense_sums_rows(rows) * N);
}

}  // namespace arcn

using namespace arcn;

#define ARCN_DENSE_DISPATCH(call_)                                            \
    (dtype == ARCN_DTYPE_F32 ? DenseOps<float>::call_                         \
                             : dtype == ARCN_DTYPE_BF16 ? DenseOps<__bf16>::call_ : DenseOps<_Float16>::call_)

ARCN_EXPORT int arcn_dense_fwd(const void *x, int64_t ld_x, const void *w, const void *bias, const void *residual, int64_t ld_res, void *y, int dtype, int act,
                               float beta, int64_t n_rows, int K, int N, void *stream) {
    if (!dense_type(dtype) || !dense_act(act, beta) || !dense_sizes(n_rows, K, N)) return einval("dense_fwd: unsupported type, activation or size");
    if (n_rows == 0) return ARCN_OK;
    if (!x || !w || !y || ld_x < K || (residual && ld_res < N)) return einval("dense_fwd: missing / invalid argument");
    return ARCN_DENSE_DISPATCH(fwd(x, ld_x, w, bias, residual, ld_res, y, act, beta, n_rows, K, N, as_stream(stream)));
}

ARCN_EXPORT int64_t arcn_bias_sums_floats(int64_t n_rows, int N) { return n_rows < 0 || N < 1 ? 0 : dense_sums_rows(n_rows) * N; }

ARCN_EXPORT int arcn_dense_dz_sums(const void *x, int64_t ld_x, const void *w, const void *bias, const void *dy, int64_t ld_dy, void *dz, void *dx, float *sums,
                                   int64_t sums_floats, int64_t *n_sums, int dtype, int act, float beta, int64_t n_rows, int K, int N, void *stream) {
    if (!dense_type(dtype) || !dense_act(act, beta) || !dense_sizes(n_rows, K, N)) return einval("dense_dz: unsupported type, activation or size");
    if (!dense_sums(dtype, sums, sums_floats, n_sums, n_rows, N)) return einval("dense_dz: sums of f32, sums without n_sums or fewer than arcn_bias_sums_floats");
    if (n_rows == 0) return ARCN_OK;
    if (!x || !w || !dy || !dz || ld_x < K || ld_dy < N) return einval("dense_dz: missing / invalid argument");
    return ARCN_DENSE_DISPATCH(dz_dx(x, ld_x, w, bias, dy, ld_dy, dz, dx, act, beta, sums, n_sums, n_rows, K, N, as_stream(stream)));
}

ARCN_EXPORT int arcn_dense_dz(const void *x, int64_t ld_x, const void *w, const void *bias, const void *dy, int64_t ld_dy, void *dz, void *dx, int dtype, int act,
                              float beta, int64_t n_rows, int K, int N, void *stream) {
    return arcn_dense_dz_sums(x, ld_x, w, bias, dy, ld_dy, dz, dx, nullptr, 0, nullptr, dtype, act, beta, n_rows, K, N, stream);
}

ARCN_EXPORT int arcn_dense_dx(const void *dz, int64_t ld_dz, const void *w, const void *w2, void *dx, int dtype, int64_t n_rows, int N, int K, void *stream) {
    if (!dense_type(dtype) || !dense_sizes_n(n_rows, K, N) || (w2 && (N & 1))) return einval("dense_dx: unsupported type or size");
    if (n_rows == 0) return ARCN_OK;
    if (!dz || !w || !dx || ld_dz < N) return einval("dense_dx: missing / invalid argument");
    return ARCN_DENSE_DISPATCH(dx(dz, ld_dz, w, w2, dx, n_rows, N, K, as_stream(stream)));
}

ARCN_EXPORT int64_t arcn_dense_dw_scratch_floats(int64_t n_rows, int N, int K, int dtype) {
    if (!dense_sizes_n(n_rows, K, N) || !dense_type(dtype)) return 0;
    return (int64_t)dense_dw_slabs(dtype == ARCN_DTYPE_F32 ? 4 : 2, n_rows, N, K) * ((int64_t)N * K + N);
}

ARCN_EXPORT int arcn_dense_dw_sums(const void *dz, int64_t ld_dz, const void *x, int64_t ld_x, const float *sums, int64_t n_sums, void *dw, void *db, int dtype,
                                   float *scratch, int64_t scratch_floats, int64_t n_rows, int N, int K, void *stream) {
    if (!dense_type(dtype) || !dense_sizes_n(n_rows, K, N)) return einval("dense_dw: unsupported type or size");
    if (sums && (dtype == ARCN_DTYPE_F32 || n_sums < 0 || n_sums > dense_sums_rows(n_rows))) return einval("dense_dw: sums of f32, or not as many as arcn_dense_dz_sums gave");
    if (!dw || !scratch || (n_rows > 0 && (!dz || !x || ld_dz < N || ld_x < K))) return einval("dense_dw: missing / invalid argument");
    if (scratch_floats < arcn_dense_dw_scratch_floats(n_rows, N, K, dtype)) return einval("dense_dw: scratch smaller than arcn_dense_dw_scratch_floats");
    return ARCN_DENSE_DISPATCH(dw(dz, ld_dz, x, ld_x, sums, n_sums, dw, db, scratch, n_rows, N, K, as_stream(stream)));
}

ARCN_EXPORT int arcn_dense_dw(const void *dz, int64_t ld_dz, const void *x, int64_t ld_x, void *dw, void *db, int dtype, float *scratch, int64_t scratch_floats,
                              int64_t n_rows, int N, int K, void *stream) {
    return arcn_dense_dw_sums(dz, ld_dz, x, ld_x, nullptr, 0, dw, db, dtype, scratch, scratch_floats, n_rows, N, K, stream);
}

ARCN_EXPORT int arcn_gated_fwd(const void *x, int64_t ld_x, const void *w_gate, const void *w_up, const void *b_gate, const void *b_up, void *h, int dtype, int act,
                               float beta, int64_t n_rows, int K, int H, void *stream) {
    if (!dense_type(dtype) || !dense_act(act, beta) || !dense_sizes(n_rows, K, H)) return einval("gated_fwd: unsupported type, activation or size");
    if (n_rows == 0) return ARCN_OK;
    if (!x || !w_gate || !w_up || !h || ld_x < K) return einval("gated_fwd: missing / invalid argument");
    return ARCN_DENSE_DISPATCH(gated_fwd(x, ld_x, w_gate, w_up, b_gate, b_up, h, act, beta, n_rows, K, H, as_stream(stream)));
}

ARCN_EXPORT int arcn_gated_bwd_sums(const void *x, int64_t ld_x, const void *w_gate, const void *w_up, const void *b_gate, const void *b_up, const void *dy, int64_t ld_dy,
                                    const void *w_down, void *dgu, float *sums, int64_t sums_floats, int64_t *n_sums, int dtype, int act, float beta, int64_t n_rows, int K,
                                    int H, int N, void *stream) {
    if (!dense_type(dtype) || !dense_act(act, beta) || !dense_sizes(n_rows, K, H) || !dense_sizes(n_rows, H, N))
        return einval("gated_bwd: unsupported type, activation or size");
    if (!dense_sums(dtype, sums, sums_floats, n_sums, n_rows, 2 * (int64_t)H)) return einval("gated_bwd: sums of f32, sums without n_sums or fewer than arcn_bias_sums_floats");
    if (n_rows == 0) return ARCN_OK;
    if (!x || !w_gate || !w_up || !dy || !w_down || !dgu || ld_x < K || ld_dy < N) return einval("gated_bwd: missing / invalid argument");
    return ARCN_DENSE_DISPATCH(gated_bwd(x, ld_x, w_gate, w_up, b_gate, b_up, dy, ld_dy, w_down, dgu, act, beta, sums, n_sums, n_rows, K, H, N, as_stream(stream)));
}

ARCN_EXPORT int arcn_gated_bwd(const void *x, int64_t ld_x, const void *w_gate, const void *w_up, const void *b_gate, const void *b_up, const void *dy, int64_t ld_dy,
                               const void *w_down, void *dgu, int dtype, int act, float beta, int64_t n_rows, int K, int H, int N, void *stream) {
    return arcn_gated_bwd_sums(x, ld_x, w_gate, w_up, b_gate, b_up, dy, ld_dy, w_down, dgu, nullptr, 0, nullptr, dtype, act, beta, n_rows, K, H, N, stream);
}
