// Layer norm of feature rows, forward and backward, for f32, bf16 and f16 rows (statistics and sums in f32).
//
//   y = (x - mean(x)) r w + b,   r = 1 / sqrt(mean((x - mean)^2) + eps)
//   with n = (x - mean) r and g = dy w:   dx = r (g - mean(g) - n mean(g n)),   dw = sum over rows of dy n,   db = sum over rows of dy
//
// Both directions are one pass over HBM: a row stays in the registers of its lanes between the mean, the centred sum of squares (a
// second look at registers, not the E[x^2] - mean^2 form, which cancels for rows far from zero) and the result.  LPR lanes hold a row
// in NCH 16-byte packs each; rows start at any element (a column slice of a wider buffer, an odd width).  The backward keeps each
// lane's share of dw and db in registers over all the rows that its workgroup meets (a fixed grid strides over the rows), adds the
// workgroup's lanes in LDS and writes ONE partial row per workgroup; a second small kernel adds those in a fixed order: no atomics, the
// same bits on every run.
//
// Bound by HBM: 2 (forward) and 3 (backward) row-sized streams.
#include "elem.hpp"
#include "partials.hpp"

#pragma clang fp contract(fast)

namespace arcn {

constexpr int kNormThreads = 256;
constexpr int kNormMaxBlocks = 2048;   // backward: workgroups, hence partial rows
constexpr int kNormRegWidth = 8192;    // widest row the register kernels hold

// sum over the LPR lanes of a row (LPR = 256: the whole workgroup, through `lds`), the same value in every lane
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float *lds) {
    v += dpp_take<0xB1>(0.f, v);
    v += dpp_take<0x4E>(0.f, v);
    v += dpp_take<0x141>(0.f, v);
    if (LPR >= 16) v += dpp_take<0x140>(0.f, v);
    if (LPR >= 32) v += __shfl_xor(v, 16);
    if (LPR >= 64) v += __shfl_xor(v, 32);
    if (LPR == 256) {
        __syncthreads();   // the previous sum's readers are done
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    }
    return v;
}

// the lane's packs of a row (`rows` operands of one layout): a width that ends inside a pack is read by tail_at / tail_fix, rows narrower than a
// pack element by element; `live` false: nothing is read
template <typename T, int LPR, int NCH>
__device__ __forceinline__ void load_row(const T *p, int lane, int C, bool live, u4v *r) {
    if (C % Elem<T>::VEC == 0 || C < Elem<T>::VEC) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int col = (c * LPR + lane) * Elem<T>::VEC;
            r[c] = load_pack(p + col, live ? C - col : 0);
        }
    } else {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int col = (c * LPR + lane) * Elem<T>::VEC;
            r[c] = live ? load16(tail_at<T>(p + col, C - col)) : u4v{0u, 0u, 0u, 0u};
        }
    }
}
template <typename T, int LPR, int NCH>
__device__ __forceinline__ void unpack_row(u4v *r, int lane, int C, float (*v)[Elem<T>::VEC]) {
    const bool tail = C % Elem<T>::VEC != 0 && C >= Elem<T>::VEC;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        if (tail) r[c] = tail_fix<T>(r[c], C - (c * LPR + lane) * Elem<T>::VEC);
        Elem<T>::unpack(r[c], v[c]);
    }
}

// the lane's columns of the weight or bias (f32, or the rows' type), `fill` where the pointer is NULL or the row has ended
template <typename T, typename WT>
__device__ __forceinline__ void load_param(const WT *w, int col, int C, float fill, float *out) {
    constexpr int V = Elem<T>::VEC, WV = Elem<WT>::VEC;
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = fill;
    if (!w || col >= C) return;
    if (col + V <= C) {
#pragma unroll
        for (int h = 0; h < V / WV; ++h) Elem<WT>::unpack(load16(w + col + h * WV), out + h * WV);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (col + e < C) out[e] = (float)w[col + e];
    }
}

template <typename T, typename WT, int LPR, int NCH>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_fwd_kernel(const T *__restrict__ x, int64_t ld_x, const WT *__restrict__ w, const WT *__restrict__ b, float eps, T *__restrict__ y,
                      float2 *__restrict__ stats, int64_t rows, int C) {
    constexpr int VEC = Elem<T>::VEC, ROWS = kNormThreads / LPR;
    __shared__ float lds[4];
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const float inv_c = 1.0f / (float)C;
    float wv[NCH][VEC], bv[NCH][VEC];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        load_param<T, WT>(w, (c * LPR + lane) * VEC, C, 1.f, wv[c]);
        load_param<T, WT>(b, (c * LPR + lane) * VEC, C, 0.f, bv[c]);
    }
    // every lane of a wave takes part in the sums: a row behind the last one reads nothing and writes nothing
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < rows; r0 += (int64_t)gridDim.x * ROWS) {
        const int64_t r = r0 + sub;
        const bool live = r < rows;
        float v[NCH][VEC], s = 0.f;
        u4v raw[NCH];
        load_row<T, LPR, NCH>(x + r * ld_x, lane, C, live, raw);
        unpack_row<T, LPR, NCH>(raw, lane, C, v);
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += v[c][e];
        const float mean = row_sum<LPR>(s, lds) * inv_c;
        float q = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = ((c * LPR + lane) * VEC + e < C) ? v[c][e] - mean : 0.f;
                v[c][e] = d;
                q += d * d;
            }
        const float rstd = 1.0f / sqrtf(row_sum<LPR>(q, lds) * inv_c + eps);
        if (live && lane == 0 && stats) stats[r] = make_float2(mean, rstd);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int col = (c * LPR + lane) * VEC;
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = v[c][e] * rstd * wv[c][e] + bv[c][e];
            if (live) store_pack(y + r * C + col, Elem<T>::pack(o), C - col);
        }
    }
}

template <typename T, typename WT, int LPR, int NCH>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_bwd_kernel(const T *__restrict__ x, int64_t ld_x, const T *__restrict__ dy, int64_t ld_dy, const WT *__restrict__ w,
                      const float2 *__restrict__ stats, T *__restrict__ dx, float *__restrict__ partial, int64_t rows, int C) {
    constexpr int VEC = Elem<T>::VEC, ROWS = kNormThreads / LPR, COLS = LPR * NCH * VEC;
    __shared__ float lds[LPR == 256 ? 4 : 4 * COLS];
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const float inv_c = 1.0f / (float)C;
    float wv[NCH][VEC], dw[NCH][VEC] = {}, db[NCH][VEC] = {};
#pragma unroll
    for (int c = 0; c < NCH; ++c) load_param<T, WT>(w, (c * LPR + lane) * VEC, C, 1.f, wv[c]);
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < rows; r0 += (int64_t)gridDim.x * ROWS) {
        const int64_t r = r0 + sub;
        const bool live = r < rows;
        const float2 st = live ? stats[r] : make_float2(0.f, 0.f);
        float n[NCH][VEC], d[NCH][VEC], sg = 0.f, sgn = 0.f;
        u4v raw_x[NCH], raw_dy[NCH];
        load_row<T, LPR, NCH>(x + r * ld_x, lane, C, live, raw_x);
        load_row<T, LPR, NCH>(dy + r * ld_dy, lane, C, live, raw_dy);
        unpack_row<T, LPR, NCH>(raw_x, lane, C, n);
        unpack_row<T, LPR, NCH>(raw_dy, lane, C, d);
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                n[c][e] = ((c * LPR + lane) * VEC + e < C) ? (n[c][e] - st.x) * st.y : 0.f;
                dw[c][e] += d[c][e] * n[c][e];
                db[c][e] += d[c][e];
                d[c][e] *= wv[c][e];
                sg += d[c][e];
                sgn += d[c][e] * n[c][e];
            }
        if (dx) {
            const float mg = row_sum<LPR>(sg, lds) * inv_c, mgn = row_sum<LPR>(sgn, lds) * inv_c;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int col = (c * LPR + lane) * VEC;
                float o[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) o[e] = st.y * (d[c][e] - mg - n[c][e] * mgn);
                if (live) store_pack(dx + r * C + col, Elem<T>::pack(o), C - col);
            }
        }
    }
    if (!partial) return;
    // partial[block][0] = dw, [1] = db: the rows of a wave by shuffles, the four waves through LDS
    float *mine = partial + (int64_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (LPR < 256) __syncthreads();
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float v = h ? db[c][e] : dw[c][e];
                const int col = (c * LPR + lane) * VEC + e;
                if (LPR == 256) {
                    if (col < C) mine[h * C + col] = v;
                } else {
#pragma unroll
                    for (int o = LPR; o < 64; o <<= 1) v += __shfl_xor(v, o);
                    if ((threadIdx.x & 63) < LPR) lds[(threadIdx.x >> 6) * COLS + col] = v;
                }
            }
        if (LPR < 256) {
            __syncthreads();
            for (int col = threadIdx.x; col < C; col += kNormThreads)
                mine[h * C + col] = (lds[col] + lds[COLS + col]) + (lds[2 * COLS + col] + lds[3 * COLS + col]);
        }
    }
}

// rows wider than the registers hold: a workgroup per row, the row read again for each step (from L2)
template <typename T, typename WT>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_fwd_wide_kernel(const T *__restrict__ x, int64_t ld_x, const WT *__restrict__ w, const WT *__restrict__ b, float eps, T *__restrict__ y,
                           float2 *__restrict__ stats, int64_t rows, int C) {
    __shared__ float lds[4];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *xr = x + r * ld_x;
        float s = 0.f, q = 0.f;
        for (int c = threadIdx.x; c < C; c += kNormThreads) s += (float)xr[c];
        const float mean = row_sum<256>(s, lds) / (float)C;
        for (int c = threadIdx.x; c < C; c += kNormThreads) q += ((float)xr[c] - mean) * ((float)xr[c] - mean);
        const float rstd = 1.0f / sqrtf(row_sum<256>(q, lds) / (float)C + eps);
        if (threadIdx.x == 0 && stats) stats[r] = make_float2(mean, rstd);
        for (int c = threadIdx.x; c < C; c += kNormThreads)
            y[r * C + c] = (T)(((float)xr[c] - mean) * rstd * (w ? (float)w[c] : 1.f) + (b ? (float)b[c] : 0.f));
    }
}

template <typename T, typename WT>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_dx_wide_kernel(const T *__restrict__ x, int64_t ld_x, const T *__restrict__ dy, int64_t ld_dy, const WT *__restrict__ w,
                          const float2 *__restrict__ stats, T *__restrict__ dx, int64_t rows, int C) {
    __shared__ float lds[4];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float2 st = stats[r];
        float sg = 0.f, sgn = 0.f;
        for (int c = threadIdx.x; c < C; c += kNormThreads) {
            const float g = (float)dy[r * ld_dy + c] * (w ? (float)w[c] : 1.f);
            sg += g;
            sgn += g * ((float)x[r * ld_x + c] - st.x) * st.y;
        }
        const float mg = row_sum<256>(sg, lds) / (float)C, mgn = row_sum<256>(sgn, lds) / (float)C;
        for (int c = threadIdx.x; c < C; c += kNormThreads) {
            const float g = (float)dy[r * ld_dy + c] * (w ? (float)w[c] : 1.f), n = ((float)x[r * ld_x + c] - st.x) * st.y;
            dx[r * C + c] = (T)(st.y * (g - mg - n * mgn));
        }
    }
}

// a thread per column, a workgroup's share of the rows: blockIdx.x = the share, blockIdx.y = 256 columns
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_dw_wide_kernel(const T *__restrict__ x, int64_t ld_x, const T *__restrict__ dy, int64_t ld_dy, const float2 *__restrict__ stats,
                          float *__restrict__ partial, int64_t rows, int C) {
    const int c = blockIdx.y * kNormThreads + threadIdx.x;
    if (c >= C) return;
    float dw = 0.f, db = 0.f;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float d = (float)dy[r * ld_dy + c];
        dw += d * ((float)x[r * ld_x + c] - stats[r].x) * stats[r].y;
        db += d;
    }
    partial[(int64_t)blockIdx.x * 2 * C + c] = dw;
    partial[(int64_t)blockIdx.x * 2 * C + C + c] = db;
}

// workgroups of a register kernel: rows_per = rows per workgroup and trip
static inline unsigned norm_grid(int64_t rows, int rows_per, int most) {
    const int64_t g = ceil_div<int64_t>(rows, rows_per);
    return (unsigned)(g < most ? g : most);
}

static inline int norm_lpr(int dtype, int C) {      // as norm_shape has it
    const int nv = ceil_div<int>(C, dtype == ARCN_DTYPE_F32 ? 4 : 8);
    return nv <= 8 ? 8 : nv <= 16 ? 16 : nv <= (dtype == ARCN_DTYPE_F32 ? 32 : 64) ? 32 : C <= 2048 ? 64 : 256;
}

static inline int norm_parts(int64_t rows, int dtype, int C) {
    if (C > kNormRegWidth) return (int)norm_grid(rows, 64, 256);
    return (int)norm_grid(rows, 4 * kNormThreads / norm_lpr(dtype, C), kNormMaxBlocks);
}

// calls f with the (LPR, NCH) of a width as compile-time numbers
template <typename T, typename Fn>
static void norm_shape(int C, Fn &&f) {
#define ARCN_NS(L_, N_) f(std::integral_constant<int, L_>{}, std::integral_constant<int, N_>{})
    if constexpr (sizeof(T) == 4) {
        if (C <= 32) ARCN_NS(8, 1);
        else if (C <= 64) ARCN_NS(16, 1);
        else if (C <= 128) ARCN_NS(32, 1);
        else if (C <= 256) ARCN_NS(64, 1);
        else if (C <= 512) ARCN_NS(64, 2);
        else if (C <= 1024) ARCN_NS(64, 4);
        else if (C <= 2048) ARCN_NS(64, 8);
        else if (C <= 4096) ARCN_NS(256, 4);
        else ARCN_NS(256, 8);
    } else {
        if (C <= 64) ARCN_NS(8, 1);
        else if (C <= 128) ARCN_NS(16, 1);
        else if (C <= 256) ARCN_NS(32, 1);
        else if (C <= 512) ARCN_NS(32, 2);      // two rows to a wave
        else if (C <= 1024) ARCN_NS(64, 2);
        else if (C <= 2048) ARCN_NS(64, 4);
        else if (C <= 4096) ARCN_NS(256, 2);
        else ARCN_NS(256, 4);
    }
#undef ARCN_NS
}

template <typename T, typename WT>
static void norm_fwd(const void *x, int64_t ld_x, const void *w, const void *b, float eps, void *y, float *stats, int64_t rows, int C, hipStream_t st) {
    const T *xp = static_cast<const T *>(x);
    const WT *wp = static_cast<const WT *>(w), *bp = static_cast<const WT *>(b);
    T *yp = static_cast<T *>(y);
    float2 *sp = reinterpret_cast<float2 *>(stats);
    if (C > kNormRegWidth) {
        hipLaunchKernelGGL((layer_norm_fwd_wide_kernel<T, WT>), dim3(norm_grid(rows, 1, 4096)), dim3(kNormThreads), 0, st, xp, ld_x, wp, bp, eps, yp, sp, rows, C);
        return;
    }
    norm_shape<T>(C, [&](auto lpr, auto nch) {
        hipLaunchKernelGGL((layer_norm_fwd_kernel<T, WT, lpr(), nch()>), dim3(norm_grid(rows, kNormThreads / lpr(), kNormMaxBlocks)), dim3(kNormThreads), 0, st,
                           xp, ld_x, wp, bp, eps, yp, sp, rows, C);
    });
}

template <typename T, typename WT>
static void norm_bwd(const void *x, int64_t ld_x, const void *dy, int64_t ld_dy, const void *w, const float *stats, int dtype, void *dx, void *dw, void *db,
                     float *partial, int64_t rows, int C, hipStream_t st) {
    const T *xp = static_cast<const T *>(x), *gp = static_cast<const T *>(dy);
    const WT *wp = static_cast<const WT *>(w);
    const float2 *sp = reinterpret_cast<const float2 *>(stats);
    float *part = (dw || db) ? partial : nullptr;
    const int parts = norm_parts(rows, dtype, C);
    if (C > kNormRegWidth) {
        if (dx)
            hipLaunchKernelGGL((layer_norm_dx_wide_kernel<T, WT>), dim3(norm_grid(rows, 1, 4096)), dim3(kNormThreads), 0, st, xp, ld_x, gp, ld_dy, wp, sp,
                               static_cast<T *>(dx), rows, C);
        if (part)
            hipLaunchKernelGGL((layer_norm_dw_wide_kernel<T>), dim3((unsigned)parts, (unsigned)ceil_div<int>(C, kNormThreads)), dim3(kNormThreads), 0, st, xp, ld_x,
                               gp, ld_dy, sp, part, rows, C);
    } else {
        norm_shape<T>(C, [&](auto lpr, auto nch) {
            hipLaunchKernelGGL((layer_norm_bwd_kernel<T, WT, lpr(), nch()>), dim3((unsigned)parts), dim3(kNormThreads), 0, st, xp, ld_x, gp, ld_dy, wp, sp,
                               static_cast<T *>(dx), part, rows, C);
        });
    }
    if (part)
        sum_partials<WT>(part, parts, C, C, static_cast<WT *>(dw), static_cast<WT *>(db), st);
}

static int norm_args(const char *what, int dtype, int w_dtype, int64_t n_rows, int C) {
    if (dtype < ARCN_DTYPE_F32 || dtype > ARCN_DTYPE_F16 || (w_dtype != dtype && w_dtype != ARCN_DTYPE_F32)) return einval(what);
    if (n_rows < 0 || C < 1 || C > (1 << 24)) return einval(what);
    return ARCN_OK;
}

}  // namespace arcn

using namespace arcn;

// f<T, WT>(...) for the pair of type codes (checked by norm_args)
#define ARCN_NORM_DISPATCH(fn_, ...)                                                          \
    do {                                                                                      \
        if (dtype == ARCN_DTYPE_F32) fn_<float, float>(__VA_ARGS__);                          \
        else if (dtype == ARCN_DTYPE_BF16 && w_dtype == dtype) fn_<__bf16, __bf16>(__VA_ARGS__); \
        else if (dtype == ARCN_DTYPE_BF16) fn_<__bf16, float>(__VA_ARGS__);                   \
        else if (w_dtype == dtype) fn_<_Float16, _Float16>(__VA_ARGS__);                      \
        else fn_<_Float16, float>(__VA_ARGS__);                                               \
    } while (0)

ARCN_EXPORT int arcn_layer_norm_fwd(const void *x, int64_t ld_x, const void *weight, const void *bias, int dtype, int w_dtype, float eps, void *y,
                                    float *stats, int64_t n_rows, int C, void *stream) {
    if (int rc = norm_args("layer_norm_fwd: unsupported type or size", dtype, w_dtype, n_rows, C)) return rc;
    if (n_rows == 0) return ARCN_OK;
    if (!x || !y || ld_x < C) return einval("layer_norm_fwd: missing / invalid argument");
    ARCN_NORM_DISPATCH(norm_fwd, x, ld_x, weight, bias, eps, y, stats, n_rows, C, as_stream(stream));
    return check_launch("layer_norm_fwd");
}

ARCN_EXPORT int64_t arcn_layer_norm_bwd_scratch_floats(int64_t n_rows, int C, int dtype) {
    if (n_rows < 1 || C < 1) return 0;
    return (int64_t)norm_parts(n_rows, dtype, C) * 2 * C;
}

ARCN_EXPORT int arcn_layer_norm_bwd(const void *x, int64_t ld_x, const void *dy, int64_t ld_dy, const void *weight, const float *stats, int dtype, int w_dtype,
                                    void *dx, void *dweight, void *dbias, float *scratch, int64_t scratch_floats, int64_t n_rows, int C, void *stream) {
    if (int rc = norm_args("layer_norm_bwd: unsupported type or size", dtype, w_dtype, n_rows, C)) return rc;
    if (n_rows == 0) return (dweight || dbias) ? einval("layer_norm_bwd: no rows to sum the weight gradient over") : ARCN_OK;
    if (!x || !dy || !stats || ld_x < C || ld_dy < C) return einval("layer_norm_bwd: missing / invalid argument");
    if ((dweight || dbias) && (!scratch || scratch_floats < arcn_layer_norm_bwd_scratch_floats(n_rows, C, dtype)))
        return einval("layer_norm_bwd: scratch smaller than arcn_layer_norm_bwd_scratch_floats");
    ARCN_NORM_DISPATCH(norm_bwd, x, ld_x, dy, ld_dy, weight, stats, dtype, dx, dweight, dbias, scratch, n_rows, C, as_stream(stream));
    return check_launch("layer_norm_bwd");
}
