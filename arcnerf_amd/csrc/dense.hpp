// Dense layers with their epilogues, for f32, bf16 and f16, on the matrix cores: the products behind arcn_dense_* and arcn_gated_*.
//
//   dense         y = act(x W^T + b) + res                       dz = dy act'(x W^T + b)      dx = dz W      dW = dz^T x, db = sum dz
//   gated         h = act(x Wg^T + bg) (x Wu^T + bu)             with dh = dy Wd:  du = dh act(g),  dg = dh u act'(g)
//
// Every product is D[i, j] = sum_r I[i, r] J[j, r]: i = MFMA rows = the features that are contiguous in the output's memory, j = MFMA
// columns = its rows.  An operand in memory has either r contiguous (x, dy and the weights of a forward pass: fragments are 16-byte LDS
// reads) or its output index contiguous (TR: the weights of an input gradient, both operands of a weight gradient: fragments are
// transposing LDS reads, ds_read_b64_tr_b16), so nothing is ever transposed in memory.
//
// Nothing of the forward pass but its inputs (and h) is kept for the backward: a pre-activation is computed again in the tile that needs
// its slope, in f32, where a saved one would have been rounded to the layer's type and cost its bytes twice (2 K operations per 4 bytes:
// at K = 256 a tile computes it faster than HBM would return it).  The gated backward computes g, u AND dh of a tile in registers; only
// dg and du, each rounded once, are written.
//
// f32 operands are split into three bf16 planes on their way into LDS, x = hi + mid + lo, and six products (hi hi, hi mid, mid hi, hi lo,
// lo hi, mid mid) are accumulated in f32; what is dropped is below 2^-25 of a product.  416 TFLOP/s of f32-accurate products against 157
// on the f32 MFMA.  Infinities and NaN in such an operand give NaN.
//
// A tile's I rows are dealt to MFMA tiles in pairs: MFMA row 4 g + r of tile m is feature 32 (m / 2) + 8 g + 4 (m % 2) + r, so that a
// lane's accumulators of two tiles are 8 CONSECUTIVE features of one row: residual, gradient and result move as 16 bytes per lane.
#pragma once

#include <type_traits>

#include "elem.hpp"

#pragma clang fp contract(fast)

namespace arcn {

typedef short s4v __attribute__((ext_vector_type(4)));
typedef short s8v __attribute__((ext_vector_type(8)));

enum DenseMode { kDenseFwd, kDenseDz, kGatedFwd, kGatedBwd, kDenseDx, kDenseDw };

// ---- activations: value and slope -----------------------------------------------------------------------------------------------------
// e^x for x <= 0 (or NaN): 2^(x log2 e) on the hardware's exponential, the rounding of the product put back to first order; zero from -150 on
__device__ __forceinline__ float exp_hw(float x) {
    x = x < -150.f ? -150.f : x;
    const float t = x * 1.44269504f, lo = fmaf(x, 1.44269504f, -t) + x * 1.92596299e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e * 0.693147181f, lo, e);
}

template <bool SLOPE>
__device__ __forceinline__ float act_eval(float z, int act, float beta, float &slope) {
    switch (act) {
    case ARCN_ACT_RELU:
        if (SLOPE) slope = z <= 0.f ? 0.f : 1.f;
        return z <= 0.f ? 0.f : z;      // (a NaN stays one)
    case ARCN_ACT_SIGMOID:
    case ARCN_ACT_SILU: {
        const float e = exp_hw(-fabsf(z)), q = __builtin_amdgcn_rcpf(1.f + e);
        const float s = z >= 0.f ? q : e * q;
        if (act == ARCN_ACT_SIGMOID) {
            if (SLOPE) slope = e * q * q;
            return s;
        }
        const float one_minus = z >= 0.f ? e * q : q;
        if (SLOPE) slope = s * (1.f + z * one_minus);
        return z * s;
    }
    case ARCN_ACT_SOFTPLUS: {
        // log1p(t) = log(u) t / (u - 1) with u = fl(1 + t): the rounding of 1 + t cancels
        const float bz = beta * z;
        const float t = exp_hw(-fabsf(bz)), u = 1.f + t, q = __builtin_amdgcn_rcpf(u);
        if (SLOPE) slope = bz > 20.f ? 1.f : (bz >= 0.f ? q : t * q);
        const float l = u == 1.f ? t : __logf(u) * (t / (u - 1.f));
        return bz > 20.f ? z : (fmaxf(bz, 0.f) + l) / beta;
    }
    case ARCN_ACT_GELU: {
        const float cdf = 0.5f * (1.f + erff(z * 0.707106781f));
        if (SLOPE) slope = fmaf(z * 0.398942280f, exp_hw(-0.5f * z * z), cdf);
        return z * cdf;
    }
    default:
        if (SLOPE) slope = 1.f;
        return z;
    }
}

// ---- operand fragments ------------------------------------------------------------------------------------------------------------------
template <typename T>
struct Mma;
template <>
struct Mma<__bf16> {
    static constexpr int P = 1, BK = 64, NBUF = 2;
    static __device__ __forceinline__ f4v mma(const s8v *a, const s8v *b, f4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[0]), __builtin_bit_cast(bf16x8, b[0]), c, 0, 0, 0);
    }
    static constexpr short kOne = 0x3f80;
};
template <>
struct Mma<_Float16> {
    static constexpr int P = 1, BK = 64, NBUF = 2;
    static __device__ __forceinline__ f4v mma(const s8v *a, const s8v *b, f4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a[0]), __builtin_bit_cast(f16x8, b[0]), c, 0, 0, 0);
    }
    static constexpr short kOne = 0x3c00;
};
template <>
struct Mma<float> {
    static constexpr int P = 3, BK = 32, NBUF = 1;
    static __device__ __forceinline__ f4v one(s8v a, s8v b, f4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f4v mma(const s8v *a, const s8v *b, f4v c) {   // smallest terms first
        c = one(a[1], b[1], c);
        c = one(a[0], b[2], c);
        c = one(a[2], b[0], c);
        c = one(a[0], b[1], c);
        c = one(a[1], b[0], c);
        return one(a[0], b[0], c);
    }
    static constexpr short kOne = 0x3f80;
};

// eight consecutive elements as they come from memory
template <typename T>
struct Raw8 {
    u4v v[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T *p) {
    Raw8<T> r;
#pragma unroll
    for (int h = 0; h < (int)sizeof(T) / 2; ++h) r.v[h] = load16(p + h * Elem<T>::VEC);
    return r;
}
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T *p, int64_t left) {   // `left` elements remain (<= 0: nothing is read), zero behind them
    Raw8<T> r;
#pragma unroll
    for (int h = 0; h < (int)sizeof(T) / 2; ++h) r.v[h] = load_pack(p + h * Elem<T>::VEC, left - h * Elem<T>::VEC);
    return r;
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T> &r, float *v) {
#pragma unroll
    for (int h = 0; h < (int)sizeof(T) / 2; ++h) Elem<T>::unpack(r.v[h], v + h * Elem<T>::VEC);
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float *v, int64_t left) {
#pragma unroll
    for (int h = 0; h < (int)sizeof(T) / 2; ++h) store_pack(p + h * Elem<T>::VEC, Elem<T>::pack(v + h * Elem<T>::VEC), left - h * Elem<T>::VEC);
}

// the planes of eight elements: themselves for the 16-bit types; hi, mid, lo for f32 (each rounded to nearest: the remainders are exact)
template <typename T>
__device__ __forceinline__ void planes8(const Raw8<T> &r, s8v *pl) {
    if constexpr (sizeof(T) == 2) {
        pl[0] = __builtin_bit_cast(s8v, r.v[0]);
    } else {
        float v[8];
        unpack8<T>(r, v);
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            const u4v q = Elem<__bf16>::pack(v);
            float b[8];
            Elem<__bf16>::unpack(q, b);
            pl[p] = __builtin_bit_cast(s8v, q);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] -= b[e];
        }
    }
}

template <typename T>
struct Operand {
    const T *a, *b;   // b: the second matrix of an operand made of two (gated: the rows in groups of 32 from a, b, a, b, ...; TR: reduction
                      // rows from `split` on)
    int64_t ld;
    int64_t n_out, n_red;
    int64_t split;
};

// R: output indices of the tile.  PAIR: the I operand (MFMA tiles in pairs), else the J operand.  GATED: rows alternate between two matrices.
template <typename T, int R, int THREADS, bool TR, bool PAIR, bool GATED>
struct Tile {
    static constexpr int BK = Mma<T>::BK, P = Mma<T>::P;
    static constexpr int CHUNKS = R * BK / 8, N = (CHUNKS + THREADS - 1) / THREADS;
    static constexpr int kElems = P * R * BK;   // of one LDS buffer
    Raw8<T> raw[N];

    // place of chunk c (8 elements) of tile row `row` in a plane, in elements.  The swizzles spread what one read instruction's lanes
    // touch over all banks: 8 lanes of a 16-byte read over eight 16-byte places, 16 lanes of an 8-byte transposing read (4 rows) over
    // sixteen 8-byte ones.
    static __device__ __forceinline__ int place(int row, int c) {
        if (!TR) {
            const int q = row * (BK / 8) + c, line = q >> 3;
            const int s = BK == 64 ? (PAIR ? ((line & 3) | ((line >> 1) & 4)) : (line & 7)) : (PAIR ? ((line & 1) | ((line >> 1) & 2)) : (line & 3));
            return 8 * (q ^ s);
        }
        if (R < 64) return 8 * (row * (R / 8) + c);
        return 8 * (row * (R / 8) + (c ^ (PAIR ? ((row & 1) << 2) : ((row & 3) << 1))));
    }
    static __device__ __forceinline__ bool halves_swapped(int row) { return TR && PAIR && R >= 64 && (row & 2); }

    __device__ __forceinline__ void fetch(const Operand<T> &op, int64_t out0, int64_t k0, int64_t k_end, int tid) {
        const bool full = k0 + BK <= k_end && (!TR || out0 + R <= op.n_out);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int q = tid + n * THREADS;
            if (CHUNKS % THREADS && q >= CHUNKS) break;
            if (!TR) {
                const int row = q / (BK / 8), c = q % (BK / 8);
                // (a row behind the operand's last one is computed and dropped: it reads the last one)
                int64_t out = out0 + (GATED ? ((row >> 6) * 32 + (row & 31)) : row);
                out = out < op.n_out ? out : op.n_out - 1;
                const T *p = (GATED && (row & 32) ? op.b : op.a) + out * op.ld + k0 + 8 * c;
                raw[n] = full ? load8<T>(p) : load8<T>(p, k_end - (k0 + 8 * c));
            } else {
                const int row = q / (R / 8), c = q % (R / 8);
                const int64_t r = k0 + row, out = out0 + 8 * c;
                const T *p = (op.b && r >= op.split ? op.b + (r - op.split) * op.ld : op.a + r * op.ld) + out;
                raw[n] = full ? load8<T>(p) : load8<T>(p, r < k_end ? op.n_out - out : 0);
            }
        }
    }

    __device__ __forceinline__ void stash(short *lds, int tid) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int q = tid + n * THREADS;
            if (CHUNKS % THREADS && q >= CHUNKS) break;
            const int row = TR ? q / (R / 8) : q / (BK / 8), c = TR ? q % (R / 8) : q % (BK / 8);
            s8v pl[P];
            planes8<T>(raw[n], pl);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                u4v v = __builtin_bit_cast(u4v, pl[p]);
                if (TR && PAIR && R >= 64) {
                    const bool sw = halves_swapped(row);
                    v = u4v{sw ? v[2] : v[0], sw ? v[3] : v[1], sw ? v[0] : v[2], sw ? v[1] : v[3]};
                }
                *reinterpret_cast<u4v *>(lds + p * R * BK + place(row, c)) = v;
            }
        }
    }

    // fragment of MFMA tile m (from tile row / column `base`) at reduction step kk (32 elements): lane l holds output index l % 16 (as
    // dealt), reduction elements 8 (l / 16) .. + 7
    static __device__ __forceinline__ void frag(const short *lds, int base, int m, int kk, int lane, s8v *f) {
        const int o = lane & 15, g = lane >> 4;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const short *pl = lds + p * R * BK;
            if (!TR) {
                const int row = base + (PAIR ? 32 * (m >> 1) + 8 * (o >> 2) + 4 * (m & 1) + (o & 3) : 16 * m + o);
                f[p] = *reinterpret_cast<const s8v *>(pl + place(row, 4 * kk + g));
            } else {
                // lane o of a group of 16 asks for 4 output indices (quad o % 4) of reduction row o / 4 and receives 4 reduction rows of
                // output index o
                const int col = base + (PAIR ? 32 * (m >> 1) + 8 * (o & 3) + 4 * (m & 1) : 16 * m + 4 * (o & 3));
                s4v h[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = 32 * kk + 8 * g + 4 * e + (o >> 2);
                    const int at = place(row, col >> 3) + ((col & 4) ^ (halves_swapped(row) ? 4 : 0));
                    h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v *)(pl + at));
                }
                f[p] = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
            }
        }
    }
};

template <typename T>
struct DenseArgs {
    Operand<T> i, j;         // the product
    Operand<T> i2, j2;       // kGatedBwd: dh = dy Wd (i2 = Wd, j2 = dy)
    const T *bias, *bias2;   // by i; may be NULL
    const T *res;            // kDenseFwd: the residual (or NULL); kDenseDz: dy
    int64_t ld_res;
    T *out;
    int64_t ld_out;
    float *partial;          // kDenseDw: [slab][n_j * n_i (+ n_j column sums of j)]
    int want_sums;
    int act;
    float beta;
    int64_t tiles_i, tiles;  // tiles: of the whole product (times the slabs)
    int slabs;
};

// blockIdx -> tile: workgroups are dealt to the 8 XCDs in turn, so each XCD gets a contiguous range of tiles and the tiles that share
// their J rows (the large operand) meet in one L2
__device__ __forceinline__ int64_t xcd_tile() {
    const int64_t per = gridDim.x >> 3;
    return (int64_t)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
}

template <typename T, int MODE, int WI, int WJ, int MI, int NJ>
__global__ void __launch_bounds__(64 * WI *WJ, 2)
dense_kernel(const DenseArgs<T> p) {
    constexpr int THREADS = 64 * WI * WJ, BI = 16 * MI * WI, BJ = 16 * NJ * WJ;
    constexpr int BK = Mma<T>::BK, P = Mma<T>::P, NBUF = Mma<T>::NBUF;
    constexpr bool GATED = MODE == kGatedFwd || MODE == kGatedBwd;
    constexpr bool I_TR = MODE == kDenseDx || MODE == kDenseDw, J_TR = MODE == kDenseDw;
    constexpr int OUT_I = GATED ? BI / 2 : BI;      // features per tile
    typedef Tile<T, BI, THREADS, I_TR, true, GATED> TI;
    typedef Tile<T, BJ, THREADS, J_TR, false, false> TJ;
    typedef Tile<T, BI / 2, THREADS, true, true, false> TI2;
    constexpr int BUF = TI::kElems + TJ::kElems;
    __shared__ __attribute__((aligned(16))) short lds[NBUF * BUF];

    const int64_t t = xcd_tile();
    if (t >= p.tiles) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wi = wave % WI, wj = wave / WI;
    const int64_t i0 = (t % p.tiles_i) * OUT_I;
    int64_t rest = t / p.tiles_i, slab = 0, k_lo = 0, k_hi = p.i.n_red;
    if (MODE == kDenseDw) {
        const int64_t tiles_j = p.tiles / p.tiles_i / p.slabs;
        slab = rest / tiles_j;
        rest %= tiles_j;
        const int64_t per = (ceil_div_dev(p.i.n_red, p.slabs) + BK - 1) / BK * BK;
        k_lo = slab * per;
        k_hi = k_lo + per < p.i.n_red ? k_lo + per : p.i.n_red;
    }
    const int64_t j0 = rest * BJ;

    f4v acc[MI][NJ];
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NJ; ++n) acc[m][n] = f4v{0.f, 0.f, 0.f, 0.f};
    f4v sums[MODE == kDenseDw ? NJ : 1];
#pragma unroll
    for (int n = 0; n < (MODE == kDenseDw ? NJ : 1); ++n) sums[n] = f4v{0.f, 0.f, 0.f, 0.f};
    const bool my_sums = MODE == kDenseDw && p.want_sums && i0 == 0 && wi == 0;   // wave-uniform

    auto step = [&](auto &ti, auto &tj, const short *buf, auto &c, bool add_sums) {
        typedef std::remove_reference_t<decltype(ti)> Ti;
        typedef std::remove_reference_t<decltype(tj)> Tj;
        constexpr int M = sizeof(c) / sizeof(c[0]);
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk) {
            s8v a[M][P], b[NJ][P];
#pragma unroll
            for (int m = 0; m < M; ++m) Ti::frag(buf, wi * 16 * M, m, kk, lane, a[m]);
#pragma unroll
            for (int n = 0; n < NJ; ++n) Tj::frag(buf + TI::kElems, wj * 16 * NJ, n, kk, lane, b[n]);
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int n = 0; n < NJ; ++n) c[m][n] = Mma<T>::mma(a[m], b[n], c[m][n]);
            if (MODE == kDenseDw && add_sums) {
                const short o = Mma<T>::kOne;
                s8v ones[P] = {};
                ones[0] = s8v{o, o, o, o, o, o, o, o};
#pragma unroll
                for (int n = 0; n < NJ; ++n) sums[n] = Mma<T>::mma(ones, b[n], sums[n]);
            }
        }
    };
    auto product = [&](auto &ti, auto &tj, const Operand<T> &oi, const Operand<T> &oj, auto &c) {
        const int64_t n_steps = k_lo < k_hi ? (k_hi - k_lo + BK - 1) / BK : 0;
        if (n_steps > 0) {
            ti.fetch(oi, i0, k_lo, k_hi, tid);
            tj.fetch(oj, j0, k_lo, k_hi, tid);
        }
        if (NBUF == 2 && n_steps > 0) {
            ti.stash(lds, tid);
            tj.stash(lds + TI::kElems, tid);
            __syncthreads();
        }
        for (int64_t s = 0; s < n_steps; ++s) {
            const int64_t k = k_lo + (s + 1) * BK;
            if (NBUF == 2) {
                short *buf = lds + (s & 1) * BUF, *next = lds + ((s & 1) ^ 1) * BUF;
                if (s + 1 < n_steps) {
                    ti.fetch(oi, i0, k, k_hi, tid);
                    tj.fetch(oj, j0, k, k_hi, tid);
                }
                step(ti, tj, buf, c, my_sums);
                if (s + 1 < n_steps) {
                    ti.stash(next, tid);   // last read one step ago, behind the barrier below
                    tj.stash(next + TI::kElems, tid);
                }
                __syncthreads();
            } else {
                ti.stash(lds, tid);
                tj.stash(lds + TI::kElems, tid);
                __syncthreads();
                if (s + 1 < n_steps) {
                    ti.fetch(oi, i0, k, k_hi, tid);
                    tj.fetch(oj, j0, k, k_hi, tid);
                }
                step(ti, tj, lds, c, my_sums);
                __syncthreads();
            }
        }
    };
    {
        TI ti;
        TJ tj;
        product(ti, tj, p.i, p.j, acc);
    }
    f4v acc2[MODE == kGatedBwd ? MI / 2 : 1][NJ];
    if (MODE == kGatedBwd) {
#pragma unroll
        for (int m = 0; m < (MODE == kGatedBwd ? MI / 2 : 1); ++m)
#pragma unroll
            for (int n = 0; n < NJ; ++n) acc2[m][n] = f4v{0.f, 0.f, 0.f, 0.f};
        k_hi = p.i2.n_red;
        TI2 ti;
        TJ tj;
        product(ti, tj, p.i2, p.j2, acc2);
    }

    // ---- epilogue: lane (g, o) holds features 8 g .. 8 g + 7 of a pair of tiles, row o -------------------------------------------------
    const int g = lane >> 4, o = lane & 15;
    auto pair8 = [&](auto &c, int pr, int n, float *v) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            v[r] = c[2 * pr][n][r];
            v[4 + r] = c[2 * pr + 1][n][r];
        }
    };
    auto bias8 = [&](const T *b, int64_t i, float *v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
        if (b) unpack8<T>(load8<T>(b + i, p.i.n_out - i), v);
    };
    if constexpr (MODE == kDenseDw) {
        float *part = p.partial + slab * (p.i.n_out * p.j.n_out + (p.want_sums ? p.j.n_out : 0));
#pragma unroll
        for (int n = 0; n < NJ; ++n) {
            const int64_t j = j0 + (wj * NJ + n) * 16 + o;
            if (j >= p.j.n_out) continue;
#pragma unroll
            for (int pr = 0; pr < MI / 2; ++pr) {
                const int64_t i = i0 + wi * 16 * MI + 32 * pr + 8 * g;
                float v[8];
                pair8(acc, pr, n, v);
                store8<float>(part + j * p.i.n_out + i, v, p.i.n_out - i);
            }
            if (my_sums && g == 0) part[p.i.n_out * p.j.n_out + j] = sums[n][0];
        }
    } else if constexpr (GATED) {
#pragma unroll
        for (int pr = 0; pr < MI / 4; ++pr) {
            const int64_t i = i0 + wi * 8 * MI + 32 * pr + 8 * g;
            if (i >= p.i.n_out) continue;
            float bg[8], bu[8];
            bias8(p.bias, i, bg);
            bias8(p.bias2, i, bu);
#pragma unroll
            for (int n = 0; n < NJ; ++n) {
                const int64_t j = j0 + (wj * NJ + n) * 16 + o;
                if (j >= p.j.n_out) continue;
                float gv[8], uv[8];
                pair8(acc, 2 * pr, n, gv);
                pair8(acc, 2 * pr + 1, n, uv);
                T *dst = p.out + j * p.ld_out + i;
                if constexpr (MODE == kGatedFwd) {
                    float slope;
#pragma unroll
                    for (int e = 0; e < 8; ++e) gv[e] = act_eval<false>(gv[e] + bg[e], p.act, p.beta, slope) * (uv[e] + bu[e]);
                    store8<T>(dst, gv, p.i.n_out - i);
                } else {
                    float dh[8];
                    pair8(acc2, pr, n, dh);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float slope;
                        const float a = act_eval<true>(gv[e] + bg[e], p.act, p.beta, slope);
                        gv[e] = dh[e] * (uv[e] + bu[e]) * slope;
                        uv[e] = dh[e] * a;
                    }
                    store8<T>(dst, gv, p.i.n_out - i);
                    store8<T>(dst + p.i.n_out, uv, p.i.n_out - i);   // du behind dg in a row of 2 H
                }
            }
        }
    } else {
#pragma unroll
        for (int pr = 0; pr < MI / 2; ++pr) {
            const int64_t i = i0 + wi * 16 * MI + 32 * pr + 8 * g;
            if (i >= p.i.n_out) continue;
            float b[8];
            bias8(MODE == kDenseDx ? nullptr : p.bias, i, b);
#pragma unroll
            for (int n = 0; n < NJ; ++n) {
                const int64_t j = j0 + (wj * NJ + n) * 16 + o;
                if (j >= p.j.n_out) continue;
                float v[8];
                pair8(acc, pr, n, v);
                if (MODE != kDenseDx) {
                    float r[8] = {};
                    if (p.res) unpack8<T>(load8<T>(p.res + j * p.ld_res + i, p.i.n_out - i), r);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float slope = 1.f;
                        if (MODE == kDenseFwd) {
                            v[e] = act_eval<false>(v[e] + b[e], p.act, p.beta, slope) + r[e];
                        } else {
                            act_eval<true>(v[e] + b[e], p.act, p.beta, slope);
                            v[e] = r[e] * slope;
                        }
                    }
                }
                store8<T>(p.out + j * p.ld_out + i, v, p.i.n_out - i);
            }
        }
    }
}

// dw (and the column sums db) = the sums of the slabs' partials, in their order
template <typename T>
__global__ void __launch_bounds__(256)
dense_dw_sum_kernel(const float *__restrict__ partial, int slabs, int64_t n, int64_t n_db, T *__restrict__ dw, T *__restrict__ db) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, stride = n + n_db;
    if (e >= stride) return;
    float s[4] = {};
    int k = 0;
    for (; k + 3 < slabs; k += 4)
#pragma unroll
        for (int u = 0; u < 4; ++u) s[u] += partial[(k + u) * stride + e];
    for (; k < slabs; ++k) s[0] += partial[k * stride + e];
    const float v = (s[0] + s[1]) + (s[2] + s[3]);
    if (e < n) dw[e] = (T)v;
    else db[e - n] = (T)v;
}

// ---- few rows -------------------------------------------------------------------------------------------------------------------------
// A handful of rows leaves the tiles above with a few workgroups that wait on memory.  Here a workgroup makes 16 features (gated: 16 of
// both matrices) of all rows, its four waves share the reduction in steps of 32 and read their operands straight into fragments; the
// partial sums meet in LDS.  The weights are read once, by n_i / 16 workgroups at a time.
template <typename T, bool GATED, int NJ>
__global__ void __launch_bounds__(256)
dense_few_kernel(const DenseArgs<T> p) {
    constexpr int P = Mma<T>::P, NG = GATED ? 2 : 1;
    __shared__ float lds[4][NG * NJ][16][17];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, o = lane & 15, g = lane >> 4;
    const int64_t i0 = (int64_t)blockIdx.x * 16, K = p.i.n_red;
    const int64_t iw = i0 + o < p.i.n_out ? i0 + o : p.i.n_out - 1;
    const T *wp[2] = {p.i.a + iw * p.i.ld, GATED ? p.i.b + iw * p.i.ld : nullptr};
    const T *xp[NJ];
#pragma unroll
    for (int n = 0; n < NJ; ++n) {
        const int64_t j = 16 * n + o;
        xp[n] = p.j.a + (j < p.j.n_out ? j : p.j.n_out - 1) * p.j.ld;
    }
    f4v acc[NG][NJ];
#pragma unroll
    for (int q = 0; q < NG; ++q)
#pragma unroll
        for (int n = 0; n < NJ; ++n) acc[q][n] = f4v{0.f, 0.f, 0.f, 0.f};
    auto step = [&](int64_t k, auto full) {
        s8v a[NG][P], b[NJ][P];
#pragma unroll
        for (int q = 0; q < NG; ++q) planes8<T>(full() ? load8<T>(wp[q] + k) : load8<T>(wp[q] + k, K - k), a[q]);
#pragma unroll
        for (int n = 0; n < NJ; ++n) planes8<T>(full() ? load8<T>(xp[n] + k) : load8<T>(xp[n] + k, K - k), b[n]);
#pragma unroll
        for (int q = 0; q < NG; ++q)
#pragma unroll
            for (int n = 0; n < NJ; ++n) acc[q][n] = Mma<T>::mma(a[q], b[n], acc[q][n]);
    };
    const int64_t n_full = K / 32;   // whole steps of 32
    int64_t s = wave;
    for (; s + 12 < n_full; s += 16) {      // four steps' loads in flight
#pragma unroll
        for (int u = 0; u < 4; ++u) step(32 * (s + 4 * u) + 8 * g, std::true_type{});
    }
    for (; s < n_full; s += 4) step(32 * s + 8 * g, std::true_type{});
    if (K % 32 && (n_full & 3) == wave) step(32 * n_full + 8 * g, std::false_type{});
#pragma unroll
    for (int q = 0; q < NG; ++q)
#pragma unroll
        for (int n = 0; n < NJ; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) lds[wave][q * NJ + n][o][4 * g + r] = acc[q][n][r];
    __syncthreads();
    const int li = tid & 15, lj = tid >> 4;
    const int64_t i = i0 + li;
    if (i >= p.i.n_out) return;
#pragma unroll
    for (int n = 0; n < NJ; ++n) {
        const int64_t j = 16 * n + lj;
        if (j >= p.j.n_out) break;
        float v[NG];
#pragma unroll
        for (int q = 0; q < NG; ++q) {
            v[q] = (lds[0][q * NJ + n][lj][li] + lds[1][q * NJ + n][lj][li]) + (lds[2][q * NJ + n][lj][li] + lds[3][q * NJ + n][lj][li]);
            const T *b = q ? p.bias2 : p.bias;
            if (b) v[q] += (float)b[i];
        }
        float slope, y = act_eval<false>(v[0], p.act, p.beta, slope);
        if (GATED) y *= v[NG - 1];
        else if (p.res) y += (float)p.res[j * p.ld_res + i];
        p.out[j * p.ld_out + i] = (T)y;
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------------
constexpr int64_t kFewRows = 32;

// Tiles: 128 x 128 (four waves of 64 x 64) where they fill the chip, else 64 x 64 (four waves of 64 x 16): a product of few tiles is
// bound by how many CUs take part.
template <typename T, int MODE>
static int launch_tiles(DenseArgs<T> &p, hipStream_t st) {
    constexpr bool GATED = MODE == kGatedFwd || MODE == kGatedBwd;
    const int64_t oi = GATED ? p.i.n_out * 2 : p.i.n_out;
    const bool big = ceil_div<int64_t>(oi, 128) * ceil_div<int64_t>(p.j.n_out, 128) * (MODE == kDenseDw ? p.slabs : 1) >= 256;
    const int b = big ? 128 : 64;
    p.tiles_i = ceil_div<int64_t>(oi, b);
    p.tiles = p.tiles_i * ceil_div<int64_t>(p.j.n_out, b) * (MODE == kDenseDw ? p.slabs : 1);
    const int64_t grid = ceil_div<int64_t>(p.tiles, 8) * 8;
    if (grid > 0x7fffffff) return einval("dense: too many tiles for one launch");
    if (big) hipLaunchKernelGGL((dense_kernel<T, MODE, 2, 2, 4, 4>), dim3((unsigned)grid), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((dense_kernel<T, MODE, 1, 4, 4, 1>), dim3((unsigned)grid), dim3(256), 0, st, p);
    return check_launch("dense");
}

// slabs of a weight gradient (rows cut so that the tiles times the slabs fill the chip twice over, none shorter than 256 rows)
static inline int dense_dw_slabs(int64_t rows, int64_t n, int64_t k) {
    const int64_t tiles = ceil_div<int64_t>(n, 128) * ceil_div<int64_t>(k, 128);
    int64_t s = ceil_div<int64_t>(512, tiles);
    const int64_t most = ceil_div<int64_t>(rows, 256);
    s = s < most ? s : most;
    return (int)(s > 0 ? s : 1);
}

template <typename T>
struct DenseOps {
    static int fwd(const void *x, int64_t ld_x, const void *w, const void *b, const void *res, int64_t ld_res, void *y, int act, float beta, int64_t rows, int K, int N,
                   hipStream_t st);
    static int dz(const void *x, int64_t ld_x, const void *w, const void *b, const void *dy, int64_t ld_dy, void *dz, int act, float beta, int64_t rows, int K, int N,
                  hipStream_t st);
    static int dx(const void *dz, int64_t ld_dz, const void *w, const void *w2, void *dx, int64_t rows, int N, int K, hipStream_t st);
    static int dw(const void *dz, int64_t ld_dz, const void *x, int64_t ld_x, void *dw, void *db, float *scratch, int64_t rows, int N, int K, hipStream_t st);
    static int gated_fwd(const void *x, int64_t ld_x, const void *wg, const void *wu, const void *bg, const void *bu, void *h, int act, float beta, int64_t rows, int K,
                         int H, hipStream_t st);
    static int gated_bwd(const void *x, int64_t ld_x, const void *wg, const void *wu, const void *bg, const void *bu, const void *dy, int64_t ld_dy, const void *wd,
                         void *dgu, int act, float beta, int64_t rows, int K, int H, int N, hipStream_t st);
};

}  // namespace arcn
