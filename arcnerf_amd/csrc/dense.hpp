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
// Nothing of the forward pass but its inputs (and h) is kept for the backward: a pre-activation is computed again, in f32, in the tile that
// needs its slope.  A 16-bit layer's saved one would have been rounded to its type and cost its bytes twice (2 K operations per 4 bytes: at
// K = 256 a tile computes it faster than HBM would return it).  An f32 layer loses nothing by saving it and pays for the product from K of
// about 160 on (at 256 2.7 ps an element at the split products' rate below against 1.7 for its 8 bytes): what it gets is the memory.  The
// gated backward computes g, u AND dh of a tile in registers; only dg and du, each rounded once, are written.  (That rounding, and h's and
// dz's, are the 16-bit types' only ones between a call's inputs and its results: dx and dW are made from the rounded values, which costs
// them as much again as their own rounding, 1.4 x in all; in f32 these tensors would be twice the traffic and the products six times the
// operations.  The bias gradients are sums of the values before that.)
//
// f32 operands are split into three bf16 planes on their way into LDS, x = hi + mid + lo, and six products (hi hi, hi mid, mid hi, hi lo,
// lo hi, mid mid) are accumulated in f32; what is dropped is below 2^-25 of a product.  A sixth of the bf16 rate, 193 TFLOP/s at the 1156 of a
// large library product here, whose f32 products reach 154; the gated forward 32768 x 256 -> 2 x 512 runs at 155 (111 us).  Infinities, NaN and
// what rounds to infinity as bf16 (from 3.39e38 on) in such an operand give NaN.
//
// A lane's accumulators of one MFMA tile are 4 consecutive features of a row; the tiles are taken in pairs and lane rows 1 and 3 of the
// first are swapped with lane rows 0 and 2 of the second (v_permlane16_swap_b32), which leaves 8 CONSECUTIVE features of one row in each
// lane: residual, gradient and result move as 16 bytes per lane, 64 bytes per row and instruction.
#pragma once

#include <type_traits>

#include "elem.hpp"
#include "partials.hpp"

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

// FAST (16-bit results): the exponential without that correction (x 2^-24 of itself, 2^-18 at most where the result counts) and
// erfc(x) = t P(t) e^(-x^2), t = 1 / (1 + 0.38 x), which shares its exponential with the slope: a third of the instructions of an epilogue that
// is all of a wide tile's vector work.  P: our own fit of degree 6, by the largest error relative to erfc in its tail (1.5e-5, 2^-5 of half a
// step of f16, where a form with a small absolute error loses steps) and absolute towards zero (2.5e-7).
template <int ACT, bool SLOPE, bool FAST>
__device__ __forceinline__ float act_eval(float z, float beta, float inv_beta, float &slope) {
    if constexpr (ACT == ARCN_ACT_RELU) {
        if (SLOPE) slope = z <= 0.f ? 0.f : 1.f;
        return z <= 0.f ? 0.f : z;      // (a NaN stays one)
    } else if constexpr (FAST && ACT == ARCN_ACT_SIGMOID && !SLOPE) {
        return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
    } else if constexpr (FAST && ACT == ARCN_ACT_SILU) {
        const float q = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
        if (SLOPE) slope = q * fmaf(z, 1.f - q, 1.f);
        return z * q;
    } else if constexpr (ACT == ARCN_ACT_SIGMOID || ACT == ARCN_ACT_SILU) {
        // (the slope as e q^2: q (1 - q) cancels from z of about 8 on, its digits are gone at 17)
        const float e = FAST ? __builtin_amdgcn_exp2f(fabsf(z) * -1.44269504f) : exp_hw(-fabsf(z)), q = __builtin_amdgcn_rcpf(1.f + e), eq = e * q;
        const bool up = z >= 0.f;
        const float s = up ? q : eq;
        if constexpr (ACT == ARCN_ACT_SIGMOID) {
            if (SLOPE) slope = eq * q;
            return s;
        } else {
            if (SLOPE) slope = s * (1.f + z * (up ? eq : q));
            return z * s;
        }
    } else if constexpr (ACT == ARCN_ACT_SOFTPLUS) {
        // log1p(t) = log(u) t / (u - 1) with u = fl(1 + t): the rounding of 1 + t cancels
        const float bz = beta * z;
        const float t = FAST ? __builtin_amdgcn_exp2f(fabsf(bz) * -1.44269504f) : exp_hw(-fabsf(bz)), u = 1.f + t;
        if (SLOPE) {
            const float q = __builtin_amdgcn_rcpf(u);
            slope = bz > 20.f ? 1.f : (bz >= 0.f ? q : t * q);
        }
        const float l = u == 1.f ? t : __logf(u) * (t * __builtin_amdgcn_rcpf(u - 1.f));
        return bz > 20.f ? z : (fmaxf(bz, 0.f) + l) * inv_beta;
    } else if constexpr (FAST && ACT == ARCN_ACT_GELU) {
        const float e = __builtin_amdgcn_exp2f(z * z * -0.721347520f);             // e^(-z^2 / 2)
        const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.26870057f, 1.f));   // 1 / (1 + 0.38 |z| / sqrt 2)
        float q = fmaf(t, -0.0584391914f, 0.152983919f);
        q = fmaf(t, q, -0.0142182391f);
        q = fmaf(t, q, 0.109800145f);
        q = fmaf(t, q, 0.0951927528f);
        q = fmaf(t, q, 0.107490107f);
        q = fmaf(t, q, 0.107190385f) * t * e;                                      // half of erfc(|z| / sqrt 2)
        const float cdf = z > 0.f ? 1.f - q : q;
        if (SLOPE) slope = fmaf(z * 0.398942280f, e, cdf);
        return z * cdf;
    } else if constexpr (ACT == ARCN_ACT_GELU) {
        const float cdf = 0.5f * erfcf(z * -0.707106781f);      // (1 + erf cancels for negative z: nothing of it is left at -6)
        if (SLOPE) slope = fmaf(z * 0.398942280f, exp_hw(-0.5f * z * z), cdf);
        return z * cdf;
    } else {
        if (SLOPE) slope = 1.f;
        return z;
    }
}

// f(activation as a compile-time number): the choice is made once per tile, not once per element (64 copies of a switch over all the
// activations do not fit the instruction cache: a 256-wide bf16 layer of 262144 rows took 249 us with them, 135 without)
template <typename Fn>
__device__ __forceinline__ void with_act(int act, Fn &&f) {
    switch (act) {
    case ARCN_ACT_RELU: f(std::integral_constant<int, ARCN_ACT_RELU>{}); break;
    case ARCN_ACT_SIGMOID: f(std::integral_constant<int, ARCN_ACT_SIGMOID>{}); break;
    case ARCN_ACT_SOFTPLUS: f(std::integral_constant<int, ARCN_ACT_SOFTPLUS>{}); break;
    case ARCN_ACT_SILU: f(std::integral_constant<int, ARCN_ACT_SILU>{}); break;
    case ARCN_ACT_GELU: f(std::integral_constant<int, ARCN_ACT_GELU>{}); break;
    default: f(std::integral_constant<int, ARCN_ACT_NONE>{}); break;
    }
}

// ---- operand fragments ------------------------------------------------------------------------------------------------------------------
template <typename T>
struct Mma;
template <>
struct Mma<__bf16> {
    static constexpr int P = 1, BK = 64, NBUF = 2;
    static __device__ __forceinline__ f4v mma(const s8v *a, const s8v *b, f4v c, float) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[0]), __builtin_bit_cast(bf16x8, b[0]), c, 0, 0, 0);
    }
    static constexpr short kOne = 0x3f80;
};
template <>
struct Mma<_Float16> {
    static constexpr int P = 1, BK = 64, NBUF = 2;
    static __device__ __forceinline__ f4v mma(const s8v *a, const s8v *b, f4v c, float) {
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
    // The six terms of 32 reduction elements among themselves, smallest first, then ONE addition (rounded to nearest) to the running sum:
    // six accumulations straight into it would round at its size six times.  The matrix cores round their sums downwards, a bias that
    // adds up in a column sum over many rows: the I operand of every other step comes negated (sign = -1), which turns it around.
    static __device__ __forceinline__ f4v mma(const s8v *a, const s8v *b, f4v c, float sign) {
        f4v t = {0.f, 0.f, 0.f, 0.f};
        t = one(a[1], b[1], t);
        t = one(a[0], b[2], t);
        t = one(a[2], b[0], t);
        t = one(a[0], b[1], t);
        t = one(a[1], b[0], t);
        t = one(a[0], b[0], t);
#pragma unroll
        for (int r = 0; r < 4; ++r) c[r] = fmaf(sign, t[r], c[r]);
        return c;
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
// the branch-free form (rows of at least 8 elements): tail8 loads, tail8_fix puts in place
template <typename T>
__device__ __forceinline__ Raw8<T> tail8(const T *p, int64_t left) {
    Raw8<T> r;
#pragma unroll
    for (int h = 0; h < (int)sizeof(T) / 2; ++h) r.v[h] = load16(tail_at<T>(p + h * Elem<T>::VEC, left - h * Elem<T>::VEC));
    return r;
}
template <typename T>
__device__ __forceinline__ void tail8_fix(Raw8<T> &r, int64_t left) {
#pragma unroll
    for (int h = 0; h < (int)sizeof(T) / 2; ++h) r.v[h] = tail_fix<T>(r.v[h], left - h * Elem<T>::VEC);
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
__device__ __forceinline__ void planes8(const Raw8<T> &r, s8v *pl, float sign = 1.f) {
    if constexpr (sizeof(T) == 2) {
        pl[0] = __builtin_bit_cast(s8v, r.v[0]);
    } else {
        float v[8];
        unpack8<T>(r, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= sign;
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

// R: output indices of the tile.  GATED: its rows alternate, in groups of 32, between two matrices.
template <typename T, int R, int THREADS, bool TR, bool GATED>
struct Tile {
    static constexpr int BK = Mma<T>::BK, P = Mma<T>::P;
    static constexpr int CHUNKS = R * BK / 8, N = (CHUNKS + THREADS - 1) / THREADS;   // chunk: 8 elements
    static constexpr int PER_ROW = TR ? R / 8 : BK / 8;                              // chunks of an LDS row (TR: a reduction row)
    static constexpr int kElems = P * R * BK;                                        // of one LDS buffer
    Raw8<T> raw[N];

    // chunk c of LDS row `row` is kept at chunk c ^ swizzle(row): the 8 lanes that one cycle of a 16-byte read serves, and the 16 of an
    // 8-byte transposing read (4 rows), fall on different banks.  (Its own inverse.  A row of 4 chunks shares its 128 bytes with the next.)
    static __device__ __forceinline__ int place(int row, int c) {
        if (TR) return 8 * (row * PER_ROW + (PER_ROW >= 8 ? c ^ ((row & 3) << 1) : c));
        if (BK == 64) return 8 * (row * PER_ROW + (c ^ (row & 7)));
        return 8 * ((row * PER_ROW + c) ^ ((row >> 1) & 3));
    }

    // address of chunk c of LDS row `row` when the reduction stands at k0
    static __device__ __forceinline__ const T *source(const Operand<T> &op, int64_t out0, int64_t k0, int row, int c) {
        if (!TR) {
            // (a row behind the operand's last one is computed and dropped: it reads the last one)
            int64_t out = out0 + (GATED ? ((row >> 6) * 32 + (row & 31)) : row);
            out = out < op.n_out ? out : op.n_out - 1;
            return (GATED && (row & 32) ? op.b : op.a) + out * op.ld + k0 + 8 * c;
        }
        const int64_t r = k0 + row;
        return (op.b && r >= op.split ? op.b + (r - op.split) * op.ld : op.a + r * op.ld) + out0 + 8 * c;
    }

    // How a step is loaded (the same for the whole workgroup): all of it there; some of it behind an end of the operand, rows of 8 elements or
    // more (no branches: a lane that waited for its tail would hold up the loads of the wave); narrow rows, element by element.
    enum How { kWhole, kTail, kNarrow };
    static __device__ __forceinline__ How how(const Operand<T> &op, int64_t out0, int64_t k0, int64_t k_end) {
        if (k0 + BK <= k_end && (!TR || out0 + R <= op.n_out)) return kWhole;
        return (TR ? op.n_out : op.n_red) >= 8 ? kTail : kNarrow;
    }
    // elements of its row from chunk c of LDS row `row` on; 0 or less: none
    static __device__ __forceinline__ int64_t left(const Operand<T> &op, int64_t out0, int64_t k0, int64_t k_end, int row, int c) {
        return TR ? (k0 + row < k_end ? op.n_out - (out0 + 8 * c) : 0) : k_end - (k0 + 8 * c);
    }

    __device__ __forceinline__ void fetch(const Operand<T> &op, int64_t out0, int64_t k0, int64_t k_end, int tid) {
        const How h = how(op, out0, k0, k_end);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int q = tid + n * THREADS;
            if (CHUNKS % THREADS && q >= CHUNKS) break;
            const int row = q / PER_ROW, c = q % PER_ROW;
            if (h == kWhole) {
                raw[n] = load8<T>(source(op, out0, k0, row, c));
            } else if (h == kTail) {
                // (a reduction row behind the last one reads the last one; stash makes it zero)
                const int at = TR && k0 + row >= k_end ? (int)(k_end - 1 - k0) : row;
                raw[n] = tail8<T>(source(op, out0, k0, at, c), left(op, out0, k0, k_end, at, c));
            } else {
                raw[n] = load8<T>(source(op, out0, k0, row, c), left(op, out0, k0, k_end, row, c));
            }
        }
    }

    // sums (TR, f32; or NULL): the thread's 8 output indices' sums over the rows that it loads (its chunk is the same in all of them)
    __device__ __forceinline__ void stash(const Operand<T> &op, int64_t out0, int64_t k0, int64_t k_end, short *lds, int tid, float sign = 1.f, float *sums = nullptr) {
        if (how(op, out0, k0, k_end) == kTail) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int q = tid + n * THREADS;
                tail8_fix<T>(raw[n], left(op, out0, k0, k_end, q / PER_ROW, q % PER_ROW));
            }
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int q = tid + n * THREADS;
            if (CHUNKS % THREADS && q >= CHUNKS) break;
            if (TR && P == 3 && sums) {
                static_assert(THREADS % PER_ROW == 0, "a thread keeps its chunk");
                float v[8];
                unpack8<T>(raw[n], v);
#pragma unroll
                for (int e = 0; e < 8; ++e) sums[e] += v[e];
            }
            s8v pl[P];
            planes8<T>(raw[n], pl, sign);
#pragma unroll
            for (int p = 0; p < P; ++p) *reinterpret_cast<s8v *>(lds + p * R * BK + place(q / PER_ROW, q % PER_ROW)) = pl[p];
        }
    }

    // memory to LDS without registers (16-bit types, 16-byte aligned rows, whole steps of the reduction): a wave's 64 chunks land in
    // consecutive places, so the lane whose place it is asks for the chunk that belongs there
    static __device__ __forceinline__ void copy(const Operand<T> &op, int64_t out0, int64_t k0, short *lds, int tid) {
        const int wave0 = __builtin_amdgcn_readfirstlane(tid & ~63);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (CHUNKS % THREADS && n * THREADS + wave0 >= CHUNKS) break;
            const int q = tid + n * THREADS, row = q / PER_ROW;
            int c = (place(row, q % PER_ROW) >> 3) - row * PER_ROW;
            int64_t o0 = out0;
            if (TR && o0 + 8 * c + 8 > op.n_out) o0 = op.n_out - 8 - 8 * c;   // (dropped outputs read the last ones)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)source(op, o0, k0, row, c),
                                             (__attribute__((address_space(3))) void *)(lds + 8 * (n * THREADS + wave0)), 16, 0, 0);
        }
    }

    // fragment of MFMA tile m (from tile row / column `base`) at reduction step kk (32 elements): lane l holds output index l % 16,
    // reduction elements 8 (l / 16) .. + 7
    static __device__ __forceinline__ void frag(const short *lds, int base, int m, int kk, int lane, s8v *f) {
        const int o = lane & 15, g = lane >> 4;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const short *pl = lds + p * R * BK;
            if (!TR) {
                f[p] = *reinterpret_cast<const s8v *>(pl + place(base + 16 * m + o, 4 * kk + g));
            } else {
                // lane o of a group of 16 asks for 4 output indices (quad o % 4) of reduction row o / 4 and receives 4 reduction rows of
                // output index o
                const int col = base + 16 * m + 4 * (o & 3);
                s4v h[2];
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) s4v *)(pl + place(32 * kk + 8 * g + 4 * e + (o >> 2), col >> 3) + (col & 4)));
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
    T *out2;                 // dense_dz_dx_kernel: dx
    int64_t ld_out2;
    float *partial;          // kDenseDw: [slab][n_j * n_i (+ n_j column sums of j)]
    int want_sums;
    // Column sums of dz (dg | du) before they are rounded, 16-bit types: [n_sums][features], a row per workgroup of rows.  Written by kDenseDz,
    // kGatedBwd and dense_dz_dx_kernel (or NULL), read by kDenseDw in place of its own sums of j (or NULL).
    float *sums;
    int64_t n_sums;
    int act;
    float beta, inv_beta;
    uint32_t tiles_i, tiles_j, tiles;  // tiles: of the whole product (times the slabs)
    int slabs;
};

// blockIdx -> tile: workgroups are dealt to the 8 XCDs in turn, so each XCD gets a contiguous range of tiles and the tiles that share
// their J rows (the large operand) meet in one L2 (gridDim.x is a multiple of 8; y: wide_grid)
__device__ __forceinline__ uint32_t xcd_tile() { return blockIdx.y * gridDim.x + (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3); }

// the 8 consecutive features that a lane ends up with of a pair of MFMA tiles (every lane takes part)
__device__ __forceinline__ void swap8(f4v a, f4v b, float *v) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const auto sw = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, (float)a[r]), __builtin_bit_cast(uint32_t, (float)b[r]), false, false);
        v[r] = __builtin_bit_cast(float, (uint32_t)sw[0]);
        v[4 + r] = __builtin_bit_cast(float, (uint32_t)sw[1]);
    }
}

// the sum over the 16 lanes of a row (the 16 rows of an MFMA tile), the same value in each of them
__device__ __forceinline__ float sum16(float v) {
    v += dpp_take<0xB1>(0.f, v);
    v += dpp_take<0x4E>(0.f, v);
    v += dpp_take<0x141>(0.f, v);
    return v + dpp_take<0x140>(0.f, v);
}

// ASYNC: operands straight from memory to LDS (Tile::copy; launch_tiles checks what it needs)
template <typename T, int MODE, int WI, int WJ, int MI, int NJ, bool ASYNC>
__global__ void __launch_bounds__(64 * WI *WJ, 2)
dense_kernel(const DenseArgs<T> p) {
    constexpr int THREADS = 64 * WI * WJ, BI = 16 * MI * WI, BJ = 16 * NJ * WJ;
    constexpr int BK = Mma<T>::BK, P = Mma<T>::P, NBUF = Mma<T>::NBUF;
    constexpr bool GATED = MODE == kGatedFwd || MODE == kGatedBwd;
    constexpr bool I_TR = MODE == kDenseDx || MODE == kDenseDw, J_TR = MODE == kDenseDw;
    constexpr int OUT_I = GATED ? BI / 2 : BI;      // features per tile
    typedef Tile<T, BI, THREADS, I_TR, GATED> TI;
    typedef Tile<T, BJ, THREADS, J_TR, false> TJ;
    typedef Tile<T, BI / 2, THREADS, true, false> TI2;
    constexpr int BUF = TI::kElems + TJ::kElems;
    __shared__ __attribute__((aligned(16))) short lds[NBUF * BUF];

    const uint32_t t = xcd_tile();
    if (t >= p.tiles) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wi = wave % WI, wj = wave / WI;
    uint32_t rest = t / p.tiles_i;
    const int64_t i0 = (int64_t)(t - rest * p.tiles_i) * OUT_I;
    int64_t slab = 0, k_lo = 0, k_hi = p.i.n_red;
    if (MODE == kDenseDw) {
        slab = rest / p.tiles_j;
        rest -= (uint32_t)slab * p.tiles_j;
        const int64_t per = (ceil_div_dev(p.i.n_red, p.slabs) + BK - 1) / BK * BK;
        k_lo = slab * per;
        k_hi = k_lo + per < p.i.n_red ? k_lo + per : p.i.n_red;
    }
    const int64_t j0 = (int64_t)rest * BJ;

    f4v acc[MI][NJ];
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NJ; ++n) acc[m][n] = f4v{0.f, 0.f, 0.f, 0.f};
    // column sums of the J operand (the bias gradient), by the tiles of the first i: 16-bit types by a product with ones (the waves of the first
    // wi), f32 as its rows are staged (8 registers instead of 16)
    constexpr bool SUM_MMA = MODE == kDenseDw && P == 1, SUM_ADD = MODE == kDenseDw && P == 3;
    f4v sums[SUM_MMA ? NJ : 1];
    float add_sums[SUM_ADD ? 8 : 1] = {};
#pragma unroll
    for (int n = 0; n < (SUM_MMA ? NJ : 1); ++n) sums[n] = f4v{0.f, 0.f, 0.f, 0.f};
    const bool given_sums = SUM_MMA && p.want_sums && i0 == 0 && p.sums;
    const bool my_sums = MODE == kDenseDw && p.want_sums && i0 == 0 && (wi == 0 || SUM_ADD) && !given_sums;   // wave-uniform

    // given column sums: the slab's share of their rows, THREADS / BJ threads to a column (in front of the product, which hides the loads)
    float given = 0.f;
    if constexpr (SUM_MMA) {
        if (given_sums && j0 + tid % BJ < p.j.n_out) {
            const int64_t lo = p.n_sums * slab / p.slabs, hi = p.n_sums * (slab + 1) / p.slabs;
#pragma unroll 4
            for (int64_t k = lo + tid / BJ; k < hi; k += THREADS / BJ) given += p.sums[k * p.j.n_out + j0 + tid % BJ];
        }
    }

    // after the swap a lane holds 8 features of a pair of tiles from 32 pr + f8, row o
    const int g = lane >> 4, o = lane & 15, f8 = 16 * (g & 1) + 8 * (g >> 1);
    // residual (or dy) of the lane's results.  16-bit types with registers to spare fetch it in front of the product, which hides the
    // latency; else the registers are free only behind it
    constexpr bool RES = MODE == kDenseFwd || MODE == kDenseDz;
    constexpr bool RES_EARLY = RES && sizeof(T) == 2 && MI * NJ <= 16;
    Raw8<T> res[RES ? MI / 2 : 1][RES ? NJ : 1];
    const bool inner = i0 + OUT_I <= p.i.n_out && j0 + BJ <= p.j.n_out;    // a whole tile
    auto fetch_res = [&]() {
        if constexpr (RES) {
#pragma unroll
            for (int pr = 0; pr < MI / 2; ++pr)
#pragma unroll
                for (int n = 0; n < NJ; ++n) {
                    const int64_t i = i0 + wi * 16 * MI + 32 * pr + f8, j = j0 + (wj * NJ + n) * 16 + o;
                    const T *src = p.res + j * p.ld_res + i;
                    if (inner) res[pr][n] = load8<T>(src);
                    else if (p.i.n_out >= 8) res[pr][n] = tail8<T>(j < p.j.n_out ? src : src + (p.j.n_out - 1 - j) * p.ld_res, p.i.n_out - i);
                    else res[pr][n] = load8<T>(src, j < p.j.n_out ? p.i.n_out - i : 0);
                }
        }
    };
    if (RES_EARLY && p.res) fetch_res();

    auto step = [&](auto &ti, auto &tj, const short *buf, auto &c, int64_t k_left, float sign = 1.f) {
        typedef std::remove_reference_t<decltype(ti)> Ti;
        typedef std::remove_reference_t<decltype(tj)> Tj;
        constexpr int M = sizeof(c) / sizeof(c[0]);
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk) {
            if (kk > 0 && 32 * kk >= k_left) break;
            s8v b[NJ][P];
#pragma unroll
            for (int n = 0; n < NJ; ++n) Tj::frag(buf + TI::kElems, wj * 16 * NJ, n, kk, lane, b[n]);
#pragma unroll
            for (int m = 0; m < M; ++m) {
                s8v a[P];
                Ti::frag(buf, wi * 16 * M, m, kk, lane, a);
#pragma unroll
                for (int n = 0; n < NJ; ++n) c[m][n] = Mma<T>::mma(a, b[n], c[m][n], sign);
            }
            if (SUM_MMA && my_sums) {
                const short one = Mma<T>::kOne;
                s8v ones[P] = {};
                ones[0] = s8v{one, one, one, one, one, one, one, one};
#pragma unroll
                for (int n = 0; n < NJ; ++n) sums[n] = Mma<T>::mma(ones, b[n], sums[n], 1.f);
            }
        }
    };
    auto product = [&](auto &ti, auto &tj, const Operand<T> &oi, const Operand<T> &oj, auto &c) {
        const int64_t n_steps = k_lo < k_hi ? (k_hi - k_lo + BK - 1) / BK : 0;
        if constexpr (NBUF == 1) {
            if (n_steps > 0) {
                ti.fetch(oi, i0, k_lo, k_hi, tid);
                tj.fetch(oj, j0, k_lo, k_hi, tid);
            }
            for (int64_t s = 0; s < n_steps; ++s) {
                const int64_t k = k_lo + (s + 1) * BK;
                const float sign = s & 1 ? -1.f : 1.f;
                ti.stash(oi, i0, k - BK, k_hi, lds, tid, sign);
                tj.stash(oj, j0, k - BK, k_hi, lds + TI::kElems, tid, 1.f, SUM_ADD && my_sums ? add_sums : nullptr);
                __syncthreads();
                if (s + 1 < n_steps) {
                    ti.fetch(oi, i0, k, k_hi, tid);
                    tj.fetch(oj, j0, k, k_hi, tid);
                }
                step(ti, tj, lds, c, BK, sign);
                __syncthreads();
            }
        } else {
            // step s + 1 is on its way to the other buffer while step s is computed; a buffer is written again behind the barrier that
            // follows its last read.  A last partial step goes through registers, where what lies behind the end is made zero.
            auto through_regs = [&](int64_t s) {
                ti.fetch(oi, i0, k_lo + s * BK, k_hi, tid);
                tj.fetch(oj, j0, k_lo + s * BK, k_hi, tid);
            };
            auto put = [&](int64_t s) {
                ti.stash(oi, i0, k_lo + s * BK, k_hi, lds + (s & 1) * BUF, tid);
                tj.stash(oj, j0, k_lo + s * BK, k_hi, lds + (s & 1) * BUF + TI::kElems, tid);
                __syncthreads();
            };
            if constexpr (ASYNC) {
                auto copy = [&](int64_t s) {
                    ti.copy(oi, i0, k_lo + s * BK, lds + (s & 1) * BUF, tid);
                    tj.copy(oj, j0, k_lo + s * BK, lds + (s & 1) * BUF + TI::kElems, tid);
                };
                auto landed = [&]() {
                    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
                    __syncthreads();
                };
                const int64_t whole = k_lo < k_hi ? (k_hi - k_lo) / BK : 0;
                if (whole > 0) {
                    copy(0);
                    landed();
                }
                for (int64_t s = 0; s < whole; ++s) {
                    if (s + 1 < whole) copy(s + 1);
                    step(ti, tj, lds + (s & 1) * BUF, c, BK);
                    landed();
                }
                if (whole < n_steps) {
                    through_regs(whole);
                    put(whole);
                    step(ti, tj, lds + (whole & 1) * BUF, c, k_hi - k_lo - whole * BK);
                    __syncthreads();
                }
            } else {
                if (n_steps > 0) {
                    through_regs(0);
                    put(0);
                }
                for (int64_t s = 0; s < n_steps; ++s) {
                    if (s + 1 < n_steps) through_regs(s + 1);
                    step(ti, tj, lds + (s & 1) * BUF, c, k_hi - k_lo - s * BK);
                    if (s + 1 < n_steps) put(s + 1);
                    else __syncthreads();
                }
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

    // ---- epilogue -----------------------------------------------------------------------------------------------------------------------
    // the column sums of what is stored, not rounded: a wave's rows in registers, the WJ waves of a tile in LDS ([wave][column of out])
    constexpr bool SUMS = (MODE == kDenseDz || MODE == kGatedBwd) && sizeof(T) == 2;
    constexpr int SUM_COLS = GATED ? 2 * OUT_I : OUT_I;
    float *const red = reinterpret_cast<float *>(lds);      // behind the products' last barrier
    auto keep_sums = [&](float *v, int col) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = sum16(v[e]);
        if (o == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) red[wj * SUM_COLS + col + e] = v[e];
        }
    };
    auto pair8 = [&](auto &c, int pr, int n, float *v) { swap8(c[2 * pr][n], c[2 * pr + 1][n], v); };
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
#pragma unroll
            for (int pr = 0; pr < MI / 2; ++pr) {
                const int64_t i = i0 + wi * 16 * MI + 32 * pr + f8;
                float v[8];
                pair8(acc, pr, n, v);
                if (j < p.j.n_out) store8<float>(part + j * p.i.n_out + i, v, p.i.n_out - i);
            }
            if (SUM_MMA && my_sums && g == 0 && j < p.j.n_out) part[p.i.n_out * p.j.n_out + j] = sums[n][0];
        }
        if constexpr (SUM_MMA) {
            if (given_sums) {
                float *f = reinterpret_cast<float *>(lds);      // behind the product's last barrier
                f[tid] = given;
                __syncthreads();
                if (tid < BJ && j0 + tid < p.j.n_out) {
                    float v = 0.f;
#pragma unroll
                    for (int k = 0; k < THREADS / BJ; ++k) v += f[k * BJ + tid];
                    part[p.i.n_out * p.j.n_out + j0 + tid] = v;
                }
            }
        }
        if (SUM_ADD && my_sums) {
            float *f = reinterpret_cast<float *>(lds);      // [thread][8]; behind the product's last barrier
#pragma unroll
            for (int e = 0; e < 8; ++e) f[8 * tid + e] = add_sums[e];
            __syncthreads();
            if (tid < BJ && j0 + tid < p.j.n_out) {
                float v = 0.f;
                for (int k = tid >> 3; k < THREADS; k += TJ::PER_ROW) v += f[8 * k + (tid & 7)];
                part[p.i.n_out * p.j.n_out + j0 + tid] = v;
            }
        }
    } else if constexpr (GATED) {
        with_act(p.act, [&](auto A) {
#pragma unroll
        for (int pr = 0; pr < MI / 4; ++pr) {
            const int64_t i = i0 + wi * 8 * MI + 32 * pr + f8;
            float bg[8], bu[8];
            bias8(p.bias, i, bg);
            bias8(p.bias2, i, bu);
            float sg[8] = {}, su[8] = {};
#pragma unroll
            for (int n = 0; n < NJ; ++n) {
                const int64_t j = j0 + (wj * NJ + n) * 16 + o;
                const int64_t left = j < p.j.n_out ? p.i.n_out - i : 0;
                float gv[8], uv[8];
                pair8(acc, 2 * pr, n, gv);      // (every lane takes part in the swaps)
                pair8(acc, 2 * pr + 1, n, uv);
                T *dst = p.out + j * p.ld_out + i;
                if constexpr (MODE == kGatedFwd) {
                    float slope;
#pragma unroll
                    for (int e = 0; e < 8; ++e) gv[e] = act_eval<A(), false, sizeof(T) == 2>(gv[e] + bg[e], p.beta, p.inv_beta, slope) * (uv[e] + bu[e]);
                    store8<T>(dst, gv, left);
                } else {
                    float dh[8];
                    pair8(acc2, pr, n, dh);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float slope;
                        const float a = act_eval<A(), true, sizeof(T) == 2>(gv[e] + bg[e], p.beta, p.inv_beta, slope);
                        gv[e] = dh[e] * (uv[e] + bu[e]) * slope;
                        uv[e] = dh[e] * a;
                    }
                    if (SUMS && p.sums) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            sg[e] += j < p.j.n_out ? gv[e] : 0.f;
                            su[e] += j < p.j.n_out ? uv[e] : 0.f;
                        }
                    }
                    store8<T>(dst, gv, left);
                    store8<T>(dst + p.i.n_out, uv, left);   // du behind dg in a row of 2 H
                }
            }
            if (SUMS && p.sums) {
                keep_sums(sg, wi * 8 * MI + 32 * pr + f8);
                keep_sums(su, OUT_I + wi * 8 * MI + 32 * pr + f8);
            }
        }
        });
    } else {
        if (RES && !RES_EARLY && p.res) fetch_res();
        with_act(RES ? p.act : ARCN_ACT_NONE, [&](auto A) {
#pragma unroll
        for (int pr = 0; pr < MI / 2; ++pr) {
            const int64_t i = i0 + wi * 16 * MI + 32 * pr + f8;
            float b[8];
            bias8(MODE == kDenseDx ? nullptr : p.bias, i, b);
            float sz[8] = {};
#pragma unroll
            for (int n = 0; n < NJ; ++n) {
                const int64_t j = j0 + (wj * NJ + n) * 16 + o;
                float v[8];
                pair8(acc, pr, n, v);
                if constexpr (RES) {
                    float r[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) r[e] = 0.f;
                    if (p.res) {
                        if (!inner && p.i.n_out >= 8) tail8_fix<T>(res[pr][n], p.i.n_out - i);
                        unpack8<T>(res[pr][n], r);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float slope = 1.f;
                        if (MODE == kDenseFwd) {
                            v[e] = act_eval<A(), false, sizeof(T) == 2>(v[e] + b[e], p.beta, p.inv_beta, slope) + r[e];
                        } else {
                            act_eval<A(), true, sizeof(T) == 2>(v[e] + b[e], p.beta, p.inv_beta, slope);
                            v[e] = r[e] * slope;
                        }
                    }
                }
                if (SUMS && p.sums) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) sz[e] += j < p.j.n_out ? v[e] : 0.f;
                }
                store8<T>(p.out + j * p.ld_out + i, v, j < p.j.n_out ? p.i.n_out - i : 0);
            }
            if (SUMS && p.sums) keep_sums(sz, wi * 16 * MI + 32 * pr + f8);
        }
        });
    }
    if constexpr (SUMS) {
        if (p.sums) {
            __syncthreads();
            for (int c = tid; c < SUM_COLS; c += THREADS) {
                const int64_t i = i0 + c % OUT_I;
                if (i >= p.i.n_out) continue;
                float v = 0.f;
#pragma unroll
                for (int k = 0; k < WJ; ++k) v += red[k * SUM_COLS + c];
                p.sums[(int64_t)rest * p.ld_out + (c / OUT_I) * p.i.n_out + i] = v;
            }
        }
    }
}

// ---- few rows -------------------------------------------------------------------------------------------------------------------------
// A handful of rows leaves the tiles above with a few workgroups that wait on memory.  Here a workgroup makes 16 features (gated: 16 of
// both matrices) of up to 32 rows, its four waves share the reduction in steps of 32 and read their operands straight into fragments; the
// partial sums meet in LDS.  The weights are read once per 32 rows, by n_i / 16 workgroups.
// One row, 1024 x 1024 bf16: 3.5 us, 2 MB of weight.
template <typename T, bool GATED, int NJ>
__global__ void __launch_bounds__(256)
dense_few_kernel(const DenseArgs<T> p) {
    constexpr int P = Mma<T>::P, NG = GATED ? 2 : 1;
    __shared__ float lds[4][NG * NJ][16][17];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, o = lane & 15, g = lane >> 4;
    const int64_t i0 = (int64_t)blockIdx.x * 16, j0 = (int64_t)blockIdx.y * 16 * NJ, K = p.i.n_red;
    const int64_t iw = i0 + o < p.i.n_out ? i0 + o : p.i.n_out - 1;
    const T *wp[2] = {p.i.a + iw * p.i.ld, GATED ? p.i.b + iw * p.i.ld : nullptr};
    const T *xp[NJ];
#pragma unroll
    for (int n = 0; n < NJ; ++n) {
        const int64_t j = j0 + 16 * n + o;
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
            for (int n = 0; n < NJ; ++n) acc[q][n] = Mma<T>::mma(a[q], b[n], acc[q][n], 1.f);
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
        const int64_t j = j0 + 16 * n + lj;
        if (j >= p.j.n_out) break;
        float v[NG];
#pragma unroll
        for (int q = 0; q < NG; ++q) {
            v[q] = (lds[0][q * NJ + n][lj][li] + lds[1][q * NJ + n][lj][li]) + (lds[2][q * NJ + n][lj][li] + lds[3][q * NJ + n][lj][li]);
            const T *b = q ? p.bias2 : p.bias;
            if (b) v[q] += (float)b[i];
        }
        float slope, y = 0.f;
        with_act(p.act, [&](auto A) { y = act_eval<A(), false, sizeof(T) == 2>(v[0], p.beta, p.inv_beta, slope); });
        if (GATED) y *= v[NG - 1];
        else if (p.res) y += (float)p.res[j * p.ld_res + i];
        p.out[j * p.ld_out + i] = (T)y;
    }
}

// ---- a weight that stays in LDS: dz and dx in one kernel -----------------------------------------------------------------------------------
// The backward of a layer whose whole weight fits LDS (16-bit types, up to 128 inputs and 512 outputs: 128 KB) moves 8 bytes per 4 K operations:
// it is bound by HBM, and as two products dz alone goes out and comes back.  Here a workgroup loads the weight once and its waves run on
// their own, 16 rows at a time, without another barrier.  A lane's fragments of x come straight from memory (its row's 16 bytes); the
// pre-activation is computed again for 128 features at a time, and because a lane's 8 consecutive features of dz are what the next
// product wants as its J fragment, dx = dz W follows in registers on the SAME weight, read the other way round (transposing reads).  The
// reduction over features is dealt to the lanes as the features fell (f8).  x and dy in, dz and dx out: 128 -> 112, 317560 rows, bf16 71 us
// (4.3 TB/s) against 67 + 47 as two products, 80 with the column sums.  (With 256 inputs the accumulators of dx do not fit beside the rest: 236 us
// against 127 + 75.)
template <typename T, int KS>
__global__ void __launch_bounds__(512, 2)
dense_dz_dx_kernel(const DenseArgs<T> p) {
    constexpr int WAVES = 8, NT = 8, ROW = KS * 4;      // NT: feature tiles of a pass; ROW: 16-byte chunks per LDS row
    extern __shared__ __attribute__((aligned(16))) short w[];      // [N up to a multiple of 128][KS * 32], the bias, if wanted the waves' sums
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, o = lane & 15, g = lane >> 4, f8 = 16 * (g & 1) + 8 * (g >> 1);
    int K = (int)p.i.n_red, N = (int)p.i.n_out;
    const int ks = (K + 31) / 32, n_pad = (N + 127) / 128 * 128;
    T *bias = reinterpret_cast<T *>(w + n_pad * ROW * 8);
    // chunk c of row n at c ^ swizzle(n): 8 rows of one chunk, and 4 rows of two, fall on different banks
    auto swizzle = [](int n) { return ((n & 3) << 1) | ((n >> 2) & 1); };
    for (int q = tid; q < n_pad * ROW; q += 64 * WAVES) {
        const int n = q / ROW, c = q % ROW;
        *reinterpret_cast<u4v *>(w + 8 * (n * ROW + (c ^ swizzle(n)))) = load8<T>(p.i.a + (int64_t)(n < N ? n : 0) * p.i.ld + 8 * c, n < N ? K - 8 * c : 0).v[0];
    }
    for (int n = tid; n < n_pad; n += 64 * WAVES) bias[n] = p.bias && n < N ? p.bias[n] : (T)0.f;
    float *const sums = reinterpret_cast<float *>(bias + n_pad), *const mine = sums + wave * n_pad;
    if (p.sums)
        for (int n = tid; n < WAVES * n_pad; n += 64 * WAVES) sums[n] = 0.f;
    __syncthreads();

    const int64_t rows = p.j.n_out, step = (int64_t)gridDim.x * WAVES * 16;
    u4v x[KS];
    auto fetch = [&](int64_t r) {
        const T *row = p.j.a + (r + o < rows ? r + o : rows - 1) * p.j.ld;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
            if (kk < ks) x[kk] = load16(tail_at<T>(row + 32 * kk + 8 * g, K - 32 * kk - 8 * g));
    };
    int64_t r0 = ((int64_t)blockIdx.x * WAVES + wave) * 16;
    if (r0 < rows) fetch(r0);
    for (; r0 < rows; r0 += step) {
        const int64_t r = r0 + o < rows ? r0 + o : rows - 1;
        const bool live = r0 + o < rows;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
            if (kk < ks && 32 * kk + 32 > K) x[kk] = tail_fix<T>(x[kk], K - 32 * kk - 8 * g);
        f4v dx[2 * KS];
#pragma unroll
        for (int m = 0; m < 2 * KS; ++m) dx[m] = f4v{0.f, 0.f, 0.f, 0.f};
        for (int n0 = 0; n0 < n_pad; n0 += 128) {
            // What the loops could keep they must not: weight and bias are read again for every group, the masks of the last columns and the
            // addresses of the weight's fragments (a few per lane, everything else is in the instructions' offsets) are computed again:
            // hundreds of registers.
            asm volatile("" : "+s"(K), "+s"(N) : : "memory");
            uint32_t af[2], at[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                af[h] = 16 * ((n0 + o) * ROW + ((4 * h + g) ^ swizzle(o)));      // row o, chunk 4 h + g
                asm volatile("" : "+v"(af[h]));
#pragma unroll
                for (int m = 0; m < 4; ++m) {      // row f8 + 4 h + o / 4, column 16 m + 4 (o % 4)
                    at[h][m] = 16 * ((n0 + f8 + 4 * h + (o >> 2)) * ROW + 2 * (m ^ (o >> 2)) + (((o >> 1) & 1) ^ h)) + 8 * (o & 1);
                    asm volatile("" : "+v"(at[h][m]));
                }
            }
            const char *const wb = reinterpret_cast<const char *>(w);
            u4v dy[NT / 2];
#pragma unroll
            for (int pr = 0; pr < NT / 2; ++pr) dy[pr] = load16(tail_at<T>(p.res + r * p.ld_res + n0 + 32 * pr + f8, N - n0 - 32 * pr - f8));
            f4v z[NT];
#pragma unroll
            for (int m = 0; m < NT; ++m) z[m] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                if (kk >= ks) break;
                const s8v b = __builtin_bit_cast(s8v, x[kk]);
#pragma unroll
                for (int m = 0; m < NT; ++m) {
                    const s8v a = *reinterpret_cast<const s8v *>(wb + af[kk & 1] + 16 * m * ROW * 16 + (kk >> 1) * 128);
                    z[m] = Mma<T>::mma(&a, &b, z[m], 1.f);
                }
            }
            if (n0 + 128 >= n_pad && r0 + step < rows) fetch(r0 + step);      // the next rows', behind the rest of this group
            with_act(p.act, [&](auto A) {
#pragma unroll
                for (int pr = 0; pr < NT / 2; ++pr) {
                    float v[8], b[8], q[8];
                    swap8(z[2 * pr], z[2 * pr + 1], v);
                    Elem<T>::unpack(*reinterpret_cast<const u4v *>(bias + n0 + 32 * pr + f8), b);
                    if (n0 + 32 * pr + 32 > N) dy[pr] = tail_fix<T>(dy[pr], N - n0 - 32 * pr - f8);
                    Elem<T>::unpack(dy[pr], q);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float slope;
                        act_eval<A(), true, true>(v[e] + b[e], p.beta, p.inv_beta, slope);
                        v[e] = q[e] * slope;
                    }
                    if (n0 + 32 * pr + 32 > N) {      // features behind the last: zero, whatever an infinity in x made of their slope
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = n0 + 32 * pr + f8 + e < N ? v[e] : 0.f;
                    }
                    dy[pr] = Elem<T>::pack(v);      // dz from here on
                    if (p.sums && n0 + 32 * pr < N) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = sum16(live ? v[e] : 0.f);
                        if (o == 0) {
                            float *const at = mine + n0 + 32 * pr + f8;
#pragma unroll
                            for (int e = 0; e < 8; ++e) at[e] += v[e];
                        }
                    }
                }
            });
#pragma unroll
            for (int pr = 0; pr < NT / 2; ++pr) {
                const int i = n0 + 32 * pr + f8;
                if (N % 32 == 0) {
                    if (live && i < N) store16(p.out + r * p.ld_out + i, dy[pr]);
                } else {
                    store_pack(p.out + r * p.ld_out + i, dy[pr], live ? N - i : 0);
                }
            }
#pragma unroll
            for (int pr = 0; pr < NT / 2; ++pr) {
                if (n0 + 32 * pr >= N) break;
                const s8v b = __builtin_bit_cast(s8v, dy[pr]);
#pragma unroll
                for (int m = 0; m < 2 * KS; ++m) {
                    s4v h[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s4v *)(wb + at[e][m & 3] + 32 * pr * ROW * 16 + (m >> 2) * 128));
                    const s8v a = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
                    dx[m] = Mma<T>::mma(&a, &b, dx[m], 1.f);
                }
            }
        }
#pragma unroll
        for (int pr = 0; pr < KS; ++pr) {
            if (pr >= ks) break;
            const int i = 32 * pr + f8;
            float v[8];
            swap8(dx[2 * pr], dx[2 * pr + 1], v);
            if (K % 32 == 0) {
                if (live) store16(p.out2 + r * p.ld_out2 + i, Elem<T>::pack(v));
            } else {
                store_pack(p.out2 + r * p.ld_out2 + i, Elem<T>::pack(v), live ? K - i : 0);
            }
        }
    }
    if (p.sums) {
        __syncthreads();
        for (int n = tid; n < N; n += 64 * WAVES) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < WAVES; ++k) v += sums[k * n_pad + n];
            p.sums[(int64_t)blockIdx.x * N + n] = v;
        }
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------------
// dense_few_kernel: as long as two of its workgroups to a CU (f32: four) do the product.  One feature block of it costs 3 - 5 us whatever the rows,
// the tiles' first step waits longer and in f32 computes six products on a few CUs.  us here / by tiles, 1024 outputs, at the limit and at twice
// that, reductions of 32, 256, 1024, 4096:  bf16, 256 rows 3.1 / 4.0, 4.1 / 4.4, 8.0 / 7.8, 24 / 34, 512 rows 3.3 / 4.1, 5.5 / 4.5, 13 / 7.9, 45 / 34;
// f32, 512 rows 4.1 / 4.8, 8.8 / 11, 25 / 35, 87 / 124, 1024 rows 6.0 / 5.2, 15 / 12, 46 / 35, 170 / 125.
static inline bool dense_few(int elem_bytes, int64_t rows, int64_t n) {
    return rows <= 1024 && ceil_div<int64_t>(n, 16) * ceil_div<int64_t>(rows, 32) <= (elem_bytes == 2 ? 512 : 1024);
}

// dense_dz_dx_kernel's layers: 16 bits, enough rows for the weight that every CU loads first.  us here / as two products, with the column sums,
// 16384, 24576, 32768 and 65536 rows:  16 -> 16 8.3 / 8.8, 8.4 / 9.6, 8.6 / 12, 16 / 15;  64 -> 64 8.4 / 7.2, 8.8 / 8.4, 9.1 / 15, 16 / 20;
// 128 -> 128 11 / 9.8, 11 / 12, 13 / 16, 23 / 25;  128 -> 512 28 / 24, 30 / 31, 31 / 39, 52 / 62.
constexpr int64_t kStayRows = 24576;
template <typename T>
static bool dense_stays(int64_t rows, int K, int N) {
    return sizeof(T) == 2 && K >= 8 && N >= 8 && K <= 128 && N <= 512 && rows >= kStayRows;
}
template <typename T>
static int launch_dz_dx(DenseArgs<T> &p, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        // the weight's rows of 128 inputs, the bias, the eight waves' sums
        const int bytes = ceil_div<int>((int)p.i.n_out, 128) * 128 * (256 + 2 + (p.sums ? 32 : 0));
        const int64_t g = ceil_div<int64_t>(p.j.n_out, 128), most = bytes <= 80 * 1024 ? 512 : 256;
        p.n_sums = g < most ? g : most;
        hipLaunchKernelGGL((dense_dz_dx_kernel<T, 4>), dim3((unsigned)p.n_sums), dim3(512), bytes, st, p);
    }
    return check_launch("dense_dz");
}

// slabs of a weight gradient: the rows are cut so that tiles times slabs fill the chip (256 x 256 tiles: once; 128 x 128: two workgroups to a
// CU), none shorter than 256 rows.  A rule on sizes and type only: the scratch a caller brings is as large whatever its pointers' alignment.
// (256 x 256 tiles make twice the partial sums, 64 MB of them, and 1.2 x the rate: 271 against 326 us for a 2048 x 512 weight and 65536 rows;
// 101 against 96 us for one of 256 x 256 and 262144 rows.)
static inline bool dense_dw_wide(int elem_bytes, int64_t n, int64_t k) { return elem_bytes == 2 && n >= 256 && k >= 256 && n * k >= 512 * 512; }
static inline int dense_dw_slabs(int elem_bytes, int64_t rows, int64_t n, int64_t k) {
    const int64_t b = dense_dw_wide(elem_bytes, n, k) ? 256 : 128;
    const int64_t tiles = ceil_div<int64_t>(n, b) * ceil_div<int64_t>(k, b);
    int64_t s = (b == 256 ? 256 : 512) / tiles;
    const int64_t most = ceil_div<int64_t>(rows, 256);
    s = s < most ? s : most;
    return (int)(s > 0 ? s : 1);
}

// The tile of a product, by how many there would be: the chip takes part with as many CUs as there are tiles, and a larger tile reads less
// LDS per operation and computes longer on what it has loaded.  (64 x 64: four waves of 64 x 16; 128 x 128: four of 64 x 64, two workgroups
// to a CU; 256 x 256: eight of 128 x 64, one workgroup - gated backward, with its third accumulator, 256 x 192.)  65536 rows, 512 x 2048, bf16,
// 256 against 128: gated forward 361 / 472 us, gated backward 728 / 843, input gradient 351 / 398, 2048 -> 512 152 / 180.  A short reduction
// (below 256) is all epilogue, which only a second workgroup on the CU overlaps; a single step of it is all latency, which five small
// workgroups hide better than two (20 -> 543, 129871 rows, bf16: 118 / 140 us).
template <typename T, int MODE>
static int launch_tiles(DenseArgs<T> &p, hipStream_t st) {
    constexpr bool GATED = MODE == kGatedFwd || MODE == kGatedBwd;
    constexpr bool TR_I = MODE == kDenseDx || MODE == kDenseDw, TR_J = MODE == kDenseDw;
    const int64_t oi = GATED ? p.i.n_out * 2 : p.i.n_out, z = MODE == kDenseDw ? p.slabs : 1;
    auto count = [&](int bi, int bj) { return ceil_div<int64_t>(oi, bi) * ceil_div<int64_t>(p.j.n_out, bj) * z; };
    auto aligned = [](const Operand<T> &q, bool tr) {
        return ((reinterpret_cast<uintptr_t>(q.a) | reinterpret_cast<uintptr_t>(q.b)) & 15) == 0 && q.ld % 8 == 0 && (!tr || q.n_out % 8 == 0);
    };
    const bool async = sizeof(T) == 2 && aligned(p.i, TR_I) && aligned(p.j, TR_J) && (MODE != kGatedBwd || (aligned(p.i2, true) && aligned(p.j2, false)));
    const bool wide = async && (MODE == kDenseDw ? dense_dw_wide(2, p.j.n_out, p.i.n_out) && count(256, 256) >= 128
                                                 : oi >= 256 && p.i.n_red >= 256 && count(256, 256) >= 256);
    const bool one_step = (MODE == kDenseFwd || MODE == kDenseDz) && p.i.n_red <= 32;
    const bool big = count(128, 128) >= 256 && !one_step;
    const int bi = wide ? 256 : big ? 128 : 64, bj = wide ? (MODE == kGatedBwd ? 192 : 256) : bi;
    const int64_t grid = ceil_div<int64_t>(count(bi, bj), 8) * 8;
    if (grid > 0xff000000) return einval("dense: too many tiles for one launch");      // (tile numbers have 32 bits)
    p.tiles_i = (uint32_t)ceil_div<int64_t>(oi, bi);
    p.tiles_j = (uint32_t)ceil_div<int64_t>(p.j.n_out, bj);
    p.tiles = (uint32_t)count(bi, bj);
    if (MODE != kDenseDw) p.n_sums = p.tiles_j;
#define ARCN_DK(WI_, WJ_, MI_, NJ_, A_) hipLaunchKernelGGL((dense_kernel<T, MODE, WI_, WJ_, MI_, NJ_, A_>), wide_grid(grid), dim3(64 * WI_ * WJ_), 0, st, p)
    if constexpr (sizeof(T) == 2) {
        if (wide) ARCN_DK(2, 4, 8, (MODE == kGatedBwd ? 3 : 4), true);
        else if (big && async) ARCN_DK(2, 2, 4, 4, true);
        else if (async) ARCN_DK(1, 4, 4, 1, true);
    }
    if (!async) {
        if (big) ARCN_DK(2, 2, 4, 4, false);
        else ARCN_DK(1, 4, 4, 1, false);
    }
#undef ARCN_DK
    return check_launch("dense");
}

// rows of column sums that a kernel may write: the smallest tile has 64 rows
static inline int64_t dense_sums_rows(int64_t rows) { return ceil_div<int64_t>(rows, 64); }

// sums, n_sums: of DenseArgs; NULL or, 16-bit types, where the column sums go and how many rows of them there are
template <typename T>
struct DenseOps {
    static int fwd(const void *x, int64_t ld_x, const void *w, const void *b, const void *res, int64_t ld_res, void *y, int act, float beta, int64_t rows, int K, int N,
                   hipStream_t st);
    static int dx(const void *dz, int64_t ld_dz, const void *w, const void *w2, void *dx, int64_t rows, int N, int K, hipStream_t st);
    static int dz_dx(const void *x, int64_t ld_x, const void *w, const void *b, const void *dy, int64_t ld_dy, void *dz, void *dx, int act, float beta, float *sums,
                     int64_t *n_sums, int64_t rows, int K, int N, hipStream_t st);
    static int dw(const void *dz, int64_t ld_dz, const void *x, int64_t ld_x, const float *sums, int64_t n_sums, void *dw, void *db, float *scratch, int64_t rows, int N, int K,
                  hipStream_t st);
    static int gated_fwd(const void *x, int64_t ld_x, const void *wg, const void *wu, const void *bg, const void *bu, void *h, int act, float beta, int64_t rows, int K,
                         int H, hipStream_t st);
    static int gated_bwd(const void *x, int64_t ld_x, const void *wg, const void *wu, const void *bg, const void *bu, const void *dy, int64_t ld_dy, const void *wd,
                         void *dgu, int act, float beta, float *sums, int64_t *n_sums, int64_t rows, int K, int H, int N, hipStream_t st);
};

}  // namespace arcn
