// Element types of the feed-forward operators (f32, bf16, f16): 16-byte loads and stores of rows that start at any element, and the
// conversion to and from f32, in which everything is computed.
#pragma once

#include "common.hpp"

namespace arcn {

typedef float f4v __attribute__((ext_vector_type(4)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef uint32_t u4v_any __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes at any 2-byte boundary: one global_load_dwordx4 here
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// VEC: elements of one 16-byte access; Pack: their registers
template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int VEC = 4;
    static __device__ __forceinline__ void unpack(u4v p, float *v) {
        const f4v f = __builtin_bit_cast(f4v, p);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = f[e];
    }
    static __device__ __forceinline__ u4v pack(const float *v) { return __builtin_bit_cast(u4v, f4v{v[0], v[1], v[2], v[3]}); }
};
template <>
struct Elem<__bf16> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ void unpack(u4v p, float *v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {   // a bf16 is the upper half of an f32
            v[2 * e] = __builtin_bit_cast(float, p[e] << 16);
            v[2 * e + 1] = __builtin_bit_cast(float, p[e] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u4v pack(const float *v) {
        bf16x8 r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = (__bf16)v[e];   // round to nearest even (v_cvt_pk_bf16_f32)
        return __builtin_bit_cast(u4v, r);
    }
};
template <>
struct Elem<_Float16> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ void unpack(u4v p, float *v) {
        const f16x8 f = __builtin_bit_cast(f16x8, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)f[e];
    }
    static __device__ __forceinline__ u4v pack(const float *v) {
        f16x8 r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = (_Float16)v[e];
        return __builtin_bit_cast(u4v, r);
    }
};

template <typename T>
__device__ __forceinline__ u4v load16(const T *p) {
    return *reinterpret_cast<const u4v_any *>(p);
}
template <typename T>
__device__ __forceinline__ void store16(T *p, u4v v) {
    *reinterpret_cast<u4v_any *>(p) = v;
}

// The same without a branch that waits: a row of at least VEC elements is read up to its LAST 16 bytes (`tail_at` moves the address there), and
// what was loaded is shifted down to its place once it has arrived (`tail_fix`).  p: the pack's place in the row, left: elements of the row
// from there on (any number).
template <typename T>
__device__ __forceinline__ const T *tail_at(const T *p, int64_t left) {
    return left >= Elem<T>::VEC ? p : p + (left - Elem<T>::VEC);
}
template <typename T>
__device__ __forceinline__ u4v tail_fix(u4v v, int64_t left) {
    const int drop = left >= Elem<T>::VEC ? 0 : Elem<T>::VEC - (int)(left > 0 ? left : 0);   // elements in front of the pack
    if (sizeof(T) == 2) {
        if (drop & 8) v = u4v{0u, 0u, 0u, 0u};
        if (drop & 4) v = u4v{v[2], v[3], 0u, 0u};
        if (drop & 2) v = u4v{v[1], v[2], v[3], 0u};
        if (drop & 1)
            v = u4v{__builtin_amdgcn_alignbit(v[1], v[0], 16), __builtin_amdgcn_alignbit(v[2], v[1], 16), __builtin_amdgcn_alignbit(v[3], v[2], 16), v[3] >> 16};
    } else {
        if (drop & 4) v = u4v{0u, 0u, 0u, 0u};
        if (drop & 2) v = u4v{v[2], v[3], 0u, 0u};
        if (drop & 1) v = u4v{v[1], v[2], v[3], 0u};
    }
    return v;
}

// one 16-byte pack of a row of which `left` elements remain (<= 0: nothing is read); what lies behind the row's end reads as zero
template <typename T>
__device__ __forceinline__ u4v load_pack(const T *p, int64_t left) {
    if (left >= Elem<T>::VEC) return load16(p);
    u4v r = {0u, 0u, 0u, 0u};
    if (left > 0) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < left) r[e] = reinterpret_cast<const uint32_t *>(p)[e];
        } else {
#pragma unroll
            for (int e = 0; e < 7; ++e)
                if (e < left) r[e >> 1] |= (uint32_t) reinterpret_cast<const uint16_t *>(p)[e] << (16 * (e & 1));
        }
    }
    return r;
}

template <typename T>
__device__ __forceinline__ void store_pack(T *p, u4v v, int64_t left) {
    if (left >= Elem<T>::VEC) {
        store16(p, v);
        return;
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < left) reinterpret_cast<uint32_t *>(p)[e] = v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < left) reinterpret_cast<uint16_t *>(p)[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
    }
}

}  // namespace arcn
