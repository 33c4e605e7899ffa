// Sums of partial results over workgroups, in a fixed order: out[e] = sum_p partial[p][e].
#pragma once

#include "common.hpp"

namespace arcn {

// A launch has fewer than 2^32 threads along one dimension (2^33 were cut short here without an error): many workgroups lie in rows of 2^21.
static inline dim3 wide_grid(int64_t blocks) {
    const int64_t row = 1 << 21;
    return blocks <= row ? dim3((unsigned)blocks) : dim3((unsigned)row, (unsigned)ceil_div<int64_t>(blocks, row));
}

// A workgroup sums E elements; 1024 / E threads share an element's partials, eight loads in flight each, and meet in LDS.  The elements
// are few and the partials many (a 64 x 64 weight gradient of 10^5 rows: 4096 elements of 390 partials): one thread per element would walk
// them alone, 600 ns a load (59 us there, 6 with E = 16).
// n_a elements go to a (if not NULL), the others to b (if not NULL).
template <typename T, int E>
__global__ void __launch_bounds__(1024)
sum_partials_kernel(const float *__restrict__ partial, int n_part, int64_t n_a, int64_t n_b, T *__restrict__ a, T *__restrict__ b) {
    constexpr int SHARES = 1024 / E;
    __shared__ float lds[SHARES][E + 1];
    const int le = threadIdx.x % E, share = threadIdx.x / E;
    const int64_t e = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * E + le, stride = n_a + n_b;
    float s[8] = {};
    if (e < stride) {
        int p = share;
        for (; p + 7 * SHARES < n_part; p += 8 * SHARES)
#pragma unroll
            for (int u = 0; u < 8; ++u) s[u] += partial[(int64_t)(p + u * SHARES) * stride + e];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (p + u * SHARES < n_part) s[u] += partial[(int64_t)(p + u * SHARES) * stride + e];
    }
    lds[share][le] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
#pragma unroll
    for (int h = SHARES / 2; h > 0; h >>= 1) {
        if (share < h) lds[share][le] += lds[share + h][le];
        __syncthreads();
    }
    if (share == 0 && e < stride) {
        if (e < n_a) {
            if (a) a[e] = (T)lds[0][le];
        } else if (b) {
            b[e - n_a] = (T)lds[0][le];
        }
    }
}

template <typename T>
static inline void sum_partials(const float *partial, int n_part, int64_t n_a, int64_t n_b, T *a, T *b, hipStream_t st) {
    const int64_t n = n_a + n_b;
#define ARCN_SP(E_) \
    hipLaunchKernelGGL((sum_partials_kernel<T, E_>), wide_grid(ceil_div<int64_t>(n, E_)), dim3(1024), 0, st, partial, n_part, n_a, n_b, a, b)
    if (n_part <= 8) ARCN_SP(1024);      // (nothing to share: 2 M elements of 4 partials 12 us, 26 with E = 256)
    else if (n <= 8192) ARCN_SP(16);
    else if (n <= 131072) ARCN_SP(64);
    else ARCN_SP(256);
#undef ARCN_SP
}

}  // namespace arcn
