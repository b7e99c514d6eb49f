// linear_i8.hip.h -- out[m][n] = (sum_k x[m][k] w[n][k]) x_scale[m] w_scale[n] + bias[n] for 8-bit x and w.
//
// The sum is exact in 32 bits (|product| <= 2^14, k < 2^17) and does not depend on its order.  Both operands have k contiguous,
// which is how the matrix instruction wants them: a lane holds 16 consecutive k of one row.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "element.hip.h"

namespace apr {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

struct LinearI8Args {
    const int8_t *x, *w;
    const float *x_scale, *w_scale, *bias;
    void *out;
    unsigned long long ld_x, ld_w, ld_out;
    unsigned m, n, k;
};

// 64 x 64 outputs at a time, four waves of 32 x 32; 64 k a step through LDS, byte by byte: any alignment.
template <typename T>
__global__ __launch_bounds__(256) void linear_i8_kernel(LinearI8Args a)
{
    __shared__ __align__(16) int8_t s_x[64][80], s_w[64][80];   // 80: neighbouring rows start in other banks
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
    const unsigned long long tiles_n = (a.n + 63u) / 64u, tiles = (a.m + 63u) / 64u * tiles_n;
    for (unsigned long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const unsigned m0 = (unsigned)(tile / tiles_n) * 64u, n0 = (unsigned)(tile % tiles_n) * 64u;
        i32x16 acc = {};
        for (unsigned k0 = 0; k0 < a.k; k0 += 64) {
            __syncthreads();
            for (unsigned i = threadIdx.x; i < 64 * 64; i += 256) {
                const unsigned r = i >> 6, c = i & 63, k = k0 + c;
                s_x[r][c] = m0 + r < a.m && k < a.k ? a.x[(m0 + r) * a.ld_x + k] : (int8_t)0;
                s_w[r][c] = n0 + r < a.n && k < a.k ? a.w[(n0 + r) * a.ld_w + k] : (int8_t)0;
            }
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < 64; kk += 32) {
                const i32x4 xa = *(const i32x4 *)&s_x[wm + (lane & 31)][kk + 16 * (lane >> 5)];
                const i32x4 wb = *(const i32x4 *)&s_w[wn + (lane & 31)][kk + 16 * (lane >> 5)];
                acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(xa, wb, acc, 0, 0, 0);
            }
        }
        const unsigned n = n0 + wn + (lane & 31);
        if (n < a.n) {
            const float ws = a.w_scale[n], b = a.bias ? a.bias[n] : 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const unsigned m = m0 + wm + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
                if (m < a.m) ((T *)a.out)[m * a.ld_out + n] = from_f32<T>((float)acc[i] * a.x_scale[m] * ws + b);
            }
        }
    }
}

}  // namespace apr
