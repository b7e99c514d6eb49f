// rowquant.hip.h -- rows of real numbers as 8-bit whole numbers with one scale each.
//
// a = max |x|, scale = a / 127, q = 127 x / a rounded to nearest even.  The quotient is the exact one: t = x (127 / a) in 64 bits is
// within 2^-45 of it, and a quotient of two 24-bit numbers that is not itself halfway between two whole numbers is at least 2^-33
// away from there, so t rounded to a multiple of 2^-36 is on the right side, and exactly halfway where the quotient is.
// A row of zeros, or of nothing above 2^-119 (its scale would leave the normal range): q = 0, scale 0.  A row that holds a NaN or an
// infinity: q = 0, scale NaN.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "element.hip.h"

namespace apr {

constexpr float kLeastRow = 0x1p-119f;

__device__ __forceinline__ int quantize_one(float x, double inv)
{
    const double snap = 0x1.8p+16, whole = 0x1.8p+52;   // adding these rounds at 2^-36 and at 1
    double t = (double)x * inv;
    t = (t + snap) - snap;
    return (int)(uint32_t)__builtin_bit_cast(uint64_t, t + whole);
}

struct RowQuantArgs {
    const void *x;
    int8_t *q;
    float *scale;
    unsigned long long n, ld, ld_q;
    unsigned k;
};

// One workgroup per row.
template <typename T>
__global__ __launch_bounds__(256) void rowquant_kernel(RowQuantArgs a)
{
    __shared__ uint32_t s_part[4];
    for (unsigned long long row = blockIdx.x; row < a.n; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.ld;
        // magnitudes as bit patterns: NaN above infinity above every number
        uint32_t most = 0;
        for (unsigned j = threadIdx.x; j < a.k; j += 256) most = max(most, __builtin_bit_cast(uint32_t, to_f32(x[j])) & 0x7FFFFFFFu);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = most;
        __syncthreads();
        most = max(max(s_part[0], s_part[1]), max(s_part[2], s_part[3]));
        const float am = __builtin_bit_cast(float, most);
        const bool bad = most >= 0x7F800000u, none = bad || am < kLeastRow;
        const double inv = none ? 0.0 : 127.0 / (double)am;
        if (threadIdx.x == 0) a.scale[row] = bad ? __builtin_nanf("") : none ? 0.0f : am / 127.0f;
        for (unsigned j = threadIdx.x; j < a.k; j += 256) a.q[row * a.ld_q + j] = none ? (int8_t)0 : (int8_t)quantize_one(to_f32(x[j]), inv);
    }
}

}  // namespace apr
