// rowquant.hip.h -- rows of real numbers as 8-bit whole numbers with one scale each.
//
// a = max |x|, scale = a / 127, q = 127 x / a rounded to nearest even.  The quotient is the exact one: t = x (127 / a) in 64 bits is
// within 2^-45 of it, and a quotient of two 24-bit numbers that is not itself halfway between two whole numbers is at least 2^-33
// away from there, so t rounded to a multiple of 2^-36 is on the right side, and exactly halfway where the quotient is.
// In 32 bits x (127 / a) is within 127 * 2^-23 < 2^-16 of the quotient, so that values which are 2^-15 or more from halfway are right without
// that; the 64 bits, an instruction of which takes twice as long, are for the waves that hold another one.
// A row of zeros, or of nothing above 2^-119 (its scale would leave the normal range): q = 0, scale 0.  A row that holds a NaN or an
// infinity: q = 0, scale NaN.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "element.hip.h"

namespace apr {

constexpr float kLeastRow = 0x1p-119f, kToWhole = 0x1.8p+23f;   // adding kToWhole rounds to whole numbers, whose lowest 8 bits come out

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

// G waves per row, U units of 16 bytes a lane in registers, read once (a row that is longer than that is read twice).
// HBM-bound: 35999 x 1024 f32 takes 35.2 us, 5.2 TB/s (a multiplication by a number: 5.6 to 6.0), 4096 x 8191 bf16 25.8 us, 3.9 TB/s; in a
// captured row of calls 35.5 and 24.3, and with every quotient in 64 bits 38.6 and 26.1.  16-byte loads
// begin at the 16-byte unit that the row begins in (which is inside the allocation, as the row's first element is); what does not belong
// to the row counts as 0 and is not written.  A lane writes the 4 or 8 values of its unit together, at whatever alignment they have.
template <typename T, int G, int U>
__global__ __launch_bounds__(G == 1 ? 256 : G * 64) void rowquant_kernel(RowQuantArgs a)
{
    constexpr int V = 16 / (int)sizeof(T), LANES = G * 64;
    typedef T txv __attribute__((ext_vector_type(V)));
    typedef int8_t qxv __attribute__((ext_vector_type(V)));
    __shared__ uint32_t s_part[2][G];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), me = G == 1 ? lane : (int)threadIdx.x;
    constexpr unsigned ROWS = G == 1 ? 4 : 1;   // rows that a workgroup has at hand
    int flip = 0;
    for (unsigned long long row = (unsigned long long)blockIdx.x * ROWS + (G == 1 ? wave : 0); row < a.n; row += (unsigned long long)gridDim.x * ROWS) {
        const T *x = (const T *)a.x + row * a.ld;
        int8_t *q = a.q + row * a.ld_q;
        const unsigned off = (unsigned)(((unsigned long long)x & 15) / sizeof(T));
        const txv *units = (const txv *)(x - off);
        const unsigned long long len = (unsigned long long)a.k + off;
        const unsigned n_units = (unsigned)((len + V - 1) / V);
        txv v[U];
        // magnitudes as bit patterns: NaN above infinity above every number
        uint32_t most = 0;
        const auto load = [&](unsigned base) {
#pragma unroll
            for (int i = 0; i < U; i++) {
                const unsigned w = base + i * LANES + me;
                if (w < n_units) v[i] = units[w];
                else v[i] = (T)0.0f;
            }
#pragma unroll
            for (int i = 0; i < U; i++) {
                const unsigned w = base + i * LANES + me;
                if (w == 0 || w == n_units - 1) {
#pragma unroll
                    for (int e = 0; e < V; e++)
                        if ((unsigned long long)w * V + e < off || (unsigned long long)w * V + e >= len) v[i][e] = (T)0.0f;
                }
            }
        };
        for (unsigned base = 0; base < n_units; base += U * LANES) {
            load(base);
#pragma unroll
            for (int i = 0; i < U; i++)
#pragma unroll
                for (int e = 0; e < V; e++) most = max(most, __builtin_bit_cast(uint32_t, to_f32(v[i][e])) & 0x7FFFFFFFu);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));
        if (G > 1) {
            if (lane == 0) s_part[flip][wave] = most;   // two sets: the next row's may be written while this one's are read
            __syncthreads();
#pragma unroll
            for (int w = 0; w < G; w++) most = max(most, s_part[flip][w]);
            flip ^= 1;
        }
        const float am = __builtin_bit_cast(float, most);
        const bool bad = most >= 0x7F800000u, none = bad || am < kLeastRow;
        const float inv = none ? 0.0f : 127.0f / am;
        if (me == 0) a.scale[row] = bad ? __builtin_nanf("") : none ? 0.0f : am / 127.0f;
        for (unsigned base = 0; base < n_units; base += U * LANES) {
            if (n_units > U * LANES) load(base);   // otherwise the row is still there
#pragma unroll
            for (int i = 0; i < U; i++) {
                asm volatile("" : "+v"(v[i]));   // or the compiler keeps what the loop above made of it, in twice the registers
                qxv r;
                float far = 0.0f;   // from a whole number
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float t = to_f32(v[i][e]) * inv, n = t + kToWhole;
                    far = fmaxf(far, fabsf(t - (n - kToWhole)));
                    r[e] = (int8_t)(uint8_t)__builtin_bit_cast(uint32_t, n);
                }
                if (__ballot(far > 0.5f - 0x1p-15f)) {
                    const double exact = none ? 0.0 : 127.0 / (double)am;
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        r[e] = (int8_t)quantize_one(to_f32(v[i][e]), exact);
                        __builtin_amdgcn_sched_barrier(0);   // one after the other, in few registers
                    }
                }
                if (none) r = (int8_t)0;
                const unsigned w = base + i * LANES + me;
                if (w >= n_units) continue;
                const long long j = (long long)w * V - off;
                if (j >= 0 && j + V <= (long long)a.k) __builtin_memcpy(q + j, &r, V);
                else {
#pragma unroll
                    for (int e = 0; e < V; e++)
                        if (j + e >= 0 && j + e < (long long)a.k) q[j + e] = r[e];
                }
            }
        }
    }
}

}  // namespace apr
