// logprob.hip.h -- log probabilities of given labels over rows of class scores, with entropy and the best alternatives, and
// their gradient.
//
// For a row x of C scores and a scale (1 / temperature): m = max x, d_j = scale (x_j - m), s = sum exp(d_j),
//   stat = (m, log s)      logprob = d_t - log s      entropy = log s - sum exp(d_j) d_j / s
//   gradient of sum (g logprob + h entropy):  scale (g [j = t] - p_j (g + h (log p_j + entropy))),  p_j = exp(d_j - log s)
// Everything is relative to the row's maximum and held in 32 bits: no score overflows, whatever its size.  -inf is a label
// that is ruled out: p = 0, no alternative.  A row of nothing else has stat (-inf, -inf), logprob -inf, entropy 0, gradient 0.
// A row that holds a NaN or +inf gives NaN, and no alternatives.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "element.hip.h"

namespace apr {

constexpr float kNegInf = -__builtin_inff();
constexpr float kNaN = __builtin_nanf("");

// A score and its label as one whole number: larger is better, equal scores go to the lowest label, +0 and -0 are equal.
__device__ __forceinline__ unsigned long long score_key(float x, unsigned label)
{
    uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    b ^= (uint32_t)((int32_t)b >> 31) | 0x80000000u;
    return ((unsigned long long)b << 32) | (unsigned)~label;
}
__device__ __forceinline__ float key_score(unsigned long long key)
{
    uint32_t b = (uint32_t)(key >> 32);
    b ^= (b >> 31) ? 0x80000000u : 0xFFFFFFFFu;
    return __builtin_bit_cast(float, b);
}
__device__ __forceinline__ int key_label(unsigned long long key) { return (int)~(uint32_t)key; }

struct LogprobArgs {
    const void *x;
    unsigned long long n, ld;
    unsigned n_labels;
    float scale;
    const int32_t *target;
    int top;
    float *logprob, *entropy, *stat;
    int32_t *top_label;
    float *top_logprob;
};

template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, V *s_part, F f)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o));
    const int wave = threadIdx.x >> 6, n_waves = blockDim.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_part[wave] = v;
    __syncthreads();
    v = s_part[0];
    for (int w = 1; w < n_waves; w++) v = f(v, s_part[w]);
    return v;
}

// One workgroup per row.
template <typename T>
__global__ __launch_bounds__(256) void logprob_rows_kernel(LogprobArgs a)
{
    __shared__ float s_f[4];
    __shared__ unsigned long long s_k[4];
    const auto add = [](float p, float q) { return p + q; };
    const auto larger = [](float p, float q) { return fmaxf(p, q); };
    const auto better = [](unsigned long long p, unsigned long long q) { return p > q ? p : q; };
    for (unsigned long long row = blockIdx.x; row < a.n; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.ld;
        float m = kNegInf, bad = 0.0f;
        for (unsigned j = threadIdx.x; j < a.n_labels; j += 256) {
            const float v = to_f32(x[j]);
            m = fmaxf(m, v);
            if (!(v < __builtin_inff())) bad = 1.0f;
        }
        m = block_reduce(m, s_f, larger);
        bad = block_reduce(bad, s_f, larger);
        const int t = a.target ? a.target[row] : -1;
        const bool has_t = t >= 0 && (unsigned)t < a.n_labels;
        float s = 0.0f, u = 0.0f;
        for (unsigned j = threadIdx.x; j < a.n_labels; j += 256) {
            const float v = to_f32(x[j]);
            if (v > kNegInf) {
                const float d = a.scale * (v - m), e = __expf(d);
                s += e;
                u += e * fmaxf(d, -200.0f);   // exp(-200) = 0 in 32 bits; a d of -inf would make 0 * inf
            }
        }
        s = block_reduce(s, s_f, add);
        u = block_reduce(u, s_f, add);
        const bool empty = m == kNegInf;
        const float log_s = logf(s);
        if (threadIdx.x == 0) {
            if (a.stat) {
                a.stat[2 * row] = bad ? kNaN : m;
                a.stat[2 * row + 1] = bad ? kNaN : log_s;
            }
            if (a.entropy) a.entropy[row] = bad ? kNaN : empty ? 0.0f : fmaxf(log_s - u / s, 0.0f);
            if (a.logprob) a.logprob[row] = !has_t ? 0.0f : bad ? kNaN : empty ? kNegInf : a.scale * (to_f32(x[t]) - m) - log_s;
        }
        unsigned long long last = ~0ull;
        for (int k = 0; k < a.top; k++) {
            unsigned long long best = 0;
            if (!bad && last)
                for (unsigned j = threadIdx.x; j < a.n_labels; j += 256) {
                    const float v = to_f32(x[j]);
                    const unsigned long long key = score_key(v, j);
                    if (v > kNegInf && key < last && key > best) best = key;
                }
            last = block_reduce(best, s_k, better);
            if (threadIdx.x == 0) {
                if (a.top_label) a.top_label[row * a.top + k] = last ? key_label(last) : -1;
                if (a.top_logprob) a.top_logprob[row * a.top + k] = last ? a.scale * (key_score(last) - m) - log_s : bad ? kNaN : kNegInf;
            }
        }
    }
}

struct LogprobGradArgs {
    const void *x;
    void *grad;
    unsigned long long n, ld, ld_grad;
    unsigned n_labels;
    float scale;
    const int32_t *target;
    const float *stat, *entropy, *g_logprob, *g_entropy;
};

// One workgroup per row; an element is read before the same thread writes it, so grad may be x.
template <typename T>
__global__ __launch_bounds__(256) void logprob_grad_kernel(LogprobGradArgs a)
{
    for (unsigned long long row = blockIdx.x; row < a.n; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.ld;
        T *grad = (T *)a.grad + row * a.ld_grad;
        const float m = a.stat[2 * row], log_s = a.stat[2 * row + 1];
        const int t = a.target ? a.target[row] : -1;
        const bool has_t = t >= 0 && (unsigned)t < a.n_labels;
        const float g = has_t && a.g_logprob ? a.g_logprob[row] : 0.0f;
        const float h = a.g_entropy ? a.g_entropy[row] : 0.0f;
        const float ent = a.g_entropy ? a.entropy[row] : 0.0f;
        for (unsigned j = threadIdx.x; j < a.n_labels; j += 256) {
            const float l = m == kNegInf ? kNegInf : a.scale * (to_f32(x[j]) - m) - log_s;
            const float p = __expf(l);
            float r = -p * (g + h * (fmaxf(l, -200.0f) + ent));
            if (has_t && j == (unsigned)t && m != kNegInf) r += g;
            grad[j] = from_f32<T>(a.scale * r);
        }
    }
}

}  // namespace apr
