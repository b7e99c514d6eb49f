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

// ---- reductions of a wave (64 lanes) ----
template <int CTRL, int ROWS>
__device__ __forceinline__ float lane_move(float v)
{
    const int b = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(b, b, CTRL, ROWS, 0xf, false));
}
// over the four lanes of a quad, and over the sixteen of a row: every lane has the result
template <typename F>
__device__ __forceinline__ float quad_reduce(float v, F f)
{
    v = f(v, lane_move<0xB1, 0xf>(v));   // lane ^ 1
    return f(v, lane_move<0x4E, 0xf>(v));   // lane ^ 2
}
template <typename F>
__device__ __forceinline__ float row_reduce(float v, F f)
{
    v = quad_reduce(v, f);
    v = f(v, lane_move<0x141, 0xf>(v));   // mirrored within eight
    return f(v, lane_move<0x140, 0xf>(v));   // mirrored within sixteen
}
// over all lanes, from row results; wave-uniform
template <typename F>
__device__ __forceinline__ float wave_of_rows(float v, F f)
{
    const int b = __builtin_bit_cast(int, v);
    const auto at = [b](int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, lane)); };
    return f(f(at(0), at(16)), f(at(32), at(48)));
}
template <typename F>
__device__ __forceinline__ float wave_reduce(float v, F f) { return wave_of_rows(row_reduce(v, f), f); }

struct MaxOf { __device__ __forceinline__ float operator()(float p, float q) const { return fmaxf(p, q); } };
struct SumOf { __device__ __forceinline__ float operator()(float p, float q) const { return p + q; } };

constexpr float kLog2E = 1.44269504088896340736f;

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
    // rows cut in pieces: [row][piece] partial results
    struct LogprobPart *part;
    unsigned long long *part_top;   // [row][piece][top], best first, 0 = none
    unsigned pieces, piece_len;
};

// Sums of a piece of a row relative to its own maximum m (as a score): s = sum exp(scale (x - m)), u = sum exp(..) (x - m).
struct LogprobPart { float m, s, u; };

// exp(scale (x - m)) and its product with x - m.  m = -inf (nothing but ruled-out labels) counts as 0, so that x - m is -inf; the
// product takes x - m no lower than where the exponential is 0 anyway, so that there is no 0 * inf.  NaN and +inf end up in s.
struct ExpSum {
    float m, c, least, s = 0.0f, u = 0.0f;
    __device__ __forceinline__ ExpSum(float max, float scale) : m(max == kNegInf ? 0.0f : max), c(scale * kLog2E), least(-200.0f / scale) {}
    __device__ __forceinline__ void add(float x)
    {
        const float t = x - m, e = __builtin_amdgcn_exp2f(t * c);
        s += e;
        u = fmaf(e, fmaxf(t, least), u);
    }
};

// The outputs of a row from its sums; called by one lane.
__device__ __forceinline__ void logprob_write(const LogprobArgs &a, unsigned long long row, LogprobPart r, float x_target, bool has_target)
{
    const bool bad = r.s != r.s, empty = r.m == kNegInf && !bad;
    const float log_s = logf(r.s);
    if (a.stat) {
        a.stat[2 * row] = bad ? kNaN : r.m;
        a.stat[2 * row + 1] = bad ? kNaN : log_s;
    }
    if (a.entropy) a.entropy[row] = bad ? kNaN : empty ? 0.0f : fmaxf(log_s - a.scale * (r.u / r.s), 0.0f);
    if (a.logprob) a.logprob[row] = !has_target ? 0.0f : bad ? kNaN : empty ? kNegInf : a.scale * (x_target - r.m) - log_s;
}
__device__ __forceinline__ void logprob_write_top(const LogprobArgs &a, unsigned long long row, LogprobPart r, int place, unsigned long long key)
{
    const bool bad = r.s != r.s, none = bad || !key;
    if (a.top_label) a.top_label[row * a.top + place] = none ? -1 : key_label(key);
    if (a.top_logprob) a.top_logprob[row * a.top + place] = bad ? kNaN : none ? kNegInf : a.scale * (key_score(key) - r.m) - logf(r.s);
}

// ---- the best `top` of many keys, by one wave ----
//
// A score that at least `top` of the wave's 64 values reach: the binary search over the ordered bits counts lanes with a ballot.  The
// highest 16 bits are enough, a score that is a little lower lets a few more candidates through.  Never below the lowest finite
// score: what is ruled out is no candidate.
__device__ __forceinline__ float reached_by(float v, int top)
{
    const uint32_t k = (uint32_t)(score_key(v, 0) >> 32);
    uint32_t t = 0;
#pragma unroll
    for (int b = 31; b >= 16; b--) {
        const uint32_t c = t | (1u << b);
        if (__builtin_popcountll(__ballot(k >= c)) >= top) t = c;
    }
    t = t < 0x00800000u ? 0x00800000u : t;
    return key_score((unsigned long long)t << 32);
}

// The `top`-th largest of the keys that count() counts (each key is there once): the largest K that at least `top` of them reach.
template <typename F>
__device__ __forceinline__ unsigned long long key_reached_by(int top, F count)
{
    unsigned long long t = 0;
    for (int b = 63; b >= 0; b--) {
        const unsigned long long c = t | (1ull << b);
        if (count(c) >= top) t = c;
    }
    return t;
}

// Place of a lane's key among the first n lanes' keys, best first
__device__ __forceinline__ int key_place(unsigned long long key, int n)
{
    int place = 0;
    const int lo = (int)(uint32_t)key, hi = (int)(uint32_t)(key >> 32);
    for (int i = 0; i < n; i++) {
        const unsigned long long other = ((unsigned long long)(uint32_t)__builtin_amdgcn_readlane(hi, i) << 32) | (uint32_t)__builtin_amdgcn_readlane(lo, i);
        place += other > key ? 1 : 0;
    }
    return place;
}

// Keeps the best `top` of the n keys in `list` (LDS, n <= 16 * 64) there, in any order; returns how many that are (<= 64)
__device__ __forceinline__ int keep_best(unsigned long long *list, int n, int top, int lane)
{
    if (n <= 64) return n;
    unsigned long long k[16];
#pragma unroll
    for (int i = 0; i < 16; i++) k[i] = 64 * i + lane < n ? list[64 * i + lane] : 0;
    const unsigned long long t = key_reached_by(top, [&](unsigned long long c) {
        int count = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) count += __builtin_popcountll(__ballot(k[i] >= c));
        return count;
    });
    int kept = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const unsigned long long in = __ballot(k[i] >= t && k[i]);
        if (k[i] >= t && k[i]) list[kept + __builtin_popcountll(in & ((1ull << lane) - 1))] = k[i];
        kept += __builtin_popcountll(in);
    }
    return kept;
}

// ---- short rows: a wave per row, E scores a lane ----
//
// Candidates for the alternatives are the scores that at least `top` lanes' best scores reach: about as many as are wanted.
template <typename T, int E>
__global__ __launch_bounds__(256, 8) void logprob_wave_kernel(LogprobArgs a)
{
    __shared__ unsigned long long s_list[4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned long long *list = s_list[wave];
    for (unsigned long long row = (unsigned long long)blockIdx.x * 4 + wave; row < a.n; row += (unsigned long long)gridDim.x * 4) {
        const T *x = (const T *)a.x + row * a.ld;
        const int t = a.target ? a.target[row] : -1;
        const bool has_t = t >= 0 && (unsigned)t < a.n_labels;
        const float xt = has_t ? to_f32(x[t]) : 0.0f;
        float v[E], best = kNegInf;
#pragma unroll
        for (int i = 0; i < E; i++) v[i] = 64u * i + lane < a.n_labels ? to_f32(x[64 * i + lane]) : kNegInf;
#pragma unroll
        for (int i = 0; i < E; i++) best = fmaxf(best, v[i]);
        LogprobPart r;
        r.m = wave_reduce(best, MaxOf());
        ExpSum sum(r.m, a.scale);
#pragma unroll
        for (int i = 0; i < E; i++) sum.add(v[i]);
        r.s = wave_reduce(sum.s, SumOf());
        r.u = wave_reduce(sum.u, SumOf());
        if (lane == 0) logprob_write(a, row, r, xt, has_t);
        if (!a.top) continue;
        const float least = reached_by(best, a.top);
        int n = 0;
#pragma unroll
        for (int i = 0; i < E; i++) n += __builtin_popcountll(__ballot(v[i] >= least));
        unsigned long long reach = 0;
        if (n > 64)   // many equal scores: the exact border, over the scores in memory (this is rare, and they would take registers)
            reach = key_reached_by(a.top, [&](unsigned long long c) {
                int count = 0;   // lane 0 is in every round
                for (unsigned j = lane; j < a.n_labels; j += 64) {
                    const float y = to_f32(x[j]);
                    count += __builtin_popcountll(__ballot(y >= least && score_key(y, j) >= c));
                }
                return __builtin_amdgcn_readfirstlane(count);
            });
        n = 0;
#pragma unroll
        for (int i = 0; i < E; i++) {
            const unsigned long long key = score_key(v[i], 64 * i + lane);
            const bool in = v[i] >= least && key >= reach;
            const unsigned long long mask = __ballot(in);
            if (in) list[n + __builtin_popcountll(mask & ((1ull << lane) - 1))] = key;
            n += __builtin_popcountll(mask);
        }
        __builtin_amdgcn_wave_barrier();   // the wave's LDS operations are in order
        const unsigned long long key = lane < n ? list[lane] : 0;
        const int place = key_place(key, n);
        if (lane < n && place < a.top) logprob_write_top(a, row, r, place, key);
        if (lane >= n && lane < a.top) logprob_write_top(a, row, r, lane, 0);
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- longer rows: a workgroup per row, or per piece of one; E scores a lane in registers, read once ----
//
// 16-byte loads begin at the 16-byte unit that the piece begins in (which is inside the allocation, as the piece's first element is);
// what does not belong to the piece counts as ruled out.
// Candidates are the scores that at least `top` of 64 groups of NT / 64 lanes reach with their best; they are collected in LDS.
// If equal scores make them too many, the exact border is found by counting over the whole workgroup.
constexpr int kCandidates = 1024;

template <typename T, int NT, int E>
__global__ __launch_bounds__(NT, 8) void logprob_block_kernel(LogprobArgs a)
{
    constexpr int V = 16 / (int)sizeof(T), VECS = E / V, WAVES = NT / 64;
    typedef T txv __attribute__((ext_vector_type(V)));
    __shared__ float s_group[64], s_s[WAVES], s_u[WAVES];
    __shared__ unsigned long long s_list[kCandidates];
    __shared__ int s_n;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned long long works = a.n * a.pieces;
    for (unsigned long long work = blockIdx.x; work < works; work += gridDim.x) {
        const unsigned long long row = a.pieces == 1 ? work : work / a.pieces;
        const unsigned piece = (unsigned)(work - row * a.pieces), j0 = piece * a.piece_len, j1 = min(j0 + a.piece_len, a.n_labels);
        const T *x = (const T *)a.x + row * a.ld;
        // first unit, and the label that its first element would be (modulo 2^32; below j0 by less than V)
        const unsigned off = (unsigned)(((unsigned long long)(x + j0) & 15) / sizeof(T));
        const txv *units = (const txv *)(x + j0 - off);
        const unsigned len = j1 - j0 + off, n_units = (len + V - 1) / V;
        float v[E], best = kNegInf;
#pragma unroll
        for (int q = 0; q < VECS; q++) {
            const unsigned w = q * NT + threadIdx.x;
            if (w < n_units) {
                const txv p = units[w];
#pragma unroll
                for (int i = 0; i < V; i++) v[q * V + i] = to_f32(p[i]);
                if (w == 0 || w == n_units - 1) {
#pragma unroll
                    for (int i = 0; i < V; i++)
                        if (w * V + i < off || w * V + i >= len) v[q * V + i] = kNegInf;
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) v[q * V + i] = kNegInf;
            }
        }
        const auto label = [&](int e) { return j0 - off + (e / V * NT + threadIdx.x) * V + e % V; };
#pragma unroll
        for (int e = 0; e < E; e++) best = fmaxf(best, v[e]);
        const float group = NT == 1024 ? row_reduce(best, MaxOf()) : NT == 512 ? fmaxf(quad_reduce(best, MaxOf()), lane_move<0x141, 0xf>(quad_reduce(best, MaxOf())))
                                                                                : quad_reduce(best, MaxOf());
        if (threadIdx.x % (NT / 64) == 0) s_group[threadIdx.x / (NT / 64)] = group;
        if (threadIdx.x == 0) s_n = 0;
        __syncthreads();
        const float g = s_group[lane];
        LogprobPart r;
        r.m = wave_reduce(g, MaxOf());
        ExpSum sum(r.m, a.scale);
#pragma unroll
        for (int e = 0; e < E; e++) sum.add(v[e]);
        const float ws = wave_reduce(sum.s, SumOf()), wu = wave_reduce(sum.u, SumOf());
        if (lane == 0) { s_s[wave] = ws; s_u[wave] = wu; }
        if (a.top) {
            const float least = reached_by(g, a.top);
            if (best >= least) {
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (v[e] >= least) {
                        const int at = atomicAdd(&s_n, 1);
                        if (at < kCandidates) s_list[at] = score_key(v[e], label(e));
                    }
            }
            __syncthreads();
            if (s_n > kCandidates) {
                // over the scores in memory: this is rare, and they would take registers
                const unsigned long long reach = key_reached_by(a.top, [&](unsigned long long c) {
                    int count = 0;   // lane 0 is in every round of its wave
                    for (unsigned j = j0 + threadIdx.x; j < j1; j += NT) {
                        const float y = to_f32(x[j]);
                        count += __builtin_popcountll(__ballot(y >= least && score_key(y, j) >= c));
                    }
                    __syncthreads();
                    if (threadIdx.x == 0) s_n = 0;
                    __syncthreads();
                    if (lane == 0) atomicAdd(&s_n, count);
                    __syncthreads();
                    return s_n;
                });
                __syncthreads();
                if (threadIdx.x == 0) s_n = 0;
                __syncthreads();
                for (unsigned j = j0 + threadIdx.x; j < j1; j += NT) {
                    const float y = to_f32(x[j]);
                    if (y >= least && score_key(y, j) >= reach) s_list[atomicAdd(&s_n, 1)] = score_key(y, j);
                }
                __syncthreads();
            }
        } else {
            __syncthreads();
        }
        if (wave == 0) {
            r.s = wave_reduce(lane < WAVES ? s_s[lane] : 0.0f, SumOf());
            r.u = wave_reduce(lane < WAVES ? s_u[lane] : 0.0f, SumOf());
            if (lane == 0) {
                if (a.pieces == 1) {
                    const int t = a.target ? a.target[row] : -1;
                    const bool has_t = t >= 0 && (unsigned)t < a.n_labels;
                    logprob_write(a, row, r, has_t ? to_f32(x[t]) : 0.0f, has_t);
                } else
                    a.part[work] = r;
            }
            if (a.top) {
                const int n = keep_best(s_list, s_n, a.top, lane);
                __builtin_amdgcn_wave_barrier();
                const unsigned long long key = lane < n ? s_list[lane] : 0;
                const int place = key_place(key, n);
                if (a.pieces == 1) {
                    if (lane < n && place < a.top) logprob_write_top(a, row, r, place, key);
                    if (lane >= n && lane < a.top) logprob_write_top(a, row, r, lane, 0);
                } else {
                    if (lane < n && place < a.top) a.part_top[work * a.top + place] = key;
                    if (lane >= n && lane < a.top) a.part_top[work * a.top + lane] = 0;
                }
            }
        }
        __syncthreads();   // before the next row's s_group, s_n and s_list
    }
}

// ---- the pieces of a row joined, a wave per row ----
__global__ __launch_bounds__(64) void logprob_join_kernel(LogprobArgs a, int type)
{
    __shared__ unsigned long long s_list[kCandidates];
    const int lane = threadIdx.x;
    for (unsigned long long row = blockIdx.x; row < a.n; row += gridDim.x) {
        const LogprobPart *part = a.part + row * a.pieces;
        LogprobPart r;
        float m = kNegInf;
        for (unsigned p = lane; p < a.pieces; p += 64) m = fmaxf(m, part[p].m);
        r.m = wave_reduce(m, MaxOf());
        const ExpSum to(r.m, a.scale);
        float s = 0.0f, u = 0.0f;
        for (unsigned p = lane; p < a.pieces; p += 64) {
            const LogprobPart q = part[p];
            const float d = q.m - to.m, e = __builtin_amdgcn_exp2f(d * to.c);
            s = fmaf(e, q.s, s);
            u = fmaf(e, fmaf(fmaxf(d, to.least), q.s, q.u), u);
        }
        r.s = wave_reduce(s, SumOf());
        r.u = wave_reduce(u, SumOf());
        if (lane == 0) {
            const int t = a.target ? a.target[row] : -1;
            const bool has_t = t >= 0 && (unsigned)t < a.n_labels;
            float xt = 0.0f;
            if (has_t) {
                const unsigned long long at = row * a.ld + (unsigned)t;
                xt = type == 0 ? ((const float *)a.x)[at] : type == 1 ? to_f32(((const f16_t *)a.x)[at]) : to_f32(((const bf16_t *)a.x)[at]);
            }
            logprob_write(a, row, r, xt, has_t);
        }
        if (!a.top) continue;
        // the pieces' lists through LDS, as many at a time as fit beside the best so far
        const unsigned long long *keys = a.part_top + row * a.pieces * a.top, all = (unsigned long long)a.pieces * a.top;
        int n = 0;
        for (unsigned long long k0 = 0; k0 < all;) {
            const int more = (int)min(all - k0, (unsigned long long)(kCandidates - n));
            int kept = n;
            for (int i = 0; i < more; i += 64) {
                const unsigned long long key = i + lane < more ? keys[k0 + i + lane] : 0, in = __ballot(key != 0);
                if (key) s_list[kept + __builtin_popcountll(in & ((1ull << lane) - 1))] = key;
                kept += __builtin_popcountll(in);
            }
            k0 += more;
            __builtin_amdgcn_wave_barrier();
            n = keep_best(s_list, kept, a.top, lane);
            __builtin_amdgcn_wave_barrier();
        }
        const unsigned long long key = lane < n ? s_list[lane] : 0;
        const int place = key_place(key, n);
        if (lane < n && place < a.top) logprob_write_top(a, row, r, place, key);
        if (lane >= n && lane < a.top) logprob_write_top(a, row, r, lane, 0);
        __builtin_amdgcn_wave_barrier();
    }
}

// How a call's rows are cut: lanes and scores a lane of a workgroup (0 lanes: a wave per row), pieces of a row and their length.
struct LogprobPlan {
    int threads, each;
    unsigned pieces, piece_len;
    size_t work;   // bytes
};
inline LogprobPlan logprob_plan(size_t n, size_t c, int top)
{
    LogprobPlan p = {0, 1, 1, (unsigned)c, 0};
    if (c <= 1024) {
        while (64 * p.each < (int)c) p.each *= 2;
        return p;
    }
    // rows to spare for every CU: the shortest workgroup that holds a row, or the longest; otherwise short pieces, so that the rows
    // at hand reach more CUs (a piece loses up to 7 places to alignment)
    const bool many = n * ((c + 32759) / 32760) >= 256;
    p.threads = c <= 4088 || !many ? 256 : c <= 8184 ? 256 : c <= 16376 ? 512 : 1024;
    p.each = p.threads == 256 && (c <= 4088 || !many) ? 16 : 32;
    const size_t room = (size_t)p.threads * p.each - 8;
    p.pieces = (unsigned)((c + room - 1) / room);
    p.piece_len = (unsigned)(((c + p.pieces - 1) / p.pieces + 7) / 8 * 8);
    p.pieces = (unsigned)((c + p.piece_len - 1) / p.piece_len);
    if (p.pieces > 1) p.work = n * p.pieces * (size_t)top * 8 + (n * p.pieces * sizeof(LogprobPart) + 15) / 16 * 16;
    return p;
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
