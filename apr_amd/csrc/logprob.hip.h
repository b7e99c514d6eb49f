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

#include <algorithm>

#include "../../include/apr.h"
#include "element.hip.h"

namespace apr {

constexpr float kNegInf = -__builtin_inff();
constexpr float kLowest = -3.402823466e+38f;   // of the finite ones
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
// Another lane's value, by a pattern in which every lane has a source: folds into the instruction that uses it
template <int CTRL>
__device__ __forceinline__ float lane_move(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true)); }
// over the four lanes of a quad, and over the sixteen of a row: every lane has the result
template <typename F>
__device__ __forceinline__ float quad_reduce(float v, F f)
{
    v = f(v, lane_move<0xB1>(v));   // lane ^ 1
    return f(v, lane_move<0x4E>(v));   // lane ^ 2
}
template <typename F>
__device__ __forceinline__ float row_reduce(float v, F f)
{
    v = quad_reduce(v, f);
    v = f(v, lane_move<0x141>(v));   // mirrored within eight
    return f(v, lane_move<0x140>(v));   // mirrored within sixteen
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

// The sums of two values over all lanes, wave-uniform.  The first step leaves p's in the lower and q's in the upper half of one register.
__device__ __forceinline__ void wave_sums(float &p, float &q)
{
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    const auto both = [](u32x2 v) {
        const unsigned lower = v.x, upper = v.y;   // by value: a bit cast of an element itself takes the first one
        return __builtin_bit_cast(float, lower) + __builtin_bit_cast(float, upper);
    };
    float v = both(__builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, p), __builtin_bit_cast(unsigned, q), false, false));
    v = v + lane_move<0xB1>(v);
    v = v + lane_move<0x4E>(v);
    v = v + lane_move<0x141>(v);
    v = v + lane_move<0x140>(v);
    const unsigned b = __builtin_bit_cast(unsigned, v);
    const int w = __builtin_bit_cast(int, both(__builtin_amdgcn_permlane16_swap(b, b, false, false)));
    p = __builtin_bit_cast(float, __builtin_amdgcn_readlane(w, 0));
    q = __builtin_bit_cast(float, __builtin_amdgcn_readlane(w, 32));
}

// The largest of all lanes, wave-uniform, as whole numbers, whose maximum folds with the move (a float's is made quiet first)
__device__ __forceinline__ int wave_max(int v)
{
    const int none = (int)0x80000000;
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_update_dpp(none, v, 0x142, 0xa, 0xf, false));   // a row's last lane to the next row
    v = max(v, __builtin_amdgcn_update_dpp(none, v, 0x143, 0xc, 0xf, false));   // lane 31 to the upper half
    return __builtin_amdgcn_readlane(v, 63);
}
// A float as a whole number of the same order, and back
__device__ __forceinline__ int ordered(float v)
{
    const int b = __builtin_bit_cast(int, v);
    return b ^ (b >> 31 & 0x7FFFFFFF);
}
__device__ __forceinline__ float of_ordered(int b) { return __builtin_bit_cast(float, b ^ (b >> 31 & 0x7FFFFFFF)); }

struct MaxOf { __device__ __forceinline__ float operator()(float p, float q) const { return fmaxf(p, q); } };

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
    // short rows: a wave's, at most kRows, and 65536 / top rounded up
    unsigned rows, per_top;
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

// log of a sum of exponentials: 1 <= s, or 0, or NaN; the instruction's error is 2^-24 of log2 s or of 1
__device__ __forceinline__ float log_of_sum(float s) { return __builtin_amdgcn_logf(s) * 0.69314718055994530942f; }

// scale (x - m), also where x - m is beyond the largest float and the product is not (halves are exact, subnormals aside)
__device__ __forceinline__ float scaled_distance(float x, float m, float scale) { return (0.5f * x - 0.5f * m) * (2.0f * scale); }

// The outputs of a row from its sums and their logarithm; called by one lane.
__device__ __forceinline__ void logprob_write(const LogprobArgs &a, unsigned long long row, LogprobPart r, float log_s, float x_target, bool has_target)
{
    const bool bad = r.s != r.s, empty = r.m == kNegInf && !bad;
    if (a.stat) {
        a.stat[2 * row] = bad ? kNaN : r.m;
        a.stat[2 * row + 1] = bad ? kNaN : log_s;
    }
    if (a.entropy) a.entropy[row] = bad ? kNaN : empty ? 0.0f : fmaxf(log_s - a.scale * (r.u * __builtin_amdgcn_rcpf(r.s)), 0.0f);
    if (a.logprob) a.logprob[row] = !has_target ? 0.0f : bad ? kNaN : empty ? kNegInf : scaled_distance(x_target, r.m, a.scale) - log_s;
}
__device__ __forceinline__ void logprob_write_top(const LogprobArgs &a, unsigned long long row, LogprobPart r, float log_s, int place, unsigned long long key)
{
    const bool bad = r.s != r.s, none = bad || !key;
    if (a.top_label) a.top_label[row * a.top + place] = none ? -1 : key_label(key);
    if (a.top_logprob) a.top_logprob[row * a.top + place] = bad ? kNaN : none ? kNegInf : scaled_distance(key_score(key), r.m, a.scale) - log_s;
}

// ---- the best `top` of many keys, by one wave ----
//
// A score that at least `top` of the wave's 64 values reach: the binary search over the ordered bits counts lanes with a ballot.  The
// highest 16 bits are enough, a score that is a little lower lets a few more candidates through.  Never below the lowest finite
// score: what is ruled out is no candidate.
__device__ __forceinline__ float reached_by(uint32_t k, int top)
{
    uint32_t t = 0;
#pragma unroll
    for (int b = 31; b >= 16; b--) {
        const uint32_t c = t | (1u << b);
        if (__builtin_popcountll(__ballot(k >= c)) >= top) t = c;
    }
    t = t < 0x00800000u ? 0x00800000u : t;
    return key_score((unsigned long long)t << 32);
}
__device__ __forceinline__ float reached_by(float v, int top) { return reached_by((uint32_t)(score_key(v, 0) >> 32), top); }

typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));

// Place of a lane's key among the wave's first n, best first (n <= 64; the other lanes' keys are 0).  All lanes read them from LDS, two a time.
__device__ __forceinline__ int key_place(unsigned long long key, int n, unsigned long long *list, int lane)
{
    list[lane] = key;
    __builtin_amdgcn_wave_barrier();   // the wave's LDS operations are in order
    int place = 0;
    for (int i = 0; i < n; i += 4) {
        const u64x2 p = *(const u64x2 *)(list + i), q = *(const u64x2 *)(list + i + 2);
        place += (p.x > key ? 1 : 0) + (p.y > key ? 1 : 0) + (q.x > key ? 1 : 0) + (q.y > key ? 1 : 0);
    }
    __builtin_amdgcn_wave_barrier();
    return place;
}

// Lanes below this one in a mask
__device__ __forceinline__ int below(unsigned long long mask) { return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0)); }

// Of the wave's keys k[0..N-1] (0: none) at most 64 that hold the best `top` are put at places 0, 1, ..; returns how many, and in
// `border` a key that none of the dropped ones reaches.  Counting reached candidates of a binary search: 16 bits of the score first, and
// if equal scores leave more than 64, all other bits, which ends at the `top`-th key itself, as every key is there once.
template <int N, typename F>
__device__ __forceinline__ int keep_best(const unsigned long long (&k)[N], int top, unsigned long long &border, F put)
{
    uint32_t t = 0;
#pragma unroll
    for (int b = 31; b >= 16; b--) {
        const uint32_t c = t | (1u << b);
        int count = 0;
#pragma unroll
        for (int i = 0; i < N; i++) count += __builtin_popcountll(__ballot((uint32_t)(k[i] >> 32) >= c));
        if (count >= top) t = c;
    }
    unsigned long long reach = (unsigned long long)t << 32;
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; i++) n += __builtin_popcountll(__ballot(k[i] >= reach && k[i]));
    if (n > 64)
        for (int b = 47; b >= 0; b--) {
            const unsigned long long c = reach | (1ull << b);
            int count = 0;
#pragma unroll
            for (int i = 0; i < N; i++) count += __builtin_popcountll(__ballot(k[i] >= c));
            if (count >= top) reach = c;
        }
    n = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const bool in = k[i] >= reach && k[i];
        const unsigned long long mask = __ballot(in);
        if (in) put(n + below(mask), k[i]);
        n += __builtin_popcountll(mask);
    }
    border = reach;
    return n;
}

// The alternatives of a row from at most 64 keys, one each of the first n lanes
__device__ __forceinline__ void logprob_write_list(const LogprobArgs &a, unsigned long long row, LogprobPart r, float log_s, unsigned long long key, int n, unsigned long long *list, int lane)
{
    const int place = key_place(key, n, list, lane);
    if (lane < n && place < a.top) logprob_write_top(a, row, r, log_s, place, key);
    if (lane >= n && lane < a.top) logprob_write_top(a, row, r, log_s, lane, 0);
}

// A wave's candidates for the alternatives, collected in LDS as its scores come by.  Taken are scores of at least `least`; when the list
// is full, the best are kept and `least` rises.  If equal scores still are too many, they are taken one by one, and only those whose key
// passes `border`.  An entry is the score's bits above the label; keys are made of them when the list is looked at, which is much rarer.
constexpr int kList = 128;
struct Candidates {
    unsigned long long *list;
    unsigned long long border = 0;
    int n = 0;
    float least = __builtin_inff();
    __device__ __forceinline__ explicit Candidates(unsigned long long *l) : list(l) {}
    __device__ __forceinline__ unsigned long long key_at(int i) const
    {
        if (i >= n) return 0;
        return score_key(__builtin_bit_cast(float, (uint32_t)(list[i] >> 32)), (unsigned)list[i]);
    }
    static __device__ __forceinline__ unsigned long long entry(float v, unsigned label) { return (unsigned long long)__builtin_bit_cast(uint32_t, v) << 32 | label; }
    __device__ __forceinline__ void shrink(int top, int lane)
    {
        __builtin_amdgcn_wave_barrier();   // the wave's LDS operations are in order
        unsigned long long k[kList / 64];
#pragma unroll
        for (int i = 0; i < kList / 64; i++) k[i] = key_at(64 * i + lane);
        __builtin_amdgcn_wave_barrier();
        n = keep_best(k, top, border, [&](int at, unsigned long long key) { list[at] = entry(key_score(key), (unsigned)key_label(key)); });
        least = fmaxf(least, key_score(border));
        __builtin_amdgcn_wave_barrier();
    }
    // N scores of every lane, their labels label(i), and the same score again from memory
    template <int N, typename L, typename M>
    __device__ __forceinline__ void offer(const float (&v)[N], int top, int lane, L label, M again)
    {
        for (bool full = false;; full = true) {
            int more = 0;
#pragma unroll
            for (int i = 0; i < N; i++) more += __builtin_popcountll(__ballot(v[i] >= least));
            if (n + more <= kList) {
                if (more) {
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const unsigned long long mask = __ballot(v[i] >= least);
                        if (!mask) continue;
                        if (mask >> lane & 1) list[n + below(mask)] = entry(v[i], label(i));
                        n += __builtin_popcountll(mask);
                    }
                }
                return;
            }
            if (full) break;
            if (n > 0) shrink(top, lane);
        }
        // a loop over memory: this is rare, and unrolled over the registers it would take more of them
        for (int i = 0; i < N; i++) {
            const float y = again(i);
            unsigned long long mask = __ballot(y >= least && score_key(y, label(i)) >= border);
            if (n + __builtin_popcountll(mask) > kList) {   // then n > 64, and no more than 64 are left
                shrink(top, lane);
                mask = __ballot(y >= least && score_key(y, label(i)) >= border);
            }
            if (mask >> lane & 1) list[n + below(mask)] = entry(y, label(i));
            n += __builtin_popcountll(mask);
        }
    }
    // at most 64 keys, one a lane (0: none)
    __device__ __forceinline__ unsigned long long finish(int top, int lane)
    {
        if (n > 64) shrink(top, lane);
        __builtin_amdgcn_wave_barrier();
        const unsigned long long key = key_at(lane);
        __builtin_amdgcn_wave_barrier();
        return key;
    }
};

// ---- short rows: a wave holds a row, E scores a lane, one row after the other ----
//
// Candidates for the alternatives are the scores that at least `top` lanes' best scores reach: about as many as are wanted.
// Bound by instruction issue, so what belongs to a row and not to its scores is done by a lane for each of the wave's rows, at the end.
// 35999 x 527 bf16 takes 13.2 us without alternatives and 20.6 with five (38 MB: 6.3 us at 6 TB/s), 100000 x 64 f32 with five
// 31.  With one row a wave these are 3, 3 and 10 us more; eight are no faster than four, and much slower while they leave waves unused.
// Candidates looked up by a lane each instead of picked out of all scores: 1.7 us less for the 527 labels.
constexpr unsigned kRows = 4;
template <typename T, int E>
__global__ __launch_bounds__(256, E > 12 ? 7 : 8) void logprob_wave_kernel(LogprobArgs a)
{
    __shared__ __align__(16) unsigned long long s_list[4][kList], s_top[4][kRows * APR_MAX_TOP];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (unsigned long long row0 = ((unsigned long long)blockIdx.x * 4 + wave) * a.rows; row0 < a.n; row0 += (unsigned long long)gridDim.x * 4 * a.rows) {
        const unsigned rows = (unsigned)min((unsigned long long)a.rows, a.n - row0);
        const int targets = a.target && (unsigned)lane < rows ? a.target[row0 + lane] : -1;
        LogprobPart mine = {0.0f, 0.0f, 0.0f};   // lane i: row i's
        T mine_t = (T)0.0f;
        const bool has_t = (unsigned)targets < a.n_labels;
        for (unsigned i_row = 0; i_row < rows; i_row++) {
            const T *x = (const T *)a.x + (row0 + i_row) * a.ld;
            float v[E], best = kNegInf;
#pragma unroll
            for (int i = 0; i < E; i++) v[i] = i < E - 1 || 64u * i + lane < a.n_labels ? to_f32(x[64 * i + lane]) : kNegInf;
            if (i_row == 0 && has_t) mine_t = x[lane * a.ld + (unsigned)targets];   // behind the first row's loads, not before them
#pragma unroll
            for (int i = 0; i < E; i++) best = fmaxf(best, v[i]);
            const int key_best = ordered(best);
            LogprobPart r;
            r.m = of_ordered(wave_max(key_best));
            ExpSum sum(r.m, a.scale);
#pragma unroll
            for (int i = 0; i < E; i++) sum.add(v[i]);
            wave_sums(sum.s, sum.u);
            const bool me = (unsigned)lane == i_row;
            mine.m = me ? r.m : mine.m;
            mine.s = me ? sum.s : mine.s;
            mine.u = me ? sum.u : mine.u;
            if (!a.top) continue;
            if (a.top == 1) {   // the lowest label that has the row's maximum
                unsigned label = 0;
#pragma unroll
                for (int i = E - 1; i >= 0; i--) {
                    const unsigned long long mask = __ballot(v[i] == r.m);
                    if (mask) label = 64 * i + __builtin_ctzll(mask);
                }
                if (lane == 0) s_top[wave][i_row] = r.m == kNegInf ? 0 : score_key(r.m, label);
                continue;
            }
            // of a few labels all may be candidates
            const float least = a.n_labels <= 16 ? kLowest : reached_by((uint32_t)key_best ^ 0x80000000u, a.top);
            // the lanes that have a candidate; while all their scores are no more than the wave's lanes, each lane looks one of them up
            const unsigned long long hits = __ballot(best >= least);
            unsigned long long *list = s_list[wave], key;
            int n;
            if (__builtin_popcountll(hits) * E <= 64) {
                unsigned label = lane;
                float y = v[0];
                if (E > 1) {
                    if (hits >> lane & 1) list[below(hits)] = lane;
                    __builtin_amdgcn_wave_barrier();   // the wave's LDS operations are in order
                    label = lane < __builtin_popcountll(hits) * E ? lane % E * 64u + (unsigned)list[lane / E] : a.n_labels;
                    y = label < a.n_labels ? to_f32(x[label]) : kNegInf;
                    __builtin_amdgcn_wave_barrier();
                }
                const unsigned long long mask = __ballot(y >= least);
                n = __builtin_popcountll(mask);
                if (mask >> lane & 1) list[below(mask)] = score_key(y, label);
                __builtin_amdgcn_wave_barrier();
                key = lane < n ? list[lane] : 0;
                __builtin_amdgcn_wave_barrier();
            } else {
                Candidates c(list);
                c.least = least;
                c.offer(v, a.top, lane, [&](int i) { return 64u * i + lane; }, [&](int i) { return 64u * i + lane < a.n_labels ? to_f32(x[64 * i + lane]) : kNegInf; });
                key = c.finish(a.top, lane);
                n = c.n;
            }
            const int place = key_place(key, n, list, lane);
            unsigned long long *to = s_top[wave] + i_row * a.top;
            if (lane < n && place < a.top) to[place] = key;
            if (lane >= n && lane < a.top) to[lane] = 0;
        }
        const float log_s = log_of_sum(mine.s);
        if ((unsigned)lane < rows) logprob_write(a, row0 + lane, mine, log_s, to_f32(mine_t), has_t);
        if (!a.top) continue;
        __builtin_amdgcn_wave_barrier();   // the wave's LDS operations are in order
        for (unsigned i = lane; i < (rows * a.top + 63u & ~63u); i += 64) {   // every lane, as they read each other's rows
            const unsigned i_row = min(i * a.per_top >> 16, rows - 1);
            LogprobPart r;
            r.m = __shfl(mine.m, i_row);
            r.s = __shfl(mine.s, i_row);
            const float l = __shfl(log_s, i_row);
            if (i < rows * a.top) logprob_write_top(a, row0, r, l, i, s_top[wave][i]);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- longer rows: a wave per row, or per piece of one, 1024 scores at a time, the next ones on their way ----
//
// No lane waits for another wave.  The sums are relative to the best score so far, which the wave shares: it is new in the k-th of many
// steps once in k times or so, where a lane's own maximum would be new in some lane at nearly every step.  It is renewed for any better score:
// relative to one that is g lower, s and u hold terms up to e^(scale g) and g e^(scale g), and what is left of their roundings when u is
// moved to the maximum, scale g times that of s, is too much for the entropy of a nearly sure answer (off by 3e-6 with g of up to
// 8 / scale).  A step's 16 terms of a lane are summed before they are added.
// 16-byte loads begin at the 16-byte unit that the row begins in (which is inside the allocation, as the row's first element is);
// what does not belong to the row counts as ruled out.
// The alternatives are among the `top` best units of 16 bytes, by a unit's best score, equal ones by their place: whatever a score
// outside of them is, each of them holds a better one, or an equal one in front of it.  So units are collected, two or four a step and lane
// instead of 16 scores, and the scores of those that are left are looked at when the row is done.
// HBM-bound without alternatives: 8192 x 32000 bf16 takes 96 us a call among others, 5.5 TB/s (97 to 101 by the
// profiler; 122 with 20 alternatives, and 141 when each score is offered by itself); a workgroup per row, whose waves meet three times
// a row, took 158.  Few rows are bound by latency: 64 x 131072 with 20 alternatives takes 11.2 us in 64 pieces a row.
// TOP: with alternatives, whose code takes registers (68 to 77: six or seven waves a SIMD instead of eight).
template <typename T, bool TOP>
__global__ __launch_bounds__(256, TOP ? 6 : 8) void logprob_stream_kernel(LogprobArgs a)
{
    constexpr int V = 16 / (int)sizeof(T), U = 16 / V;
    typedef T txv __attribute__((ext_vector_type(V)));
    __shared__ __align__(16) unsigned long long s_list[4][kList];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const unsigned long long works = a.n * a.pieces;
    const float c = a.scale * kLog2E, least_t = -200.0f / a.scale;
    for (unsigned long long work = (unsigned long long)blockIdx.x * waves + wave; work < works; work += (unsigned long long)gridDim.x * waves) {
        const unsigned long long row = a.pieces == 1 ? work : work / a.pieces;
        const unsigned piece = (unsigned)(work - row * a.pieces);
        const T *x = (const T *)a.x + row * a.ld;
        // all pieces but the first begin with a 16-byte unit, so that none but the last takes a step for what a unit holds of its neighbour
        const unsigned out = (unsigned)(((unsigned long long)x & 15) / sizeof(T)), off = piece ? 0 : out;
        const unsigned j0 = piece ? piece * a.piece_len - out : 0, j1 = piece + 1 < a.pieces ? (piece + 1) * a.piece_len - out : a.n_labels;
        const txv *units = (const txv *)(x + j0 - off);
        const unsigned len = j1 - j0 + off, n_units = (len + V - 1) / V, steps = (n_units + 64 * U - 1) / (64 * U);
        const unsigned keep = len - (n_units - 1) * V;   // elements of the last unit
        txv cur[U], next[U];
        const auto load = [&](txv(&to)[U], unsigned step) {
#pragma unroll
            for (int q = 0; q < U; q++) {
                const unsigned w = (step * U + q) * 64 + lane;
                if (w < n_units) to[q] = units[w];
                else to[q] = (T)kNegInf;
            }
        };
        load(cur, 0);
        float m = kNegInf, s = 0.0f, u = 0.0f;   // m: wave-uniform
        Candidates best(s_list[wave]);
        for (unsigned step = 0; step < steps; step++) {
            if (step + 1 < steps) load(next, step + 1);
            float v[16], top = kNegInf;
#pragma unroll
            for (int e = 0; e < 16; e++) v[e] = to_f32(cur[e / V][e % V]);
            if (step == 0 && off) {   // the first unit is lane 0's
#pragma unroll
                for (int i = 0; i < V - 1; i++) v[i] = lane == 0 && (unsigned)i < off ? kNegInf : v[i];
            }
            if (step == steps - 1 && keep < V) {
#pragma unroll
                for (int q = 0; q < U; q++) {
                    const bool last = (step * U + q) * 64 + lane == n_units - 1;
#pragma unroll
                    for (int i = 1; i < V; i++) v[q * V + i] = last && (unsigned)i >= keep ? kNegInf : v[q * V + i];
                }
            }
            float unit_max[U];
#pragma unroll
            for (int q = 0; q < U; q++) {
                unit_max[q] = v[q * V];
#pragma unroll
                for (int e = 1; e < V; e++) unit_max[q] = fmaxf(unit_max[q], v[q * V + e]);
                top = fmaxf(top, unit_max[q]);
            }
            if (__ballot(top > m)) {
                const float higher = wave_reduce(top, MaxOf()), d = m - higher, w = __builtin_amdgcn_exp2f(d * c);
                u = w * fmaf(fmaxf(d, least_t), s, u);
                s *= w;
                m = higher;
            }
            const float r = m == kNegInf ? 0.0f : m;
            float es = 0.0f, eu = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float t = v[e] - r, p = __builtin_amdgcn_exp2f(t * c);
                es += p;
                eu = fmaf(p, fmaxf(t, least_t), eu);
            }
            s += es;
            u += eu;
            if (TOP) {
                if (step == 0) best.least = reached_by(top, a.top);
                if (__ballot(top >= best.least))
                    best.offer(unit_max, a.top, lane, [&](int q) { return (step * U + q) * 64 + lane; }, [&](int q) {
                        float y = unit_max[0];
#pragma unroll
                        for (int i = 1; i < U; i++) y = q == i ? unit_max[i] : y;
                        return y;
                    });
            }
#pragma unroll
            for (int q = 0; q < U; q++) cur[q] = next[q];
        }
        LogprobPart r;
        wave_sums(s, u);
        r.m = m;
        r.s = s;
        r.u = u;
        const float log_s = log_of_sum(r.s);
        if (lane == 0) {
            if (a.pieces == 1) {
                const int t = a.target ? a.target[row] : -1;
                const bool has_t = t >= 0 && (unsigned)t < a.n_labels;
                logprob_write(a, row, r, log_s, has_t ? to_f32(x[t]) : 0.0f, has_t);
            } else
                a.part[work] = r;
        }
        if (!TOP) continue;
        // the best units, a lane each, once more: their scores are the candidates
        const unsigned long long unit_key = best.finish(a.top, lane);
        const bool has_unit = lane < best.n;
        const unsigned first = has_unit ? (unsigned)key_label(unit_key) * V : 0;   // of the unit's scores, from the piece's first unit on
        txv unit;
        if (has_unit) unit = units[first / V];
        else unit = (T)kNegInf;
        float y[V];
#pragma unroll
        for (int e = 0; e < V; e++) y[e] = has_unit && first + e >= off && first + e < len ? to_f32(unit[e]) : kNegInf;
        Candidates c_top(s_list[wave]);
        c_top.least = reached_by(has_unit ? key_score(unit_key) : kNegInf, a.top);
        c_top.offer(y, a.top, lane, [&](int e) { return j0 - off + first + e; }, [&](int e) {
            const unsigned at = first + e;
            return has_unit && at >= off && at < len ? to_f32(x[j0 - off + at]) : kNegInf;
        });
        const unsigned long long key = c_top.finish(a.top, lane);
        if (a.pieces == 1)
            logprob_write_list(a, row, r, log_s, key, c_top.n, c_top.list, lane);
        else {
            const int place = key_place(key, c_top.n, c_top.list, lane);
            if (lane < c_top.n && place < a.top) a.part_top[work * a.top + place] = key;
            if (lane >= c_top.n && lane < a.top) a.part_top[work * a.top + lane] = 0;
        }
    }
}

constexpr unsigned kJoined = 1024, kHeads = 8;
static_assert(2 * kHeads == kJoined / 64, "one set of registers for both");

// ---- the pieces of a row joined, a wave per row: 5.8 us for one row, 5.4 for 64, most of it the launch and two loads in a row ----
__global__ __launch_bounds__(64) void logprob_join_kernel(LogprobArgs a, int type)
{
    __shared__ __align__(16) unsigned long long s_list[64];
    const int lane = threadIdx.x;
    for (unsigned long long row = blockIdx.x; row < a.n; row += gridDim.x) {
        // The pieces' lists, asked for before the sums are joined: all their keys where those are 1024 at most, otherwise the best kHeads of
        // each of at most 128 pieces (logprob_plan), lane i's and i + 64's.
        const unsigned long long *keys = a.part_top + row * a.pieces * a.top;
        const unsigned all = a.pieces * a.top;
        unsigned long long k[kJoined / 64];
        if (all <= kJoined) {
#pragma unroll
            for (unsigned i = 0; i < kJoined / 64; i++) k[i] = 64u * i + lane < all ? keys[64 * i + lane] : 0;
        } else {
#pragma unroll
            for (unsigned i = 0; i < 2 * kHeads; i++) {
                const unsigned p = lane + i / kHeads * 64;
                k[i] = p < a.pieces ? keys[p * a.top + i % kHeads] : 0;
            }
        }
        unsigned long long sample = 0;
        if (a.top && a.pieces < 64) {
            const unsigned each = 64 / a.pieces, p = lane / each, j = lane - p * each;
            if (p < a.pieces && j < (unsigned)a.top) sample = keys[(unsigned long long)p * a.top + j];
        } else if (a.top)
            for (unsigned p = lane; p < a.pieces; p += 64) sample = max(sample, keys[(unsigned long long)p * a.top]);
        const LogprobPart *part = a.part + row * a.pieces;
        const int t = a.target ? a.target[row] : -1;
        const bool has_t = t >= 0 && (unsigned)t < a.n_labels;
        float xt = 0.0f;
        if (has_t) {
            const unsigned long long at = row * a.ld + (unsigned)t;
            xt = type == 0 ? ((const float *)a.x)[at] : type == 1 ? to_f32(((const f16_t *)a.x)[at]) : to_f32(((const bf16_t *)a.x)[at]);
        }
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
        wave_sums(s, u);
        r.s = s;
        r.u = u;
        const float log_s = log_of_sum(r.s);
        if (lane == 0) logprob_write(a, row, r, log_s, xt, has_t);
        if (!a.top) continue;
        // A score that `top` of 64 of the keys reach, each piece's best or as many of each as make 64, bounds the ones that matter: about
        // as many as are wanted.  keep_best, which counts all keys 16 times, is for what is left over that.
        unsigned long long border;
        const auto put = [&](int at, unsigned long long key) { s_list[at] = key; };
        const float least = reached_by(sample ? key_score(sample) : kNegInf, a.top);
        const unsigned long long reach = score_key(least, 0) >> 32 << 32;
        const bool behind = all > kJoined && (k[kHeads - 1] >= reach || k[2 * kHeads - 1] >= reach);   // the heads' last ones count, so what is behind them may
        int n = 0;
#pragma unroll
        for (unsigned i = 0; i < kJoined / 64; i++) {
            if (k[i] < reach) k[i] = 0;
            n += __builtin_popcountll(__ballot(k[i] != 0));
        }
        if (__ballot(behind)) {
            // some piece holds many of the best: all keys, 64 at a time, to what is kept of those before
            n = 0;
            for (unsigned i = 0; i < all; i += 64) {
                const unsigned long long two[2] = {lane < n ? s_list[lane] : 0, i + lane < all ? keys[i + lane] : 0};
                __builtin_amdgcn_wave_barrier();
                n = keep_best(two, a.top, border, put);
                __builtin_amdgcn_wave_barrier();
            }
        } else if (n <= 64) {
            n = 0;
#pragma unroll
            for (unsigned i = 0; i < kJoined / 64; i++) {
                const unsigned long long mask = __ballot(k[i] != 0);
                if (k[i]) put(n + below(mask), k[i]);
                n += __builtin_popcountll(mask);
            }
        } else
            n = keep_best(k, a.top, border, put);
        __builtin_amdgcn_wave_barrier();
        logprob_write_list(a, row, r, log_s, lane < n ? s_list[lane] : 0, n, s_list, lane);
        __builtin_amdgcn_wave_barrier();
    }
}

// How a call's rows are cut: scores a lane of a wave that holds a whole row (0: rows are streamed), pieces of a row and their length.
struct LogprobPlan {
    int each;
    unsigned pieces, piece_len;
    size_t work;   // bytes
};
// Waves that have places at the same time in the form with alternatives (2000 rows of 100000 take 93 us in three pieces, 97 in two).
// Pieces are whole steps (64 rows of 131072, 20 alternatives: 16.4 us in 64 pieces of two steps, about 2 more in 50 of two and a half), and
// with alternatives there are no more than the join's registers hold (one row of 131071, 20 alternatives: 10.2 us in 128 pieces, 13.0 in
// 51, 15.1 in 33, 20.9 in 17).
constexpr size_t kPlaces = 6144, kStep = 1024;
// Up to here a row is not cut: 2000 scores take 5.6 us as one and 8.7 as two pieces and their join, 4000 8.3 and 8.7, 6000 9.9 and 9.0.
constexpr size_t kWhole = 4096;
inline LogprobPlan logprob_plan(size_t n, size_t c, int top)
{
    LogprobPlan p = {0, 1, (unsigned)c, 0};
    if (c <= kStep) {
        p.each = (int)((c + 63) / 64);
        return p;
    }
    if (c <= kWhole) return p;
    size_t pieces = std::max<size_t>(kPlaces / std::max<size_t>(n, 1), 1);
    if (top > 0) pieces = std::min(pieces, std::max<size_t>(kJoined / (size_t)top, 128));
    const size_t steps = (c + kStep - 1) / kStep;
    p.piece_len = (unsigned)((steps + pieces - 1) / pieces * kStep);
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
    unsigned pieces, piece_units;   // a row's units of 16 bytes (of grad) that a wave takes
};

// A wave per row, or per piece of one.  Reads and writes every score once; an element is read before its place is written by the same
// lane, so grad may be x.  Stores are whole 16-byte units of grad, wherever its rows begin (what a row has before its first
// and behind its last whole unit goes element by element); the loads follow them at whatever alignment x has then, which the hardware takes.
// p = exp2(scale log2 e (x - m) - log2 e log s): x - m is exact for the scores that matter, the rest rounds once.
// HBM-bound: 8192 x 32000 bf16 takes 179 us a call among others, 5.8 TB/s (182 to 185 by the profiler),
// 509 x 50257 f32 38 us, 5.3 TB/s (39 to 40; a multiplication by a number of as many bytes: 6.1 and 6.0).  Stores that pass the caches by: 183 us against 192.
template <typename T, bool ENTROPY>
__global__ __launch_bounds__(256) void logprob_grad_kernel(LogprobGradArgs a)
{
    constexpr int V = 16 / (int)sizeof(T);
    typedef T txv __attribute__((ext_vector_type(V)));
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const unsigned long long works = a.n * a.pieces;
    const float c = a.scale * kLog2E;
    for (unsigned long long work = (unsigned long long)blockIdx.x * waves + wave; work < works; work += (unsigned long long)gridDim.x * waves) {
        const unsigned long long row = a.pieces == 1 ? work : work / a.pieces;
        const unsigned piece = (unsigned)(work - row * a.pieces);
        const T *x = (const T *)a.x + row * a.ld;
        T *grad = (T *)a.grad + row * a.ld_grad;
        // the row: `head` elements up to grad's first 16-byte unit, whole units, `tail` elements
        const unsigned off = (unsigned)(((unsigned long long)grad & 15) / sizeof(T));
        const unsigned head = off ? min(V - off, a.n_labels) : 0, n_units = (a.n_labels - head) / V, tail = a.n_labels - head - n_units * V;
        const unsigned w0 = piece * a.piece_units, w1 = min(w0 + a.piece_units, n_units);
        const float m = a.stat[2 * row], log_s = a.stat[2 * row + 1];
        const int t = a.target ? a.target[row] : -1;
        const bool empty = m == kNegInf, has_t = t >= 0 && (unsigned)t < a.n_labels && !empty;
        const float g = has_t && a.g_logprob ? a.g_logprob[row] : 0.0f, h = ENTROPY ? a.g_entropy[row] : 0.0f, ent = ENTROPY ? a.entropy[row] : 0.0f;
        const float gs = -a.scale * g, hs = -a.scale * h, ls2 = log_s * kLog2E;
        const auto one = [&](float v) {
            const float l2 = fmaf(v - m, c, -ls2), p = __builtin_amdgcn_exp2f(l2);
            float f = gs;
            if (ENTROPY) f = fmaf(hs, fmaf(fmaxf(l2, -300.0f), 0.69314718055994530942f, ent), gs);   // exp2(-300) = 0; no 0 * inf
            return empty ? 0.0f : p * f;
        };
        const unsigned tu = has_t && (unsigned)t >= head ? ((unsigned)t - head) / V : 0xFFFFFFFFu, tv = ((unsigned)t - head) % V;
        const T *xb = x + head;
        T *gb = grad + head;
#pragma unroll 4
        for (unsigned w = w0 + lane; w < w1; w += 64) {
            txv v, r;
            __builtin_memcpy(&v, xb + (unsigned long long)w * V, 16);
            float f[V];
#pragma unroll
            for (int i = 0; i < V; i++) f[i] = one(to_f32(v[i]));
            if (w == tu) {
#pragma unroll
                for (int i = 0; i < V; i++) f[i] -= i == (int)tv ? gs : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < V; i++) r[i] = from_f32<T>(f[i]);
            __builtin_nontemporal_store(r, (txv *)(gb + (unsigned long long)w * V));
        }
        if (piece == 0) {
            const unsigned e = (unsigned)lane < head ? lane : a.n_labels - tail + (lane - 32);
            if ((unsigned)lane < head || (lane >= 32 && lane - 32 < (int)tail)) grad[e] = from_f32<T>(one(to_f32(x[e])) - (has_t && e == (unsigned)t ? gs : 0.0f));
        }
    }
}

}  // namespace apr
