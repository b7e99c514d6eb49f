// linear_i8.hip.h -- out[m][n] = (sum_k x[m][k] w[n][k]) x_scale[m] w_scale[n] + bias[n] for 8-bit x and w.
//
// The sum is exact in 32 bits (|product| <= 2^14, k < 2^17) and does not depend on its order.  Both operands have k contiguous,
// which is how the matrix instruction wants them: a lane holds 16 consecutive k of one row.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
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

// 16 bytes of a row from k on, 0 from `end` on.  WHOLE: the rows are 16-byte aligned, and the unit that k ends in is read whole (it lies in
// the row's stride, and inside the allocation, as its first byte is); otherwise a unit begins at any byte, and the one that k ends in is
// read byte by byte.
template <bool WHOLE>
__device__ __forceinline__ i32x4 linear_unit(const int8_t *row, unsigned k, unsigned end)
{
    i32x4 v = {0, 0, 0, 0};
    if (k >= end) return v;
    if (WHOLE) return *(const i32x4 *)(row + k);
    if (k + 16u <= end) {
        __builtin_memcpy(&v, row + k, 16);
        return v;
    }
    for (unsigned c = 0; k + c < end; c++) v[c >> 2] |= (int)(uint8_t)row[k + c] << (8 * (c & 3));
    return v;
}

// The sum times both scales, one after the other.  The larger one is last where 2^31 of it are beyond the largest float (the product itself
// then is only if the other one is as large); a whole number of the smaller one loses nothing below the normal range.
__device__ __forceinline__ bool linear_large(float x_scale) { return fabsf(x_scale) >= 0x1p+97f; }
__device__ __forceinline__ float linear_scaled(int sum, float x_scale, float w_scale)
{
    const bool large = linear_large(x_scale);
    return (float)sum * (large ? w_scale : x_scale) * (large ? x_scale : w_scale);
}

// ---- tiled kernel: operands 16 bytes at a time, straight from memory to LDS ----
//
// A stage is 128 bytes of k of every row of the tile, eight units of 16 bytes; unit c of row r lies at place c ^ ((r >> 1) & 7).  An LDS
// read of 16 bytes a lane serves 16 lanes at a time, which hit all 64 banks once if their places differ modulo 256 bytes: the
// hardware's sixteen (lanes 0-3, 12-15, 20-23, 24-27 and so on) are eight even and eight odd rows whose r >> 1 differ modulo 8.
// (With r & 7 they pair up: 104 million cycles of bank conflicts in a product of 16384 x 8192 x 8192 instead of 3, though not more time.)
// A DMA instruction fills 1 KiB of LDS, eight rows, lane by lane; the swizzle is which unit each lane asks for.  Rows past the matrix
// and units past k are out of the buffer's range, which reads as 0.
//
// What bounds 256 x 256 tiles: the chip's power.  16384 x 8192 x 8192 takes 0.92-0.94 ms a call among others (2.3-2.4 POPS;
// 0.94-0.98 by the profiler) at 1.8 GHz, where the matrix units work 62 % of the cycles; matrix instructions alone, without loads, take
// 0.69 ms, since random operands bring the clock down (from registers 3.1-3.5 POPS, and 4.6 on zeros), and with the LDS reads 0.78.
// LDS-DMA: 64 lanes x 16 B from a buffer to 1 KiB of LDS at byte address lds (wave-uniform).  The caller waits on vmcnt.
__device__ __forceinline__ void linear_dma(i32x4 rs, unsigned voff, unsigned lds)
{
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\t"
                 "buffer_load_dwordx4 %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(voff), "s"(rs), "s"(lds)
                 : "memory");
}

template <int N>
__device__ __forceinline__ void wait_dma_and_meet()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// the 256 or so tiles that run together share rows of x and w in their XCD's L2: the tiles are cut into one run for each of the
// 8 XCDs (workgroups go to them in turn), and a run walks G tiles down m for each step along n
__device__ __forceinline__ void linear_tile(unsigned block, unsigned tiles_m, unsigned tiles_n, unsigned &tm, unsigned &tn)
{
    const unsigned tiles = tiles_m * tiles_n, xcd = block & 7u, q = tiles >> 3, r = tiles & 7u;
    const unsigned t = xcd * q + min(xcd, r) + (block >> 3);
    const unsigned G = 8, per = G * tiles_n, g = t / per, in = t - g * per;
    const unsigned rows = min(G, tiles_m - g * G);
    tn = in / rows;
    tm = g * G + in - tn * rows;
}

// EVERY: a DMA instruction in front of every EVERY-th matrix instruction, so that the 64 KiB of a stage do not queue up before the step's
// first product (128 x 128 tiles: 2-3 % less time, 256 x 256: 1 %); 0: all at the top (64 x 64 tiles have too few instructions a step).
// DMA false: rows that are not 16-byte aligned.  The stages come through registers, a step ahead, and are written to the same places.
template <typename T, int BM, int BN, int BK, int NBUF, int WM, int WN, bool DMA, int EVERY>
__global__ __launch_bounds__(WM * WN * 64, 1) void linear_i8_tile_kernel(LinearI8Args a, unsigned tiles_m, unsigned tiles_n)
{
    constexpr int WAVES = WM * WN, FM = BM / WM / 32, FN = BN / WN / 32, KS = BK / 32, UNITS = BK / 16, RPD = 64 / UNITS;
    constexpr int DA = BM / RPD / WAVES, DB = BN / RPD / WAVES, ABYTES = BM * BK, STAGE = (BM + BN) * BK;
    extern __shared__ __align__(128) int8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned tm, tn;
    linear_tile(blockIdx.x, tiles_m, tiles_n, tm, tn);
    tm = __builtin_amdgcn_readfirstlane(tm);   // the division is vector code
    tn = __builtin_amdgcn_readfirstlane(tn);
    const unsigned m0 = tm * BM, n0 = tn * BN;
    const unsigned rows_x = min((unsigned)BM, a.m - m0), rows_w = min((unsigned)BN, a.n - n0);
    const unsigned k16 = (a.k + 15u) & ~15u;
    const unsigned ld_x = (unsigned)a.ld_x, ld_w = (unsigned)a.ld_w;
    unsigned long long bx = (unsigned long long)(a.x + (unsigned long long)m0 * a.ld_x), bw = (unsigned long long)(a.w + (unsigned long long)n0 * a.ld_w);
    // Range of the tile's rows: a row past the matrix begins beyond it (k16 <= ld) and reads as 0, at every stage, since a stage moves
    // the base along k and not the range
    const unsigned nx = (rows_x - 1) * ld_x + k16, nw = (rows_w - 1) * ld_w + k16;

    // this lane's row of a DMA instruction's eight, and its unit: the rows of every other instruction are 8 to 15 modulo 16
    static_assert(BK == 128 && DA % 2 == 0 && DB % 2 == 0, "units and their places");
    const int dr = lane / UNITS, dp = lane % UNITS;
    const int du[2] = {dp ^ (dr >> 1), dp ^ (dr >> 1) ^ 4};
    unsigned vx[DA], vw[DB];
#pragma unroll
    for (int i = 0; i < DA; i++) vx[i] = (unsigned)((wave * DA + i) * RPD + dr) * ld_x + 16u * du[i & 1];
#pragma unroll
    for (int i = 0; i < DB; i++) vw[i] = (unsigned)((wave * DB + i) * RPD + dr) * ld_w + 16u * du[i & 1];
    const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) int8_t *)lds;

    const unsigned full = a.k / BK, steps = (a.k + BK - 1) / BK;
    unsigned k_next = 0;   // first k of the next stage to fetch
    int slot_in = 0;
    static_assert(DMA || NBUF == 2, "one stage is in registers");
    static_assert(EVERY * (DA + DB - 1) < (KS - 1) * FM * FN || EVERY == 0, "all of a stage is asked for before the waves meet");
    i32x4 hx[DMA ? 1 : DA], hw[DMA ? 1 : DB], rx, rw;
    bool past[2];
    unsigned to;
    auto piece = [&](int i) {   // one DMA instruction of the stage that fetch has begun
        if (i < DA) linear_dma(rx, past[i & 1] ? 0xFFFFFFF0u : vx[i], to + (wave * DA + i) * 1024);
        else linear_dma(rw, past[i & 1] ? 0xFFFFFFF0u : vw[i - DA], to + ABYTES + (wave * DB + i - DA) * 1024);
    };
    auto fetch = [&]() {
        if (!DMA) {
#pragma unroll
            for (int i = 0; i < DA; i++) {
                const unsigned r = (wave * DA + i) * RPD + dr;
                hx[DMA ? 0 : i] = linear_unit<false>(a.x + (m0 + r) * a.ld_x, k_next + 16u * du[i & 1], r < rows_x ? a.k : 0);
            }
#pragma unroll
            for (int i = 0; i < DB; i++) {
                const unsigned r = (wave * DB + i) * RPD + dr;
                hw[DMA ? 0 : i] = linear_unit<false>(a.w + (n0 + r) * a.ld_w, k_next + 16u * du[i & 1], r < rows_w ? a.k : 0);
            }
            k_next += BK;
            return;
        }
        // past k an empty stage keeps the count of loads in flight: a range of 0
        const unsigned left = k_next < a.k ? a.k - k_next : 0;
        rx = {(int)(unsigned)bx, (int)(unsigned)(bx >> 32), left ? (int)nx : 0, 0x00020000};
        rw = {(int)(unsigned)bw, (int)(unsigned)(bw >> 32), left ? (int)nw : 0, 0x00020000};
        past[0] = 16u * du[0] >= left;
        past[1] = 16u * du[1] >= left;
        to = lds0 + slot_in * STAGE;
        if (left > BK) { bx += BK; bw += BK; }
        k_next += BK;
        slot_in = slot_in + 1 == NBUF ? 0 : slot_in + 1;
        if (EVERY == 0) {
#pragma unroll
            for (int i = 0; i < DA + DB; i++) piece(i);
        }
    };
    auto commit = [&]() {   // what fetch left in registers
        if (DMA) return;
        int8_t *to = lds + slot_in * STAGE + lane * 16;
#pragma unroll
        for (int i = 0; i < DA; i++) *(i32x4 *)(to + (wave * DA + i) * 1024) = hx[DMA ? 0 : i];
#pragma unroll
        for (int i = 0; i < DB; i++) *(i32x4 *)(to + ABYTES + (wave * DB + i) * 1024) = hw[DMA ? 0 : i];
        slot_in ^= 1;
    };

    const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN), r32 = lane & 31, half = lane >> 5;
    unsigned pa[KS];   // this lane's place in a row for each k of 32
#pragma unroll
    for (int kk = 0; kk < KS; kk++) pa[kk] = (unsigned)(((2 * kk + half) ^ ((r32 >> 1) & 7)) * 16);
    const int8_t *la = lds + (wm + r32) * BK, *lb = lds + ABYTES + (wn + r32) * BK;

    i32x16 acc[FM][FN] = {};
    i32x4 fa[2][FM], fb[2][FN];
    auto read = [&](int set, unsigned stage, int kk) {
#pragma unroll
        for (int i = 0; i < FM; i++) fa[set][i] = *(const i32x4 *)(la + stage + i * 32 * BK + pa[kk]);
#pragma unroll
        for (int j = 0; j < FN; j++) fb[set][j] = *(const i32x4 *)(lb + stage + j * 32 * BK + pa[kk]);
    };
    // at: matrix instructions of this step before these; every EVERY-th has a DMA instruction in front of it
    auto multiply = [&](int set, int at) {
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
            for (int j = 0; j < FN; j++) {
                if (EVERY > 0) {
                    const int q = at + i * FN + j;
                    if (q >= 0 && q % (EVERY ? EVERY : 1) == 0 && q / (EVERY ? EVERY : 1) < DA + DB) {
                        __builtin_amdgcn_sched_barrier(0);
                        piece(q / (EVERY ? EVERY : 1));
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[set][j], fa[set][i], acc[i][j], 0, 0, 0);
            }
    };

    constexpr int FLY = (NBUF - 2) * (DA + DB);   // loads that may still be on their way when the next stage has to be there
#pragma unroll
    for (int s = 0; s < NBUF - 1; s++) {
        fetch();
        if (DMA && EVERY > 0) {
#pragma unroll
            for (int i = 0; i < DA + DB; i++) piece(i);
        }
    }
    commit();
    wait_dma_and_meet<FLY>();
    unsigned stage = 0;
    if (full) read(0, 0, 0);
    for (unsigned s = 0; s < full; s++) {
        fetch();   // into the stage that was read before the last meeting
        const unsigned next = stage + STAGE == NBUF * STAGE ? 0 : stage + STAGE;
#pragma unroll
        for (int kk = 0; kk < KS; kk++) {
            if (kk + 1 < KS) read((kk + 1) & 1, stage, kk + 1);
            else {
                commit();
                wait_dma_and_meet<FLY>();
                read(0, next, 0);   // past the last whole stage: the tail's, or zeros
            }
            multiply(kk & 1, kk * FM * FN);
        }
        stage = next;
    }
    if (steps > full) {
        // the tail: units past k are 0; the unit that k ends in is cut in x, which is enough
#pragma unroll
        for (int kk = 0; kk < KS; kk++) {
            read(kk & 1, stage, kk);
            const int left = (int)a.k - (int)(full * BK + 32 * kk + 16 * half);
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const int keep = left - 4 * d;
                const int mask = keep >= 4 ? -1 : keep <= 0 ? 0 : (1 << (8 * keep)) - 1;
#pragma unroll
                for (int i = 0; i < FM; i++) fa[kk & 1][i][d] &= mask;
            }
            multiply(kk & 1, -1000);
        }
    }
    // The end of a tile.  w is the instruction's first operand, so a lane holds runs of four neighbouring n of one m: 32 rows of the
    // wave's outputs at a time go through the wave's own piece of the LDS and out again in whole 16-byte units of a row.
    constexpr int TN = BN / WN, ROW = TN * (int)sizeof(T) + 16;   // + 16: rows start in other banks
    static_assert(WAVES * 32 * ROW + 2 * BN * 4 <= NBUF * STAGE, "the outputs fit in the stages");
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");   // every stage is read, every load has landed
    float *s_ws = (float *)(lds + WAVES * 32 * ROW), *s_b = s_ws + BN;
    for (int c = threadIdx.x; c < BN; c += WAVES * 64) {
        const bool in = n0 + c < a.n;
        s_ws[c] = in ? a.w_scale[n0 + c] : 0.0f;
        s_b[c] = in && a.bias ? a.bias[n0 + c] : 0.0f;
    }
    __syncthreads();
    int8_t *mine = lds + wave * 32 * ROW;
    constexpr int V = 16 / (int)sizeof(T), LPR = TN / V, RPI = 64 / LPR;   // values of a unit, lanes a row, rows an instruction
    typedef T tx4 __attribute__((ext_vector_type(4)));
    typedef T txv __attribute__((ext_vector_type(V)));
    const bool units = ((a.ld_out * sizeof(T) | (unsigned long long)a.out) & 15) == 0;
    T *out = (T *)a.out + (unsigned long long)m0 * a.ld_out + n0 + wn;
    const unsigned m_left = a.m - m0, n_left = a.n - n0 > (unsigned)wn ? a.n - n0 - wn : 0;
#pragma unroll
    for (int i = 0; i < FM; i++) {
        const unsigned mr = wm + 32 * i;
        const float xs = mr + r32 < m_left ? a.x_scale[m0 + mr + r32] : 0.0f;
        const auto put = [&](auto scaled) {
#pragma unroll
            for (int j = 0; j < FN; j++)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const int c = 32 * j + 8 * g + 4 * half;
                    tx4 v;
#pragma unroll
                    for (int q = 0; q < 4; q++) v[q] = from_f32<T>(scaled(acc[i][j][4 * g + q], s_ws[wn + c + q]) + s_b[wn + c + q]);
                    *(tx4 *)(mine + r32 * ROW + c * (int)sizeof(T)) = v;
                }
        };
        // apart from each other: chosen for each output, the order takes 3 % more time of 4096 x 4096 x 1024 (28.5 us against 27.7)
        if (__builtin_expect(__ballot(linear_large(xs)) != 0, 0)) put([&](int sum, float ws) { return linear_scaled(sum, xs, ws); });
        else put([&](int sum, float ws) { return (float)sum * xs * ws; });
        __builtin_amdgcn_wave_barrier();   // the wave's LDS operations are in order
        if (units) {
#pragma unroll
            for (int r = 0; r < 32; r += RPI) {
                const unsigned row = r + lane / LPR, c = lane % LPR * V;
                const txv v = *(const txv *)(mine + row * ROW + c * sizeof(T));
                T *o = out + (mr + row) * a.ld_out + c;
                if (mr + row < m_left) {
                    if (c + V <= n_left) *(txv *)o = v;
                    else
                        for (int q = 0; q < V; q++)
                            if (c + q < n_left) o[q] = v[q];
                }
            }
        } else {
#pragma unroll 8
            for (int r = 0; r < TN / 2; r++) {
                const unsigned idx = 64 * r + lane, row = idx / TN, c = idx % TN;
                if (mr + row < m_left && c < n_left) out[(mr + row) * a.ld_out + c] = *(const T *)(mine + row * ROW + c * sizeof(T));
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- few tiles: every wave takes a part of k for the same 16 n and G x 16 m, straight from memory to registers ----
//
// Blocks of 256 k go to the W waves in turn.  A load takes 64 neighbouring bytes of 16 rows (the 16 x 16 x 64 instruction's layout: with the
// 32 x 32 x 32 one a load takes 32 bytes of 32 rows, and the lines of 16 waves do not stay in the L1 until the rest is asked for:
// 1 x 8192 x 8192 takes 14.3 us against 19.4, 4.7 TB/s of weights; twice as many loads in flight: the same).  The waves' partial sums, exact whole numbers, meet in LDS.
template <typename T, int W, int G, bool WHOLE>
__global__ __launch_bounds__(W * 64) void linear_i8_few_kernel(LinearI8Args a)
{
    __shared__ int s_part[W][G * 4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, quarter = lane >> 4;
    const unsigned long long tiles_n = (a.n + 15u) / 16u, tiles = (a.m + 16u * G - 1u) / (16u * G) * tiles_n;
    const unsigned blocks = (a.k + 255u) / 256u;
    for (unsigned long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const unsigned m0 = (unsigned)(tile / tiles_n) * (16u * G), n0 = (unsigned)(tile % tiles_n) * 16u;
        const unsigned k_w = n0 + r16 < a.n ? a.k : 0;   // a row past the matrix has no units
        const int8_t *w = a.w + (n0 + r16) * a.ld_w, *x[G];
        unsigned k_x[G];
#pragma unroll
        for (int g = 0; g < G; g++) {
            k_x[g] = m0 + 16 * g + r16 < a.m ? a.k : 0;
            x[g] = a.x + (m0 + 16 * g + r16) * a.ld_x;
        }
        i32x4 acc[G] = {}, fw[4], fx[G][4];
        auto load = [&](unsigned b) {
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const unsigned k = b * 256u + 64u * u + 16u * quarter;
                fw[u] = linear_unit<WHOLE>(w, k, k_w);
#pragma unroll
                for (int g = 0; g < G; g++) fx[g][u] = linear_unit<WHOLE>(x[g], k, k_x[g]);
            }
        };
        load(wave);
        for (unsigned b = wave; b < blocks; b += W) {
            if (WHOLE && b * 256u + 256u > a.k) {
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        const int keep = (int)a.k - (int)(b * 256u + 64u * u + 16u * quarter) - 4 * d;
                        const int mask = keep >= 4 ? -1 : keep <= 0 ? 0 : (1 << (8 * keep)) - 1;
#pragma unroll
                        for (int g = 0; g < G; g++) fx[g][u][d] &= mask;
                    }
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int g = 0; g < G; g++) acc[g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fx[g][u], fw[u], acc[g], 0, 0, 0);
            load(b + W);
        }
        __syncthreads();   // the last tile's sums are read
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int e = 0; e < 4; e++) s_part[wave][4 * g + e][lane] = acc[g][e];
        __syncthreads();
        for (int e = wave; e < 4 * G; e += W) {
            int sum = 0;
#pragma unroll
            for (int v = 0; v < W; v++) sum += s_part[v][e][lane];
            const unsigned m = m0 + 16 * (e >> 2) + 4 * quarter + (e & 3), n = n0 + r16;
            if (m < a.m && n < a.n) ((T *)a.out)[m * a.ld_out + n] = from_f32<T>(linear_scaled(sum, a.x_scale[m], a.w_scale[n]) + (a.bias ? a.bias[n] : 0.0f));
        }
    }
}

// ---- which kernel ----
//
// Microseconds of a variant: t0 for each tile that a CU walks one after the other, and a step of 128 k takes `alone` (its latency,
// shared by the `beside` tiles that fit a CU together) or `full` for each tile (its throughput), whichever is longer.  Measured with
// one to eight rounds of tiles, bf16 out; 1024 x 8192 x 8192: 98 / 73 / 121 / 103 us by 256 x 256, 128 x 128, 64 x 64 with four and with
// two stages (the rule: 98 / 73 / 127 / 105), 256 x 8192 x 8192: 85 / 50 / 32 / 39 (98 / 50 / 34 / 39), 16384 x 8192 x 8192: 925 / 1113 / 1780 / 1612.
// The few kernel: 2.3 us and, for each tile of a CU, 0.8 ns a k (16 m) or 1.4 ns a k (32 m): 256 x 527 x 1024 takes
// 5.1 us in a captured row of calls (5.8 by the profiler) against 6.7 by 64 x 64 tiles, 64 x 2000 x 4096 8.7; 4096 x 527 x 1024 would take 30 against 9.4.
struct LinearCost {
    int tile, beside;
    float t0, alone, full;
};
constexpr LinearCost kLinearCost[4] = {{256, 1, 5.0f, 1.45f, 1.72f}, {128, 2, 3.6f, 0.73f, 0.54f}, {64, 2, 3.5f, 0.29f, 0.24f}, {64, 5, 2.5f, 0.57f, 0.20f}};
enum { kLinear256, kLinear128, kLinear64Deep, kLinear64, kLinearFew };

// whole: the rows are 16-byte aligned; otherwise there are 128 x 128 tiles, whose steps then take about twice as long, and the few kernel,
// which takes four times as long
inline int linear_variant(unsigned m, unsigned n, unsigned k, bool whole, int n_cus)
{
    const float steps = (float)((k + 127) / 128), cus = (float)n_cus;
    const float few_tiles = (float)(m <= 16 ? 1 : (m + 31) / 32) * (float)((n + 15) / 16);
    float best = 2.3f + ceilf(few_tiles / cus) * (m <= 16 ? 0.8e-3f : 1.4e-3f) * (float)k * (whole ? 1.0f : 4.0f);
    int variant = kLinearFew;
    for (int v = 0; v < 4; v++) {
        if (!whole && v != kLinear128) continue;
        const LinearCost &c = kLinearCost[v];
        const float tiles = (float)((m + c.tile - 1) / c.tile) * (float)((n + c.tile - 1) / c.tile);
        const float per_cu = ceilf(tiles / cus), rounds = ceilf(per_cu / (float)c.beside);
        const float us = c.t0 * rounds + steps * fmaxf(c.alone * rounds, c.full * per_cu) * (whole ? 1.0f : 2.0f);
        if (us < best) { best = us; variant = v; }
    }
    return variant;
}

}  // namespace apr
