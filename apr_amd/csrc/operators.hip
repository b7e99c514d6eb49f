// operators.hip -- C ABI of the operators behind a label head (include/apr.h): argument checks and launches.
//
// Every entry checks its arguments before it looks at the engine, so that a bad call is an error code on a host without a GPU too,
// allocates nothing, and issues kernels only, on the engine's stream: it may be captured into a graph.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <type_traits>

#include "../../include/apr.h"
#include "engine_view.h"
#include "linear_i8.hip.h"
#include "logprob.hip.h"
#include "rowquant.hip.h"

using namespace apr;

namespace {

constexpr size_t kMostRows = 0x7FFFFFFF, kMostStride = (size_t)1 << 40;
constexpr double kLeastScale = 1e-30, kMostScale = 1e30;   // what is divided by it or multiplied with it stays in the range of a float
constexpr unsigned kMostBlocks = 1u << 20;   // grids stride over their rows beyond that

size_t element_size(int dtype) { return dtype == APR_F32 ? 4 : 2; }
bool dtype_ok(int dtype) { return dtype == APR_F32 || dtype == APR_F16 || dtype == APR_BF16; }
bool aligned(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

int refuse(apr_engine *e, const char *entry, const char *why)
{
    char text[256];
    snprintf(text, sizeof text, "%s: bad argument (%s)", entry, why);
    return engine_fail(e, APR_ERR_INVALID, text);
}

// the launches of one entry: on the engine's GPU and stream, the caller's device back afterwards
template <class F>
int on_engine(apr_engine *e, const char *entry, F launch)
{
    EngineView v;
    char text[256];
    if (!engine_view(e, v)) {
        snprintf(text, sizeof text, "%s: null engine", entry);
        return engine_fail(e, APR_ERR_INVALID, text);
    }
    DeviceScope scope(v.device);
    if (!scope.ok()) return engine_fail(e, APR_ERR_DEVICE, "hipSetDevice failed");
    Launches go(v.stream);
    launch(v, go);
    if (go.error() == hipSuccess) return APR_OK;
    snprintf(text, sizeof text, "%s: %s", entry, hipGetErrorString(go.error()));
    return engine_fail(e, APR_ERR_DEVICE, text);
}

// calls f with a null pointer of the element type
template <class F>
void with_type(int dtype, F f)
{
    if (dtype == APR_F32) f((float *)nullptr);
    else if (dtype == APR_F16) f((f16_t *)nullptr);
    else f((bf16_t *)nullptr);
}
#define APR_TYPE_OF(p) std::remove_pointer_t<decltype(p)>

template <typename T>
void launch_logprobs(const EngineView &v, Launches &go, const LogprobArgs &a, const LogprobPlan &p)
{
    if (p.each) {
        const unsigned rows = 4 * a.rows;
        const dim3 grid((unsigned)std::min<unsigned long long>((a.n + rows - 1) / rows, kMostBlocks)), block(256);
        const auto launch = [&](auto kernel) { go(kernel, grid, block, 0, a); };
        switch (p.each) {   // scores a lane: what a row has beyond them is computed for nothing
        case 1: return launch(logprob_wave_kernel<T, 1>);
        case 2: return launch(logprob_wave_kernel<T, 2>);
        case 3: return launch(logprob_wave_kernel<T, 3>);
        case 4: return launch(logprob_wave_kernel<T, 4>);
        case 5: return launch(logprob_wave_kernel<T, 5>);
        case 6: return launch(logprob_wave_kernel<T, 6>);
        case 7: return launch(logprob_wave_kernel<T, 7>);
        case 8: return launch(logprob_wave_kernel<T, 8>);
        case 9: return launch(logprob_wave_kernel<T, 9>);
        case 10: return launch(logprob_wave_kernel<T, 10>);
        case 11: return launch(logprob_wave_kernel<T, 11>);
        case 12: return launch(logprob_wave_kernel<T, 12>);
        case 13: return launch(logprob_wave_kernel<T, 13>);
        case 14: return launch(logprob_wave_kernel<T, 14>);
        case 15: return launch(logprob_wave_kernel<T, 15>);
        default: return launch(logprob_wave_kernel<T, 16>);
        }
    }
    // few waves: one in a workgroup, so that they spread over the CUs
    const unsigned long long works = a.n * a.pieces;
    const unsigned waves = works < 4ull * v.n_cus ? 1 : 4;
    const dim3 grid((unsigned)std::min<unsigned long long>((works + waves - 1) / waves, kMostBlocks)), block(64 * waves);
    if (a.top) go(logprob_stream_kernel<T, true>, grid, block, 0, a);
    else go(logprob_stream_kernel<T, false>, grid, block, 0, a);
}

// The smallest group of lanes that holds a row's 16-byte units in registers
template <typename T>
void launch_rowquant(Launches &go, const RowQuantArgs &a)
{
    constexpr unsigned V = 16 / sizeof(T);
    const bool whole = aligned(a.x, 16) && a.ld % V == 0;
    const unsigned long long units = (a.k + (whole ? 0ull : V - 1) + V - 1) / V;   // a row may begin inside a unit
    const auto launch = [&](auto kernel, unsigned rows, unsigned threads) {
        go(kernel, dim3((unsigned)std::min<unsigned long long>((a.n + rows - 1) / rows, kMostBlocks)), dim3(threads), 0, a);
    };
    if (units <= 512) {
        switch ((units + 63) / 64) {
        case 1: return launch(rowquant_kernel<T, 1, 1>, 4, 256);
        case 2: return launch(rowquant_kernel<T, 1, 2>, 4, 256);
        case 3: return launch(rowquant_kernel<T, 1, 3>, 4, 256);
        case 4: return launch(rowquant_kernel<T, 1, 4>, 4, 256);
        case 5: return launch(rowquant_kernel<T, 1, 5>, 4, 256);
        case 6: return launch(rowquant_kernel<T, 1, 6>, 4, 256);
        case 7: return launch(rowquant_kernel<T, 1, 7>, 4, 256);
        default: return launch(rowquant_kernel<T, 1, 8>, 4, 256);
        }
    }
    if (units <= 2048) {
        switch ((units + 255) / 256) {
        case 3: return launch(rowquant_kernel<T, 4, 3>, 1, 256);
        case 4: return launch(rowquant_kernel<T, 4, 4>, 1, 256);
        case 5: return launch(rowquant_kernel<T, 4, 5>, 1, 256);
        case 6: return launch(rowquant_kernel<T, 4, 6>, 1, 256);
        case 7: return launch(rowquant_kernel<T, 4, 7>, 1, 256);
        default: return launch(rowquant_kernel<T, 4, 8>, 1, 256);
        }
    }
    launch(rowquant_kernel<T, 16, 8>, 1, 1024);
}

// Tiles of BM x BN outputs
template <typename T, int BM, int BN, int NBUF, int WM, int WN, bool DMA, int EVERY>
constexpr auto linear_tiles() { return linear_i8_tile_kernel<T, BM, BN, 128, NBUF, WM, WN, DMA, EVERY>; }
template <int BM, int BN, int NBUF>
constexpr int kLinearLds = (BM + BN) * 128 * NBUF;

template <typename T, int BM, int BN, int NBUF, int WM, int WN, bool DMA, int EVERY>
void launch_linear_tiles(Launches &go, const LinearI8Args &a)
{
    const unsigned tiles_m = (a.m + BM - 1) / BM, tiles_n = (a.n + BN - 1) / BN;
    go(linear_tiles<T, BM, BN, NBUF, WM, WN, DMA, EVERY>(), dim3(tiles_m * tiles_n), dim3(WM * WN * 64), kLinearLds<BM, BN, NBUF>, a, tiles_m, tiles_n);
}

template <typename T>
void launch_linear(const EngineView &v, Launches &go, const LinearI8Args &a)
{
    const unsigned long long few = (unsigned long long)(a.m <= 16 ? 1 : (a.m + 31) / 32) * ((a.n + 15) / 16);
    const dim3 few_grid((unsigned)std::min<unsigned long long>(few, kMostBlocks));
    const bool whole = aligned(a.x, 16) && aligned(a.w, 16) && a.ld_x % 16 == 0 && a.ld_w % 16 == 0;
    int variant = linear_variant(a.m, a.n, a.k, whole, v.n_cus);
    // the tiles address their rows with 32 bits, and a grid has less than 2^32 threads
    if (a.ld_x > (1u << 22) || a.ld_w > (1u << 22) || few > (1ull << 25)) variant = kLinearFew;
    if (variant == kLinearFew) {
        if (a.m <= 16 && whole) go(linear_i8_few_kernel<T, 8, 1, true>, few_grid, dim3(512), 0, a);
        else if (a.m <= 16) go(linear_i8_few_kernel<T, 8, 1, false>, few_grid, dim3(512), 0, a);
        else if (whole) go(linear_i8_few_kernel<T, 8, 2, true>, few_grid, dim3(512), 0, a);
        else go(linear_i8_few_kernel<T, 8, 2, false>, few_grid, dim3(512), 0, a);
    } else if (!whole) launch_linear_tiles<T, 128, 128, 2, 2, 2, false, 0>(go, a);
    else if (variant == kLinear256) launch_linear_tiles<T, 256, 256, 2, 2, 4, true, 1>(go, a);
    else if (variant == kLinear128) launch_linear_tiles<T, 128, 128, 2, 2, 2, true, 1>(go, a);
    else if (variant == kLinear64Deep) launch_linear_tiles<T, 64, 64, 4, 2, 2, true, 0>(go, a);
    else launch_linear_tiles<T, 64, 64, 2, 2, 2, true, 0>(go, a);
}

template <typename T>
bool allow_lds()
{
    return hipFuncSetAttribute(reinterpret_cast<const void *>(linear_tiles<T, 256, 256, 2, 2, 4, true, 1>()), hipFuncAttributeMaxDynamicSharedMemorySize,
                               kLinearLds<256, 256, 2>) == hipSuccess;
}

}  // namespace

namespace apr {

// More than 64 KiB of LDS has to be allowed, once on each device; it loads this file's kernels there, too, so that the first call may
// be one that is captured.
bool operators_prepare() noexcept { return allow_lds<float>() && allow_lds<f16_t>() && allow_lds<bf16_t>(); }

}  // namespace apr

extern "C" {

size_t apr_label_logprobs_workspace(size_t n, size_t n_labels, int top)
{
    if (n < 1 || n > kMostRows || n_labels < 1 || n_labels > kMostRows || top < 0 || top > APR_MAX_TOP) return 0;
    // Without lists a row may be cut in more pieces than with them, so the most for any `top` up to this one: a call that leaves the lists
    // out has enough with what its `top` asks for.
    size_t work = 0;
    for (int t = 0; t <= top; t++) work = std::max(work, logprob_plan(n, n_labels, t).work);
    return work;
}

int apr_label_logprobs_device(apr_engine *e, int dtype, const void *d_logits, size_t n, size_t n_labels, size_t ld, double scale,
                              const int32_t *d_target, int top, float *d_logprob, float *d_entropy, float *d_stat, int32_t *d_top_label,
                              float *d_top_logprob, void *d_work, size_t work_bytes)
{
    const char *me = "apr_label_logprobs_device";
    if (!dtype_ok(dtype)) return refuse(e, me, "dtype is APR_F32, APR_F16 or APR_BF16");
    if (n > kMostRows || n_labels < 1 || n_labels > kMostRows) return refuse(e, me, "1 <= n_labels < 2^31, n < 2^31");
    if (ld < n_labels || ld > kMostStride) return refuse(e, me, "ld is at least n_labels");
    if (!(scale >= kLeastScale && scale <= kMostScale)) return refuse(e, me, "1e-30 <= scale <= 1e30");
    if (top < 0 || top > APR_MAX_TOP) return refuse(e, me, "0 <= top <= APR_MAX_TOP");
    if (d_logprob && !d_target) return refuse(e, me, "d_logprob needs d_target");
    if (top == 0 && (d_top_label || d_top_logprob)) d_top_label = nullptr, d_top_logprob = nullptr;
    if (!d_top_label && !d_top_logprob) top = 0;
    if (!n) return on_engine(e, me, [](const EngineView &, Launches &) {});
    if (!d_logits) return refuse(e, me, "null d_logits");
    if (!aligned(d_logits, element_size(dtype)) || !aligned(d_target, 4) || !aligned(d_logprob, 4) || !aligned(d_entropy, 4) || !aligned(d_stat, 4) ||
        !aligned(d_top_label, 4) || !aligned(d_top_logprob, 4))
        return refuse(e, me, "pointers are aligned to their element");
    const LogprobPlan plan = logprob_plan(n, n_labels, top);
    if (plan.work && (!d_work || work_bytes < plan.work || !aligned(d_work, 16))) return refuse(e, me, "d_work holds apr_label_logprobs_workspace bytes, 16-aligned");
    LogprobArgs a;
    a.x = d_logits; a.n = n; a.ld = ld; a.n_labels = (unsigned)n_labels; a.scale = (float)scale; a.target = d_target; a.top = top;
    a.logprob = d_logprob; a.entropy = d_entropy; a.stat = d_stat; a.top_label = d_top_label; a.top_logprob = d_top_logprob;
    a.pieces = plan.pieces; a.piece_len = plan.piece_len;
    a.part_top = (unsigned long long *)d_work;
    a.part = (LogprobPart *)((char *)d_work + (plan.pieces > 1 ? n * plan.pieces * (size_t)top * 8 : 0));
    a.per_top = top ? (65536u + top - 1) / top : 0;
    return on_engine(e, me, [&](const EngineView &v, Launches &go) {
        // 32 waves fit a CU: a wave takes a row until the chip is full
        a.rows = (unsigned)std::max<size_t>(1, std::min<size_t>(kRows, n / (32 * (size_t)v.n_cus)));
        with_type(dtype, [&](auto *p) { launch_logprobs<APR_TYPE_OF(p)>(v, go, a, plan); });
        if (plan.pieces > 1) go(logprob_join_kernel, dim3((unsigned)std::min<size_t>(n, kMostBlocks)), dim3(64), 0, a, dtype);
    });
}

int apr_label_logprobs_backward_device(apr_engine *e, int dtype, const void *d_logits, size_t n, size_t n_labels, size_t ld, double scale,
                                       const int32_t *d_target, const float *d_stat, const float *d_entropy, const float *d_g_logprob,
                                       const float *d_g_entropy, void *d_grad, size_t ld_grad)
{
    const char *me = "apr_label_logprobs_backward_device";
    if (!dtype_ok(dtype)) return refuse(e, me, "dtype is APR_F32, APR_F16 or APR_BF16");
    if (n > kMostRows || n_labels < 1 || n_labels > kMostRows) return refuse(e, me, "1 <= n_labels < 2^31, n < 2^31");
    if (ld < n_labels || ld > kMostStride || ld_grad < n_labels || ld_grad > kMostStride) return refuse(e, me, "ld and ld_grad are at least n_labels");
    if (!(scale >= kLeastScale && scale <= kMostScale)) return refuse(e, me, "1e-30 <= scale <= 1e30");
    if (d_g_logprob && !d_target) return refuse(e, me, "d_g_logprob needs d_target");
    if (d_g_entropy && !d_entropy) return refuse(e, me, "d_g_entropy needs d_entropy");
    if (!n) return on_engine(e, me, [](const EngineView &, Launches &) {});
    if (!d_logits || !d_stat || !d_grad) return refuse(e, me, "null d_logits, d_stat or d_grad");
    if (!aligned(d_logits, element_size(dtype)) || !aligned(d_grad, element_size(dtype)) || !aligned(d_target, 4) || !aligned(d_stat, 4) ||
        !aligned(d_entropy, 4) || !aligned(d_g_logprob, 4) || !aligned(d_g_entropy, 4))
        return refuse(e, me, "pointers are aligned to their element");
    if (d_grad == d_logits && ld_grad != ld) return refuse(e, me, "a gradient in the place of the scores has their stride");
    LogprobGradArgs a;
    a.x = d_logits; a.grad = d_grad; a.n = n; a.ld = ld; a.ld_grad = ld_grad; a.n_labels = (unsigned)n_labels; a.scale = (float)scale;
    a.target = d_target; a.stat = d_stat; a.entropy = d_entropy; a.g_logprob = d_g_logprob; a.g_entropy = d_g_entropy;
    // A wave's piece of a row: 4 KiB, so that waves which run together are at neighbouring places of memory (8192 x 32000 bf16 takes 183 us,
    // whole rows 236, pieces of 8 KiB 192, of 2 KiB 194), and less while that leaves waves unused (1 x 131071 f32: 2.6 us against 3.7)
    constexpr size_t kGradWaves = 4096;
    const size_t units = std::max<size_t>(n_labels * element_size(dtype) / 16, 1), share = n >= kGradWaves ? units : n * units / kGradWaves;
    a.piece_units = (unsigned)std::min<size_t>(std::max<size_t>((share + 63) / 64 * 64, 64), 256);
    a.pieces = (unsigned)((units + a.piece_units - 1) / a.piece_units);
    return on_engine(e, me, [&](const EngineView &, Launches &go) {
        const dim3 grid((unsigned)std::min<size_t>((n * a.pieces + 3) / 4, kMostBlocks)), block(256);
        with_type(dtype, [&](auto *p) {
            if (a.g_entropy) go(logprob_grad_kernel<APR_TYPE_OF(p), true>, grid, block, 0, a);
            else go(logprob_grad_kernel<APR_TYPE_OF(p), false>, grid, block, 0, a);
        });
    });
}

int apr_quantize_rows_device(apr_engine *e, int dtype, const void *d_x, size_t n, size_t k, size_t ld, int8_t *d_q, size_t ld_q, float *d_scale)
{
    const char *me = "apr_quantize_rows_device";
    if (!dtype_ok(dtype)) return refuse(e, me, "dtype is APR_F32, APR_F16 or APR_BF16");
    if (n > kMostRows || k < 1 || k > kMostRows) return refuse(e, me, "1 <= k < 2^31, n < 2^31");
    if (ld < k || ld > kMostStride || ld_q < k || ld_q > kMostStride) return refuse(e, me, "ld and ld_q are at least k");
    if (!n) return on_engine(e, me, [](const EngineView &, Launches &) {});
    if (!d_x || !d_q || !d_scale) return refuse(e, me, "null pointer");
    if (!aligned(d_x, element_size(dtype)) || !aligned(d_scale, 4)) return refuse(e, me, "pointers are aligned to their element");
    RowQuantArgs a;
    a.x = d_x; a.q = d_q; a.scale = d_scale; a.n = n; a.ld = ld; a.ld_q = ld_q; a.k = (unsigned)k;
    return on_engine(e, me, [&](const EngineView &, Launches &go) {
        with_type(dtype, [&](auto *p) { launch_rowquant<APR_TYPE_OF(p)>(go, a); });
    });
}

int apr_linear_i8_device(apr_engine *e, const int8_t *d_x, size_t ld_x, const float *d_x_scale, const int8_t *d_w, size_t ld_w,
                         const float *d_w_scale, const float *d_bias, size_t m, size_t n, size_t k, int dtype, void *d_out, size_t ld_out)
{
    const char *me = "apr_linear_i8_device";
    if (!dtype_ok(dtype)) return refuse(e, me, "dtype is APR_F32, APR_F16 or APR_BF16");
    if (m > APR_LINEAR_MAX_ROWS || n > APR_LINEAR_MAX_ROWS) return refuse(e, me, "m and n are at most APR_LINEAR_MAX_ROWS");
    if (k < 1 || k > APR_LINEAR_MAX_K) return refuse(e, me, "1 <= k <= APR_LINEAR_MAX_K: the sum has 32 bits");
    if (ld_x < k || ld_x > kMostStride || ld_w < k || ld_w > kMostStride || ld_out < n || ld_out > kMostStride)
        return refuse(e, me, "ld_x and ld_w are at least k, ld_out at least n");
    if (!m || !n) return on_engine(e, me, [](const EngineView &, Launches &) {});
    if (!d_x || !d_w || !d_x_scale || !d_w_scale || !d_out) return refuse(e, me, "null pointer");
    if (!aligned(d_out, element_size(dtype)) || !aligned(d_x_scale, 4) || !aligned(d_w_scale, 4) || !aligned(d_bias, 4))
        return refuse(e, me, "pointers are aligned to their element");
    LinearI8Args a;
    a.x = d_x; a.w = d_w; a.x_scale = d_x_scale; a.w_scale = d_w_scale; a.bias = d_bias; a.out = d_out;
    a.ld_x = ld_x; a.ld_w = ld_w; a.ld_out = ld_out; a.m = (unsigned)m; a.n = (unsigned)n; a.k = (unsigned)k;
    return on_engine(e, me, [&](const EngineView &v, Launches &go) {
        with_type(dtype, [&](auto *p) { launch_linear<APR_TYPE_OF(p)>(v, go, a); });
    });
}

}  // extern "C"
