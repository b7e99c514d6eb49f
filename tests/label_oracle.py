"""The label operators in 64 bits, from their definitions, with the distance a 32-bit computation may be from them.

Tolerances count roundings, each of at most half a step: H = 2^-24 relative for a 32-bit result, eps / 2 of a narrower type.
A sum of C terms is made of partial sums of at most C / 256 + 32 additions one after the other (each worker's own, then a tree), so
its relative error is at most (C / 256 + 32) H on top of its terms' errors.  A term exp(d) is off by 2 |d| H (d and its product with
log2 e are rounded) + 4 H (the exponential itself, 2 steps), so the sum s of the terms by (2 E|d| + 4 + C / 256 + 32) H relative, where
E is the mean under p; log s by that absolutely, + 4 H |log s| (the logarithm, 2 steps).
"""
import torch

H = 2.0 ** -24
INF = float("inf")


def logprobs(x, scale=1.0, target=None, top=0):
    """x [n, C] of any type -> dict of float64 / int results and their absolute tolerances ``tol_*``."""
    x = x.double()
    n, c = x.shape
    bad = (torch.isnan(x) | (x == INF)).any(1)
    m = torch.where(torch.isnan(x), -INF, x).amax(1)
    empty = (m == -INF) & ~bad
    mm = torch.where(torch.isfinite(m), m, 0.0)
    d = scale * (torch.where(torch.isfinite(x), x, -INF) - mm[:, None])
    e = torch.exp(d)
    s = e.sum(1)
    d0 = torch.where(d > -INF, d, 0.0)
    log_s = torch.log(s)
    p = e / torch.where(s > 0, s, 1.0)[:, None]
    mean_d, mean_d2 = (p * d0.abs()).sum(1), (p * d0 * d0).sum(1)
    adds = c / 256 + 32
    ls0 = torch.where(empty | bad, 0.0, log_s)
    tol_s = H * (2 * mean_d + 4 + adds + 4 * ls0.abs())
    entropy = ls0 + mean_d
    tol_e = tol_s + H * (2 * mean_d2 + (4 + 2 * adds + 2 * mean_d) * mean_d + 2 * ls0.abs())
    nan = float("nan")
    out = dict(stat=torch.stack([torch.where(bad, nan, m), torch.where(bad, nan, torch.where(empty, -INF, log_s))], 1),
               entropy=torch.where(bad, nan, torch.where(empty, 0.0, entropy)), tol_stat=tol_s, tol_entropy=tol_e, bad=bad, empty=empty)
    if target is not None:
        t = target.long()
        has = (t >= 0) & (t < c)
        dt = d.gather(1, torch.where(has, t, 0)[:, None])[:, 0]
        lp = torch.where(bad, nan, torch.where(empty, -INF, dt - ls0))
        out["logprob"] = torch.where(has, lp, 0.0)
        out["tol_logprob"] = tol_s + H * (4 * torch.where(torch.isfinite(dt), dt, 0.0).abs() + ls0.abs())
    if top:
        k = min(top, c)
        score, place = torch.sort(torch.where(torch.isnan(x), -INF, x), dim=1, descending=True, stable=True)
        score, place = score[:, :k], place[:, :k]
        none = (score == -INF) | bad[:, None]
        lab = torch.full((n, top), -1, dtype=torch.int32, device=x.device)
        val = torch.full((n, top), -INF, dtype=torch.float64, device=x.device)
        lab[:, :k] = torch.where(none, -1, place).int()
        dk = d.gather(1, place)
        val[:, :k] = torch.where(none, -INF, dk - ls0[:, None])
        val[bad] = nan
        out["top_label"], out["top_logprob"] = lab, val
        dk0 = torch.zeros(n, top, dtype=torch.float64, device=x.device)
        dk0[:, :k] = torch.where(torch.isfinite(dk), dk, 0.0).abs()
        out["tol_top_logprob"] = tol_s[:, None] + H * (4 * dk0 + ls0.abs()[:, None])
    return out


def value(x, scale, target, g, h):
    """sum_i g_i logprob_i + h_i entropy_i in 64 bits: what the gradient is the gradient of."""
    o = logprobs(x, scale, target)
    return (g * o["logprob"]).sum() + (h * o["entropy"]).sum()


def gradient(x, scale, target, g=None, h=None):
    """-> (gradient [n, C] float64, its tolerance before the rounding to x's type), for the stat and entropy of 32 bits."""
    o = logprobs(x, scale, target)
    dtype, x = x.dtype, x.double()
    n, c = x.shape
    zero = torch.zeros(n, dtype=torch.float64, device=x.device)
    t = target.long() if target is not None else torch.full((n,), -1, device=x.device)
    has = (t >= 0) & (t < c) & ~o["empty"]
    g = torch.where(has, g.double(), 0.0) if g is not None else zero
    h = h.double() if h is not None else zero
    lp = scale * (x - o["stat"][:, :1]) - o["stat"][:, 1:]
    lp = torch.where(o["empty"][:, None], -INF, lp)
    p = torch.exp(lp)
    l0 = torch.where(lp > -INF, lp, 0.0)
    ent = o["entropy"][:, None]
    inner = g[:, None] + h[:, None] * (l0 + ent)
    grad = -p * inner
    grad[torch.arange(n, device=x.device)[has], t[has]] += g[has]
    nan = o["bad"][:, None]
    grad = torch.where(nan, float("nan"), scale * grad)
    # p: 2 |l| H + 4 H from the exponential, |l| H from l, the error of log s and of the largest score's product
    ls = o["stat"][:, 1:].abs()
    ls = torch.where(torch.isfinite(ls), ls, 0.0)
    rel = H * (4 * l0.abs() + 4 * ls + 8) + o["tol_stat"][:, None]
    size = g.abs()[:, None] + h.abs()[:, None] * (l0.abs() + ent.abs())
    tol = p * size * (rel + 4 * H) + p * h.abs()[:, None] * (o["tol_entropy"][:, None] + rel * 2) + 2 * H * g.abs()[:, None] * (p + 1e-30)
    at = torch.zeros_like(tol)
    at[torch.arange(n, device=x.device)[has], t[has]] = 4 * H * g.abs()[has]
    tol = scale * (tol + at) + 4 * H * grad.abs() + 1e-37
    tol = torch.where(torch.isfinite(tol), tol, 0.0)
    half = torch.finfo(dtype).eps / 2
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2     # half the step of its subnormals
    return grad, tol * (1 + half) + half * grad.abs().nan_to_num(0.0) + least


def quantize(x):
    """-> (q int8, scale float32): the quotient 127 x / max|x| of 32-bit numbers is exact enough in 64 bits (a quotient that is not
    halfway between whole numbers is 2^-33 away from there, one that is comes out exactly)."""
    x = x.float()
    a = x.abs().nan_to_num(INF, INF, INF).amax(1)
    none = (a < 2.0 ** -119) | (a == INF)
    safe = torch.where(none, 1.0, a)
    q = torch.round(x.double() * 127.0 / safe.double()[:, None])
    q = torch.where(none[:, None], 0.0, q).to(torch.int8)
    scale = torch.where(a == INF, float("nan"), torch.where(none, 0.0, (a.double() / 127.0).float()))   # torch divides a 32-bit tensor by its reciprocal
    return q, scale


def linear(x, xs, w, ws, bias, dtype):
    """-> (out float64, tolerance): float(sum) (H), two products (H each), the sum with the bias (H), and the type's rounding."""
    acc = x.double() @ w.double().t().contiguous()
    prod = acc * xs.double()[:, None] * ws.double()[None, :]
    out = prod if bias is None else prod + bias.double()
    half = torch.finfo(dtype).eps / 2
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    tol = 4 * H * prod.abs() + 2 * H * out.abs() + 1e-37
    return out, tol * (1 + half) + (half if dtype != torch.float32 else 0.0) * out.abs() + least
