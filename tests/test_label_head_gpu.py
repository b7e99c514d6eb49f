"""GPU: the operators behind a label head through the C ABI against the 64-bit oracle, at the sizes, masks and strides where they
can go wrong; then the chain of them on an engine's features.  The tolerances are derived in label_oracle.py."""
import numpy as np
import pytest
import torch

import label_oracle as oracle_l
import oracle
from apr_amd import _capi, model, weights as W
from apr_amd._capi import AprError

pytestmark = pytest.mark.gpu

INF = float("inf")
TYPES = [torch.float32, torch.float16, torch.bfloat16]
GUARD = -77.0            # what outputs hold behind the last row: has to stay


@pytest.fixture(scope="module")
def eng():
    e = model.Engine(None, 0, 1)
    yield e
    e.close()


def dev():
    return torch.device("cuda", 0)


def rows(n, c, dtype, seed, masked=0.0, ld=None, spread=3.0):
    """[n, c] scores inside rows of ld elements, at an address that is aligned to nothing but the type"""
    ld = c if ld is None else ld
    g = torch.Generator(device=dev()).manual_seed(seed)
    store = torch.full((n * ld + 1,), 1e4, device=dev(), dtype=dtype)
    x = store[1:].view(n, ld)[:, :c] if ld != c else store[1:].view(n, c)
    v = torch.randn(n, c, generator=g, device=dev()) * spread
    t = torch.randint(0, c, (n,), generator=g, device=dev(), dtype=torch.int32)
    v.scatter_add_(1, t.long()[:, None], torch.full((n, 1), 6.0, device=dev()))
    if masked:
        v.masked_fill_(torch.rand(n, c, generator=g, device=dev()) < masked, -INF)
    x.copy_(v)
    return x, t


def run(eng, x, target=None, top=0, scale=1.0):
    n, c = x.shape
    out = dict(logprob=torch.full((n + 1,), GUARD, device=dev()), entropy=torch.full((n + 1,), GUARD, device=dev()),
               stat=torch.full((n + 1, 2), GUARD, device=dev()), top_label=torch.full((n + 1, max(top, 1)), -77, device=dev(), dtype=torch.int32),
               top_logprob=torch.full((n + 1, max(top, 1)), GUARD, device=dev()))
    need = eng.label_logprobs_workspace(n, c, top)
    work = torch.full((need + 64,), 0xAB, device=dev(), dtype=torch.uint8) if need else None
    torch.cuda.synchronize()
    eng.label_logprobs_device(x, n, c, d_target=target, top=top, d_logprob=out["logprob"] if target is not None else None,
                              d_entropy=out["entropy"], d_stat=out["stat"], d_top_label=out["top_label"],
                              d_top_logprob=out["top_logprob"], d_work=work, scale=scale, work_bytes=need)
    eng.sync()
    if need:
        assert (work[need:] == 0xAB).all()
    for k, v in out.items():
        if k.startswith("top") and not top or k == "logprob" and target is None:
            assert (v == GUARD).all()
        else:
            assert (v[n:] == GUARD).all(), k
    if not top:
        out.pop("top_label"), out.pop("top_logprob")
    if target is None:
        out.pop("logprob")
    return {k: v[:n] for k, v in out.items()}


def near(got, want, tol, what):
    # a result beyond the type's largest value, (2 - eps / 2) * 2^emax at the least, rounds to infinity: 2.5 * the lowest float is one
    most = torch.finfo(got.dtype)
    want = torch.where(want.abs() >= most.max * (1 + most.eps / 4), torch.sign(want) * INF, want)
    got = got.double()
    special = ~torch.isfinite(want)
    same = torch.where(torch.isnan(want), torch.isnan(got), got == want)
    assert same[special].all(), (what, "special values")
    far = ((got - want).abs() - tol)[~special]
    assert far.numel() == 0 or far.max() <= 0, (what, float(far.max()), far.numel())


def check(eng, x, target=None, top=0, scale=1.0):
    want, got = oracle_l.logprobs(x, np.float32(scale).item(), target, top), run(eng, x, target, top, scale)
    near(got["stat"][:, 0], want["stat"][:, 0], torch.zeros_like(want["tol_stat"]), "largest")
    near(got["stat"][:, 1], want["stat"][:, 1], want["tol_stat"], "log s")
    near(got["entropy"], want["entropy"], want["tol_entropy"], "entropy")
    if target is not None:
        near(got["logprob"], want["logprob"], want["tol_logprob"], "logprob")
    if top:
        assert torch.equal(got["top_label"], want["top_label"])
        near(got["top_logprob"], want["top_logprob"], want["tol_top_logprob"], "top_logprob")
    return got


# one label to a long list; the borders of every power of two that a kernel may cut rows at
SIZES = [1, 2, 3, 4, 15, 16, 17, 63, 64, 65, 127, 255, 257, 511, 512, 513, 527, 1000, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097,
         8191, 8192, 8193, 16383, 16384, 16385, 32767, 32768, 32769, 50257, 65536, 65537, 131071, 200003]


@pytest.mark.parametrize("c", SIZES)
def test_logprobs_over_list_lengths(eng, c):
    for i, dtype in enumerate(TYPES):
        n = (5, 1, 3)[i]
        x, t = rows(n, c, dtype, 100 + i, masked=(0.0, 0.3, 0.0)[i])
        check(eng, x, t, top=(5, 32, 1)[i], scale=(1.0, 1.0, 0.7)[i])


@pytest.mark.parametrize("n", [1, 2, 4, 7, 64, 255, 256, 257, 1000, 4099])
@pytest.mark.parametrize("c,dtype", [(4, torch.float32), (64, torch.float32), (527, torch.bfloat16), (5003, torch.float16), (40000, torch.bfloat16)])
def test_logprobs_over_row_counts(eng, n, c, dtype):
    if n * c > 5e7:
        n = max(1, int(5e7 // c))
    x, t = rows(n, c, dtype, n, masked=0.1, ld=c + 13)
    check(eng, x, t, top=3)


@pytest.mark.parametrize("n,c,top", [(16385, 700, 5), (20001, 64, 32), (24577, 527, 0), (35999, 100, 1), (36003, 17, 3), (140002, 3, 2), (140003, 40, 31)])
def test_logprobs_of_many_rows(eng, n, c, top):
    # several rows to a wave, the last wave's rows cut short; some without labels, some of NaN, between the others
    for dtype in (torch.float32, torch.bfloat16):
        x, t = rows(n, c, dtype, n, masked=0.05, ld=c + 5)
        x[5::37] = -INF
        x[n - 1] = -INF
        x[7::41, c // 2] = float("nan")
        x[9::43] = 0.5
        t[::11], t[3::13] = -1, c
        check(eng, x, t, top=top)


@pytest.mark.parametrize("top", [0, 1, 2, 3, 7, 8, 16, 31, 32])
@pytest.mark.parametrize("c", [5, 64, 700, 9000, 100000])
def test_logprobs_top_counts(eng, top, c):
    x, t = rows(6, c, torch.bfloat16, top)      # bf16: many equal scores
    check(eng, x, t, top=top)


@pytest.mark.parametrize("c", [3, 64, 300, 3000, 30000, 90000])
@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_rows_that_are_hard(eng, c, dtype):
    lowest = torch.finfo(dtype).min
    x, t = rows(16, c, dtype, 9, ld=c + 3)
    x[0] = -INF                                  # every label ruled out
    x[1] = lowest                                # the type's lowest value everywhere: all alike
    x[2] = -INF
    x[2, c - 1] = 2.0                            # one label left, the last
    x[3] = 0.0                                   # all equal
    x[4, c // 2] = float("nan")
    x[5, 0] = INF
    x[6] = torch.arange(c, device=dev()).to(dtype)          # the best at the end
    x[7] = -torch.arange(c, device=dev()).float().to(dtype)  # the best at the start
    x[8, :] = lowest
    x[8, c // 3] = 1.0                           # lowest as a mask
    x[9] = torch.finfo(dtype).max / 2            # large, alike
    x[10, :] = -0.0
    x[10, c - 1] = 0.0                           # equal scores
    x[11] = -INF
    x[11, : min(c, 3)] = -5.0                    # fewer labels than places
    x[12, c - 1] = -INF
    x[13] *= 100
    t[14], t[15] = -1, c                         # no label
    t[2], t[12] = 0, c - 1                       # labels that are ruled out
    got = check(eng, x, t, top=8)
    assert got["logprob"][14] == 0 and got["logprob"][15] == 0 and got["top_label"][0].tolist() == [-1] * 8
    check(eng, x, t, top=32, scale=2.5)
    check(eng, x, None, top=2)
    check(eng, x, t, top=0, scale=0.01)


def test_logprobs_with_many_equal_scores(eng):
    # every score equal in every list length: the lowest labels win, whatever a kernel keeps as candidates
    for c in (40, 1000, 5000, 33000, 140000):
        x = torch.full((3, c), 1.5, device=dev(), dtype=torch.bfloat16)
        x[1, ::2] = 1.25
        x[2, : c // 2] = -INF
        got = check(eng, x, torch.tensor([0, 1, c - 1], device=dev(), dtype=torch.int32), top=32)
        assert got["top_label"][0].tolist() == list(range(32)) and got["top_label"][1].tolist() == (list(range(1, c, 2)) + list(range(0, c, 2)))[:32]


@pytest.mark.parametrize("scale", [1e-30, 1e-10, 1e10, 1e30])
@pytest.mark.parametrize("c", [60, 3000])
def test_logprobs_at_the_ends_of_the_scale(eng, scale, c):
    # scores of the size that the scale wants, one row with a label ruled out, one with the range's largest spread
    g = torch.Generator(device=dev()).manual_seed(2)
    x = torch.randn(4, c, generator=g, device=dev()) * 3.0 / scale
    x[1, c // 2] = -INF
    x[2, 0], x[2, 1:] = 3e38, -3e38
    t = torch.randint(1, c, (4,), generator=g, device=dev(), dtype=torch.int32)
    check(eng, x, t, top=3, scale=scale)
    gradient_case(eng, x, t, scale, torch.full((4,), 1e-3, device=dev()), None)


def test_logprobs_outputs_are_each_optional(eng):
    x, t = rows(5, 777, torch.float32, 3)
    want = run(eng, x, t, 4)
    for keep in ("logprob", "entropy", "stat", "top_label", "top_logprob"):
        out = {"d_" + keep: torch.full_like(want[keep].contiguous(), -1)}
        torch.cuda.synchronize()
        eng.label_logprobs_device(x, 5, 777, d_target=t, top=4, **out)
        eng.sync()
        assert torch.equal(out["d_" + keep], want[keep]), keep
    eng.label_logprobs_device(x, 5, 777, d_target=t)                     # none at all
    eng.label_logprobs_device(x[:0], 0, 777, d_target=t[:0], top=3)      # no rows
    eng.sync()


def test_logprobs_repeat_bit_for_bit(eng):
    for n, c in ((1, 150000), (70, 60000), (300, 512)):
        x, t = rows(n, c, torch.bfloat16, 4)
        a, b = run(eng, x, t, 20), run(eng, x, t, 20)
        assert all(torch.equal(a[k], b[k]) for k in a)


def test_offsets_beyond_32_bits(eng):
    # three rows 1.5 * 2^31 elements apart (bf16): the last one starts beyond 2^32 elements; only the rows are touched
    c, ld = 5000, 3 << 30
    store = torch.empty(2 * ld + c, device=dev(), dtype=torch.bfloat16)
    x = torch.as_strided(store, (3, c), (ld, 1))
    src, t = rows(3, c, torch.bfloat16, 8)
    x.copy_(src)
    assert torch.equal(x, src)
    got = check(eng, x, t, 5)    # not src's bits: a row that begins elsewhere in a 16-byte unit is summed in another order
    stat, ent = got["stat"].contiguous(), got["entropy"].contiguous()
    g = torch.full((3,), -0.5, device=dev())
    a, b = torch.empty(3, c, device=dev(), dtype=torch.bfloat16), x
    torch.cuda.synchronize()
    eng.label_logprobs_backward_device(src, 3, c, t, stat, a, d_g_logprob=g)
    eng.label_logprobs_backward_device(x, 3, c, t, stat, b, d_g_logprob=g)            # in place, too
    eng.sync()
    assert torch.equal(a, b)
    q, s = torch.empty(3, c, device=dev(), dtype=torch.int8), torch.empty(3, device=dev())
    torch.cuda.synchronize()
    eng.quantize_rows_device(x, 3, c, q, s)
    eng.sync()
    wq, wsc = oracle_l.quantize(x)
    assert torch.equal(q, wq) and torch.equal(s, wsc)


def gradient_case(eng, x, t, scale=1.0, g=None, h=None, in_place=False, ld_grad=None):
    n, c = x.shape
    o = oracle_l.logprobs(x, np.float32(scale).item(), t)
    stat, ent = o["stat"].float().contiguous(), o["entropy"].float().contiguous()
    want, tol = oracle_l.gradient(x, np.float32(scale).item(), t, g, h)
    ld = c if ld_grad is None else ld_grad
    store = torch.full((n, ld), GUARD, device=dev(), dtype=x.dtype)
    grad = x if in_place else store[:, :c]
    torch.cuda.synchronize()
    eng.label_logprobs_backward_device(x, n, c, t, stat, grad, d_g_logprob=g, d_entropy=ent if h is not None else None, d_g_entropy=h, scale=scale)
    eng.sync()
    near(grad, want, tol, "gradient")
    assert (store[:, c:] == GUARD).all()


@pytest.mark.parametrize("c", [1, 2, 7, 8, 9, 63, 64, 65, 255, 256, 257, 527, 1023, 2048, 2049, 5000, 32768, 50257, 131073])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_over_list_lengths(eng, c, dtype):
    n = 9
    x, t = rows(n, c, dtype, c, masked=0.2, ld=c + (c % 3))
    gen = torch.Generator(device=dev()).manual_seed(1)
    g, h = torch.randn(n, generator=gen, device=dev()), torch.randn(n, generator=gen, device=dev())
    t[3], t[4] = -1, c
    gradient_case(eng, x, t, 1.0, g, h, ld_grad=c + 5)
    gradient_case(eng, x, t, 0.6, g, None)
    gradient_case(eng, x, None, 1.7, None, h)
    gradient_case(eng, x, t, 1.0, g, h, in_place=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [5, 700, 40000])
def test_gradient_rows_that_are_hard(eng, c, dtype):
    lowest = torch.finfo(dtype).min
    x, t = rows(10, c, dtype, 2)
    x[0] = -INF
    x[1] = lowest
    x[2] = -INF
    x[2, c - 1] = 1.0
    x[3, 1] = float("nan")
    x[4, 0] = INF
    x[5, :] = lowest
    x[5, 2] = 0.0
    x[6, t[6].long()] = -INF
    x[7] *= 50
    g, h = torch.full((10,), -0.25, device=dev()), torch.full((10,), 0.1, device=dev())
    gradient_case(eng, x, t, 1.0, g, h)
    gradient_case(eng, x, t, 3.0, g, None)


def test_gradient_of_many_short_rows(eng):
    x, t = rows(70001, 4, torch.float32, 6)
    g = torch.full((70001,), -1.0, device=dev())
    gradient_case(eng, x, t, 1.0, g, None)
    gradient_case(eng, x, t, 1.0, g, g)


@pytest.mark.parametrize("k", [1, 2, 7, 8, 15, 16, 17, 64, 100, 255, 256, 1000, 1024, 2047, 2048, 4095, 4097, 8191, 8192, 8193, 16384, 40000])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_rows(eng, k, dtype):
    n, ld, ld_q = 13, k + (k % 5), -(-k // 16) * 16
    x, _ = rows(n, k, dtype, k, ld=ld)
    x[0] = 0.0
    x[1, k // 2] = float("nan")
    x[2, k - 1] = -INF
    x[3] = 0.0
    x[3, k - 1] = -3.0                                       # the largest magnitude is negative
    x[4] = (torch.arange(k, device=dev()) % 255 - 127).to(dtype)
    x[5] = ((torch.arange(k, device=dev()) % 255 - 127).float() + 0.5).to(dtype)       # halves: quotients exactly between two whole numbers
    x[5, 0] = 127.0
    x[6] = 1e-30 if dtype != torch.float16 else 2.0 ** -24
    x[7] = 2.0 ** -119 if dtype != torch.float16 else 0.0
    x[8] = 2.0 ** -120 if dtype != torch.float16 else 0.0
    x[9] = torch.finfo(dtype).max
    x[10] = -0.0
    store = torch.full((n + 1, ld_q), 99, device=dev(), dtype=torch.int8)
    scale = torch.full((n + 1,), GUARD, device=dev())
    torch.cuda.synchronize()
    eng.quantize_rows_device(x, n, k, store, scale, ld_q=ld_q)
    eng.sync()
    q, s = oracle_l.quantize(x)
    assert torch.equal(store[:n, :k], q)
    assert torch.equal(torch.isnan(scale[:n]), torch.isnan(s)) and torch.equal(scale[:n].nan_to_num(0.0), s.nan_to_num(0.0))
    assert (store[n] == 99).all() and (store[:n, k:] == 99).all() and scale[n] == GUARD


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_next_to_halves_in_every_row_length(eng, dtype):
    # rows of every number of 16-byte units a lane, filled with the type's numbers on both sides of (j + 1/2) a / 127
    unit = 16 // torch.empty(0, dtype=dtype).element_size()
    for units in (50, 100, 170, 230, 300, 370, 420, 500, 700, 1000, 1200, 1500, 1700, 2000, 2300):
        k, n = units * unit - 3, 6
        g = torch.Generator(device=dev()).manual_seed(units)
        a = torch.exp2(torch.tensor([0.0, 0.3, -7.7, 9.1, -13.4, 3.9], device=dev(), dtype=torch.float64)).to(dtype)
        half = torch.randint(-127, 127, (n, k), generator=g, device=dev()).double() + 0.5
        v = (half * a.double()[:, None] / 127).to(dtype)
        bits = {2: torch.int16, 4: torch.int32}[v.element_size()]
        v = (v.view(bits) + torch.randint(-1, 2, (n, k), generator=g, device=dev()).to(bits)).view(dtype)
        v[:, k // 3] = a
        q, s = torch.empty(n, k, device=dev(), dtype=torch.int8), torch.empty(n, device=dev())
        torch.cuda.synchronize()
        eng.quantize_rows_device(v, n, k, q, s)
        eng.sync()
        wq, ws = oracle_l.quantize(v)
        assert torch.equal(q, wq) and torch.equal(s, ws), units


def test_quantize_many_rows_and_odd_strides(eng):
    for n, k, ld_q in ((40000, 33, 33), (3001, 1024, 1024), (2000, 527, 529)):
        x, _ = rows(n, k, torch.float32, n)
        q, s = torch.empty(n, ld_q, device=dev(), dtype=torch.int8), torch.empty(n, device=dev())
        torch.cuda.synchronize()
        eng.quantize_rows_device(x, n, k, q, s)
        eng.sync()
        wq, ws = oracle_l.quantize(x)
        assert torch.equal(q[:, :k], wq) and torch.equal(s, ws)


def whole(rows_, k, ld, seed, shift=0, most=127):
    """[rows, k] int8 inside rows of ld bytes that hold 77 elsewhere, at 16-byte aligned addresses + shift"""
    g = torch.Generator(device=dev()).manual_seed(seed)
    store = torch.full((rows_ * ld + 16,), 77, device=dev(), dtype=torch.int8)
    v = store[shift : shift + rows_ * ld].view(rows_, ld)[:, :k]
    v.copy_(torch.randint(-most - 1, most + 1, (rows_, k), generator=g, device=dev(), dtype=torch.int16).to(torch.int8))
    return v


def linear_case(eng, m, n, k, dtype, bias=True, ld_x=None, ld_w=None, shift=0, ld_out=None, x=None, w=None):
    pad = lambda v: -(-v // 16) * 16   # noqa: E731
    x = whole(m, k, ld_x or pad(k), 1, shift) if x is None else x
    w = whole(n, k, ld_w or pad(k), 2, shift) if w is None else w
    g = torch.Generator(device=dev()).manual_seed(3)
    xs, ws = (torch.rand(r, generator=g, device=dev()) * 0.01 + 1e-4 for r in (m, n))
    b = torch.randn(n, generator=g, device=dev()) if bias else None
    ld_out = n if ld_out is None else ld_out
    out = torch.full((m + 1, ld_out), GUARD, device=dev(), dtype=dtype)
    torch.cuda.synchronize()
    eng.linear_i8_device(x, xs, w, ws, m, n, k, out[:m], d_bias=b, ld_x=ld_x or pad(k), ld_w=ld_w or pad(k))
    eng.sync()
    want, tol = oracle_l.linear(x, xs, w, ws, b, dtype)
    near(out[:m, :n], want, tol, "product")
    assert (out[m] == GUARD).all() and (out[:m, n:] == GUARD).all()


@pytest.mark.parametrize("m", [1, 2, 3, 4, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 511, 513])
def test_linear_over_row_counts(eng, m):
    for i, dtype in enumerate(TYPES):
        linear_case(eng, m, (64, 527, 260)[i], (1024, 300, 2048)[i], dtype, bias=i != 1)


@pytest.mark.parametrize("n", [1, 2, 5, 16, 31, 64, 65, 127, 128, 130, 255, 256, 257, 1000, 4096, 5001])
def test_linear_over_label_counts(eng, n):
    linear_case(eng, 7, n, 1024, torch.float32)
    linear_case(eng, 300, n, 640, torch.bfloat16, bias=False)


@pytest.mark.parametrize("k", [1, 2, 3, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 191, 255, 256, 257, 383, 384, 385, 512, 1000, 1024, 4000, 8191, 16385])
def test_linear_over_depths(eng, k):
    linear_case(eng, 5, 70, k, torch.float32)
    linear_case(eng, 70, 300, k, torch.float16, bias=False)
    linear_case(eng, 520, 270, k, torch.bfloat16)


@pytest.mark.parametrize("m,n,k", [(1, 33, 100), (20, 70, 333), (130, 300, 1025), (600, 520, 257)])
def test_linear_any_alignment_and_stride(eng, m, n, k):
    linear_case(eng, m, n, k, torch.float32, ld_x=k, ld_w=k + 3)
    linear_case(eng, m, n, k, torch.float32, shift=5)
    linear_case(eng, m, n, k, torch.bfloat16, shift=8, ld_out=n + 7)
    linear_case(eng, m, n, k, torch.float16, ld_x=1040, ld_w=2048, ld_out=n + 1)


def test_linear_largest_sums_are_exact(eng):
    # k = 131071 of -128 * -128: 2^31 - 2^14, the largest sum that 32 bits hold; and the same sum with opposite signs
    k = _capi_max_k()
    for m in (1, 40, 300):
        x = torch.full((m, k + 1), -128, device=dev(), dtype=torch.int8)[:, :k]
        w = torch.full((3, k + 1), -128, device=dev(), dtype=torch.int8)[:, :k]
        w[1] = 127
        linear_case(eng, m, 3, k, torch.float32, bias=False, ld_x=k + 1, ld_w=k + 1, x=x, w=w)


def _capi_max_k():
    return 131071


def test_linear_marked_rows_and_overflow(eng):
    m, n, k = 4, 6, 64
    x, w = whole(m, k, 64, 1), whole(n, k, 64, 2)
    xs, ws = torch.tensor([1.0, float("nan"), 0.0, 1e6], device=dev()), torch.full((n,), 1.0, device=dev())
    out = torch.empty(m, n, device=dev(), dtype=torch.float16)
    torch.cuda.synchronize()
    eng.linear_i8_device(x, xs, w, ws, m, n, k, out)
    eng.sync()
    acc = x.double() @ w.double().t()
    assert torch.isnan(out[1]).all() and (out[2] == 0).all()
    assert torch.equal(torch.isinf(out[3]), (acc[3] * 1e6).abs() >= 65520) and torch.equal(torch.sign(out[3].double()), torch.sign(acc[3]))


def test_chain_quantize_linear_logprobs_backward(eng):
    # features -> 8 bits -> scores -> log probabilities -> gradient, queued without a wait between, against the chain of oracles
    m, n, k = 517, 1000, 1024
    g = torch.Generator(device=dev()).manual_seed(11)
    f, wt = torch.rand(m, k, generator=g, device=dev()), torch.randn(n, k, generator=g, device=dev()) * 0.1
    t = torch.randint(0, n, (m,), generator=g, device=dev(), dtype=torch.int32)
    E = lambda *s, d=torch.float32: torch.empty(*s, device=dev(), dtype=d)   # noqa: E731
    xq, xs, wq, ws = E(m, k, d=torch.int8), E(m), E(n, k, d=torch.int8), E(n)
    z, lp, ent, stat, tl, tp, dz = E(m, n), E(m), E(m), E(m, 2), E(m, 5, d=torch.int32), E(m, 5), E(m, n)
    gl = torch.full((m,), -1.0 / m, device=dev())
    need = eng.label_logprobs_workspace(m, n, 5)
    work = torch.empty(max(need, 16), device=dev(), dtype=torch.uint8)
    torch.cuda.synchronize()
    eng.quantize_rows_device(wt, n, k, wq, ws)
    eng.quantize_rows_device(f, m, k, xq, xs)
    eng.linear_i8_device(xq, xs, wq, ws, m, n, k, z)
    eng.label_logprobs_device(z, m, n, d_target=t, top=5, d_logprob=lp, d_entropy=ent, d_stat=stat, d_top_label=tl, d_top_logprob=tp, d_work=work)
    eng.label_logprobs_backward_device(z, m, n, t, stat, dz, d_g_logprob=gl)
    eng.sync()
    (oq, os_), (owq, ows) = oracle_l.quantize(f), oracle_l.quantize(wt)
    assert torch.equal(xq, oq) and torch.equal(wq, owq)
    want, tol = oracle_l.linear(oq, os_, owq, ows, None, torch.float32)
    near(z, want, tol, "product")
    o = oracle_l.logprobs(z, 1.0, t, 5)
    near(lp, o["logprob"], o["tol_logprob"], "logprob")
    assert torch.equal(tl, o["top_label"])
    grad, gtol = oracle_l.gradient(z, 1.0, t, gl)
    near(dz, grad, gtol + 4 * o["tol_stat"][:, None] * grad.abs(), "gradient")      # stat is the kernel's own here


def test_captured_and_replayed(eng):
    # two graphs with workspaces of their own, replayed several times with eager work between, on new inputs each time
    stream = model.torch_stream(eng)
    parts = []
    for n, c in ((2, 140000), (300, 527)):
        x, t = rows(n, c, torch.bfloat16, n)
        E = lambda *s, d=torch.float32: torch.zeros(*s, device=dev(), dtype=d)   # noqa: E731
        b = dict(lp=E(n), ent=E(n), stat=E(n, 2), tl=E(n, 9, d=torch.int32), tp=E(n, 9), grad=torch.zeros(n, c, device=dev(), dtype=x.dtype),
                 q=E(n, c, d=torch.int8), s=E(n), out=E(n, n), g=torch.full((n,), -1.0, device=dev()),
                 work=torch.zeros(max(16, eng.label_logprobs_workspace(n, c, 9)), device=dev(), dtype=torch.uint8))

        def calls(x=x, t=t, b=b, n=n, c=c):
            eng.label_logprobs_device(x, n, c, d_target=t, top=9, d_logprob=b["lp"], d_entropy=b["ent"], d_stat=b["stat"], d_top_label=b["tl"],
                                      d_top_logprob=b["tp"], d_work=b["work"])
            eng.label_logprobs_backward_device(x, n, c, t, b["stat"], b["grad"], d_g_logprob=b["g"])
            eng.quantize_rows_device(x, n, c, b["q"], b["s"])
            if c <= _capi_max_k():
                eng.linear_i8_device(b["q"], b["s"], b["q"], b["s"], n, n, c, b["out"])
        torch.cuda.synchronize()
        calls()
        eng.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            calls()
        parts.append((x, b, calls, graph))
    for k in range(4):
        for x, b, _, graph in parts:
            x.copy_(torch.randn(x.shape, device=dev(), generator=torch.Generator(device=dev()).manual_seed(k)) * 4)
        torch.cuda.synchronize()
        for _, b, _, graph in parts:
            graph.replay()
        torch.cuda.synchronize()
        for x, b, calls, graph in parts:
            got = {q: v.clone() for q, v in b.items() if q != "work"}
            for q in ("lp", "ent", "tl", "grad", "q"):
                b[q].zero_()
            torch.cuda.synchronize()
            calls()
            eng.sync()
            assert all(torch.equal(got[q], b[q]) for q in got), k


def test_in_order_with_torch_on_the_engines_stream(eng):
    # torch work under torch_stream(engine) needs no wait before or after the engine's calls, and the current device stays
    stream = model.torch_stream(eng)
    x, t = rows(4096, 5000, torch.float32, 1)
    E = lambda *s: torch.empty(*s, device=dev())   # noqa: E731
    lp, twice = E(4096), E(4096)
    torch.cuda.synchronize()
    before = torch.cuda.current_device()
    with torch.cuda.stream(stream):
        y = x * 2.0
        eng.label_logprobs_device(y, 4096, 5000, d_target=t, d_logprob=lp)
        torch.mul(lp, 2.0, out=twice)
    eng.sync()
    assert torch.cuda.current_device() == before
    o = oracle_l.logprobs(x * 2.0, 1.0, t)
    near(twice / 2, o["logprob"], o["tol_logprob"], "logprob")


def test_refused_calls_leave_the_engine_working(eng):
    x, t = rows(3, 100, torch.float32, 1)
    with pytest.raises(AprError) as ei:
        eng.label_logprobs_device(x, 3, 100, d_target=t, top=33, d_top_label=torch.zeros(99, device=dev(), dtype=torch.int32))
    assert ei.value.code == _capi.ERR_INVALID and "APR_MAX_TOP" in str(ei.value)
    with pytest.raises(ValueError):
        eng.label_logprobs_device(x, 4, 100)
    with pytest.raises(ValueError):
        eng.label_logprobs_device(x.t(), 100, 3)
    with pytest.raises(ValueError):
        eng.label_logprobs_device(x, 3, 100, d_target=t, d_logprob=torch.zeros(2, device=dev()))
    c, n = 140000, 1
    need = eng.label_logprobs_workspace(n, c, 3)
    if need:
        big, _ = rows(n, c, torch.float32, 2)
        with pytest.raises(AprError, match="workspace"):
            eng.label_logprobs_device(big, n, c, d_entropy=torch.zeros(1, device=dev()), top=3, d_top_label=torch.zeros(3, device=dev(), dtype=torch.int32))
    check(eng, x, t, top=3)


def test_label_head_on_the_engines_features(he_weights, clips):
    # a head that is the CNN's own Linear: its answers agree with the CNN's to the error of 8 bits; then its loss and gradient
    C = 4
    full = model.Engine(W.pack_blob(he_weights, C), 0, 4)
    assert full.num_features == 1024
    with pytest.raises(AprError):
        model.Engine(None, 0, 1).features_device(torch.zeros(1, 128, 188, device=dev()), 1, torch.zeros(1, 1024, device=dev()))
    sd = W.to_state_dict(he_weights, C)
    wt, b = (np.asarray(sd[k], np.float32) for k in ("classifier.3.weight", "classifier.3.bias"))
    pcm = np.concatenate([clips[c] for c in sorted(clips)])
    spec = full.prepare_batch(pcm, 4, stride=192000)
    spec = np.concatenate([spec, spec[::-1], spec[:2]])                     # ten windows: three passes of four
    cnn = full.classify(spec)
    f = torch.empty(10, 1024, device=dev())
    d_spec = torch.from_numpy(spec).to(dev())
    torch.cuda.synchronize()
    full.features_device(d_spec, 10, f)
    full.sync()
    logits = f.double().cpu().numpy() @ wt.T.astype(np.float64) + b
    assert np.abs(logits - cnn["logits"]).max() <= 2e-4                     # the tolerance of the engine's logits
    want = oracle.cnn_forward(he_weights, C, spec[:4])
    assert np.abs(logits[:4] - want).max() <= 2e-4

    head = model.LabelHead(full, wt, b, max_rows=4)
    target = np.array([0, 1, 2, 3, 3, 2, 1, -1, 4, 0], np.int32)
    got = head.score(spec, target, top=3)
    # the head's logits from the definition: both operands rounded to 8 bits
    (fq, fs), (wq, ws) = oracle_l.quantize(f), oracle_l.quantize(torch.from_numpy(wt).to(dev()))
    z, tol = oracle_l.linear(fq, fs, wq, ws, torch.from_numpy(b).to(dev()), torch.float32)
    o = oracle_l.logprobs(z, 1.0, torch.from_numpy(target).to(dev()), 3)
    slack = 4 * tol.amax(1)
    near(torch.from_numpy(got["logprob"]).to(dev()), o["logprob"], o["tol_logprob"] + slack, "logprob")
    near(torch.from_numpy(got["entropy"]).to(dev()), o["entropy"], o["tol_entropy"] + slack * (2 + o["entropy"]), "entropy")
    assert np.array_equal(got["top_label"], o["top_label"].cpu().numpy())
    near(torch.from_numpy(got["top_logprob"]).to(dev()), o["top_logprob"], o["tol_top_logprob"] + slack[:, None], "top_logprob")
    assert got["logprob"][7] == 0 and got["logprob"][8] == 0
    # 8 bits: half a step of each operand, summed over the products, bounds a logit's distance from the CNN's own
    worst = 0.5 * fs.double()[:, None] * torch.from_numpy(np.abs(wt).sum(1)).to(dev()) + 0.5 * ws.double() * (f.double().abs().sum(1, keepdim=True) + 512 * fs.double()[:, None])
    assert (np.abs(z.cpu().numpy() - cnn["logits"]) <= worst.cpu().numpy() + 4e-4).all()

    r = head.loss(spec, target)
    n_used = int(((target >= 0) & (target < C)).sum())
    assert abs(r["loss"] + float(o["logprob"].sum()) / n_used) <= float((o["tol_logprob"] + slack).sum()) / n_used
    g = torch.full((10,), -1.0 / n_used, device=dev())
    grad, gtol = oracle_l.gradient(z.float(), 1.0, torch.from_numpy(target).to(dev()), g)
    near(torch.from_numpy(r["d_logits"]).to(dev()), grad, gtol + 8 * slack[:, None] / n_used + 4 * o["tol_stat"][:, None] / n_used, "d_logits")
    assert np.array_equal(r["features"], f.cpu().numpy())
    assert head.score(spec, top=0)["top_label"].shape == (10, 0) and head.score(spec[:0], target[:0])["entropy"].shape == (0,)
    again = head.score(spec, target, top=3)
    assert all(np.array_equal(again[k], got[k]) for k in got)
    assert np.array_equal(full.classify(spec)["logits"], cnn["logits"])     # the CNN's own head is as it was
    with pytest.raises(ValueError):
        model.LabelHead(full, wt[:, :5])
    with pytest.raises(ValueError):
        head.score(spec, target[:3])
    with pytest.raises(ValueError):
        head.score(spec, top=33)
    head.close()
    full.close()
