"""GPU: calls of the label operators that the documents allow, beside other users of the GPU and at the ends of the numbers."""
import ctypes as C

import numpy as np
import pytest
import torch

import label_oracle as oracle_l
from apr_amd import _capi, model, weights as W
from test_label_head_gpu import check, dev, near, rows, whole

pytestmark = pytest.mark.gpu

INVALID_DEVICE = 101          # hipErrorInvalidDevice


@pytest.fixture(scope="module")
def cnn(he_weights):
    e = model.Engine(W.pack_blob(he_weights, 4), 0, 4)
    yield e
    e.close()


class AnErrorBefore:
    """The thread's last HIP error is somebody else's: a device that there is not.  It has to be there still afterwards."""

    def __enter__(self):
        torch.cuda.synchronize()
        self.hip = _capi.lib()            # its dependencies' symbols are found through it
        self.hip.hipGetLastError()
        assert self.hip.hipSetDevice(10000) == INVALID_DEVICE and self.hip.hipPeekAtLastError() == INVALID_DEVICE

    def __exit__(self, *exc):
        left = self.hip.hipGetLastError()
        assert exc[0] is not None or left == INVALID_DEVICE


def test_an_error_of_somebody_else_is_not_the_operators(cnn):
    x, t = rows(70, 9000, torch.bfloat16, 1)
    E = lambda *s, d=torch.float32: torch.zeros(*s, device=dev(), dtype=d)   # noqa: E731
    stat, ent, lp, tl, grad, q, s, out = E(70, 2), E(70), E(70), E(70, 3, d=torch.int32), E(70, 9000, d=torch.bfloat16), E(70, 9000, d=torch.int8), E(70), E(70, 70)
    g = torch.full((70,), -1.0, device=dev())
    work = E(cnn.label_logprobs_workspace(70, 9000, 3), d=torch.uint8)
    with AnErrorBefore():
        cnn.label_logprobs_device(x, 70, 9000, d_target=t, top=3, d_logprob=lp, d_entropy=ent, d_stat=stat, d_top_label=tl, d_work=work)
        cnn.label_logprobs_backward_device(x, 70, 9000, t, stat, grad, d_g_logprob=g)
        cnn.quantize_rows_device(x, 70, 9000, q, s)
        cnn.linear_i8_device(q, s, q, s, 70, 70, 9000, out)
        cnn.label_logprobs_device(x[:0], 0, 9000, d_target=t[:0])
    cnn.sync()
    o = oracle_l.logprobs(x, 1.0, t, 3)
    near(lp, o["logprob"], o["tol_logprob"], "logprob")
    assert torch.equal(tl, o["top_label"]) and torch.equal(q, oracle_l.quantize(x)[0]) and torch.isfinite(out).all() and grad.abs().sum() > 0


def test_an_error_of_somebody_else_is_not_the_engines(cnn, clips):
    # the engine's other entry points: the same answers with it as without it
    pcm = clips["test_bigdog"]
    host = cnn.prepare_batch(pcm, 1, stride=192000)
    spec = torch.from_numpy(host).to(dev())
    f, z, hits = torch.zeros(1, 1024, device=dev()), torch.zeros(1, 4, device=dev()), torch.zeros(1, 4, device=dev(), dtype=torch.uint8)
    label, match = torch.tensor([2], device=dev(), dtype=torch.int32), torch.tensor([1], device=dev(), dtype=torch.uint8)
    taps = np.ones(2 * 4)
    up_in = np.arange(50, dtype=np.int16)

    def calls():
        f.zero_(), z.zero_(), hits.zero_()
        torch.cuda.synchronize()
        up_out = np.zeros(100, np.int16)
        with AnErrorBefore() if foreign else torch.no_grad():
            cnn.features_device(spec, 1, f)
            cnn.infer_device(spec, 1, z)
            cnn.bucket_hits_device(label, match, 1, 4, hits, 1)
            scored = [cnn.score(pcm, 1, 192000), cnn.classify(host), cnn.prepare(pcm)[0]]
            assert _capi.lib().apr_upsample(cnn._h, up_in.ctypes.data, 50, 2, taps.ctypes.data, 4, up_out.ctypes.data) == 0
        cnn.sync()
        return [f.cpu().numpy(), z.cpu().numpy(), hits.cpu().numpy(), up_out, scored[2]] + [v for s in scored[:2] for v in s.values()]

    foreign = False
    want = calls()
    foreign = True
    got = calls()
    assert all(np.array_equal(a, b) for a, b in zip(got, want)) and want[0].any() and want[1].any() and want[2].any()


@pytest.mark.parametrize("m,n,k", [(3, 70, 100), (10, 70, 100), (40, 70, 100), (520, 520, 1024), (1030, 1500, 129), (1500, 4100, 129), (2305, 3841, 129)])
def test_product_of_a_large_and_a_small_scale(cnn, m, n, k):
    # the whole sum times one scale may be beyond the largest float where the product with both is not; a scale of zero makes zeros
    x, w = whole(m, k, -(-k // 16) * 16, 1), whole(n, k, -(-k // 16) * 16, 2)
    x[1], w[1] = -128, -128
    x[m - 1] = 0
    one = torch.tensor([1.5, -0.75, 1.0, 1.25], device=dev())
    xs = one.repeat(m)[:m] * torch.exp2((torch.arange(m, device=dev()) % 5 - 2) * 60.0)      # 2^-120 to 2^120
    for dtype in (torch.float32, torch.bfloat16):
        for ws in (torch.full((n,), 2.0 ** -118, device=dev()), torch.exp2((torch.arange(n, device=dev()) % 5 - 2) * 60.0), torch.zeros(n, device=dev()),
                   torch.full((n,), 2.0 ** -140, device=dev())):
            out = torch.empty(m, n, device=dev(), dtype=dtype)
            b = torch.randn(n, generator=torch.Generator(device=dev()).manual_seed(1), device=dev())
            for bias in (None, b):
                torch.cuda.synchronize()
                cnn.linear_i8_device(x, xs, w, ws, m, n, k, out, d_bias=bias, ld_x=x.stride(0), ld_w=w.stride(0))
                cnn.sync()
                want, tol = oracle_l.linear(x, xs, w, ws, bias, dtype)
                near(out, want, tol, "product")


def test_the_chain_from_spectrograms_captured_and_replayed(cnn, clips):
    # features -> 8 bits -> scores -> log probabilities in one graph, on new spectrograms each time, with eager work between the replays
    n, c = 4, 300
    E = lambda *s, d=torch.float32: torch.zeros(*s, device=dev(), dtype=d)   # noqa: E731
    host = [cnn.prepare_batch(np.concatenate([clips[k] for k in order]), n, stride=192000)
            for order in (sorted(clips), sorted(clips)[::-1], sorted(clips)[2:] + sorted(clips)[:2])]
    gen = torch.Generator(device=dev()).manual_seed(1)
    w, ws = torch.randint(-127, 128, (c, 1024), generator=gen, device=dev(), dtype=torch.int16).to(torch.int8), torch.rand(c, generator=gen, device=dev()) * 0.01
    spec, f, q, qs, z, ent, tl = E(n, 128, 188), E(n, 1024), E(n, 1024, d=torch.int8), E(n), E(n, c), E(n), E(n, 5, d=torch.int32)
    outs = (f, q, qs, z, ent, tl)

    def calls():
        cnn.features_device(spec, n, f)
        cnn.quantize_rows_device(f, n, 1024, q, qs)
        cnn.linear_i8_device(q, qs, w, ws, n, c, 1024, z)
        cnn.label_logprobs_device(z, n, c, top=5, d_entropy=ent, d_top_label=tl)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=model.torch_stream(cnn)):
        calls()
    for k in range(4):
        spec.copy_(torch.from_numpy(host[k % 3]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        for t in outs:
            t.zero_()
        torch.cuda.synchronize()
        calls()
        cnn.sync()
        assert all(torch.equal(a, b) for a, b in zip(got, outs)) and f.any() and ent.all()


def test_a_tensor_of_the_engines_stream_dropped_while_its_call_waits(cnn):
    # made under the engine's stream and dropped behind the call: torch hands its memory out again in that stream's order
    n, c = 512, 3000
    x, t = rows(n, c, torch.float32, 1)
    x = x.contiguous()
    lp = torch.zeros(n, device=dev())
    torch.cuda.synchronize()
    with torch.cuda.stream(model.torch_stream(cnn)):
        y = x * 2.0
        torch.cuda._sleep(1_000_000)              # the call waits behind it
        cnn.label_logprobs_device(y, n, c, d_target=t, d_logprob=lp)
        place = y.data_ptr()
        del y
        other = torch.full_like(x, 7.0)
    cnn.sync()
    assert other.data_ptr() == place              # the same memory
    o = oracle_l.logprobs(x * 2.0, 1.0, t)
    near(lp, o["logprob"], o["tol_logprob"], "logprob")


@pytest.mark.parametrize("c", [1100, 1239, 4000, 20000])
@pytest.mark.parametrize("scale", [1.0, 7.0])
def test_a_best_score_behind_one_that_is_nearly_as_good(cnn, c, scale):
    # a first part of the row with a maximum of its own, then the row's, up to 8 nats higher: the sums stay relative to the largest score,
    # so that the entropy of an answer that is nearly sure is as exact as any
    n = 3000
    gen = torch.Generator(device=dev()).manual_seed(c)
    x = torch.rand(n, c, generator=gen, device=dev()) * 2 - 5
    x[:, 1000] = 0.0
    at = torch.randint(1060, c, (n,), generator=gen, device=dev())
    x.scatter_(1, at[:, None], 6.0 + 2 * torch.rand(n, 1, generator=gen, device=dev()))
    for dtype in (torch.float32, torch.bfloat16):
        check(cnn, (x / scale).to(dtype), at.int(), top=2, scale=scale)
