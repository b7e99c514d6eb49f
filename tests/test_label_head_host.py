"""CPU: refusals of the label operators (argument checks come before the engine is looked at, so they need no GPU), the checks of
their Python side, and the oracle's gradient against differences."""
import ctypes as C
import weakref

import numpy as np
import pytest
import torch

import label_oracle as oracle_l
from apr_amd import _capi, model

P = 0x1000        # a non-null, aligned address that no refused call touches
OK = dict(
    logprobs=dict(e=None, dtype=0, x=P, n=4, c=10, ld=10, scale=1.0, target=P, top=3, lp=P, ent=P, stat=P, tl=P, tp=P, work=P, nwork=1 << 20),
    backward=dict(e=None, dtype=0, x=P, n=4, c=10, ld=10, scale=1.0, target=P, stat=P, ent=P, g=P, h=P, grad=2 * P, ldg=10),
    quantize=dict(e=None, dtype=0, x=P, n=4, k=10, ld=10, q=P, ldq=10, s=P),
    linear=dict(e=None, x=P, ldx=32, xs=P, w=P, ldw=32, ws=P, b=P, m=4, n=5, k=20, dtype=0, out=P, ldo=5),
)
ENTRY = dict(logprobs="apr_label_logprobs_device", backward="apr_label_logprobs_backward_device", quantize="apr_quantize_rows_device",
             linear="apr_linear_i8_device")


def call(op, **change):
    args = dict(OK[op], **change)
    rc = getattr(_capi.lib(), ENTRY[op])(*args.values())
    return rc, (_capi.lib().apr_last_error(None) or b"").decode()


@pytest.mark.parametrize("op", list(ENTRY))
def test_good_arguments_reach_the_engine(op):
    rc, why = call(op)
    assert rc == _capi.ERR_INVALID and why == ENTRY[op] + ": null engine"


@pytest.mark.parametrize("op,change", [
    ("logprobs", dict(dtype=3)), ("logprobs", dict(dtype=-1)), ("logprobs", dict(c=0)), ("logprobs", dict(c=1 << 31, ld=1 << 31)),
    ("logprobs", dict(n=1 << 31)), ("logprobs", dict(ld=9)), ("logprobs", dict(ld=1 << 41)), ("logprobs", dict(scale=0.0)),
    ("logprobs", dict(scale=-1.0)), ("logprobs", dict(scale=float("nan"))), ("logprobs", dict(scale=float("inf"))),
    ("logprobs", dict(scale=1e-60)), ("logprobs", dict(scale=1e39)), ("logprobs", dict(scale=0.9e-30)), ("logprobs", dict(scale=1.1e30)), ("logprobs", dict(top=-1)), ("logprobs", dict(top=33)),
    ("logprobs", dict(target=None)), ("logprobs", dict(x=None)), ("logprobs", dict(x=P + 2)), ("logprobs", dict(dtype=1, x=P + 1)),
    ("logprobs", dict(target=P + 2)), ("logprobs", dict(lp=P + 1)), ("logprobs", dict(ent=P + 2)), ("logprobs", dict(stat=P + 2)),
    ("logprobs", dict(tl=P + 3)), ("logprobs", dict(tp=P + 2)),
    ("backward", dict(dtype=7)), ("backward", dict(c=0)), ("backward", dict(n=1 << 31)), ("backward", dict(ld=9)), ("backward", dict(ldg=9)),
    ("backward", dict(scale=0.0)), ("backward", dict(scale=float("nan"))), ("backward", dict(scale=1e-31)), ("backward", dict(scale=1e31)), ("backward", dict(target=None)), ("backward", dict(ent=None)),
    ("backward", dict(x=None)), ("backward", dict(stat=None)), ("backward", dict(grad=None)), ("backward", dict(grad=P + 2)),
    ("backward", dict(grad=P, ldg=11)), ("backward", dict(g=P + 1)), ("backward", dict(h=P + 2)),
    ("quantize", dict(dtype=3)), ("quantize", dict(k=0)), ("quantize", dict(ld=9)), ("quantize", dict(ldq=9)), ("quantize", dict(x=None)),
    ("quantize", dict(q=None)), ("quantize", dict(s=None)), ("quantize", dict(x=P + 1)), ("quantize", dict(s=P + 2)), ("quantize", dict(n=1 << 31)),
    ("linear", dict(dtype=3)), ("linear", dict(k=0)), ("linear", dict(k=131072, ldx=131072, ldw=131072)), ("linear", dict(ldx=19)),
    ("linear", dict(ldw=19)), ("linear", dict(ldo=4)), ("linear", dict(m=(1 << 24) + 1)), ("linear", dict(n=(1 << 24) + 1, ldo=1 << 25)),
    ("linear", dict(x=None)), ("linear", dict(w=None)), ("linear", dict(xs=None)), ("linear", dict(ws=None)), ("linear", dict(out=None)),
    ("linear", dict(out=P + 2)), ("linear", dict(xs=P + 1)), ("linear", dict(ws=P + 2)), ("linear", dict(b=P + 2)),
])
def test_bad_arguments_are_refused(op, change):
    rc, why = call(op, **change)
    assert rc == _capi.ERR_INVALID and why.startswith(ENTRY[op] + ": bad argument"), why


def test_a_workspace_that_is_needed_is_asked_for():
    L = _capi.lib()
    for n, c, top in ((1, 131071, 20), (64, 131072, 20), (1, 2_000_000, 0), (7, 200_000, 32)):
        need = L.apr_label_logprobs_workspace(n, c, top)
        if need:
            for bad in (dict(nwork=need - 1), dict(work=None), dict(work=P + 4)):
                rc, why = call("logprobs", n=n, c=c, ld=c, top=top, nwork=bad.pop("nwork", need), **bad)
                assert rc == _capi.ERR_INVALID and "apr_label_logprobs_workspace" in why
        rc, why = call("logprobs", n=n, c=c, ld=c, top=top, nwork=need)
        assert why.endswith("null engine")
    assert L.apr_label_logprobs_workspace(0, 10, 3) == 0


def test_features_of_no_engine():
    L = _capi.lib()
    assert L.apr_engine_num_features(None) == 0 and L.apr_features_device(None, P, 1, P) == _capi.ERR_INVALID


def test_python_side_refuses_host_and_foreign_tensors():
    e = object.__new__(model.Engine)
    e.device = 0
    with pytest.raises(TypeError):
        e._matrix("d_x", np.zeros((2, 3), np.float32), 2, 3, None)
    with pytest.raises(ValueError, match="on cpu"):
        e._matrix("d_x", torch.zeros(2, 3), 2, 3, None)
    with pytest.raises(ValueError, match="element type"):
        e._matrix("d_x", torch.zeros(2, 3, dtype=torch.float64), 2, 3, None)
    with pytest.raises(ValueError, match="element type"):
        e._matrix("d_q", torch.zeros(2, 3), 2, 3, None, None, (model._I8,))
    with pytest.raises(TypeError):
        e._vector("d_scale", np.zeros(2, np.float32), 2)
    with pytest.raises(ValueError, match="float32"):
        e._vector("d_scale", torch.zeros(2, dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="on cpu"):
        e._vector("d_scale", torch.zeros(2), 2)
    assert e._matrix("d_x", 4096, 2, 3, None) == (4096, 3, _capi.F32) and e._matrix("d_x", 4096, 2, 3, 8, _capi.BF16) == (4096, 8, _capi.BF16)
    assert e._vector("d_scale", None, 2) == 0


def test_a_closed_engine_or_head_refuses():
    e = object.__new__(model.Engine)
    e._lib, e.device, e._h, e._fin = _capi.lib(), 0, 1, lambda: None      # a handle that must not be looked at
    e.close()
    for call_ in (lambda: e.quantize_rows_device(P, 2, 3, P, P), lambda: e.linear_i8_device(P, P, P, P, 1, 2, 3, P),
                  lambda: e.label_logprobs_device(P, 2, 3), lambda: e.label_logprobs_backward_device(P, 2, 3, P, P, P),
                  lambda: e.features_device(P, 1, P)):
        with pytest.raises(model.AprError):
            call_()
    assert e.num_features == 0
    with pytest.raises(ValueError, match="contiguous float32"):
        e.features_device(torch.zeros(1, 128, 188), 2, P)
    h = object.__new__(model.LabelHead)
    h.labels, h._fin = 5, weakref.finalize(h, int)
    spec = np.zeros((4, 128, 188), np.float32)
    assert h._arguments(spec, np.array([0, 4, 5, -100]))[1].tolist() == [0, 4, -1, -1]
    assert h._arguments(spec, np.array([0, 4, 2**32, -2**32 + 1]))[1].tolist() == [0, 4, -1, -1]
    assert h._arguments(spec, np.array([0, 4, 2**63 + 1, 1], np.uint64))[1].tolist() == [0, 4, -1, 1]
    assert h._arguments(spec[:0], [])[1].dtype == np.int32
    for bad in ([0, 1], [0.0, 1.0, 2.0, 3.0], [[0, 1, 2, 3]]):
        with pytest.raises(ValueError, match="whole numbers"):
            h._arguments(spec, bad)
    h.close()
    with pytest.raises(ValueError, match="closed"):
        h.score(spec)
    with pytest.raises(ValueError, match="closed"):
        h.loss(spec, [0, 0, 0, 0])


@pytest.mark.parametrize("scale", [1.0, 0.37])
def test_oracle_gradient_against_differences(scale):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(4, 7, generator=g, dtype=torch.float64) * 2
    x[1, 3] = -float("inf")
    x[3] = -float("inf")
    target = torch.tensor([2, 0, -1, 4], dtype=torch.int32)
    a, b = torch.randn(4, generator=g, dtype=torch.float64), torch.randn(4, generator=g, dtype=torch.float64)
    a_used = torch.where(torch.tensor([True, True, True, False]), a, 0.0)      # -inf * a: the empty row has no gradient
    grad, _ = oracle_l.gradient(x, scale, target, a, b)
    step = 1e-6
    for i in range(4):
        for j in range(7):
            if x[i, j] == -float("inf"):
                assert grad[i, j] == 0.0
                continue
            up, down = x.clone(), x.clone()
            up[i, j] += step
            down[i, j] -= step
            rows = [0, 1, 2]
            diff = (oracle_l.value(up[rows], scale, target[rows], a_used[rows], b[rows])
                    - oracle_l.value(down[rows], scale, target[rows], a_used[rows], b[rows])) / (2 * step)
            assert abs(diff - grad[i, j]) < 1e-8      # a third derivative of order 1 times step^2, and 1e-16 / step of the two values
