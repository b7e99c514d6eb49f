"""CPU: calls of the label operators that the documents allow, up to the point where they need a GPU (argument checks come before the
engine is looked at), and what their Python side refuses."""
import numpy as np
import pytest
import torch

from apr_amd import _capi, model

P = 0x1000        # a non-null, aligned address that no call here touches


def logprobs(n, c, top, work_bytes, lists=True):
    """the error text of a call of those sizes without an engine"""
    tops = (P, P) if lists else (None, None)
    rc = _capi.lib().apr_label_logprobs_device(None, 0, P, n, c, c, 1.0, P, top, P, P, P, *tops, P, work_bytes)
    assert rc == _capi.ERR_INVALID
    return _capi.lib().apr_last_error(None).decode()


LENGTHS = (1, 64, 1000, 1025, 4096, 4097, 5000, 131071, 149505, 300000, 749000, 790000, 1050000, 2885000, 3000000, 6300000, 2**31 - 1)


def test_scratch_for_the_lists_is_enough_without_them():
    # any output may be NULL: a call that leaves both lists out has the scratch of the `top` it names
    for n in (1, 2, 3, 7, 48, 64, 700, 6144):
        for c in LENGTHS:
            for top in (0, 1, 2, 7, 8, 20, 32):
                need = _capi.lib().apr_label_logprobs_workspace(n, c, top)
                for lists in (True, False):
                    why = logprobs(n, c, top, need, lists)
                    assert why.endswith("null engine"), (n, c, top, lists, why)


def test_scratch_does_not_fall_with_the_lists_length():
    for n in (1, 2, 5, 60, 1000):
        for c in LENGTHS:
            sizes = [_capi.lib().apr_label_logprobs_workspace(n, c, top) for top in range(_capi.MAX_TOP + 1)]
            assert sizes == sorted(sizes), (n, c, sizes)


class Recorder:
    """An engine's memory and sizes without a GPU"""
    num_features = 1

    def __init__(self):
        self.sizes, self._fin = {}, type("Gone", (), {"alive": False})

    def device_alloc(self, nbytes):
        self.sizes[len(self.sizes) + 1] = nbytes
        return len(self.sizes)

    def label_logprobs_workspace(self, n, c, top):
        return _capi.lib().apr_label_logprobs_workspace(n, c, top)

    def device_upload(self, p, a):
        pass

    device_free = quantize_rows_device = sync = lambda self, *a, **k: None


@pytest.mark.parametrize("labels,max_rows", [(2885000, 1), (3100000, 2), (800000, 3), (5000, 64), (527, 8)])
def test_a_heads_scratch_is_enough_for_every_pass(labels, max_rows):
    e = Recorder()
    head = model.LabelHead(e, np.zeros((labels, 1), np.float32), max_rows=max_rows)
    have = e.sizes[head._work] if head._work else 0
    assert have == head._work_bytes
    for n in range(1, max_rows + 1):
        for top in (0, 1, 5, 8, 20, 32):
            assert logprobs(n, labels, top, have, lists=top > 0).endswith("null engine"), (n, top)


def no_engine():
    """An engine's Python side without a GPU: a call that passes its checks ends as 'null engine'"""
    e = object.__new__(model.Engine)
    e._lib, e.device, e._h = _capi.lib(), 0, None
    return e


class OnGpu:
    """What the checks ask of a tensor on GPU 0"""
    dtype = None

    def __init__(self, count):
        self.count = count

    def is_contiguous(self):
        return True

    def get_device(self):
        return 0

    def numel(self):
        return self.count

    def element_size(self):
        return 1

    def data_ptr(self):
        return P


def test_scratch_of_a_size_that_is_none_is_refused():
    # a negative size must not come round to a large one
    e = no_engine()
    need = e.label_logprobs_workspace(1, 131071, 20)
    lists = dict(d_top_label=P, d_top_logprob=P, top=20)
    for work, size in ((P, -1), (P, -(2**63)), (OnGpu(16), -1), (OnGpu(need), -need)):
        with pytest.raises(ValueError, match="work_bytes"):
            e.label_logprobs_device(P, 1, 131071, d_work=work, work_bytes=size, **lists)
    for work, size in ((P, need - 1), (P, 0), (P, None), (OnGpu(need - 1), None), (OnGpu(need - 1), need), (OnGpu(need), need - 1), (None, None)):
        with pytest.raises(model.AprError, match="apr_label_logprobs_workspace"):
            e.label_logprobs_device(P, 1, 131071, d_work=work, work_bytes=size, **lists)
    for work, size in ((P, need), (OnGpu(need), None), (OnGpu(need), need + 5)):
        with pytest.raises(model.AprError, match="null engine"):
            e.label_logprobs_device(P, 1, 131071, d_work=work, work_bytes=size, **lists)


def test_the_stream_of_a_closed_engine_is_refused():
    for cached in (True, False):
        e = no_engine()
        e._fin = lambda: None
        if cached:
            e._torch_stream = object()       # what an earlier torch_stream(e) kept
            assert model.torch_stream(e) is e._torch_stream
        e.close()
        with pytest.raises(model.AprError, match="closed") as why:
            model.torch_stream(e)
        assert why.value.code == _capi.ERR_INVALID
        e.close()                            # a second time: nothing


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.float16])
def test_a_head_takes_the_parameters_of_a_linear(dtype):
    # tensors that train, as torch.nn.Linear keeps them, of any type, and rows that are not one after the other
    linear = torch.nn.Linear(1, 5).to(dtype)
    assert linear.weight.requires_grad
    wide = torch.randn(1, 5, dtype=dtype).t()
    for weight in (linear.weight, wide, linear.weight.detach().float().numpy()):
        e, up = Recorder(), []
        e.device_upload = lambda p, a: up.append(a)
        head = model.LabelHead(e, weight, linear.bias)
        want = torch.as_tensor(weight).detach().float().numpy()
        assert head.labels == 5 and all(a.dtype == np.float32 and a.flags.c_contiguous for a in up)
        assert np.array_equal(up[0], linear.bias.detach().float().numpy()) and np.array_equal(up[1], want)
    with pytest.raises(ValueError, match="weight"):
        model.LabelHead(Recorder(), linear.weight[:, :0])
    with pytest.raises(ValueError, match="bias"):
        model.LabelHead(Recorder(), linear.weight, linear.bias[:3])
