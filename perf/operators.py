"""The operators behind a label head, as cases that can be measured: the log probabilities of given labels with entropy and top
alternatives, their gradient, rows quantised to 8 bits, and the matrix product of 8-bit rows.

``run`` computes them in their plain form (torch, 32 bits) where ``own`` is false and through ``apr_amd.model.Engine`` where it is
true; ``exact`` gives the same outputs from the definitions in 64 bits.  The sizes are the engine's own (64 classes at most in a
CNN's own head, 1024 features, 256 live streams, the 35 999 windows of ten hours) and generic ones for long label lists.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MOST_LOGITS = 8192 * 32000          # values of the largest drawn table of logits
MOST_PRODUCT = 16384 * 8192 * 8192  # multiplications of the largest drawn product

_engine = None


def engine():
    """A front-end-only engine: the operators need its GPU and stream, no CNN."""
    global _engine
    if _engine is None:
        from apr_amd import model
        _engine = model.Engine(None, torch.cuda.current_device(), 1)
    return _engine


def listed():
    return [
        # one tick of 256 live streams scored by a CNN with as many classes as a model may have: launch latency
        dict(name="logprobs 256x64", op="logprobs", n=256, labels=64, dtype="f32", top=5, masked=0.0),
        # the 35 999 windows of a ten-hour sweep against an audio-tagging list of 527 labels
        dict(name="logprobs 35999x527", op="logprobs", n=35999, labels=527, dtype="bf16", top=5, masked=0.0),
        # one row over a long list, half of it ruled out beforehand
        dict(name="logprobs 1x131071", op="logprobs", n=1, labels=131071, dtype="f32", top=20, masked=0.5),
        # a served batch, one row for each request
        dict(name="logprobs 64x131072", op="logprobs", n=64, labels=131072, dtype="bf16", top=20, masked=0.0),
        # a training batch: label and entropy, no alternatives
        dict(name="logprobs 8192x32000", op="logprobs", n=8192, labels=32000, dtype="bf16", top=0, masked=0.0),
        # the gradient of that batch
        dict(name="gradient 8192x32000", op="gradient", n=8192, labels=32000, dtype="bf16", masked=0.0),
        # an odd list in 32 bits
        dict(name="gradient 509x50257", op="gradient", n=509, labels=50257, dtype="f32", masked=0.1),
        # the features of ten hours
        dict(name="quantize 35999x1024", op="quantize", n=35999, k=1024, dtype="f32"),
        # activations of a wide layer
        dict(name="quantize 4096x8191", op="quantize", n=4096, k=8191, dtype="bf16"),
        # one row through a wide layer: the weights' bytes
        dict(name="linear 1x8192x8192", op="linear", m=1, n=8192, k=8192, dtype="bf16", bias=False),
        # the features of a tick of 256 live streams against 527 labels
        dict(name="linear 256x527x1024", op="linear", m=256, n=527, k=1024, dtype="f32", bias=True),
        # a whole pass of windows through a wide layer: the matrix rate
        dict(name="linear 16384x8192x8192", op="linear", m=16384, n=8192, k=8192, dtype="bf16", bias=False),
    ]


def _size(rng, low, high):
    """A whole number, spread over the logarithm of its range."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["logprobs", "gradient", "quantize", "linear"])
    if op in ("logprobs", "gradient"):
        labels = _size(rng, 2, 200000)
        n = _size(rng, 1, min(36000, MOST_LOGITS // labels))
        case = dict(op=op, n=n, labels=labels, dtype=rng.choice(["f32", "f16", "bf16"]), masked=rng.choice([0.0, 0.1, 0.5]))
        if op == "logprobs":
            case["top"] = rng.choice([0, 1, 2, 5, 10, 20, 32])
        return case
    if op == "quantize":
        k = _size(rng, 16, 16384)
        return dict(op=op, n=_size(rng, 1, min(36000, MOST_LOGITS // k)), k=k, dtype=rng.choice(["f32", "f16", "bf16"]))
    n, k = _size(rng, 4, 16384), _size(rng, 16, 16384)
    return dict(op=op, m=_size(rng, 1, min(36000, MOST_PRODUCT // (n * k))), n=n, k=k, dtype=rng.choice(["f32", "f16", "bf16"]),
                bias=rng.random() < 0.5)


def _logits(case, g, device):
    """Scores of rows of which most are sure of one label, with a share of the labels ruled out (-inf)."""
    n, c = case["n"], case["labels"]
    x = torch.empty(n, c, device=device, dtype=torch.float32).normal_(0.0, 2.5, generator=g)
    target = torch.randint(0, c, (n,), device=device, generator=g, dtype=torch.int32)
    sure = torch.rand(n, device=device, generator=g) < 0.8
    at = target.long()[:, None]
    x.scatter_add_(1, at, torch.where(sure, 12.0, 0.0)[:, None])
    if case["masked"]:
        out = torch.rand(n, c, device=device, generator=g) < case["masked"]
        out.scatter_(1, at, False)
        x.masked_fill_(out, -math.inf)
    return x.to(DTYPES[case["dtype"]]), target


def _stats(x):
    """(largest score, logarithm of the sum of the exponentials relative to it, entropy) of rows of scores in 32 bits."""
    m = x.amax(1)
    d = (x - m[:, None]).clamp_(min=-200.0)
    e = torch.exp(d)
    s = e.sum(1)
    log_s = torch.log(s)
    return m, log_s, log_s - (e * d).sum(1) / s


def _padded(n):
    """Rows of 8-bit values lie 16 bytes apart, or a multiple of that."""
    return -(-n // 16) * 16


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    state = dict(case=case)
    if case["op"] == "logprobs":
        n, top = case["n"], case["top"]
        state["x"], state["target"] = _logits(case, g, device)
        state["logprob"] = torch.empty(n, device=device)
        state["entropy"] = torch.empty(n, device=device)
        state["stat"] = torch.empty(n, 2, device=device)
        state["top_label"] = torch.empty(n, top, device=device, dtype=torch.int32)
        state["top_logprob"] = torch.empty(n, top, device=device)
        state["work"] = torch.empty(64 << 20, device=device, dtype=torch.uint8)   # this program's scratch
    elif case["op"] == "gradient":
        n = case["n"]
        state["x"], state["target"] = _logits(case, g, device)
        m, log_s, entropy = _stats(state["x"].float())
        state["stat"], state["entropy"] = torch.stack([m, log_s], 1), entropy
        state["g_logprob"] = torch.empty(n, device=device).normal_(-1.0, 0.25, generator=g)
        state["g_entropy"] = torch.empty(n, device=device).normal_(0.0, 0.1, generator=g)
        state["grad"] = torch.empty_like(state["x"])
    elif case["op"] == "quantize":
        n, k = case["n"], case["k"]
        spread = torch.rand(n, 1, device=device, generator=g) * 4.0 + 0.01
        x = torch.empty(n, k, device=device).normal_(0.0, 1.0, generator=g) * spread
        state["x"] = x.to(DTYPES[case["dtype"]])
        state["q"] = torch.empty(n, _padded(k), device=device, dtype=torch.int8)
        state["scale"] = torch.empty(n, device=device)
        state["values"] = torch.empty(n, k, device=device)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        for name, rows in (("x", m), ("w", n)):
            q = torch.zeros(rows, _padded(k), device=device, dtype=torch.int8)
            q[:, :k] = torch.empty(rows, k, device=device).normal_(0.0, 36.0, generator=g).round_().clamp_(-127, 127).to(torch.int8)
            state[name] = q
            state[name + "_scale"] = torch.rand(rows, device=device, generator=g) * 0.02 + 0.001
        state["bias"] = torch.empty(n, device=device).normal_(0.0, 1.0, generator=g) if case["bias"] else None
        state["out"] = torch.empty(m, n, device=device, dtype=DTYPES[case["dtype"]])
    return state


def _own_logprobs(s):
    c = s["case"]
    engine().label_logprobs_device(s["x"], c["n"], c["labels"], d_target=s["target"], top=c["top"], d_logprob=s["logprob"],
                                   d_entropy=s["entropy"], d_stat=s["stat"], d_top_label=s["top_label"],
                                   d_top_logprob=s["top_logprob"], d_work=s["work"])
    return dict(logprob=s["logprob"], entropy=s["entropy"], top_label=s["top_label"], top_logprob=s["top_logprob"])


def _plain_logprobs(s):
    c = s["case"]
    x = s["x"].float()
    m, log_s, entropy = _stats(x)
    at = s["target"].long()[:, None]
    logprob = x.gather(1, at)[:, 0] - m - log_s
    k = min(c["top"], c["labels"])
    label = torch.full((c["n"], c["top"]), -1, device=x.device, dtype=torch.int32)
    best = torch.full((c["n"], c["top"]), -math.inf, device=x.device)
    if k:
        # a score and its place as one whole number, so that equal scores go to the lowest label
        bits = (x + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
        key = (order << 32) | (0xFFFFFFFF - torch.arange(c["labels"], device=x.device))
        at = 0xFFFFFFFF - (key.topk(k, dim=1).values & 0xFFFFFFFF)
        score = x.gather(1, at)
        label[:, :k] = torch.where(score > -math.inf, at, -1).int()
        best[:, :k] = score - m[:, None] - log_s[:, None]
    return dict(logprob=logprob, entropy=entropy, top_label=label, top_logprob=best)


def _own_gradient(s):
    c = s["case"]
    engine().label_logprobs_backward_device(s["x"], c["n"], c["labels"], d_target=s["target"], d_stat=s["stat"], d_grad=s["grad"],
                                            d_g_logprob=s["g_logprob"], d_entropy=s["entropy"], d_g_entropy=s["g_entropy"])
    return s["grad"]


def _plain_gradient(s):
    x = s["x"].float()
    log_p = x - s["stat"][:, :1] - s["stat"][:, 1:]
    p = torch.exp(log_p)
    inner = s["g_logprob"][:, None] + s["g_entropy"][:, None] * (log_p.clamp(min=-200.0) + s["entropy"][:, None])
    grad = -p * inner
    grad.scatter_add_(1, s["target"].long()[:, None], s["g_logprob"][:, None])
    return grad.to(s["x"].dtype)


def _own_quantize(s):
    from apr_amd import model
    c, e = s["case"], engine()
    e.quantize_rows_device(s["x"], c["n"], c["k"], s["q"], s["scale"], ld_q=s["q"].shape[1])
    with torch.cuda.stream(model.torch_stream(e)):     # the values that the 8 bits stand for
        torch.mul(s["q"][:, :c["k"]], s["scale"][:, None], out=s["values"])
    return dict(values=s["values"], scale=s["scale"])


def _plain_quantize(s):
    x = s["x"].float()
    most = x.abs().amax(1)
    scale = most / 127.0
    q = torch.round(x.double() * 127.0 / most.double()[:, None]).float()     # in 64 bits: next to a half, 32 round the other way
    return dict(values=q * scale[:, None], scale=scale)


def _own_linear(s):
    c = s["case"]
    engine().linear_i8_device(s["x"], s["x_scale"], s["w"], s["w_scale"], c["m"], c["n"], c["k"], s["out"], d_bias=s["bias"],
                              ld_x=s["x"].shape[1], ld_w=s["w"].shape[1])
    return s["out"]


def _plain_linear(s):
    k = s["case"]["k"]
    out = torch.mm(s["x"][:, :k].float(), s["w"][:, :k].float().t())
    out = out * s["x_scale"][:, None] * s["w_scale"]
    if s["bias"] is not None:
        out = out + s["bias"]
    return out.to(s["out"].dtype)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"logprobs": _own_logprobs, "gradient": _own_gradient, "quantize": _own_quantize, "linear": _own_linear}[op](state)
    return {"logprobs": _plain_logprobs, "gradient": _plain_gradient, "quantize": _plain_quantize, "linear": _plain_linear}[op](state)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "logprobs":
        values = case["n"] * case["labels"]
        return dict(bytes=values * size + case["n"] * (4 + 8 + 8 * case["top"]), flops=6 * values)
    if case["op"] == "gradient":
        values = case["n"] * case["labels"]
        return dict(bytes=2 * values * size + case["n"] * 24, flops=8 * values)
    if case["op"] == "quantize":
        values = case["n"] * case["k"]
        return dict(bytes=values * (size + 4) + case["n"] * 4, flops=4 * values)
    m, n, k = case["m"], case["n"], case["k"]
    return dict(bytes=m * k + n * k + m * n * size + 4 * (m + n), flops=2 * m * n * k)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        k = case["k"]
        w = s["w"][:, :k].double() * s["w_scale"].double()[:, None]
        out = torch.matmul(s["x"][:, :k].double(), w.t().contiguous()) * s["x_scale"].double()[:, None]
        return out if s["bias"] is None else out + s["bias"].double()
    x = s["x"].double()
    if case["op"] == "quantize":
        most = torch.linalg.vector_norm(x, math.inf, dim=1, keepdim=True)
        return dict(values=torch.round((127.0 * x).div(most)) * most / 127.0, scale=most[:, 0] / 127.0)
    # the definitions: p = exp(x) / sum(exp(x)), H = -sum(p log p)
    log_p = x - torch.logsumexp(x, 1, keepdim=True)
    p = torch.exp(log_p)
    entropy = torch.special.entr(p).sum(1)
    at = torch.arange(case["n"], device=x.device), s["target"].long()
    if case["op"] == "gradient":
        # of sum_i g_i log p_i[t_i] + h_i H_i, by the chain rule over p
        g, h = s["g_logprob"].double(), s["g_entropy"].double()
        by_log_p = -h[:, None] * p * torch.where(p > 0, log_p, 0.0)
        by_log_p[at] += g
        through_entropy = (h * entropy)[:, None] * p
        grad = by_log_p - through_entropy
        grad -= g[:, None] * p
        return grad
    top, k = case["top"], min(case["top"], case["labels"])
    label = torch.full((case["n"], top), -1, device=x.device, dtype=torch.int32)
    best = torch.full((case["n"], top), -math.inf, device=x.device, dtype=torch.float64)
    if k:
        score, place = torch.sort(x, dim=1, descending=True, stable=True)
        score, place = score[:, :k], place[:, :k]
        label[:, :k] = torch.where(torch.isinf(score), -1, place).int()
        best[:, :k] = log_p.gather(1, place)
    return dict(logprob=log_p[at], entropy=entropy, top_label=label, top_logprob=best)
