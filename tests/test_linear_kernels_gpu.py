"""GPU: every kernel of the 8-bit product at sizes that end inside a tile, a stage and a unit, against 64 bits (label_oracle.py)."""
import pytest
import torch

from linear_shapes import CASES
from test_label_head_gpu import dev, eng, linear_case, near, whole as rows_of_8_bits  # noqa: F401
import label_oracle as oracle_l

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("kernel,whole,m,n,k", CASES)
def test_every_kernel_at_odd_sizes(eng, kernel, whole, m, n, k):  # noqa: F811
    for i, dtype in enumerate(TYPES):
        strides = {} if whole else (dict(ld_x=k + (k % 2 == 0), ld_w=k + 3), dict(shift=5), dict(shift=8))[i]
        # out at 16-byte units, at a stride that is none, and both again by the other types
        linear_case(eng, m, n, k, dtype, bias=i != 1, ld_out=(n + 7, -(-n // 8) * 8, n)[(i + k) % 3], **strides)


@pytest.mark.parametrize("kernel,whole,m,n,k", [next(c for c in CASES if c[:2] == head and c[4] == 1025) for head in dict.fromkeys(c[:2] for c in CASES)])
def test_every_kernel_writes_at_any_place(eng, kernel, whole, m, n, k):  # noqa: F811
    # out one element behind a 16-byte unit, rows of whole units apart: what lies around them stays
    x, w = (rows_of_8_bits(r, k, 1040 if whole else 1025, s) for s, r in enumerate((m, n)))
    xs, ws = (torch.linspace(1e-4, 1e-2, r, device=dev()) for r in (m, n))
    for dtype in TYPES:
        ld = -(-(n + 1) // 8) * 8
        store = torch.full((m * ld + 1,), -77.0, device=dev(), dtype=dtype)
        out = store[1:].view(m, ld)[:, :n]
        torch.cuda.synchronize()
        eng.linear_i8_device(x, xs, w, ws, m, n, k, out)
        eng.sync()
        want, tol = oracle_l.linear(x, xs, w, ws, None, dtype)
        near(out, want, tol, "product")
        assert store[0] == -77 and (store[1:].view(m, ld)[:, n:] == -77).all()
