"""Rows of h and w further apart than the kernels reach."""
import pytest
import torch

from tests.test_linear_ce_gpu import DEV, dev, make

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from multimodalspectraltransformer_amd import ops


@pytest.mark.parametrize("apart", [1 << 20, (1 << 20) + 8, 1 << 21])
def test_rows_far_apart(apart):
    h, w, b, t, dl = dev(*make(70, 64, 90, seed=3, ignored=7))
    want = ops.linear_ce(h, w, t, bias=b) + ops.linear_ce_grad(h, w, t, bias=b, dloss=dl)
    memory = torch.full((91, apart), float("nan"), dtype=torch.bfloat16, device=DEV)
    for far in ("h", "w"):
        x = h if far == "h" else w
        y = memory[:x.shape[0], 8:72]
        y.copy_(x)
        pair = (y, w) if far == "h" else (h, y)
        got = ops.linear_ce(*pair, t, bias=b) + ops.linear_ce_grad(*pair, t, bias=b, dloss=dl)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        memory.fill_(float("nan"))
