"""Equal calls of the linear layer with cross entropy give equal bits, also where losses are NaN or infinite."""
import pytest
import torch

from tests.test_linear_ce_gpu import dev, make

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from multimodalspectraltransformer_amd import ops

DEV = "cuda"


def bits(x):
    return x.view(torch.int32 if x.dtype == torch.float32 else torch.int16)


# logits in parts, small and large tiles, tiles of 160 words, the stream, one launch for the loss, rows that are numbered
@pytest.mark.parametrize("n,d,v", [(70, 1032, 45), (200, 4096, 1001), (130, 1024, 129), (16, 2048, 8003), (600, 8192, 7),
                                   (520, 96, 4096), (600, 640, 33000), (333, 136, 50001), (1000, 128, 20001), (300, 64, 100),
                                   (2100, 1024, 50001), (17000, 64, 3001)])
def test_equal_calls_give_equal_bits(n, d, v):
    h, w, b, t, dl = make(n, d, v, seed=n + d, ignored=n // 6)
    b[v // 2] = float("-inf")
    t[t >= 0] %= max(1, v // 2)
    t[1], t[n // 2], t[2] = v, -7, v // 2   # no words, and a masked one
    h, w, b, t, dl = dev(h, w, b, t, dl)
    for rows in (0, 256):
        calls = [ops.linear_ce(h, w, t, bias=b) + ops.linear_ce_grad(h, w, t, bias=b, dloss=dl, rows_per_piece=rows) for _ in range(4)]
        assert calls[0][0].isnan().any() and torch.isinf(calls[0][0]).any()
        for again in calls[1:]:
            assert all(torch.equal(bits(x), bits(y)) for x, y in zip(calls[0], again))
