"""The loss alone at sizes where its rows go in pieces, against 64-bit arithmetic on picked rows."""
import pytest
import torch

from tests.test_linear_ce_gpu import IGN, check_loss, oracle

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from multimodalspectraltransformer_amd import ops

DEV = "cuda"


def big(n, d, v, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.randn(n, d, device=DEV, generator=g).bfloat16()
    w = (torch.randn(v, d, device=DEV, generator=g) * (scale / d ** 0.5)).bfloat16()
    return h, w, 0.3 * torch.randn(v, device=DEV, generator=g), torch.randint(0, v, (n,), device=DEV, generator=g)


def test_streamed_loss_whose_pairs_need_pieces():
    """A row has 128 bytes of pairs in the eight parts of the vocabulary: 2^30 bytes of them and 1 MiB are 8380416 rows."""
    cut, d, v = 8380416, 8, 8100
    n = cut + 300
    h, w, b, t = big(n, d, v, seed=3)
    t[cut - 2], t[cut + 1], t[5] = IGN, v, IGN
    loss, lse = ops.linear_ce(h, w, t, bias=b)
    pick = [0, 5, n // 2] + list(range(cut - 3, cut + 3)) + [n - 1]
    check_loss(oracle(h[pick].cpu(), w.cpu(), b.cpu(), t[pick].cpu(), None), loss[pick], lse[pick])
    assert int((loss == 0).sum()) == 2 and int(loss.isnan().sum()) == 1
    torch.cuda.empty_cache()
