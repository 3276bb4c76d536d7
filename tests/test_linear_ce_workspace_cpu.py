"""How much workspace mmst_linear_ce asks for, against what its header says."""
import ctypes as C

import pytest

from multimodalspectraltransformer_amd import _lib as L
from multimodalspectraltransformer_amd import ops


def need(grad, n, d, v, **kw):
    a, size = L.LinearCeArgs(N=n, D=d, V=v, **kw), C.c_size_t()
    assert ops._function("mmst_linear_ce_ws")(C.byref(a), grad, C.byref(size)) == 0
    return size.value


ROWS = [0, 1, 100, 256, 5000, 65536, 1 << 20, (1 << 23) - 256, 1 << 24]


@pytest.mark.parametrize("d", [8, 128, 136, 1016, 1024, 32768])
@pytest.mark.parametrize("v", [1, 43, 128, 129, 1000, 8064, 8065, 50001, 1 << 20])
def test_the_loss_alone_needs_what_the_header_says(d, v):
    for n in ROWS:
        if (n + 127) // 128 * ((v + 127) // 128) >= 0x7FFFFFFF:
            continue
        rows = max(256, (n + 255) // 256 * 256)
        if d <= 128 and v <= 128:
            assert need(0, n, d, v) == 256
            continue
        pairs = 8 * rows * ((v + 255) // 256 * 4)
        if d <= 128:
            pairs = max(pairs, (1 << 20) + rows * (128 if v > 8064 else 16))
        most = min(pairs, 1 << 30) + 4 * rows + (32 << 20 if d >= 1024 else 0)
        if 2 * n * d * v >= 1e10:   # rows that may be numbered
            most += 8 * rows + min(2 * d * rows, 1 << 30) + 4096
        assert need(0, n, d, v) <= most + 4 * 256, (n, d, v)   # (every buffer begins at a multiple of 256 bytes)


def test_fp32_sums_of_pieces_only_for_bf16_gradients():
    size = dict(n=4096, d=512, v=20000, rows_per_piece=256, dbias=1)
    bf16, both, alone = (need(1, grad_f32=f, **size) for f in (0, 1, 2))
    assert bf16 >= both + 20000 * 512 * 4 + 20000 * 4 and alone == both + 20000 * 512 * 4
