"""What mmst_linear_ce and its wrappers refuse before they touch the device, and how much workspace they ask for."""
import ctypes as C

import pytest
import torch

from multimodalspectraltransformer_amd import _lib as L
from multimodalspectraltransformer_amd import ops

P = 0x10000   # stands for a device address: a refused call never follows it


def _args(**kw):
    a = L.LinearCeArgs()
    d = dict(h=P, ldh=64, w=2 * P, ldw=64, target=3 * P, ignore_index=-100, N=10, D=64, V=100, loss=4 * P, dh=5 * P, lddh=64,
             dw=6 * P, ws=7 * P, ws_bytes=1 << 30, grad_scale=1.0)
    d.update(kw)
    for k, v in d.items():
        setattr(a, k, v)
    return a


def _call(grad, **kw):
    return ops._function("mmst_linear_ce")(C.byref(_args(**kw)), grad, None)


@pytest.mark.parametrize("kw", [dict(h=None), dict(w=None), dict(target=None), dict(loss=None), dict(N=-1), dict(V=0), dict(D=0),
                                dict(D=12, ldh=16, ldw=16), dict(D=40000, ldh=40000, ldw=40000), dict(V=1 << 23), dict(N=1 << 25),
                                dict(N=1 << 24, V=1 << 22), dict(ldh=63), dict(ldh=56), dict(ldw=68), dict(ldw=0), dict(h=P + 8),
                                dict(w=P + 2), dict(ws=None), dict(ws=P + 16), dict(ws_bytes=64), dict(rows_per_piece=-1),
                                dict(ldw=1 << 21)])
def test_linear_ce_refusals(kw):
    assert _call(0, **kw) == -1
    assert _call(1, **kw) == -1


@pytest.mark.parametrize("kw", [dict(dh=None), dict(dw=None), dict(lddh=63), dict(dh=P + 4), dict(dw=P + 8), dict(ws_bytes=4096)])
def test_linear_ce_gradient_refusals(kw):
    assert _call(1, **kw) == -1


@pytest.mark.parametrize("kw", [dict(target=3 * P + 4), dict(bias=8 * P + 2), dict(loss=4 * P + 1), dict(lse=8 * P + 2)])
def test_linear_ce_refuses_misaligned_vectors(kw):
    assert _call(0, **kw) == -1
    assert _call(1, **kw) == -1
    assert _call(1, dloss=8 * P + 2) == -1
    assert _call(1, dbias=8 * P + 1) == -1
    assert _call(1, dbias=8 * P + 2, grad_f32=1) == -1


def test_linear_ce_workspace():
    def need(grad, **kw):
        n = C.c_size_t()
        assert ops._function("mmst_linear_ce_ws")(C.byref(_args(**kw)), grad, C.byref(n)) == 0
        return n.value
    # a piece's gradient of the logits is what counts, and it is bounded by rows_per_piece
    whole, piece = need(1, N=4096, V=50000), need(1, N=4096, V=50000, rows_per_piece=256)
    assert 4096 * 50000 * 2 <= whole <= 4096 * 50176 * 2 * 1.2
    assert 256 * 50000 * 2 <= piece <= 256 * 50176 * 2 * 1.2 + 50000 * 64 * 4 + (1 << 20)
    assert need(0, N=4096, V=50000) < 4096 * 50000 * 2 / 10
    assert need(1, N=1 << 20, V=131072, D=1024, ldh=1024, ldw=1024) < 7 << 30
    n = C.c_size_t()
    assert ops._function("mmst_linear_ce_ws")(C.byref(_args(V=0)), 1, C.byref(n)) == -1
    assert ops._function("mmst_linear_ce_ws")(C.byref(_args()), 1, None) == -1
    assert ops._function("mmst_linear_ce_ws")(None, 1, C.byref(n)) == -1


def test_wrappers_refuse_cpu_tensors():
    h, w, t = torch.zeros(4, 64).bfloat16(), torch.zeros(9, 64).bfloat16(), torch.zeros(4, dtype=torch.int64)
    for f in (ops.linear_ce, ops.linear_ce_grad):
        with pytest.raises(L.MMSTError):
            f(h, w, t)
