"""Row operators of any width, without a GPU: the generator against its published vectors, and what the entry points and
their Python wrappers refuse before they touch the device."""
import ctypes as C

import numpy as np
import pytest
import torch

from multimodalspectraltransformer_amd import _lib as L
from multimodalspectraltransformer_amd import ops
from tests.philox_oracle import factor, philox


def test_philox_published_vectors():
    """Known answers of philox4x32-10 published with the paper's reference code."""
    def words(c, k):
        return [int(w) for w in philox([np.array(v) for v in c], k)]
    assert words([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert words([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert words([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_mask_keeps_the_asked_share():
    """Kept share of 2^16 elements: binomial, standard deviation at most 2^-9; five of them."""
    for p in (0.1, 0.5, 0.9):
        kept = (factor((256, 256), p, 77, 3) > 0).double().mean().item()
        assert abs(kept - (1 - p)) < 5 * 2.0 ** -9
    assert (factor((256, 256), 1.0, 77, 3) == 0).all() and (factor((16, 16), 0.0, 77, 3) == 1).all()


P = 0x10000   # stands for a device address: a refused call never follows it


def _rc(name, *args):
    return ops._function(name)(*args)


def _dropout(**kw):
    a = dict(x=P, ldx=128, y=2 * P, ldy=128, dtype=1, rows=4, cols=128, p=0.1, seed=1, offset=2)
    a.update(kw)
    return _rc("mmst_dropout", *a.values(), None)


def _ln(**kw):
    a = dict(x=P, ldx=128, res=None, ldr=0, gamma=None, beta=None, y=2 * P, ldy=128, z=None, ldz=0, stats=None, dtype=1,
             rows=4, cols=128, eps=1e-5, p=0.0, seed=0, offset=0)
    a.update(kw)
    return _rc("mmst_layer_norm", *a.values(), None)


def _ln_bwd(**kw):
    a = dict(dy=P, lddy=128, z=2 * P, ldz=128, stats=3 * P, gamma=None, dz_in=None, lddz_in=0, dz=4 * P, lddz=128, dx=None,
             lddx=0, dgamma=5 * P, dbeta=6 * P, accumulate=0, dtype=1, rows=4, cols=128, p=0.0, seed=0, offset=0, ws=7 * P,
             ws_bytes=1 << 20)
    a.update(kw)
    return _rc("mmst_layer_norm_bwd", *a.values(), None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(y=None), dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(cols=-1),
                                dict(ldx=127), dict(ldy=0), dict(p=-0.1), dict(p=1.1), dict(p=float("nan")),
                                dict(rows=1 << 40, cols=1 << 40, ldx=1 << 40, ldy=1 << 40)])
def test_dropout_refusals(kw):
    assert _dropout(**kw) == -1


def test_dropout_of_nothing():
    assert _dropout(rows=0) == 0 and _dropout(cols=0, x=None, y=None) == 0


@pytest.mark.parametrize("kw", [dict(x=None), dict(y=None), dict(dtype=5), dict(rows=-1), dict(cols=0), dict(cols=16385, ldx=16385, ldy=16385),
                                dict(ldx=100), dict(ldy=100), dict(res=P, ldr=5), dict(z=P, ldz=5), dict(eps=-1.0),
                                dict(eps=float("nan")), dict(p=2.0)])
def test_layer_norm_refusals(kw):
    assert _ln(**kw) == -1
    assert _ln(rows=0) == 0


@pytest.mark.parametrize("kw", [dict(dy=None), dict(z=None), dict(stats=None), dict(dz=None), dict(p=0.5), dict(dtype=9),
                                dict(cols=0), dict(cols=20000), dict(ws=None), dict(ws_bytes=16), dict(lddy=1), dict(ldz=1),
                                dict(lddz=1), dict(dz_in=P, lddz_in=3), dict(p=0.5, dx=P, lddx=3), dict(rows=-5)])
def test_layer_norm_bwd_refusals(kw):
    assert _ln_bwd(**kw) == -1


def test_workspace_query():
    n = C.c_size_t()
    assert _rc("mmst_layer_norm_bwd_ws", 1, 1000, 128, C.byref(n)) == 0 and n.value >= 2 * 128 * 4
    assert _rc("mmst_layer_norm_bwd_ws", 1, 0, 128, C.byref(n)) == 0
    assert _rc("mmst_layer_norm_bwd_ws", 1, 10, 0, C.byref(n)) == -1
    assert _rc("mmst_layer_norm_bwd_ws", 1, 10, 128, None) == -1


def test_wrappers_refuse_cpu_tensors_and_bad_arguments():
    x = torch.zeros(4, 128)
    for call in (lambda: ops.dropout(x, 0.1, 1), lambda: ops.layer_norm(x), lambda: ops.layer_norm_bwd(x, x, torch.zeros(4, 2))):
        with pytest.raises(L.MMSTError):
            call()
