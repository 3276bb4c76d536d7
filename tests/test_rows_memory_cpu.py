"""The check for outputs that share memory with inputs, against sets of elements."""
import random

import torch

from multimodalspectraltransformer_amd import ops


def test_overlap_of_strided_rows():
    memory, rng = torch.zeros(400), random.Random(1)
    found = [0, 0]
    for _ in range(5000):
        rows, cols = rng.randint(1, 6), rng.randint(1, 9)
        lda = cols + rng.randint(0, 9)
        ldb = rng.choice([lda, cols + rng.randint(0, 9)])
        at, bt = rng.randint(0, 60), rng.randint(0, 60)
        elements = [{first + r * ld + c for r in range(rows) for c in range(cols)} for first, ld in ((at, lda), (bt, ldb))]
        want = bool(elements[0] & elements[1])
        a, b = memory.as_strided((rows, cols), (lda, 1), at), memory.as_strided((rows, cols), (ldb, 1), bt)
        assert ops._overlap(a, lda, b, ldb) == want, (rows, cols, lda, ldb, at, bt)
        found[want] += 1
    assert min(found) > 1000
    assert not ops._overlap(memory[:0], 1, memory[:0], 1)


P = 0x10000   # stands for a device address: a refused call never follows it


def _layer_norm(**kw):
    a = dict(x=P, ldx=128, res=None, ldr=0, gamma=None, beta=None, y=2 * P, ldy=128, z=3 * P, ldz=128, stats=None, dtype=1,
             rows=4, cols=128, eps=1e-5, p=0.0, seed=0, offset=0)
    a.update(kw)
    return ops._function("mmst_layer_norm")(*a.values(), None)


def _layer_norm_bwd(**kw):
    a = dict(dy=P, lddy=128, z=2 * P, ldz=128, stats=3 * P, gamma=None, dz_in=None, lddz_in=0, dz=4 * P, lddz=128, dx=8 * P,
             lddx=128, dgamma=5 * P, dbeta=6 * P, accumulate=0, dtype=1, rows=4, cols=128, p=0.5, seed=0, offset=0, ws=7 * P,
             ws_bytes=1 << 20)
    a.update(kw)
    return ops._function("mmst_layer_norm_bwd")(*a.values(), None)


def test_one_tensor_as_two_outputs_is_refused():
    assert _layer_norm(z=2 * P) == -1 and _layer_norm(y=P, z=P) == -1
    assert _layer_norm_bwd(dx=4 * P) == -1
    for by in (0, 4, 127 * 4, -127 * 4):
        assert _layer_norm_bwd(dbeta=5 * P + by) == -1
        assert _layer_norm_bwd(dbeta=5 * P + by, rows=0) == -1
