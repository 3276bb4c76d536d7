"""Row operators whose outputs are given: what the calls return stays what it is said to be, whatever memory the output
shares with the inputs.  The comparisons are of equal bits: the same kernels on the same values."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from multimodalspectraltransformer_amd import _lib as L
    from multimodalspectraltransformer_amd import ops

DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rnd(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols,pad", [(21, 200, 0), (21, 200, 8), (5, 1003, 3), (1, 7, 0)])
def test_layer_norm_over_its_input_keeps_z_for_the_backward_pass(t, rows, cols, pad):
    """out=x: z is what x held, and the backward pass from it gives what it gives without `out`."""
    x = rnd(rows, cols, seed=rows).to(t).to(DEV)
    dy = rnd(rows, cols, seed=rows + 1).to(t).to(DEV)
    gamma, beta = (1 + 0.2 * rnd(cols, seed=3)).to(DEV), rnd(cols, seed=4).to(DEV)
    y, z, stats = ops.layer_norm(x, gamma, beta)
    assert z is x
    want = ops.layer_norm_bwd(dy, z, stats, gamma)
    wide = torch.zeros(rows, cols + pad, dtype=t, device=DEV)
    over = wide[:, :cols]
    over.copy_(x)
    got = ops.layer_norm(over, gamma, beta, out=over)
    assert got[0] is over and torch.equal(over, y) and torch.equal(got[1], x) and torch.equal(got[2], stats)
    assert all(torch.equal(a, b) for a, b in zip(ops.layer_norm_bwd(dy, got[1], got[2], gamma), want))
    assert (wide[:, cols:] == 0).all()


def test_layer_norm_into_another_tensor_returns_its_input_as_z():
    """No copy where none is needed: another tensor, and other columns of the same one."""
    x = rnd(9, 64, seed=1).to(DEV)
    assert ops.layer_norm(x, out=torch.empty_like(x))[1] is x
    wide = torch.zeros(9, 128, device=DEV)
    left, right = wide[:, :64], wide[:, 64:]
    left.copy_(x)
    y, z, _ = ops.layer_norm(left, out=right)
    assert y is right and z is left and torch.equal(left, x) and torch.equal(right, ops.layer_norm(x)[0])


def test_layer_norm_over_a_transposed_input_that_is_copied():
    """x is read from a copy; an output over x's own memory leaves z what x held."""
    memory = rnd(12, 12, seed=2).to(DEV)
    x, held = memory.t(), memory.t().contiguous()
    y, z, stats = ops.layer_norm(x, out=memory)
    want = ops.layer_norm(held)
    assert torch.equal(y, want[0]) and torch.equal(z, held) and torch.equal(stats, want[2])


def test_outputs_that_share_some_elements_are_refused():
    memory, w = torch.zeros(20, 40, device=DEV), torch.zeros(40, device=DEV)
    x, below, right, left, wide = memory[:4, 8:16], memory[1:5, 8:16], memory[:4, 9:17], memory[:4, 1:9], memory[::2][:4, 8:16]
    res = torch.zeros(4, 8, device=DEV)
    for o in (below, right, left, wide):
        for call in (lambda: ops.dropout(x, 0.5, 1, out=o), lambda: ops.layer_norm(x, out=o), lambda: ops.layer_norm(x, z_out=o),
                     lambda: ops.layer_norm(res, residual=x, out=o), lambda: ops.layer_norm(res, residual=x, z_out=o),
                     lambda: ops.layer_norm(res, out=x, z_out=o), lambda: ops.layer_norm(res, out=x, z_out=x)):
            with pytest.raises(L.MMSTError):
                call()
    with pytest.raises(L.MMSTError):
        ops.layer_norm_bwd(x, x, torch.zeros(4, 2, device=DEV), dgamma=w[:8], dbeta=w[7:15])
    assert (memory == 0).all() and (w == 0).all()
    # what shares none: rows in turn, and columns beside one another
    x.copy_(rnd(4, 8, seed=1))
    for o in (memory[4:8, 8:16], memory[:4, 16:24], memory[:4, :8]):
        assert torch.equal(ops.dropout(x, 0.5, 1, out=o), ops.dropout(x, 0.5, 1))
        assert torch.equal(ops.layer_norm(x, out=o)[0], ops.layer_norm(x)[0])
    even, odd = memory[8::2][:4, :8], memory[9::2][:4, :8]
    even.copy_(x)
    assert torch.equal(ops.dropout(even, 0.5, 1, out=odd), ops.dropout(x, 0.5, 1)) and torch.equal(even, x)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 2.0 ** -17, 0.5])
def test_dropout_returns_one_layout_for_every_p(t, p):
    """Rows one after another, whatever the input's strides and whether anything is dropped."""
    base = rnd(12, 30, seed=5).to(t).to(DEV)
    for x in (base[:, :17], base[:, 3:11], base.t(), base[::3], base[:1].expand(12, 30), base):
        y = ops.dropout(x, p, 7)
        assert y.is_contiguous() and (y.data_ptr() != x.data_ptr() or x is base)
        if p < 2.0 ** -17:
            assert torch.equal(y, x)
