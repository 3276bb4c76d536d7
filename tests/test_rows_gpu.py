"""Row operators of any width on the GPU -- counter-based dropout, layer norm forward and backward -- against 64-bit
arithmetic on the same inputs.

Tolerances count roundings, u = 2^-24 for fp32 and half = finfo(type).eps / 2 for the stored type.  A row sum adds at most
16 values per lane, 6 steps across a wave and 16 waves: fewer than 64 roundings of partial sums that the sum of the
magnitudes bounds, hence 64 u * sum |.|.  Column sums add at most 64 rows per lane here, 64 lane groups and 16 + 64
partial sums: 256 u * sum |.|."""
import numpy as np
import pytest
import torch

from tests.philox_oracle import factor, factor_at

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from multimodalspectraltransformer_amd import _lib as L
    from multimodalspectraltransformer_amd import ops

DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SEED, OFFSET = 0x9E3779B97F4A7C15, (5 << 32) + 3


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """half a step among the numbers below the smallest normal one"""
    return torch.finfo(t).smallest_normal * half(t)


def rnd(*shape, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g) * scale + shift


def strided(t, pad, lead=0):
    """the same values as rows of a wider tensor on the GPU, `lead` elements behind its start"""
    wide = torch.full((t.shape[0], t.shape[1] + pad + lead), float("nan"), dtype=t.dtype, device=DEV)
    wide[:, lead:lead + t.shape[1]] = t.to(DEV)
    return wide[:, lead:lead + t.shape[1]]


def inside(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.double()
    bad = ~((got - want).abs() <= tol) & ~((got == want) | (got.isnan() & want.isnan()))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((got - want).abs().max()):.3g} " \
                          f"(first at {bad.nonzero()[0].tolist()})"


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (17,), (1, 1), (64, 128), (33, 1001), (700, 3), (1000, 1), (2, 3, 40), (3, 4104)])
def test_dropout(t, shape):
    x = rnd(*shape, seed=1).to(t)
    for p in (0.0, 0.1, 0.5, 1.0):
        y = ops.dropout(x.to(DEV), p, SEED, OFFSET)
        f = factor(shape, p, SEED, OFFSET)
        want = x.double() * f
        assert ((y.cpu() == 0) == ((f == 0) | (x == 0))).all()
        # the scale's rounding, the product's and the stored one
        inside(y, want, want.abs() * (2 * U + half(t)) + tiny(t), f"dropout {shape} p={p}")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols,pad,lead", [(128, 8, 0), (128, 3, 1), (1001, 7, 0), (40, 24, 8), (5, 1, 1), (72, 0, 0)])
def test_dropout_strided_in_place_and_unaligned(t, cols, pad, lead):
    x = rnd(37, cols, seed=2).to(t)
    f = factor(x.shape, 0.3, 11, 0)
    want = x.double() * f
    tol = want.abs() * (2 * U + half(t)) + tiny(t)
    xs = strided(x, pad, lead)
    inside(ops.dropout(xs, 0.3, 11), want, tol, "strided input")
    out = strided(torch.zeros(37, cols, dtype=t), pad + 8, lead)
    whole = out._base if out._base is not None else out
    before = whole.clone()
    assert ops.dropout(xs, 0.3, 11, out=out) is out
    inside(out, want, tol, "strided output")
    mark = torch.ones_like(whole, dtype=torch.bool)
    mark[:, lead:lead + cols] = False
    assert torch.equal(whole[mark].isnan(), before[mark].isnan())   # columns beside the rows are left alone
    inside(ops.dropout(xs, 0.3, 11, out=xs), want, tol, "in place")
    flat = torch.zeros(37 * cols + 1, dtype=t, device=DEV)
    flat[1:] = x.reshape(-1).to(DEV)
    inside(ops.dropout(flat[1:], 0.3, 11), want.reshape(-1), tol.reshape(-1), "unaligned start")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols,pad", [(1003, 31, 2), (1003, 33, 1), (517, 127, 5), (517, 129, 3), (2, 4099, 13), (301, 257, 1), (9, 9, 9), (1, 130, 1)])
def test_dropout_of_odd_rows(t, rows, cols, pad):
    """Blocks of eight elements that begin in one row and end in the next, and the widths at which they are taken."""
    x = rnd(rows, cols, seed=rows).to(t)
    want = x.double() * factor(x.shape, 0.3, 11, 5)
    tol = want.abs() * (2 * U + half(t)) + tiny(t)
    wide = torch.full((rows + 1, cols + pad), float("nan"), dtype=t, device=DEV)
    out = wide[:rows, :cols]
    xs = strided(x, pad + 2)
    ops.dropout(xs, 0.3, 11, 5, out=out)
    inside(out, want, tol, "strided")
    assert wide[:, cols:].isnan().all() and wide[rows:].isnan().all()
    ops.dropout(xs, 0.3, 11, 5, out=xs)
    inside(xs, want, tol, "in place")
    y = ops.dropout(strided(x, pad + 2), 0.0, 11)
    assert torch.equal(y.cpu(), x)


def test_dropout_of_nothing_dropped_is_its_input():
    x = rnd(40, 17, seed=1).to(DEV)
    assert ops.dropout(x, 0.0, 1) is x and ops.dropout(x, 2.0 ** -18, 1) is x
    out = torch.empty_like(x)
    assert ops.dropout(x, 0.0, 1, out=out) is out and torch.equal(out, x)
    assert ops.dropout(x, 2.0 ** -17, 1) is not x


def test_dropout_clears_infinities_and_nan():
    x = torch.full((64, 128), float("nan"), device=DEV)
    x[::2] = float("inf")
    f = factor(x.shape, 0.5, 3, 1)
    y = ops.dropout(x, 0.5, 3, 1).cpu()
    assert (y[f == 0] == 0).all() and not torch.isfinite(y[f > 0]).any()
    assert (ops.dropout(x, 1.0, 3, 1) == 0).all()


def test_dropout_mask_depends_on_every_bit_of_seed_and_offset():
    x = torch.ones(64, 64, device=DEV)
    masks = [ops.dropout(x, 0.5, s, o) for s, o in ((1, 0), (1 | 1 << 33, 0), (1, 1), (1, 1 << 40), (2, 0))]
    for i in range(len(masks)):
        for j in range(i):
            assert not torch.equal(masks[i], masks[j])
    assert torch.equal(masks[0], ops.dropout(x, 0.5, 1, 0))


@pytest.mark.parametrize("rows,cols,pad", [(1, (1 << 32) + 4100, 0), (65600, 65599, 1)])
def test_dropout_past_32_bits_of_elements(rows, cols, pad):
    """More than 2^32 elements, as one vector and as odd rows of a wider tensor."""
    wide = torch.ones(rows, cols + pad, dtype=torch.bfloat16, device=DEV)
    y = ops.dropout(wide[:, :cols], 0.25, SEED, OFFSET).reshape(-1)
    n = rows * cols
    for first in (0, (1 << 32) - 700, (1 << 32) + 1, n - 1000):
        idx = np.arange(first, min(n, first + 1000), dtype=np.uint64)
        want = torch.from_numpy(factor_at(idx, 0.25, SEED, OFFSET)).bfloat16()
        assert torch.equal(y[first:first + len(idx)].cpu(), want)
    del y, wide
    torch.cuda.empty_cache()


def test_dropout_of_nothing():
    for shape in ((0,), (0, 5), (5, 0)):
        assert ops.dropout(torch.zeros(shape, device=DEV), 0.5, 1).shape == torch.Size(shape)


# ------------------------------------------------------------------------------------------------ layer norm
def ln_oracle(x, res, gamma, beta, eps, f):
    z = x.double() * f if f is not None else x.double()
    if res is not None:
        z = z + res.double()
    mean = z.mean(-1, keepdim=True)
    rstd = ((z - mean) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    g = torch.ones(x.shape[-1], dtype=torch.float64) if gamma is None else gamma.double()
    b = torch.zeros(x.shape[-1], dtype=torch.float64) if beta is None else beta.double()
    return z, mean, rstd, (z - mean) * rstd * g + b, g, b


def check_forward(x, res, gamma, beta, p, y, z, stats, eps=1e-5):
    t = x.dtype
    f = factor(x.shape, p, SEED, OFFSET) if p > 0 else None
    wz, mean, rstd, wy, g, b = ln_oracle(x, res, gamma, beta, eps, f)
    top = wz.abs().amax(-1, keepdim=True)
    dmean = 68 * U * top                                            # the row sum, z's own roundings, 1 / cols
    # variance: its sum, and centred values that are off by 3 u top each (the mean's own error only enters squared,
    # rstd * dmean < 1 for the rows here); rstd has half of that
    drstd = (72 + 8 * top * rstd) * U + (dmean * rstd) ** 2
    inside(stats[..., :1], mean, dmean, "mean")
    inside(stats[..., 1:], rstd, rstd * drstd, "rstd")
    centred = (wy - b).abs()
    tol = (g * rstd).abs() * (dmean + 3 * U * top) + centred * (drstd + 4 * U) + wy.abs() * (half(t) + U) + tiny(t)
    inside(y, wy, tol * 1.01, "y")   # 1.01: products of two of these terms
    if res is not None or p > 0:
        inside(z, wz, wz.abs() * half(t) + 3 * U * top + tiny(t), "z")


WIDTHS = [1, 2, 7, 16, 100, 128, 136, 250, 512, 1003, 1024, 2048, 2056, 4096, 4099, 8192, 8193, 16384, 16383]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_layer_norm(t, cols):
    rows = 9 if cols > 1024 else 77
    x, res = rnd(rows, cols, seed=cols, scale=1.5, shift=0.3).to(t), rnd(rows, cols, seed=cols + 1).to(t)
    gamma, beta = 1 + 0.3 * rnd(cols, seed=5), 0.3 * rnd(cols, seed=6)
    for use_res, p, affine in ((False, 0.0, True), (True, 0.0, False), (False, 0.2, True), (True, 0.2, True)):
        g, b = (gamma, beta) if affine else (None, None)
        y, z, stats = ops.layer_norm(x.to(DEV), None if g is None else g.to(DEV), None if b is None else b.to(DEV),
                                     residual=res.to(DEV) if use_res else None, p=p, seed=SEED, offset=OFFSET)
        check_forward(x, res if use_res else None, g, b, p, y, z, stats)


def bwd_oracle(dy, z, stats, gamma, dz_in, f):
    dy, z, st = dy.double(), z.double(), stats.double()
    mean, rstd = st[..., :1], st[..., 1:]
    g = torch.ones(dy.shape[-1], dtype=torch.float64) if gamma is None else gamma.double()
    xh = (z - mean) * rstd
    q = dy * g
    dz = rstd * (q - q.mean(-1, keepdim=True) - xh * (q * xh).mean(-1, keepdim=True))
    if dz_in is not None:
        dz = dz + dz_in.double()
    return xh, q, dz, dz if f is None else dz * f, (dy * xh).sum(0), dy.sum(0)


def check_backward(dy, z, stats, gamma, dz_in, p, got, base=None):
    t = dy.dtype
    f = factor(dy.shape, p, SEED, OFFSET) if p > 0 else None
    xh, q, dz, dx, dg, db = bwd_oracle(dy, z, stats, gamma, dz_in, f)
    rstd = stats[..., 1:].double()
    top = torch.maximum(z.double().abs().amax(-1, keepdim=True), stats[..., :1].double().abs())
    dxh = U * top * rstd + 2 * U * xh.abs()                          # z - mean, times rstd
    s2 = (q * xh).mean(-1, keepdim=True).abs()
    ds1 = 66 * U * q.abs().mean(-1, keepdim=True)
    ds2 = 68 * U * (q * xh).abs().mean(-1, keepdim=True) + (q.abs() * dxh).mean(-1, keepdim=True)
    err = rstd * (5 * U * q.abs() + ds1 + 4 * U * q.abs().mean(-1, keepdim=True) + xh.abs() * ds2 + s2 * dxh
                  + 4 * U * xh.abs() * s2)
    if dz_in is not None:
        err = err + 2 * U * (dz_in.double().abs() + dz.abs())
    gdz, gdx, gdg, gdb = got
    inside(gdz, dz, 1.01 * err + dz.abs() * half(t) + tiny(t), "dz")
    scale = 1.0 if f is None else f
    inside(gdx, dx, 1.01 * err * scale + dx.abs() * (half(t) + 2 * U) + tiny(t), "dx")
    b0 = (0.0, 0.0) if base is None else [v.double() for v in base]
    terms = (dy.double() * xh).abs().sum(0)
    inside(gdg, dg + b0[0], 256 * U * terms + (dy.double().abs() * dxh).sum(0) + U * (dg + b0[0]).abs(), "dgamma")
    inside(gdb, db + b0[1], 256 * U * dy.double().abs().sum(0) + U * (db + b0[1]).abs(), "dbeta")


def stats_of(z, eps=1e-5):
    zd = z.double()
    mean = zd.mean(-1, keepdim=True)
    return torch.cat([mean, ((zd - mean) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()], -1).float()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_layer_norm_bwd(t, cols):
    rows = 9 if cols > 1024 else 77
    z, dy = rnd(rows, cols, seed=cols, scale=1.5, shift=0.3).to(t), rnd(rows, cols, seed=cols + 2).to(t)
    add, gamma, stats = rnd(rows, cols, seed=cols + 3).to(t), 1 + 0.3 * rnd(cols, seed=5), stats_of(z)
    for use_add, p, affine in ((False, 0.0, True), (True, 0.0, False), (False, 0.2, True), (True, 0.2, True)):
        g = gamma if affine else None
        a = add if use_add else None
        got = ops.layer_norm_bwd(dy.to(DEV), z.to(DEV), stats.to(DEV), None if g is None else g.to(DEV),
                                 dz_in=None if a is None else a.to(DEV), p=p, seed=SEED, offset=OFFSET)
        check_backward(dy, z, stats, g, a, p, got)


@pytest.mark.parametrize("rows,cols", [(1 << 20, 4104), ((1 << 22) + 5, 1027)])
def test_layer_norm_past_32_bits_of_elements(rows, cols):
    """The last of more than 2^32 elements.  Half of them dropped and the others doubled is exact in bf16, so those rows by
    themselves, without dropout, have to give the same bits."""
    t = torch.bfloat16
    x = rnd(64, cols, seed=1).to(t).to(DEV).repeat(rows // 64 + 1, 1)[:rows]
    gamma, beta = (1 + 0.2 * rnd(cols, seed=2)).to(DEV), rnd(cols, seed=3).to(DEV)
    y, z, stats = ops.layer_norm(x, gamma, beta, p=0.5, seed=SEED, offset=OFFSET)
    k = 5
    idx = np.arange((rows - k) * cols, rows * cols, dtype=np.uint64)
    f = torch.from_numpy(factor_at(idx, 0.5, SEED, OFFSET)).reshape(k, cols)
    assert torch.equal(z[-k:].cpu().double(), x[-k:].cpu().double() * f)
    alone = ops.layer_norm(z[-k:].contiguous(), gamma, beta)
    assert torch.equal(y[-k:], alone[0]) and torch.equal(stats[-k:], alone[2])
    dz, dx = ops.layer_norm_bwd(x, z, stats, gamma, p=0.5, seed=SEED, offset=OFFSET)[:2]
    want = ops.layer_norm_bwd(x[-k:].contiguous(), z[-k:].contiguous(), stats[-k:].contiguous(), gamma)[0]
    assert torch.equal(dz[-k:], want) and torch.equal(dx[-k:].cpu().double(), want.cpu().double() * f)
    del x, y, z, dz, dx
    torch.cuda.empty_cache()


# on both sides of every change of the number of lanes per row and of the accesses per lane
EDGES = [3, 8, 9, 24, 31, 32, 33, 63, 64, 65, 127, 129, 255, 256, 257, 300, 511, 513, 768, 769, 777, 1025, 1536, 1537, 2047, 2049, 4095,
         4097, 6144, 6145, 8191]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols", EDGES)
def test_layer_norm_at_the_edges_of_its_shapes(t, cols):
    rows = 9 if cols > 1024 else 77
    x, res, dy = (rnd(rows, cols, seed=cols + i, scale=1.5, shift=0.3).to(t) for i in range(3))
    gamma, beta = 1 + 0.3 * rnd(cols, seed=5), 0.3 * rnd(cols, seed=6)
    # rows apart, and nothing but NaN between them
    xs, rs, ds = strided(x, 5), strided(res, 3, 1), strided(dy, 8, 8)
    y, z, stats = ops.layer_norm(xs, gamma.to(DEV), beta.to(DEV), residual=rs, p=0.2, seed=SEED, offset=OFFSET)
    check_forward(x, res, gamma, beta, 0.2, y, z, stats)
    wide = torch.full((rows, cols + 2), float("nan"), dtype=t, device=DEV)
    again = ops.layer_norm(xs, gamma.to(DEV), beta.to(DEV), residual=rs, p=0.2, seed=SEED, offset=OFFSET, out=wide[:, 1:-1])
    assert torch.equal(again[0], y) and wide[:, 0].isnan().all() and wide[:, -1].isnan().all()
    got = ops.layer_norm_bwd(ds, z, stats, gamma.to(DEV), dz_in=rs, p=0.2, seed=SEED, offset=OFFSET)
    check_backward(dy, z.cpu(), stats.cpu(), gamma, res, 0.2, got)


@pytest.mark.parametrize("rows,cols", [(1, 128), (3, 200), (5000, 64), (4100, 1000), (1500, 1536)])
def test_layer_norm_many_rows_both_passes(rows, cols):
    """More rows than one sweep of the grid; the backward pass from what the forward pass returned."""
    t = torch.bfloat16
    x, res = rnd(rows, cols, seed=1).to(t), rnd(rows, cols, seed=2).to(t)
    gamma, beta, dy = 1 + 0.2 * rnd(cols, seed=3), rnd(cols, seed=4), rnd(rows, cols, seed=5).to(t)
    y, z, stats = ops.layer_norm(x.to(DEV), gamma.to(DEV), beta.to(DEV), residual=res.to(DEV), p=0.1, seed=SEED, offset=OFFSET)
    check_forward(x, res, gamma, beta, 0.1, y, z, stats)
    base = (rnd(cols, seed=6), rnd(cols, seed=7))
    acc = [b.to(DEV) for b in base]
    got = ops.layer_norm_bwd(dy.to(DEV), z, stats, gamma.to(DEV), p=0.1, seed=SEED, offset=OFFSET, dgamma=acc[0], dbeta=acc[1])
    assert got[2] is acc[0] and got[3] is acc[1]
    check_backward(dy, z.cpu(), stats.cpu(), gamma, None, 0.1, got, base=base)
    again = ops.layer_norm_bwd(dy.to(DEV), z, stats, gamma.to(DEV), p=0.1, seed=SEED, offset=OFFSET)
    twice = ops.layer_norm_bwd(dy.to(DEV), z, stats, gamma.to(DEV), p=0.1, seed=SEED, offset=OFFSET)
    assert all(torch.equal(a, b) for a, b in zip(again, twice))   # sums in a fixed order


@pytest.mark.parametrize("t", TYPES)
def test_layer_norm_strided_shapes_and_in_place(t):
    x, res = rnd(21, 200, seed=1).to(t), rnd(21, 200, seed=2).to(t)
    gamma, beta = 1 + 0.2 * rnd(200, seed=3), rnd(200, seed=4)
    g, b = gamma.to(DEV), beta.to(DEV)
    want = ops.layer_norm(x.to(DEV), g, b, residual=res.to(DEV), p=0.1, seed=SEED, offset=OFFSET)
    check_forward(x, res, gamma, beta, 0.1, *want)
    for pad, lead in ((8, 0), (5, 1)):
        xs, rs = strided(x, pad, lead), strided(res, pad + 8, lead)
        got = ops.layer_norm(xs, g, b, residual=rs, p=0.1, seed=SEED, offset=OFFSET, out=xs, z_out=rs)
        assert got[0] is xs and got[1] is rs
        check_forward(x, res, gamma, beta, 0.1, *got)
    got = ops.layer_norm(x.to(DEV).view(3, 7, 200), g, b, residual=res.to(DEV).view(3, 7, 200), p=0.1, seed=SEED, offset=OFFSET)
    assert all(torch.equal(a.reshape(w.shape), w) for a, w in zip(got, want))
    broad = ops.layer_norm(x.to(DEV), g, b, residual=res[:1].to(DEV).expand(21, 200))   # copied: rows without a stride
    check_forward(x, res[:1].expand(21, 200), gamma, beta, 0.0, *broad)
    dy = rnd(1, 200, seed=8).to(t)
    got = ops.layer_norm_bwd(dy.to(DEV).expand(21, 200), strided(want[1].cpu(), 3, 1), want[2], g)
    check_backward(dy.expand(21, 200), want[1].cpu(), want[2].cpu(), gamma, None, 0.0, got)
    # a transposed input is copied as well, a transposed output refused
    y = ops.layer_norm(x.to(DEV).t().contiguous().t(), g, b)[0]
    check_forward(x, None, gamma, beta, 0.0, y, None, ops.layer_norm(x.to(DEV), g, b)[2])
    with pytest.raises(L.MMSTError):
        ops.layer_norm(x.to(DEV), g, b, out=torch.empty(200, 21, dtype=t, device=DEV).t())


def test_layer_norm_of_large_means_and_constant_rows():
    """A mean a thousand times the spread costs no more digits than the type of z has; a constant row has rstd = eps^-1/2."""
    x = rnd(40, 500, seed=1) + 1000.0
    x[7] = 3.25
    y, z, stats = ops.layer_norm(x.to(DEV))
    check_forward(x, None, None, None, 0.0, y, z, stats)
    assert z.data_ptr() != y.data_ptr() and (y[7] == 0).all()


def test_layer_norm_keeps_bad_rows_to_themselves():
    x = rnd(70, 256, seed=1)
    x[3, 5], x[64, 0] = float("nan"), float("inf")
    y = ops.layer_norm(x.to(DEV))[0].cpu()
    fine = torch.ones(70, dtype=torch.bool)
    fine[[3, 64]] = False
    assert y[3].isnan().all() and y[64].isnan().any() and torch.isfinite(y[fine]).all()
    assert torch.equal(y[fine], ops.layer_norm(x[fine].to(DEV))[0].cpu())


def test_layer_norm_of_no_rows():
    e = torch.zeros(0, 128, device=DEV)
    y, z, stats = ops.layer_norm(e)
    assert y.shape == (0, 128) and stats.shape == (0, 2)
    dz, dx, dg, db = ops.layer_norm_bwd(e, e, stats)
    assert dz.shape == (0, 128) and (dg == 0).all() and (db == 0).all()
    acc = [torch.ones(128, device=DEV), torch.ones(128, device=DEV)]
    ops.layer_norm_bwd(e, e, stats, dgamma=acc[0], dbeta=acc[1])
    assert (acc[0] == 1).all() and (acc[1] == 1).all()


def test_layer_norm_gradients_against_differences():
    """sum(w * y) of the 64-bit definition, central differences with step h: the second-order term is below
    h^2 * max|d3| <= 1e-8 here; the kernel's fp32 gradients agree to 2e-5 of their scale (64 u plus that)."""
    torch.manual_seed(4)
    x, res, w = torch.randn(3, 24).double(), torch.randn(3, 24).double(), torch.randn(3, 24).double()
    gamma, beta = 1 + 0.2 * torch.randn(24).double(), torch.randn(24).double()
    x, res, w, gamma, beta = (v.float().double() for v in (x, res, w, gamma, beta))
    f = factor((3, 24), 0.25, SEED, OFFSET)

    def loss(x, res, gamma, beta):
        return (ln_oracle(x, res, gamma, beta, 1e-5, f)[3] * w).sum()

    def numeric(i, args, h=1e-5):
        out = torch.zeros_like(args[i])
        for k in range(out.numel()):
            hi, lo = [a.clone() for a in args], [a.clone() for a in args]
            hi[i].view(-1)[k] += h
            lo[i].view(-1)[k] -= h
            out.view(-1)[k] = (loss(*hi) - loss(*lo)) / (2 * h)
        return out

    args = [x, res, gamma, beta]
    y, z, stats = ops.layer_norm(x.float().to(DEV), gamma.float().to(DEV), beta.float().to(DEV), residual=res.float().to(DEV),
                                 p=0.25, seed=SEED, offset=OFFSET)
    dz, dx, dg, db = ops.layer_norm_bwd(w.float().to(DEV), z, stats, gamma.float().to(DEV), p=0.25, seed=SEED, offset=OFFSET)
    for got, i in ((dx, 0), (dz, 1), (dg, 2), (db, 3)):
        want = numeric(i, args)
        inside(got, want, 2e-5 * want.abs().max(), f"argument {i}")


def test_one_mask_in_all_three_operators():
    for shape in ((13, 128), (13, 77)):
        ones, zero = torch.ones(shape, device=DEV), torch.zeros(shape, device=DEV)
        m = ops.dropout(ones, 0.4, 9, 2)
        y, z, stats = ops.layer_norm(ones, residual=zero, p=0.4, seed=9, offset=2)
        assert torch.equal(z, m)
        dz, dx, _, _ = ops.layer_norm_bwd(zero, z, stats, dz_in=ones, p=0.4, seed=9, offset=2)
        assert torch.equal(dx, m) and torch.equal(dz, ones)


def test_row_operators_on_another_stream_and_in_a_replayed_graph():
    x, res, dy = (rnd(300, 264, seed=s).bfloat16().to(DEV) for s in (1, 2, 3))
    gamma = (1 + 0.2 * rnd(264, seed=4)).to(DEV)

    def step():
        d = ops.dropout(x, 0.3, 5, 1)
        y, z, stats = ops.layer_norm(d, gamma, residual=res, p=0.1, seed=5, offset=2)
        return (d, y, z, stats) + ops.layer_norm_bwd(dy, z, stats, gamma, p=0.1, seed=5, offset=2)

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        x.copy_(rnd(300, 264, seed=10 + k).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager)), f"replay {k}"


def test_wrappers_refuse():
    x = torch.zeros(4, 128, device=DEV)
    bad = [lambda: ops.dropout(x.double(), 0.1, 1), lambda: ops.dropout(x, 1.5, 1), lambda: ops.dropout(x, 0.1, -1),
           lambda: ops.dropout(x, 0.1, 1, out=torch.zeros(4, 127, device=DEV)),
           lambda: ops.dropout(x, 0.1, 1, out=torch.zeros(4, 128, device=DEV, dtype=torch.bfloat16)),
           lambda: ops.layer_norm(x, gamma=torch.ones(127, device=DEV)),
           lambda: ops.layer_norm(x, gamma=torch.ones(128, device=DEV).bfloat16()),
           lambda: ops.layer_norm(x, residual=x.bfloat16()), lambda: ops.layer_norm(torch.zeros(2, 16385, device=DEV)),
           lambda: ops.layer_norm(torch.zeros(2, 0, device=DEV)), lambda: ops.layer_norm(x, eps=-1.0),
           lambda: ops.layer_norm_bwd(x, x, torch.zeros(4, 3, device=DEV)),
           lambda: ops.layer_norm_bwd(x, x[:3], torch.zeros(4, 2, device=DEV)),
           lambda: ops.layer_norm_bwd(x, x, torch.zeros(4, 2, device=DEV), dgamma=torch.zeros(128, device=DEV))]
    for i, call in enumerate(bad):
        with pytest.raises(L.MMSTError):
            call()
            print("not refused:", i)
