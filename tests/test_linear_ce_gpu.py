"""Linear layer + softmax cross entropy over a large vocabulary against 64-bit arithmetic on the same bf16 inputs.

Tolerances count roundings (u = 2^-24, half = finfo(bf16).eps / 2 = 2^-8).  A logit is a sum of D products in fp32,
in any order: at most D u sum |h w| off, plus the bias's addition; call the worst of a row E.  The exponent differences
carry two more roundings of the row's largest magnitude M, so a probability is off by the factor exp(2 E + 4 u M + 8 u)
(exp2's and the sums' own roundings: each term's at most V / 16 + 300 partial sums are bounded by u * that many), and lse by
E + that.  The gradient of the logits is rounded to bf16 once (twice where it is made from the exponentials of a tile, which are
kept in 16 bits of their own, 2^-10): within 2 half each term, and products of N (dw) or V (dh) such terms in fp32."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from multimodalspectraltransformer_amd import _lib as L
    from multimodalspectraltransformer_amd import ops

DEV = "cuda"
U = 2.0 ** -24
HALF = torch.finfo(torch.bfloat16).eps / 2
IGN = -100


def make(n, d, v, seed=0, ignored=0, bias=True, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(n, d, generator=g).bfloat16()
    w = (torch.randn(v, d, generator=g) * (scale / d ** 0.5)).bfloat16()
    b = 0.3 * torch.randn(v, generator=g) if bias else None
    t = torch.randint(0, v, (n,), generator=g)
    t[torch.randperm(n, generator=g)[:ignored]] = IGN
    dl = 0.5 + torch.rand(n, generator=g)
    return h, w, b, t, dl


def dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def oracle(h, w, b, t, dl):
    """64-bit values and the error bounds of the head comment"""
    n, d, v = h.shape[0], h.shape[1], w.shape[0]
    keep = (t != IGN) & (t >= 0) & (t < v)
    hd = torch.where(keep[:, None], h.double(), torch.zeros(1, dtype=torch.float64))
    wd = w.double()
    logits = hd @ wd.t() + (0 if b is None else b.double())
    mag = hd.abs() @ wd.abs().t() + (0 if b is None else torch.where(b > -1e30, b.double().abs(), torch.zeros(1, dtype=torch.float64)))
    e_row = (d + 1) * U * mag.amax(1)
    top = torch.where(logits > -1e30, logits.abs(), torch.zeros(1, dtype=torch.float64)).amax(1)
    rel = 2 * e_row + 4 * U * top + (v / 16 + 308) * U
    lse = torch.logsumexp(logits, 1)
    hot = torch.where(keep, t, torch.zeros_like(t))
    loss = lse - logits.gather(1, hot[:, None])[:, 0]
    loss = torch.where(lse == -float("inf"), torch.full_like(loss, float("inf")), loss)
    bad = ~keep & (t != IGN)
    zero, nan = torch.zeros_like(loss), torch.full_like(loss, float("nan"))
    dloss = e_row * 2 + rel + 2 * U * (top + lse.abs().nan_to_num(0, 0, 0))
    out = dict(loss=torch.where(keep, loss, torch.where(bad, nan, zero)), lse=torch.where(keep, lse, torch.where(bad, nan, zero)), dloss=dloss)
    if dl is None:
        return out
    p = torch.exp(logits - lse[:, None])
    ok = keep & (lse != -float("inf"))
    onehot = torch.zeros_like(p).scatter_(1, hot[:, None], 1.0)
    wt = torch.where(ok, dl.double(), torch.zeros(1, dtype=torch.float64))[:, None]
    p = torch.where(ok[:, None], p, torch.zeros(1, dtype=torch.float64))
    g = (p - onehot) * wt
    # 1.01: rounded values of values already off
    dg = 1.01 * ((p * (rel[:, None] + 3 * U + HALF) + U) * wt.abs() + g.abs() * (HALF + 2 * U))
    dg = torch.where(ok[:, None], dg, torch.zeros(1, dtype=torch.float64))
    out["dh"], out["dw"], out["db"] = g @ wd, g.t() @ hd, g.sum(0)
    out["ddh"] = dg @ wd.abs() + (v + 40) * U * (g.abs() @ wd.abs())
    out["ddw"] = dg.t() @ hd.abs() + (n + 8) * U * (g.abs().t() @ hd.abs())
    out["ddb"] = dg.sum(0) + (n + 8) * U * g.abs().sum(0)
    return out


def inside(got, want, tol, what):
    got = got.detach().cpu().double()
    bad = ~((got - want).abs() <= tol) & ~((got == want) | (got.isnan() & want.isnan()))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((got - want).abs().nan_to_num().max()):.3g} " \
                          f"(first at {bad.nonzero()[0].tolist()}: {float(got[tuple(bad.nonzero()[0])]):.6g} for " \
                          f"{float(want[tuple(bad.nonzero()[0])]):.6g})"


def check_loss(o, loss, lse):
    inside(lse, o["lse"], o["dloss"], "lse")
    inside(loss, o["loss"], o["dloss"], "loss")


def check_grad(o, dh, dw, db):
    inside(dh, o["dh"], o["ddh"] + o["dh"].abs() * HALF * 1.01, "dh")
    stored = HALF * 1.01 if dw.dtype == torch.bfloat16 else U
    inside(dw, o["dw"], o["ddw"] + o["dw"].abs() * stored, "dw")
    if db is not None:
        inside(db, o["db"], o["ddb"] + o["db"].abs() * stored, "dbias")


SIZES = [(1, 8, 1, 0), (1, 64, 43, 0), (3, 72, 7, 1), (64, 128, 43, 5), (129, 128, 1000, 40), (255, 256, 257, 0), (256, 64, 256, 255),
         (300, 200, 511, 300), (257, 8, 2049, 100), (1000, 128, 3001, 0), (70, 1032, 12345, 11), (520, 96, 4096, 1)]


@pytest.mark.parametrize("n,d,v,ignored", SIZES)
@pytest.mark.parametrize("bias", [False, True])
def test_loss(n, d, v, ignored, bias):
    h, w, b, t, _ = make(n, d, v, seed=n, ignored=ignored, bias=bias)
    loss, lse = ops.linear_ce(*dev(h, w, t), bias=dev(b)[0])
    check_loss(oracle(h, w, b, t, None), loss, lse)


@pytest.mark.parametrize("n,d,v,ignored", SIZES)
@pytest.mark.parametrize("bias", [False, True])
def test_gradients(n, d, v, ignored, bias):
    h, w, b, t, dl = make(n, d, v, seed=n, ignored=ignored, bias=bias)
    loss, lse, dh, dw, db = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    o = oracle(h, w, b, t, dl)
    check_loss(o, loss, lse)
    check_grad(o, dh, dw, db)
    assert dw.dtype == torch.bfloat16 and (db is None) == (b is None)
    assert (dh.cpu()[t == IGN] == 0).all()


@pytest.mark.parametrize("n,d,v", [(600, 640, 33000), (4100, 264, 9000)])
def test_gradients_of_many_tiles(n, d, v):
    """Enough tiles for the large ones, and a split contraction of dh."""
    h, w, b, t, dl = make(n, d, v, seed=1, ignored=n // 7)
    loss, lse, dh, dw, db = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    o = oracle(h, w, b, t, dl)
    check_loss(o, loss, lse)
    check_grad(o, dh, dw, db)
    l2, s2 = ops.linear_ce(*dev(h, w, t), bias=dev(b)[0])
    check_loss(o, l2, s2)


@pytest.mark.parametrize("rows", [1, 256, 300, 700, 5000])
@pytest.mark.parametrize("f32", [False, True])
def test_pieces_and_accumulation(rows, f32):
    h, w, b, t, dl = make(1100, 136, 1500, seed=3, ignored=200)
    o = oracle(h, w, b, t, dl * 0.25)
    kw = {}
    if f32:
        g = torch.Generator().manual_seed(9)
        base = torch.randn(1500, 136, generator=g), torch.randn(1500, generator=g)
        kw = dict(dw=base[0].to(DEV), dbias=base[1].to(DEV))
        o["dw"], o["db"] = o["dw"] + base[0].double(), o["db"] + base[1].double()
        o["ddw"], o["ddb"] = o["ddw"] + 8 * U * base[0].abs(), o["ddb"] + 8 * U * base[1].abs()
    loss, lse, dh, dw, db = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0], grad_scale=0.25, rows_per_piece=rows, **kw)
    check_loss(o, loss, lse)
    check_grad(o, dh, dw, db)
    if f32:
        assert dw is kw["dw"] and db is kw["dbias"]


def test_equal_calls_give_equal_bits():
    h, w, b, t, dl = make(900, 512, 20000, seed=5, ignored=100)
    first = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    again = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    assert all(torch.equal(x, y) for x, y in zip(first, again))


def test_what_padding_holds_reaches_nothing():
    h, w, b, t, dl = make(400, 128, 2000, seed=6, ignored=150)
    clean = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    pad = t == IGN
    h2, dl2 = h.clone(), dl.clone()
    h2[pad] = float("nan")
    h2[pad.nonzero()[0]] = float("inf")
    dl2[pad] = float("nan")
    dirty = ops.linear_ce_grad(*dev(h2, w, t), bias=dev(b)[0], dloss=dev(dl2)[0])
    assert all(torch.equal(x, y) for x, y in zip(clean, dirty))
    loss, lse = ops.linear_ce(*dev(h2, w, t), bias=dev(b)[0])
    assert (loss.cpu()[pad] == 0).all() and (lse.cpu()[pad] == 0).all()
    check_loss(oracle(h, w, b, t, None), loss, lse)


def test_every_row_ignored_and_no_rows():
    h, w, b, t, _ = make(70, 64, 300, seed=6, ignored=70)
    loss, lse, dh, dw, db = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0])
    assert all((x == 0).all() for x in (loss, lse, dh, dw, db))
    e = [x[:0] for x in dev(h, t)]
    loss, lse, dh, dw, db = ops.linear_ce_grad(e[0], dev(w)[0], e[1], bias=dev(b)[0])
    assert loss.shape == (0,) and dh.shape == (0, 64) and (dw == 0).all() and (db == 0).all()
    assert ops.linear_ce(e[0], dev(w)[0], e[1])[0].shape == (0,)
    acc = torch.ones(300, 64, device=DEV)
    ops.linear_ce_grad(e[0], dev(w)[0], e[1], dw=acc)
    assert (acc == 1).all()


@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float32).min])
def test_masked_words(low):
    """A bias that masks words, among them whole tiles of the vocabulary: no probability and no gradient there."""
    h, w, b, t, dl = make(200, 128, 3000, seed=7)
    b[600:2000] = low
    b[2500:] = low
    t = t % 600
    o = oracle(h, w, b, t, dl)
    loss, lse, dh, dw, db = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    check_loss(o, loss, lse)
    check_grad(o, dh, dw, db)
    assert (dw[600:2000] == 0).all() and (db[2500:] == 0).all()
    check_loss(o, *ops.linear_ce(*dev(h, w, t), bias=dev(b)[0]))


def test_rows_whose_mask_leaves_nothing():
    h, w, b, t, dl = make(100, 64, 700, seed=8)
    b[:] = float("-inf")
    for loss, lse in (ops.linear_ce(*dev(h, w, t), bias=dev(b)[0]), ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0])[:2]):
        assert (loss == float("inf")).all() and (lse == float("-inf")).all()
    _, _, dh, dw, db = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    assert (dh == 0).all() and (dw == 0).all() and (db == 0).all()
    b[:] = torch.finfo(torch.float32).min   # everything at the lowest value: the words are equally likely
    loss, lse = ops.linear_ce(*dev(h, w, t), bias=dev(b)[0])
    assert (lse <= 0).all() and torch.isfinite(loss).all()


def test_a_masked_target_costs_infinity():
    h, w, b, t, dl = make(50, 64, 300, seed=9)
    b[17] = float("-inf")
    t[5] = 17
    o = oracle(h, w, b, t, dl)
    loss, lse, dh, dw, db = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    assert loss[5] == float("inf")
    check_loss(o, loss, lse)
    check_grad(o, dh, dw, db)


def test_targets_that_are_no_words():
    h, w, b, t, dl = make(300, 64, 500, seed=10, ignored=20)
    t[3], t[100], t[299] = 500, -1, 1 << 40
    o = oracle(h, w, b, t, dl)
    out = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    check_loss(o, *out[:2])
    check_grad(o, *out[2:])
    assert out[0][[3, 100, 299]].isnan().all() and (out[2][[3, 100, 299]] == 0).all()
    check_loss(o, *ops.linear_ce(*dev(h, w, t), bias=dev(b)[0]))
    # an ignore_index that is a word ignores that word
    t2 = t.clamp(0, 499)
    t2[::3] = 42
    loss, _ = ops.linear_ce(*dev(h, w, t2), ignore_index=42)
    assert (loss.cpu()[t2 == 42] == 0).all() and (loss.cpu()[t2 != 42] > 0).all()


def test_bad_rows_poison_what_they_touch():
    h, w, b, t, dl = make(300, 64, 500, seed=11)
    h[7, 3] = float("nan")
    loss, lse, dh, dw, db = (x.cpu() for x in ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0]))
    rest = torch.arange(300) != 7
    assert loss[7].isnan() and dh[7].isnan().all() and torch.isfinite(loss[rest]).all() and torch.isfinite(dh[rest]).all()
    assert dw.isnan().all()


def test_confident_rows_keep_small_gradients():
    """A target of probability near 1: g = p - 1 is small, and as exact as the bounds say relative to p, not to 1 - p only
    where p itself is not the tile's largest."""
    h, w, _, t, dl = make(128, 64, 1000, seed=12, bias=False, scale=0.5)
    t = torch.arange(128)
    w[:128] = (h.float() * 0.15).bfloat16()
    o = oracle(h, w, None, t, dl)
    assert float(o["loss"].min()) < 0.05
    loss, lse, dh, dw, _ = ops.linear_ce_grad(*dev(h, w, t), dloss=dev(dl)[0])
    check_loss(o, loss, lse)
    check_grad(o, dh, dw, None)


@pytest.mark.parametrize("pad,lead", [(8, 0), (3, 0), (8, 8), (8, 1)])
def test_strides_and_alignment(pad, lead):
    h, w, b, t, dl = make(150, 72, 600, seed=13, ignored=10)
    o = oracle(h, w, b, t, dl)

    def wide(x):
        y = torch.full((x.shape[0], x.shape[1] + pad + lead), float("nan"), dtype=x.dtype, device=DEV)
        y[:, lead:lead + x.shape[1]] = x.to(DEV)
        return y[:, lead:lead + x.shape[1]]
    t2 = torch.stack([t, t], 1).to(DEV)[:, 0]
    out = ops.linear_ce_grad(wide(h), wide(w), t2, bias=dev(b)[0], dloss=dev(dl)[0])
    check_loss(o, *out[:2])
    check_grad(o, *out[2:])
    check_loss(o, *ops.linear_ce(wide(h), wide(w), t2, bias=dev(b)[0]))


def test_gradients_against_differences():
    """Central differences of the 64-bit loss, step 1e-5 (error below 1e-8); the kernels' bf16 results are off by their own
    bounds."""
    h, w, b, t, dl = make(5, 16, 11, seed=14, ignored=1)
    out = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    keep = t != IGN
    args = [h.double(), w.double(), b.double()]

    def loss(h, w, b):
        z = h @ w.t() + b
        l = torch.logsumexp(z, 1) - z.gather(1, t.clamp(min=0)[:, None])[:, 0]
        return (l * dl.double())[keep].sum()
    o = oracle(h, w, b, t, dl)
    for i, (got, key) in enumerate(((out[2], "ddh"), (out[3], "ddw"), (out[4], "ddb"))):
        num = torch.zeros_like(args[i])
        for k in range(num.numel()):
            hi, lo = [a.clone() for a in args], [a.clone() for a in args]
            hi[i].view(-1)[k] += 1e-5
            lo[i].view(-1)[k] -= 1e-5
            num.view(-1)[k] = (loss(*hi) - loss(*lo)) / 2e-5
        inside(got, num, o[key] + num.abs() * HALF * 1.01 + 1e-8, f"argument {i}")


def test_another_stream_and_a_replayed_graph():
    h, w, b, t, dl = dev(*make(300, 136, 3000, seed=15, ignored=30))

    def step():
        return ops.linear_ce_grad(h, w, t, bias=b, dloss=dl) + ops.linear_ce(h, w, t, bias=b)
    want = [x.clone() for x in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        h2, _, _, t2, _ = make(300, 136, 3000, seed=20 + k, ignored=60 * k)
        h.copy_(h2)
        t.copy_(t2)
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(x, y) for x, y in zip(captured, eager)), f"replay {k}"


def test_gradient_of_logits_past_32_bits():
    """A piece of more than 2^32 bytes (and elements past 2^31) of the logits' gradient: the last rows and words by value."""
    n, d, v = 17408, 8, 131073
    g = torch.Generator(device=DEV).manual_seed(1)
    h = torch.randn(n, d, device=DEV, generator=g).bfloat16()
    w = torch.randn(v, d, device=DEV, generator=g).bfloat16()
    t = torch.randint(0, v, (n,), device=DEV, generator=g)
    t[-1] = v - 1
    loss, lse, dh, dw, _ = ops.linear_ce_grad(h, w, t, rows_per_piece=n)
    pick = [0, 1, n // 2, n - 2, n - 1]
    o = oracle(h[pick].cpu(), w.cpu(), None, t[pick].cpu(), torch.ones(len(pick)))
    check_loss(o, loss[pick], lse[pick])
    inside(dh[pick], o["dh"], o["ddh"] + o["dh"].abs() * HALF * 1.01, "dh")
    lo = v - 3   # dw of the last words: g of every row there
    z = h.double() @ w[lo:].double().t()
    p = torch.exp(z - lse.double()[:, None]).cpu()
    tail = p - torch.nn.functional.one_hot((t - lo).clamp(min=-1).cpu() + 1, v - lo + 1)[:, 1:].double()
    want = tail.t() @ h.double().cpu()
    tol = (p * (HALF * 2 + 1e-5) + tail.abs() * HALF).t() @ h.double().abs().cpu()
    inside(dw[lo:], want, tol * 1.01 + want.abs() * HALF * 1.01, "dw")
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,v", [(70001, 43), (66000, 128), (66000, 129)])
def test_loss_of_few_words_over_many_rows(n, v):
    """More tiles of rows than workgroups; a bias and weights of the loss that start at any float."""
    h, w, b, t, dl = make(n, 64, v, seed=n + v, ignored=n // 9)
    t[5], t[n - 1] = v, -3
    b[1] = float("-inf")
    t[7] = 1
    o = oracle(h, w, b, t, dl)
    b1, dl1 = torch.empty(v + 1, device=DEV), torch.empty(n + 1, device=DEV)
    b1[1:], dl1[1:] = b.to(DEV), dl.to(DEV)
    check_loss(o, *ops.linear_ce(*dev(h, w, t), bias=b1[1:]))
    out = ops.linear_ce_grad(*dev(h, w, t), bias=b1[1:], dloss=dl1[1:])
    check_loss(o, *out[:2])
    check_grad(o, *out[2:])


def test_loss_whose_pairs_need_pieces():
    """More than 2^30 bytes of (maximum, sum) pairs: rows on both sides of the cut, and the last ones, by value."""
    n, d, v = 8192 + 300, 136, 1 << 20
    g = torch.Generator(device=DEV).manual_seed(2)
    h = torch.randn(n, d, device=DEV, generator=g).bfloat16()
    w = (0.1 * torch.randn(v, d, device=DEV, generator=g)).bfloat16()
    t = torch.randint(0, v, (n,), device=DEV, generator=g)
    t[8190] = IGN
    loss, lse = ops.linear_ce(h, w, t)
    pick = [0, 8189, 8190, 8191, 8192, 8193, n - 1]
    o = oracle(h[pick].cpu(), w.cpu(), None, t[pick].cpu(), None)
    check_loss(o, loss[pick], lse[pick])
    assert torch.isfinite(loss).all() and int((loss == 0).sum()) == 1


@pytest.mark.parametrize("n,d,v,ignored", [(1000, 128, 20001, 77), (1300, 40, 13000, 5), (140, 128, 70001, 0), (66000, 64, 300, 9), (33100, 8, 513, 33000)])
def test_narrow_layers_as_a_stream(n, d, v, ignored):
    """More than two tiles per workgroup, one part of the vocabulary or eight: masked words, targets that are none, padding."""
    h, w, b, t, dl = make(n, d, v, seed=n + 1, ignored=ignored)
    b[v // 3:v // 2] = float("-inf")
    b[v - 2] = torch.finfo(torch.float32).min
    t[t >= 0] = t[t >= 0] % (v // 3)
    t[11], t[n - 2], t[n // 2] = -1, v, 1 << 33
    h[(t == IGN).nonzero()[:1, 0]] = float("nan")
    o = oracle(h, w, b, t, dl)
    loss, lse, dh, dw, db = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    check_loss(o, loss, lse)
    check_grad(o, dh, dw, db)
    assert (dh[(t == IGN).to(DEV)] == 0).all() and (dw[v // 3:v // 2] == 0).all()
    check_loss(o, *ops.linear_ce(*dev(h, w, t), bias=dev(b)[0]))
    o = oracle(h, w, None, t, dl)
    out = ops.linear_ce_grad(*dev(h, w, t), dloss=dev(dl)[0])
    check_loss(o, *out[:2])
    check_grad(o, *out[2:])
    check_loss(o, *ops.linear_ce(*dev(h, w, t)))


@pytest.mark.parametrize("n,d,v", [(300, 512, 32000), (1024, 136, 16000), (2100, 520, 6000), (4100, 136, 7000), (3000, 264, 40)])
def test_every_tile_size_and_split(n, d, v):
    """Large tiles of dw; of the logits, one round; of the logits and of dh, split; two rounds; dw split over the rows."""
    h, w, b, t, dl = make(n, d, v, seed=n + v, ignored=n // 5)
    b[v // 2] = float("-inf")
    o = oracle(h, w, b, t, dl)
    out = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    check_loss(o, *out[:2])
    check_grad(o, *out[2:])
    again = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    assert all(torch.equal(x, y) for x, y in zip(out, again))
    check_loss(o, *ops.linear_ce(*dev(h, w, t), bias=dev(b)[0]))
    f32 = torch.ones(v, d, device=DEV), torch.ones(v, device=DEV)
    ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0], dw=f32[0], dbias=f32[1])
    inside(f32[0] - 1, o["dw"], o["ddw"] + 8 * U * (1 + o["dw"].abs()), "dw added to")
    inside(f32[1] - 1, o["db"], o["ddb"] + 8 * U * (1 + o["db"].abs()), "dbias added to")


@pytest.mark.parametrize("low", [-2.0 ** 14, -1e9, -1e10, -1e30, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("n,d,v", [(200, 128, 3000), (140, 64, 70001), (300, 200, 2100), (150, 64, 100)])
def test_masks_of_large_finite_numbers(n, d, v, low):
    """Words masked by a low finite bias, whole tiles of them."""
    h, w, b, t, dl = make(n, d, v, seed=n)
    b[v // 4:] = low
    t = t % (v // 4)
    o = oracle(h, w, b, t, dl)
    loss, lse, dh, dw, db = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    # the oracle's bound of the whole row counts the mask's magnitude, which reaches nothing: that of the unmasked words
    u = oracle(h, w[:v // 4], b[:v // 4], t, dl)
    check_loss(dict(loss=o["loss"], lse=o["lse"], dloss=u["dloss"] + v * U), loss, lse)
    inside(dh, u["dh"], u["ddh"] + u["dh"].abs() * HALF * 1.01, "dh")
    inside(dw[:v // 4], u["dw"], u["ddw"] + u["dw"].abs() * HALF * 1.01, "dw")
    assert (dw[v // 4:] == 0).all() and (db[v // 4:] == 0).all()
    check_loss(dict(loss=o["loss"], lse=o["lse"], dloss=u["dloss"] + v * U), *ops.linear_ce(*dev(h, w, t), bias=dev(b)[0]))


@pytest.mark.parametrize("n,d,v", [(200, 128, 3000), (140, 64, 70001), (300, 200, 2100), (150, 64, 100)])
@pytest.mark.parametrize("low", [-2.0 ** 40, 2.0 ** 40, -1e30, torch.finfo(torch.float32).min])
def test_rows_of_nothing_but_a_large_finite_mask(n, d, v, low):
    """low + l is low in fp32 for every word (|l| < 2^10, half a step of 2^40 is 2^16): equally likely words, so loss log v
    and g = dloss (1 / v - [target]).  The loss is off by log's and the sum's rounding, g by bf16's and those."""
    h, w, b, t, dl = make(n, d, v, seed=n)
    b[:] = low
    loss, lse, dh, dw, db = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    rel = (v / 16 + 308) * U
    want = torch.full((n,), float(torch.tensor(v, dtype=torch.float64).log()), dtype=torch.float64)
    for x in (loss, ops.linear_ce(*dev(h, w, t), bias=dev(b)[0])[0]):
        inside(x, want, want * 0 + rel + 4 * U * want, "loss")
    inside(lse, want * 0 + low, want * 0 + abs(low) * U * 2, "lse")
    hd, wd, wt = h.double(), w.double(), dl.double()[:, None]
    p = torch.full((n, v), 1.0 / v, dtype=torch.float64)
    g = (p - torch.nn.functional.one_hot(t, v)) * wt
    dg = 1.01 * (p * (rel + HALF + 3 * U) * wt + g.abs() * (HALF + 2 * U))
    o = dict(dh=g @ wd, dw=g.t() @ hd, db=g.sum(0), ddh=dg @ wd.abs() + (v + 40) * U * (g.abs() @ wd.abs()),
             ddw=dg.t() @ hd.abs() + (n + 8) * U * (g.abs().t() @ hd.abs()), ddb=dg.sum(0) + (n + 8) * U * g.abs().sum(0))
    check_grad(o, dh, dw, db)


def test_tiles_keep_more_than_bf16_of_a_probability():
    """dbias of words that are no row's target is a sum of probabilities.  A rounding to bf16 has steps of 2^-7 of a number's
    power of two: its relative error has the standard deviation 2^-7 / sqrt(12) times the root of the mean of 1 / x^2 over x in
    [1, 2) (mantissas spread over their logarithm: 3 / (8 log 2)), 0.00166; the one to 9 bits before it a quarter of that.
    Together 0.00171, of the root of the sum of p^2; over 990 words the mean of that has a deviation of 1 / sqrt(2 * 990) =
    2.2 %, five of which leave it below 0.0019.  (Two roundings to bf16 would be at 0.00235.)"""
    n, d, v = 2000, 136, 1000
    h, w, b, t, _ = make(n, d, v, seed=31)
    t = t % 10
    s = torch.zeros(v, device=DEV)
    ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dw=torch.zeros(v, d, device=DEV), dbias=s)
    p = torch.softmax(h.double() @ w.double().t() + b.double(), 1)[:, 10:]
    off = (s.cpu().double()[10:] - p.sum(0)) / p.pow(2).sum(0).sqrt()
    assert float(off.pow(2).mean().sqrt()) < 0.0019


@pytest.mark.parametrize("n,d,v", [(333, 136, 5000), (3000, 128, 8000)])
@pytest.mark.parametrize("weights", ["dloss", "scale"])
def test_equal_weights_are_not_rounded(n, d, v, weights):
    """The mean's 1 / n, whose nearest bf16 number is up to 2^-8 off: sums of g would all be.  dbias summed over the words that
    are targets, each of probability below 2^-9, is minus the weights' sum and what their probabilities add: g of a target is
    off by at most 2^-9 of it (the step below 1 is 2^-8) and by its probability where that rounds away."""
    h, w, b, t, _ = make(n, d, v, seed=41, scale=0.5)
    s = torch.zeros(v, device=DEV)
    kw = dict(dloss=torch.full((n,), 1 / n, device=DEV)) if weights == "dloss" else dict(grad_scale=1 / n)
    dh = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dw=torch.zeros(v, d, device=DEV), dbias=s, **kw)[2]
    p = torch.softmax(h.double() @ w.double().t() + b.double(), 1)
    g = (p - torch.nn.functional.one_hot(t, v)) / n
    pt = p.gather(1, t[:, None])
    assert float(pt.max()) < 2.0 ** -9
    hot = torch.zeros(v, dtype=torch.bool)
    hot[t] = True
    off = abs(float(s.cpu().double()[hot].sum() - g.sum(0)[hot].sum()))
    assert off <= float(pt.mean()) * 1.01 + 2.0 ** -8 * float(p[:, hot].sum()) / n + 1e-5
    # and without a weight the same bits of g: dh is that times the weight, rounded once more
    one = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0])[2].cpu().double() / n
    inside(dh, one, one.abs() * 2.02 * HALF, "dh")


@pytest.mark.parametrize("n,d,v", [(64, 136, 500), (1000, 64, 20001)])
def test_weights_of_every_kind(n, d, v):
    """Zeros, negative ones, and one of infinity or NaN, which stays with its row (and the words, all of which it reaches)."""
    h, w, b, t, dl = make(n, d, v, seed=43, ignored=n // 8)
    dl[::3] = 0
    dl[1::3] *= -1e-3
    o = oracle(h, w, b, t, dl)
    check_grad(o, *ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])[2:])
    zero = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=torch.zeros(n, device=DEV))
    assert all((x == 0).all() for x in zero[2:])
    k = int((t != IGN).nonzero()[2, 0])
    for bad in (float("nan"), float("inf")):
        dl2 = dl.clone()
        dl2[k] = bad
        dh = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl2)[0])[2].cpu()
        rest = torch.arange(n) != k
        inside(dh[rest], o["dh"][rest], (o["ddh"] + o["dh"].abs() * HALF * 1.01)[rest], "dh")
        assert not torch.isfinite(dh[k]).any()


def test_an_expanded_gradient_of_the_loss():
    """What autograd hands back for a mean: one number with a stride of 0."""
    h, w, b, t, _ = make(150, 64, 700, seed=44, ignored=9)
    want = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=torch.full((150,), 0.125, device=DEV))
    got = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=torch.tensor(0.125, device=DEV).expand(150))
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("n,d,v", [(333, 136, 50001), (300, 200, 50000)])
def test_loss_of_wide_tiles(n, d, v):
    """Tiles of 160 words: targets in every part of them, masked words, an odd end."""
    h, w, b, t, _ = make(n, d, v, seed=n, ignored=n // 10)
    b[:170] = float("-inf")
    b[v // 2] = torch.finfo(torch.float32).min
    t[t >= 0] = t[t >= 0].clamp(min=170)
    t[:160] = 10400 + torch.arange(160)   # every column of a tile
    t[200], t[201] = v, v - 1
    o = oracle(h, w, b, t, None)
    check_loss(o, *ops.linear_ce(*dev(h, w, t), bias=dev(b)[0]))
    check_loss(oracle(h, w, None, t, None), *ops.linear_ce(*dev(h, w, t)))


@pytest.mark.parametrize("n,d,v", [(3, 32768, 70), (2, 8, 1 << 22), (2, 1032, 1 << 18), (1, 8, 1)])
def test_largest_widths_and_vocabularies(n, d, v):
    h, w, b, t, dl = make(n, d, v, seed=45)
    t[-1] = v - 1
    o = oracle(h, w, b, t, dl)
    out = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    check_loss(o, *out[:2])
    check_grad(o, *out[2:])
    check_loss(o, *ops.linear_ce(*dev(h, w, t), bias=dev(b)[0]))


def test_the_most_rows():
    """2^24 rows, in two pieces: first and last ones by value, every row's loss against the sum of its equal copies."""
    n, d, v = 1 << 24, 8, 5
    h, w, b, t, _ = make(1 << 10, d, v, seed=46, ignored=100)
    many = n >> 10
    o = oracle(h, w, b, t, torch.ones(1 << 10))
    hd, td = h.to(DEV).repeat(many, 1), t.to(DEV).repeat(many)
    s = torch.zeros(v, d, device=DEV), torch.zeros(v, device=DEV)
    loss, lse, dh, _, _ = ops.linear_ce_grad(hd, w.to(DEV), td, bias=b.to(DEV), dw=s[0], dbias=s[1])
    for rows in (slice(0, 1 << 10), slice(n - (1 << 10), n)):
        check_loss(o, loss[rows], lse[rows])
        inside(dh[rows], o["dh"], o["ddh"] + o["dh"].abs() * HALF * 1.01, "dh")
    assert torch.equal(loss.view(many, -1), loss[:1 << 10].expand(many, -1))
    assert torch.equal(dh.view(many, -1), dh[:1 << 10].reshape(-1).expand(many, -1))
    # a piece of 2^23 rows is summed in 32 parts: at most 2^18 roundings in a row, each of the magnitudes' sum
    z = h.double() @ w.double().t() + b.double()
    g = ((torch.softmax(z, 1) - torch.nn.functional.one_hot(t.clamp(min=0), v)) * (t != IGN)[:, None]).abs()
    inside(s[1] / many, o["db"], o["ddb"] + (2 ** 18 + 100) * U * g.sum(0), "dbias")
    check_loss(o, *(x[-(1 << 10):] for x in ops.linear_ce(hd, w.to(DEV), td, bias=b.to(DEV))))
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,d,v", [(70, 1032, 45), (200, 4096, 1001), (1, 2000, 300), (130, 1024, 129), (16, 2048, 8003), (600, 8192, 7)])
def test_logits_in_parts_of_a_long_contraction(n, d, v):
    h, w, b, t, dl = make(n, d, v, seed=n + d, ignored=n // 6)
    if v > 40:
        b[v // 3:v // 3 + 20], b[v - 1] = float("-inf"), -1e30
        t[t >= 0] %= v // 3
    if n > 60:
        t[3], t[50] = v, -7
        h[(t == IGN).nonzero()[0, 0]] = float("nan")
    # the oracle's bound counts the mask's magnitude, which reaches nothing
    b2 = torch.where(b < -1e20, torch.full_like(b, float("-inf")), b)
    o = oracle(h, w, b2, t, dl)
    out = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    check_loss(o, *out[:2])
    check_grad(o, *out[2:])
    check_loss(o, *ops.linear_ce(*dev(h, w, t), bias=dev(b)[0]))
    again = ops.linear_ce_grad(*dev(h, w, t), bias=dev(b)[0], dloss=dev(dl)[0])
    assert all(torch.equal(x, y) or x.isnan().any() for x, y in zip(out, again))
    none = torch.full((v,), float("-inf"))
    out = ops.linear_ce_grad(*dev(h, w, t), bias=dev(none)[0])
    keep = ((t >= 0) & (t < v)).to(DEV)
    assert (out[1][keep] == float("-inf")).all() and (out[2] == 0).all() and (out[3] == 0).all()


def test_wrappers_refuse():
    h, w, b, t, dl = dev(*make(20, 64, 100))
    bad = [lambda: ops.linear_ce(h.float(), w, t), lambda: ops.linear_ce(h, w.half(), t), lambda: ops.linear_ce(h, w, t.int()),
           lambda: ops.linear_ce(h[:, :60], w[:, :60], t), lambda: ops.linear_ce(h, w[:, :32], t), lambda: ops.linear_ce(h, w, t[:5]),
           lambda: ops.linear_ce(h, w, t, bias=b.bfloat16()), lambda: ops.linear_ce(h, w, t, bias=b[:50]), lambda: ops.linear_ce(h[0], w, t),
           lambda: ops.linear_ce(h, w[:0], t), lambda: ops.linear_ce_grad(h, w, t, dloss=dl[:3]),
           lambda: ops.linear_ce_grad(h, w, t, dw=torch.zeros(100, 64, device=DEV).bfloat16()),
           lambda: ops.linear_ce_grad(h, w, t, dw=torch.zeros(100, 63, device=DEV)),
           lambda: ops.linear_ce_grad(h, w, t, bias=b, dw=torch.zeros(100, 64, device=DEV)),
           lambda: ops.linear_ce_grad(h, w, t, dbias=b), lambda: ops.linear_ce_grad(h, w, t, rows_per_piece=-1),
           lambda: ops.linear_ce_grad(h, w, t, rows_per_piece=1 << 32),
           lambda: ops.linear_ce(h[:1].expand((1 << 32) + 20, 64), w, t[:1].expand((1 << 32) + 20))]
    for i, call in enumerate(bad):
        with pytest.raises(L.MMSTError):
            call()
            print("not refused:", i)
