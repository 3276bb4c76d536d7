"""The row operators and the linear layer with cross entropy in one run, as the end of a decoder uses them:

    x = dropout(e)    y = layer_norm(residual + dropout(x))    loss = cross entropy of y w^T + bias

and back to e, the residual, gamma, beta, w and bias, against 64-bit arithmetic on the same inputs.

Between the operators tensors are rounded to bf16 (x, y, z, dh, dz, dx): each by at most half = 2^-8 of the value.  The
bounds follow those roundings through the chain row by row in the Euclidean norm |.|, with rstd and gamma a row's own
(s: the factor 1 / (1 - p) of kept elements, L = max |gamma| rstd, k = 1.05 for products of two roundings and for what fp32
adds, which is below 2^-14 of any of them at these sizes):
  x off by half |x|, z by s half |x| (its own rounding, half |z|, matters to the backward pass only)
  y off by k L |dz_in| + half |y|: layer norm is Lipschitz in z with rstd max |gamma| (I minus two projections)
  g off by dl / 2 |dy| |w|_2 (the softmax is Lipschitz with 1/2), hence dh by that times |w|_2 more, and by its own
     operator's roundings: 2 half |p| |w|_2 dl for g (stored twice in bf16 on the way) and half |dh|
  dz = rstd (a - mean a - xhat mean(a xhat)), a = gamma dh: a's error passes without growing, times rstd; xhat, off by
     D = rstd (s half |x| + half |z|), adds rstd |a| (2 sqrt(C) D + D^2) / C; rstd itself is off by the factor 1 + rstd s
     half |x| / sqrt(C); the result's rounding adds half |dz|
  dx: s times that and half |dx|; de: s times that and half |de|
The loss is Lipschitz in y with sqrt(2) |w|_2.  Differences of the 64-bit loss along a direction are off by less than 1e-6
of it with steps of 1e-4."""
import pytest
import torch

from tests.philox_oracle import factor

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from multimodalspectraltransformer_amd import ops

DEV = "cuda"
HALF = torch.finfo(torch.bfloat16).eps / 2
K = 1.05
IGN = -100
P1, P2, S1, S2 = 0.125, 0.25, (11, 1), (12, 1 << 33)


def make(n, c, v, ignored, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    t = torch.randint(0, v, (n,), generator=g)
    t[torch.randperm(n, generator=g)[:ignored]] = IGN
    return dict(e=r(n, c).bfloat16(), residual=r(n, c).bfloat16(), gamma=1 + 0.1 * r(c), beta=0.1 * r(c),
                w=(r(v, c) / c ** 0.5).bfloat16(), bias=0.3 * r(v), t=t, dl=0.5 + torch.rand(n, generator=g))


def run(i):
    x = ops.dropout(i["e"], P1, *S1)
    y, z, stats = ops.layer_norm(x, i["gamma"], i["beta"], residual=i["residual"], p=P2, seed=S2[0], offset=S2[1])
    loss, lse, dh, dw, db = ops.linear_ce_grad(y, i["w"], i["t"], bias=i["bias"], dloss=i["dl"])
    dz, dx, dgamma, dbeta = ops.layer_norm_bwd(dh, y if z is None else z, stats, i["gamma"], p=P2, seed=S2[0], offset=S2[1])
    de = ops.dropout(dx, P1, *S1)
    return dict(loss=loss, e=de, residual=dz, gamma=dgamma, beta=dbeta, w=dw, bias=db)


class Reference:
    """The same in 64 bits, and how far the run may be off."""
    def __init__(self, i, eps=1e-5):
        self.i, self.eps = i, eps
        self.f1, self.f2 = factor(i["e"].shape, P1, *S1), factor(i["e"].shape, P2, *S2)
        self.keep = i["t"] != IGN
        self.v = {k: i[k].double().requires_grad_() for k in ("e", "residual", "gamma", "beta", "w", "bias")}

    def forward(self, e, residual, gamma, beta, w, bias):
        x = e * self.f1
        z = residual + x * self.f2
        mean, var = z.mean(1, keepdim=True), z.var(1, unbiased=False, keepdim=True)
        rstd = (var + self.eps).rsqrt()
        y = (z - mean) * rstd * gamma + beta
        logits = y @ w.t() + bias
        loss = torch.logsumexp(logits, 1) - logits.gather(1, self.i["t"].clamp(min=0)[:, None])[:, 0]
        return x, z, rstd, y, torch.where(self.keep, loss, torch.zeros_like(loss)), logits

    def total(self, **v):
        return (self.forward(**v)[4] * self.i["dl"].double()).sum()

    def solve(self):
        x, z, rstd, y, loss, logits = self.forward(**self.v)
        z.retain_grad(), y.retain_grad(), x.retain_grad()
        (loss * self.i["dl"].double()).sum().backward()
        d = lambda t: t.detach()
        norm = lambda t: d(t).norm(dim=1)
        c = y.shape[1]
        rstd, gmax = d(rstd)[:, 0], d(self.v["gamma"]).abs().max()
        w2 = torch.linalg.matrix_norm(d(self.v["w"]), 2)
        s1, s2 = 1 / (1 - P1), 1 / (1 - P2)
        dl = self.i["dl"].double() * self.keep
        off_z = s2 * HALF * norm(x)
        off_y = K * gmax * rstd * off_z + HALF * norm(y)
        p = torch.softmax(d(logits), 1).norm(dim=1) + 1 * self.keep   # g before the target's 1 and behind it
        off_dh = K * (dl * w2 * (off_y * w2 / 2 + 2 * HALF * p) + HALF * norm(y.grad))
        a, off_a = (d(self.v["gamma"]) * y.grad).norm(dim=1), gmax * off_dh
        off_x = rstd * (off_z + HALF * norm(z))
        off_dz = K * (rstd * (off_a + a * (2 * c ** 0.5 * off_x + off_x ** 2) / c + a * rstd * off_z / c ** 0.5) + HALF * norm(z.grad))
        off_dx = s2 * off_dz + HALF * norm(x.grad)
        off_de = s1 * K * off_dx + HALF * norm(self.v["e"].grad)
        self.loss, self.tol = d(loss), dict(loss=2 ** 0.5 * w2 * off_y * K, e=off_de, residual=off_dz)
        # sums over the rows: each row's error in one column is at most its norm
        xhat = (d(z) - d(z).mean(1, keepdim=True)) * rstd[:, None]
        self.tol["beta"] = off_dh.sum()
        self.tol["gamma"] = (off_dh * xhat.abs().amax(1) + y.grad.abs().amax(1) * K * off_x).sum()
        g = (torch.softmax(d(logits), 1) - torch.nn.functional.one_hot(self.i["t"].clamp(min=0), logits.shape[1])) * dl[:, None]
        off_g = dl * (off_y * w2 / 2 + 2 * HALF * p)
        self.tol["w"] = K * ((off_g * norm(y) + norm(g) * off_y).sum() + HALF * self.v["w"].grad.abs().max())
        self.tol["bias"] = K * (off_g.sum() + HALF * self.v["bias"].grad.abs().max())
        return self


def check(ref, got):
    got = {k: t.cpu().double() for k, t in got.items()}
    assert ((got["loss"] - ref.loss).abs() <= ref.tol["loss"] * ref.keep).all(), "loss"
    for k in ("e", "residual"):
        off = (got[k] - ref.v[k].grad).norm(dim=1)
        assert (off <= ref.tol[k]).all(), (k, float((off / ref.tol[k].clamp(min=1e-30)).max()))
        assert (got[k][~ref.keep] == 0).all(), k
    for k in ("gamma", "beta", "w", "bias"):
        off = (got[k] - ref.v[k].grad).abs().max()
        assert off <= ref.tol[k], (k, float(off / ref.tol[k]))


SHAPES = [(1, 8, 1, 0), (64, 128, 43, 9), (200, 128, 1000, 50), (131, 1000, 517, 0), (70, 256, 9000, 69)]


@pytest.mark.parametrize("n,c,v,ignored", SHAPES)
def test_a_run_forward_and_backward(n, c, v, ignored):
    i = make(n, c, v, ignored, seed=n)
    check(Reference(i).solve(), run({k: t.to(DEV) for k, t in i.items()}))


def test_a_runs_gradients_against_differences():
    i = make(40, 64, 90, 7, seed=3)
    ref = Reference(i).solve()
    got = {k: t.cpu().double() for k, t in run({k: t.to(DEV) for k, t in i.items()}).items()}
    v = {k: t.detach() for k, t in ref.v.items()}
    g = torch.Generator().manual_seed(4)
    for k in ("e", "residual", "gamma", "beta", "w", "bias"):
        step = torch.randn(v[k].shape, generator=g, dtype=torch.float64)
        num = (ref.total(**{**v, k: v[k] + 1e-4 * step}) - ref.total(**{**v, k: v[k] - 1e-4 * step})) / 2e-4
        tol = (ref.tol[k] * step.norm(dim=1)).sum() if k in ("e", "residual") else ref.tol[k] * step.abs().sum()
        assert abs((got[k] * step).sum() - num) <= tol + 1e-6 * ref.loss.sum(), k


def test_a_run_in_two_replayed_graphs():
    """Two captured runs, replayed in turn and with eager runs between them: each gives what the eager run does."""
    ins = [{k: t.to(DEV) for k, t in make(200, 128, 1000, 50, seed=s).items()} for s in (5, 6)]
    eager = [run(i) for i in ins]
    graphs = []
    for i in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(i)
        graphs.append((g, out))
    for k in range(6):
        for (g, out), want in zip(graphs, eager):
            g.replay()
            run(ins[k % 2])
            torch.cuda.synchronize()
            assert all(torch.equal(out[n], want[n]) for n in out), f"replay {k}"


def test_runs_on_two_streams_at_once():
    """Two runs enqueued in turn on streams of their own: nothing is shared between calls."""
    ins = [{k: t.to(DEV) for k, t in make(n, c, v, 20, seed=n).items()} for n, c, v in ((300, 128, 9000), (257, 1000, 517))]
    want = [run(i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = [[], []]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(run(ins[k]))
    torch.cuda.synchronize()
    for k, w in enumerate(want):
        assert all(torch.equal(g[n], w[n]) for g in got[k] for n in w)
