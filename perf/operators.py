"""The measured cases of the framework's wide-row operators: counter-based dropout, layer norm with residual and dropout
(forward and backward) and the linear layer with softmax cross entropy over a large vocabulary (loss, and loss with
gradients).  `own` selects the framework's entry points (multimodalspectraltransformer_amd.ops) or the plain forms: the
operators' formulas in elementary torch operations, 32-bit, rounded once."""
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5
IGNORE = -100


def listed():
    return [
        # one target position of 64 molecules: the rows a decoder step drops out (latency counts)
        dict(name="dropout 64x128", op="dropout", rows=64, cols=128, pad=0, dtype="bf16", p=0.1),
        # hidden activation of the feed-forward block, 64 molecules x 582 memory rows
        dict(name="dropout 37248x2048", op="dropout", rows=37248, cols=2048, pad=0, dtype="bf16", p=0.1),
        # fp32 rows cut out of a wider tensor, odd width
        dict(name="dropout 1023x4099 fp32 strided", op="dropout", rows=1023, cols=4099, pad=13, dtype="fp32", p=0.3),
        # post-norm sub-block of one target position of 64 molecules
        dict(name="ln fwd 64x128 res drop", op="ln_fwd", rows=64, cols=128, dtype="bf16", residual=True, p=0.1),
        # post-norm sub-block of the cross encoder's rows
        dict(name="ln fwd 37248x128 res drop", op="ln_fwd", rows=37248, cols=128, dtype="bf16", residual=True, p=0.1),
        # the same rows' backward pass
        dict(name="ln bwd 37248x128 drop", op="ln_bwd", rows=37248, cols=128, dtype="bf16", add=False, p=0.1),
        # plain layer norm of an odd width in fp16
        dict(name="ln fwd 4099x1003 fp16", op="ln_fwd", rows=4099, cols=1003, dtype="fp16", residual=False, p=0.0),
        # a wide pre-norm block's backward pass: the residual stream's gradient is added
        dict(name="ln bwd 8192x4096 add", op="ln_bwd", rows=8192, cols=4096, dtype="bf16", add=True, p=0.0),
        # teacher-forced loss of 64 molecules x 63 positions over the SMILES vocabulary
        dict(name="ce loss 4032x128x43", op="ce_loss", rows=4032, ignored=0, dim=128, vocab=43, bias=True),
        # scoring a few sequences over a large odd vocabulary
        dict(name="ce loss 333x1024x50001", op="ce_loss", rows=333, ignored=33, dim=1024, vocab=50001, bias=False),
        # training step of this width over a large vocabulary, padded batch
        dict(name="ce grad 4032x128x32000", op="ce_grad", rows=4032, ignored=1000, dim=128, vocab=32000, bias=True),
        # training step of a wide model
        dict(name="ce grad 8192x2048x65536", op="ce_grad", rows=8192, ignored=0, dim=2048, vocab=65536, bias=False),
    ]


def _log_int(rng, lo, hi):
    """An integer whose logarithm is uniform over [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["dropout", "ln_fwd", "ln_bwd", "ce_loss", "ce_grad"])
    if op == "dropout":
        cols = _log_int(rng, 1, 16384)
        rows = _log_int(rng, 1, max(1, min(65536, 37248 * 2048 // cols // 2)))
        return dict(op=op, rows=rows, cols=cols, pad=rng.choice([0, 0, 8, rng.randint(1, 40)]),
                    dtype=rng.choice(list(DTYPES)), p=rng.choice([0.0, 0.05, 0.1, 0.5, rng.random()]))
    if op in ("ln_fwd", "ln_bwd"):
        cols = _log_int(rng, 16, 16384)
        if rng.random() < 0.5:
            cols = max(16, cols // 8 * 8)
        rows = _log_int(rng, 1, max(1, min(65536, 8192 * 4096 // cols // 2)))
        c = dict(op=op, rows=rows, cols=cols, dtype=rng.choice(list(DTYPES)), p=rng.choice([0.0, 0.0, 0.1, rng.random() * 0.9]))
        c["residual" if op == "ln_fwd" else "add"] = rng.random() < 0.5
        return c
    dim = 8 * _log_int(rng, 4, 512)
    vocab = _log_int(rng, 43, 65536)
    most = int(min(16384, 8192 * 2048 * 65536 / dim / vocab / 2))
    rows = _log_int(rng, 1, max(1, most))
    return dict(op=op, rows=rows, ignored=rng.choice([0, rows // 5, rows // 2]), dim=dim, vocab=vocab, bias=rng.random() < 0.5)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = dict(case, seed=(seed * 0x9E3779B97F4A7C15 + 12345) % (1 << 63), offset=seed % 1000 + 1)
    if op == "dropout":
        t = DTYPES[case["dtype"]]
        wide = torch.randn(case["rows"], case["cols"] + case["pad"], device="cuda", generator=g).to(t)
        s["x"] = wide[:, :case["cols"]]
    elif op == "ln_fwd":
        t, shape = DTYPES[case["dtype"]], (case["rows"], case["cols"])
        s["x"] = (torch.randn(shape, device="cuda", generator=g) * 1.5 + 0.25).to(t)
        s["res"] = torch.randn(shape, device="cuda", generator=g).to(t) if case["residual"] else None
        s["gamma"] = 1 + 0.2 * torch.randn(case["cols"], device="cuda", generator=g)
        s["beta"] = 0.2 * torch.randn(case["cols"], device="cuda", generator=g)
    elif op == "ln_bwd":
        t, shape = DTYPES[case["dtype"]], (case["rows"], case["cols"])
        s["z"] = (torch.randn(shape, device="cuda", generator=g) * 1.5 + 0.25).to(t)
        s["dy"] = torch.randn(shape, device="cuda", generator=g).to(t)
        s["add"] = torch.randn(shape, device="cuda", generator=g).to(t) if case["add"] else None
        s["gamma"] = 1 + 0.2 * torch.randn(case["cols"], device="cuda", generator=g)
        var, mean = torch.var_mean(s["z"].double(), dim=1, correction=0)  # what the forward pass has kept
        s["stats"] = torch.stack([mean, (var + EPS).rsqrt()], dim=1).float()
    else:
        n, d, v = case["rows"], case["dim"], case["vocab"]
        s["h"] = torch.randn(n, d, device="cuda", generator=g).bfloat16()
        s["w"] = (torch.randn(v, d, device="cuda", generator=g) * (2.0 / d ** 0.5)).bfloat16()
        s["b"] = 0.1 * torch.randn(v, device="cuda", generator=g) if case["bias"] else None
        target = torch.randint(0, v, (n,), device="cuda", generator=g)
        target[torch.randperm(n, device="cuda", generator=g)[:case["ignored"]]] = IGNORE
        s["target"] = target
        # the mean over the rows that count, as a training step weighs them
        s["dloss"] = torch.full((n,), 1.0 / max(1, n - case["ignored"]), device="cuda")
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------
M32 = 0xFFFFFFFF
ROUND_KEYS = [((k * 0x9E3779B9) & M32, (k * 0xBB67AE85) & M32) for k in range(10)]


def _keep(shape, p, seed, offset):
    """The mask: element i of the tensor read row by row takes 16 bits of Philox4x32-10 (Salmon et al., 2011) of key
    `seed` and counter (i // 8, offset), and is kept where they are at least round(65536 p)."""
    rows, cols = shape
    n = rows * cols
    block = torch.arange((n + 7) // 8, device="cuda")
    c0, c1 = block & M32, block >> 32
    c2, c3 = torch.full_like(block, offset & M32), torch.full_like(block, offset >> 32)
    for a, b in ROUND_KEYS:
        k0, k1 = (a + seed) & M32, (b + (seed >> 32)) & M32
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64-bit products, their upper halves by an arithmetic shift and a mask
        c0, c1, c2, c3 = ((p1 >> 32) & M32) ^ c1 ^ k0, p1 & M32, ((p0 >> 32) & M32) ^ c3 ^ k1, p0 & M32
    words = torch.stack([c0, c1, c2, c3], dim=1)
    bits = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)[:n]
    return (bits >= int(p * 65536 + 0.5)).reshape(rows, cols)


def _scale(p):
    thr = int(p * 65536 + 0.5)
    return 65536.0 / (65536 - thr) if thr < 65536 else 0.0


def _dropped(x, s):
    return x if s["p"] == 0 else torch.where(_keep(x.shape, s["p"], s["seed"], s["offset"]), x * _scale(s["p"]), 0.0)


def _plain_ln_fwd(s):
    z = _dropped(s["x"].float(), s)
    if s["res"] is not None:
        z = s["res"].float() + z
    mean = z.mean(dim=1, keepdim=True)
    centred = z - mean
    rstd = (centred * centred).mean(dim=1, keepdim=True).add(EPS).rsqrt()
    y = centred * rstd * s["gamma"] + s["beta"]
    out = dict(y=y.to(s["x"].dtype), stats=torch.cat([mean, rstd], dim=1))
    if s["res"] is not None or s["p"] > 0:
        out["z"] = z.to(s["x"].dtype)
    return out


def _plain_ln_bwd(s):
    dy, mean, rstd = s["dy"].float(), s["stats"][:, :1], s["stats"][:, 1:]
    xh = (s["z"].float() - mean) * rstd
    q = dy * s["gamma"]
    dz = rstd * (q - q.mean(dim=1, keepdim=True) - xh * (q * xh).mean(dim=1, keepdim=True))
    if s["add"] is not None:
        dz = dz + s["add"].float()
    out = dict(dz=dz.to(s["dy"].dtype), dgamma=(dy * xh).sum(dim=0), dbeta=dy.sum(dim=0))
    if s["p"] > 0:
        out["dx"] = _dropped(dz, s).to(s["dy"].dtype)
    return out


def _plain_ce(s, grad):
    h, w = s["h"].float(), s["w"].float()
    logits = h @ w.t()
    if s["b"] is not None:
        logits = logits + s["b"]
    counts = s["target"] != IGNORE
    hot = torch.where(counts, s["target"], 0).unsqueeze(1)
    top = logits.amax(dim=1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(dim=1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(1)
    loss = torch.where(counts, lse - logits.gather(1, hot).squeeze(1), 0.0)
    lse = torch.where(counts, lse, 0.0)
    if not grad:
        return dict(loss=loss, lse=lse)
    weight = torch.where(counts, s["dloss"], 0.0).unsqueeze(1)
    g = e.mul_(weight / total)
    g.scatter_add_(1, hot, -weight)
    out = dict(loss=loss, lse=lse, dh=(g @ w).bfloat16(), dw=(g.t() @ h).bfloat16())
    if s["b"] is not None:
        out["dbias"] = g.sum(dim=0).bfloat16()
    return out


# ---- the framework's calls ------------------------------------------------------------------------------------------
def _own_ln_fwd(s):
    from multimodalspectraltransformer_amd import ops
    y, z, stats = ops.layer_norm(s["x"], s["gamma"], s["beta"], eps=EPS, residual=s["res"], p=s["p"], seed=s["seed"], offset=s["offset"])
    out = dict(y=y, stats=stats)
    if s["res"] is not None or s["p"] > 0:
        out["z"] = z
    return out


def _own_ln_bwd(s):
    from multimodalspectraltransformer_amd import ops
    dz, dx, dgamma, dbeta = ops.layer_norm_bwd(s["dy"], s["z"], s["stats"], s["gamma"], dz_in=s["add"], p=s["p"], seed=s["seed"], offset=s["offset"])
    out = dict(dz=dz, dgamma=dgamma, dbeta=dbeta)
    if s["p"] > 0:
        out["dx"] = dx
    return out


def _own_ce(s, grad):
    from multimodalspectraltransformer_amd import ops
    if not grad:
        loss, lse = ops.linear_ce(s["h"], s["w"], s["target"], bias=s["b"], ignore_index=IGNORE)
        return dict(loss=loss, lse=lse)
    loss, lse, dh, dw, dbias = ops.linear_ce_grad(s["h"], s["w"], s["target"], bias=s["b"], dloss=s["dloss"], ignore_index=IGNORE)
    out = dict(loss=loss, lse=lse, dh=dh, dw=dw)
    if s["b"] is not None:
        out["dbias"] = dbias
    return out


def run(state):
    op = state["op"]
    if op == "dropout":
        if own:
            from multimodalspectraltransformer_amd import ops
            return ops.dropout(state["x"], state["p"], state["seed"], state["offset"])
        return _dropped(state["x"].float(), state).to(state["x"].dtype)
    if op == "ln_fwd":
        return _own_ln_fwd(state) if own else _plain_ln_fwd(state)
    if op == "ln_bwd":
        return _own_ln_bwd(state) if own else _plain_ln_bwd(state)
    return _own_ce(state, op == "ce_grad") if own else _plain_ce(state, op == "ce_grad")


def work(case):
    op = case["op"]
    if op.startswith("ce"):
        n, d, v = case["rows"] - case["ignored"], case["dim"], case["vocab"]
        passes = 3 if op == "ce_grad" else 1  # logits; and the two products of their gradient
        moved = 2 * (n * d + v * d) * (2 if op == "ce_grad" else 1) + 16 * case["rows"] + 4 * v * case["bias"]
        return {"bytes": moved, "flops": 2 * passes * n * d * v + 4 * n * v}
    n, size = case["rows"] * case["cols"], DTYPES[case["dtype"]].itemsize
    if op == "dropout":
        return {"bytes": 2 * n * size, "flops": 30 * n}
    if op == "ln_fwd":
        tensors = 2 + case["residual"] + (case["residual"] or case["p"] > 0)
    else:
        tensors = 3 + case["add"] + (case["p"] > 0)
    return {"bytes": tensors * n * size + 8 * case["rows"] + 8 * case["cols"], "flops": (30 if case["p"] > 0 else 10) * n}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _mul32(a, m):
    """(upper, lower) 32 bits of a product of two 32-bit numbers, from 16-bit halves."""
    a0, a1, m0, m1 = a & 0xFFFF, a >> 16, m & 0xFFFF, m >> 16
    mid = a1 * m0 + ((a0 * m0) >> 16)
    low = a0 * m1 + (mid & 0xFFFF)
    return a1 * m1 + (mid >> 16) + (low >> 16), ((low & 0xFFFF) << 16) | ((a0 * m0) & 0xFFFF)


def _exact_factor(rows, cols, p, seed, offset):
    """What each element is multiplied with, in 64 bits."""
    i = torch.arange(rows * cols, device="cuda").reshape(-1)
    block = torch.arange(-(-rows * cols // 8), device="cuda")
    x = [block % (1 << 32), block // (1 << 32), torch.full_like(block, offset % (1 << 32)), torch.full_like(block, offset // (1 << 32))]
    k = [seed % (1 << 32), seed // (1 << 32)]
    for _ in range(10):
        (h0, l0), (h1, l1) = _mul32(x[0], 0xD2511F53), _mul32(x[2], 0xCD9E8D57)
        x = [h1 ^ x[1] ^ k[0], l1, h0 ^ x[3] ^ k[1], l0]
        k = [(k[0] + 0x9E3779B9) % (1 << 32), (k[1] + 0xBB67AE85) % (1 << 32)]
    word = torch.cat([w.unsqueeze(1) for w in x], dim=1)[i // 8, i % 8 // 2]
    sixteen = torch.where(i % 2 == 0, word % 65536, word // 65536)
    thr = int(p * 65536 + 0.5)
    return ((sixteen >= thr).double() * (65536 / max(1, 65536 - thr))).reshape(rows, cols)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op.startswith("ce"):
        return _exact_ce(s, op == "ce_grad")
    factor = _exact_factor(case["rows"], case["cols"], s["p"], s["seed"], s["offset"]) if s["p"] > 0 else None
    if op == "dropout":
        return s["x"].double() if factor is None else s["x"].double() * factor
    gamma = s["gamma"].double()
    if op == "ln_fwd":
        z = s["x"].double() if factor is None else s["x"].double() * factor
        z = z if s["res"] is None else z + s["res"].double()
        mean = z.sum(1) / z.shape[1]
        rstd = 1 / torch.sqrt(((z - mean[:, None]) ** 2).sum(1) / z.shape[1] + EPS)
        out = {"y": (z - mean[:, None]) * rstd[:, None] * gamma + s["beta"].double(), "stats": torch.stack([mean, rstd], 1)}
        if s["res"] is not None or factor is not None:
            out["z"] = z
        return out
    dy, mean, rstd = s["dy"].double(), s["stats"][:, 0:1].double(), s["stats"][:, 1:2].double()
    xh = (s["z"].double() - mean) * rstd
    n = dy.shape[1]
    dz = rstd / n * (n * dy * gamma - (dy @ gamma)[:, None] - xh * ((dy * xh) @ gamma)[:, None])
    dz = dz if s["add"] is None else dz + s["add"].double()
    out = {"dz": dz, "dgamma": torch.ones(dy.shape[0], dtype=torch.float64, device="cuda") @ (dy * xh), "dbeta": dy.sum(0)}
    if factor is not None:
        out["dx"] = dz * factor
    return out


def _exact_ce(s, grad):
    h, w = s["h"].double(), s["w"].double()
    bias = torch.zeros(w.shape[0], dtype=torch.float64, device="cuda") if s["b"] is None else s["b"].double()
    n, v = h.shape[0], w.shape[0]
    loss, lse = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    dh, dw, db = torch.zeros_like(h), torch.zeros_like(w), torch.zeros_like(bias)
    rows = (s["target"] != IGNORE).nonzero()[:, 0]
    for part in rows.split(max(1, (1 << 27) // v)):  # the rows that count, some at a time
        logits = torch.addmm(bias, h[part], w.t())
        t, at = s["target"][part], torch.arange(part.numel(), device="cuda")
        lse[part] = torch.logsumexp(logits, dim=1)
        loss[part] = lse[part] - logits[at, t]
        if grad:
            g = torch.softmax(logits, dim=1)
            g[at, t] -= 1
            g *= s["dloss"][part].double()[:, None]
            dh[part] = g @ w
            dw += g.t() @ h[part]
            db += g.sum(0)
    out = {"loss": loss, "lse": lse}
    if grad:
        out.update(dh=dh, dw=dw)
        if s["b"] is not None:
            out["dbias"] = db
    return out
