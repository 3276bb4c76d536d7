"""Thin Python wrappers that fill the C structs of libmmst.so from torch tensors.

Every function enqueues HIP kernels on torch's current stream and returns
immediately; nothing here computes on the host.
"""
import ctypes as C
import functools

import torch

from . import _lib as L

_PTR_FIELDS = ("P", "Q", "C", "bias", "R", "gamma", "beta", "Z", "stats", "C2", "dgamma", "dbeta", "dbias")


def gemm_batch(groups):
    """groups: list of dicts with GemmProb field names; tensors for pointer fields."""
    if not 1 <= len(groups) <= L.GEMM_MAX_GROUPS:
        raise L.MMSTError("gemm: 1..%d groups" % L.GEMM_MAX_GROUPS)
    b = L.GemmBatch()
    b.n = len(groups)
    for i, g in enumerate(groups):
        p = b.p[i]
        for k, v in g.items():
            if k in _PTR_FIELDS:
                setattr(p, k, L.ptr(v) if isinstance(v, torch.Tensor) else v)
            else:
                setattr(p, k, v)
    return b


def gemm_launch(batch, epi, pt=False, qt=False):
    L.check(L.lib().mmst_gemm(C.byref(batch), epi, int(pt), int(qt), L.stream_ptr()), "mmst_gemm")


def gemm(groups, epi, pt=False, qt=False):
    gemm_launch(gemm_batch(groups), epi, pt, qt)


_APTR = ("Q", "K", "V", "kbias", "O", "lse", "dO", "delta", "dQ", "dK", "dV")


def attn_batch(groups, hd, causal=False, drop_p=0.0):
    if not 1 <= len(groups) <= L.MAX_GROUPS:
        raise L.MMSTError("attn: 1..%d groups" % L.MAX_GROUPS)
    b = L.AttnBatch()
    b.n = len(groups)
    b.hd = hd
    b.causal = int(causal)
    b.drop_p = float(drop_p)
    for i, g in enumerate(groups):
        p = b.p[i]
        for k, v in g.items():
            if k in _APTR:
                setattr(p, k, v if (v is None or isinstance(v, int)) else L.ptr(v))
            else:
                setattr(p, k, v)
    return b


def attn_fwd_launch(batch):
    L.check(L.lib().mmst_attn_fwd(C.byref(batch), L.stream_ptr()), "mmst_attn_fwd")


def attn_bwd_launch(batch):
    L.check(L.lib().mmst_attn_bwd(C.byref(batch), L.stream_ptr()), "mmst_attn_bwd")


_FPTR = ("X", "W1", "W2", "b1", "H", "dH", "ws", "Wn", "Cn", "Hs", "A", "Wp", "Wq", "bq", "Cq")


def ffn_batch(groups):
    """groups: list of dicts; key "epi" holds a dict of GemmProb fields for the final row epilogue."""
    if not 1 <= len(groups) <= L.MAX_GROUPS:
        raise L.MMSTError("ffn: 1..%d groups" % L.MAX_GROUPS)
    b = L.FfnBatch()
    b.n = len(groups)
    for i, g in enumerate(groups):
        p = b.p[i]
        for k, v in g.items():
            if k in ("epi", "pre"):
                sub = getattr(p, k)
                for ek, ev in v.items():
                    setattr(sub, ek, (L.ptr(ev) if isinstance(ev, torch.Tensor) else ev) if ek in _PTR_FIELDS else ev)
            elif k in _FPTR:
                setattr(p, k, L.ptr(v) if isinstance(v, torch.Tensor) else v)
            else:
                setattr(p, k, v)
    return b


def ffn_launch(batch, backward=False):
    """Returns 1 when a backward launch also wrote the chained Cn = E Wn of every problem, else 0."""
    rc = L.lib().mmst_ffn(C.byref(batch), int(backward), L.stream_ptr())
    if rc < 0:
        L.check(rc, "mmst_ffn")
    return rc


def ffn_wgrad(groups):
    """groups: list of dicts with FfnWgradProb fields (tensors for pointers)."""
    b = L.FfnWgradBatch()
    b.n = len(groups)
    for i, g in enumerate(groups):
        for k, v in g.items():
            setattr(b.p[i], k, L.ptr(v) if isinstance(v, torch.Tensor) else v)
    L.check(L.lib().mmst_ffn_wgrad(C.byref(b), L.stream_ptr()), "mmst_ffn_wgrad")


def eptr(t, offset_elems):
    """Device address of element `offset_elems` of tensor t."""
    return t.data_ptr() + offset_elems * t.element_size()


# ---------------------------------------------------------------------------------------------
# row operators of any width: dropout, layer norm (mmst_dropout, mmst_layer_norm, mmst_layer_norm_bwd)
#
# A call on a few rows takes the GPU 2 us and the host several times that, so these wrappers look at a tensor once and
# build their messages only where they raise.  They record no graph: what they compute does not require gradients, also
# where an input does, and the backward pass is the call that is named for it.
# ---------------------------------------------------------------------------------------------
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # mmst_dtype
_P, _I, _LONG, _SIZE, _F, _D, _U64 = C.c_void_p, C.c_int, C.c_long, C.c_size_t, C.c_float, C.c_double, C.c_uint64
_SIGNATURES = {
    "mmst_dropout": [_P, _LONG, _P, _LONG, _I, _LONG, _LONG, _D, _U64, _U64, _P],
    "mmst_layer_norm": [_P, _LONG, _P, _LONG, _P, _P, _P, _LONG, _P, _LONG, _P, _I, _LONG, _I, _F, _D, _U64, _U64, _P],
    "mmst_layer_norm_bwd": [_P, _LONG, _P, _LONG, _P, _P, _P, _LONG, _P, _LONG, _P, _LONG, _P, _P, _I, _I, _LONG, _I, _D,
                            _U64, _U64, _P, _SIZE, _P],
    "mmst_layer_norm_bwd_ws": [_I, _LONG, _I, _P],
    "mmst_linear_ce": [_P, _I, _P],
    "mmst_linear_ce_ws": [_P, _I, _P],
}
_functions = {}


def _function(name):
    """The library's entry point with its argument types declared (ctypes converts plain numbers faster that way)."""
    f = _functions.get(name)
    if f is None:
        f = getattr(L.lib(), name)
        f.argtypes = _SIGNATURES[name]
        _functions[name] = f
    return f


# the stream's handle without the Stream object around it (0.1 us instead of 2.7)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _call(name, device, *args):
    """One call on the current stream of `device` (the tensors' own, which need not be the current one)."""
    f = _functions.get(name) or _function(name)
    index = device.index
    if index == _current_device():
        rc = f(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(*args, _raw_stream(index))
    if rc != 0:
        raise L.MMSTError(f"{name} failed with code {rc}")


def _new_like(t):
    """A contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


def _rows(t, like, name, out=False):
    """(tensor, row stride) of a tensor of the shape, type and device of `like`, whose leading dimensions can be counted
    through with one stride and whose columns follow one another.  An input of another layout is copied, an output refused."""
    shape = like.shape
    if t is not like and (t.dtype is not like.dtype or t.shape != shape or t.device != like.device):
        raise L.MMSTError(f"{name}: {tuple(shape)} {like.dtype} on {like.device} expected, got {tuple(t.shape)} {t.dtype} on {t.device}")
    cols = shape[-1]
    if t.is_contiguous():
        return t, cols
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= cols:
        return t, t.stride(0)
    if t.stride(-1) == 1 or cols == 1:
        try:
            flat = t.view(-1, cols)
        except RuntimeError:
            flat = None
        if flat is not None and (flat.size(0) <= 1 or flat.stride(0) >= cols):
            return t, max(flat.stride(0), cols)
    if out:
        raise L.MMSTError(f"{name}: rows of consecutive columns, one stride apart, expected")
    return t.contiguous(), cols


def _overlap(a, lda, b, ldb):
    """Whether two tensors of one shape and type, their rows lda and ldb elements apart, have an element in common."""
    cols, size = a.shape[-1], a.element_size()
    if a.numel() == 0:
        return False
    rows, gap = a.numel() // cols, b.data_ptr() - a.data_ptr()
    if gap >= ((rows - 1) * lda + cols) * size or -gap >= ((rows - 1) * ldb + cols) * size:
        return False
    if rows == 1 or lda == ldb:   # a row of one begins `at` bytes behind one of the other
        at = gap % (lda * size)
        return rows == 1 or at < cols * size or lda * size - at < cols * size
    first = torch.arange(rows) * (lda * size)
    other = gap + torch.arange(rows) * (ldb * size)
    i = torch.searchsorted(first, other, right=True)   # rows of a that begin no later
    before = other - first[(i - 1).clamp(min=0)]
    behind = first[i.clamp(max=rows - 1)] - other
    return bool((((i > 0) & (before < cols * size)) | ((i < rows) & (behind < cols * size))).any())


def _clear(out, ldo, t, ldt, name, same=True):
    """Refuses an output that has some elements in common with another tensor of the call: a row could be written before
    it is read.  `same`: the very same rows may be written over."""
    if same and out.data_ptr() == t.data_ptr() and (ldo == ldt or t.numel() == t.shape[-1]):
        return
    if _overlap(out, ldo, t, ldt):
        raise L.MMSTError(f"{name} shares some of its elements with another tensor of the call")


def _vector(t, n, device, name):
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.shape != (n,) or not t.is_contiguous() or t.device != device:
        raise L.MMSTError(f"{name}: contiguous fp32 [{n}] on {device} expected, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


def _dtype_of(x, what):
    dt = _DTYPES.get(x.dtype) if isinstance(x, torch.Tensor) else None
    if dt is None or not x.is_cuda or x.dim() < 1:
        raise L.MMSTError(f"{what}: an fp32, bf16 or fp16 tensor of at least one dimension on the GPU expected (there is no "
                          f"CPU path), got {type(x).__name__ if not isinstance(x, torch.Tensor) else (x.dtype, tuple(x.shape), x.device)}")
    return dt


def _check_mask(p, seed, offset, what):
    if not 0.0 <= p <= 1.0:
        raise L.MMSTError(f"{what}: p = {p} is not a probability")
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        raise L.MMSTError(f"{what}: seed and offset are 64-bit numbers")


def dropout(x, p, seed, offset=0, out=None):
    """x with each element set to 0 with probability p and scaled by 1 / (1 - p) otherwise (p rounded to a multiple of
    1 / 65536).  The mask is a function of (seed, offset, element of x read row by row) and never stored: the same call on
    the gradient of the result is the backward pass.  `out` may be x, but share no other elements with it.  Without
    `out` the result is contiguous, and x itself where x is that and p rounds to 0: with a p that may be 0, a result that is
    changed in place needs an `out`.  fp32, bf16, fp16; any shape of at least one dimension."""
    dt = _dtype_of(x, "dropout")
    _check_mask(p, seed, offset, "dropout")
    y = None
    if out is None:
        if p * 65536.0 + 0.5 < 1.0 and x.is_contiguous():
            return x
        out = _new_like(x)
        ldy = x.shape[-1]
    else:
        y, ldy = _rows(out, x, "dropout: out", out=True)
    n = x.numel()
    if n == 0:
        return out
    x, ldx = _rows(x, x, "dropout: x")
    if y is not None:
        _clear(y, ldy, x, ldx, "dropout: out")
    cols = x.shape[-1]
    _call("mmst_dropout", x.device, x.data_ptr(), ldx, out.data_ptr(), ldy, dt, n // cols, cols, p, seed, offset)
    return out


def layer_norm(x, gamma=None, beta=None, eps=1e-5, residual=None, p=0.0, seed=0, offset=0, out=None, z_out=None):
    """(y, z, stats): z = residual + dropout(x) and its layer norm over the last dimension, y = (z - mean) rstd gamma +
    beta; stats [..., 2] = (mean, rstd) in fp32.  z is x itself where there is neither residual nor dropout, and a copy of
    it where `out` overwrites x.  gamma / beta fp32 or None; at most 16384 columns.  (p, seed, offset) as in dropout().
    `out` and `z_out` may each be x or the residual, but share no other elements with these and none with each other."""
    dt = _dtype_of(x, "layer_norm")
    _check_mask(p, seed, offset, "layer_norm")
    shape, device = x.shape, x.device
    cols = shape[-1]
    if not 1 <= cols <= 16384 or not eps >= 0.0:
        raise L.MMSTError(f"layer_norm: 1 to 16384 columns and eps >= 0 expected, got {cols} and {eps}")
    gp, bp = _vector(gamma, cols, device, "layer_norm: gamma"), _vector(beta, cols, device, "layer_norm: beta")
    x2, ldx = _rows(x, x, "layer_norm: x")
    rp, ldr = None, cols
    if residual is not None:
        residual, ldr = _rows(residual, x, "layer_norm: residual")
        rp = residual.data_ptr()
    ldy = ldz = cols
    if out is None:
        y = _new_like(x)
    else:
        y, ldy = _rows(out, x, "layer_norm: out", out=True)
    z, zp = x, None
    if z_out is not None:
        z, ldz = _rows(z_out, x, "layer_norm: z_out", out=True)
        zp = z.data_ptr()
    elif rp is not None or p > 0.0:
        z = _new_like(x)
        zp = z.data_ptr()
    elif out is not None:   # z is x, unless y is written over it
        if x2 is not x:
            z = x2
        elif _overlap(x, ldx, y, ldy):
            z = _new_like(x)
            zp = z.data_ptr()
    if out is not None or z_out is not None:
        for given, t, ld, name in ((out, y, ldy, "layer_norm: out"), (z_out, z, ldz, "layer_norm: z_out")):
            if given is not None:
                _clear(t, ld, x2, ldx, name)
                if residual is not None:
                    _clear(t, ld, residual, ldr, name)
        if out is not None and z_out is not None:
            _clear(y, ldy, z, ldz, "layer_norm: out", same=False)
    stats = x.new_empty(shape[:-1] + (2,), dtype=torch.float32)
    _call("mmst_layer_norm", device, x2.data_ptr(), ldx, rp, ldr, gp, bp, y.data_ptr(), ldy, zp, ldz, stats.data_ptr(), dt,
          x.numel() // cols, cols, eps, p, seed, offset)
    return y, z, stats


@functools.lru_cache(maxsize=1024)
def _layer_norm_bwd_ws(dt, rows, cols):
    n = C.c_size_t()
    if _function("mmst_layer_norm_bwd_ws")(dt, rows, cols, C.byref(n)) != 0:
        raise L.MMSTError(f"layer_norm_bwd: 1 to 16384 columns expected, got {cols}")
    return n.value


def layer_norm_bwd(dy, z, stats, gamma=None, dz_in=None, p=0.0, seed=0, offset=0, dgamma=None, dbeta=None):
    """(dz, dx, dgamma, dbeta) from the gradient at y and what layer_norm() returned: dz = gradient at z (the residual's
    too), plus dz_in where z is also used elsewhere; dx = dz through the dropout mask (dz itself where p is 0).  dgamma /
    dbeta (fp32): given ones are added to, as the framework's parameter gradients are, and share no elements; None makes new
    ones."""
    dt = _dtype_of(dy, "layer_norm_bwd")
    _check_mask(p, seed, offset, "layer_norm_bwd")
    shape, device = dy.shape, dy.device
    cols = shape[-1]
    if cols < 1 or (dgamma is None) != (dbeta is None):
        raise L.MMSTError("layer_norm_bwd: at least one column expected, and dgamma and dbeta together")
    rows = dy.numel() // cols
    nbytes = _layer_norm_bwd_ws(dt, rows, cols)
    gp = _vector(gamma, cols, device, "layer_norm_bwd: gamma")
    dy2, lddy = _rows(dy, dy, "layer_norm_bwd: dy")
    z2, ldz = _rows(z, dy, "layer_norm_bwd: z")
    if stats.dtype != torch.float32 or stats.shape != shape[:-1] + (2,) or stats.device != device:
        raise L.MMSTError(f"layer_norm_bwd: stats as layer_norm() returns them expected, got {tuple(stats.shape)} {stats.dtype}")
    if not stats.is_contiguous():
        stats = stats.contiguous()
    ap, ldadd = None, cols
    if dz_in is not None:
        dz_in, ldadd = _rows(dz_in, dy, "layer_norm_bwd: dz_in")
        ap = dz_in.data_ptr()
    accumulate = 0
    if dgamma is None:
        dgamma, dbeta = torch.empty((2, cols), dtype=torch.float32, device=device).unbind(0)
        dgp = dgamma.data_ptr()
        dbp = dgp + 4 * cols
    else:
        accumulate = 1
        dgp = _vector(dgamma, cols, device, "layer_norm_bwd: dgamma")
        dbp = _vector(dbeta, cols, device, "layer_norm_bwd: dbeta")
        if abs(dgp - dbp) < 4 * cols:
            raise L.MMSTError("layer_norm_bwd: dgamma and dbeta share elements")
    dz = _new_like(dy)
    dx = torch.empty_like(dz) if int(p * 65536.0 + 0.5) > 0 else dz
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _call("mmst_layer_norm_bwd", device, dy2.data_ptr(), lddy, z2.data_ptr(), ldz, stats.data_ptr(), gp, ap, ldadd,
          dz.data_ptr(), cols, dx.data_ptr(), cols, dgp, dbp, accumulate, dt, rows, cols, p, seed, offset, ws.data_ptr(), nbytes)
    return dz, dx, dgamma, dbeta


# ---------------------------------------------------------------------------------------------
# linear layer + softmax cross entropy over a large vocabulary (mmst_linear_ce)
# ---------------------------------------------------------------------------------------------
def _matrix(t, d, what):
    """(tensor, row stride) of a bf16 matrix of d columns as the kernels read it: rows 16-byte aligned and at most 2^20
    elements apart; copied otherwise."""
    ld = t.stride(0) if t.shape[0] > 1 else d
    if t.stride(1) != 1 or ld % 8 or not d <= ld <= 1 << 20 or t.data_ptr() % 16:
        t = torch.empty_like(t, memory_format=torch.contiguous_format).copy_(t)
        ld = d
    return t, ld


def _share(a, b):
    """Whether two tensors without strides share memory."""
    p, q = a.data_ptr(), b.data_ptr()
    return p < q + b.numel() * b.element_size() and q < p + a.numel() * a.element_size()


def _linear_ce_args(h, w, target, bias, ignore_index, what):
    if not (isinstance(h, torch.Tensor) and isinstance(w, torch.Tensor) and h.is_cuda and h.dtype == w.dtype == torch.bfloat16
            and h.dim() == w.dim() == 2 and h.device == w.device and h.shape[1] == w.shape[1]):
        raise L.MMSTError(f"{what}: h [N, D] and w [V, D] in bf16 on one GPU expected (there is no CPU path)")
    device, (n, d), v = h.device, h.shape, w.shape[0]
    if not 1 <= v <= 1 << 22 or not 8 <= d <= 32768 or d % 8 or n > 1 << 24:
        raise L.MMSTError(f"{what}: at most 2^24 rows, 1 to 2^22 words and a width that is a multiple of 8 and at most 32768 "
                          f"expected, got {n}, {v} and {d}")
    if target.dtype != torch.int64 or target.shape != (n,) or target.device != device:
        raise L.MMSTError(f"{what}: target as int64 [{n}] on {device} expected, got {target.dtype} {tuple(target.shape)} on {target.device}")
    h, ldh = _matrix(h, d, what)
    w, ldw = _matrix(w, d, what)
    if not target.is_contiguous():
        target = target.contiguous()
    # positional, in the order of the struct: half the time of setting the fields one by one
    a = L.LinearCeArgs(h.data_ptr(), ldh, w.data_ptr(), ldw, _vector(bias, v, device, what + ": bias"), target.data_ptr(),
                       ignore_index, n, d, v)
    return a, (h, w, target)   # the copies, if any, live until the call


@functools.lru_cache(maxsize=1024)
def _linear_ce_ws(n, d, v, grad, rows_per_piece, bias, f32):
    a = L.LinearCeArgs(N=n, D=d, V=v, rows_per_piece=rows_per_piece, dbias=1 if bias else None, grad_f32=f32)
    nbytes = C.c_size_t()
    if _function("mmst_linear_ce_ws")(C.byref(a), grad, C.byref(nbytes)) != 0:
        raise L.MMSTError(f"linear_ce: sizes outside the limits: {n} rows, {v} words, width {d}")
    return nbytes.value


def linear_ce(h, w, target, bias=None, ignore_index=-100):
    """(loss, lse), both fp32 [N]: softmax cross entropy of the logits h w^T + bias against target, and the rows' log sum
    exp, without the logits in memory.  h [N, D], w [V, D] bf16, target int64 [N], bias fp32 [V] or None; D a multiple of 8.
    Rows whose target is ignore_index have loss and lse 0; a target that is no word gives NaN."""
    a, keep = _linear_ce_args(h, w, target, bias, ignore_index, "linear_ce")
    device, n = h.device, a.N
    loss, lse = torch.empty((2, n), dtype=torch.float32, device=device).unbind(0)
    a.loss = loss.data_ptr()
    a.lse = a.loss + 4 * n if n else None
    a.ws_bytes = _linear_ce_ws(n, a.D, a.V, 0, 0, False, 0)
    ws = torch.empty(a.ws_bytes, dtype=torch.uint8, device=device)
    a.ws = ws.data_ptr()
    _call("mmst_linear_ce", device, C.byref(a), 0)
    return loss, lse


def linear_ce_grad(h, w, target, bias=None, dloss=None, grad_scale=1.0, ignore_index=-100, dw=None, dbias=None,
                   rows_per_piece=0):
    """(loss, lse, dh, dw, dbias): linear_ce() and the gradients of sum(grad_scale * dloss * loss) (dloss fp32 [N], None:
    ones).  dh is bf16; dw and dbias are bf16 as well, or, where fp32 tensors are given, added to those: dbias, or dw and
    with a bias dbias (which may be the bias itself: an update in place).  dbias is None without a bias.  rows_per_piece
    bounds the workspace: that many rows' gradient of the logits, in bf16, at a time."""
    given = [x for x in (dw, dbias) if x is not None]
    if given:   # gradients are written while later rows are still to come: what lies under them is read from a copy
        if len(given) == 2 and _share(dw, dbias):
            raise L.MMSTError("linear_ce_grad: dw and dbias share memory")
        if bias is not None and any(_share(x, bias) for x in given):
            bias = bias.clone()
        if dloss is not None and any(_share(x, dloss) for x in given):
            dloss = dloss.clone()
    a, keep = _linear_ce_args(h, w, target, bias, ignore_index, "linear_ce_grad")
    device, n, d, v = h.device, a.N, a.D, a.V
    if not 0 <= rows_per_piece <= 1 << 24:
        raise L.MMSTError("linear_ce_grad: rows_per_piece between 0 and 2^24 expected")
    loss, lse = torch.empty((2, n), dtype=torch.float32, device=device).unbind(0)
    dh = torch.empty((n, d), dtype=torch.bfloat16, device=device)
    a.loss, a.dh, a.lddh = loss.data_ptr(), dh.data_ptr(), d
    a.lse = a.loss + 4 * n if n else None
    if isinstance(dloss, torch.Tensor) and not dloss.is_contiguous():   # a mean's gradient is one number, expanded
        dloss = dloss.contiguous()
    a.dloss = _vector(dloss, n, device, "linear_ce_grad: dloss")
    a.grad_scale, a.rows_per_piece = grad_scale, rows_per_piece
    if dw is None:
        dw = torch.empty((v, d), dtype=torch.bfloat16, device=device)
        if dbias is not None:
            if bias is None:
                raise L.MMSTError("linear_ce_grad: dbias comes with bias")
            _vector(dbias, v, device, "linear_ce_grad: dbias")
            a.grad_f32 = 2
        elif bias is not None:
            dbias = torch.empty(v, dtype=torch.bfloat16, device=device)
    else:
        if dw.dtype != torch.float32 or dw.device != device or dw.shape != (v, d) or not dw.is_contiguous() or dw.data_ptr() % 16:
            raise L.MMSTError(f"linear_ce_grad: dw as contiguous fp32 [{v}, {d}] on {device} expected")
        if (dbias is None) != (bias is None):
            raise L.MMSTError("linear_ce_grad: dbias comes with bias")
        _vector(dbias, v, device, "linear_ce_grad: dbias")
        a.grad_f32 = 1
    a.dw = dw.data_ptr()
    if dbias is not None:
        a.dbias = dbias.data_ptr()
    a.ws_bytes = _linear_ce_ws(n, d, v, 1, rows_per_piece, dbias is not None, a.grad_f32)
    ws = torch.empty(a.ws_bytes, dtype=torch.uint8, device=device)
    a.ws = ws.data_ptr()
    _call("mmst_linear_ce", device, C.byref(a), 1)
    return loss, lse, dh, dw, dbias
