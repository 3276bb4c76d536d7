"""Thin Python wrappers that fill the C structs of libmmst.so from torch tensors.

Every function enqueues HIP kernels on torch's current stream and returns
immediately; nothing here computes on the host.
"""
import ctypes as C

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
# ---------------------------------------------------------------------------------------------
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # mmst_dtype
_P, _I, _LONG, _SIZE, _F, _D, _U64 = C.c_void_p, C.c_int, C.c_long, C.c_size_t, C.c_float, C.c_double, C.c_uint64
_SIGNATURES = {
    "mmst_dropout": [_P, _LONG, _P, _LONG, _I, _LONG, _LONG, _D, _U64, _U64, _P],
    "mmst_layer_norm": [_P, _LONG, _P, _LONG, _P, _P, _P, _LONG, _P, _LONG, _P, _I, _LONG, _I, _F, _D, _U64, _U64, _P],
    "mmst_layer_norm_bwd": [_P, _LONG, _P, _LONG, _P, _P, _P, _LONG, _P, _LONG, _P, _LONG, _P, _P, _I, _I, _LONG, _I, _D,
                            _U64, _U64, _P, _SIZE, _P],
    "mmst_layer_norm_bwd_ws": [_LONG, _I, _P],
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


def _call(name, device, *args):
    """One call on the current stream of `device` (the tensors' own, which need not be the current one)."""
    f = _function(name)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            rc = f(*args, torch.cuda.current_stream().cuda_stream)
    else:
        rc = f(*args, torch.cuda.current_stream().cuda_stream)
    if rc != 0:
        raise L.MMSTError(f"{name} failed with code {rc}")


def _check(cond, message):
    if not cond:
        raise L.MMSTError(message)


def _rows(t, shape, dtype, device, name, out=False):
    """(tensor, row stride) of a tensor whose leading dimensions can be counted through with one stride and whose columns
    follow one another.  An input of another layout is copied, an output refused."""
    if t.dtype != dtype or t.device != device or t.shape != shape:
        raise L.MMSTError(f"{name}: {tuple(shape)} {dtype} on {device} expected, got {tuple(t.shape)} {t.dtype} on {t.device}")
    cols = shape[-1]
    if t.is_contiguous():
        return t, cols
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


def _vector(t, n, device, name):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.device != device or t.shape != (n,) or not t.is_contiguous():
        raise L.MMSTError(f"{name}: contiguous fp32 [{n}] on {device} expected, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


def _check_rows_input(x, what):
    _check(isinstance(x, torch.Tensor) and x.is_cuda, f"{what}: a tensor on the GPU expected (there is no CPU path)")
    _check(x.dtype in _DTYPES, f"{what}: fp32, bf16 or fp16 expected, got {x.dtype}")
    _check(x.dim() >= 1, f"{what}: at least one dimension expected")


def _check_mask(p, seed, offset, what):
    _check(0.0 <= p <= 1.0, f"{what}: p = {p} is not a probability")
    _check(0 <= seed < 1 << 64 and 0 <= offset < 1 << 64, f"{what}: seed and offset are 64-bit numbers")


def dropout(x, p, seed, offset=0, out=None):
    """x with each element set to 0 with probability p and scaled by 1 / (1 - p) otherwise (p rounded to a multiple of
    1 / 65536).  The mask is a function of (seed, offset, element of x read row by row) and never stored: the same call on
    the gradient of the result is the backward pass.  `out` may be x.  fp32, bf16, fp16; any shape."""
    _check_rows_input(x, "dropout")
    _check_mask(p, seed, offset, "dropout")
    shape, device = x.shape, x.device
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=device)
    if x.numel() == 0:
        return out
    x, ldx = _rows(x, shape, x.dtype, device, "dropout: x")
    y, ldy = _rows(out, shape, x.dtype, device, "dropout: out", out=True)
    cols = shape[-1]
    _call("mmst_dropout", device, x.data_ptr(), ldx, y.data_ptr(), ldy, _DTYPES[x.dtype], x.numel() // cols, cols, p, seed,
          offset)
    return out


def layer_norm(x, gamma=None, beta=None, eps=1e-5, residual=None, p=0.0, seed=0, offset=0, out=None, z_out=None):
    """(y, z, stats): z = residual + dropout(x) and its layer norm over the last dimension, y = (z - mean) rstd gamma +
    beta; stats [..., 2] = (mean, rstd) in fp32.  z is x itself where there is neither residual nor dropout.  gamma / beta
    fp32 or None; at most 16384 columns.  (p, seed, offset) as in dropout()."""
    _check_rows_input(x, "layer_norm")
    _check_mask(p, seed, offset, "layer_norm")
    shape, dtype, device = x.shape, x.dtype, x.device
    cols = shape[-1]
    _check(1 <= cols <= 16384, f"layer_norm: 1 to 16384 columns, got {cols}")
    _check(eps >= 0.0, "layer_norm: eps must not be negative")
    gp, bp = _vector(gamma, cols, device, "layer_norm: gamma"), _vector(beta, cols, device, "layer_norm: beta")
    x2, ldx = _rows(x, shape, dtype, device, "layer_norm: x")
    rp, ldr = None, cols
    if residual is not None:
        residual, ldr = _rows(residual, shape, dtype, device, "layer_norm: residual")
        rp = residual.data_ptr()
    y = torch.empty(shape, dtype=dtype, device=device) if out is None else out
    y2, ldy = (y, cols) if out is None else _rows(y, shape, dtype, device, "layer_norm: out", out=True)
    z, zp, ldz = x, None, cols
    if residual is not None or p > 0.0 or z_out is not None:
        z = torch.empty(shape, dtype=dtype, device=device) if z_out is None else z_out
        z2, ldz = (z, cols) if z_out is None else _rows(z, shape, dtype, device, "layer_norm: z_out", out=True)
        zp = z2.data_ptr()
    stats = torch.empty(shape[:-1] + (2,), dtype=torch.float32, device=device)
    _call("mmst_layer_norm", device, x2.data_ptr(), ldx, rp, ldr, gp, bp, y2.data_ptr(), ldy, zp, ldz, stats.data_ptr(),
          _DTYPES[dtype], x.numel() // cols, cols, eps, p, seed, offset)
    return y, z, stats


def layer_norm_bwd(dy, z, stats, gamma=None, dz_in=None, p=0.0, seed=0, offset=0, dgamma=None, dbeta=None):
    """(dz, dx, dgamma, dbeta) from the gradient at y and what layer_norm() returned: dz = gradient at z (the residual's
    too), plus dz_in where z is also used elsewhere; dx = dz through the dropout mask (dz itself where p is 0).  dgamma /
    dbeta (fp32): given ones are added to, as the framework's parameter gradients are, None makes new ones."""
    _check_rows_input(dy, "layer_norm_bwd")
    _check_mask(p, seed, offset, "layer_norm_bwd")
    shape, dtype, device = dy.shape, dy.dtype, dy.device
    cols = shape[-1]
    _check(1 <= cols <= 16384, f"layer_norm_bwd: 1 to 16384 columns, got {cols}")
    _check((dgamma is None) == (dbeta is None), "layer_norm_bwd: dgamma and dbeta come together")
    rows = dy.numel() // cols
    gp = _vector(gamma, cols, device, "layer_norm_bwd: gamma")
    dy2, lddy = _rows(dy, shape, dtype, device, "layer_norm_bwd: dy")
    z2, ldz = _rows(z, shape, dtype, device, "layer_norm_bwd: z")
    stats, _ = _rows(stats, shape[:-1] + (2,), torch.float32, device, "layer_norm_bwd: stats")
    if not stats.is_contiguous():
        stats = stats.contiguous()
    ap, ldadd = None, cols
    if dz_in is not None:
        dz_in, ldadd = _rows(dz_in, shape, dtype, device, "layer_norm_bwd: dz_in")
        ap = dz_in.data_ptr()
    accumulate = dgamma is not None
    if not accumulate:
        dgamma, dbeta = torch.empty(2, cols, dtype=torch.float32, device=device).unbind(0)
    dgp, dbp = _vector(dgamma, cols, device, "layer_norm_bwd: dgamma"), _vector(dbeta, cols, device, "layer_norm_bwd: dbeta")
    dz = torch.empty(shape, dtype=dtype, device=device)
    masked = int(p * 65536.0 + 0.5) > 0
    dx = torch.empty(shape, dtype=dtype, device=device) if masked else dz
    nbytes = C.c_size_t()
    rc = _function("mmst_layer_norm_bwd_ws")(rows, cols, C.byref(nbytes))
    _check(rc == 0, "mmst_layer_norm_bwd_ws failed")
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=device)
    _call("mmst_layer_norm_bwd", device, dy2.data_ptr(), lddy, z2.data_ptr(), ldz, stats.data_ptr(), gp, ap, ldadd,
          dz.data_ptr(), cols, dx.data_ptr(), cols, dgp, dbp, int(accumulate), _DTYPES[dtype], rows, cols, p, seed, offset,
          ws.data_ptr(), nbytes.value)
    return dz, dx, dgamma, dbeta


# ---------------------------------------------------------------------------------------------
# linear layer + softmax cross entropy over a large vocabulary (mmst_linear_ce)
# ---------------------------------------------------------------------------------------------
def _linear_ce_args(h, w, target, bias, ignore_index, what):
    for t, name in ((h, "h"), (w, "w")):
        _check(isinstance(t, torch.Tensor) and t.is_cuda, f"{what}: {name} on the GPU expected (there is no CPU path)")
        _check(t.dtype == torch.bfloat16 and t.dim() == 2, f"{what}: {name} as a bf16 matrix expected, got {t.dtype} {tuple(t.shape)}")
    device, (n, d), v = h.device, h.shape, w.shape[0]
    _check(w.device == device and w.shape[1] == d, f"{what}: h {tuple(h.shape)} and w {tuple(w.shape)} do not fit")
    _check(v >= 1 and d >= 8 and d % 8 == 0, f"{what}: a vocabulary and a width that is a multiple of 8 expected, got {v} and {d}")
    _check(target.dtype == torch.int64 and target.device == device and target.shape == (n,),
           f"{what}: target as int64 [{n}] on {device} expected, got {target.dtype} {tuple(target.shape)} on {target.device}")
    a = L.LinearCeArgs()
    keep = []   # copies of inputs whose layout the kernels do not read
    for t, name in ((h, "h"), (w, "w")):
        if t.stride(1) != 1 or t.stride(0) % 8 or (t.shape[0] > 1 and t.stride(0) < d) or t.data_ptr() % 16:
            t = torch.empty_like(t, memory_format=torch.contiguous_format).copy_(t)
            keep.append(t)
        setattr(a, name, t.data_ptr())
        setattr(a, "ld" + name, t.stride(0) if t.shape[0] > 1 else d)
    if not target.is_contiguous():
        target = target.contiguous()
        keep.append(target)
    a.target = target.data_ptr()
    a.bias = _vector(bias, v, device, f"{what}: bias")
    a.ignore_index = ignore_index
    a.N, a.D, a.V = n, d, v
    return a, keep


def _linear_ce_call(a, grad, device):
    nbytes = C.c_size_t()
    _check(_function("mmst_linear_ce_ws")(C.byref(a), grad, C.byref(nbytes)) == 0,
           f"linear_ce: sizes outside the limits: {a.N} rows, {a.V} words, width {a.D}")
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=device)
    a.ws, a.ws_bytes = ws.data_ptr(), nbytes.value
    _call("mmst_linear_ce", device, C.byref(a), grad)


def linear_ce(h, w, target, bias=None, ignore_index=-100):
    """(loss, lse), both fp32 [N]: softmax cross entropy of the logits h w^T + bias against target, and the rows' log sum
    exp, without the logits in memory.  h [N, D], w [V, D] bf16, target int64 [N], bias fp32 [V] or None; D a multiple of 8.
    Rows whose target is ignore_index have loss and lse 0; a target that is no word gives NaN."""
    a, keep = _linear_ce_args(h, w, target, bias, ignore_index, "linear_ce")
    loss, lse = torch.empty(2, a.N, dtype=torch.float32, device=h.device).unbind(0)
    a.loss, a.lse = loss.data_ptr(), lse.data_ptr()
    _linear_ce_call(a, 0, h.device)
    return loss, lse


def linear_ce_grad(h, w, target, bias=None, dloss=None, grad_scale=1.0, ignore_index=-100, dw=None, dbias=None,
                   rows_per_piece=0):
    """(loss, lse, dh, dw, dbias): linear_ce() and the gradients of sum(grad_scale * dloss * loss) (dloss fp32 [N], None:
    ones).  dh is bf16; dw and dbias are bf16 as well, or, where fp32 tensors are given, added to those.  dbias is None
    without a bias.  rows_per_piece bounds the workspace: that many rows' gradient of the logits, in bf16, at a time."""
    a, keep = _linear_ce_args(h, w, target, bias, ignore_index, "linear_ce_grad")
    device, n, d, v = h.device, a.N, a.D, a.V
    _check(rows_per_piece >= 0, "linear_ce_grad: rows_per_piece must not be negative")
    loss, lse = torch.empty(2, n, dtype=torch.float32, device=device).unbind(0)
    dh = torch.empty(n, d, dtype=torch.bfloat16, device=device)
    a.loss, a.lse, a.dh, a.lddh = loss.data_ptr(), lse.data_ptr(), dh.data_ptr(), d
    a.dloss = _vector(dloss, n, device, "linear_ce_grad: dloss")
    a.grad_scale, a.rows_per_piece = grad_scale, rows_per_piece
    if dw is None:
        _check(dbias is None, "linear_ce_grad: dbias to be added to comes with dw")
        dw = torch.empty(v, d, dtype=torch.bfloat16, device=device)
        dbias = None if bias is None else torch.empty(v, dtype=torch.bfloat16, device=device)
    else:
        _check(dw.dtype == torch.float32 and dw.device == device and dw.shape == (v, d) and dw.is_contiguous() and dw.data_ptr() % 16 == 0,
               f"linear_ce_grad: dw as contiguous fp32 [{v}, {d}] on {device} expected")
        _check((dbias is None) == (bias is None), "linear_ce_grad: dbias comes with bias")
        _vector(dbias, v, device, "linear_ce_grad: dbias")
        a.grad_f32 = 1
    a.dw, a.dbias = dw.data_ptr(), None if dbias is None else dbias.data_ptr()
    _linear_ce_call(a, 1, device)
    return loss, lse, dh, dw, dbias
