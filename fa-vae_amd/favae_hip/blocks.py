"""The operators of a residual block: group norm with an activation (channels last), matrix product with bias, activation and
residual in its epilogue, both with their gradients, and activations kept for the backward pass in 8 bits (csrc/groupnorm.hip,
linear.hip, ckpt8.hip).

    y, mean, rstd, x8 = group_norm_act(x, groups, gamma, beta, act="silu", ckpt=True)
    out, pre          = linear_act(y, w, bias, act="gelu_tanh", residual=r, save_pre=True)
    y8, pre8          = ckpt8_pack(y), ckpt8_pack(pre)                       # y and pre need not be kept
    dy, dw, db        = linear_act_bwd(dout, y8, w, act="gelu_tanh", pre=pre8)   # the gradient of r is dout
    dx, dgamma, dbeta = group_norm_act_bwd(dy, x8, groups, gamma, beta, mean, rstd, act="silu")

Tensors are fp32 or bf16 (one type per call), scale, shift, bias and statistics fp32.  Every call is asynchronous on the current
stream of its tensors' device, may be captured into a graph, and takes its workspace from torch's allocator on that stream.
Activations: "none", "lrelu" (slope 0.01), "silu", "gelu_tanh".  Wrong arguments raise ValueError or TypeError before anything is
launched (sizes past a limit of the library: lib.FavaeArgError, a ValueError and a FavaeHipError); there is no CPU fallback.

Nothing here enters an autograd graph: gradients come from the *_bwd calls, made by hand under torch.no_grad() or from an
autograd.Function.  With grad mode on and an input that requires a gradient, the values are the same, differentiating them raises, and
`out` is refused.  What a *_bwd call or ckpt8_unpack returns is a constant.
"""
import ctypes
import math

import torch

from . import lib as L

_raw = L.raw()
_p, _ll, _i, _sz = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int, ctypes.c_size_t
_raw.favae_ckpt8_pack.argtypes = [_p, _ll, _ll, _i, _p, _ll, _p, _ll, _i, _p]
_raw.favae_ckpt8_unpack.argtypes = [_p, _ll, _p, _ll, _ll, _i, _p, _ll, _i, _p]
_raw.favae_gn_act_scratch.argtypes = [_ll, _ll, _i, _i, _i, _i]
_raw.favae_gn_act_scratch.restype = _sz
_raw.favae_gn_act_fwd.argtypes = [_p, _ll, _ll, _ll, _ll, _i, _i, _p, _p, ctypes.c_float, _i, _p, _ll, _ll, _p, _p, _p, _p, _p, _sz, _i, _p]
_raw.favae_gn_act_bwd.argtypes = [_p, _ll, _ll, _p, _ll, _ll, _p, _p, _ll, _ll, _i, _i, _p, _p, _p, _p, _i, _p, _ll, _ll, _p, _p, _p, _sz,
                                  _i, _p]
_raw.favae_linear_act_fwd_scratch.argtypes = [_ll, _i, _i, _i, _i]
_raw.favae_linear_act_fwd_scratch.restype = _sz
_raw.favae_linear_act_fwd.argtypes = [_p, _ll, _p, _ll, _p, _p, _ll, _p, _ll, _p, _ll, _ll, _i, _i, _i, _p, _sz, _i, _p]
_raw.favae_linear_act_bwd_scratch.argtypes = [_ll, _i, _i, _i, _i, _i, _i]
_raw.favae_linear_act_bwd_scratch.restype = _sz
_raw.favae_linear_act_bwd.argtypes = [_p, _ll, _p, _ll, _p, _ll, _p, _ll, _p, _ll, _p, _ll, _ll, _i, _i, _i, _p, _ll, _p, _ll, _i, _p, _p, _sz,
                                      _i, _p]

ACTS = {"none": 0, "lrelu": 1, "silu": 2, "gelu_tanh": 3}
CKPT_BLOCK = 32
F32, BF16 = torch.float32, torch.bfloat16


class Ckpt8:
    """An activation in 8 bits: q int8 [..., C] and e uint8 [..., ceil(C / 32)], value = q * 2^(e - 127); dtype is the type it was
    packed from.  A decoded value is exact in bf16.  A block of 32 channels that held an infinity or a NaN decodes to NaN."""

    __slots__ = ("q", "e", "dtype")

    def __init__(self, q, e, dtype):
        if q.dtype != torch.int8 or e.dtype != torch.uint8:
            raise TypeError("Ckpt8: q is int8 and e is uint8")
        if dtype not in (F32, BF16):
            raise TypeError("Ckpt8: dtype is float32 or bfloat16")
        if q.dim() < 1 or e.shape != q.shape[:-1] + ((q.shape[-1] + CKPT_BLOCK - 1) // CKPT_BLOCK,):
            raise ValueError("Ckpt8: e has the shape of q with ceil(C / 32) in place of C")
        if q.device != e.device or not (q.is_contiguous() and e.is_contiguous()):
            raise ValueError("Ckpt8: q and e are contiguous and on one device")
        self.q, self.e, self.dtype = q, e, dtype

    @property
    def shape(self):
        return self.q.shape

    @property
    def device(self):
        return self.q.device


# ---- arguments -----------------------------------------------------------------------------------------------------------
def _code(t, name):
    if t.dtype == F32:
        return L.F32
    if t.dtype == BF16:
        return L.BF16
    raise TypeError("%s: float32 or bfloat16, not %s" % (name, t.dtype))


def _act(name):
    if name not in ACTS:
        raise ValueError("act: one of %s, not %r" % (", ".join(sorted(ACTS)), name))
    return ACTS[name]


def _rows(t, name):
    """Stride between the rows of t seen as [R, C]; its leading dimensions must collapse and its last one be contiguous."""
    if t.dim() < 1:
        raise ValueError("%s: a tensor of at least one dimension" % name)
    if t.is_contiguous():
        return t.shape[-1]
    sh, st = t.shape, t.stride()
    if 0 in sh:
        return sh[-1]
    if sh[-1] > 1 and st[-1] != 1:
        raise ValueError("%s: the last dimension must be contiguous" % name)
    ld, span = None, 1
    for n, s in zip(reversed(sh[:-1]), reversed(st[:-1])):
        if n == 1:
            continue
        if ld is None:
            ld = s
        elif s != ld * span:
            raise ValueError("%s: its leading dimensions are not one run of rows" % name)
        span *= n
    if ld is None:
        return sh[-1]
    if ld < sh[-1]:
        raise ValueError("%s: its rows overlap" % name)
    return ld


def _maps(t, name):
    """(sample stride, position stride) of t [N, ..., C]; the middle dimensions must be one run of positions."""
    c = t.shape[-1]
    if t.is_contiguous() or t.numel() == 0:
        s = 1
        for n in t.shape[1:-1]:
            s *= n
        return s * c, c
    pos = _rows(t[0], name)
    return (t.stride(0) if t.shape[0] > 1 else 0), pos


def _vec(t, n, name, dev):
    if t.dtype != F32 or t.shape != (n,):
        raise ValueError("%s: float32 [%d]" % (name, n))
    if t.device != dev or not t.is_contiguous():
        raise ValueError("%s: contiguous and on the device of the call" % name)
    return t.data_ptr()


def _on(dev, **tensors):
    if dev.type != "cuda":
        raise ValueError("tensors must be on the GPU; there is no CPU fallback")
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError("%s is on %s, the call is on %s" % (name, t.device, dev))


def _span(t):
    """First and one-past-last byte that t can touch."""
    if t.numel() == 0:
        return 0, 0
    n = 1 + sum((k - 1) * s for k, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def _same_place(a, b):
    return a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype


def _beside(a, b):
    """Whether a and b, whose spans meet, are different columns of one buffer: modulo the largest pitch that all their strides but the last
    are multiples of, the bytes of their rows do not meet."""
    pitch, width = 0, []
    for t in (a, b):
        es, inner = t.element_size(), t.dim() - 1
        for k in range(inner):
            if t.shape[k] > 1:
                pitch = math.gcd(pitch, t.stride(k) * es)
        width.append(((t.shape[inner] - 1) * t.stride(inner) + 1) * es)
    if pitch == 0:
        return False
    d = (b.data_ptr() - a.data_ptr()) % pitch
    return width[0] <= d and d + width[1] <= pitch


def _apart(out, name, ins, may_be=None):
    """`out` shares no memory with the inputs, but that it may be `may_be` itself."""
    lo, hi = _span(out)
    for t in ins:
        if t is None or (t is may_be and _same_place(out, t)):
            continue
        a, b = _span(t)
        if lo < b and a < hi and not _beside(out, t):
            raise ValueError("%s overlaps an input" % name)


def _distinct(t, name):
    """Every element of t, which a call writes, has a place of its own."""
    span = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if st < span:
            raise ValueError("%s overlaps itself" % name)
        span = st * n                                        # (at least: strides that interleave otherwise are refused too)
    return t


def _out(out, name, like, shape, dtype, ins, may_be=None):
    if out is None:
        return like.new_empty(shape, dtype=dtype)
    dev = like.device
    if out.dtype != dtype or out.shape != torch.Size(shape) or out.device != dev:
        raise ValueError("%s: %s %s on %s" % (name, dtype, list(shape), dev))
    _apart(out, name, ins, may_be)
    return out if out.is_contiguous() or out.numel() == 0 else _distinct(out, name)


def _no_out(out):
    """An output of the caller's is refused where autograd would follow the inputs, as torch's own operators do."""
    if out is not None:
        raise ValueError("out: takes no part in autograd, and an input requires a gradient (call under torch.no_grad())")


def _no_graph(name, *outs):
    """The outputs, with a node of autograd that raises: to be differentiated they would have to come from a graph, and there is none.  The node
    hangs on a leaf of its own, so that an output that lives on keeps nothing of the caller's."""
    node = torch._C._functions.DelayedError("%s leaves no autograd graph: its gradients are %s_bwd's (call both under torch.no_grad(), or from an "
                                            "autograd.Function)" % (name, name), len(outs) + 1)
    return node(*outs, torch.empty(0, device="cpu", requires_grad=True))[:-1]


_grad_mode = torch.is_grad_enabled
_stream_of, _current = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice    # torch.cuda.current_stream builds an object: 2 us


def _call(dev, fn, *args):
    """fn(*args, stream) on the current stream of `dev`, whichever device is current."""
    i = dev.index
    if i == _current():
        rc = fn(*args, _stream_of(i))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream_of(i))
    if rc == L.ERR_ARG:
        raise L.FavaeArgError(L.last_error())
    if rc:
        L.check(rc)


def _scratch(nbytes, like):
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---- 8-bit activations ---------------------------------------------------------------------------------------------------
def _new_ckpt(x):
    shape = x.shape
    ck = Ckpt8.__new__(Ckpt8)                                # right by construction
    ck.q = x.new_empty(shape, dtype=torch.int8)
    ck.e = x.new_empty(shape[:-1] + (-(-shape[-1] // CKPT_BLOCK),), dtype=torch.uint8)
    ck.dtype = x.dtype
    return ck


def ckpt8_pack(x):
    """x [..., C] (fp32 or bf16, rows of any stride) -> Ckpt8."""
    code, ld, dev = _code(x, "x"), _rows(x, "x"), x.device
    if dev.type != "cuda":
        _on(dev)
    c = x.shape[-1]
    ck = _new_ckpt(x)
    n = x.numel()
    if n:
        _call(dev, _raw.favae_ckpt8_pack, x.data_ptr(), ld, n // c, c, ck.q.data_ptr(), c, ck.e.data_ptr(), -(-c // CKPT_BLOCK), code)
    return ck


def ckpt8_unpack(ck, dtype=None, out=None):
    """The values of a checkpoint, in the type it was packed from or in `dtype`; out: rows of any stride."""
    q, e = ck.q, ck.e
    dtype = ck.dtype if dtype is None and out is None else out.dtype if dtype is None else dtype
    if dtype not in (F32, BF16):
        raise TypeError("dtype: float32 or bfloat16")
    dev = q.device
    if dev.type != "cuda":
        _on(dev)
    c = q.shape[-1]
    if out is None:
        out, ld = q.new_empty(q.shape, dtype=dtype), c
    else:
        out = _out(out, "out", q, q.shape, dtype, (q, e))
        ld = _rows(out, "out")
    n = q.numel()
    if n:
        _call(dev, _raw.favae_ckpt8_unpack, q.data_ptr(), c, e.data_ptr(), -(-c // CKPT_BLOCK), n // c, c, out.data_ptr(), ld,
              L.F32 if dtype == F32 else L.BF16)
    return out


# ---- group norm ----------------------------------------------------------------------------------------------------------
def _gn_sizes(shape, groups):
    if len(shape) < 2:
        raise ValueError("x: [N, ..., C]")
    n, c = shape[0], shape[-1]
    if not isinstance(groups, int) or groups < 1 or c < 1 or c % groups:
        raise ValueError("groups: a divisor of the %d channels, not %r" % (c, groups))
    s = 1
    for k in shape[1:-1]:
        s *= k
    return n, s, c


def group_norm_act(x, groups, gamma, beta, act="none", eps=1e-5, ckpt=False, out=None):
    """y = act(gamma * (x - mean) * rstd + beta) over x [N, ..., C], channels last, per sample and group of C / groups neighbouring
    channels.  Returns y, mean [N, groups], rstd [N, groups] (fp32) and, with ckpt, x as a Ckpt8.  A sample of no positions has mean
    0 and variance 0.  out may be x (without ckpt)."""
    shape = x.shape
    n, s, c = _gn_sizes(shape, groups)
    code, a, dev = _code(x, "x"), _act(act), x.device
    if dev.type != "cuda":
        _on(dev)
    g, b = _vec(gamma, c, "gamma", dev), _vec(beta, c, "beta", dev)
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError("eps: not negative")
    cut = _grad_mode() and (x.requires_grad or gamma.requires_grad or beta.requires_grad)
    if cut:
        _no_out(out)
    xn, xs = (s * c, c) if x.is_contiguous() else _maps(x, "x")
    if out is None:
        y, yn, ys = x.new_empty(shape), s * c, c
    else:
        y = _out(out, "out", x, shape, x.dtype, (x, gamma, beta), None if ckpt else x)
        yn, ys = _maps(y, "out")
    mean, rstd = gamma.new_empty((2, n, groups)).unbind()
    ck = _new_ckpt(x) if ckpt else None
    if n:
        nbytes = _raw.favae_gn_act_scratch(n, s, c, groups, 0, code)
        ws = _scratch(nbytes, x)
        _call(dev, _raw.favae_gn_act_fwd, x.data_ptr(), xn, xs, n, s, c, groups, g, b, eps, a, y.data_ptr(), yn, ys, mean.data_ptr(),
              rstd.data_ptr(), ck.q.data_ptr() if ckpt else None, ck.e.data_ptr() if ckpt else None, _ptr(ws), nbytes, code)
    if cut:
        y, mean, rstd = _no_graph("group_norm_act", y, mean, rstd)
    return (y, mean, rstd, ck) if ckpt else (y, mean, rstd)


def group_norm_act_bwd(dy, x, groups, gamma, beta, mean, rstd, act="none", out=None):
    """Gradients of group_norm_act: dx (dy's type), dgamma, dbeta (fp32 [C]).  x: the forward's input or its Ckpt8; mean and rstd as
    the forward returned them.  out may be dy."""
    n, s, c = _gn_sizes(dy.shape, groups)
    code, a, dev = _code(dy, "dy"), _act(act), dy.device
    ck = isinstance(x, Ckpt8)
    if x.shape != dy.shape or x.dtype != dy.dtype:
        raise ValueError("x: %s %s, as dy" % (dy.dtype, list(dy.shape)))
    if dev.type != "cuda" or x.device != dev or mean.device != dev or rstd.device != dev:
        _on(dev, x=x, mean=mean, rstd=rstd)
    g, b = _vec(gamma, c, "gamma", dev), _vec(beta, c, "beta", dev)
    stat = (n, groups)
    if not (mean.dtype == rstd.dtype == F32 and mean.shape == rstd.shape == stat and mean.is_contiguous() and rstd.is_contiguous()):
        raise ValueError("mean and rstd: contiguous float32 [%d, %d]" % stat)
    dn, ds = (s * c, c) if dy.is_contiguous() else _maps(dy, "dy")
    xn, xs = (0, 0) if ck else (s * c, c) if x.is_contiguous() else _maps(x, "x")
    if out is None:
        dx, dxn, dxs = dy.new_empty(dy.shape), s * c, c
    else:
        dx = _out(out, "out", dy, dy.shape, dy.dtype, (dy, x.q, x.e, gamma, beta, mean, rstd) if ck else (dy, x, gamma, beta, mean, rstd), dy)
        dxn, dxs = _maps(dx, "out")
    dgamma, dbeta = gamma.new_empty((2, c)).unbind()
    nbytes = _raw.favae_gn_act_scratch(n, s, c, groups, 1, code)
    ws = _scratch(nbytes, dy)
    _call(dev, _raw.favae_gn_act_bwd, dy.data_ptr(), dn, ds, None if ck else x.data_ptr(), xn, xs, x.q.data_ptr() if ck else None,
          x.e.data_ptr() if ck else None, n, s, c, groups, g, b, mean.data_ptr(), rstd.data_ptr(), a, dx.data_ptr(), dxn, dxs,
          dgamma.data_ptr(), dbeta.data_ptr(), _ptr(ws), nbytes, code)
    return dx, dgamma, dbeta


def _odd(t, ld, ptr):
    """How t lies: 0 in 16-byte aligned rows, 1 not, 2 in rows more than 4 MB apart (the size of a product's workspace depends on it)."""
    row = ld * t.element_size()
    return 2 if row > 1 << 22 else 1 if ptr % 16 or row % 16 else 0


# ---- matrix product ------------------------------------------------------------------------------------------------------
def linear_act(x, w, bias=None, act="none", residual=None, save_pre=False, out=None):
    """act(x w^T + bias) + residual: x [..., K], w [N, K], bias fp32 [N], residual and the result [..., N] of x's type, rows of any
    stride.  Sums, bias, activation and residual are fp32, the result is rounded once.  With save_pre returns (y, pre), pre = x w^T +
    bias rounded to x's type, for linear_act_bwd.  out may be residual."""
    xsh, wsh = x.shape, w.shape
    if len(wsh) != 2 or not xsh or xsh[-1] != wsh[1]:
        raise ValueError("x [..., K] and w [N, K], not %s and %s" % (list(xsh), list(wsh)))
    code, a, dev = _code(x, "x"), _act(act), x.device
    if w.dtype != x.dtype:
        raise TypeError("w: %s, as x" % x.dtype)
    if dev.type != "cuda" or w.device != dev or residual is not None:
        _on(dev, w=w, residual=residual)
    n, k = wsh
    lead = xsh[:-1]
    m = 1
    for v in lead:
        m *= v
    shape = lead + (n,)
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype):
        raise ValueError("residual: %s %s" % (x.dtype, list(shape)))
    bp = None if bias is None else _vec(bias, n, "bias", dev)
    cut = _grad_mode() and (x.requires_grad or w.requires_grad or (bias is not None and bias.requires_grad) or
                            (residual is not None and residual.requires_grad))
    if cut:
        _no_out(out)
    if out is None:
        y, ldy = x.new_empty(shape), n
    else:
        y = _out(out, "out", x, shape, x.dtype, (x, w, bias, residual), residual)
        ldy = _rows(y, "out")
    pre = x.new_empty(shape) if save_pre else None
    if m and n:
        ldx = k if x.is_contiguous() else _rows(x, "x")
        ldw = k if w.is_contiguous() else _rows(w, "w")
        xp, wp = x.data_ptr(), w.data_ptr()
        nbytes = _raw.favae_linear_act_fwd_scratch(m, n, k, max(_odd(x, ldx, xp), _odd(w, ldw, wp)), code)
        ws = _scratch(nbytes, x)
        _call(dev, _raw.favae_linear_act_fwd, xp, ldx, wp, ldw, bp, _ptr(residual),
              0 if residual is None else _rows(residual, "residual"), _ptr(pre), n, y.data_ptr(), ldy, m, n, k, a, _ptr(ws), nbytes, code)
    if cut:
        return _no_graph("linear_act", y, pre) if save_pre else _no_graph("linear_act", y)[0]
    return (y, pre) if save_pre else y


_ALL = ("x", "w", "b")


def linear_act_bwd(dy, x, w, act="none", pre=None, need=_ALL, dw=None):
    """Gradients of linear_act: (dx, dw, db), None for what `need` leaves out.  x and pre: tensors or Ckpt8; pre is needed unless act
    is "none".  dx [..., K] is of dy's type, dw [N, K] of w's type or, into a float32 `dw`, as it was summed, db fp32 [N].  Both products
    read du = dy act'(pre) rounded once to dy's type (db sums it unrounded).  The gradient of the residual is dy."""
    code, a, dev = _code(dy, "dy"), _act(act), dy.device
    if w.dim() != 2 or dy.dim() < 1 or dy.shape[-1] != w.shape[0] or x.shape != dy.shape[:-1] + (w.shape[1],):
        raise ValueError("dy [..., N], x [..., K], w [N, K], not %s, %s, %s" % (list(dy.shape), list(x.shape), list(w.shape)))
    if w.dtype != dy.dtype or x.dtype != dy.dtype:
        raise TypeError("x and w: %s, as dy" % dy.dtype)
    if need is not _ALL and not set(need) <= set(_ALL):
        raise ValueError("need: of 'x', 'w', 'b'")
    if act == "none":
        pre = None
    elif pre is None:
        raise ValueError("pre: the gradient of %s needs the pre-activation" % act)
    elif pre.shape != dy.shape or pre.dtype != dy.dtype:
        raise ValueError("pre: %s %s, as dy" % (dy.dtype, list(dy.shape)))
    if dev.type != "cuda" or x.device != dev or w.device != dev or pre is not None:
        _on(dev, x=x, w=w, pre=pre)
    n, k = w.shape
    m = 1
    for v in dy.shape[:-1]:
        m *= v
    xck, pck = isinstance(x, Ckpt8), isinstance(pre, Ckpt8)
    lddw = k
    if dw is not None and "w" in need:
        if dw.dtype not in (F32, w.dtype) or dw.shape != w.shape or dw.device != dev:
            raise ValueError("dw: float32 or %s, %s" % (w.dtype, list(w.shape)))
        lddw = _rows(dw, "dw")
        _apart(dw, "dw", (dy, w) + ((x.q, x.e) if xck else (x,)) + ((pre.q, pre.e) if pck else (pre,)))
    dx = dy.new_empty(x.shape) if "x" in need else None
    dw = None if "w" not in need else w.new_empty((n, k)) if dw is None else dw
    db = dy.new_empty(n, dtype=F32) if "b" in need else None
    xp = x.q if xck else x
    pp = pre.q if pck else pre
    ldd = n if dy.is_contiguous() else _rows(dy, "dy")
    ldx = k if xp.is_contiguous() else _rows(xp, "x")
    ldw = k if w.is_contiguous() else _rows(w, "w")
    dyp, wp, xptr = dy.data_ptr(), w.data_ptr(), xp.data_ptr()
    odd = max(_odd(dy, ldd, dyp), _odd(w, ldw, wp), 0 if xck else _odd(x, ldx, xptr))
    nbytes = _raw.favae_linear_act_bwd_scratch(m, n, k, a, xck and dw is not None, odd, code)
    ws = _scratch(nbytes, dy)
    _call(dev, _raw.favae_linear_act_bwd, dyp, ldd, xptr, ldx, x.e.data_ptr() if xck else None,
          x.e.shape[-1] if xck else 0, wp, ldw, _ptr(pp), 0 if pp is None else _rows(pp, "pre"),
          pre.e.data_ptr() if pck else None, pre.e.shape[-1] if pck else 0, m, n, k, a, _ptr(dx), k, _ptr(dw), lddw,
          L.F32 if dw is not None and dw.dtype == F32 else code, _ptr(db), _ptr(ws), nbytes, code)
    return dx, dw, db
