"""Activations in 8 bits, the norms that write and read them, and the root-mean-square norm (csrc/act8.hip, csrc/norm8_fwd.hip, csrc/norm8_bwd.hip).

A token is one position of an activation [N, C, ...] (a pixel of [N, C, H, W], a row of [N, C]).  Its C values are held as int8 or
e4m3 numbers with ONE power-of-two exponent per token, so a restored value is exact in bfloat16.  `Act8` is such an activation;
`checkpoint8` / `restore8` pack and restore one, `rms_norm8` writes its output in that form, `rms_norm(fmt=)` and `channel_norm8`
keep what their backward pass needs in it (1 byte per element in the place of a bfloat16 input, and of the next layer's input),
and `conv2d_weight_grad8` / `conv_transpose2d_weight_grad8` contract one.  The functions are part of `hific_amd.ops`.
"""
import contextlib
import functools
import os

import torch
from torch.autograd import Function, forward_ad

from . import lib, ops
from .lib import ptr, stream, require_gpu

FORMATS = {"int8": (0, torch.int8), "e4m3": (1, torch.float8_e4m3fn)}
_CODE = {torch.int8: 0, torch.float8_e4m3fn: 1}
_INF = float("inf")
_INT = 2 ** 31 - 1
_MAX_C = 2 ** 20                          # channels that a token's sums and exponent are formed over; strides and pads


def _fmt(fmt):
    if fmt not in FORMATS:
        raise lib.HificError(f"8-bit format must be one of {sorted(FORMATS)}, not {fmt!r}")
    return FORMATS[fmt]


def _nchw(x, name="x"):
    """(N, C, positions) of an activation [N, C, ...]."""
    d = x.dim()
    if d < 2 or x.size(1) < 1:
        raise lib.HificError(f"{name} must be [N, C, ...] with at least one channel, got {tuple(x.shape)}")
    n, c, hw = x.size(0), x.size(1), 1
    for i in range(2, d):
        hw *= x.size(i)
    if n > _INT or c > _MAX_C or hw > _INT:
        raise lib.HificError(f"{name}: {tuple(x.shape)} has a dimension beyond 32 bits or more than {_MAX_C} channels")
    return n, c, hw


def _tokens(x):
    return x.shape[:1] + x.shape[2:]


def _one_device(first, *rest):
    """All on the GPU, and on one (strided tensors are copied later: no contiguity rule)."""
    if not first.is_cuda:
        require_gpu(first)
    dev = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != dev:
            if not t.is_cuda:
                require_gpu(t)
            raise lib.HificError(f"tensors on {first.device} and {t.device}")


def c16(t):
    """Contiguous and 16-byte aligned: a strided or oddly placed view is copied."""
    if not t.is_contiguous():
        return t.contiguous()
    return t if (t.data_ptr() & 15) == 0 else t.clone(memory_format=torch.contiguous_format)


def _param(w, C, name):
    if w.dtype is not torch.float32 or w.numel() != C or not w.is_contiguous():
        raise lib.HificError(f"{name} must be a contiguous float32 tensor of {C} values, got {w.dtype} {tuple(w.shape)}")


def _like(t, x, name):
    if t.dtype is not x.dtype or t.shape != x.shape:
        raise lib.HificError(f"{name} must be {x.dtype} {tuple(x.shape)}, got {t.dtype} {tuple(t.shape)}")


def _eps(eps):
    if not 0.0 < eps < _INF:
        raise lib.HificError(f"eps must be positive and finite, got {eps}")
    return float(eps)


def _launch(name, t, *args):
    """Entry point `name` on the device of `t` and its current stream (the last argument)."""
    fn = getattr(lib._lib, name)
    if t.get_device() == lib._cur_device():
        rc = fn(*args, stream())
    else:
        with _on(t):
            rc = fn(*args, stream())
    if rc != 0:
        raise lib.HificError(f"{name} failed: {lib._ERR.get(rc, rc)} (rc={rc})")


_here = contextlib.nullcontext()


def _on(t):
    """Context in which launches (and the stream's workspace) belong to the device of `t`."""
    return _here if t.get_device() == lib._cur_device() else torch.cuda.device(t.device)


class _SecondOrder(Function):
    """Passes gradients on; differentiating them raises."""

    @staticmethod
    def forward(ctx, *grads):
        return tuple(g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *grads):
        raise lib.HificError(_NO_SECOND)


_NO_SECOND = "the 8-bit activation operators have no second derivative"


def _first_order(backward):
    """A backward pass that has no derivative of its own.  Grad mode is on in it with create_graph=True only: an incoming gradient that
    requires grad is refused, and what is computed from the saved tensors raises where it is differentiated in turn - returned as
    constants, a penalty on it would drop out of another loss without a word.  Gradients that are passed through are constants in truth."""
    @functools.wraps(backward)
    def run(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        if any(g is not None and g.requires_grad for g in grads):
            raise lib.HificError(_NO_SECOND)
        with torch.no_grad():
            grads = [g if g is None else c16(g) for g in grads]
            out = backward(ctx, *grads)
        made = {id(g): g for g in out if g is not None and not any(g is t for t in grads)}
        if not made:
            return out
        made = dict(zip(made, _SecondOrder.apply(*(g.detach().requires_grad_() for g in made.values()))))
        return tuple(made.get(id(g), g) if g is not None else None for g in out)
    return run


def _arena(t):
    slot = ops._slot(t)
    return None if slot is None else slot.arena


def _token(t, arena):
    """Changes with the values of a parameter: torch counts writes in place (not of inference tensors), an arena its optimizer's steps."""
    return 0 if t.is_inference() else t._version, 0 if arena is None else arena.epoch


class Act8:
    """An activation in 8 bits: `q` (int8 or float8_e4m3fn) [N, C, ...] and `e` (uint8, exponent + 127, from 1 on) [N, ...].  With `gamma` /
    `beta` (float32, C values) it stands for relu?(gamma * (q * 2^e) + beta): a norm's output held as its normalised values.  It holds
    these tensors themselves, not copies: one that channel_norm8 or conv_norm8 returned stands for their output until its norm's
    parameters change (an optimizer step), and is refused from then on."""
    __slots__ = ("q", "e", "gamma", "beta", "relu", "_made")

    def __init__(self, q, e, gamma=None, beta=None, relu=False):
        if q.dtype not in _CODE or e.dtype != torch.uint8:
            raise lib.HificError(f"Act8: q must be int8 or float8_e4m3fn and e uint8, got {q.dtype} and {e.dtype}")
        _, C, _ = _nchw(q, "q")
        if e.shape != _tokens(q):
            raise lib.HificError(f"Act8: e must be {tuple(_tokens(q))} for q {tuple(q.shape)}, got {tuple(e.shape)}")
        if (gamma is None) != (beta is None) or (relu and gamma is None):
            raise lib.HificError("Act8: gamma and beta come together, and relu with them")
        _one_device(q, e, gamma, beta)
        for t, name in ((gamma, "gamma"), (beta, "beta")):
            if t is not None:
                _param(t, C, name)
        self.q, self.e, self.gamma, self.beta, self.relu, self._made = c16(q), c16(e), gamma, beta, bool(relu), None

    @classmethod
    def _of(cls, q, e, gamma=None, beta=None, relu=False):
        """Without the checks: tensors that were just made; gamma and beta a norm's parameters."""
        a = object.__new__(cls)
        a.q, a.e, a.relu = q, e, relu
        if gamma is None:
            a.gamma = a.beta = a._made = None
        else:
            a.gamma, a.beta = g, b = gamma.detach(), beta.detach()       # (the same version counters)
            ga, ba = _arena(gamma), _arena(beta)
            a._made = ga, _token(g, ga), ba, _token(b, ba)
        return a

    @classmethod
    def _held(cls, *values):
        a = object.__new__(cls)
        a.q, a.e, a.gamma, a.beta, a.relu, a._made = *values, None
        return a

    def __reduce__(self):
        """Copied and saved with the parameters as they are, which nobody else changes then; not with the arena they live in."""
        self._current()
        return Act8._held, (self.q, self.e, self.gamma, self.beta, self.relu)

    def __copy__(self):
        a = Act8._held(self.q, self.e, self.gamma, self.beta, self.relu)
        a._made = self._made
        return a

    def _current(self):
        """Refuses values of a norm whose parameters have changed since."""
        m = self._made
        if m is not None and (_token(self.gamma, m[0]) != m[1] or _token(self.beta, m[2]) != m[3]):
            raise lib.HificError("this Act8 holds a norm's output as its normalised values, and the norm's gamma or beta have changed since")
        return self

    @property
    def fmt(self):
        return "int8" if self.q.dtype == torch.int8 else "e4m3"

    @property
    def shape(self):
        return self.q.shape

    @property
    def nbytes(self):
        return self.q.numel() + self.e.numel()

    def tensors(self):
        """What an autograd node saves."""
        return self.q, self.e, self.gamma, self.beta


def _new8(x, dt):
    return torch.empty_like(x, dtype=dt), torch.empty(_tokens(x), dtype=torch.uint8, device=x.device)


def checkpoint8(x, fmt="int8"):
    """x (float32 or bfloat16, [N, C, ...]) -> Act8.  Carries no gradient: it is what a backward pass keeps of x."""
    code, dt = _fmt(fmt)
    N, C, HW = _nchw(x)
    _one_device(x)
    x = c16(x)
    cd = lib.dtype_code(x)
    q, e = _new8(x, dt)
    if N and HW:
        _launch("hific_act8_pack", x, x.data_ptr(), q.data_ptr(), e.data_ptr(), code, N, C, HW, cd)
    return Act8._of(q, e)


def restore8(a, dtype=torch.bfloat16):
    """The values that `a` stands for, in float32 or bfloat16."""
    if not isinstance(a, Act8):
        raise lib.HificError(f"restore8 needs an Act8, got {type(a).__name__}")
    if dtype not in (torch.float32, torch.bfloat16):
        raise lib.HificError(f"restore8: dtype must be torch.float32 or torch.bfloat16, not {dtype}")
    a._current()
    return _restore(a.q, a.e, a.gamma, a.beta, a.relu, dtype)


def _restore(q, e, gamma, beta, relu, dtype):
    out = torch.empty_like(q, dtype=dtype)
    N, C, HW = _nchw(q)
    if N and HW:
        _launch("hific_act8_restore", q, q.data_ptr(), e.data_ptr(), _CODE[q.dtype], ptr(gamma), ptr(beta), int(relu), out.data_ptr(),
                N, C, HW, lib.HIFIC_F32 if dtype is torch.float32 else lib.HIFIC_BF16)
    return out


# ---- root-mean-square norm ---------------------------------------------------------------------------------------------
def _rms_fwd(x, weight, resid, eps, geom, cd, code, dt, want_y, want_rstd):
    """-> y, h, rstd, q, e (None where not asked for; q holds y where y is not asked for, else the normalised values)."""
    N, C, HW = geom
    y = torch.empty_like(x) if want_y else None
    h = torch.empty_like(x) if resid is not None else None
    rstd = torch.empty(_tokens(x), dtype=torch.float32, device=x.device) if want_rstd else None
    q, e = _new8(x, dt) if dt is not None else (None, None)
    if N and HW:
        _launch("hific_rms_norm_fwd", x, x.data_ptr(), ptr(resid), weight.data_ptr(), ptr(y), ptr(h), ptr(rstd), ptr(q), ptr(e), code,
                0 if want_y else 1, N, C, HW, eps, cd)
    return y, h, rstd, q, e


@functools.lru_cache(maxsize=1024)
def _bwd_ws_bytes(N, C, HW):
    return int(lib.raw("hific_norm8_bwd_ws_bytes")(N, C, HW))


def _bwd_ws(N, C, HW, rstd):
    # its own allocation per call (float32, like rstd), not the stream's workspace: two captured graphs that replay on two streams share
    # nothing
    n = _bwd_ws_bytes(N, C, HW)
    return rstd.new_empty(n >> 2), n


class RmsNormFn(Function):
    """y = weight * h * rsqrt(mean_c h^2 + eps), h = x + resid.  Keeps h (or x), or with a format its normalised form in 8 bits."""

    @staticmethod
    def forward(ctx, x, weight, resid, eps, geom, cd, code, dt):
        y, h, rstd, q, e = _rms_fwd(x, weight, resid, eps, geom, cd, code, dt, True, True)
        ctx.geom, ctx.cd, ctx.code, ctx.slot = geom, cd, code, ops._slot(weight)
        ctx.has_resid = resid is not None
        ctx.set_materialize_grads(False)
        if dt is not None:
            ctx.save_for_backward(q, e, rstd, weight)
        else:
            ctx.save_for_backward(x if h is None else h, None, rstd, weight)
        return y if h is None else (y, h)

    @staticmethod
    @_first_order
    def backward(ctx, dy, dstream=None):
        kept, e, rstd, weight = ctx.saved_tensors
        none = (None,) * 5
        if dy is None:                                   # only the stream was used
            return (dstream, None, dstream if ctx.has_resid else None) + none
        dy = c16(dy)
        if dstream is not None:
            dstream = c16(dstream)
        want_w = ctx.needs_input_grad[1]
        dwt, acc, dw = ops._grad_target(ctx.slot, weight) if want_w else (torch.empty_like(weight), 0, None)
        dx = torch.empty_like(dy)
        N, C, HW = ctx.geom
        if N and HW:
            ws, n = _bwd_ws(N, C, HW, rstd)
            h, q = (kept.data_ptr(), None) if e is None else (None, kept.data_ptr())
            _launch("hific_rms_norm_bwd", dy, h, q, ptr(e), ctx.code, rstd.data_ptr(), dy.data_ptr(), ptr(dstream), weight.data_ptr(),
                    dx.data_ptr(), dwt.data_ptr(), acc, N, C, HW, ctx.cd, ws.data_ptr(), n)
        elif not acc:
            dwt.zero_()
        if want_w:
            ops._written(ctx.slot)
        return (dx, dw, dx if ctx.has_resid else None) + none


def _rms_args(x, weight, resid):
    """-> x, resid (contiguous, aligned), (N, C, positions), type code."""
    geom = _nchw(x)
    _one_device(x, weight, resid)
    _param(weight, geom[1], "weight")
    if resid is not None:
        _like(resid, x, "resid")
        resid = c16(resid)
    return c16(x), resid, geom, lib.dtype_code(x)


def _needs_grad(x, weight, resid):
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (x, weight, resid)):
        raise lib.HificError("the root-mean-square norm has no forward-mode derivative")
    return torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (resid is not None and resid.requires_grad))


def rms_norm(x, weight, resid=None, eps=1e-6, fmt=None):
    """weight * h / sqrt(mean_c h^2 + eps) over dim 1 of x [N, C, ...] (float32 or bfloat16; weight float32, C values).
    With `resid` (like x): h = x + resid rounded to x's type, and (y, h) is returned - h is the new residual stream, and the norm
    and its backward pass see what it holds.  `fmt` ("int8" | "e4m3"): the backward pass keeps h in 8 bits, normalised."""
    x, resid, geom, cd = _rms_args(x, weight, resid)
    eps = _eps(eps)
    code, dt = (0, None) if fmt is None else _fmt(fmt)
    if _needs_grad(x, weight, resid):
        return RmsNormFn.apply(x, weight, resid, eps, geom, cd, code, dt)
    y, h, _, _, _ = _rms_fwd(x, weight, resid, eps, geom, cd, 0, None, True, False)
    return y if h is None else (y, h)


def rms_norm8(x, weight, resid=None, eps=1e-6, fmt="e4m3"):
    """rms_norm with its output in 8 bits: Act8, or (Act8, h) with `resid`.  For inference: it carries no gradient."""
    x, resid, geom, cd = _rms_args(x, weight, resid)
    eps = _eps(eps)
    code, dt = _fmt(fmt)
    if _needs_grad(x, weight, resid):
        raise lib.HificError("rms_norm8 carries no gradient: call it under torch.no_grad(), or rms_norm(fmt=...) in training")
    _, h, _, q, e = _rms_fwd(x, weight, resid, eps, geom, cd, code, dt, False, False)
    return Act8._of(q, e) if h is None else (Act8._of(q, e), h)


# ---- channel norm with an 8-bit checkpoint ---------------------------------------------------------------------------------
def _cn8_fwd(x, gamma, beta, resid, eps, relu, geom, cd, code, dt):
    """-> y, rstd, q, e (normalised values), q2, e2 (y in 8 bits, with resid)."""
    N, C, HW = geom
    y = torch.empty_like(x)
    rstd = torch.empty(_tokens(x), dtype=torch.float32, device=x.device)
    q, e = _new8(x, dt)
    q2, e2 = _new8(x, dt) if resid is not None else (None, None)
    if N and HW:
        _launch("hific_channelnorm8_fwd", x, x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), ptr(resid), y.data_ptr(), rstd.data_ptr(),
                q.data_ptr(), e.data_ptr(), ptr(q2), ptr(e2), code, N, C, HW, eps, int(relu), cd)
    return y, rstd, q, e, q2, e2


def _cn8_bwd(q, e, rstd, dy, gamma, beta, relu, dg, db, acc, dprev=None, acc_prev=0, geom=None):
    N, C, HW = geom or _nchw(dy)
    dx = torch.empty_like(dy)
    if N and HW:
        ws, n = _bwd_ws(N, C, HW, rstd)
        _launch("hific_channelnorm8_bwd", dy, q.data_ptr(), e.data_ptr(), _CODE[q.dtype], rstd.data_ptr(), dy.data_ptr(), gamma.data_ptr(),
                beta.data_ptr(), dx.data_ptr(), dg.data_ptr(), db.data_ptr(), acc, ptr(dprev), acc_prev, N, C, HW, int(relu),
                lib.dtype_code(dy), ws.data_ptr(), n)
    else:
        for t, a in ((dg, acc), (db, acc), (dprev, acc_prev)):
            if t is not None and not a:
                t.zero_()
    return dx


def _norm_targets(want, g_slot, gamma, b_slot, beta):
    """(tensors to write for gamma and beta, accumulate flag, values to return to autograd).  The kernel has one flag for both: where one
    of them is added to and the other is written for the first time (one in an arena, one not), the other starts from zeros."""
    if not want:
        return torch.empty_like(gamma), torch.empty_like(beta), 0, None, None
    dgt, acc_g, dg = ops._grad_target(g_slot, gamma)
    dbt, acc_b, db = ops._grad_target(b_slot, beta)
    if acc_g != acc_b:
        (dbt if acc_g else dgt).zero_()
    return dgt, dbt, acc_g | acc_b, dg, db


class ChannelNorm8Fn(Function):
    """ChannelNormFn whose backward pass reads the normalised activation in 8 bits."""

    @staticmethod
    def forward(ctx, x, gamma, beta, eps, relu, resid, geom, cd, code, dt):
        y, rstd, q, e, q2, e2 = _cn8_fwd(x, gamma, beta, resid, eps, relu, geom, cd, code, dt)
        ctx.relu, ctx.has_resid = relu, resid is not None
        ctx.g_slot, ctx.b_slot = ops._slot(gamma), ops._slot(beta)
        ctx.save_for_backward(q, e, rstd, gamma, beta)
        kept = (q, e) if resid is None else (q2, e2)
        ctx.mark_non_differentiable(*kept)
        ctx.set_materialize_grads(False)
        return (y,) + kept

    @staticmethod
    @_first_order
    def backward(ctx, dy, _q, _e):
        if dy is None:
            return (None,) * 10
        q, e, rstd, gamma, beta = ctx.saved_tensors
        dy = c16(dy)
        want = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dgt, dbt, acc, dg, db = _norm_targets(want, ctx.g_slot, gamma, ctx.b_slot, beta)
        dx = _cn8_bwd(q, e, rstd, dy, gamma, beta, ctx.relu, dgt, dbt, acc)
        if want:
            ops._written(ctx.g_slot, ctx.b_slot)
        return (dx, dg, db, None, None, dy if ctx.has_resid else None) + (None,) * 4


def _norm_args(x, gamma, beta, name):
    geom = _nchw(x)
    if geom[1] < 2:
        raise lib.HificError(f"{name} needs at least two channels (unbiased variance)")
    _one_device(x, gamma, beta)
    _param(gamma, geom[1], "gamma")
    _param(beta, geom[1], "beta")
    return geom


def channel_norm8(x, gamma, beta, eps=1e-3, relu=False, resid=None, fmt="int8"):
    """channel_norm (src/normalisation/channel.py:48-59, with the ReLU or the residual behind it) -> (y, Act8): y as channel_norm
    gives it (but for a position with an infinity or NaN, which stays NaN behind the ReLU too, and one of values above 1e19, whose
    squares leave float32: it is normalised here), and the Act8 stands for y too - what the next convolution's weight gradient reads
    (conv2d(x8=)).  The backward pass of the norm keeps its normalised input in 8 bits and nothing else of x or y.  With `relu` the
    kept values are on the same side of the ReLU as the forward values."""
    geom = _norm_args(x, gamma, beta, "channel_norm8")
    code, dt = _fmt(fmt)
    cd = lib.dtype_code(x)
    if resid is not None:
        _one_device(x, resid)
        _like(resid, x, "resid")
        resid = c16(resid)
    y, q, e = ChannelNorm8Fn.apply(c16(x), gamma, beta, _eps(eps), bool(relu), resid, geom, cd, code, dt)
    if resid is not None:
        return y, Act8._of(q, e)
    return y, Act8._of(q, e, gamma, beta, bool(relu))


def channel_norm_grad8(a, dy, gamma, beta, rstd, relu=False):
    """(dx, dgamma, dbeta) of channel_norm8 from what its forward pass kept: `a` the normalised values (q, e), `rstd` float32
    [N, ...] the reciprocal standard deviations, dy float32 or bfloat16.  Carries no gradient."""
    if not isinstance(a, Act8) or a.gamma is not None:
        raise lib.HificError("channel_norm_grad8 needs the normalised values as an Act8 without gamma / beta")
    geom = _norm_args(a.q, gamma, beta, "channel_norm_grad8")
    if dy.shape != a.q.shape:
        raise lib.HificError(f"dy must be {tuple(a.shape)}, got {tuple(dy.shape)}")
    _one_device(a.q, dy, rstd)
    _param(rstd, a.e.numel(), "rstd")
    lib.dtype_code(dy)
    dg, db = torch.empty_like(gamma), torch.empty_like(beta)
    return _cn8_bwd(a.q, a.e, rstd, c16(dy), gamma, beta, bool(relu), dg, db, 0, geom=geom), dg, db


# ---- training with 8-bit checkpoints ---------------------------------------------------------------------------------------------
# Every conv -> ChannelNorm block of the Generator (and of the Encoder where it runs the plain chain) keeps, for its backward pass,
# the normalised values in 8 bits and nothing else: they serve the norm's own backward pass and, with gamma / beta, stand for the
# block's output in the next convolution's weight gradient - 1 byte per element in the place of two bfloat16 tensors (4).
# HIFIC_CHECKPOINT8=int8|e4m3 / hific_amd.set_checkpoint8(...); off by default.
_CHECKPOINT8 = os.environ.get("HIFIC_CHECKPOINT8", "") or None
if _CHECKPOINT8 is not None:
    _fmt(_CHECKPOINT8)


def set_checkpoint8(fmt):
    """"int8" | "e4m3": training forwards keep 8-bit activations (see above); None: bfloat16 / float32 ones.  Where it acts: the Generator's
    fused conv -> ChannelNorm chain, and the Encoder's with set_exact_index(False).  Everything else keeps what it kept: the exact chains
    (set_exact_training, set_exact_reconstruction, set_exact_index), instance norms, a Generator that samples noise, the hyperprior and
    the Discriminator."""
    global _CHECKPOINT8
    if fmt is not None:
        _fmt(fmt)
    _CHECKPOINT8 = fmt


def checkpoint8_fmt():
    return _CHECKPOINT8


def _conv_geom(x, weight, geom):
    """(N, C, H, W, K, R, S, OH, OW); geom of 3 entries: nn.ConvTranspose2d, of 6: nn.Conv2d."""
    N, C, H, W = x.shape
    if len(geom) == 3:
        stride, pad, outpad = geom
        Cw, K, R, S = weight.shape
        OH, OW = (H - 1) * stride - 2 * pad + R + outpad, (W - 1) * stride - 2 * pad + S + outpad
    else:
        stride, pt, pl, pb, pr, _ = geom
        K, Cw, R, S = weight.shape
        OH, OW = (H + pt + pb - R) // stride + 1, (W + pl + pr - S) // stride + 1
    if Cw != C:
        raise lib.HificError(f"channel mismatch: input {C}, weight {Cw}")
    return N, C, H, W, K, R, S, OH, OW


def _conv_fwd(x, weight, bias, geom, out_f32):
    cd = ops._cd()
    if cd == lib.HIFIC_F32 and x.dtype != torch.float32:
        raise lib.HificError("float32 compute mode needs float32 activations")
    N, C, H, W, K, R, S, OH, OW = _conv_geom(x, weight, geom)
    z = torch.empty((N, K, OH, OW), dtype=torch.float32 if cd == lib.HIFIC_F32 or out_f32 else torch.bfloat16, device=x.device)
    flags = (ops._is_f32(x) | ops._is_f32(z) << 1) if cd == lib.HIFIC_BF16 else 0
    wsp, wsb = ops._ws(x)
    if len(geom) == 3:
        wc = ops._wcache(weight, 0, (N, C, H, W, K, R, S) + geom, cd, flags, None, transposed=True)
        lib.call("hific_conv_transpose2d_fwd", ptr(x), ptr(weight), ptr(bias), ptr(z), N, C, H, W, K, R, S, *geom, lib.ACT_NONE, cd,
                 flags, wsp, wsb, *wc, stream())
    else:
        wc = ops._wcache(weight, 0, (N, C, H, W, K, R, S) + geom, cd, flags, None)
        lib.call("hific_conv2d_fwd", ptr(x), ptr(weight), None, ptr(bias), None, ptr(z), N, C, H, W, K, R, S, *geom, lib.ACT_NONE, cd,
                 flags, wsp, wsb, *wc, stream())
    return z


def _conv_bwd_data(dz, weight, geom, shape, dtype, cd):
    dx = torch.empty(shape, dtype=dtype, device=dz.device)
    N, C, H, W, K, R, S, _, _ = _conv_geom(dx, weight, geom)
    flags = (ops._is_f32(dz) | ops._is_f32(dx) << 1) if cd == lib.HIFIC_BF16 else 0
    wsp, wsb = ops._ws(dz)
    wc = ops._wcache(weight, 1, (N, C, H, W, K, R, S) + geom, cd, flags, None, transposed=len(geom) == 3)
    if len(geom) == 3:
        lib.call("hific_conv_transpose2d_bwd_data", ptr(dz), ptr(weight), ptr(dx), N, C, H, W, K, R, S, *geom, cd, flags, wsp, wsb, *wc,
                 stream())
    else:
        lib.call("hific_conv2d_bwd_data", ptr(dz), ptr(weight), None, ptr(dx), N, C, H, W, K, R, S, *geom, cd, flags, wsp, wsb, *wc,
                 stream())
    return dx


def _kept_input(x, q, e, gamma, beta):
    """What a convolution keeps of its input: the 8-bit form of it, or (no q) the tensor itself."""
    return (x, None, None, None) if q is None else (q, e, gamma, beta)


def _weight_grad(kept, relu, dz, dw, acc, geom, cd):
    x, e, gamma, beta = kept
    if e is not None:
        return _conv_wgrad8(kept, relu, dz, dw, acc, geom, cd)
    N, C, H, W = x.shape
    R, S = dw.shape[2], dw.shape[3]
    K = dz.shape[1]
    flags = (ops._is_f32(x) | ops._is_f32(dz) << 1) if cd == lib.HIFIC_BF16 else 0
    if len(geom) == 3:        # (the transposed form's first operand is the input)
        lib.call("hific_conv_transpose2d_bwd_weight", ptr(x), ptr(dz), ptr(dw), N, C, H, W, K, R, S, *geom, acc, cd, flags, *ops._ws(x),
                 stream())
    else:
        lib.call("hific_conv2d_bwd_weight", ptr(x), ptr(dz), ptr(dw), N, C, H, W, K, R, S, *geom, acc, cd, flags, *ops._ws(x), stream())


def _conv_backward(ctx, kept, relu, dz, weight, want_x, want_w, after=None, after_slot=None):
    """Data gradient on the current stream; weight gradient (and `after`, which writes `after_slot`) next to it on the side stream where
    every gradient made there is written into an arena: one that autograd gets is read on the current stream at once.  -> dx, dw"""
    side = want_w and ops._use_side(ctx.w_slot, after_slot if after is not None else True)
    ev = lib.stream_obj().record_event() if side else None
    dx = _conv_bwd_data(dz, weight, ctx.geom, ctx.x_shape, ctx.x_dtype, ctx.mode) if want_x else None
    dw = None

    def params():
        nonlocal dw
        if want_w:
            dwt, acc, dw = ops._grad_target(ctx.w_slot, weight)
            _weight_grad(kept, relu, dz, dwt, acc, ctx.geom, ctx.mode)
        if after is not None:
            after()
    if side:
        with ops._SideLaunch(ev, *kept, dz, key=ctx.w_slot):
            params()
    else:
        params()
    if want_w:
        ops._written(ctx.w_slot)
    return dx, dw


class ConvNorm8Fn(Function):
    """ops.ConvNormFn that keeps 8-bit activations: conv (nn.ConvTranspose2d: geom of 3 entries) -> ChannelNorm[+ReLU][+residual].
    q, e, xg, xb, xrelu: the 8-bit form of x (its weight gradient reads it); without q, x itself is kept."""

    @staticmethod
    def forward(ctx, x, q, e, xg, xb, xrelu, weight, bias, geom, gamma, beta, eps, relu, resid, code, dt):
        require_gpu(x, weight, bias, gamma, beta, resid)
        with _on(x):
            z = _conv_fwd(x, weight, bias, geom, False)
            _param(gamma, z.size(1), "gamma")
            _param(beta, z.size(1), "beta")
            if resid is not None:
                _like(resid, z, "resid")
            y, rstd, nq, ne, q2, e2 = _cn8_fwd(z, gamma, beta, resid, eps, relu, _nchw(z), lib.dtype_code(z), code, dt)
        ctx.geom, ctx.relu, ctx.xrelu, ctx.mode = geom, relu, xrelu, ops._cd()
        ctx.x_shape, ctx.x_dtype, ctx.has_bias, ctx.has_resid = x.shape, x.dtype, bias is not None, resid is not None
        ctx.w_slot, ctx.b_slot, ctx.g_slot, ctx.be_slot = (ops._slot(t) for t in (weight, bias, gamma, beta))
        ctx.save_for_backward(*_kept_input(x, q, e, xg, xb), weight, nq, ne, rstd, gamma, beta)
        kept = (nq, ne) if resid is None else (q2, e2)
        ctx.mark_non_differentiable(*kept)
        ctx.set_materialize_grads(False)
        return (y,) + kept

    @staticmethod
    @_first_order
    def backward(ctx, dy, _q, _e):
        if dy is None:
            return (None,) * 16
        x, e, xg, xb, weight, nq, ne, rstd, gamma, beta = ctx.saved_tensors
        dy = c16(dy)
        need = ctx.needs_input_grad
        with _on(dy):
            want_n = need[9] or need[10]
            dgt, dbt, acc_g, dg, dbe = _norm_targets(want_n, ctx.g_slot, gamma, ctx.be_slot, beta)
            want_b = ctx.has_bias and need[7]
            dpt, acc_p, db = ops._grad_target(ctx.b_slot, gamma.new_empty(gamma.numel())) if want_b else (None, 0, None)
            dz = _cn8_bwd(nq, ne, rstd, dy, gamma, beta, ctx.relu, dgt, dbt, acc_g, dpt, acc_p)
            if want_n:
                ops._written(ctx.g_slot, ctx.be_slot)
            if want_b:
                ops._written(ctx.b_slot)
            dx, dw = _conv_backward(ctx, (x, e, xg, xb), ctx.xrelu, dz, weight, need[0], need[6])
        return (dx, None, None, None, None, None, dw, db, None, dg, dbe, None, None, dy if ctx.has_resid else None, None, None)


def conv_norm8(x, x8, conv, norm, resid=None, fmt="int8"):
    """ops.conv_norm with 8-bit checkpoints -> (y, Act8 of y).  `x8`: the Act8 that stands for x (the previous block's, or
    checkpoint8(x)), or None to keep x itself."""
    code, dt = _fmt(fmt)
    if conv.transposed:
        geom = (conv.stride[0], conv.padding[0], conv.output_padding[0])
    else:
        geom = (conv.stride[0],) + tuple(conv.pads) + (conv.hip_pad_mode,)
    q, e, xg, xb, xrelu = _split8(x8, x)
    y, q, e = ConvNorm8Fn.apply(c16(x), q, e, xg, xb, xrelu, conv.weight, conv.bias, geom, norm.gamma, norm.beta, _eps(norm.eps),
                                bool(norm.fuse_relu), None if resid is None else c16(resid), code, dt)
    if resid is not None:
        return y, Act8._of(q, e)
    return y, Act8._of(q, e, norm.gamma, norm.beta, bool(norm.fuse_relu))


def _split8(x8, x):
    if x8 is None:
        return None, None, None, None, False
    if not isinstance(x8, Act8) or x8.shape != x.shape:
        raise lib.HificError(f"x8 must be the Act8 of x {tuple(x.shape)}")
    _one_device(x, x8.q)
    x8._current()
    return x8.q, x8.e, x8.gamma, x8.beta, x8.relu


class Conv8Fn(Function):
    """conv2d whose weight gradient reads the 8-bit form of its input (ops.conv2d with x8=)."""

    @staticmethod
    def forward(ctx, x, q, e, xg, xb, xrelu, weight, bias, geom, out_f32, bias_grad):
        require_gpu(x, weight, bias)
        with _on(x):
            y = _conv_fwd(x, weight, bias, geom, out_f32)
        ctx.geom, ctx.xrelu, ctx.mode = geom, xrelu, ops._cd()
        ctx.x_shape, ctx.x_dtype, ctx.has_bias, ctx.bias_grad = x.shape, x.dtype, bias is not None, bool(bias_grad)
        ctx.w_slot, ctx.b_slot = ops._slot(weight), ops._slot(bias)
        ctx.save_for_backward(q, e, xg, xb, weight)
        return y

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        q, e, xg, xb, weight = ctx.saved_tensors
        dy = c16(dy)
        need = ctx.needs_input_grad
        db = None
        want_b = ctx.has_bias and need[7] and ctx.bias_grad

        def bias():
            nonlocal db
            K, plane = dy.shape[1], dy.shape[2] * dy.shape[3]
            dbt, acc, db = ops._grad_target(ctx.b_slot, weight.new_empty(K))
            lib.call("hific_channel_sum", ptr(dy), ptr(dbt), dy.shape[0], K, plane, acc, lib.dtype_code(dy), *ops._ws(dy), stream())
        with _on(dy):
            dx, dw = _conv_backward(ctx, (q, e, xg, xb), ctx.xrelu, dy, weight, need[0], need[6], bias if want_b else None, ctx.b_slot)
            if want_b:
                ops._written(ctx.b_slot)
        return (dx, None, None, None, None, None, dw, db, None, None, None)


def conv2d8(x, x8, weight, bias, geom, out_f32, bias_grad):
    q, e, xg, xb, xrelu = _split8(x8, x)
    return Conv8Fn.apply(c16(x), q, e, xg, xb, xrelu, weight, bias, geom, out_f32, bias_grad)


# ---- weight gradients of convolutions from an 8-bit input ------------------------------------------------------------------
# The convolution kernels address one call's tensors with 32-bit element offsets: larger batches go in slices of whole samples
_MAX_ELEMENTS = 2 ** 31 - 1


def _slices(N, per_sample):
    if per_sample > _MAX_ELEMENTS:
        raise lib.HificError(f"weight gradient: one sample of {per_sample} elements is beyond 32-bit offsets")
    step = max(1, min(N, _MAX_ELEMENTS // max(1, per_sample)))
    return [(i, min(N, i + step)) for i in range(0, N, step)]


@functools.lru_cache(maxsize=1024)
def _wgrad8_ws_bytes(*shape):
    """Workspace of the kernel that reads the 8-bit tensor itself; 0 where restoring it for the natural-order kernels is faster."""
    return int(lib.raw("hific_wgrad8_ws_bytes")(*shape)) if lib.raw("hific_wgrad8_prefer")(*shape) else 0


def _graph_ws(x, tr, geom, N, C, H, W, K, R, S, cd):
    """Workspace of the restored form: the stream's, or inside a graph capture one of the graph's own (two graphs captured on one
    stream may replay on two)."""
    if not torch.cuda.is_current_stream_capturing():
        return ops._ws(x)
    if tr:
        n = lib.raw("hific_conv_transpose2d_ws_bytes")(N, C, H, W, K, R, S, *geom, cd)
    else:
        n = lib.raw("hific_conv2d_ws_bytes")(N, C, H, W, K, R, S, *geom[:5], cd)
    ws = torch.empty(n, dtype=torch.uint8, device=x.device)
    return ws.data_ptr(), n


def _conv_wgrad8(saved, relu, dy, dw, acc, geom, cd, own_ws=False):
    """dw (=|+=) sum dy * pad(x), x the values of `saved` (q, e, gamma, beta) restored to the compute type `cd`; geom of 3 entries:
    nn.ConvTranspose2d."""
    q, e, gamma, beta = saved
    N, C, H, W = q.shape
    K, R, S = dy.shape[1], dw.shape[2], dw.shape[3]
    name = "hific_conv_transpose2d_bwd_weight" if len(geom) == 3 else "hific_conv2d_bwd_weight"
    xt = torch.float32 if cd == lib.HIFIC_F32 else torch.bfloat16
    flags = ops._is_f32(dy) << 1 if cd == lib.HIFIC_BF16 else 0
    tr, OH, OW = int(len(geom) == 3), dy.shape[2], dy.shape[3]
    small = max(C * H * W, K * OH * OW)
    for lo, hi in ((0, N),) if N * small <= _MAX_ELEMENTS else _slices(N, small):
        qs, es, d = (q, e, dy) if hi - lo == N else (q[lo:hi], e[lo:hi], c16(dy[lo:hi]))
        n = _wgrad8_ws_bytes(tr, hi - lo, C, H, W, K, R, S, OH, OW, geom[0]) if dy.dtype is torch.bfloat16 and cd == lib.HIFIC_BF16 else 0
        if n:
            ws = torch.empty(n, dtype=torch.uint8, device=dy.device)
            pt, pl, mode = (geom[1], geom[1], lib.PAD_ZERO) if tr else (geom[1], geom[2], geom[5])
            lib.call("hific_wgrad8", tr, qs.data_ptr(), es.data_ptr(), _CODE[q.dtype], ptr(gamma), ptr(beta), int(relu), d.data_ptr(),
                     dw.data_ptr(), hi - lo, C, H, W, K, R, S, OH, OW, geom[0], pt, pl, mode, acc, ws.data_ptr(), n, stream())
        else:
            x = _restore(qs, es, gamma, beta, relu, xt)
            ws = _graph_ws(x, tr, geom, hi - lo, C, H, W, K, R, S, cd) if own_ws else ops._ws(x)
            lib.call(name, ptr(x), ptr(d), ptr(dw), hi - lo, C, H, W, K, R, S, *geom, acc, cd, flags, *ws, stream())
        acc = 1


def _wgrad_args(a, dy, kernel, name):
    if not isinstance(a, Act8) or a.q.dim() != 4:
        raise lib.HificError(f"{name} needs a 4-dimensional Act8")
    a._current()
    if dy.dim() != 4 or dy.shape[0] != a.shape[0] or dy.shape[1] < 1:
        raise lib.HificError(f"{name}: dy must be [{a.shape[0]}, K, OH, OW], got {tuple(dy.shape)}")
    R, S = (int(k) for k in kernel)
    if R < 1 or S < 1 or R * S > 64:
        raise lib.HificError(f"{name}: kernel {(R, S)} is not supported (1 to 64 taps)")
    _one_device(a.q, dy)
    lib.dtype_code(dy)
    return R, S, c16(dy)


def conv2d_weight_grad8(a, dy, kernel, stride=1, pads=(0, 0, 0, 0), pad_mode=lib.PAD_ZERO):
    """Weight gradient [K, C, R, S] (float32) of conv2d whose input is held as `a`, dy [N, K, OH, OW] float32 or bfloat16: what
    conv2d's backward pass gives for restore8(a, dy.dtype).  In bfloat16 the restored values of a plain Act8 are exact, so the
    products are exact and the sum is float32.  Carries no gradient."""
    R, S, dy = _wgrad_args(a, dy, kernel, "conv2d_weight_grad8")
    N, C, H, W = a.shape
    pt, pl, pb, pr = (int(v) for v in pads)
    stride = int(stride)
    if not 1 <= stride <= _MAX_C or min(pt, pl, pb, pr) < 0 or max(pt, pl, pb, pr) > _MAX_C or pad_mode not in (lib.PAD_ZERO, lib.PAD_REFLECT):
        raise lib.HificError("conv2d_weight_grad8: bad stride, pads or pad_mode")
    if pad_mode == lib.PAD_REFLECT and (max(pt, pb) >= H or max(pl, pr) >= W):
        raise lib.HificError("conv2d_weight_grad8: reflection pads must be smaller than the plane")
    oh, ow = (H + pt + pb - R) // stride + 1, (W + pl + pr - S) // stride + 1
    if oh < 1 or ow < 1 or tuple(dy.shape[2:]) != (oh, ow):
        raise lib.HificError(f"conv2d_weight_grad8: dy must be {(oh, ow)} for planes {(H, W)}, got {tuple(dy.shape[2:])}")
    dw = torch.empty((dy.shape[1], C, R, S), dtype=torch.float32, device=dy.device)
    if N == 0:
        return dw.zero_()
    with _on(dy):
        _conv_wgrad8(a.tensors(), a.relu, dy, dw, 0, (stride, pt, pl, pb, pr, pad_mode), lib.dtype_code(dy), True)
    return dw


def conv_transpose2d_weight_grad8(a, dy, kernel, stride, pad, outpad):
    """Weight gradient [C, K, R, S] (float32) of conv_transpose2d whose input is held as `a`; see conv2d_weight_grad8."""
    R, S, dy = _wgrad_args(a, dy, kernel, "conv_transpose2d_weight_grad8")
    N, C, H, W = a.shape
    stride, pad, outpad = int(stride), int(pad), int(outpad)
    if not 1 <= stride <= _MAX_C or not 0 <= pad <= _MAX_C or not 0 <= outpad <= _MAX_C:
        raise lib.HificError("conv_transpose2d_weight_grad8: bad stride or padding")
    size = ((H - 1) * stride - 2 * pad + R + outpad, (W - 1) * stride - 2 * pad + S + outpad)
    if min(size) < 1 or tuple(dy.shape[2:]) != size:
        raise lib.HificError(f"conv_transpose2d_weight_grad8: dy must be {size} for planes {(H, W)}, got {tuple(dy.shape[2:])}")
    dw = torch.empty((C, dy.shape[1], R, S), dtype=torch.float32, device=dy.device)
    if N == 0:
        return dw.zero_()
    with _on(dy):
        _conv_wgrad8(a.tensors(), a.relu, dy, dw, 0, (stride, pad, outpad), lib.dtype_code(dy), True)
    return dw
