"""Activations in 8 bits, the norms that write and read them, and the root-mean-square norm (csrc/act8.hip, csrc/norm8.hip).

A token is one position of an activation [N, C, ...] (a pixel of [N, C, H, W], a row of [N, C]).  Its C values are held as int8 or
e4m3 numbers with ONE power-of-two exponent per token, so a restored value is exact in bfloat16.  `Act8` is such an activation;
`checkpoint8` / `restore8` pack and restore one, `rms_norm8` writes its output in that form, `rms_norm(fmt=)` and `channel_norm8`
keep what their backward pass needs in it (1 byte per element in the place of a bfloat16 input, and of the next layer's input),
and `conv2d_weight_grad8` / `conv_transpose2d_weight_grad8` contract one.  The functions are part of `hific_amd.ops`.
"""
import contextlib

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import lib
from .lib import call, ptr, stream, require_gpu

FORMATS = {"int8": (0, torch.int8), "e4m3": (1, torch.float8_e4m3fn)}
_CODE = {torch.int8: 0, torch.float8_e4m3fn: 1}
_here = contextlib.nullcontext()


def _on(t):
    """Context in which launches go to the device of `t` (and to that device's current stream)."""
    return _here if t.device.index == lib._cur_device() else torch.cuda.device(t.device)


def _fmt(fmt):
    if fmt not in FORMATS:
        raise lib.HificError(f"8-bit format must be one of {sorted(FORMATS)}, not {fmt!r}")
    return FORMATS[fmt]


def _nchw(x, name="x"):
    """(N, C, positions) of an activation [N, C, ...]."""
    if x.dim() < 2 or x.shape[1] < 1:
        raise lib.HificError(f"{name} must be [N, C, ...] with at least one channel, got {tuple(x.shape)}")
    hw = 1
    for d in x.shape[2:]:
        hw *= d
    return x.shape[0], x.shape[1], hw


def _tokens(x):
    return x.shape[:1] + x.shape[2:]


def _act(x):
    require_gpu_any(x)
    lib.dtype_code(x)                                   # float32 or bfloat16
    return c16(x)


def require_gpu_any(*tensors):
    """require_gpu without the contiguity rule (strided tensors are copied), and all on one device."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            require_gpu(t)
        if dev is not None and t.device != dev:
            raise lib.HificError(f"tensors on {dev} and {t.device}")
        dev = t.device


def c16(t):
    """Contiguous and 16-byte aligned (the wide kernels' accesses): a strided or oddly placed view is copied."""
    t = t.contiguous()
    return t if (t.data_ptr() & 15) == 0 else t.clone(memory_format=torch.contiguous_format)


def _param(w, C, name):
    if w.dtype != torch.float32 or w.numel() != C or not w.is_contiguous():
        raise lib.HificError(f"{name} must be a contiguous float32 tensor of {C} values, got {w.dtype} {tuple(w.shape)}")


def _like(t, x, name):
    if t.shape != x.shape or t.dtype != x.dtype:
        raise lib.HificError(f"{name} must be {x.dtype} {tuple(x.shape)}, got {t.dtype} {tuple(t.shape)}")


def _eps(eps):
    if not 0.0 < eps < float("inf"):
        raise lib.HificError(f"eps must be positive and finite, got {eps}")
    return float(eps)


class Act8:
    """An activation in 8 bits: `q` (int8 or float8_e4m3fn) [N, C, ...] and `e` (uint8, exponent + 127) [N, ...].  With `gamma` /
    `beta` (float32, C values) it stands for relu?(gamma * (q * 2^e) + beta): a norm's output held as its normalised values."""
    __slots__ = ("q", "e", "gamma", "beta", "relu")

    def __init__(self, q, e, gamma=None, beta=None, relu=False):
        if q.dtype not in _CODE or e.dtype != torch.uint8:
            raise lib.HificError(f"Act8: q must be int8 or float8_e4m3fn and e uint8, got {q.dtype} and {e.dtype}")
        _, C, _ = _nchw(q, "q")
        if e.shape != _tokens(q):
            raise lib.HificError(f"Act8: e must be {tuple(_tokens(q))} for q {tuple(q.shape)}, got {tuple(e.shape)}")
        if (gamma is None) != (beta is None) or (relu and gamma is None):
            raise lib.HificError("Act8: gamma and beta come together, and relu with them")
        require_gpu_any(q, e, gamma, beta)
        for t, name in ((gamma, "gamma"), (beta, "beta")):
            if t is not None:
                _param(t, C, name)
        self.q, self.e, self.gamma, self.beta, self.relu = c16(q), c16(e), gamma, beta, bool(relu)

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
    return torch.empty(x.shape, dtype=dt, device=x.device), torch.empty(_tokens(x), dtype=torch.uint8, device=x.device)


def checkpoint8(x, fmt="int8"):
    """x (float32 or bfloat16, [N, C, ...]) -> Act8.  Carries no gradient: it is what a backward pass keeps of x."""
    code, dt = _fmt(fmt)
    N, C, HW = _nchw(x)
    x = _act(x.detach())
    q, e = _new8(x, dt)
    if x.numel():
        with _on(x):
            call("hific_act8_pack", ptr(x), ptr(q), ptr(e), code, N, C, HW, lib.dtype_code(x), stream())
    return Act8(q, e)


def restore8(a, dtype=torch.bfloat16):
    """The values that `a` stands for, in float32 or bfloat16."""
    if not isinstance(a, Act8):
        raise lib.HificError(f"restore8 needs an Act8, got {type(a).__name__}")
    if dtype not in (torch.float32, torch.bfloat16):
        raise lib.HificError(f"restore8: dtype must be torch.float32 or torch.bfloat16, not {dtype}")
    return _restore(a.q, a.e, a.gamma, a.beta, a.relu, dtype)


def _restore(q, e, gamma, beta, relu, dtype):
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    if out.numel():
        N, C, HW = _nchw(q)
        with _on(q):
            call("hific_act8_restore", ptr(q), ptr(e), _CODE[q.dtype], ptr(gamma), ptr(beta), int(relu), ptr(out), N, C, HW,
                 lib.dtype_code(out), stream())
    return out


# ---- root-mean-square norm ---------------------------------------------------------------------------------------------
def _rms_fwd(x, weight, resid, eps, code, dt, want_y, want_rstd, q_of_y):
    """-> y, h, rstd, q, e (None where not asked for; h is x without a residual)."""
    N, C, HW = _nchw(x)
    y = torch.empty_like(x) if want_y else None
    h = torch.empty_like(x) if resid is not None else None
    rstd = torch.empty(_tokens(x), dtype=torch.float32, device=x.device) if want_rstd else None
    q, e = _new8(x, dt) if dt is not None else (None, None)
    if x.numel():
        with _on(x):
            call("hific_rms_norm_fwd", ptr(x), ptr(resid), ptr(weight), ptr(y), ptr(h), ptr(rstd), ptr(q), ptr(e), code,
                 int(q_of_y), N, C, HW, eps, lib.dtype_code(x), stream())
    return y, h, rstd, q, e


def _bwd_ws(N, C, HW, device):
    # its own allocation per call, not the stream's workspace: two captured graphs that replay on two streams share nothing
    n = int(lib.raw("hific_norm8_bwd_ws_bytes")(N, C, HW))
    return torch.empty(n, dtype=torch.uint8, device=device), n


def _rms_bwd(h, q, e, rstd, dy, dstream, weight, dw, acc):
    N, C, HW = _nchw(dy)
    dx = torch.empty_like(dy)
    if dy.numel():
        ws, n = _bwd_ws(N, C, HW, dy.device)
        call("hific_rms_norm_bwd", ptr(h), ptr(q), ptr(e), 0 if q is None else _CODE[q.dtype], ptr(rstd), ptr(dy), ptr(dstream),
             ptr(weight), ptr(dx), ptr(dw), acc, N, C, HW, lib.dtype_code(dy), ptr(ws), n, stream())
    elif not acc:
        dw.zero_()
    return dx


class RmsNormFn(Function):
    """y = weight * h * rsqrt(mean_c h^2 + eps), h = x + resid.  Keeps h (or x), or with `fmt` its normalised form in 8 bits."""

    @staticmethod
    def forward(ctx, x, weight, resid, eps, fmt):
        from . import ops
        code, dt = _fmt(fmt) if fmt is not None else (0, None)
        y, h, rstd, q, e = _rms_fwd(x, weight, resid, eps, code, dt, True, True, False)
        ctx.slot = ops._slot(weight)
        ctx.has_resid, ctx.kept8 = resid is not None, fmt is not None
        ctx.set_materialize_grads(False)
        if fmt is not None:
            ctx.save_for_backward(q, e, rstd, weight)
        else:
            ctx.save_for_backward(x if resid is None else h, rstd, weight)
        return y if resid is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstream=None):
        from . import ops
        if ctx.kept8:
            q, e, rstd, weight = ctx.saved_tensors
            h = None
        else:
            h, rstd, weight = ctx.saved_tensors
            q = e = None
        want_w = ctx.needs_input_grad[1]
        if dy is None:                                   # only the stream was used
            return dstream, None, (dstream if ctx.has_resid else None), None, None
        dy = c16(dy)
        dstream = None if dstream is None else c16(dstream)
        with _on(dy):
            if want_w:
                dwt, acc, dw = ops._grad_target(ctx.slot, weight)
            else:
                dwt, acc, dw = torch.empty_like(weight), 0, None
            dx = _rms_bwd(h, q, e, rstd, dy, dstream, weight, dwt, acc)
            if want_w:
                ops._written(ctx.slot)
        return dx, dw, (dx if ctx.has_resid else None), None, None


def _rms_args(x, weight, resid, eps):
    _, C, _ = _nchw(x)
    require_gpu_any(x, weight, resid)
    _param(weight, C, "weight")
    if resid is not None:
        _like(resid, x, "resid")
        resid = _act(resid)
    return _act(x), resid, _eps(eps)


def rms_norm(x, weight, resid=None, eps=1e-6, fmt=None):
    """weight * h / sqrt(mean_c h^2 + eps) over dim 1 of x [N, C, ...] (float32 or bfloat16; weight float32, C values).
    With `resid` (like x): h = x + resid rounded to x's type, and (y, h) is returned - h is the new residual stream, and the norm
    and its backward pass see what it holds.  `fmt` ("int8" | "e4m3"): the backward pass keeps h in 8 bits, normalised."""
    x, resid, eps = _rms_args(x, weight, resid, eps)
    if fmt is not None:
        _fmt(fmt)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (resid is not None and resid.requires_grad)):
        return RmsNormFn.apply(x, weight, resid, eps, fmt)
    y, h, _, _, _ = _rms_fwd(x, weight, resid, eps, 0, None, True, False, False)
    return y if resid is None else (y, h)


def rms_norm8(x, weight, resid=None, eps=1e-6, fmt="e4m3"):
    """rms_norm with its output in 8 bits: Act8, or (Act8, h) with `resid`.  For inference: it carries no gradient."""
    x, resid, eps = _rms_args(x, weight, resid, eps)
    code, dt = _fmt(fmt)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (resid is not None and resid.requires_grad)):
        raise lib.HificError("rms_norm8 carries no gradient: call it under torch.no_grad(), or rms_norm(fmt=...) in training")
    _, h, _, q, e = _rms_fwd(x, weight, resid, eps, code, dt, False, False, True)
    return Act8(q, e) if resid is None else (Act8(q, e), h)


# ---- channel norm with an 8-bit checkpoint ---------------------------------------------------------------------------------
def _cn8_fwd(x, gamma, beta, resid, eps, relu, fmt):
    code, dt = _fmt(fmt)
    N, C, HW = _nchw(x)
    y = torch.empty_like(x)
    rstd = torch.empty(_tokens(x), dtype=torch.float32, device=x.device)
    q, e = _new8(x, dt)
    q2, e2 = _new8(x, dt) if resid is not None else (None, None)
    if x.numel():
        call("hific_channelnorm8_fwd", ptr(x), ptr(gamma), ptr(beta), ptr(resid), ptr(y), ptr(rstd), ptr(q), ptr(e), ptr(q2),
             ptr(e2), code, N, C, HW, eps, int(relu), lib.dtype_code(x), stream())
    return y, rstd, q, e, q2, e2


def _cn8_bwd(q, e, rstd, dy, gamma, beta, relu, dg, db, acc, dprev=None, acc_prev=0):
    N, C, HW = _nchw(dy)
    dx = torch.empty_like(dy)
    if dy.numel():
        ws, n = _bwd_ws(N, C, HW, dy.device)
        call("hific_channelnorm8_bwd", ptr(q), ptr(e), _CODE[q.dtype], ptr(rstd), ptr(dy), ptr(gamma), ptr(beta), ptr(dx), ptr(dg),
             ptr(db), acc, ptr(dprev), acc_prev, N, C, HW, int(relu), lib.dtype_code(dy), ptr(ws), n, stream())
    else:
        for t, a in ((dg, acc), (db, acc), (dprev, acc_prev)):
            if t is not None and not a:
                t.zero_()
    return dx


class ChannelNorm8Fn(Function):
    """ChannelNormFn whose backward pass reads the normalised activation in 8 bits."""

    @staticmethod
    def forward(ctx, x, gamma, beta, eps, relu, resid, fmt):
        from . import ops
        with _on(x):
            y, rstd, q, e, q2, e2 = _cn8_fwd(x, gamma, beta, resid, eps, relu, fmt)
        ctx.relu, ctx.has_resid = relu, resid is not None
        ctx.g_slot, ctx.b_slot = ops._slot(gamma), ops._slot(beta)
        ctx.save_for_backward(q, e, rstd, gamma, beta)
        kept = (q, e) if resid is None else (q2, e2)
        ctx.mark_non_differentiable(*kept)
        ctx.set_materialize_grads(False)
        return (y,) + kept

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, _q, _e):
        from . import ops
        if dy is None:
            return (None,) * 7
        q, e, rstd, gamma, beta = ctx.saved_tensors
        dy = c16(dy)
        want = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        with _on(dy):
            dgt, acc, dg = ops._grad_target(ctx.g_slot, gamma) if want else (torch.empty_like(gamma), 0, None)
            dbt, acc_b, db = ops._grad_target(ctx.b_slot, beta) if want else (torch.empty_like(beta), 0, None)
            assert acc == acc_b
            dx = _cn8_bwd(q, e, rstd, dy, gamma, beta, ctx.relu, dgt, dbt, acc)
            if want:
                ops._written(ctx.g_slot, ctx.b_slot)
        return dx, dg, db, None, None, (dy if ctx.has_resid else None), None


def channel_norm8(x, gamma, beta, eps=1e-3, relu=False, resid=None, fmt="int8"):
    """channel_norm (src/normalisation/channel.py:48-59, with the ReLU or the residual behind it) -> (y, Act8): y as channel_norm
    gives it, and the Act8 stands for y too - what the next convolution's weight gradient reads (conv2d(x8=)).  The backward pass
    of the norm keeps its normalised input in 8 bits and nothing else of x or y.  With `relu` the kept values are on the same
    side of the ReLU as the forward values."""
    _, C, _ = _nchw(x)
    if C < 2:
        raise lib.HificError("channel_norm8 needs at least two channels (unbiased variance)")
    require_gpu_any(x, gamma, beta, resid)
    _param(gamma, C, "gamma")
    _param(beta, C, "beta")
    _fmt(fmt)
    if resid is not None:
        _like(resid, x, "resid")
        resid = _act(resid)
    y, q, e = ChannelNorm8Fn.apply(_act(x), gamma, beta, _eps(eps), bool(relu), resid, fmt)
    if resid is not None:
        return y, Act8(q, e)
    return y, Act8(q, e, gamma.detach(), beta.detach(), relu)


def channel_norm_grad8(a, dy, gamma, beta, rstd, relu=False):
    """(dx, dgamma, dbeta) of channel_norm8 from what its forward pass kept: `a` the normalised values (q, e), `rstd` float32
    [N, ...] the reciprocal standard deviations, dy float32 or bfloat16."""
    if not isinstance(a, Act8) or a.gamma is not None:
        raise lib.HificError("channel_norm_grad8 needs the normalised values as an Act8 without gamma / beta")
    _, C, _ = _nchw(a.q)
    if C < 2:
        raise lib.HificError("channel_norm_grad8 needs at least two channels (unbiased variance)")
    if dy.shape != a.shape:
        raise lib.HificError(f"dy must be {tuple(a.shape)}, got {tuple(dy.shape)}")
    require_gpu_any(a.q, dy, gamma, beta, rstd)
    _param(gamma, C, "gamma")
    _param(beta, C, "beta")
    _param(rstd, a.e.numel(), "rstd")
    dy = _act(dy.detach())
    dg, db = torch.empty_like(gamma), torch.empty_like(beta)
    with _on(dy):
        dx = _cn8_bwd(a.q, a.e, rstd, dy, gamma, beta, bool(relu), dg, db, 0)
    return dx, dg, db


# ---- weight gradients of convolutions from an 8-bit input ------------------------------------------------------------------
# The convolution kernels address one call's tensors with 32-bit element offsets: larger batches go in slices of whole samples
_MAX_ELEMENTS = 2 ** 31 - 1


def _slices(N, per_sample):
    if per_sample > _MAX_ELEMENTS:
        raise lib.HificError(f"weight gradient: one sample of {per_sample} elements is beyond 32-bit offsets")
    step = max(1, min(N, _MAX_ELEMENTS // max(1, per_sample)))
    return [(i, min(N, i + step)) for i in range(0, N, step)]


def _conv_wgrad8(saved, relu, dy, dw, acc, geom):
    """dw (=|+=) sum dy * pad(x), x the values of `saved` (q, e, gamma, beta) restored to dy's type."""
    from . import ops
    q, e, gamma, beta = saved
    stride, pt, pl, pb, pr, pad_mode = geom
    N, C, H, W = q.shape
    K, R, S = dw.shape[0], dw.shape[2], dw.shape[3]
    cd = lib.dtype_code(dy)
    per = max(C * H * W, K * dy.shape[2] * dy.shape[3])
    for lo, hi in _slices(N, per):
        x = _restore(q[lo:hi], e[lo:hi], gamma, beta, relu, dy.dtype)
        d = c16(dy[lo:hi])
        call("hific_conv2d_bwd_weight", ptr(x), ptr(d), ptr(dw), hi - lo, C, H, W, K, R, S, stride, pt, pl, pb, pr, pad_mode, acc,
             cd, 0, *ops._ws(x), stream())
        acc = 1


def _convt_wgrad8(saved, relu, dy, dw, acc, geom):
    from . import ops
    q, e, gamma, beta = saved
    stride, pad, outpad = geom
    N, C, H, W = q.shape
    K, R, S = dw.shape[1], dw.shape[2], dw.shape[3]
    cd = lib.dtype_code(dy)
    for lo, hi in _slices(N, max(C * H * W, K * dy.shape[2] * dy.shape[3])):
        x = _restore(q[lo:hi], e[lo:hi], gamma, beta, relu, dy.dtype)
        d = c16(dy[lo:hi])
        call("hific_conv_transpose2d_bwd_weight", ptr(x), ptr(d), ptr(dw), hi - lo, C, H, W, K, R, S, stride, pad, outpad, acc,
             cd, 0, *ops._ws(x), stream())
        acc = 1


def _wgrad_args(a, dy, kernel, name):
    if not isinstance(a, Act8) or a.q.dim() != 4:
        raise lib.HificError(f"{name} needs a 4-dimensional Act8")
    if dy.dim() != 4 or dy.shape[0] != a.shape[0] or dy.shape[1] < 1:
        raise lib.HificError(f"{name}: dy must be [{a.shape[0]}, K, OH, OW], got {tuple(dy.shape)}")
    R, S = (int(k) for k in kernel)
    if R < 1 or S < 1 or R * S > 64:
        raise lib.HificError(f"{name}: kernel {(R, S)} is not supported (1 to 64 taps)")
    require_gpu_any(a.q, dy)
    return R, S, _act(dy.detach())


def conv2d_weight_grad8(a, dy, kernel, stride=1, pads=(0, 0, 0, 0), pad_mode=lib.PAD_ZERO):
    """Weight gradient [K, C, R, S] (float32) of conv2d whose input is held as `a`, dy [N, K, OH, OW] float32 or bfloat16: what
    conv2d's backward pass gives for restore8(a, dy.dtype).  In bfloat16 the restored values of a plain Act8 are exact, so the
    products are exact and the sum is float32."""
    R, S, dy = _wgrad_args(a, dy, kernel, "conv2d_weight_grad8")
    N, C, H, W = a.shape
    pt, pl, pb, pr = (int(v) for v in pads)
    stride = int(stride)
    if stride < 1 or min(pt, pl, pb, pr) < 0 or pad_mode not in (lib.PAD_ZERO, lib.PAD_REFLECT):
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
        _conv_wgrad8(a.tensors(), a.relu, dy, dw, 0, (stride, pt, pl, pb, pr, pad_mode))
    return dw


def conv_transpose2d_weight_grad8(a, dy, kernel, stride, pad, outpad):
    """Weight gradient [C, K, R, S] (float32) of conv_transpose2d whose input is held as `a`; see conv2d_weight_grad8."""
    R, S, dy = _wgrad_args(a, dy, kernel, "conv_transpose2d_weight_grad8")
    N, C, H, W = a.shape
    stride, pad, outpad = int(stride), int(pad), int(outpad)
    if stride < 1 or pad < 0 or outpad < 0:
        raise lib.HificError("conv_transpose2d_weight_grad8: bad stride or padding")
    size = ((H - 1) * stride - 2 * pad + R + outpad, (W - 1) * stride - 2 * pad + S + outpad)
    if min(size) < 1 or tuple(dy.shape[2:]) != size:
        raise lib.HificError(f"conv_transpose2d_weight_grad8: dy must be {size} for planes {(H, W)}, got {tuple(dy.shape[2:])}")
    dw = torch.empty((C, dy.shape[1], R, S), dtype=torch.float32, device=dy.device)
    if N == 0:
        return dw.zero_()
    with _on(dy):
        _convt_wgrad8(a.tensors(), a.relu, dy, dw, 0, (stride, pad, outpad))
    return dw
