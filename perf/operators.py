"""Cases of the 8-bit activation operators: root-mean-square norm (with the residual's addition, and with an 8-bit
output), activation checkpoints in 8 bits, the channel norm that keeps such a checkpoint, and the weight gradient of a
convolution that reads one.

A token is one position of an activation tensor [N, C, ...]: a pixel of a plane [N, C, H, W] or a row of [N, C].  All
operators work on the C values of a token.  Eight bits are held as (q, e): q is int8 or e4m3 (finite-only, largest value
448) of the tensor's shape, e one exponent per token stored with a bias of 127; the value is q * 2^e, and e is the
smallest exponent with max|v| <= QMAX * 2^e.  Powers of two make every restored value exact in bfloat16.
"""
import math

import torch
import torch.nn.functional as F

own = False

RMS_EPS, NORM_EPS = 1e-6, 1e-3
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one token through a pre-norm block when the output is wanted at once: latency
        dict(name="rms one token", op="rms", n=1, c=960, h=1, w=1, type="bf16", resid=True, grad=False),
        # a training step's pre-norm over the tokens of 16 planes of 64x64 at the residual trunk's width
        dict(name="rms train tokens", op="rms", n=65536, c=960, h=1, w=1, type="bf16", resid=True, grad=True),
        # the same in the framework's plane layout, at the width of the 64x64 stage
        dict(name="rms train planes", op="rms", n=16, c=240, h=64, w=64, type="bf16", resid=True, grad=True),
        # a batch of tokens whose normalised form goes on in 8 bits
        dict(name="rms8 tokens", op="rms8", n=256, c=960, h=1, w=1, type="bf16", resid=True, fmt="e4m3"),
        # float32 latents of a wide image, 220 channels
        dict(name="rms8 latents f32", op="rms8", n=4, c=220, h=64, w=96, type="f32", resid=False, fmt="int8"),
        # latents of images whose planes are odd: nothing is aligned
        dict(name="checkpoint odd planes", op="checkpoint", n=3, c=220, h=45, w=31, type="bf16", fmt="int8"),
        # the largest activation of a 256x256 training batch: 60 channels at full resolution
        dict(name="checkpoint full planes", op="checkpoint", n=16, c=60, h=256, w=256, type="bf16", fmt="e4m3"),
        # norm + ReLU behind an up-convolution of the Generator in training, kept in 8 bits
        dict(name="norm8 upconv", op="norm8", n=16, c=120, h=128, w=128, type="bf16", relu=True, resid=False, fmt="int8"),
        # its backward pass in the residual trunk, and at full resolution
        dict(name="norm8 grad trunk", op="norm8_grad", n=16, c=960, h=16, w=16, type="bf16", relu=True, fmt="int8"),
        dict(name="norm8 grad full planes", op="norm8_grad", n=16, c=60, h=256, w=256, type="bf16", relu=True, fmt="int8"),
        # weight gradients: the residual trunk's 3x3, and a strided layer on odd planes
        dict(name="weight grad trunk", op="wgrad", n=16, c=960, h=16, w=16, k=960, r=3, stride=1, pad="reflect", fmt="int8"),
        dict(name="weight grad odd stride 2", op="wgrad", n=2, c=120, h=61, w=47, k=240, r=3, stride=2, pad="zero", fmt="e4m3"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rms", "rms", "rms8", "checkpoint", "norm8", "norm8_grad", "wgrad"])
    fmt = rng.choice(["int8", "e4m3"])
    kind = rng.choice(["f32", "bf16", "bf16"])
    if op == "wgrad":
        r = rng.choice([1, 3, 3, 5])
        case = dict(op=op, n=_log(rng, 1, 16), c=_log(rng, 16, 960), h=_log(rng, 8, 96), w=_log(rng, 8, 96),
                    k=_log(rng, 16, 960), r=r, stride=rng.choice([1, 2]), pad=rng.choice(["zero", "reflect"]), fmt=fmt)
        while case["n"] * case["h"] * case["w"] * case["c"] * r * r > 36_000_000 or work(case)["flops"] > 6.7e10:
            case[rng.choice(["c", "k"])] = _log(rng, 16, 240)
            case["n"] = max(1, case["n"] // 2)
        return case
    rows = op in ("rms", "rms8") and rng.random() < 0.5
    c = _log(rng, 2, 4096 if rows else 1024)
    most = 60_000_000
    if rows:
        n, h, w = _log(rng, 1, max(1, min(65536, most // c))), 1, 1
    else:
        h, w = _log(rng, 2, 256), _log(rng, 2, 256)
        if rng.random() < 0.5:
            w = max(8, w // 8 * 8)
        while h * w * c > most // 2:
            h = max(1, h // 2)
        n = _log(rng, 1, max(1, min(16, most // (c * h * w))))
    case = dict(op=op, n=n, c=c, h=h, w=w, type=kind)
    if op == "rms":
        case.update(resid=rng.random() < 0.6, grad=rng.random() < 0.6)
    elif op == "rms8":
        case.update(resid=rng.random() < 0.6, fmt=fmt)
    elif op == "checkpoint":
        case.update(fmt=fmt)
    elif op == "norm8":
        case.update(type="bf16", relu=rng.random() < 0.6, resid=rng.random() < 0.4, fmt=fmt)
    else:
        case.update(relu=rng.random() < 0.6, fmt=fmt)
    return case


def _out_size(case):
    p = case["r"] // 2
    return ((case["h"] + 2 * p - case["r"]) // case["stride"] + 1, (case["w"] + 2 * p - case["r"]) // case["stride"] + 1)


def work(case):
    n, c, hw = case["n"], case["c"], case["h"] * case["w"]
    el, tok = n * c * hw, n * hw
    if case["op"] == "wgrad":
        oh, ow = _out_size(case)
        taps = case["r"] ** 2
        return {"bytes": el + tok + 2 * n * case["k"] * oh * ow + 4 * case["k"] * c * taps,
                "flops": 2 * n * oh * ow * case["k"] * c * taps}
    t = 2 if case["type"] == "bf16" else 4
    if case["op"] == "rms":
        b = t * el * (4 if case["resid"] else 2) + 4 * c                       # x, resid -> y, stream
        if case["grad"]:
            b += t * el * (4 if case["resid"] else 3) + 8 * c                  # stream (or x), dy, dstream -> dx; weight -> dweight
        return {"bytes": b, "flops": (14 if case["grad"] else 5) * el}
    if case["op"] == "rms8":
        # int8 is restored to the values it stands for
        back = 0 if case["fmt"] == "e4m3" else (1 + t) * el + tok
        return {"bytes": t * el * (3 if case["resid"] else 1) + el + tok + 4 * c + back, "flops": 6 * el}
    if case["op"] == "checkpoint":
        return {"bytes": 2 * ((t + 1) * el + tok), "flops": 4 * el}
    if case["op"] == "norm8":
        # x (and resid) -> y, q and, with resid, the 8 bits of y; restored once
        return {"bytes": (2 * t + 1) * el + (t + 1) * el * case["resid"] + 9 * tok + 8 * c + (1 + t) * el, "flops": 14 * el}
    return {"bytes": (2 * t + 1) * el + 5 * tok + 16 * c, "flops": 16 * el}     # q, dy -> dx


def _shape(case):
    return (case["n"], case["c"]) if case["h"] * case["w"] == 1 else (case["n"], case["c"], case["h"], case["w"])


def _qmax(fmt):
    return 127.0 if fmt == "int8" else 448.0


def _exponent(amax, fmt):
    """Smallest e with amax <= QMAX * 2^e (at least -126): QMAX is 0.9921875 * 2^7 or 0.875 * 2^9."""
    m, k = torch.frexp(amax)
    frac, bits = (0.9921875, 7) if fmt == "int8" else (0.875, 9)
    e = k - bits + (m > frac)
    return torch.where(amax > 0, e.clamp(min=-126), torch.full_like(e, -126))


def _pow2(e, like):
    return torch.ldexp(torch.ones((), dtype=like.dtype, device=like.device), e)


def _round_to(t, fmt):
    """t rounded to the format's values (half to even)."""
    return torch.round(t) if fmt == "int8" else t.float().to(torch.float8_e4m3fn).to(t.dtype)


def _next_to(q, up, fmt):
    """The format's value next to q, above or below."""
    step = torch.where(up, 1, -1)
    if fmt == "int8":
        return q + step
    bits = q.float().to(torch.float8_e4m3fn).view(torch.uint8).to(torch.int16)
    key = torch.where(bits > 127, -(bits & 127), bits) + step
    code = torch.where(key < 0, 128 - key, key).to(torch.uint8)
    return code.view(torch.float8_e4m3fn).to(q.dtype)


def _quantise(v, fmt):
    """(q as values, e) of v, one exponent per token."""
    e = _exponent(v.abs().amax(1, keepdim=True), fmt)
    return _round_to(v * _pow2(-e, v), fmt), e


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    shape, op = _shape(case), case["op"]

    def normal(*size):
        return torch.randn(*size, generator=g, device="cuda")

    s = dict(case=case)
    n, c = case["n"], case["c"]
    if op in ("wgrad", "norm8_grad"):
        # a checkpoint as the forward pass leaves it: behind a ReLU for a convolution, normalised values for a norm
        v = normal(*shape)
        if op == "wgrad":
            v = torch.relu(v * (1.0 + 0.2 * normal(1, c, 1, 1)))
        q, e = _quantise(v, case["fmt"])
        s["q"] = q.to(torch.int8 if case["fmt"] == "int8" else torch.float8_e4m3fn)
        s["e"] = (e + 127).to(torch.uint8).reshape(shape[:1] + shape[2:])
        if op == "wgrad":
            s["dy"] = (1e-3 * normal(n, case["k"], *_out_size(case))).to(torch.bfloat16)
            return s
    t = TYPES[case["type"]]
    if op == "norm8_grad":
        s["dy"] = (1e-3 * normal(*shape)).to(t)
        s["rstd"] = 0.5 + torch.rand(n, case["h"] * case["w"], generator=g, device="cuda")
        s["gamma"], s["beta"] = 1.0 + 0.2 * normal(1, c, 1, 1), 0.2 * normal(1, c, 1, 1)
        return s
    # some channels are much larger than the rest, as in trained networks
    s["x"] = (normal(*shape) * torch.exp(0.5 * normal(1, c, *([1] * (len(shape) - 2)))) + 0.1).to(t)
    if case.get("resid"):
        s["resid"] = normal(*shape).to(t)
    if op in ("rms", "rms8"):
        s["weight"] = 1.0 + 0.2 * normal(c)
        if case.get("grad"):
            s["dy"] = (1e-3 * normal(*shape)).to(t)
            s["dstream"] = (1e-3 * normal(*shape)).to(t)
    elif op == "norm8":
        s["gamma"], s["beta"] = 1.0 + 0.2 * normal(1, c, 1, 1), 0.2 * normal(1, c, 1, 1)
    return s


def run(state):
    return _own(state) if own else _plain(state)


# ---- the framework's calls ---------------------------------------------------------------------------------------------
def _own(s):
    from hific_amd import lib, ops
    case, op = s["case"], s["case"]["op"]
    if op == "rms":
        if not case["grad"]:
            with torch.no_grad():
                out = ops.rms_norm(s["x"], s["weight"], resid=s.get("resid"), eps=RMS_EPS)
            return dict(y=out[0], stream=out[1]) if case["resid"] else dict(y=out)
        x, wt = s["x"].detach().requires_grad_(), s["weight"].detach().requires_grad_()
        if case["resid"]:
            y, stream = ops.rms_norm(x, wt, resid=s["resid"], eps=RMS_EPS)
            dx, dw = torch.autograd.grad((y, stream), (x, wt), (s["dy"], s["dstream"]))
            return dict(y=y, stream=stream, dx=dx, dweight=dw)
        y = ops.rms_norm(x, wt, eps=RMS_EPS)
        dx, dw = torch.autograd.grad(y, (x, wt), s["dy"])
        return dict(y=y, dx=dx, dweight=dw)
    if op == "rms8":
        out = ops.rms_norm8(s["x"], s["weight"], resid=s.get("resid"), eps=RMS_EPS, fmt=case["fmt"])
        a = out[0] if case["resid"] else out
        r = dict(y=ops.restore8(a)) if case["fmt"] == "int8" else dict(y=a.q, scale=a.e.view(torch.float8_e8m0fnu))
        return dict(r, stream=out[1]) if case["resid"] else r
    if op == "checkpoint":
        return dict(x=ops.restore8(ops.checkpoint8(s["x"], fmt=case["fmt"]), dtype=s["x"].dtype))
    if op == "norm8":
        with torch.no_grad():
            y, a = ops.channel_norm8(s["x"], s["gamma"], s["beta"], eps=NORM_EPS, relu=case["relu"], resid=s.get("resid"),
                                     fmt=case["fmt"])
        return dict(y=y, kept=ops.restore8(a, dtype=y.dtype))
    a = ops.Act8(s["q"], s["e"])
    if op == "norm8_grad":
        dx, dgamma, dbeta = ops.channel_norm_grad8(a, s["dy"], s["gamma"], s["beta"], s["rstd"], relu=case["relu"])
        return dict(dx=dx, dgamma=dgamma, dbeta=dbeta)
    p = case["r"] // 2
    return dict(dw=ops.conv2d_weight_grad8(a, s["dy"], (case["r"], case["r"]), stride=case["stride"], pads=(p, p, p, p),
                                           pad_mode=lib.PAD_REFLECT if case["pad"] == "reflect" else lib.PAD_ZERO))


# ---- the plain form ----------------------------------------------------------------------------------------------------
def _channels(v, like):
    return v.reshape([1, -1] + [1] * (like.dim() - 2))


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op in ("rms", "rms8"):
        t = s["x"].dtype
        # the stream is what is stored: the norm and its backward pass see the same rounded sum
        stream = (s["x"].float() + s["resid"].float()).to(t) if case["resid"] else s["x"]
        h, wt = stream.float(), _channels(s["weight"], s["x"])
        r = torch.rsqrt((h * h).mean(1, keepdim=True) + RMS_EPS)
        out = dict(stream=stream) if case["resid"] else {}
        if op == "rms8":
            q, e = _quantise(h * r * wt, case["fmt"])
            if case["fmt"] == "int8":
                return dict(out, y=(q * _pow2(e, q)).to(torch.bfloat16))
            e = e.reshape(e.shape[:1] + e.shape[2:])
            return dict(out, y=q.to(torch.float8_e4m3fn), scale=(e + 127).to(torch.uint8).view(torch.float8_e8m0fnu))
        xh = h * r
        out["y"] = (xh * wt).to(t)
        if case["grad"]:
            dy = s["dy"].float()
            g = dy * wt
            dx = r * (g - xh * (g * xh).mean(1, keepdim=True))
            out["dx"] = ((dx + s["dstream"].float()) if case["resid"] else dx).to(t)
            out["dweight"] = (dy * xh).sum([0] + list(range(2, dy.dim())))
        return out
    if op == "checkpoint":
        q, e = _quantise(s["x"].float(), case["fmt"])
        return dict(x=(q * _pow2(e, q)).to(s["x"].dtype))
    if op == "norm8":
        x, gamma, beta, t = s["x"].float(), s["gamma"], s["beta"], s["x"].dtype
        d = x - x.mean(1, keepdim=True)
        r = torch.rsqrt((d * d).sum(1, keepdim=True) / (x.shape[1] - 1) + NORM_EPS)
        v, kept = _norm8_values(d * r, gamma, beta, case)
        if not case["resid"]:
            return dict(y=v.to(t), kept=kept.to(t))
        y = v.to(t).float() + s["resid"].float()
        q, e = _quantise(y, case["fmt"])
        return dict(y=y.to(t), kept=(q * _pow2(e, q)).to(t))
    e = (s["e"].to(torch.int32) - 127).unsqueeze(1)
    v = s["q"].float()
    v = v * _pow2(e, v)
    dy = s["dy"].float()
    if op == "norm8_grad":
        return _norm8_grad(v, dy, s["gamma"], s["beta"], s["rstd"], case, s["dy"].dtype)
    return dict(dw=_weight_grad(v, dy, case))


def _norm8_values(xh, gamma, beta, case):
    """Values of the norm, and what the 8 bits kept of them stand for.  Behind a ReLU a kept value is rounded to its other
    neighbour where the nearest one would be on the wrong side of zero: the backward pass then masks as the forward pass."""
    v = gamma * xh + beta
    e = _exponent(xh.abs().amax(1, keepdim=True), case["fmt"])
    t = xh * _pow2(-e, xh)
    q, scale = _round_to(t, case["fmt"]), _pow2(e, xh)
    if case["relu"]:
        # the side of zero in 64 bits, where gamma * x is exact
        g64, b64 = gamma.double(), beta.double()
        wrong = (g64 * (q * scale).double() + b64 > 0) != (g64 * xh.double() + b64 > 0)
        q = torch.where(wrong, _next_to(q, t > q, case["fmt"]), q)
    kept = gamma * (q * scale) + beta
    return (torch.relu(v), torch.relu(kept)) if case["relu"] else (v, kept)


def _norm8_grad(xh, dy, gamma, beta, rstd, case, t):
    if case["relu"]:
        dy = torch.where(gamma.double() * xh.double() + beta.double() > 0, dy, torch.zeros((), device=dy.device, dtype=dy.dtype))
    c = xh.shape[1]
    g = dy * gamma
    r = rstd.reshape(xh.shape[0], 1, *xh.shape[2:])
    dx = r * (g - g.mean(1, keepdim=True) - xh * ((g * xh).sum(1, keepdim=True) / (c - 1)))
    return dict(dx=dx.to(t), dgamma=(dy * xh).sum((0, 2, 3)).reshape(gamma.shape), dbeta=dy.sum((0, 2, 3)).reshape(beta.shape))


def _weight_grad(x, dy, case):
    r, st, p = case["r"], case["stride"], case["r"] // 2
    if p:
        x = F.pad(x, (p, p, p, p), mode="reflect" if case["pad"] == "reflect" else "constant")
    cols = x.unfold(2, r, st).unfold(3, r, st).permute(0, 2, 3, 1, 4, 5).reshape(-1, x.shape[1] * r * r)
    return (dy.permute(1, 0, 2, 3).reshape(dy.shape[1], -1) @ cols).reshape(dy.shape[1], x.shape[1], r, r)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "checkpoint":
        v = s["x"].double()
        return dict(x=_exact8(v, case["fmt"])[0])
    if op in ("rms", "rms8"):
        h = s["x"].double()
        out = {}
        if case["resid"]:
            h = out["stream"] = (h + s["resid"].double()).to(s["x"].dtype).double()
        w = s["weight"].double().view(-1, *[1] * (h.dim() - 2))
        inv = 1.0 / (h.square().sum(1, keepdim=True) / case["c"] + RMS_EPS).sqrt()
        y = h * inv * w
        if op == "rms8":
            val, q, e = _exact8(y, case["fmt"])
            if case["fmt"] == "int8":
                return dict(out, y=val)
            return dict(out, y=q, scale=torch.exp2(e.squeeze(1).double()))
        out["y"] = y
        if case["grad"]:
            dy = s["dy"].double()
            # d/dh of sum(dy * w * h * inv): inv depends on every h of the token
            dot = (dy * w * h).sum(1, keepdim=True)
            out["dx"] = dy * w * inv - h * inv ** 3 * dot / case["c"]
            if case["resid"]:
                out["dx"] = out["dx"] + s["dstream"].double()
            out["dweight"] = (dy * h * inv).transpose(0, 1).reshape(case["c"], -1).sum(1)
        return out
    if op == "norm8":
        x, gamma, beta = s["x"].double(), s["gamma"].double(), s["beta"].double()
        var, mean = torch.var_mean(x, dim=1, keepdim=True, correction=1)
        xh = (x - mean) / (var + NORM_EPS).sqrt()
        v = xh * gamma + beta
        y = v.clamp_min(0) if case["relu"] else v
        if case["resid"]:
            y = y.to(s["x"].dtype).double() + s["resid"].double()
            return dict(y=y, kept=_exact8(y, case["fmt"])[0])
        near = _exact8(xh, case["fmt"])[0]
        if case["relu"]:
            other = _exact8(xh, case["fmt"], far=True)[0]
            side = (near * gamma + beta > 0) == (v > 0)
            near = torch.where(side, near, other)
        kept = near * gamma + beta
        return dict(y=y, kept=kept.clamp_min(0) if case["relu"] else kept)
    scale = torch.exp2(s["e"].double() - 127).unsqueeze(1)
    v = s["q"].double() * scale
    dy = s["dy"].double()
    if op == "norm8_grad":
        gamma, beta = s["gamma"].double(), s["beta"].double()
        if case["relu"]:
            dy = dy * (v * gamma + beta > 0)
        r = s["rstd"].double().view(v.shape[0], 1, *v.shape[2:])
        c = case["c"]
        g = dy * gamma
        dx = (g - g.sum(1, keepdim=True) / c - v * (g * v).sum(1, keepdim=True) / (c - 1)) * r
        per = lambda a: a.transpose(0, 1).reshape(c, -1).sum(1).view(1, c, 1, 1)  # noqa: E731
        return dict(dx=dx, dgamma=per(dy * v), dbeta=per(dy))
    # the weight gradient, one tap at a time
    r, st, p = case["r"], case["stride"], case["r"] // 2
    oh, ow = _out_size(case)
    iy = torch.arange(oh, device=v.device) * st - p
    ix = torch.arange(ow, device=v.device) * st - p
    dyk = dy.transpose(0, 1).reshape(case["k"], -1)
    taps = []
    for a in range(r):
        for b in range(r):
            y, x = iy + a, ix + b
            if case["pad"] == "reflect":
                y, x = _mirror(y, case["h"]), _mirror(x, case["w"])
            inside = ((y >= 0) & (y < case["h"])).double()[:, None] * ((x >= 0) & (x < case["w"])).double()[None, :]
            part = v[:, :, y.clamp(0, case["h"] - 1)][:, :, :, x.clamp(0, case["w"] - 1)] * inside
            taps.append(dyk @ part.transpose(0, 1).reshape(case["c"], -1).t())
    return dict(dw=torch.stack(taps, -1).view(case["k"], case["c"], r, r))


def _mirror(i, n):
    i = i.abs()
    return torch.minimum(i, 2 * (n - 1) - i)


def _exact8(v, fmt, far=False):
    """(value, q, e) of the format's value next to v in the scale of v's tokens: the nearest (ties to even), or the one on
    the other side of v."""
    amax = v.abs().amax(1, keepdim=True)
    e = torch.ceil(torch.log2(amax / _qmax(fmt)))
    e = torch.where(amax <= _qmax(fmt) * torch.exp2(e - 1), e - 1, e)
    e = torch.where(amax > _qmax(fmt) * torch.exp2(e), e + 1, e)
    e = torch.where(amax > 0, e, torch.full_like(e, -126)).clamp_min(-126)
    t = v / torch.exp2(e)
    if fmt == "int8":
        step = torch.ones_like(t)
    else:
        # three bits behind the leading one, down to 2^-9
        step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3)
    near = torch.round(t / step) * step
    if far:
        lo, hi = torch.floor(t / step) * step, torch.ceil(t / step) * step
        near = torch.where(near == lo, hi, lo)
    return near * torch.exp2(e), near, e
