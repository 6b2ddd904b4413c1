"""Activations in 8 bits and the norms around them in float64, from their definitions: the oracle of tests/test_act8.py and
tests/test_gpu_act8.py.  Tensors are [N, C, ...]; a token is one position, its C values share one power-of-two exponent."""
import torch

QMAX = {"int8": 127.0, "e4m3": 448.0}


def e4m3_values():
    """The 127 magnitudes of the finite-only e4m3 format, by code 0 .. 126: sign, 4 exponent bits (bias 7), 3 mantissa bits."""
    out = []
    for code in range(127):
        e, m = code >> 3, code & 7
        out.append(m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return torch.tensor(out, dtype=torch.float64)


def grid(fmt):
    """Every value of the format, ascending (one zero)."""
    if fmt == "int8":
        return torch.arange(-127, 128, dtype=torch.float64)
    v = e4m3_values()
    return torch.cat((-v.flip(0)[:-1], v))


def exponent(amax, fmt):
    """Smallest e >= -126 with amax <= QMAX * 2^e, by trying; -126 for 0."""
    e = torch.floor(torch.log2(torch.where(amax > 0, amax, torch.ones_like(amax)) / QMAX[fmt])) - 2
    for _ in range(4):
        e = torch.where(amax > QMAX[fmt] * torch.exp2(e), e + 1, e)
    e = torch.where(amax > 0, e, torch.full_like(e, -126.0))
    return e.clamp_min(-126.0)


def nearest(t, fmt):
    """(index into grid(fmt) of the value nearest to t, ties to the one whose code is even)."""
    g = grid(fmt)
    hi = torch.searchsorted(g, t.contiguous()).clamp(1, len(g) - 1)
    lo = hi - 1
    dl, dh = t - g[lo], g[hi] - t
    # codes count outwards from zero: the parity of the distance from the middle is the parity of the code
    lo_even = ((lo - len(g) // 2) % 2) == 0
    pick_lo = (dl < dh) | ((dl == dh) & lo_even)
    return torch.where(pick_lo, lo, hi)


def quantise(v, fmt, gamma=None, beta=None):
    """(values q * 2^e, exponents [N, ...]) of float64 v.  With gamma / beta ([C]): rounded to the side of the ReLU that v is on.
    A token with an infinity or NaN gives NaN and exponent 128.  Where the nearest value would leave float32 (2^128) it is the next one
    towards zero: a finite token stays finite."""
    v = v.double()
    bad = ~torch.isfinite(v).all(1, keepdim=True)
    vv = torch.where(bad, torch.zeros_like(v), v)
    e = exponent(vv.abs().amax(1, keepdim=True), fmt)
    t = vv / torch.exp2(e)
    idx, g = nearest(t, fmt), grid(fmt)
    if gamma is not None:
        sh = [1, -1] + [1] * (v.dim() - 2)
        ga, be = gamma.double().reshape(sh), beta.double().reshape(sh)
        wrong = (ga * (g[idx] * torch.exp2(e)) + be > 0) != (ga * vv + be > 0)
        other = torch.where(t > g[idx], idx + 1, idx - 1).clamp(0, len(g) - 1)
        idx = torch.where(wrong, other, idx)
    over = g[idx].abs() * torch.exp2(e) >= 2.0 ** 128
    idx = torch.where(over, torch.where(g[idx] > 0, idx - 1, idx + 1), idx)
    out = torch.where(bad, torch.full_like(v, float("nan")), g[idx] * torch.exp2(e))
    return out, torch.where(bad, torch.full_like(e, 128.0), e).squeeze(1)


def values(q, e):
    """What int8 / float8_e4m3fn q and uint8 e stand for."""
    s = torch.where(e == 255, torch.full(e.shape, float("nan"), dtype=torch.float64), torch.exp2(e.double() - 127))
    return q.float().double() * s.unsqueeze(1)


def _ch(w, like):
    return w.double().reshape([1, -1] + [1] * (like.dim() - 2))


def rms_norm(x, weight, resid=None, eps=1e-6):
    """(y, h, rstd): h = x + resid rounded to x's type."""
    h = x if resid is None else (x.float() + resid.float()).to(x.dtype)
    hd = h.double()
    r = 1.0 / torch.sqrt((hd * hd).mean(1, keepdim=True) + eps)
    return hd * r * _ch(weight, x), h, r


def rms_norm_grad(xh, r, weight, dy, dstream=None):
    """(dx, dweight) from the normalised xh and r [N, 1, ...]."""
    xh, dy = xh.double(), dy.double()
    g = dy * _ch(weight, xh)
    dx = r * (g - xh * (g * xh).mean(1, keepdim=True))
    if dstream is not None:
        dx = dx + dstream.double()
    return dx, (dy * xh).sum([0] + list(range(2, xh.dim())))


def channel_norm(x, gamma, beta, eps=1e-3):
    """(v = gamma xh + beta, xh, rstd) with the unbiased variance."""
    xd = x.double()
    d = xd - xd.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((d * d).sum(1, keepdim=True) / (x.shape[1] - 1) + eps)
    return _ch(gamma, x) * d * r + _ch(beta, x), d * r, r


def channel_norm_grad(xh, r, gamma, beta, dy, relu):
    """(dx, dgamma, dbeta) from the normalised xh and r [N, 1, ...]."""
    xh, dy = xh.double(), dy.double()
    if relu:
        dy = torch.where(_ch(gamma, xh) * xh + _ch(beta, xh) > 0, dy, torch.zeros_like(dy))
    g = dy * _ch(gamma, xh)
    dx = r * (g - g.mean(1, keepdim=True) - xh * ((g * xh).sum(1, keepdim=True) / (xh.shape[1] - 1)))
    dims = [0] + list(range(2, xh.dim()))
    return dx, (dy * xh).sum(dims), dy.sum(dims)


def conv2d_weight_grad(x, dy, kernel, stride, pads, reflect):
    """[K, C, R, S] = sum dy * pad(x), one tap at a time."""
    x, dy = x.double(), dy.double()
    pt, pl, pb, pr = pads
    xp = torch.nn.functional.pad(x, (pl, pr, pt, pb), mode="reflect" if reflect else "constant")
    K, OH, OW = dy.shape[1], dy.shape[2], dy.shape[3]
    dw = torch.zeros(K, x.shape[1], *kernel, dtype=torch.float64)
    for r in range(kernel[0]):
        for s in range(kernel[1]):
            t = xp[:, :, r:r + (OH - 1) * stride + 1:stride, s:s + (OW - 1) * stride + 1:stride]
            dw[:, :, r, s] = torch.einsum("nkp,ncp->kc", dy.flatten(2), t.flatten(2))
    return dw
