"""8-bit activations and the norms around them on the GPU against the float64 oracle (oracle/act8_oracle.py).

Tolerances.  A result rounded to type t once is off by half a step, finfo(t).eps / 2 relative to the value; float32 arithmetic in
front of it adds a few 2^-24 relative to the largest term.  F32 below is 2^-24 times 32: sums over the channels are trees or short
chains per thread (at most 16 terms in a row for the sizes here, then pairwise), and a handful of products follow.  8-bit values are
off by half a step of their format, or by a whole one where the ReLU decides the side."""
import math

import pytest
import torch

from oracle import act8_oracle as O

pytestmark = pytest.mark.gpu
F32 = 32 * 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# [N, C, ...]: one token, one channel, rows (even, odd, wide), planes (multiples of eight, odd, tiny, one row of blocks and more)
SHAPES = [(1, 1), (1, 960), (3, 7), (5, 64), (33, 220), (70, 961), (4, 4100), (2, 5, 1, 1), (1, 3, 2, 2), (2, 16, 3, 5), (3, 60, 8, 8),
          (2, 220, 13, 11), (1, 2, 1, 8), (2, 33, 24, 40), (1, 960, 16, 16), (2, 240, 9, 64), (5, 8, 64), (1, 2100, 4, 8), (2, 1030, 3, 3)]
NORM_SHAPES = [s for s in SHAPES if s[1] > 1]


def _half(t):
    return torch.finfo(t).eps / 2


def _rand(shape, seed, dtype=torch.float32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype)


def _chan(shape, seed, around=1.0, spread=0.3):
    return around + spread * _rand((shape[1],), seed)


def _close(got, want, rel, absolute, what):
    """|got - want| <= rel * |want| + absolute (tensor or number), everywhere."""
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    off = (got - want).abs() - (rel * want.abs() + absolute)
    assert (off <= 0).all(), f"{what}: {float(off.max()):.3g} over the bound"


def _step8(v, e, fmt):
    """Half a step of the format at the values v with exponents e."""
    s = torch.exp2(e).unsqueeze(1)
    if fmt == "int8":
        return 0.5 * s
    mag = torch.exp2(torch.floor(torch.log2((v.abs() / s).clamp_min(2.0 ** -6))))
    return mag * 2.0 ** -4 * s


def _vals(a):
    """float64 values of an Act8's own bits (without its gamma / beta)."""
    return O.values(a.q.cpu(), a.e.cpu())


def _finish(*tensors):
    torch.cuda.synchronize()
    return tensors


# ---- pack and restore: bit for bit -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_checkpoint_is_the_oracles_bit_for_bit(hific, dev, shape, dt, fmt):
    from hific_amd import ops
    x = _rand(shape, 1, scale=3.0)
    x *= torch.exp2(_rand(shape[:1] + (1,) + shape[2:], 2, scale=20.0).round())      # exponents far apart
    x = x.to(TYPES[dt])
    a = ops.checkpoint8(x.to(dev), fmt=fmt)
    back32, back16 = ops.restore8(a, torch.float32), ops.restore8(a)
    _finish()
    want, e = O.quantise(x.double(), fmt)
    assert torch.equal(a.e.cpu().double() - 127, e)
    assert torch.equal(_vals(a), want)
    assert torch.equal(back32.cpu().double(), want)
    assert back16.dtype == torch.bfloat16 and torch.equal(back16.cpu().double(), want)   # at most 8 significant bits: exact
    assert ((want - x.double()).abs() <= _step8(x.double(), e, fmt)).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_every_code_packs_and_restores_to_itself(hific, dev, fmt):
    from hific_amd import ops
    v = O.grid(fmt)
    for e in (-100, 0, 77):
        x = (v * 2.0 ** e).float().reshape(1, -1)
        a = ops.checkpoint8(x.to(dev), fmt=fmt)
        assert torch.equal(ops.restore8(a, torch.float32).cpu(), x)
        assert int(a.e.cpu()[0]) == 127 + e


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_ties_and_borders_round_as_the_oracle(hific, dev, fmt):
    from hific_amd import ops
    g = O.grid(fmt)
    mid = (g[1:] + g[:-1]) / 2
    row = torch.cat((g[-1:], mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20))).float().reshape(1, -1)
    a = ops.checkpoint8(row.to(dev), fmt=fmt)
    assert torch.equal(_vals(a), O.quantise(row.double(), fmt)[0])
    # the exponent's own border: QMAX, one step above it, one below
    for q in (O.QMAX[fmt],):
        t = torch.tensor([[q, 1.0], [math.nextafter(q, 2 * q), 1.0], [q * (1 + 2.0 ** -23), 1.0], [q * (1 - 2.0 ** -24), 1.0]]).float()
        b = ops.checkpoint8(t.to(dev), fmt=fmt)
        want, e = O.quantise(t.double(), fmt)
        assert torch.equal(b.e.cpu().double() - 127, e) and torch.equal(_vals(b), want)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(6, 40), (6, 41), (2, 40, 8, 8), (2, 21, 3, 5)])
def test_zeros_tiny_and_not_finite_tokens(hific, dev, shape, dt, fmt):
    from hific_amd import ops
    x = _rand(shape, 4).to(TYPES[dt])
    flat = x.movedim(1, -1).reshape(-1, shape[1])
    flat[0] = 0.0
    flat[1, 3] = float("inf")
    flat[2, 5] = float("-inf")
    flat[3, 0] = float("nan")
    flat[4] = 1e-39                                      # below the smallest normal number
    flat[5] = flat[5] * 1e30
    x = flat.reshape(shape[:1] + shape[2:] + shape[1:2]).movedim(-1, 1).contiguous()
    a = ops.checkpoint8(x.to(dev), fmt=fmt)
    back = ops.restore8(a, torch.float32).cpu().double()
    want, e = O.quantise(x.double(), fmt)
    assert torch.equal(torch.isnan(back), torch.isnan(want))
    keep = ~torch.isnan(want)
    assert torch.equal(back[keep], want[keep])
    assert torch.equal(a.e.cpu().double() - 127, e)


def test_restore_with_norm_parameters(hific, dev):
    from hific_amd import ops
    shape = (2, 37, 6, 7)
    a = ops.checkpoint8(_rand(shape, 6).to(dev))
    gamma, beta = _chan(shape, 7).reshape(1, -1, 1, 1), _chan(shape, 8, 0.0)
    v = O._ch(gamma, torch.empty(shape)) * _vals(a) + O._ch(beta, torch.empty(shape))
    for relu in (False, True):
        b = ops.Act8(a.q, a.e, gamma.to(dev), beta.to(dev), relu)
        want = torch.relu(v) if relu else v
        _close(ops.restore8(b, torch.float32), want, 2.0 ** -24, 0.0, "f32")        # one fused multiply-add: one rounding
        _close(ops.restore8(b), want, _half(torch.bfloat16) + 2.0 ** -23, 0.0, "bf16")
    nan = ops.Act8(a.q, torch.full_like(a.e, 255), gamma.to(dev), beta.to(dev), True)
    assert torch.isnan(ops.restore8(nan)).all()


# ---- root-mean-square norm ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("resid", [False, True])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rms_norm_forward(hific, dev, shape, dt, resid):
    from hific_amd import ops
    t = TYPES[dt]
    x, w = _rand(shape, 11, t, 2.0, 0.5), _chan(shape, 12)
    rs = _rand(shape, 13, t) if resid else None
    y, h, _ = O.rms_norm(x, w, rs)
    got = ops.rms_norm(x.to(dev), w.to(dev), resid=None if rs is None else rs.to(dev))
    if resid:
        got, gh = got
        assert torch.equal(gh.cpu(), h)
    assert got.dtype == t
    _close(got, y, _half(t) + F32, 0.0, "y")


@pytest.mark.parametrize("kept", [None, "int8", "e4m3"])
@pytest.mark.parametrize("resid", [False, True])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rms_norm_backward(hific, dev, shape, dt, resid, kept):
    """Against the formula on what the forward pass kept: h, or the 8-bit values (read back from the node)."""
    from hific_amd import ops
    t = TYPES[dt]
    x, w = _rand(shape, 21, t, 2.0, 0.5), _chan(shape, 22)
    rs, dy, ds = _rand(shape, 23, t), _rand(shape, 24, t), _rand(shape, 25, t)
    xd, wd, rd = x.to(dev).requires_grad_(), w.to(dev).requires_grad_(), rs.to(dev).requires_grad_()
    if resid:
        y, h = ops.rms_norm(xd, wd, resid=rd, fmt=kept)
        saved = y.grad_fn.saved_tensors
        dx, dw, dr = torch.autograd.grad((y, h), (xd, wd, rd), (dy.to(dev), ds.to(dev)))
        assert torch.equal(dx, dr)
    else:
        y = ops.rms_norm(xd, wd, fmt=kept)
        saved = y.grad_fn.saved_tensors
        dx, dw = torch.autograd.grad(y, (xd, wd), dy.to(dev))
    yw, hw, r = O.rms_norm(x, w, rs if resid else None)
    _close(y, yw, _half(t) + F32, 0.0, "y")
    xh = hw.double() * r
    if kept:
        assert saved[0].dtype in (torch.int8, torch.float8_e4m3fn) and saved[0].numel() == x.numel()
        v = O.values(saved[0].cpu(), saved[1].cpu())
        e = saved[1].cpu().double() - 127
        _close(v, xh, F32, _step8(xh, e, kept) * (1 + 1e-6), "kept")
        xh = v
    wdx, wdw = O.rms_norm_grad(xh, r, w, dy, ds if resid else None)
    size = r * (dy.double() * O._ch(w, x)).abs().amax(1, keepdim=True) * (1 + xh.abs().amax(1, keepdim=True))
    _close(dx, wdx, _half(t), F32 * size + F32 * ds.double().abs().amax(), "dx")
    terms = (dy.double() * xh).abs().sum([0] + list(range(2, x.dim())))
    _close(dw, wdw, 0.0, 8 * F32 * terms + 1e-30, "dweight")


def test_rms_norm_gradient_against_differences(hific, dev):
    """(f(x + s v) - f(x - s v)) / 2 s of the kernel's own forward pass in float32.  s = 2^-6: the third-order term is
    s^2 / 6 * f''' ~ 4e-5 * f'''; the rounding of f is 2^-24 * sum|y dy| / s."""
    from hific_amd import ops
    shape, s = (2, 24, 5, 8), 2.0 ** -6
    x, w, dy, v = _rand(shape, 31).to(dev), _chan(shape, 32).to(dev), _rand(shape, 33).to(dev), _rand(shape, 34).to(dev)
    xd = x.clone().requires_grad_()
    dx, = torch.autograd.grad(ops.rms_norm(xd, w), xd, dy)
    f = lambda z: (ops.rms_norm(z, w).double() * dy.double()).sum()  # noqa: E731
    diff = float((f(x + s * v) - f(x - s * v)) / (2 * s))
    want = float((dx.double() * v.double()).sum())
    assert abs(diff - want) < 2e-3 * float((dx.double() * v.double()).abs().sum())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("resid", [False, True])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rms_norm8(hific, dev, shape, dt, resid, fmt):
    from hific_amd import ops
    t = TYPES[dt]
    x, w = _rand(shape, 41, t, 2.0, 0.5), _chan(shape, 42)
    rs = _rand(shape, 43, t) if resid else None
    y, h, _ = O.rms_norm(x, w, rs)
    got = ops.rms_norm8(x.to(dev), w.to(dev), resid=None if rs is None else rs.to(dev), fmt=fmt)
    if resid:
        got, gh = got
        assert torch.equal(gh.cpu(), h)
    assert got.fmt == fmt and got.shape == x.shape
    e = got.e.cpu().double() - 127
    amax = y.abs().amax(1)
    assert (amax <= O.QMAX[fmt] * torch.exp2(e) * (1 + F32)).all() and (amax > O.QMAX[fmt] * torch.exp2(e - 1) * (1 - F32)).all()
    _close(_vals(got), y, F32, _step8(y, e, fmt) * (1 + 1e-6), "values")


# ---- channel norm with a checkpoint -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("relu,resid", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_channel_norm8(hific, dev, shape, dt, relu, resid, fmt):
    from hific_amd import ops
    t = TYPES[dt]
    x, gamma, beta = _rand(shape, 51, t, 1.5, 0.3), _chan(shape, 52), _chan(shape, 53, 0.0)
    rs, dy = _rand(shape, 54, t), _rand(shape, 55, t)
    leaves = [v.to(dev).requires_grad_() for v in (x, gamma, beta, rs)]
    y, a = ops.channel_norm8(leaves[0], leaves[1], leaves[2], relu=relu, resid=leaves[3] if resid else None, fmt=fmt)
    q, e, rstd, _, _ = y.grad_fn.saved_tensors
    grads = torch.autograd.grad(y, leaves if resid else leaves[:3], dy.to(dev))
    v, xh, r = O.channel_norm(x, gamma, beta)
    big = 1 + xh.abs().amax(1, keepdim=True) + (x.double().abs().amax(1, keepdim=True) * r)     # what the mean cancels
    vabs = F32 * big * (1 + O._ch(gamma, x).abs())
    act = torch.relu(v) if relu else v
    if resid:       # the norm's value is rounded to the type, then the sum: two half steps
        _close(y, act + rs.double(), _half(t), _half(t) * act.abs() * (1 + _half(t)) + 2 * vabs, "y")
    else:
        _close(y, act, _half(t), 2 * vabs, "y")
    _close(rstd.reshape(r.shape), r, 4 * F32 * (1 + float(x.double().abs().amax()) ** 2), 0.0, "rstd")
    # what is kept of xh: half a step; a whole one where the ReLU decides, and then on the right side of it
    kept, ee = O.values(q.cpu(), e.cpu()), e.cpu().double() - 127
    half = _step8(xh, ee, fmt)
    off = (kept - xh).abs()
    assert (off <= (2 if relu else 1) * half * (1 + 1e-6) + F32 * big).all()
    if relu:
        side = O._ch(gamma, x) * kept + O._ch(beta, x) > 0
        clear = v.abs() > 2 * vabs                       # the float32 value is surely on the oracle's side
        assert torch.equal(side[clear], (v > 0)[clear])
        # more than half a step off only where the nearest value is on the wrong side.  (A count of such values proves nothing on a
        # small tensor: one value of twelve is 8 %.)
        moved = (off > half * (1 + 1e-6) + F32 * big) & clear
        near = O.quantise(xh, fmt)[0]
        wrong = (O._ch(gamma, x) * near + O._ch(beta, x) > 0) != (v > 0)
        assert wrong[moved].all()
    # the checkpoint stands for y
    back = ops.restore8(a, torch.float32).cpu().double()
    if resid:
        yd = y.detach().cpu().double()
        assert (a.gamma is None) and ((back - yd).abs() <= _step8(yd, a.e.cpu().double() - 127, fmt)
                                      * (1 + 1e-6) + _half(t) * yd.abs()).all()
    else:
        w = O._ch(gamma, x) * kept + O._ch(beta, x)
        _close(back, torch.relu(w) if relu else w, 2.0 ** -23, 1e-30, "restored")
    # the backward pass is the formula on what was kept
    rk = rstd.cpu().double().reshape(r.shape)
    wdx, wdg, wdb = O.channel_norm_grad(kept, rk, gamma, beta, dy, relu)
    size = rk * (dy.double() * O._ch(gamma, x)).abs().amax(1, keepdim=True) * (1 + kept.abs().amax(1, keepdim=True)) * 2
    _close(grads[0], wdx, _half(t), F32 * size, "dx")
    dims = [0] + list(range(2, x.dim()))
    _close(grads[1], wdg, 0.0, 8 * F32 * (dy.double() * kept).abs().sum(dims) + 1e-30, "dgamma")
    _close(grads[2], wdb, 0.0, 8 * F32 * dy.double().abs().sum(dims) + 1e-30, "dbeta")
    if resid:
        assert torch.equal(grads[3].cpu(), dy)
    # the function form gives the same
    dx, dg, db = ops.channel_norm_grad8(ops.Act8(q, e), dy.to(dev), leaves[1].detach(), leaves[2].detach(), rstd, relu=relu)
    assert torch.equal(dx, grads[0]) and torch.equal(dg, grads[1]) and torch.equal(db, grads[2])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("shape", [(2, 64, 8, 8), (3, 60, 24, 40), (2, 33, 5, 7), (3, 47, 2, 3), (40, 96)])
def test_masks_agree_forward_and_backward_for_any_gamma(hific, dev, shape, fmt):
    """gamma of both signs, zero and tiny: a position passes gradient exactly where its forward value is positive.  dbeta of a dy that is
    one at a single channel counts them."""
    from hific_amd import ops
    x = _rand(shape, 58, scale=1.5)
    gamma, beta = _rand((shape[1],), 59), 0.5 * _rand((shape[1],), 60)
    gamma[3], gamma[5], beta[5], gamma[7] = 0.0, 0.0, -0.25, 1e-30
    xd, gd, bd = x.to(dev).requires_grad_(), gamma.to(dev).requires_grad_(), beta.to(dev).requires_grad_()
    y, a = ops.channel_norm8(xd, gd, bd, relu=True, fmt=fmt)
    db, = torch.autograd.grad(y, bd, torch.ones_like(y), retain_graph=True)
    open_ = (y.detach() > 0).double().sum([0] + list(range(2, len(shape))))
    assert torch.equal(db.double(), open_)
    assert 0.2 < float(open_.sum() / x.numel()) < 0.8
    assert torch.equal(ops.restore8(a, torch.float32) > 0, y > 0)


def test_channel_norm8_agrees_with_channel_norm(hific, dev):
    """y as channel_norm gives it (the same formula; another order of the sums), gradients within what 8 bits cost: xh is off by
    u = half a step <= 2^-7 * max|xh|, rms u / sqrt(3) - times the two places where xh enters dx."""
    from hific_amd import ops
    shape = (4, 64, 16, 16)
    x, gamma, beta, dy = _rand(shape, 61).to(dev), _chan(shape, 62).to(dev).reshape(1, -1, 1, 1), _chan(shape, 63, 0.0).to(dev).reshape(1, -1, 1, 1), _rand(shape, 64).to(dev)
    res = []
    for f in (lambda *a: ops.channel_norm(*a, relu=True), lambda *a: ops.channel_norm8(*a, relu=True)[0]):
        leaves = [v.clone().requires_grad_() for v in (x, gamma, beta)]
        y = f(*leaves)
        res.append((y.detach(),) + torch.autograd.grad(y, leaves, dy))
    y0, y1 = res[0][0].double(), res[1][0].double()
    assert ((y0 - y1).abs() <= 1e-5 * (1 + y0.abs())).all()
    for a, b in zip(res[0][1:], res[1][1:]):
        assert float((a - b).norm() / a.norm()) < 0.02


# ---- weight gradients ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n,c,h,w,k,r,s,stride,pads,reflect", [
    (2, 64, 16, 16, 64, 3, 3, 1, (1, 1, 1, 1), True), (1, 33, 9, 7, 17, 3, 3, 1, (1, 1, 1, 1), False), (3, 20, 13, 16, 40, 3, 3, 2, (1, 0, 0, 1), True),
    (2, 16, 8, 8, 24, 1, 1, 1, (0, 0, 0, 0), False), (1, 24, 17, 19, 12, 5, 5, 2, (2, 2, 2, 2), True), (1, 130, 16, 32, 70, 3, 3, 1, (1, 1, 1, 1), True),
    (2, 64, 32, 32, 96, 3, 3, 2, (1, 1, 1, 1), False), (1, 3, 40, 48, 60, 7, 7, 1, (3, 3, 3, 3), True),
    (1, 1, 1, 1, 1, 1, 1, 1, (0, 0, 0, 0), False), (5, 7, 3, 4, 130, 3, 2, 1, (1, 1, 1, 0), True), (3, 70, 5, 9, 3, 2, 3, 2, (0, 1, 1, 1), False),
    (2, 200, 14, 10, 300, 3, 3, 1, (0, 0, 0, 0), False)])
def test_conv_weight_gradient_from_8_bits(hific, dev, n, c, h, w, k, r, s, stride, pads, reflect, dt, fmt):
    """Products of restored values and dy are exact in bfloat16 (8 + 8 bits), so only the float32 sum rounds: 2^-24 per addition.  At most
    1920 positions here, 16 of them per matrix instruction, so at most 120 additions in a row, each of a sum of 16."""
    from hific_amd import ops, lib
    a = ops.checkpoint8(_rand((n, c, h, w), 71).to(dev), fmt=fmt)
    oh, ow = (h + pads[0] + pads[2] - r) // stride + 1, (w + pads[1] + pads[3] - s) // stride + 1
    dy = _rand((n, k, oh, ow), 72, TYPES[dt])
    x = _vals(a)
    got = ops.conv2d_weight_grad8(a, dy.to(dev), (r, s), stride, pads, lib.PAD_REFLECT if reflect else lib.PAD_ZERO)
    want = O.conv2d_weight_grad(x, dy, (r, s), stride, pads, reflect)
    size = O.conv2d_weight_grad(x.abs(), dy.double().abs(), (r, s), stride, pads, reflect)
    _close(got, want, 0.0, 136 * 2.0 ** -24 * size + 1e-30, "dw")
    # and it is what the convolution's own backward pass gives for the restored tensor
    ops_x = ops.restore8(a, TYPES[dt])
    again = torch.empty_like(got)
    wsp, wsb = ops._ws(ops_x)
    lib.call("hific_conv2d_bwd_weight", lib.ptr(ops_x), lib.ptr(dy.to(dev).contiguous()), lib.ptr(again), n, c, h, w, k, r, s, stride, *pads,
             int(reflect), 0, lib.dtype_code(ops_x), 0, wsp, wsb, lib.stream())
    torch.cuda.synchronize()
    assert float((again - got).abs().max()) <= float(136 * 2.0 ** -23 * size.max())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_conv_transpose_weight_gradient_from_8_bits(hific, dev, fmt):
    from hific_amd import ops
    a = ops.checkpoint8(_rand((2, 24, 9, 8), 81).to(dev), fmt=fmt)
    dy = _rand((2, 40, 18, 16), 82, torch.bfloat16)
    got = ops.conv_transpose2d_weight_grad8(a, dy.to(dev), (3, 3), 2, 1, 1)
    x = _vals(a)

    def ref(xv, dv):          # dw[ci, co, r, s] = sum x[ci, i] dy[co, 2 i - 1 + r]
        xp = torch.nn.functional.pad(dv, (1, 2, 1, 2))
        out = torch.zeros(24, 40, 3, 3, dtype=torch.float64)
        for r in range(3):
            for s in range(3):
                t = xp[:, :, r:r + 17:2, s:s + 15:2]
                out[:, :, r, s] = torch.einsum("ncp,nkp->ck", xv.flatten(2), t.flatten(2))
        return out
    _close(got, ref(x, dy.double()), 0.0, 64 * 2.0 ** -24 * ref(x.abs(), dy.double().abs()) + 1e-30, "dw")


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("n,c,h,w,k,r,stride", [(2, 40, 16, 32, 72, 3, 1), (2, 40, 16, 32, 72, 3, 2), (1, 30, 7, 24, 20, 3, 2), (3, 21, 9, 7, 33, 3, 2), (1, 140, 24, 24, 20, 3, 1)])
def test_both_forms_of_the_weight_gradient(hific, dev, monkeypatch, transposed, n, c, h, w, k, r, stride):
    """The kernel that reads the 8-bit tensor and the restored form, on shapes that either may take: the same sums in another order, with a
    norm's gamma / beta / ReLU on the way, and accumulating."""
    from hific_amd import act8, lib, ops
    a = ops.checkpoint8(_rand((n, c, h, w), 73).to(dev))
    a = ops.Act8(a.q, a.e, _chan((1, c), 74).to(dev), _chan((1, c), 75, 0.0).to(dev), True)
    geom = (stride, 1, stride - 1) if transposed else (stride, 1, 1, 1, 1, lib.PAD_REFLECT)
    if transposed:
        oh, ow = (h - 1) * stride + 1 + stride - 1, (w - 1) * stride + 1 + stride - 1
    else:
        oh, ow = (h - 1) // stride + 1, (w - 1) // stride + 1
    dy = _rand((n, k, oh, ow), 76, torch.bfloat16).to(dev)
    start = _rand((c, k, r, r) if transposed else (k, c, r, r), 77)
    sums = []
    for own in (True, False):
        monkeypatch.setattr(act8, "_wgrad8_ws_bytes", lambda *s: int(lib.raw("hific_wgrad8_ws_bytes")(*s)) if own else 0)
        for acc in (0, 1):
            dw = start.to(dev).clone()
            act8._conv_wgrad8(a.tensors(), True, dy, dw, acc, geom, lib.HIFIC_BF16)
            sums.append(dw.cpu().double() - (start.double() if acc else 0))
    size = float((a.q.float().abs().amax() * 2.0 ** (int(a.e.max()) - 127) * 2) * dy.float().abs().amax()) * n * h * w
    for s in sums[1:]:
        assert float((s - sums[0]).abs().max()) <= 2.0 ** -22 * (size + 8)
    assert float(sums[0].abs().max()) > 0


def test_weight_gradient_in_slices_is_the_whole_one(hific, dev, monkeypatch):
    from hific_amd import act8, ops
    a = ops.checkpoint8(_rand((5, 12, 9, 7), 91).to(dev))
    dy = _rand((5, 20, 9, 7), 92, torch.bfloat16).to(dev)
    whole = ops.conv2d_weight_grad8(a, dy, (3, 3), 1, (1, 1, 1, 1))
    monkeypatch.setattr(act8, "_MAX_ELEMENTS", 2 * 20 * 63)
    parts = ops.conv2d_weight_grad8(a, dy, (3, 3), 1, (1, 1, 1, 1))
    size = O.conv2d_weight_grad(_vals(a).abs(), dy.cpu().double().abs(), (3, 3), 1, (1, 1, 1, 1), False)
    assert ((whole - parts).cpu().double().abs() <= 128 * 2.0 ** -24 * size + 1e-30).all()


# ---- how they are called ------------------------------------------------------------------------------------------------------
def test_strided_views_and_no_tokens(hific, dev):
    from hific_amd import ops
    w = _chan((1, 24), 101).to(dev)
    x = _rand((6, 24, 10), 102).to(dev)
    xt, wt = x.transpose(1, 2), w[:10].contiguous()
    assert torch.equal(ops.rms_norm(xt, wt), ops.rms_norm(xt.contiguous(), wt))
    odd = torch.empty(1 + x.numel(), device=dev)[1:].view(x.shape).copy_(x)              # 4 bytes past an aligned address
    assert torch.equal(ops.rms_norm(odd, w), ops.rms_norm(x, w))
    assert torch.equal(ops.checkpoint8(odd).q, ops.checkpoint8(x).q)
    xd, wd = torch.empty(0, 24, 4, device=dev, requires_grad=True), w.clone().requires_grad_()
    y, h = ops.rms_norm(xd, wd, resid=torch.empty(0, 24, 4, device=dev))
    dx, dw = torch.autograd.grad((y, h), (xd, wd), (y, h))
    assert y.shape == h.shape == dx.shape == xd.shape and torch.equal(dw, torch.zeros_like(dw))
    yd, a = ops.channel_norm8(xd, wd, wd.detach())
    dx, dw = torch.autograd.grad(yd, (xd, wd), yd)
    assert torch.equal(dw, torch.zeros_like(dw)) and ops.restore8(a).shape == xd.shape
    assert ops.restore8(ops.checkpoint8(torch.empty(3, 5, 0, device=dev))).shape == (3, 5, 0)
    b = ops.checkpoint8(torch.empty(0, 5, 6, 6, device=dev))
    assert torch.equal(ops.conv2d_weight_grad8(b, torch.empty(0, 7, 4, 4, device=dev), (3, 3)), torch.zeros(7, 5, 3, 3, device=dev))


def test_an_expanded_gradient_and_an_unused_output(hific, dev):
    from hific_amd import ops
    x, w, rs = (v.to(dev).requires_grad_() for v in (_rand((5, 40), 111), _chan((1, 40), 112), _rand((5, 40), 113)))
    y = ops.rms_norm(x, w)
    a, = torch.autograd.grad(y.sum(), x)
    b, = torch.autograd.grad(ops.rms_norm(x, w), x, torch.ones(5, 40, device=dev))
    assert torch.equal(a, b)
    y, h = ops.rms_norm(x, w, resid=rs)
    gx, gr = torch.autograd.grad(h.sum(), (x, rs))                                       # the norm itself is not used
    assert torch.equal(gx, torch.ones_like(gx)) and torch.equal(gr, gx)
    y, h = ops.rms_norm(x, w, resid=rs)
    gx, = torch.autograd.grad(y.sum(), x)                                                # the stream is not used
    hd = h.detach().requires_grad_()
    want, = torch.autograd.grad(ops.rms_norm(hd, w).sum(), hd)
    assert torch.equal(gx, want)


def test_refusals_on_the_device(hific, dev):
    from hific_amd import lib, ops
    x, w = torch.zeros(2, 8, 4, 4, device=dev), torch.ones(8, device=dev)
    a = ops.checkpoint8(x)
    bad = [lambda: ops.rms_norm(x, w[:7]), lambda: ops.rms_norm(x, w.half()), lambda: ops.rms_norm(x, w.cpu()), lambda: ops.rms_norm(x.half(), w),
           lambda: ops.rms_norm(x, w, resid=x[:1]), lambda: ops.rms_norm(x, w, resid=x.bfloat16()), lambda: ops.rms_norm(x, w, eps=0.0),
           lambda: ops.rms_norm(x, w, eps=float("nan")), lambda: ops.rms_norm(x, w, fmt="int4"), lambda: ops.rms_norm(x, torch.ones(16, device=dev)[::2]),
           lambda: ops.rms_norm8(x.clone().requires_grad_(), w), lambda: ops.channel_norm8(x, w, w[:4]), lambda: ops.restore8(a, torch.float16),
           lambda: ops.channel_norm_grad8(ops.Act8(a.q, a.e, w, w), x, w, w, torch.ones(2, 4, 4, device=dev)),
           lambda: ops.channel_norm_grad8(a, x[:, :, :2], w, w, torch.ones(2, 4, 4, device=dev)),
           lambda: ops.channel_norm_grad8(a, x, w, w, torch.ones(2, 4, device=dev)),
           lambda: ops.conv2d_weight_grad8(a, x, (3, 3)), lambda: ops.conv2d_weight_grad8(a, x, (3, 3), pads=(4, 4, 4, 4), pad_mode=lib.PAD_REFLECT),
           lambda: ops.conv2d_weight_grad8(a, x, (9, 9), pads=(4, 4, 4, 4)), lambda: ops.conv2d_weight_grad8(a, x, (3, 3), stride=0, pads=(1, 1, 1, 1)),
           lambda: ops.conv_transpose2d_weight_grad8(a, x, (3, 3), 2, 1, 1)]
    for i, f in enumerate(bad):
        with pytest.raises(lib.HificError):
            f()
            pytest.fail(f"refusal {i} was accepted")
    xd = x.clone().requires_grad_()
    g, = torch.autograd.grad(ops.rms_norm(xd, w), xd, torch.ones_like(x), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()                               # no second derivative, and it says so
    for f in (lambda: ops.rms_norm(xd, w), lambda: ops.channel_norm8(xd, w, w)[0]):
        with pytest.raises(lib.HificError):
            torch.autograd.grad(f().square().sum(), xd, create_graph=True)


@pytest.mark.parametrize("shape", [(5, 24), (5, 21), (2, 24, 3, 8), (2, 20, 3, 5), (2, 20, 1, 3)])
def test_tokens_that_are_not_finite_stay_so_and_alone(hific, dev, shape):
    """An infinity or NaN in a token: its 8-bit form restores to NaN, its gradient is NaN; the other tokens are as without it."""
    from hific_amd import ops
    x, w, b, dy = _rand(shape, 181), _chan(shape, 182), _chan(shape, 183, 0.0), _rand(shape, 184)
    flat = x.movedim(1, -1).reshape(-1, shape[1]).clone()
    flat[0, 3], flat[1, 7] = float("inf"), float("nan")
    bad = flat.reshape(shape[:1] + shape[2:] + shape[1:2]).movedim(-1, 1).contiguous()
    hit = ~torch.isfinite(bad).all(1, keepdim=True).expand(shape)
    for fmt in ("int8", "e4m3"):
        outs = []
        for v in (x, bad):
            xd = v.to(dev).requires_grad_()
            y, a = ops.channel_norm8(xd, w.to(dev), b.to(dev), relu=True, fmt=fmt)
            dx, = torch.autograd.grad(y, xd, dy.to(dev))
            z, c = ops.channel_norm8(v.to(dev), w.to(dev), b.to(dev), resid=v.to(dev), fmt=fmt)
            xr = v.to(dev).requires_grad_()
            dr, = torch.autograd.grad(ops.rms_norm(xr, w.to(dev), fmt=fmt), xr, dy.to(dev))
            outs.append([t.detach().cpu() for t in (y, ops.restore8(a), dx, z, ops.restore8(c), dr, ops.restore8(ops.rms_norm8(v.to(dev), w.to(dev), fmt=fmt)))])
        for i, (good, got) in enumerate(zip(*outs)):
            assert torch.isnan(got[hit]).all(), (fmt, i)
            assert torch.equal(got[~hit], good[~hit]), (fmt, i)


def test_kept_tensors_are_guarded_against_changes_in_place(hific, dev):
    from hific_amd import ops
    x, w = _rand((4, 16), 121).to(dev).requires_grad_(), _chan((1, 16), 122).to(dev)
    y, h = ops.rms_norm(x, w, resid=torch.zeros(4, 16, device=dev))
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_results_repeat_bit_for_bit(hific, dev):
    from hific_amd import ops
    for shape in ((300, 960), (3, 120, 24, 24), (3, 61, 9, 11)):
        x, w, dy = _rand(shape, 131, torch.bfloat16).to(dev), _chan(shape, 132).to(dev), _rand(shape, 133, torch.bfloat16).to(dev)
        got = []
        for _ in range(3):
            xd, wd = x.clone().requires_grad_(), w.clone().requires_grad_()
            y, a = ops.channel_norm8(xd, wd, w, relu=True)
            got.append((y.detach(), a.q.view(torch.uint8), a.e) + torch.autograd.grad(y, (xd, wd), dy))
        for g in got[1:]:
            assert all(torch.equal(p, q) for p, q in zip(g, got[0]))


def test_on_another_stream_and_two_calls_at_once(hific, dev):
    from hific_amd import ops
    shape = (8, 240, 32, 32)
    xs = [_rand(shape, 140 + i, torch.bfloat16).to(dev) for i in range(2)]
    w, dy = _chan(shape, 142).to(dev), _rand(shape, 143, torch.bfloat16).to(dev)

    def step(x):
        xd, wd = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = ops.rms_norm(xd, wd, fmt="int8")
        return (y,) + torch.autograd.grad(y, (xd, wd), dy)
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [None, None]
    for rep in range(4):
        for i, st in enumerate(streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got[i] = step(xs[i])
    torch.cuda.synchronize()
    for g, v in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, v))


def test_captured_and_replayed(hific, dev):
    """Two graphs, each a forward pass with its gradients in function form, replayed in turn with eager work between."""
    from hific_amd import ops
    shape = (2, 60, 24, 16)
    gamma, beta = _chan(shape, 151).to(dev), _chan(shape, 152, 0.0).to(dev)
    ins = [_rand(shape, 153 + i, torch.bfloat16).to(dev) for i in range(2)]
    dy = _rand(shape, 155, torch.bfloat16).to(dev)
    rstd = torch.rand(2, 24, 16, device=dev) + 0.5

    def step(x):
        with torch.no_grad():
            y, a = ops.channel_norm8(x, gamma, beta, relu=True)
            b = ops.checkpoint8(y)
            n, h = ops.rms_norm(x, gamma, resid=y)
        dx, dg, db = ops.channel_norm_grad8(ops.Act8(a.q, a.e), dy, gamma, beta, rstd, relu=True)
        return y, a.q.view(torch.uint8), b.q.view(torch.uint8), n, h, dx, dg, db, ops.conv2d_weight_grad8(b, dx, (3, 3), pads=(1, 1, 1, 1)), ops.restore8(a)
    st = torch.cuda.Stream()
    graphs, outs = [], []
    for x in ins:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            step(x)
        torch.cuda.current_stream().wait_stream(st)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st, capture_error_mode="relaxed"):
            outs.append(step(x))
        graphs.append(g)
    for rep in range(4):
        for i, x in enumerate(ins):
            x.copy_(_rand(shape, 160 + 2 * rep + i, torch.bfloat16))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x, out in zip(ins, outs):
            for k, (a, b) in enumerate(zip(out, step(x))):
                assert torch.equal(a, b), (rep, k)
        torch.cuda.synchronize()


def test_two_graphs_replayed_at_once(hific, dev):
    """Two graphs captured on one stream and replayed on two streams at the same time share nothing that is written."""
    from hific_amd import ops
    shape = (4, 120, 32, 32)
    gamma, beta = _chan(shape, 191).to(dev), _chan(shape, 192, 0.0).to(dev)
    ins = [_rand(shape, 193 + i, torch.bfloat16).to(dev) for i in range(2)]
    rstd = torch.rand(4, 32, 32, device=dev) + 0.5

    def step(x):
        with torch.no_grad():
            y, a = ops.channel_norm8(x, gamma, beta, relu=True)
            b8, h = ops.rms_norm8(x, gamma, resid=y)
        dx, dg, db = ops.channel_norm_grad8(ops.Act8(a.q, a.e), x, gamma, beta, rstd, relu=True)
        c = ops.checkpoint8(dx)
        return (y, h, dx, dg, db, ops.restore8(b8), ops.conv2d_weight_grad8(c, y, (3, 3), pads=(1, 1, 1, 1)),
                ops.conv2d_weight_grad8(c, y[:, :, :31, :31], (2, 2)))
    st = torch.cuda.Stream()
    want, graphs, outs = [], [], []
    for x in ins:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            want.append([t.clone() for t in step(x)])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st, capture_error_mode="relaxed"):
            outs.append(step(x))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for rep in range(6):
        for t in (t for o in outs for t in o):
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            for k, (p, q) in enumerate(zip(o, w)):
                assert torch.equal(p, q), (rep, k)


def test_many_small_planes(hific, dev):
    """More images than a workgroup's share of tiles: workgroups cross image borders; the channel sums are those of each image alone."""
    from hific_amd import ops
    shape = (3000, 12, 3, 4)
    x, w, dy = _rand(shape, 201, torch.bfloat16).to(dev), _chan(shape, 202).to(dev), _rand(shape, 203, torch.bfloat16).to(dev)
    xd, wd = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = ops.rms_norm(xd, wd, fmt="int8")
    q, e, rstd, _ = y.grad_fn.saved_tensors
    dx, dw = torch.autograd.grad(y, (xd, wd), dy)
    wdx, wdw = O.rms_norm_grad(O.values(q.cpu(), e.cpu()), rstd.cpu().double().unsqueeze(1), w.cpu(), dy.cpu())
    _close(dx, wdx, _half(torch.bfloat16), 64 * F32, "dx")
    _close(dw, wdw, 0.0, 8 * F32 * (dy.cpu().double() * O.values(q.cpu(), e.cpu())).abs().sum((0, 2, 3)), "dweight")
    y1 = ops.rms_norm(x[1234:1235], w)
    assert torch.equal(y1, y[1234:1235])


def test_a_tensor_beyond_32_bit_offsets(hific, dev):
    """2^31 + elements: rows of 2^16 channels; the last tokens are checked against the same rows alone."""
    from hific_amd import ops
    n, c = 32770, 65536
    x = torch.zeros(n, c, dtype=torch.bfloat16, device=dev)
    tail = _rand((3, c), 171, torch.bfloat16).to(dev)
    x[-3:] = tail
    w = torch.ones(c, device=dev)
    a, b = ops.checkpoint8(x), ops.checkpoint8(tail)
    assert torch.equal(a.q[-3:], b.q) and torch.equal(a.e[-3:], b.e) and int(a.q[:-3].abs().max()) == 0
    back = ops.restore8(a)
    assert torch.equal(back[-3:], ops.restore8(b))
    del back, a
    y = ops.rms_norm(x, w)
    assert torch.equal(y[-3:], ops.rms_norm(tail, w))
    del y, x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape", [(2 ** 21 + 37, 1, 8), (2 ** 21 + 37, 8), (2 ** 21 + 37, 9, 1, 1), (2 ** 26 + 77, 2), (2 ** 25 + 77, 2, 2)])
def test_more_tokens_than_one_launch_holds(hific, dev, shape):
    """Parts of the batch (planes, rows) or rounds of a workgroup (other shapes): every token as in a small batch, and the channel sums
    theirs.  A lane adds at most 2^21 / 512 tiles of eight values in a row, and a hundred terms follow: 33000 * 2^-24 of the terms' sum."""
    from hific_amd import ops
    n, m = shape[0], 4099
    whole, rest = divmod(n, m)

    def repeat(t):
        return torch.cat([t.repeat((whole,) + (1,) * (t.dim() - 1)), t[:rest]])
    base, dyb = (_rand((m,) + shape[1:], s, torch.bfloat16).to(dev) for s in (301, 302))
    w = _chan(shape, 303).to(dev)
    x, dy = repeat(base), repeat(dyb)
    a, b = ops.checkpoint8(x), ops.checkpoint8(base)
    assert torch.equal(a.q, repeat(b.q)) and torch.equal(a.e, repeat(b.e))
    assert torch.equal(ops.restore8(a), repeat(ops.restore8(b)))
    del a

    def count(t):                                        # sums over the large batch from the small one's terms
        return whole * t.sum(0) + t[:rest].sum(0)
    over = tuple(range(2, len(shape)))
    for kept in (None, "int8"):
        outs = []
        for xs, ds in ((base, dyb), (x, dy)):
            xd, wd = xs.clone().requires_grad_(), w.clone().requires_grad_()
            y = ops.rms_norm(xd, wd, fmt=kept)
            outs.append((y.detach(),) + torch.autograd.grad(y, (xd, wd), ds))
        (y0, dx0, _), (y1, dx1, dw1) = outs
        assert torch.equal(y1, repeat(y0)) and torch.equal(dx1, repeat(dx0)), kept
        xh = base.double() * torch.rsqrt(base.double().square().mean(1, keepdim=True) + 1e-6)
        if kept:
            y = ops.rms_norm(base.clone().requires_grad_(), w, fmt=kept)
            code = y.grad_fn.saved_tensors
            xh = O.values(code[0].cpu(), code[1].cpu()).to(dev)
        terms = (dyb.double() * xh).sum(over) if over else dyb.double() * xh
        size = (dyb.double() * xh).abs().sum(over) if over else (dyb.double() * xh).abs()
        _close(dw1, count(terms).cpu(), 0.0, 33000 * 2.0 ** -24 * count(size).cpu(), f"dweight {kept}")
    if shape[1] > 1:
        outs = []
        for xs, ds in ((base, dyb), (x, dy)):
            xd = xs.clone().requires_grad_()
            y, k = ops.channel_norm8(xd, w, w - 1, relu=True)
            outs.append((y.detach(), k.q, k.e) + torch.autograd.grad(y, xd, ds))
            del y, k
        for i, (s, t) in enumerate(zip(*outs)):
            assert torch.equal(t, repeat(s)), i
    del x, dy, outs
    torch.cuda.empty_cache()


def test_blocks_check_the_norm_against_the_convolution(hific, dev):
    from hific_amd import lib, ops
    from hific_amd.network.layers import HipConv2d
    from hific_amd.normalisation.channel import ChannelNorm2D
    conv, norm = HipConv2d(8, 16, 3).to(dev), ChannelNorm2D(12).to(dev)
    x = torch.zeros(1, 8, 10, 10, device=dev)
    with pytest.raises(lib.HificError, match="gamma"):
        ops.conv_norm8(x, None, conv, norm)
    norm = ChannelNorm2D(16).to(dev)
    for x8 in (ops.checkpoint8(x[:, :, :9]), x):
        with pytest.raises(lib.HificError, match="x8"):
            ops.conv_norm8(x, x8, conv, norm)
    with pytest.raises(lib.HificError, match="resid"):
        ops.conv_norm8(x, None, conv, norm, resid=x)


@pytest.mark.parametrize("transposed,n,c,h,w,k,r,stride,reflect", [
    (False, 2, 20, 9, 11, 24, 3, 1, False), (False, 2, 20, 9, 11, 24, 3, 1, True), (False, 1, 18, 21, 19, 33, 5, 2, True), (False, 3, 40, 17, 33, 8, 3, 2, False),
    (False, 1, 70, 8, 5, 20, 3, 1, True), (False, 2, 9, 40, 50, 40, 7, 1, True), (False, 1, 16, 30, 31, 20, 3, 3, False), (False, 9, 2, 33, 64, 5, 1, 1, False),
    (True, 2, 24, 9, 8, 40, 3, 2, False), (True, 1, 33, 7, 11, 20, 5, 2, False), (True, 2, 10, 5, 6, 12, 4, 3, False)])
def test_weight_gradient_form_of_odd_planes(hific, dev, transposed, n, c, h, w, k, r, stride, reflect):
    """The kernels that read the 8-bit tensor themselves, whatever the shape's rule says: values, and what an infinity of dy and a token
    that is not finite reach - the taps of the formula that see them (through the pad's zeros too), no others.  Products are exact; a sum
    of P positions per weight adds matrix instructions of 16 and at most 256 parts in a row."""
    from hific_amd import act8, lib, ops
    pad = r // 2
    a = ops.checkpoint8(_rand((n, c, h, w), 401).to(dev), fmt="e4m3")
    oh, ow = ((h - 1) * stride - 2 * pad + r + stride - 1, (w - 1) * stride - 2 * pad + r + stride - 1) if transposed else (
        (h + 2 * pad - r) // stride + 1, (w + 2 * pad - r) // stride + 1)
    dy = _rand((n, k, oh, ow), 402, torch.bfloat16)
    shape = (c, k, r, r) if transposed else (k, c, r, r)
    mode = lib.PAD_REFLECT if reflect else lib.PAD_ZERO

    def own(act, d):
        size = int(lib.raw("hific_wgrad8_ws_bytes")(int(transposed), n, c, h, w, k, r, r, oh, ow, stride))
        assert size > 0
        ws, dw, d = torch.empty(size, dtype=torch.uint8, device=dev), torch.empty(shape, device=dev), d.to(dev)
        lib.call("hific_wgrad8", int(transposed), lib.ptr(act.q), lib.ptr(act.e), 1, None, None, 0, lib.ptr(d), lib.ptr(dw), n, c, h, w, k, r, r, oh,
                 ow, stride, pad, pad, mode, 0, lib.ptr(ws), size, lib.stream())
        torch.cuda.synchronize()
        return dw.cpu()

    def formula(xv, dv):
        x, d = (dv, xv) if transposed else (xv, dv)          # x is padded and has the taps
        xp = torch.nn.functional.pad(x, (pad,) * 4 if not transposed else (pad, pad + r + stride) * 2, mode="reflect" if reflect else "constant")
        hh, ww = d.shape[2], d.shape[3]
        out = torch.empty(shape, dtype=torch.float64)
        for i in range(r):
            for j in range(r):
                t = xp[:, :, i:i + (hh - 1) * stride + 1:stride, j:j + (ww - 1) * stride + 1:stride]
                out[:, :, i, j] = (d.transpose(0, 1).flatten(1) @ t.transpose(0, 1).flatten(1).t())
        return out
    x = _vals(a)
    terms = n * h * w if transposed else n * oh * ow
    _close(own(a, dy), formula(x, dy.double()), 0.0, (terms / 16 + 272) * 2.0 ** -24 * formula(x.abs(), dy.double().abs()) + 1e-30, "dw")
    e = a.e.clone()
    e[0, 0, w - 1] = 255                                     # a corner, so that some taps never see it
    bad, xb, db = ops.Act8(a.q, e), x.clone(), dy.clone()
    xb[0, :, 0, w - 1] = float("nan")
    db[n - 1, 0, oh - 1, 0] = float("inf")
    for act, d, xv, dv in ((bad, dy, xb, dy), (a, db, x, db)):
        got, want = own(act, d), formula(xv, dv.double())
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
        assert torch.equal(got[torch.isinf(got)].double(), want[torch.isinf(want)])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 300, 7, 9), (1, 515, 5, 7), (3, 700, 9, 9), (1, 1100, 2, 4), (2, 513, 33, 16), (1, 2900, 5, 5), (1, 4096, 3, 3), (1, 4100, 2, 5)])
def test_planes_of_many_channels(hific, dev, shape, dt):
    """The tests above at the widths where a tile takes more waves, or none holds it."""
    for fmt in ("int8", "e4m3"):
        test_checkpoint_is_the_oracles_bit_for_bit(hific, dev, shape, dt, fmt)
        test_rms_norm8(hific, dev, shape, dt, True, fmt)
        for relu, resid in ((True, False), (False, True)):
            test_channel_norm8(hific, dev, shape, dt, relu, resid, fmt)
    for resid in (False, True):
        test_rms_norm_forward(hific, dev, shape, dt, resid)
        test_rms_norm_backward(hific, dev, shape, dt, resid, None)
    test_rms_norm_backward(hific, dev, shape, dt, True, "int8")


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 2, 24, 20), (3, 60, 8, 8), (1, 960, 16, 16), (2, 300, 7, 9), (2, 33, 2, 3), (1, 4100, 2, 5), (9, 40), (5, 3000), (6, 5)])
def test_tokens_of_equal_values(hific, dev, shape, dt, fmt):
    """Tokens without a deviation (a flat patch, zeros), and with one of the smallest numbers: normalised to nothing, never to NaN.  The
    mean of equal values is a rounded sum times a rounded 1 / C, so it misses them by up to F32 of their size (the chains that F32
    counts), and rsqrt(eps) multiplies that; of zeros and of the smallest numbers nothing is left at all."""
    from hific_amd import ops
    t = TYPES[dt]
    x, w, b = _rand(shape, 501, t), _chan(shape, 502), _chan(shape, 503, 0.0)
    flat = x.reshape(shape[0], shape[1], -1)
    tiny = torch.where(torch.arange(shape[1]) % 2 == 0, 2.0 ** -125, -2.0 ** -125).to(t)
    flat[0, :, 0], flat[-1, :, -1] = 0.0, 1.5
    flat[shape[0] // 2, :, flat.shape[2] // 2] = tiny
    alike = torch.zeros(flat[:, 0].shape, dtype=torch.bool)
    alike[0, 0] = alike[-1, -1] = alike[shape[0] // 2, flat.shape[2] // 2] = True
    dy, rs = _rand(shape, 504, t), _rand(shape, 505, t)

    def at(v):
        return v.detach().cpu().reshape(shape[0], shape[1], -1).transpose(1, 2)[alike].double()
    miss = F32 * at(x).abs().amax(1, keepdim=True) / math.sqrt(1e-3)
    for relu, resid in ((False, False), (True, False), (True, True), (False, True)):
        leaves = [v.to(dev).requires_grad_() for v in (x, w, b)]
        y, a = ops.channel_norm8(*leaves, relu=relu, resid=rs.to(dev) if resid else None, fmt=fmt)
        q, e, rstd, _, _ = y.grad_fn.saved_tensors
        kept = O.values(q.cpu(), e.cpu())
        grads = torch.autograd.grad(y, leaves, dy.to(dev))
        want = (torch.relu(b) if relu else b).double().expand(int(alike.sum()), -1)
        if resid:
            want = want.to(t).double() + at(rs)
        # (two roundings to the type with a residual: the norm's value, which miss may move across a border, and the sum)
        steps = _half(t) * want.abs() + (2 * _half(t) * (b.double().abs() + miss * w.double().abs()) if resid else 0.0)
        assert ((at(y) - want).abs() <= steps + 1.01 * miss * w.double().abs() + 2.0 ** -110).all()
        assert (at(kept).abs() <= 1.01 * miss + 2.0 ** -110).all() and torch.isfinite(kept).all()
        assert torch.isfinite(ops.restore8(a, torch.float32)).all()
        wdx, wdg, wdb = O.channel_norm_grad(kept, rstd.cpu().double().unsqueeze(1), w, b, dy, relu)
        size = rstd.cpu().double().unsqueeze(1) * (dy.double() * O._ch(w, x)).abs().amax(1, keepdim=True) * (1 + kept.abs().amax(1, keepdim=True)) * 2
        _close(grads[0], wdx, _half(t), F32 * size, "dx")
        dims = [0] + list(range(2, x.dim()))
        _close(grads[1], wdg, 0.0, 8 * F32 * (dy.double() * kept).abs().sum(dims) + 1e-30, "dgamma")
    z = x.clone()
    z.reshape(shape[0], shape[1], -1).transpose(1, 2)[alike] = 0
    zd, wd = z.to(dev).requires_grad_(), w.to(dev).requires_grad_()
    y = ops.rms_norm(zd, wd, fmt=fmt)
    q, e, rstd, _ = y.grad_fn.saved_tensors
    kept = O.values(q.cpu(), e.cpu())
    assert (at(kept) == 0).all() and (at(y) == 0).all() and torch.isfinite(kept).all()
    dx, _ = torch.autograd.grad(y, (zd, wd), dy.to(dev))
    assert torch.isfinite(dx).all()
    with torch.no_grad():
        assert (at(ops.restore8(ops.rms_norm8(zd, wd, fmt=fmt), torch.float32)) == 0).all()
