"""The 8-bit activation operators at the ends of the value range: tokens of the largest numbers, weights and values that are not finite,
sums of squares beyond float32.  Shapes reach every kernel: rows (one lane group, a wave, a workgroup, 1024 threads, too wide), rows of
few channels, planes in tiles of four and eight waves, tiny planes, planes too wide for a tile."""
import math

import pytest
import torch

from oracle import act8_oracle as O

pytestmark = pytest.mark.gpu
F32 = 32 * 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# (at least six tokens each)
SHAPES = [(7, 5), (6, 40), (6, 41), (9, 300), (6, 960), (6, 9000), (6, 16500), (2, 40, 8, 8), (2, 21, 3, 5), (1, 700, 9, 9), (3, 20, 1, 3), (2, 4100, 2, 5)]


def _rand(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _tokens(x):
    """[tokens, C] of x [N, C, ...], and the way back."""
    shape = x.shape
    flat = x.movedim(1, -1).reshape(-1, shape[1]).clone()
    return flat, lambda f: f.reshape(shape[:1] + shape[2:] + shape[1:2]).movedim(-1, 1).contiguous()


def _with_tops(shape, dt, tops, seed=1):
    """Token i holds tops[i] (of both signs, beside zeros and numbers of any size); the rest are ordinary."""
    flat, back = _tokens(_rand(shape, seed))
    for i, top in enumerate(tops):
        flat[i] *= 0.2 * top                             # (normal numbers, clipped to the largest)
        flat[i].clamp_(-top, top)
        flat[i, 1], flat[i, 2], flat[i, 3], flat[i, 4] = top, 0.0, -top, -0.0
        flat[i, 0] = 1.0 if i % 2 else -0.3 * top
    return back(flat.to(dt))


def _check_checkpoint(ops, x, fmt, dev):
    a = ops.checkpoint8(x.to(dev), fmt=fmt)
    back32, back16 = ops.restore8(a, torch.float32).cpu(), ops.restore8(a).cpu()
    want, e = O.quantise(x.double(), fmt)
    assert torch.equal(a.e.cpu().double() - 127, e)
    bad = ~torch.isfinite(x).all(1, keepdim=True).expand(x.shape)        # (rounding to the type may have reached infinity: NaN comes back)
    for v in (O.values(a.q.cpu(), a.e.cpu()), back32.double(), back16.double()):
        assert torch.isnan(v[bad]).all() and torch.isfinite(v[~bad]).all() and torch.equal(v[~bad], want[~bad])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_tokens_of_the_top_octave_restore_to_what_was_kept(hific, dev, shape, dt, fmt):
    """Around 127 * 2^120 (1.69e38), where a scale of 2^121 times 128 leaves float32, up to 127 * 2^121, the largest int8 value."""
    from hific_amd import ops
    tops = [1.6e38, 127 * 2.0 ** 120, 1.70e38, 2e38, 3e38, 127 * 2.0 ** 121 if fmt == "int8" else 448 * 2.0 ** 119]
    _check_checkpoint(ops, _with_tops(shape, TYPES[dt], tops), fmt, dev)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("transposed,n,c,h,w,k,r,stride,reflect", [
    (False, 2, 20, 9, 11, 24, 3, 1, False), (False, 1, 18, 21, 19, 33, 3, 2, True), (False, 2, 12, 6, 5, 9, 3, 1, False), (True, 2, 24, 9, 8, 40, 3, 2, False)])
def test_weight_gradients_of_the_top_octave(hific, dev, transposed, n, c, h, w, k, r, stride, reflect, fmt):
    """Exact products (of 2^121-sized values with gradients of 1e-9), at most 400 additions in a row in float32."""
    from hific_amd import act8, lib, ops
    pad = r // 2
    x = _with_tops((n, c, h, w), torch.float32, [1.6e38, 1.7e38, 2e38, 3e38], seed=3)
    a = ops.checkpoint8(x.to(dev), fmt=fmt)
    oh, ow = ((h - 1) * stride - 2 * pad + r + stride - 1, (w - 1) * stride - 2 * pad + r + stride - 1) if transposed else (
        (h + 2 * pad - r) // stride + 1, (w + 2 * pad - r) // stride + 1)
    dy = _rand((n, k, oh, ow), 4, torch.bfloat16, 1e-9)
    v = O.values(a.q.cpu(), a.e.cpu())
    if transposed:
        got = ops.conv_transpose2d_weight_grad8(a, dy.to(dev), (r, r), stride, pad, stride - 1)
        ref = lambda xv, d: O.conv2d_weight_grad(torch.nn.functional.pad(d, (pad, pad + stride) * 2), xv, (r, r), stride, (0, 0, 0, 0), False)  # noqa: E731
    else:
        got = ops.conv2d_weight_grad8(a, dy.to(dev), (r, r), stride, (pad,) * 4, lib.PAD_REFLECT if reflect else lib.PAD_ZERO)
        ref = lambda xv, d: O.conv2d_weight_grad(xv, d, (r, r), stride, (pad,) * 4, reflect)  # noqa: E731
    got = got.cpu().double()
    want, size = ref(v, dy.double()), ref(v.abs(), dy.double().abs())
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= 400 * 2.0 ** -24 * size + 1e-30).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_finite_tokens_stay_finite_up_to_the_types_maximum(hific, dev, shape, dt, fmt):
    """Above 127 * 2^121 (e4m3: 248 * 2^120) the nearest value is 2^128, which no float32 holds: the one below it is kept."""
    from hific_amd import ops
    t = TYPES[dt]
    tops = [torch.finfo(t).max, 127.5 * 2.0 ** 121, 127 * 2.0 ** 121 * (1 + 2.0 ** -7), 247 * 2.0 ** 120, 248 * 2.0 ** 120, 249 * 2.0 ** 120]
    _check_checkpoint(ops, _with_tops(shape, t, tops, seed=5), fmt, dev)
    if shape[1] > 1:                                     # and as a norm's output: y = norm(x) + resid, kept as it is stored
        x = _rand(shape, 6, t)
        rs = _with_tops(shape, t, tops, seed=7)
        y, a = ops.channel_norm8(x.to(dev), torch.zeros(shape[1], device=dev), torch.zeros(shape[1], device=dev), resid=rs.to(dev), fmt=fmt)
        assert torch.equal(y.cpu(), rs)
        want, e = O.quantise(rs.double(), fmt)
        assert torch.equal(a.e.cpu().double() - 127, e)
        assert torch.equal(torch.nan_to_num(ops.restore8(a, torch.float32).cpu().double()), torch.nan_to_num(want))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rms_norm8_of_weights_and_values_that_are_not_finite(hific, dev, shape, dt, fmt):
    """A token whose output holds an infinity or NaN is not finite as a whole, wherever that came from: a NaN or an infinity among the
    weights (times a zero too), or an infinite value in a channel of weight zero.  The other tokens are as without it."""
    from hific_amd import ops
    t = TYPES[dt]
    x, w = _rand(shape, 11, t), 1.0 + 0.3 * _rand((shape[1],), 12)
    w[1] = 0.0

    def run(xv, wv):
        a = ops.rms_norm8(xv.to(dev), wv.to(dev), fmt=fmt)
        return a.e.cpu(), ops.restore8(a, torch.float32).cpu()
    e0, good = run(x, w)
    assert torch.isfinite(good).all() and not (e0 == 255).any()
    flat, back = _tokens(x)
    flat[0, 3] = 0.0
    for value in (float("nan"), float("inf"), float("-inf")):
        bad = w.clone()
        bad[3] = value
        e, got = run(back(flat), bad)
        assert (e == 255).all() and torch.isnan(got).all(), value
    flat[0, 3] = x.movedim(1, -1).reshape(-1, shape[1])[0, 3]
    flat[2, 1] = float("inf")                            # (its weight is zero)
    flat[4, 0], flat[5, 4] = float("-inf"), float("nan")
    e, got = run(back(flat), w)
    hit = ~torch.isfinite(back(flat)).all(1)
    assert hit.sum() == 3 and torch.equal(e == 255, hit)
    hit = hit.unsqueeze(1).expand(shape)
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], good[~hit])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("channels", [5, 41, 47, 55, 61, 82, 97, 220, 301, 947, 960, 2090, 4100, 16500])
@pytest.mark.parametrize("positions", [(), (8, 9), (1, 3)])
def test_means_of_equal_terms_are_exact(hific, dev, channels, positions, dt):
    """Sums of C equal terms that float32 holds exactly, divided by C, are those terms (a product with a rounded 1 / C misses them for
    C = 41, 47, 55, ...): tokens of +-1 have the mean square 1, and a flat token of 1.5 is its own mean - normalised to zero, not to
    roundings times rsqrt(eps)."""
    from hific_amd import ops
    t = TYPES[dt]
    shape = (3, channels) + positions
    sign = torch.where(_rand(shape, 61) > 0, 1.0, -1.0).to(t)
    w, b = torch.ones(channels), 0.25 * _rand((channels,), 62)
    y = ops.rms_norm(sign.to(dev), w.to(dev), eps=1e-12)
    assert torch.equal(y.cpu(), sign)
    # dx = r (g - xh mean(g xh)) with g = xh: nothing is left
    x = sign.to(dev).requires_grad_()
    dx, = torch.autograd.grad(ops.rms_norm(x, w.to(dev), eps=1e-12), x, sign.to(dev))
    assert torch.equal(dx.cpu(), torch.zeros(shape, dtype=t))
    flat = torch.full(shape, 1.5, dtype=t).to(dev).requires_grad_()
    y, a = ops.channel_norm8(flat, w.to(dev), b.to(dev))
    assert torch.equal(y.detach().cpu(), b.reshape((1, -1) + (1,) * len(positions)).expand(shape).to(t))
    q, e, rstd, _, _ = y.grad_fn.saved_tensors
    assert (e == 1).all() and not q.any()
    # dx = r (g - mean(g)) with xh = 0 and equal g
    dx, = torch.autograd.grad(y, flat, torch.full(shape, 0.75, dtype=t).to(dev))
    assert torch.equal(dx.cpu(), torch.zeros(shape, dtype=t))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_norms_of_values_whose_squares_leave_float32(hific, dev, shape, dt):
    """Values of 1e19 to the type's maximum: normalised values are of order one, as for any other size.  rstd may be as small as 2^-128,
    where float32 has 21 bits: F32 counts 2^-19."""
    from hific_amd import ops
    t = TYPES[dt]
    C = shape[1]
    w, b = 1.0 + 0.3 * _rand((C,), 21), 0.2 * _rand((C,), 22)
    flat, back = _tokens(_rand(shape, 23))
    for i, size in enumerate((1e19, 3e20, 1e25, 1e33, 2e37)):
        flat[i] *= size
    flat[5] = torch.finfo(t).min                         # (a mask's value in every channel)
    x = back(flat.to(t))
    dy, rs = _rand(shape, 24, t), _rand(shape, 25, t)
    half = torch.finfo(t).eps / 2
    y, h, r = O.rms_norm(x, w, rs)
    assert torch.isfinite(h).all()
    for fmt in (None, "int8", "e4m3"):
        leaves = [v.to(dev).requires_grad_() for v in (x, w, rs)]
        gy, gh = ops.rms_norm(leaves[0], leaves[1], resid=leaves[2], fmt=fmt)
        rstd = gy.grad_fn.saved_tensors[2].detach().cpu().double()
        dx, dw = torch.autograd.grad(gy, leaves[:2], dy.to(dev))
        assert torch.equal(gh.cpu(), h)
        assert ((gy.cpu().double() - y).abs() <= (half + F32) * y.abs()).all(), fmt
        assert ((rstd.unsqueeze(1) - r).abs() <= F32 * r).all()
        assert torch.isfinite(dx).all() and torch.isfinite(dw).all()
        xh = h.double() * r
        if fmt is None:
            _, wdw = O.rms_norm_grad(xh, r, w, dy)
            terms = (dy.double() * xh).abs().sum([0] + list(range(2, x.dim())))
            assert ((dw.cpu().double() - wdw).abs() <= 8 * F32 * terms).all()
    a, _ = ops.rms_norm8(x.to(dev), w.to(dev), resid=rs.to(dev), fmt="int8")
    step = torch.exp2(a.e.cpu().double() - 127).unsqueeze(1)
    assert ((ops.restore8(a, torch.float32).cpu().double() - y).abs() <= 0.5 * step * (1 + 1e-6) + F32 * y.abs()).all()
    # the channel norm: sums of C values have to stay in float32 (a token whose sum does not is NaN, not a quiet zero)
    flat[4], flat[5] = flat[4].clamp(-1e38 / C, 1e38 / C), torch.where(torch.arange(C) % 2 == 0, 1e38 / C, -1e38 / C)
    x = back(flat.to(t))
    v, xh, r = O.channel_norm(x, w, b)
    big = 1 + xh.abs().amax(1, keepdim=True) + x.double().abs().amax(1, keepdim=True) * r
    for relu in (False, True):
        leaves = [z.to(dev).requires_grad_() for z in (x, w, b)]
        gy, a = ops.channel_norm8(*leaves, relu=relu)
        q, e, rstd, _, _ = gy.grad_fn.saved_tensors
        want = torch.relu(v) if relu else v
        assert ((gy.detach().cpu().double() - want).abs() <= half * want.abs() + 2 * F32 * big * (1 + O._ch(w, x).abs())).all()
        kept, scale = O.values(q.cpu(), e.cpu()), torch.exp2(e.cpu().double() - 127).unsqueeze(1)
        assert ((kept - xh).abs() <= (1.0 if relu else 0.5) * scale * (1 + 1e-6) + F32 * big).all()
        assert all(torch.isfinite(g).all() for g in torch.autograd.grad(gy, leaves, dy.to(dev)))
    flat[5] = torch.finfo(t).max
    gy, a = ops.channel_norm8(back(flat.to(t)).to(dev), w.to(dev), b.to(dev), relu=True)
    hit = (back(flat) == back(flat)[0, 0].new_tensor(torch.finfo(t).max)).all(1, keepdim=True).expand(shape)
    assert torch.isnan(gy.cpu()[hit]).all() and torch.isnan(ops.restore8(a).cpu()[hit]).all()
    assert torch.isfinite(gy.cpu()[~hit]).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rms_norm8_where_value_times_weight_leaves_float32(hific, dev, shape, fmt):
    """y = (x r) w is of ordinary size, x w is not: above 2^128 for values of 1e38 with weights of 1e3, below 2^-126 for values of 1e-20
    with weights of 1e-25 (and an eps of 1e-36).  Steps are those of y."""
    from hific_amd import ops
    flat, back = _tokens(_rand(shape, 31))
    for size, weight, eps in ((1e37, 1e3, 1e-6), (1e-20, 1e-25, 1e-36)):
        x, w = back(flat * size), weight * (1 + 0.3 * _rand((shape[1],), 32))
        xd = x.double()
        y = xd / torch.sqrt((xd * xd).mean(1, keepdim=True) + eps) * O._ch(w, x)
        a = ops.rms_norm8(x.to(dev), w.to(dev), eps=eps, fmt=fmt)
        got, e = ops.restore8(a, torch.float32).cpu().double(), a.e.cpu().double() - 127
        amax = y.abs().amax(1)
        assert (amax <= O.QMAX[fmt] * torch.exp2(e) * (1 + F32)).all() and (amax > O.QMAX[fmt] * torch.exp2(e - 1) * (1 - F32)).all()
        s = torch.exp2(e).unsqueeze(1)
        half = 0.5 * s if fmt == "int8" else torch.exp2(torch.floor(torch.log2((y.abs() / s).clamp_min(2.0 ** -6)))) * 2.0 ** -4 * s
        assert ((got - y).abs() <= half * (1 + 1e-6) + F32 * y.abs()).all()
