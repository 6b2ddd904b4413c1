"""8-bit activations, CPU side: the float64 oracle against torch's own formats, autograd and differences, and every refusal that
happens before a kernel is launched."""
import ctypes

import pytest
import torch

from oracle import act8_oracle as O


# ---- the oracle ---------------------------------------------------------------------------------------------------------
def test_e4m3_grid_is_torchs_format():
    codes = torch.arange(127, dtype=torch.uint8)
    assert torch.equal(codes.view(torch.float8_e4m3fn).double(), O.e4m3_values())
    t = torch.linspace(-448, 448, 40001, dtype=torch.float32).double()      # float32 values: torch's conversion rounds once
    assert torch.equal(O.grid("e4m3")[O.nearest(t, "e4m3")], t.float().to(torch.float8_e4m3fn).double())
    assert torch.equal(O.grid("int8")[O.nearest(t.clamp(-127, 127), "int8")], torch.round(t.clamp(-127, 127)))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_exponent_is_the_smallest_that_holds_the_largest_value(fmt):
    amax = torch.cat((torch.exp2(torch.arange(-130.0, 127.0, 0.37, dtype=torch.float64)), O.QMAX[fmt] * torch.exp2(torch.arange(-20.0, 20.0, dtype=torch.float64))))
    e = O.exponent(amax, fmt)
    assert (amax <= O.QMAX[fmt] * torch.exp2(e)).all()
    assert ((amax > O.QMAX[fmt] * torch.exp2(e - 1)) | (e == -126)).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_masked_rounding_keeps_the_side_of_the_relu(fmt):
    g = torch.Generator().manual_seed(3)
    v = torch.randn(64, 37, generator=g, dtype=torch.float64)
    gamma, beta = torch.randn(37, generator=g), 0.3 * torch.randn(37, generator=g)
    q, e = O.quantise(v, fmt, gamma, beta)
    side = lambda t: gamma.double() * t + beta.double() > 0  # noqa: E731
    assert torch.equal(side(q), side(v))
    plain, _ = O.quantise(v, fmt)
    moved = plain != q
    assert moved.any() and moved.double().mean() < 0.02            # rare: only values next to the threshold
    step = torch.exp2(e).unsqueeze(1) * (1.0 if fmt == "int8" else 32.0)
    assert ((q - v).abs() <= step).all()


def test_gradient_formulas_against_autograd_and_differences():
    g = torch.Generator().manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, b, dy, ds = rnd(3, 7, 4), rnd(7), rnd(7), rnd(3, 7, 4), rnd(3, 7, 4)

    def rms(t, wt):
        r = torch.rsqrt((t * t).mean(1, keepdim=True) + 1e-6)
        return (t * r * wt.view(1, -1, 1) * dy).sum() + (t * ds).sum()

    def chan(t, ga, be):
        return (torch.relu(O.channel_norm(t, ga, be)[0]) * dy).sum()

    xs, ws, bs = (t.clone().requires_grad_() for t in (x, w, b))
    r = torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-6)
    got = O.rms_norm_grad(x * r, r, w, dy, ds)
    want = torch.autograd.grad(rms(xs, ws), (xs, ws))
    for a, c in zip(got, want):
        assert torch.allclose(a, c, rtol=1e-9, atol=1e-11)
    _, xh, rc = O.channel_norm(x, w, b)
    gotc = O.channel_norm_grad(xh, rc, w, b, dy, True)
    wantc = torch.autograd.grad(chan(xs, ws, bs), (xs, ws, bs))
    for a, c in zip(gotc, wantc):
        assert torch.allclose(a, c, rtol=1e-9, atol=1e-11)
    # central differences along a direction: error O(eps^2)
    v, eps = rnd(3, 7, 4), 1e-5
    for f, dx in ((lambda t: rms(t, w), got[0]), (lambda t: chan(t, w, b), gotc[0])):
        diff = (f(x + eps * v) - f(x - eps * v)) / (2 * eps)
        assert abs(float(diff - (dx * v).sum())) < 1e-6 * (1 + abs(float(diff)))


def test_oracle_weight_gradient_against_autograd():
    g = torch.Generator().manual_seed(7)
    x = torch.randn(2, 3, 6, 5, generator=g, dtype=torch.float64)
    w = torch.randn(4, 3, 3, 3, generator=g, dtype=torch.float64, requires_grad=True)
    y = torch.nn.functional.conv2d(torch.nn.functional.pad(x, (1, 0, 0, 1), mode="reflect"), w, stride=2)
    dy = torch.randn(y.shape, generator=g, dtype=torch.float64)
    want, = torch.autograd.grad(y, w, dy)
    assert torch.allclose(O.conv2d_weight_grad(x, dy, (3, 3), 2, (0, 1, 1, 0), True), want, rtol=1e-10, atol=1e-12)


# ---- refusals -----------------------------------------------------------------------------------------------------------
def test_cpu_tensors_are_refused(hific):
    from hific_amd import lib, ops
    x, w = torch.zeros(2, 8, 4, 4), torch.ones(8)
    for f in (lambda: ops.rms_norm(x, w), lambda: ops.rms_norm8(x, w), lambda: ops.checkpoint8(x),
              lambda: ops.channel_norm8(x, w, w), lambda: ops.Act8(torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2, dtype=torch.uint8))):
        with pytest.raises(lib.HificError):
            f()


def test_arguments_are_checked_before_the_device(hific):
    from hific_amd import lib, ops
    x, w = torch.zeros(2, 8, 4, 4), torch.ones(8)
    bad = [lambda: ops.checkpoint8(x, fmt="int4"), lambda: ops.checkpoint8(torch.zeros(4)), lambda: ops.restore8(x),
           lambda: ops.rms_norm(torch.zeros(3), w), lambda: ops.channel_norm8(torch.zeros(2, 1, 4, 4), w[:1], w[:1]),
           lambda: ops.Act8(torch.zeros(2, 8), torch.zeros(2, dtype=torch.uint8)),
           lambda: ops.Act8(torch.zeros(2, 8, dtype=torch.int8), torch.zeros(3, dtype=torch.uint8)),
           lambda: ops.Act8(torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2, dtype=torch.uint8), relu=True),
           lambda: ops.checkpoint8(torch.empty(1, 1, 1).expand(1, 1, 2 ** 31)), lambda: ops.channel_norm_grad8(x, x, w, w, w), lambda: ops.conv2d_weight_grad8(x, x, (3, 3))]
    for f in bad:
        with pytest.raises(lib.HificError):
            f()


def test_entry_points_refuse_bad_arguments(hific):
    """Every refusal of the C entry points happens on the host, before a launch: no pointer is dereferenced."""
    from hific_amd import lib
    p = ctypes.c_void_p(4096)
    pack = lambda *a: lib.raw("hific_act8_pack")(*a)  # noqa: E731
    assert pack(None, p, p, 0, 1, 8, 4, 0, None) == -1
    assert pack(p, p, p, 2, 1, 8, 4, 0, None) == -1                       # format
    assert pack(p, p, p, 0, 1, 8, 4, 7, None) == -1                       # type
    for n, c, hw in ((0, 8, 4), (1, 0, 4), (1, 8, 0), (-1, 8, 4)):
        assert pack(p, p, p, 0, n, c, hw, 0, None) == -1
    rest = lib.raw("hific_act8_restore")
    assert rest(p, p, 0, p, None, 0, p, 1, 8, 4, 0, None) == -1           # gamma without beta
    assert rest(p, p, 0, None, None, 1, p, 1, 8, 4, 0, None) == -1        # relu without gamma
    rms = lib.raw("hific_rms_norm_fwd")
    assert rms(p, p, p, p, None, p, None, None, 0, 0, 1, 8, 4, 1e-6, 0, None) == -1     # resid without h
    assert rms(p, None, p, None, None, p, None, None, 0, 0, 1, 8, 4, 1e-6, 0, None) == -1   # nothing to write
    assert rms(p, None, p, p, None, p, p, None, 0, 0, 1, 8, 4, 1e-6, 0, None) == -1     # q without qe
    assert rms(p, None, p, p, None, p, None, None, 0, 0, 1, 8, 4, 0.0, 0, None) == -1   # eps
    assert rms(p, None, p, p, None, p, None, None, 0, 0, 1, 8, 4, float("nan"), 0, None) == -1
    rmsb = lib.raw("hific_rms_norm_bwd")
    assert rmsb(None, None, None, 0, p, p, None, p, p, p, 0, 1, 8, 4, 0, p, 1 << 20, None) == -1   # no source
    assert rmsb(p, p, p, 0, p, p, None, p, p, p, 0, 1, 8, 4, 0, p, 1 << 20, None) == -1            # two sources
    assert rmsb(p, None, None, 0, p, p, None, p, p, p, 0, 1, 8, 4, 0, p, 4, None) == -2            # workspace
    cn = lib.raw("hific_channelnorm8_fwd")
    assert cn(p, p, p, None, p, p, p, p, p, p, 0, 1, 8, 4, 1e-3, 0, 0, None) == -1      # q2 without resid
    assert cn(p, p, p, None, p, p, p, p, None, None, 0, 1, 1, 4, 1e-3, 0, 0, None) == -1    # one channel
    cnb = lib.raw("hific_channelnorm8_bwd")
    assert cnb(p, p, 0, p, p, p, p, p, p, p, 0, None, 0, 1, 8, 4, 0, 0, p, 4, None) == -2
    assert lib.raw("hific_norm8_bwd_ws_bytes")(0, 8, 4) == 0
    wg = lib.raw("hific_wgrad8")
    need = lib.raw("hific_wgrad8_ws_bytes")(0, 2, 8, 6, 6, 4, 3, 3, 6, 6, 1)
    assert need > 0 and lib.raw("hific_wgrad8_ws_bytes")(0, 2, 8, 6, 6, 0, 3, 3, 6, 6, 1) == 0
    ok = [0, p, p, 0, None, None, 0, p, p, 2, 8, 6, 6, 4, 3, 3, 6, 6, 1, 1, 1, 1, 0, p, need, None]

    def refuse(at, value):
        args = list(ok)
        args[at] = value
        return wg(*args)
    assert refuse(1, None) == refuse(3, 5) == refuse(4, p) == refuse(6, 1) == refuse(9, 0) == refuse(18, 0) == refuse(21, 3) == -1
    assert refuse(19, 6) == -1                                             # a reflection pad as large as the plane
    assert refuse(16, 99) == -1                                            # positions past the second border
    assert refuse(0, 1) == -1                                              # no reflection for the transposed form
    assert refuse(24, need - 1) == -2 and refuse(23, ctypes.c_void_p(4097)) == -2
    pref = lib.raw("hific_wgrad8_prefer")
    assert pref(0, 2, 120, 61, 47, 240, 3, 3, 31, 24, 2) == 1 and pref(0, 16, 960, 16, 16, 960, 3, 3, 16, 16, 1) == 0
    assert pref(0, 0, 120, 61, 47, 240, 3, 3, 31, 24, 2) == 0


def test_large_batches_go_in_slices(hific):
    from hific_amd import act8, lib
    assert act8._slices(5, 10) == [(0, 5)]
    per = 2 ** 30
    assert act8._slices(5, per) == [(0, 1), (1, 2), (2, 3), (3, 4), (4, 5)]
    assert act8._slices(3, 2 ** 29 + 7) == [(0, 3)]
    assert act8._slices(4, 2 ** 29 + 7) == [(0, 3), (3, 4)]
    with pytest.raises(lib.HificError):
        act8._slices(1, 2 ** 31)


def test_sizes_beyond_what_a_token_or_a_launch_may_have(hific):
    from hific_amd import act8, lib, ops
    p, wide = ctypes.c_void_p(4096), 2 ** 20 + 1
    assert lib.raw("hific_act8_pack")(p, p, p, 0, 1, wide, 1, 0, None) == -4
    assert lib.raw("hific_rms_norm_fwd")(p, None, p, p, None, p, None, None, 0, 0, 1, wide, 1, 1e-6, 0, None) == -4
    assert lib.raw("hific_rms_norm_bwd")(p, None, None, 0, p, p, None, p, p, p, 0, 1, wide, 1, 0, p, 1 << 40, None) == -4
    assert lib.raw("hific_channelnorm8_fwd")(p, p, p, None, p, p, p, p, None, None, 0, 1, wide, 4, 1e-3, 0, 0, None) == -4
    assert lib.raw("hific_channelnorm8_bwd")(p, p, 0, p, p, p, p, p, p, p, 0, None, 0, 1, wide, 4, 0, 0, p, 1 << 40, None) == -4
    assert lib.raw("hific_norm8_bwd_ws_bytes")(1, wide, 4) == 0
    with pytest.raises(lib.HificError):
        ops.checkpoint8(torch.empty(1, 1).expand(1, wide))
    assert act8._nchw(torch.empty(1, 1).expand(1, wide - 1)) == (1, wide - 1, 1)
