"""Derivatives that the 8-bit activation operators do not have are refused, never dropped: second derivatives under create_graph=True and
forward-mode derivatives."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rand(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _nodes(ops, dev):
    """name -> (function of (x, parameters), parameters)"""
    from hific_amd.network.layers import HipConv2d
    from hific_amd.normalisation.channel import ChannelNorm2D, fuse_bias_grad
    w, b = (1 + 0.2 * _rand((8,), 1)).to(dev), _rand((8,), 2).to(dev)
    r = _rand((2, 8, 6, 6), 3).to(dev)
    cw = _rand((8, 8, 3, 3), 4).to(dev)
    conv, norm = HipConv2d(8, 8, 3, stride=1, pads=(1, 1, 1, 1)).to(dev), ChannelNorm2D(8).to(dev)
    fuse_bias_grad(conv, norm)
    leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
    return {
        "rms_norm": (lambda x, p: ops.rms_norm(x, p[0]), [leaf(w)]),
        "rms_norm resid int8": (lambda x, p: ops.rms_norm(x, p[0], resid=r, fmt="int8")[0], [leaf(w)]),
        "channel_norm8": (lambda x, p: ops.channel_norm8(x, p[0], p[1])[0], [leaf(w), leaf(b)]),
        "conv2d": (lambda x, p: ops.conv2d(x, p[0], p[1], 1, (1, 1, 1, 1), x8=ops.checkpoint8(x)), [leaf(cw), leaf(b)]),
        "conv_norm8": (lambda x, p: ops.conv_norm8(x, ops.checkpoint8(x), conv, norm)[0], list(conv.parameters()) + list(norm.parameters())),
    }


@pytest.fixture(autouse=True)
def _mode(hific):
    from hific_amd import ops
    was = ops.get_compute_dtype()
    hific.set_compute_dtype(torch.float32)
    yield
    hific.set_compute_dtype(was)


@pytest.mark.parametrize("name", ["rms_norm", "rms_norm resid int8", "channel_norm8", "conv2d", "conv_norm8"])
def test_a_penalty_on_a_gradient_is_refused(hific, dev, name):
    """With a constant incoming gradient too: the gradients depend on the saved tensors.  As values they are those of a plain pass."""
    from hific_amd import lib, ops
    f, params = _nodes(ops, dev)[name]
    x, dy = _rand((2, 8, 6, 6), 5).to(dev).requires_grad_(), _rand((2, 8, 6, 6), 6).to(dev)
    plain = torch.autograd.grad(f(x, params), [x] + params, dy)
    got = torch.autograd.grad(f(x, params), [x] + params, dy, create_graph=True)
    for g, h in zip(got, plain):
        assert torch.equal(g, h) and g.requires_grad
        loss = (x * x).sum() + g.square().sum()          # the penalty may not vanish beside another term
        with pytest.raises(lib.HificError, match="second derivative"):
            loss.backward()
    x.grad = None
    f(x, params).backward(dy, create_graph=True)
    assert torch.equal(x.grad, plain[0])
    for p in [x] + params:
        p.grad = None
    with pytest.raises(lib.HificError, match="second derivative"):
        torch.autograd.grad(f(x, params).square().sum(), x, create_graph=True)


def test_gradients_that_are_passed_through_stay_constants(hific, dev):
    from hific_amd import ops
    x, r, w = (t.to(dev).requires_grad_() for t in (_rand((4, 8), 11), _rand((4, 8), 12), 1 + 0.2 * _rand((8,), 13)))
    y, h = ops.rms_norm(x, w, resid=r)
    g, = torch.autograd.grad(h.sum(), r, create_graph=True)              # the stream alone: 1, whatever x is
    assert torch.equal(g, torch.ones_like(g)) and not g.requires_grad
    z = _rand((2, 8, 4, 4), 14).to(dev)
    rs = _rand((2, 8, 4, 4), 15).to(dev).requires_grad_()
    y, _ = ops.channel_norm8(z, w, w, resid=rs)
    g, = torch.autograd.grad(y.sum(), rs, create_graph=True)
    assert torch.equal(g, torch.ones_like(g)) and not g.requires_grad


@pytest.mark.parametrize("which", ["x", "weight", "resid"])
def test_forward_mode_is_refused(hific, dev, which):
    """A tangent is refused, whether or not anything requires grad; without one a dual level changes nothing."""
    import torch.autograd.forward_ad as fwd
    from hific_amd import ops
    t = {"x": _rand((2, 8, 6, 6), 21).to(dev), "weight": _rand((8,), 22).to(dev), "resid": _rand((2, 8, 6, 6), 23).to(dev)}
    calls = [lambda a: ops.rms_norm(a["x"], a["weight"], resid=a["resid"]), lambda a: ops.rms_norm(a["x"], a["weight"], resid=a["resid"], fmt="int8"),
             lambda a: ops.rms_norm8(a["x"], a["weight"], resid=a["resid"]),
             lambda a: ops.channel_norm8(a["x"], a["weight"], t["weight"], resid=a["resid"])]
    want = ops.rms_norm(t["x"], t["weight"], resid=t["resid"])
    for grad in (False, True):
        with torch.set_grad_enabled(grad), fwd.dual_level():
            dual = dict(t, **{which: fwd.make_dual(t[which], torch.ones_like(t[which]))})
            for i, f in enumerate(calls):
                with pytest.raises(RuntimeError):
                    f(dual)
                    pytest.fail(f"call {i} lost a tangent")
            got = ops.rms_norm(t["x"], t["weight"], resid=t["resid"])
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            x = t["x"].clone()
            conv = lambda v: ops.conv2d(v, torch.ones(4, 8, 3, 3, device=dev), None, x8=ops.checkpoint8(x))  # noqa: E731
            with pytest.raises(RuntimeError):
                conv(fwd.make_dual(x, torch.ones_like(x)))
                pytest.fail("conv2d(x8=) lost a tangent")
