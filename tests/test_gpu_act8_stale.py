"""An Act8 that a norm returned stands for that norm's output: it is refused once the norm's parameters are others."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rand(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _uses(ops, x, a):
    w = _rand((4, 16, 3, 3), 9).to(x.device)
    dy = _rand((2, 4, 8, 8), 8).to(x.device)
    return {"restore8": lambda: ops.restore8(a), "conv2d": lambda: ops.conv2d(x, w, None, 1, (1, 1, 1, 1), x8=a),
            "conv2d_weight_grad8": lambda: ops.conv2d_weight_grad8(a, dy, (3, 3), 1, (1, 1, 1, 1)),
            "conv_transpose2d_weight_grad8": lambda: ops.conv_transpose2d_weight_grad8(a, dy, (3, 3), 1, 1, 0)}


@pytest.mark.parametrize("change", ["in place", "torch optimizer", "arena optimizer"])
@pytest.mark.parametrize("block", [False, True])
def test_values_of_a_changed_norm_are_refused(hific, dev, block, change):
    from hific_amd import lib, ops, optim
    from hific_amd.network.layers import HipConv2d
    from hific_amd.normalisation.channel import ChannelNorm2D, fuse_bias_grad
    was = ops.get_compute_dtype()
    hific.set_compute_dtype(torch.float32)
    try:
        conv, norm = HipConv2d(16, 16, 3, stride=1, pads=(1, 1, 1, 1)).to(dev), ChannelNorm2D(16, fuse_relu=True).to(dev)
        fuse_bias_grad(conv, norm)
        adam = optim.FusedAdam(list(norm.parameters()), lr=0.1) if change == "arena optimizer" else None
        x = _rand((2, 16, 8, 8), 1).to(dev)

        def forward():
            return ops.conv_norm8(x, None, conv, norm) if block else ops.channel_norm8(x, norm.gamma, norm.beta, relu=True)
        y, a = forward()
        before = ops.restore8(a, torch.float32)
        y.sum().backward()
        for name, use in _uses(ops, x, a).items():
            use()                                        # (a backward pass alone changes nothing)
        if adam is not None:
            adam.step()
        elif change == "torch optimizer":
            torch.optim.SGD(list(norm.parameters()), lr=0.1).step()
        else:
            with torch.no_grad():
                norm.beta.add_(1.0)
        for name, use in _uses(ops, x, a).items():
            with pytest.raises(lib.HificError, match="changed"):
                use()
                pytest.fail(f"{name} took values of another norm")
        b = ops.Act8(a.q, a.e, a.gamma, a.beta, a.relu)          # by hand it stands for what its tensors say now
        assert not torch.equal(ops.restore8(b, torch.float32), before)
        y, a = forward()
        for use in _uses(ops, x, a).values():
            use()
    finally:
        hific.set_compute_dtype(was)


def test_a_residual_output_is_held_by_itself(hific, dev):
    """With a residual the Act8 holds y's own values: nothing of it changes."""
    from hific_amd import ops
    x = _rand((2, 16, 8, 8), 2).to(dev)
    g, b = torch.nn.Parameter(torch.ones(16, device=dev)), torch.nn.Parameter(torch.zeros(16, device=dev))
    y, a = ops.channel_norm8(x, g, b, resid=x)
    before = ops.restore8(a)
    with torch.no_grad():
        g.mul_(3.0)
    assert torch.equal(ops.restore8(a), before)


def test_inference_mode(hific, dev):
    """Inference tensors have no version counter."""
    from hific_amd import ops
    x, p = _rand((2, 16, 8, 8), 3).to(dev), torch.zeros(16, device=dev)
    want, _ = ops.channel_norm8(x, 1 + p, p, relu=True)
    with torch.inference_mode():
        y, a = ops.channel_norm8(x, 1 + p, 0 * p, relu=True)
        assert torch.equal(y, want) and ops.restore8(a).shape == y.shape
        z, h = ops.rms_norm8(x, 1 + p, resid=x)
        ops.restore8(z)
    ops.restore8(a)
