"""conv2d(x8=) with its parameters in and out of an arena, the side stream on and off, and an input whose gamma / beta nothing else
holds: the same gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rand(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


@pytest.fixture(autouse=True)
def _mode(hific):
    from hific_amd import ops
    was = ops.get_compute_dtype(), ops._SIDE_ON
    hific.set_compute_dtype(torch.bfloat16)
    yield
    hific.set_compute_dtype(was[0])
    ops.set_side_stream(was[1])


@pytest.mark.parametrize("in_arena", ["none", "weight", "bias", "both"])
def test_conv_with_an_8_bit_input_and_part_of_its_parameters_in_an_arena(hific, dev, in_arena):
    from hific_amd import ops, optim
    x, dy = _rand((4, 48, 40, 40), 1, torch.bfloat16).to(dev), _rand((4, 64, 40, 40), 2, torch.bfloat16).to(dev)
    a = ops.checkpoint8(x)
    res = []
    for side in (False, True):
        ops.set_side_stream(side)
        w = torch.nn.Parameter(_rand((64, 48, 3, 3), 3).to(dev))
        b = torch.nn.Parameter(_rand((64,), 4).to(dev))
        members = [p for p, n in ((w, "weight"), (b, "bias")) if in_arena in (n, "both")]
        arena = optim.ParamArena(members) if members else None
        for rep in range(3):                             # (the later passes add)
            xd = x.clone().requires_grad_()
            y = ops.conv2d(xd, w, b, 1, (1, 1, 1, 1), x8=a)
            # the bias gradient is read as soon as autograd has it
            y.backward(dy)
        torch.cuda.synchronize()
        res.append((w.grad.clone(), b.grad.clone(), xd.grad.clone()))
        assert arena is None or len(arena.slots) == len(members)
    for p, q in zip(*res):
        assert torch.equal(p, q)
    want = 3 * dy.double().sum((0, 2, 3))
    assert ((res[1][1].double() - want).abs() <= 3 * 6400 * 2.0 ** -24 * dy.double().abs().sum((0, 2, 3))).all()


def test_an_input_whose_norm_parameters_are_temporaries(hific, dev):
    """gamma = 1 + p is held by the node alone; once the node is done its memory is the main stream's to use again."""
    from hific_amd import ops, optim
    C = 48
    x, dy = _rand((4, C, 40, 40), 11, torch.bfloat16).to(dev), _rand((4, 64, 40, 40), 12, torch.bfloat16).to(dev)
    p, beta = (0.2 * _rand((C,), 13)).to(dev), (0.2 * _rand((C,), 14)).to(dev)
    kept = ops.checkpoint8(x)
    res = []
    for side in (False, True):
        ops.set_side_stream(side)
        w, b = (torch.nn.Parameter(_rand(s, n).to(dev)) for s, n in (((64, C, 3, 3), 15), ((64,), 16)))
        optim.ParamArena([w, b])
        for rep in range(3):
            a = ops.Act8(kept.q, kept.e, 1 + p, beta + 0, True)
            y = ops.conv2d(ops.restore8(a), w, b, 1, (1, 1, 1, 1), x8=a)
            del a
            y.backward(dy)
            del y
            for _ in range(8):
                torch.full((C,), float("nan"), device=dev)
        torch.cuda.synchronize()
        res.append((w.grad.clone(), b.grad.clone()))
    assert torch.isfinite(res[0][0]).all()
    for s, t in zip(*res):
        assert torch.equal(s, t)


@pytest.mark.parametrize("block", [False, True])
@pytest.mark.parametrize("in_arena", ["gamma", "beta", "both"])
def test_a_norm_with_one_parameter_in_an_arena(hific, dev, in_arena, block):
    """The second backward pass adds to the arena's gradient and hands the other one to autograd."""
    from hific_amd import ops, optim
    from hific_amd.network.layers import HipConv2d
    from hific_amd.normalisation.channel import ChannelNorm2D, fuse_bias_grad
    C = 32
    x = _rand((2, C, 12, 12), 21, torch.bfloat16).to(dev)
    dys = [_rand((2, C, 12, 12), 22 + i, torch.bfloat16).to(dev) for i in range(3)]
    torch.manual_seed(9)
    conv = HipConv2d(C, C, 3, stride=1, pads=(1, 1, 1, 1)).to(dev)
    start = ChannelNorm2D(C, fuse_relu=True).to(dev).state_dict()

    def run(members, n):
        norm = ChannelNorm2D(C, fuse_relu=True).to(dev)
        norm.load_state_dict(start)
        fuse_bias_grad(conv, norm)
        if members:
            optim.ParamArena([getattr(norm, m) for m in members])
        for dy in dys[:n]:
            xd = x.clone().requires_grad_()
            y = ops.conv_norm8(xd, ops.checkpoint8(x), conv, norm)[0] if block else ops.channel_norm8(xd, norm.gamma, norm.beta, relu=True)[0]
            y.backward(dy)
        torch.cuda.synchronize()
        return norm.gamma.grad.clone(), norm.beta.grad.clone()
    members = ["gamma", "beta"] if in_arena == "both" else [in_arena]
    for n in (1, 2, 3):
        for got, want in zip(run(members, n), run([], n)):
            # float32 sums of the same terms; the arena's is formed inside the kernel, autograd's outside
            assert float((got - want).abs().max()) <= 4 * 2.0 ** -24 * n * 288 * 4
