"""The 8-bit activations in the framework's own training path (ops.set_checkpoint8): one conv -> norm block bit for bit against the
operators it is made of, the Generator and the Encoder against their plain forms, memory, streams and a captured training cycle.

Tolerances of the whole networks: both runs are bfloat16, so their forward values differ by roundings only (the norm sums its channels
in another order).  A weight gradient of the 8-bit run sees inputs that are off by u = step / sqrt(12) rms, step <= 2^-6 of the largest
value of a token (int8: max|v| uses at least half of 127 codes), the largest of a few hundred values being about 3.5 rms: u <= 1.6 % of
the rms; e4m3: half a step is at most 2^-4 of a value, 2^-4 / sqrt(3) = 3.6 %.  The data gradient carries a small part of that from
layer to layer (only the norm's projection reads the kept values), and the masks none.  Bounds on ||difference|| / ||gradient|| per
parameter: 3 u + 0.05 for the two bfloat16 runs' own roundings."""
import pytest
import torch

from oracle import act8_oracle as O8
from oracle import hific_oracle as O

pytestmark = pytest.mark.gpu
BOUND = {"int8": 3 * 0.016 + 0.05, "e4m3": 3 * 0.036 + 0.05}


def _rand(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


@pytest.fixture(autouse=True)
def _mode(hific):
    from hific_amd import ops
    was = ops.get_compute_dtype(), ops.exact_index_on()
    yield
    hific.set_compute_dtype(was[0])
    ops.set_exact_index(was[1])
    ops.set_checkpoint8(None)


# ---- one block ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("cd", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("transposed,relu,resid,given", [(False, True, False, True), (False, False, True, True), (False, True, False, False),
                                                         (True, True, False, True)])
def test_block_is_its_operators(hific, dev, transposed, relu, resid, given, cd, fmt):
    """conv_norm8 = convolution, channel_norm8, channel_norm_grad8, the convolution's data gradient, conv*_weight_grad8: bit for bit.
    `given`: the input comes with its 8-bit form (as values of a norm); otherwise the input itself is kept."""
    from hific_amd import lib, ops
    from hific_amd.network.layers import HipConv2d, HipConvTranspose2d
    from hific_amd.normalisation import channel
    hific.set_compute_dtype(cd)
    torch.manual_seed(3)
    if transposed:
        conv = HipConvTranspose2d(32, 48, 3, stride=2, padding=1, output_padding=1).to(dev)
    else:
        conv = HipConv2d(32, 32, 3, stride=1, pads=(1, 1, 1, 1), pad_mode="reflect").to(dev)
    K = conv.out_channels
    norm = channel.ChannelNorm2D(K, fuse_relu=relu).to(dev)
    with torch.no_grad():
        norm.gamma.add_(0.3 * torch.randn_like(norm.gamma)); norm.beta.add_(0.3 * torch.randn_like(norm.beta))
    channel.fuse_bias_grad(conv, norm)
    x = _rand((3, 32, 12, 16), 1, cd).to(dev)
    x8 = None
    if given:
        a = ops.checkpoint8(x, fmt)
        g8, b8 = (1 + 0.2 * _rand((32,), 2)).to(dev), (0.2 * _rand((32,), 3)).to(dev)
        x8 = ops.Act8(a.q, a.e, g8, b8, True)
        x = ops.restore8(x8, cd)
    out = (3, K, 24, 32) if transposed else (3, K, 12, 16)
    dy = _rand(out, 4, cd).to(dev)
    rs = _rand(out, 5, cd).to(dev).requires_grad_() if resid else None
    xd = x.clone().requires_grad_()
    y, y8 = ops.conv_norm8(xd, x8, conv, norm, resid=rs, fmt=fmt)
    if given:
        assert sum(t.numel() * t.element_size() for t in y.grad_fn.saved_tensors[:2]) <= 1.1 * x.numel()
    y.backward(dy)
    with torch.no_grad():
        if transposed:
            z = ops.conv_transpose2d(x, conv.weight, conv.bias, 2, 1, 1)
        else:
            z = ops.conv2d(x, conv.weight, conv.bias, 1, conv.pads, conv.hip_pad_mode)
    zd, rd = z.clone().requires_grad_(), None if rs is None else rs.detach()
    g, b = norm.gamma.detach(), norm.beta.detach()
    yr, ar = ops.channel_norm8(zd, g, b, norm.eps, relu, rd, fmt)
    q, e, rstd, _, _ = yr.grad_fn.saved_tensors
    assert torch.equal(y, yr) and torch.equal(y8.q.view(torch.uint8), ar.q.view(torch.uint8)) and torch.equal(y8.e, ar.e)
    assert torch.equal(ops.restore8(y8), ops.restore8(ar))
    dz, dg, db = ops.channel_norm_grad8(ops.Act8(q, e), dy, g, b, rstd, relu=relu)
    assert torch.equal(norm.gamma.grad, dg) and torch.equal(norm.beta.grad, db)
    xr = x.clone().requires_grad_()
    if transposed:
        ops.conv_transpose2d(xr, conv.weight.detach(), None, 2, 1, 1).backward(dz)
    else:
        ops.conv2d(xr, conv.weight.detach(), None, 1, conv.pads, conv.hip_pad_mode).backward(dz)
    assert torch.equal(xd.grad, xr.grad)
    kept = x8 if given else None
    if kept is not None:
        dw = ops.conv_transpose2d_weight_grad8(kept, dz, (3, 3), 2, 1, 1) if transposed else \
            ops.conv2d_weight_grad8(kept, dz, (3, 3), 1, conv.pads, conv.hip_pad_mode)
    else:
        wr = conv.weight.detach().clone().requires_grad_()
        ops.conv2d(x, wr, None, 1, conv.pads, conv.hip_pad_mode).backward(dz)
        dw = wr.grad
    assert torch.equal(conv.weight.grad, dw)
    # the bias gradient: the sum of dz as stored; 768 .. 2304 values in float32, at most 64 in a row
    want, size = dz.double().sum((0, 2, 3)), dz.double().abs().sum((0, 2, 3))
    assert ((conv.bias.grad.double() - want).abs() <= 128 * 2.0 ** -24 * size).all()
    if resid:
        assert torch.equal(rs.grad, dy)


@pytest.mark.parametrize("cd", [torch.float32, torch.bfloat16])
def test_conv_with_an_8_bit_input(hific, dev, cd):
    from hific_amd import lib, ops
    hific.set_compute_dtype(cd)
    x = _rand((2, 24, 10, 14), 11, cd).to(dev)
    a = ops.checkpoint8(x)
    w, b = _rand((20, 24, 3, 3), 12).to(dev).requires_grad_(), _rand((20,), 13).to(dev).requires_grad_()
    for out_f32 in (False, True):                            # (a float32 dy in bfloat16 mode goes the other way: restore first)
        xd = x.clone().requires_grad_()
        y = ops.conv2d(xd, w, b, 1, (1, 1, 1, 1), out_f32=out_f32, x8=a)
        dy = _rand(y.shape, 14, y.dtype).to(dev)
        got = torch.autograd.grad(y, (xd, w, b), dy)
        xr = x.clone().requires_grad_()
        yr = ops.conv2d(xr, w, b, 1, (1, 1, 1, 1), out_f32=out_f32)
        want = torch.autograd.grad(yr, (xr, w, b), dy)
        assert torch.equal(y, yr) and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
        back = ops.restore8(a, cd)
        # the weight gradient of the restored input: the same exact products, summed in another order (2^-24 per addition, chains of at
        # most 280 positions)
        ref = O8.conv2d_weight_grad(back.cpu(), dy.cpu(), (3, 3), 1, (1, 1, 1, 1), False)
        size = O8.conv2d_weight_grad(back.cpu().abs(), dy.cpu().abs(), (3, 3), 1, (1, 1, 1, 1), False)
        # (float32 out in bfloat16 mode: dy is rounded to bfloat16 by the tile loaders, half a step of 2^-8)
        half = 2.0 ** -8 if cd == torch.bfloat16 and out_f32 else 0.0
        assert ((got[1].cpu().double() - ref).abs() <= (half + 280 * 2.0 ** -24) * size).all()
    with pytest.raises(lib.HificError):
        ops.conv2d(x, w, b, 1, (1, 1, 1, 1), act="relu", x8=a)
    with pytest.raises(lib.HificError):
        ops.conv2d(x, w, b, 1, (1, 1, 1, 1), x8=ops.checkpoint8(x[:1]))


# ---- the networks ---------------------------------------------------------------------------------------------------------
def _generator(hific, dev, n_res=2):
    from hific_amd.network import generator
    torch.manual_seed(7)
    return generator.Generator((3, 8, 8), 2, C=24, n_residual_blocks=n_res).to(dev).train()


def _step(net, x, dy, fmt):
    from hific_amd import ops
    ops.set_checkpoint8(fmt)
    xd = x.clone().requires_grad_()
    net.zero_grad(set_to_none=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    y = net(xd)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated() - before
    y.backward(dy.to(y.dtype))
    torch.cuda.synchronize()
    ops.set_checkpoint8(None)
    return y.detach(), xd.grad, {n: p.grad for n, p in net.named_parameters()}, held


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_generator(hific, dev, fmt):
    hific.set_compute_dtype(torch.bfloat16)
    net = _generator(hific, dev)
    x, dy = _rand((4, 24, 16, 16), 21).to(dev), _rand((4, 3, 256, 256), 22, scale=1e-2).to(dev)
    _step(net, x, dy, None)                                  # (workspaces and packed weights exist from here on)
    y0, dx0, g0, held0 = _step(net, x, dy, None)
    y1, dx1, g1, held1 = _step(net, x, dy, fmt)
    scale = float(y0.float().abs().max())
    assert float((y0.float() - y1.float()).abs().max()) <= 0.05 * scale         # two bfloat16 forwards
    assert set(g0) == set(g1)
    for n in g0:
        a, b = g0[n].double(), g1[n].double()
        if n.endswith(".bias") and n != "conv_block_out.1.bias":
            continue      # a bias in front of a norm: its gradient is zero but for roundings
        assert float((a - b).norm()) <= BOUND[fmt] * float(a.norm()), (n, float((a - b).norm() / a.norm()))
    assert float((dx0 - dx1).norm()) <= BOUND[fmt] * float(dx0.norm())
    assert held1 < 0.5 * held0, (held0, held1)               # what a forward pass holds for its backward pass
    with torch.no_grad():
        from hific_amd import ops
        ops.set_checkpoint8(fmt)
        y2 = net(x)                                          # nothing is kept without gradients: the plain path
    assert torch.equal(y2, y0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_encoder(hific, dev, fmt):
    from hific_amd import ops
    from hific_amd.network import encoder
    hific.set_compute_dtype(torch.bfloat16)
    torch.manual_seed(8)
    net = encoder.Encoder((3, 128, 128), 2, C=24).to(dev).train()
    x, dy = torch.rand((4, 3, 128, 128), generator=torch.Generator().manual_seed(23)).to(dev), _rand((4, 24, 8, 8), 24).to(dev)
    ops.set_exact_index(True)
    ye, _, ge, _ = _step(net, x, dy, fmt)                    # the exact-index chain is not changed by the option
    yp, _, gp, _ = _step(net, x, dy, None)
    assert torch.equal(ye, yp) and all(torch.equal(ge[n], gp[n]) for n in ge)
    ops.set_exact_index(False)
    _step(net, x, dy, None)
    y0, dx0, g0, held0 = _step(net, x, dy, None)
    y1, dx1, g1, held1 = _step(net, x, dy, fmt)
    assert float((y0 - y1).abs().max()) <= 0.05 * float(y0.abs().max())
    for n in g0:
        if n.endswith(".bias") and not n.startswith("conv_block_out"):
            continue
        assert float((g0[n] - g1[n]).norm()) <= BOUND[fmt] * float(g0[n].norm()), n
    assert float((dx0 - dx1).norm()) <= BOUND[fmt] * float(dx0.norm())
    assert held1 < 0.6 * held0, (held0, held1)


def test_float32_mode(hific, dev):
    hific.set_compute_dtype(torch.float32)
    net = _generator(hific, dev, n_res=1)
    x, dy = _rand((2, 24, 8, 8), 25).to(dev), _rand((2, 3, 128, 128), 26, scale=1e-2).to(dev)
    y0, dx0, g0, _ = _step(net, x, dy, None)
    y1, dx1, g1, _ = _step(net, x, dy, "int8")
    assert float((y0 - y1).abs().max()) <= 1e-4 * float(y0.abs().max())          # float32 roundings through ten norms
    for n in g0:
        if not (n.endswith(".bias") and n != "conv_block_out.1.bias"):
            assert float((g0[n] - g1[n]).norm()) <= BOUND["int8"] * float(g0[n].norm()), n


def test_side_stream_and_arena_change_nothing(hific, dev):
    from hific_amd import ops, optim
    hific.set_compute_dtype(torch.bfloat16)
    x, dy = _rand((2, 24, 16, 16), 27).to(dev), _rand((2, 3, 256, 256), 28, scale=1e-2).to(dev)
    was, res = ops._SIDE_ON, []
    try:
        for side in (False, True, True):
            net = _generator(hific, dev)
            arena = optim.ParamArena(list(net.parameters()))
            ops.set_side_stream(side)
            ops.set_checkpoint8("int8")
            for _ in range(2):                               # the second backward pass adds
                net(x.clone().requires_grad_()).backward(dy.to(torch.bfloat16))
            torch.cuda.synchronize()
            res.append(arena.flat_grad.clone())
    finally:
        ops.set_side_stream(was)
        ops.set_checkpoint8(None)
    assert torch.isfinite(res[0]).all() and float(res[0].abs().max()) > 0
    assert torch.equal(res[0], res[1]) and torch.equal(res[0], res[2])


def test_captured_training_cycle(hific, dev):
    """The whole G-turn + D-turn cycle with 8-bit checkpoints, captured and replayed: the state that eager cycles leave, bit for bit."""
    from test_gpu_zz_graph import _run
    from hific_amd import ops
    ops.set_exact_index(False)
    ops.set_checkpoint8("int8")
    try:
        eager, graph = _run(dev, False, False), _run(dev, True, False)
        ops.set_checkpoint8(None)
        plain = _run(dev, False, False)
    finally:
        ops.pack_cache.clear(); ops.split_weights.clear()
    bad = [k for k in eager if not torch.equal(eager[k], graph[k])]
    assert not bad, bad
    assert not torch.equal(eager["amort.params"], plain["amort.params"])         # (the option was on)
    assert abs(float(eager["loss_G"]) - float(plain["loss_G"])) < 2e-2 * abs(float(plain["loss_G"]))


# ---- the root-mean-square norm as a module, and a run of the operators together ------------------------------------------------
def test_rms_norm_module_and_pre_norm_blocks(hific, dev):
    """Two pre-norm residual blocks  h += conv(relu-free norm(h))  over planes, through the public modules, against float64 autograd of the
    same formulas.  float32 compute mode: roundings only (2^-24 x a few hundred)."""
    from hific_amd import ops
    from hific_amd.network.layers import HipConv2d
    from hific_amd.normalisation import rms
    hific.set_compute_dtype(torch.float32)
    torch.manual_seed(5)
    C = 24
    norms = [rms.RMSNorm2D_wrap(C).to(dev) for _ in range(3)]
    convs = [HipConv2d(C, C, 3, stride=1, pads=(1, 1, 1, 1)).to(dev) for _ in range(2)]
    for m in norms:
        with torch.no_grad():
            m.gamma.add_(0.2 * torch.randn_like(m.gamma))
    x, dy = _rand((2, C, 9, 11), 31).to(dev), _rand((2, C, 9, 11), 32).to(dev)
    xd = x.clone().requires_grad_()
    y = norms[0](xd)
    h = xd
    for conv, norm in zip(convs, norms[1:]):
        y, h = norm(conv(y), resid=h)
    params = [p for m in norms + convs for p in m.parameters()]
    got = torch.autograd.grad(y, [xd] + params, dy)
    p64 = [p.detach().cpu().double().requires_grad_() for p in params]
    x64 = x.cpu().double().requires_grad_()
    gam, cw = p64[:3], p64[3:]
    nrm = lambda t, g: t * torch.rsqrt((t * t).mean(1, keepdim=True) + 1e-6) * g  # noqa: E731
    t, hh = nrm(x64, gam[0]), x64
    for i in range(2):
        hh = hh + torch.nn.functional.conv2d(t, cw[2 * i], cw[2 * i + 1], padding=1)
        t = nrm(hh, gam[i + 1])
    want = torch.autograd.grad(t, [x64] + p64, dy.cpu().double())
    assert float((y.detach().cpu() - t).abs().max()) <= 1e-4 * float(t.abs().max())
    for a, b in zip(got, want):
        assert float((a.cpu() - b).norm()) <= 1e-4 * float(b.norm())
    with torch.no_grad():
        a8, h8 = norms[1].forward8(x, resid=x, fmt="int8")
        ref, h = norms[1](x, resid=x)
    assert torch.equal(h, h8)
    half = 0.5 * torch.exp2(a8.e.double() - 127).unsqueeze(1)
    assert ((ops.restore8(a8, torch.float32).double() - ref.double()).abs() <= half + 1e-6).all()
    kept = rms.RMSNorm2D(C, checkpoint8="int8").to(dev)
    yk = kept(x.clone().requires_grad_())
    assert yk.grad_fn.saved_tensors[0].dtype == torch.int8
    assert "gamma" in kept.state_dict() and kept.state_dict()["gamma"].shape == (1, C, 1, 1)


def test_gradient_of_the_block_against_the_formula_in_64_bits(hific, dev):
    """norm(conv) in float32 mode with int8 checkpoints: dgamma, dbeta, dx against float64 autograd within what 8 bits cost."""
    from hific_amd import ops
    from hific_amd.network.layers import HipConv2d
    from hific_amd.normalisation import channel
    hific.set_compute_dtype(torch.float32)
    torch.manual_seed(6)
    conv, norm = HipConv2d(16, 32, 3, stride=1, pads=(1, 1, 1, 1)).to(dev), channel.ChannelNorm2D(32, fuse_relu=True).to(dev)
    channel.fuse_bias_grad(conv, norm)
    x, dy = _rand((2, 16, 12, 12), 41).to(dev), _rand((2, 32, 12, 12), 42).to(dev)
    xd = x.clone().requires_grad_()
    y, _ = ops.conv_norm8(xd, ops.checkpoint8(x), conv, norm)
    y.backward(dy)
    w, b, g, be = (p.detach().cpu().double().requires_grad_() for p in (conv.weight, conv.bias, norm.gamma, norm.beta))
    x64 = x.cpu().double().requires_grad_()
    v, _, _ = O8.channel_norm(torch.nn.functional.conv2d(x64, w, b, padding=1), g.flatten(), be.flatten())
    want = torch.autograd.grad(torch.relu(v), (x64, w, g, be), dy.cpu().double())
    for a, c in zip((xd.grad, conv.weight.grad, norm.gamma.grad, norm.beta.grad), want):
        assert float((a.cpu() - c).norm()) <= 3 * 0.016 * float(c.norm())
