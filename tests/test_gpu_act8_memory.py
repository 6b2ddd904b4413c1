"""What a training step holds and what it needs at its peak with 8-bit checkpoints: a backward pass restores one layer's input at a time
or takes a workspace of that order, so the peak falls too, not only what is held between the passes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _measure(net, x, dy):
    """(held after the forward pass, peak of forward and backward) in bytes beyond what was there before.  (The parameters' gradients,
    which outweigh the activations of small planes, lie in an arena.)"""
    torch.cuda.synchronize()
    base = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    y = net(x)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated() - base
    y.backward(dy)
    torch.cuda.synchronize()
    return held, torch.cuda.max_memory_allocated() - base


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_peak_of_the_generators_forward_and_backward_pass(hific, dev, fmt):
    """One bfloat16 tensor of full resolution (60 channels) is a fifth of what the plain pass holds; at the peak its gradient, the next
    one and the restored input live at once: three of them, beside the 8-bit ones (a third of the plain total)."""
    from hific_amd import ops, optim
    from hific_amd.network import generator
    was = ops.get_compute_dtype()
    hific.set_compute_dtype(torch.bfloat16)
    torch.manual_seed(7)
    net = generator.Generator((3, 16, 16), 4, C=24, n_residual_blocks=4).to(dev).train()
    optim.ParamArena(list(net.parameters()))
    x = torch.randn(4, 24, 16, 16, generator=torch.Generator().manual_seed(1)).to(dev)
    dy = torch.randn(4, 3, 256, 256, generator=torch.Generator().manual_seed(2)).to(dev).to(torch.bfloat16)
    res = {}
    try:
        for f in (None, fmt):
            ops.set_checkpoint8(f)
            for _ in range(2):                           # (packed weights and workspaces exist from the first pass on)
                res[f] = _measure(net, x, dy)
    finally:
        ops.set_checkpoint8(None)
        hific.set_compute_dtype(was)
    assert res[fmt][0] < 0.4 * res[None][0], res
    assert res[fmt][1] < 0.8 * res[None][1], res
