"""RMSNorm2D: root-mean-square norm over the channel dim, beside ChannelNorm2D (no mean, no shift; no counterpart in the reference).

One parameter `gamma` shaped (1, C, 1, 1).  `forward(x, resid)` with a residual adds it first and also returns the sum - the residual
stream of a pre-norm block - in one kernel (csrc/norm8_fwd.hip)."""
import torch
import torch.nn as nn

from .. import ops


def RMSNorm2D_wrap(input_channels, eps=1e-6, checkpoint8=None, **kwargs):
    return RMSNorm2D(input_channels, eps=eps, checkpoint8=checkpoint8)


class RMSNorm2D(nn.Module):
    """gamma * h / sqrt(mean_c h^2 + eps) per position of h [N, C, ...]; `checkpoint8` ("int8" | "e4m3"): the backward pass keeps
    the normalised input in 8 bits."""

    def __init__(self, input_channels, eps=1e-6, checkpoint8=None):
        super().__init__()
        self.eps = eps
        self.input_channels = input_channels
        self.checkpoint8 = checkpoint8
        self.gamma = nn.Parameter(torch.ones(1, input_channels, 1, 1))

    def forward(self, x, resid=None):
        """norm(x), or with `resid` (norm(x + resid), x + resid)."""
        return ops.rms_norm(x, self.gamma, resid=resid, eps=self.eps, fmt=self.checkpoint8)

    def forward8(self, x, resid=None, fmt="e4m3"):
        """forward with its output in 8 bits (ops.Act8); inference only."""
        return ops.rms_norm8(x, self.gamma, resid=resid, eps=self.eps, fmt=fmt)

    def extra_repr(self):
        return f"{self.input_channels}, eps={self.eps}, checkpoint8={self.checkpoint8}"
