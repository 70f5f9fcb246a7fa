"""Layer normalisation of feature rows on the MI355X: `layer_norm` (with autograd) and its module `LayerNorm`.

Beside BatchNorm (`models.blocks`) and InstanceNorm (`blocks.InstNormFn`): the channels of each pixel (row) are normalised by their own
mean and variance.  x is fp32 or bf16, statistics and sums are fp32; weight and bias are fp32 (master parameters) or bf16."""
import torch
import torch.nn as nn

from . import _lib
from .ops import UemError


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the LAST dimension of x (any leading dimensions, any of them zero).

    x: fp32 or bf16, on the device; y has its type.  weight, bias: (channels,) of fp32 or bf16 (both of one type), or None.  Gradients of
    all three; their own gradients and forward-mode derivatives are not offered.  The feature maps a `Deeplabv2` returns are logical NCHW: `LayerNorm(c, channel_dim=1)`
    normalises their channels without a copy."""
    return _lib.host().layer_norm(x, weight, bias, eps)


class LayerNorm(nn.Module):
    """`layer_norm` with its parameters.  channel_dim: -1 (rows of channels, NHWC maps) or 1 (logical NCHW maps; channels_last memory is
    used as it is, anything else is copied once, and that copy is what the backward pass reads)."""

    def __init__(self, channels, eps=1e-5, affine=True, bias=True, channel_dim=-1):
        super().__init__()
        if int(channels) < 1:
            raise UemError(f"LayerNorm: channels must be positive, got {channels}")
        if channel_dim not in (-1, 1):
            raise UemError(f"LayerNorm: channel_dim must be -1 or 1, got {channel_dim}")
        self.channels, self.eps, self.channel_dim = int(channels), float(eps), channel_dim
        self.weight = nn.Parameter(torch.ones(self.channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(self.channels)) if affine and bias else None

    def forward(self, x):
        if self.channel_dim == 1:
            if x.dim() != 4:
                raise UemError(f"LayerNorm(channel_dim=1): expected an (N, C, H, W) map, got shape {tuple(x.shape)}")
            return layer_norm(x.permute(0, 2, 3, 1), self.weight, self.bias, self.eps).permute(0, 3, 1, 2)
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.channels}, eps={self.eps}, affine={self.weight is not None}, channel_dim={self.channel_dim}"
