"""Layer normalisation of feature rows on the MI355X: `layer_norm` (with autograd) and its module `LayerNorm`.

Beside BatchNorm (`models.blocks`) and InstanceNorm (`blocks.InstNormFn`): the channels of each pixel (row) are normalised by their own
mean and variance.  x is fp32 or bf16, statistics and sums are fp32; weight and bias are fp32 (master parameters) or bf16."""
import torch
import torch.nn as nn
from torch.autograd import Function

from . import _lib, ops
from .ops import UemError, call, ptr, stream

_TYPES = (torch.float32, torch.bfloat16)


def _rows(t, c):
    """(tensor, row stride in elements) of t as rows of c channels; a copy only where no single row stride describes t"""
    if t.is_contiguous():
        return t, c
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= c:
        return t, t.stride(0)
    return t.contiguous(), c


def _flags(x, param_dtype):
    return (_lib.LN_BF16 if x.dtype == torch.bfloat16 else 0) | (_lib.LN_PARAM_BF16 if param_dtype == torch.bfloat16 else 0)


def _param_dtype(weight, bias):
    return weight.dtype if weight is not None else bias.dtype if bias is not None else None


def _forward(x, weight, bias, eps, save):
    c = x.shape[-1]
    rows = x.numel() // c
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    stats = torch.empty((2, rows), device=x.device, dtype=torch.float32) if save else None
    if rows:
        x, ld = _rows(x, c)
        mean = ptr(stats)
        with ops.on_device_of(x):
            call("uem_layernorm_fwd", ptr(x), ld, ptr(weight), ptr(bias), ptr(y), mean, mean + 4 * rows if save else None, rows, c, eps,
                 _flags(x, _param_dtype(weight, bias)), stream())
    return y, stats


class _LayerNormFn(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.param_dtype = _param_dtype(weight, bias)
        return y

    @staticmethod
    def backward(ctx, dy):
        ops.no_second_derivative("layer_norm")
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        c = x.shape[-1]
        rows = x.numel() // c
        dev = x.device
        dx = torch.empty(x.shape, device=dev, dtype=x.dtype)
        dw = torch.empty(c, device=dev, dtype=ctx.param_dtype) if need_w else None
        db = torch.empty(c, device=dev, dtype=ctx.param_dtype) if need_b else None
        if rows == 0:
            return dx, None if dw is None else dw.zero_(), None if db is None else db.zero_(), None
        xr, x_ld = _rows(x, c)
        dyr, dy_ld = _rows(dy, c)
        ws = None
        if need_w or need_b:
            ws = torch.empty(_lib.load().uem_layernorm_workspace_floats(rows, c), device=dev, dtype=torch.float32)
        mean = ptr(stats)
        with ops.on_device_of(x):
            call("uem_layernorm_bwd", ptr(xr), x_ld, ptr(dyr), dy_ld, ptr(weight), mean, mean + 4 * rows, ptr(dx), ptr(dw), ptr(db), ptr(ws),
                 rows, c, _flags(x, ctx.param_dtype), stream())
        return dx if need_x else None, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the LAST dimension of x (any leading dimensions, any of them zero).

    x: fp32 or bf16, on the device; y has its type.  weight, bias: (channels,) of fp32 or bf16 (both of one type), or None.  Gradients of
    all three; their own gradients are not offered.  The feature maps a `Deeplabv2` returns are logical NCHW: `LayerNorm(c, channel_dim=1)`
    normalises their channels without a copy."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _TYPES:
        raise UemError(f"layer_norm: x must be a float32 or bfloat16 tensor, got {getattr(x, 'dtype', type(x).__name__)}")
    ops.need_gpu(x, weight, bias)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise UemError(f"layer_norm: x needs a last dimension of at least one channel, got shape {tuple(x.shape)}")
    if not 0.0 <= eps < float("inf"):
        raise UemError(f"layer_norm: eps must be finite and not negative, got {eps}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != x.shape[-1:] or p.dtype not in _TYPES or not p.is_contiguous() or p.device != x.device:
            raise UemError(f"layer_norm: {name} must be a contiguous float32 or bfloat16 vector of {x.shape[-1]} channels on {x.device}, "
                           f"got {p.dtype} {tuple(p.shape)} strides {p.stride()} on {p.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise UemError(f"layer_norm: weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        return _LayerNormFn.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps), False)[0]


class LayerNorm(nn.Module):
    """`layer_norm` with its parameters.  channel_dim: -1 (rows of channels, NHWC maps) or 1 (logical NCHW maps; channels_last memory is
    used as it is, anything else is copied once)."""

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
