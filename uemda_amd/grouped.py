"""Products of feature rows with the weight of the group (class, domain, expert) each row belongs to, on the MI355X: `grouped_linear` (with
autograd) and its module `GroupedLinear`.

Beside the pointwise convolutions (`ops.conv2d`, `ops_bf16.conv2d`), whose one weight all rows share.  The rows come sorted by group; how
many each group has is known on the device only and never read on the host, so a step with a new partition replays from a captured graph."""
import math

import torch
import torch.nn as nn
from torch.autograd import Function

from . import _lib, ops
from .ops import UemError, call, ptr, stream

_TYPES = (torch.float32, torch.bfloat16)
_MOST_LD = 2 ** 21                                 # elements between rows that the kernels address


def _operand(t):
    """(tensor, row stride in elements) of 2-d t as rows that begin on 16-byte boundaries: t itself, or a copy with zeros behind its rows"""
    rows, cols = t.shape
    per = 16 // t.element_size()
    if cols > 1 and t.stride(1) != 1 or rows > 1 and not cols <= t.stride(0) <= _MOST_LD:
        t = t.contiguous()
    ld = t.stride(0) if rows > 1 else cols
    if cols % per == 0 and ld % per == 0 and t.data_ptr() % 16 == 0:
        return t, ld
    out_ld = -(-cols // per) * per
    out = torch.empty((rows, out_ld), device=t.device, dtype=t.dtype)
    call("uem_grouped_pad", ptr(t), ld, ptr(out), out_ld, cols, rows, _lib.GROUPED_BF16 if t.dtype == torch.bfloat16 else 0, stream())
    return out, out_ld


def _flags(x, offsets):
    return (_lib.GROUPED_BF16 if x.dtype == torch.bfloat16 else 0) | (_lib.GROUPED_OFFSETS_64 if offsets.dtype == torch.int64 else 0)


def _forward(x, weight, offsets, bias):
    """y and the operands as the kernels read them"""
    T, K = x.shape
    G, N, _ = weight.shape
    y = torch.empty((T, N), device=x.device, dtype=x.dtype)
    if T == 0:
        return y, x, weight.view(G * N, K)
    with ops.on_device_of(x):
        w = weight.reshape(G * N, K)
        if w.dtype != x.dtype:                                     # fp32 master weights under bf16 rows
            wb = torch.empty((G * N, K), device=x.device, dtype=torch.bfloat16)
            call("uem_cast_f32_bf16", ptr(w), ptr(wb), w.numel(), stream())
            w = wb
        xo, x_ld = _operand(x)
        wo, w_ld = _operand(w)
        flags = _flags(x, offsets) | (_lib.GROUPED_BIAS_BF16 if bias is not None and bias.dtype == torch.bfloat16 else 0)
        call("uem_grouped_fwd", ptr(xo), x_ld, ptr(wo), w_ld, ptr(bias), ptr(y), ptr(offsets), T, G, K, N, flags, stream())
    return y, xo, wo


class _GroupedLinearFn(Function):
    @staticmethod
    def forward(ctx, x, weight, offsets, bias):
        y, xo, wo = _forward(x, weight, offsets, bias)
        ctx.save_for_backward(xo, wo, offsets)
        ctx.sizes = (x.shape[0], weight.shape[0], x.shape[1], weight.shape[1])
        ctx.dtypes = (weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        ops.no_second_derivative("grouped_linear")
        xo, wo, offsets = ctx.saved_tensors
        T, G, K, N = ctx.sizes
        w_dtype, b_dtype = ctx.dtypes
        need_x, need_w, _, need_b = ctx.needs_input_grad
        dev = xo.device
        dx = torch.empty((T, K), device=dev, dtype=xo.dtype) if need_x else None
        dw = torch.empty((G, N, K), device=dev, dtype=w_dtype) if need_w or need_b else None      # db falls off dw's products
        db = torch.empty((G, N), device=dev, dtype=b_dtype) if need_b else None
        if T == 0:
            return dx, dw.zero_() if need_w else None, None, None if db is None else db.zero_()
        flags = _flags(xo, offsets)
        with ops.on_device_of(xo):
            dyo, dy_ld = _operand(dy)
            if need_x:
                call("uem_grouped_dgrad", ptr(dyo), dy_ld, ptr(wo), wo.stride(0) if wo.shape[0] > 1 else wo.shape[1], ptr(dx), ptr(offsets), T, G, K, N,
                     flags, stream())
            if need_w or need_b:
                ws = torch.empty(_lib.load().uem_grouped_wgrad_workspace_floats(T, G, K, N), device=dev, dtype=torch.float32)
                call("uem_grouped_wgrad", ptr(dyo), dy_ld, ptr(xo), xo.stride(0) if T > 1 else xo.shape[1], ptr(dw), ptr(db), ptr(ws), ptr(offsets),
                     T, G, K, N, flags | (_lib.GROUPED_OUT_F32 if w_dtype == torch.float32 else 0)
                     | (_lib.GROUPED_BIAS_BF16 if b_dtype == torch.bfloat16 else 0), stream())
        return dx, dw if need_w else None, None, db


def grouped_linear(x, weight, offsets, bias=None):
    """y[r] = weight[g] @ x[r] + bias[g] for the rows offsets[g] <= r < offsets[g + 1] of each group g.

    x: (rows, in) fp32 or bf16, sorted by group.  weight: (groups, out, in) of x's type, or fp32 master weights under bf16 rows (rounded to
    bf16 for the product, their gradient comes back in fp32).  bias: (groups, out) fp32 or bf16, or None.  offsets: (groups + 1,) int32 or
    int64 on the device, not decreasing; it is not read on the host: an entry below an earlier one counts as that one, entries beyond the
    rows as the number of rows.  Rows in front of offsets[0] and behind offsets[-1] belong to no group: y is zero there, as their gradient
    is, and what they hold (even NaN) reaches no weight's gradient.  Sums run in 32 bits and in a fixed order."""
    for name, t in (("x", x), ("weight", weight), ("offsets", offsets)):
        if not isinstance(t, torch.Tensor):
            raise UemError(f"grouped_linear: {name} must be a tensor, got {type(t).__name__}")
    if x.dim() != 2 or weight.dim() != 3 or weight.shape[2] != x.shape[1] or 0 in weight.shape:
        raise UemError(f"grouped_linear: expected x (rows, in) and weight (groups, out, in), none of groups, out, in zero; got {tuple(x.shape)} and {tuple(weight.shape)}")
    if x.dtype not in _TYPES or not (weight.dtype == x.dtype or (weight.dtype == torch.float32 and x.dtype == torch.bfloat16)):
        raise UemError(f"grouped_linear: x and weight must be float32, bfloat16, or bfloat16 rows with float32 weights; got {x.dtype} and {weight.dtype}")
    G, N, K = weight.shape
    if offsets.shape != (G + 1,) or offsets.dtype not in (torch.int32, torch.int64):
        raise UemError(f"grouped_linear: offsets must be int32 or int64 of {G + 1} entries, got {offsets.dtype} {tuple(offsets.shape)}")
    if bias is not None and (bias.shape != (G, N) or bias.dtype not in _TYPES):
        raise UemError(f"grouped_linear: bias must be float32 or bfloat16 of shape {(G, N)}, got {bias.dtype} {tuple(bias.shape)}")
    ops.need_gpu(x, weight, offsets, bias)
    for name, t in (("weight", weight), ("offsets", offsets), ("bias", bias)):
        if t is not None and t.device != x.device:
            raise UemError(f"grouped_linear: {name} is on {t.device}, x on {x.device}")
    if x.shape[0] >= 2 ** 30 or G >= 2 ** 16 or max(K, N) > 2 ** 20:
        raise UemError(f"grouped_linear: fewer than 2^30 rows and 2^16 groups and at most 2^20 channels, got {x.shape[0]}, {G}, {max(K, N)}")
    offsets = offsets.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _GroupedLinearFn.apply(x, weight, offsets, None if bias is None else bias.contiguous())
    return _forward(x, weight, offsets, None if bias is None else bias.contiguous())[0]


class GroupedLinear(nn.Module):
    """`grouped_linear` with its parameters, one (out, in) weight and (out,) bias a group, initialised as `nn.Linear`."""

    def __init__(self, groups, in_features, out_features, bias=True):
        super().__init__()
        if min(int(groups), int(in_features), int(out_features)) < 1:
            raise UemError(f"GroupedLinear: groups, in_features and out_features must be positive, got {groups}, {in_features}, {out_features}")
        self.groups, self.in_features, self.out_features = int(groups), int(in_features), int(out_features)
        bound = 1 / math.sqrt(self.in_features)
        self.weight = nn.Parameter(torch.empty(self.groups, self.out_features, self.in_features).uniform_(-bound, bound))
        self.bias = nn.Parameter(torch.empty(self.groups, self.out_features).uniform_(-bound, bound)) if bias else None

    def forward(self, x, offsets):
        return grouped_linear(x, self.weight, offsets, self.bias)

    def extra_repr(self):
        return f"{self.groups}, {self.in_features}, {self.out_features}, bias={self.bias is not None}"
