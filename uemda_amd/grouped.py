"""Products of feature rows with the weight of the group (class, domain, expert) each row belongs to, on the MI355X: `grouped_linear` (with
autograd) and its module `GroupedLinear`.

Beside the pointwise convolutions (`ops.conv2d`, `ops_bf16.conv2d`), whose one weight all rows share.  The rows come sorted by group; how
many each group has is known on the device only and never read on the host, so a step with a new partition replays from a captured graph."""
import math

import torch
import torch.nn as nn

from . import _lib
from .ops import UemError


def grouped_linear(x, weight, offsets, bias=None):
    """y[r] = weight[g] @ x[r] + bias[g] for the rows offsets[g] <= r < offsets[g + 1] of each group g.

    x: (rows, in) fp32 or bf16, sorted by group.  weight: (groups, out, in) of x's type, or fp32 master weights under bf16 rows (rounded to
    bf16 for the product, their gradient comes back in fp32).  bias: (groups, out) fp32 or bf16, or None.  offsets: (groups + 1,) int32 or
    int64 on the device, not decreasing; it is not read on the host: an entry below an earlier one counts as that one, entries beyond the
    rows as the number of rows.  Rows in front of offsets[0] and behind offsets[-1] belong to no group: y is zero there, as their gradient
    is, and what they hold (even NaN) reaches no weight's gradient.  Sums run in 32 bits and in a fixed order.
    Refused: 2^30 rows or 2^16 groups and more, more than 2^20 channels, more tiles than a launch holds (some ten million)."""
    return _lib.host().grouped_linear(x, weight, offsets, bias)


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
