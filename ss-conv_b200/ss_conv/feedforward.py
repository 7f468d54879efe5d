"""Gated feed-forward block on the rows of sparse tensors: what follows the convolutions voxel by voxel or point by point.

The reference's networks end in plain linear layers on the rows (LineMOD/model.py); this block widens the rows, multiplies an
activated projection with a second one and narrows them again, in two kernels."""
import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _ext
from .groupnorm import act_code
from .sp_ops.tensor import SparseTensor


def gated_feedforward(features, weight_in, weight_out, bias_in=None, bias_out=None, activation=F.silu, residual=None):
    """(act(x Wg' + bg) * (x Wu' + bu)) Wo' + bo (+ residual): features [N, C], weight_in [2, H, C] (gate, up), weight_out [C_out, H],
    bias_in [2, H], bias_out [C_out], residual [N, C_out], all float32, float16 or bfloat16 and on one device.
    activation: silu, gelu, relu, sigmoid or None.

    Sums are float32; float32 operands count to 24 bits.  In 16 bits the hidden rows and, on the way back, their gradients
    are rounded to the rows' type, so float16 needs hidden values below 65504 and gradients scaled away from zero, as for any
    float16 layer."""
    return _ext.gated_ff(features, weight_in, weight_out, bias_in, bias_out, residual, act_code(activation))


class GatedFeedForward(nn.Module):
    """gated_feedforward with its parameters, on rows or on a SparseTensor of scalars (fields of order l > 0 would not
    stay fields).  Parameters of another floating-point type than the rows are converted."""

    def __init__(self, in_channels, hidden_channels, out_channels=None, activation=F.silu, bias=False):
        super().__init__()
        out_channels = in_channels if out_channels is None else out_channels
        act_code(activation)
        self.in_channels, self.hidden_channels, self.out_channels, self.activation = in_channels, hidden_channels, out_channels, activation
        self.weight_in = nn.Parameter(torch.empty(2, hidden_channels, in_channels))
        self.weight_out = nn.Parameter(torch.empty(out_channels, hidden_channels))
        if bias:
            self.bias_in = nn.Parameter(torch.empty(2, hidden_channels))
            self.bias_out = nn.Parameter(torch.empty(out_channels))
        else:
            self.register_parameter('bias_in', None)
            self.register_parameter('bias_out', None)
        self.reset_parameters()

    def reset_parameters(self):
        for p, fan_in in ((self.weight_in, self.in_channels), (self.bias_in, self.in_channels), (self.weight_out, self.hidden_channels),
                          (self.bias_out, self.hidden_channels)):
            if p is not None:
                nn.init.uniform_(p, -1 / math.sqrt(fan_in), 1 / math.sqrt(fan_in))

    def extra_repr(self):
        return "%d, %d, %d, bias=%s" % (self.in_channels, self.hidden_channels, self.out_channels, self.bias_in is not None)

    def rows(self, x, residual=None):
        p = [t if t is None or t.dtype == x.dtype else t.to(x.dtype) for t in (self.weight_in, self.weight_out, self.bias_in, self.bias_out)]
        return gated_feedforward(x, *p, self.activation, residual)

    def forward(self, input, residual=None):
        """residual: rows to be added to the result (its shape)."""
        if not isinstance(input, SparseTensor):
            return self.rows(input, residual)
        if torch.is_grad_enabled() or residual is not None:
            input.features = self.rows(input.features, residual)
            return input
        # (row by row: a pending row count stays on the device)
        input.features = self.rows(input.raw()[0])
        if input.pending():
            input._rows.post.append(self.rows)
        return input
