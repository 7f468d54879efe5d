"""Gated feed-forward block on the rows of sparse tensors: what follows the convolutions voxel by voxel or point by point.

The reference's networks end in plain linear layers on the rows (LineMOD/model.py); this block widens the rows, multiplies an
activated projection with a second one and narrows them again, in two kernels."""
import math

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _ext
from .groupnorm import act_code
from .sp_ops.tensor import SparseTensor


class _GatedFeedForwardFn(torch.autograd.Function):
    """Saves its arguments; gate and up are computed again on the way back."""

    @staticmethod
    def forward(ctx, x, w_in, w_out, b_in, b_out, residual, act):
        ctx.save_for_backward(x, w_in, w_out, b_in)
        ctx.act = act
        return _ext.gated_ff_forward(x, w_in, w_out, b_in, b_out, residual, act)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, w_in, w_out, b_in = ctx.saved_tensors
        need = ctx.needs_input_grad
        gy = gy.contiguous()
        grads = _ext.gated_ff_backward(x, gy, w_in, w_out, b_in, ctx.act, need[:5]) if any(need[:5]) else [None] * 5
        return (*grads, gy if need[5] else None, None)


def gated_feedforward(features, weight_in, weight_out, bias_in=None, bias_out=None, activation=F.silu, residual=None):
    """(act(x Wg' + bg) * (x Wu' + bu)) Wo' + bo (+ residual): features [N, C], weight_in [2, H, C] (gate, up), weight_out [C_out, H],
    bias_in [2, H], bias_out [C_out], residual [N, C_out], all float32, float16 or bfloat16 and on one device.
    activation: silu, gelu, relu, sigmoid or None.

    Sums are float32; float32 operands count to 24 bits.  In 16 bits the hidden rows and, on the way back, their gradients
    are rounded to the rows' type, so float16 needs hidden values below 65504 and gradients scaled away from zero, as for any
    float16 layer."""
    x = features
    if not x.is_cuda:
        raise RuntimeError("ssconv_b200 runs on CUDA tensors only (got a %s tensor)" % x.device.type)
    if x.dtype not in _ext.ROW_TYPES:
        raise TypeError("features must be float32, float16 or bfloat16 (got %s)" % x.dtype)
    if x.dim() != 2 or weight_in.dim() != 3 or weight_out.dim() != 2:
        raise ValueError("features must be [N, C], weight_in [2, H, C] and weight_out [C_out, H] (got %s, %s, %s)"
                         % (tuple(x.shape), tuple(weight_in.shape), tuple(weight_out.shape)))
    hidden, c_out = weight_in.shape[1], weight_out.shape[0]
    wanted = ((weight_in, "weight_in", (2, hidden, x.shape[1])), (weight_out, "weight_out", (c_out, hidden)), (bias_in, "bias_in", (2, hidden)),
              (bias_out, "bias_out", (c_out,)), (residual, "residual", (x.shape[0], c_out)))
    for t, name, shape in wanted:
        if t is not None and (t.shape != shape or t.dtype != x.dtype or t.device != x.device):
            raise ValueError("%s must be %s %s on %s (got %s %s on %s)" % (name, x.dtype, shape, x.device, t.dtype, tuple(t.shape), t.device))
    if min(x.shape[1], hidden, c_out) < 1 or max(x.shape[1], hidden, c_out) > 65536:
        raise ValueError("widths must be 1 to 65536 (got %d, %d, %d)" % (x.shape[1], hidden, c_out))
    args = [t if t is None or t.is_contiguous() else t.contiguous() for t in (x, weight_in, weight_out, bias_in, bias_out, residual)]
    act = act_code(activation)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        return _GatedFeedForwardFn.apply(*args, act)
    return _ext.gated_ff_forward(*args, act)


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
