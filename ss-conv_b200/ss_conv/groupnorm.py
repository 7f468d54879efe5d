"""Group normalisation of sparse rows with the gated activation behind it.

The reference has batch norm only (SS_Conv_lib/ss_conv/batchnorm.py:13-136), whose statistics mix the samples of a batch;
here every sample has its own, so a row's result does not depend on what else is in the batch (but for the order of sums), and training and
inference compute the same.  Scalars are centred and scaled, fields of order l > 0 are scaled by the mean of
their squared norm, which keeps the layer equivariant."""
import functools
import itertools
import weakref

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _ext
from .activation import _act_code


def act_code(fn):
    """0 identity, 1 relu, 2 sigmoid, 3 silu, 4 gelu; ValueError for anything else."""
    code = _act_code(fn)
    if code is None and (fn is F.silu or isinstance(fn, nn.SiLU)):
        code = 3
    if code is None and (fn is F.gelu or (isinstance(fn, nn.GELU) and fn.approximate == "none")):
        code = 4
    if code is None:
        raise ValueError("the activation must be None, relu, sigmoid, silu or gelu (got %r)" % (fn,))
    return code


class _Layout(object):
    """Channel tables of rows Rs in `groups` groups for each entry; gated: the last entry's scalars are the gates of
    the fields of order l > 0 (as SS_Conv lays them out)."""

    def __init__(self, Rs, groups, gated, scalar_act):
        fields = [l for m, l in Rs for _ in range(m)]
        dims = [2 * l + 1 for l in fields]
        first = list(itertools.accumulate(dims, initial=0))[:-1]
        self.c, self.n_field, self.n_scalar = sum(dims), len(fields), fields.count(0)
        self.n_gate = sum(1 for l in fields if l > 0) if gated else 0
        if gated and (not Rs or Rs[-1][1] != 0 or Rs[-1][0] != self.n_gate):
            raise ValueError("the last entry of Rs must hold one gate scalar for each of the %d fields of order l > 0 (got %s)"
                             % (self.n_gate, Rs[-1:]))
        self.c_out = self.c - self.n_gate
        slots, slot = [], 0
        for l in fields:
            slots.append(slot if l == 0 else -1)
            slot += l == 0
        group_of_field, group_first, group_len, copies = [], [], [], []
        f = 0
        for m, l in Rs:
            if m % groups:
                raise ValueError("%d copies of order %d do not divide into %d groups" % (m, l, groups))
            for g in range(groups if m else 0):
                group_first.append(first[f])
                group_len.append(m // groups * (2 * l + 1))
                copies.append(m // groups)
                group_of_field += [len(copies) - 1] * (m // groups)
                f += m // groups
        self.n_group = len(copies)
        gates, gate_field = [], []
        for i, l in enumerate(fields):
            if gated and first[i] >= self.c_out:
                break
            if l == 0:
                gates += [-1 if scalar_act else -2]
            else:
                gates += [len(gate_field) if gated else -2] * (2 * l + 1)
                if gated:
                    gate_field.append(i)
        spread = lambda v: [x for x, d in zip(v, dims) for _ in range(d)]  # noqa: E731
        self.rows = (spread(group_of_field) + spread(range(self.n_field)) + spread(slots) + gates + first + dims + slots
                     + gate_field + group_first + group_len + copies)
        self.sizes = (self.c, self.n_field, self.n_scalar, self.n_group, self.n_gate)
        self.tables = {}

    def table(self, device):
        kept = self.tables.get(device)
        if kept is None:
            if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the channel tables of a group norm are uploaded by its first call, which cannot be inside a "
                                   "recording: call it once before")
            with torch.inference_mode(False):       # (it serves training passes as well)
                kept = self.tables[device] = torch.tensor(self.rows, dtype=torch.int32).to(device)
        return kept


# (for good: a recorded graph and a kernel on another stream hold the address of a layout's table and no reference.  At most 90 KB each.)
@functools.lru_cache(maxsize=None)
def _layout(Rs, groups, gated, scalar_act):
    if not Rs or groups < 1 or any(m < 0 or l < 0 for m, l in Rs) or sum(m for m, _ in Rs) == 0:
        raise ValueError("Rs must be [(copies, order), ...] and the number of groups positive (got %s, %s)" % (list(Rs), groups))
    return _Layout(Rs, groups, gated, scalar_act)


@functools.lru_cache(maxsize=256)
def _plan(Rs, groups, activation):
    """(channel tables, activation codes) of group_norm's arguments."""
    scalar, gate = activation if isinstance(activation, tuple) else (activation, activation)
    gated = gate is not None and any(l > 0 and m > 0 for m, l in Rs)
    codes = (act_code(scalar), act_code(gate) if gated else 0)
    return _layout(Rs, int(groups), gated, codes[0] != 0), codes


def group_norm(features, offsets, Rs, num_groups=1, weight=None, bias=None, eps=1e-5, activation=None):
    """act(norm(features)): features [N, C] float32 / float16 / bfloat16 of fields Rs = [(copies, order), ...], the samples one
    behind the other, offsets [samples + 1] int32 on the device (ascending; samples may be empty).

    The copies of every entry of Rs are split into num_groups groups, normalised over the rows of a sample and the copies of
    the group.  weight [fields] and bias [scalars] as in BatchNorm.  activation: one callable, or (scalar, gate) as in
    Activation; with a gate and fields of order l > 0 the last entry of Rs holds one gate scalar for each of them, and
    the result has the channels before it.  relu, sigmoid, silu, gelu or None.  Statistics and parameters are float32, the
    result has the type of the rows; rows of no sample (outside the offsets) come out as zeros."""
    if not eps > 0:
        raise ValueError("eps must be positive (got %r)" % (eps,))
    layout, codes = _plan(tuple(map(tuple, Rs)), num_groups, activation)
    return _ext.group_norm(features, offsets, layout, weight, bias, eps, codes)


class GroupNorm(nn.Module):
    """group_norm of a SparseTensor's rows, each sample by itself (`weight` [fields], `bias` [scalars]); takes BatchNorm's place
    in SS_Conv(norm_groups=...)."""

    def __init__(self, Rs, num_groups=1, eps=1e-5, affine=True, activation=None):
        super().__init__()
        self.Rs, self.num_groups, self.eps, self.affine, self.activation = [(int(m), int(l)) for m, l in Rs], int(num_groups), eps, affine, activation
        layout = _plan(tuple(self.Rs), self.num_groups, activation)[0]
        if affine:
            self.weight = nn.Parameter(torch.ones(layout.n_field))
            self.bias = nn.Parameter(torch.zeros(layout.n_scalar))
        else:
            self.register_parameter('weight', None)
            self.register_parameter('bias', None)

    def __repr__(self):
        return "{} (Rs={}, num_groups={}, eps={})".format(self.__class__.__name__, self.Rs, self.num_groups, self.eps)

    def rows(self, features, offsets):
        return group_norm(features, offsets, self.Rs, self.num_groups, self.weight, self.bias, self.eps, self.activation)

    @staticmethod
    def apply_rows(input, rows, parameters):
        """input (a SparseTensor) with rows(features, offsets) in the place of its features; parameters: those that `rows` uses."""
        if torch.is_grad_enabled() and (input.raw()[0].requires_grad or any(p.requires_grad for p in parameters)):
            input.features = rows(input.features, input.get_offsets())
            return input
        # (nothing to record: a pending row count stays on the device)
        input.features = rows(input.raw()[0], input.get_offsets())
        if input.pending():
            whose = weakref.ref(input)      # (called by the tensor itself; a cycle would keep its rows until the collector comes)
            input._rows.post.append(lambda f: rows(f, whose().get_offsets()))
        return input

    def norm_and_gate(self, input, act):
        """act(self(input)) in one operator where the activation is the library's (an Activation that fuses, without biases), else None."""
        if self.activation is not None or not (input.raw()[0].is_cuda and act.fusable_gate()):
            return None
        gated = act.gate_act is not None
        layout = _layout(tuple(self.Rs), self.num_groups, gated, act.scalar_act is not None)
        if act.c_in() != layout.c or act.c_out() != layout.c_out:
            return None
        codes = act._codes()

        def rows(f, offsets):
            out = f.dtype
            if out == torch.float32 and not torch.is_grad_enabled():
                out = _ext._stored_type(f.shape[0], layout.c, layout.c_out, layout.c_out, _ext.get_feature_storage()) or out
            return _ext.group_norm(f, offsets, layout, self.weight, self.bias, self.eps, codes, out)

        return self.apply_rows(input, rows, self.parameters())

    def forward(self, input):
        return self.apply_rows(input, self.rows, self.parameters())
