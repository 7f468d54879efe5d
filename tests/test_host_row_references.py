"""The 64-bit forms that the GPU tests of the row operators go by: the same numbers as torch's own derivatives, and rooms that a result of
zeros does not fit in."""
import pytest
import torch

import row_references as R
from test_gpu_groupnorm import CASES, reference
from test_gpu_feedforward import SIZES
from test_gpu_feedforward import reference as ff_reference
from test_gpu_row_precision import FF_STEPS, NORM_CASES, ff_inputs, ff_room, norm_inputs, norm_room, parts

SMALL = [i for i, c in enumerate(CASES) if sum(c[0]) <= 3000]


@pytest.mark.parametrize("case", SMALL)
def test_norm_by_formulas_and_by_torch(case):
    lengths, Rs, groups, act = CASES[case]
    x, w, b, gy, offsets = norm_inputs(lengths, Rs, act, torch.float32, 300 + case)
    found = R.group_norm(x.double(), offsets, Rs, groups, w.double(), b.double(), 1e-3, act, gy.double())
    leaves = [t.double().requires_grad_(True) for t in (x, w, b)]
    y = reference(leaves[0], offsets, Rs, groups, leaves[1], leaves[2], 1e-3, act)
    grads = torch.autograd.grad(y, leaves, found["gy"])
    for name, a in zip(("y", "x", "weight", "bias"), (y.detach(), *grads)):
        assert ((found[name][0] - a).abs() <= 2.0 ** -44 * (found[name][1] + 1)).all(), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [i for i, c in enumerate(NORM_CASES) if sum(c[0]) <= 60000])
def test_rooms_reject_zeros(case, dtype):
    """Whatever is not all rounding (the gradient of a sample of one row is none): the room is a small part of the result."""
    lengths, Rs, groups, act = NORM_CASES[case]
    x, w, b, gy, offsets = norm_inputs(lengths, Rs, act, dtype, 300 + case)
    found = R.group_norm(x.double(), offsets, Rs, groups, w.double(), b.double(), 1e-3, act, gy.double())
    for name in ("y", "x", "weight", "bias"):
        if name in ("x", "weight") and max(lengths) == 1:
            continue
        want, room = found[name][0], norm_room(found[name], torch.float32 if name in ("weight", "bias") else dtype)
        if name == "x":
            some = torch.cat([torch.full((n,), n > 1) for n in lengths])
            want, room = want[some], room[some]
        if want.numel():
            assert room.norm() < 0.03 * want.norm(), (name, (room.norm() / want.norm()).item())


SMALL_FF = [i for i, s in enumerate(SIZES) if s[0] * s[2] <= 1500000]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", SMALL_FF)
def test_feedforward_by_formulas_and_its_rooms(size, dtype):
    """The formulas' numbers are torch's; zeros do not fit in the rooms; no gate comes so near to ReLU's kink that its slope is open."""
    t, gy = ff_inputs(size, dtype)
    act = SIZES[size][-1]
    t64 = {k: None if v is None else v.double().requires_grad_(True) for k, v in t.items()}
    found = R.feedforward({k: None if v is None else v.detach() for k, v in t64.items()}, act, gy.double())
    y = ff_reference(t64, act)
    names = [k for k in t if t[k] is not None and k != "residual"]
    for name, a in zip(["y"] + names, (y.detach(), *torch.autograd.grad(y, [t64[k] for k in names], gy.double()))):
        value, size_of = found[name][:2]
        assert ((value - a).abs() <= 2.0 ** -44 * (size_of + 1)).all(), name
        for part in parts(value):
            # (one value may be small by chance: what the others around it are)
            assert ff_room(found[name], dtype, part) < 0.05 * max(part(value).norm(), part(size_of).norm() / 8), name
    assert act is not torch.nn.functional.relu or found["kink"] > 4 * FF_STEPS * R.HALF
