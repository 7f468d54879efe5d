"""How far the row operators are off, value by value: rooms of a few half steps of what each value is made of, in which no missing term, wrong
gate or forgotten last row fits (test_host_row_references.py shows that of zeros)."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

import row_references as R
from test_gpu_feedforward import SIZES, inputs
from test_gpu_groupnorm import CASES

pytestmark = pytest.mark.gpu
NORM_CASES = CASES


def norm_inputs(lengths, Rs, act, dtype, seed, c=None):
    """(x, weight, bias, gy, offsets) as the layers in front leave them: channels off centre by a few spreads."""
    g = torch.Generator().manual_seed(seed)
    c = sum(m * (2 * l + 1) for m, l in Rs)
    gate = act[1] if isinstance(act, tuple) else act
    out = c - (sum(m for m, l in Rs if l > 0) if gate is not None else 0)
    x = (torch.randn(sum(lengths), c, generator=g) * 0.7 + 2 * torch.randn(c, generator=g)).to(dtype)
    w = 1 + 0.3 * torch.randn(sum(m for m, _ in Rs), generator=g)
    b = 0.3 * torch.randn(sum(m for m, l in Rs if l == 0), generator=g)
    return x, w, b, torch.randn(x.shape[0], out, generator=g).to(dtype), np.concatenate([[0], np.cumsum(lengths)]).tolist()


# Half steps of float32 that a value may be off by, of the terms it is made of.  Means and mean squares come from chains of running values, whose
# errors shrink as rows are added: over n updates about sqrt(n / 3) roundings that go either way, 0.6 half steps each: 16 for two
# thousand, and as much for the sums of the pieces and what follows (a dozen operations).
STEPS = 32


def norm_room(found, dtype):
    value, terms = found
    room = STEPS * R.HALF * terms
    return room if dtype == torch.float32 else room + torch.finfo(dtype).eps / 2 * value.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def run_norm(cuda, x, w, b, gy, offsets, Rs, groups, eps, act):
    from ss_conv.groupnorm import group_norm
    leaves = [t.to(cuda).requires_grad_(True) for t in (x, w, b)]
    y = group_norm(leaves[0], torch.tensor(offsets, dtype=torch.int32, device=cuda), Rs, groups, leaves[1], leaves[2], eps, act)
    return [y.detach().cpu(), *(g.cpu() for g in torch.autograd.grad(y, leaves, gy.to(y.dtype).to(cuda)))]


def check_norm(cuda, x, w, b, gy, offsets, Rs, groups, eps, act):
    found = R.group_norm(x.double(), offsets, Rs, groups, w.double(), b.double(), eps, act, gy.double())
    got = run_norm(cuda, x, w, b, found["gy"], offsets, Rs, groups, eps, act)
    for name, a in zip(("y", "x", "weight", "bias"), got):
        want, room = found[name][0], norm_room(found[name], a.dtype)
        far = (a.double() - want).abs()
        assert bool((far <= room).all()), (name, (far / room.clamp(min=1e-300)).max().item(), (far.norm() / want.norm()).item())


OUTLIERS = ["channel", "row", "first piece", "last piece", "huge"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,c,groups", [(4096, 256, 1), (30001, 64, 2), (300, 2048, 1), (5000, 16, 4), (20000, 5, 1)])
@pytest.mark.parametrize("outlier", OUTLIERS)
def test_norm_with_values_far_from_the_rest(cuda, outlier, rows, c, groups, dtype):
    """A channel, a row or a range of rows a thousand spreads away keeps the others' part of the variance.  Values whose squares are beyond
    float32 do not matter, as long as the sum of the squares about the mean is within it: 2^20 squares of 2 * 10^15 are 4 * 10^36 (of 2 * 10^18
    they would be 4 * 10^42, which no float32 holds)."""
    x, w, b, gy, _ = norm_inputs([rows], [(c, 0)], F.silu, torch.float32, 7)
    if outlier == "channel":
        x[:, 0] += 1000
    elif outlier == "row":
        x[0] += 1e4
    elif outlier == "first piece":
        x[:rows // 290 + 1] += 1000
    elif outlier == "last piece":
        x[-rows // 290:] -= 1000
    else:
        x = 1e20 + 1e15 * x
    check_norm(cuda, x.to(dtype), w, b, gy.to(dtype), [0, rows], [(c, 0)], groups, 1e-5, F.silu)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(NORM_CASES)))
def test_norm_value_by_value(cuda, case, dtype):
    """Every value of the result and of all gradients, at the sizes and layouts where they can go wrong."""
    lengths, Rs, groups, act = NORM_CASES[case]
    x, w, b, gy, offsets = norm_inputs(lengths, Rs, act, dtype, 300 + case)
    check_norm(cuda, x, w, b, gy, offsets, Rs, groups, 1e-3, act)


# Half steps of a product's float32 sums: inside tensor memory an addition of sixteen terms may cut off, a step of 2^-23, half of it on average, and
# after sixteen of them the sum goes on in registers, where half a step is lost each time, either way: 16, and as much again for the planes' products that
# are left out, the parts, and the activation.
FF_STEPS = 32


def ff_room(found, dtype, part):
    """For the norm of the errors over a part of a result.  16 bits: half a step of the result, and of the terms rounded before.  Few values may
    add up to twice what many do on average."""
    value, size, rounded, stages = found
    value, size, rounded = part(value), part(size), part(rounded)
    room = stages * FF_STEPS * R.HALF * size.norm()
    half = 0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    return half * value.norm() + (2 if value.numel() < 32 else 1) * (room + half * rounded.norm())


def parts(t):
    """The whole, its first and last columns and rows, eighths of the rows and of the columns."""
    yield lambda v: v
    for i in ((0, 1), (-1, None)):
        yield lambda v, i=i: v[..., i[0]:i[1]]
        if t.dim() > 1:
            yield lambda v, i=i: v[..., i[0]:i[1], :]
    for dim in (-1, -2)[:t.dim()]:
        for k in range(8):
            if t.shape[dim] >= 8:
                yield lambda v, k=k, dim=dim: v.chunk(8, dim)[min(k, len(v.chunk(8, dim)) - 1)]


def ff_inputs(size, dtype):
    n, c, h, o, bias, residual, act = SIZES[size]
    return inputs(n, c, h, o, dtype, bias, residual, 500 + size)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", range(len(SIZES)))
def test_feedforward_part_by_part(cuda, size, dtype):
    from ss_conv.feedforward import gated_feedforward
    t, gy = ff_inputs(size, dtype)
    act = SIZES[size][-1]
    names = [k for k in t if t[k] is not None]
    on = lambda v: None if v is None else v.to(cuda)  # noqa: E731
    dev = {k: None if v is None else on(v).requires_grad_(True) for k, v in t.items()}
    y = gated_feedforward(dev["x"], dev["w_in"], dev["w_out"], dev["b_in"], dev["b_out"], act, dev["residual"])
    got = {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, [dev[k] for k in names], on(gy))))}
    found = R.feedforward({k: None if v is None else on(v).double() for k, v in t.items()}, act, on(gy).double())
    for name in got:
        if name == "residual":
            continue
        want = found[name][0]
        assert got[name].shape == want.shape
        far = got[name].double() - want
        for part in parts(want):
            room = ff_room(found[name], dtype, part)
            assert part(far).norm() <= room, (name, part(far).shape, (part(far).norm() / room).item(), (part(far).norm() / part(want).norm()).item())
