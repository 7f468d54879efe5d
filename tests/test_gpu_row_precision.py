"""How far the row operators are off, value by value: rooms of a few half steps of what each value is made of, in which no missing term, wrong
gate or forgotten last row fits (test_host_row_references.py shows that of zeros)."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

import row_references as R
from test_gpu_groupnorm import CASES, GATE

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
