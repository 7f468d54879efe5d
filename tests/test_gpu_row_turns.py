"""The feed-forward block at the widest hidden rows, whose rows are taken in turns of a few tiles."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,rows", [(torch.float32, 1100), (torch.bfloat16, 5500)])
def test_turns_of_the_widest_hidden_rows(cuda, dtype, rows):
    """Three turns, the last one no whole tile.  float32: sums leave tensor memory every 256 terms, sixteen additions that may cut off (half a
    step of 2^-23 on average), and go on in registers, 256 additions of half a step that go either way: 2^-20 and 2^-20 of the result's size in each
    of the three products behind one another, 2^-18 in all.  16 bits: hidden rows or gradients, and the result, are rounded: half a step
    each at most, and the sums inside tensor memory add up 4096 times, 2^-12 cut off at most."""
    from ss_conv.feedforward import gated_feedforward
    g = torch.Generator("cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    c, h = 16, 65536
    x, w_in, w_out = r(rows, c).to(dtype), (r(2, h, c) / 4).to(dtype), (r(c, h) / 256).to(dtype)
    b_in, b_out, gy = r(2, h).to(dtype), r(c).to(dtype), r(rows, c).to(dtype)
    leaves = [t.requires_grad_(True) for t in (x, w_in, w_out, b_in, b_out)]
    y = gated_feedforward(*leaves)
    got = [y.detach(), *torch.autograd.grad(y, leaves, gy)]
    want = [torch.empty_like(y, dtype=torch.float64)] + [torch.zeros_like(t, dtype=torch.float64) for t in leaves]
    for lo in range(0, rows, 500):
        part = [t.detach().double() for t in leaves]
        part[0] = part[0][lo:lo + 500]
        part = [t.requires_grad_(True) for t in part]
        hidden = F.silu(F.linear(part[0], part[1][0], part[3][0])) * F.linear(part[0], part[1][1], part[3][1])
        y64 = F.linear(hidden, part[2], part[4])
        grads = torch.autograd.grad(y64, part, gy[lo:lo + 500].double())
        want[0][lo:lo + 500] = y64.detach()
        want[1][lo:lo + 500] = grads[0]
        for a, b in zip(want[2:], grads[1:]):
            a += b
    most = 2.0 ** -18 if dtype == torch.float32 else torch.finfo(dtype).eps + 2.0 ** -12
    for name, a, b in zip(["y", "x", "w_in", "w_out", "b_in", "b_out"], got, want):
        assert ((a.double() - b).norm() / b.norm()).item() < most, name
        if name in ("y", "x"):
            assert ((a[-3:].double() - b[-3:]).norm() / b[-3:].norm()).item() < 2 * most, name
