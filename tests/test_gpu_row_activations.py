"""The row operators' activations, value by value over the whole range of their arguments.

A feed-forward block whose weights into the hidden units are zero and whose way out picks single units is the activation of its biases:
y[:, j] = act(b_in[0, j]), and the gradient of b_in[0, j] is the slope there, once for each row."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
ARGUMENTS = [-5.0, -30.0, -42.5, -43.5, -50.0, -87.0, -100.0, -1e4, -1e16, -1e20, -1e30, -3.4028234663852886e+38, 0.0, 3.0, 40.0, 1e4]


def arguments(dtype):
    """The values above as numbers of the type, the lowest one of the type in the place of those below it."""
    low = torch.finfo(dtype).min
    return torch.tensor([max(v, low) for v in ARGUMENTS], dtype=torch.float64).to(dtype)


def one_by_one(z, act, n, device):
    """(values, slopes) of the operator at z, each over n rows."""
    from ss_conv.feedforward import gated_feedforward
    k = z.numel()
    x = torch.ones(n, 8, dtype=z.dtype, device=device)
    b_in = torch.stack([z, torch.ones_like(z)]).to(device).requires_grad_(True)
    y = gated_feedforward(x, torch.zeros(2, k, 8, dtype=z.dtype, device=device), torch.eye(k, dtype=z.dtype, device=device), b_in, activation=act)
    g, = torch.autograd.grad(y, [b_in], torch.ones_like(y))
    return y.detach(), g[0]


def definition(z, act):
    z = z.double().requires_grad_(True)
    v = act(z)
    return v.detach(), torch.autograd.grad(v.sum(), [z])[0]


def room(z, want, dtype):
    """The exponent z log2(e) is off by half a step, the result by |z| 2^-24 of itself (up to twice that with the rounding of log2(e)), the
    other operations by a few steps; below 2^-100 planes of float32 and numbers near the smallest of a type lose bits."""
    z, want = z.double().abs().clamp(max=200), want.abs()
    least = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -100
    return want * ((z + 8) * 2.0 ** -23 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)) + least


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 8, 300])
@pytest.mark.parametrize("act", [F.silu, torch.sigmoid], ids=["silu", "sigmoid"])
def test_sigmoids_of_far_arguments(cuda, dtype, n, act):
    """Few rows and tiles: a gate switched off by a large negative bias contributes nothing."""
    z = arguments(dtype)
    value, slope = one_by_one(z, act, n, cuda)
    want, want_slope = definition(z, act)
    far = (value.double().cpu() - want).abs()
    assert bool((far <= room(z, want, dtype)).all()), (far, want)
    # (slopes: s and z s (1 - s) are added, of at most 1 + |z| times the sigmoid; a sum of n of them is off by n steps more, in 16 bits by
    # its own rounding)
    amount = n * torch.sigmoid(z.double()) * (1 + z.double().abs().clamp(max=200))
    far = (slope.double().cpu() - n * want_slope).abs()
    spare = n * room(z, amount / n, dtype) + amount * n * 2.0 ** -24 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * amount)
    assert bool((far <= spare).all()), (far, want_slope)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_with_a_channel_switched_off(cuda, dtype):
    """A bias of the lowest value: the channel's result and its share of all gradients are zero."""
    from ss_conv.groupnorm import group_norm
    g = torch.Generator().manual_seed(0)
    off = torch.tensor([0, 300, 700], dtype=torch.int32, device=cuda)
    x = torch.randn(700, 16, generator=g).to(dtype).to(cuda).requires_grad_(True)
    b = torch.zeros(16, device=cuda)
    b[[1, 6]] = torch.tensor([torch.finfo(torch.float32).min, -1e30], device=cuda)
    b.requires_grad_(True)
    y = group_norm(x, off, [(16, 0)], 4, None, b, activation=F.silu)
    gx, gb = torch.autograd.grad(y, [x, b], torch.ones_like(y))
    assert not y[:, [1, 6]].any() and not gb[[1, 6]].any() and torch.isfinite(gx).all() and gx.any()
    keep = [c for c in range(16) if c not in (1, 6)]
    # Two sigmoids share a reciprocal, 1 / d0 = d1 / (d0 d1): the neighbour's d1 is another one here.  The product, the reciprocal (a step where it
    # is approximate) and the product with d1 are rounded, half a step each, and so is the argument times the sigmoid: 5 * 2^-24 of the
    # result in either call, and a step of 16 bits between numbers that fall to different sides.
    want = group_norm(x, off, [(16, 0)], 4, activation=F.silu)[:, keep]
    step = 10 * 2.0 ** -24 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps)
    assert bool(((y[:, keep].double() - want.double()).abs() <= step * want.double().abs()).all())


@pytest.mark.parametrize("n", [1, 300])
@pytest.mark.parametrize("act", [F.silu, torch.sigmoid], ids=["silu", "sigmoid"])
def test_float32_sigmoids_to_a_few_steps(cuda, n, act):
    """From -80 to 80 the exponential is off by two steps of 2^-23 at most; what it is multiplied with to take the exponent to base two,
    the one, the shared product, its reciprocal and the two products behind it are rounded, half a step each: eleven halves, sixteen allowed; the
    slope has two more operations, one of them a sum of terms of the same sign beyond |z| = 2."""
    z = torch.linspace(-70, 80, 1023)
    z = z[z.abs() > 2]
    value, slope = one_by_one(z, act, n, cuda)
    want, want_slope = definition(z, act)
    most = ((value.double().cpu() - want).abs() / want.abs()).max().item()
    assert most < 16 * 2.0 ** -24, most
    # (1 - s of a positive argument is a difference: off by half a step of one)
    amount = want_slope.abs() + (z > 0) * (1 + z.double().abs())
    most = ((slope.double().cpu() / n - want_slope).abs() / amount).max().item()
    assert most < (20 + n / 8) * 2.0 ** -24, most
