"""Group norm with the gated activation: forward and gradients against the formula in 64 bits, at the sizes and layouts where
they can go wrong.

Tolerances.  A statistic is the end of a chain of at most a few hundred float32 additions and merges, each off by half a step
(2^-24 relative): CHAIN * 2^-24 with CHAIN = 256.  A result is off by that much of the terms it is made of, and by half a
step of its own type."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
CHAIN = 256 * 2.0 ** -24


def reference(x, offsets, Rs, groups, weight, bias, eps, activation):
    """The definition, sample by sample, on float64 tensors that may ask for gradients."""
    scalar, gate = activation if isinstance(activation, tuple) else (activation, activation)
    n_gate = sum(m for m, l in Rs if l > 0) if gate is not None else 0
    c_out = x.shape[1] - n_gate
    out = [x.new_zeros(offsets[0], c_out)]
    for lo, hi in zip(offsets[:-1], offsets[1:]):
        z, ch, f, s = [], 0, 0, 0
        for m, l in Rs:
            d = 2 * l + 1
            if m == 0:
                continue
            v = x[lo:hi, ch:ch + m * d].reshape(hi - lo, groups, m // groups, d)
            if hi > lo:
                if l == 0:
                    v = v - v.mean((0, 2), keepdim=True)
                v = v / torch.sqrt(v.pow(2).sum(3, keepdim=True).mean((0, 2), keepdim=True) + eps)
            v = v.reshape(hi - lo, m, d)
            if weight is not None:
                v = v * weight[f:f + m, None]
            if l == 0 and bias is not None:
                v = v + bias[s:s + m, None]
            z.append(v)
            ch, f, s = ch + m * d, f + m, s + (m if l == 0 else 0)
        if n_gate:
            gates, used = gate(z.pop()), 0
        rows = []
        layout = [(m, l) for m, l in Rs if m > 0]
        for (m, l), v in zip(layout[:-1] if n_gate else layout, z):
            if l == 0:
                v = scalar(v) if scalar is not None else v
            elif n_gate:
                v, used = v * gates[:, used:used + m], used + m
            rows.append(v.flatten(1))
        out.append(torch.cat(rows, 1))
    out.append(x.new_zeros(x.shape[0] - offsets[-1], c_out))
    return torch.cat(out)


def close(got, want, terms, dtype, what):
    """|got - want| <= CHAIN * terms + half a step of the result."""
    got, want = got.double().cpu(), want.double().cpu()
    room = CHAIN * terms + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal)
    far = ((got - want).abs() - room).max().item() if got.numel() else 0.0
    assert far <= 0, (what, far, (got - want).abs().max().item())


GATE = (torch.relu, torch.sigmoid)
CASES = [
    # lengths, Rs, groups, activation
    ([1], [(4, 0)], 1, None),
    ([1, 1, 1], [(8, 0)], 8, F.silu),                                   # groups of one value: variance zero
    ([5, 0, 1, 300], [(64, 0)], 32, F.silu),
    ([0, 700], [(2, 0), (2, 1), (2, 2), (2, 3), (6, 0)], 1, GATE),
    ([1021, 33], [(9, 0), (3, 1), (3, 2), (6, 0)], 3, GATE),            # 45 channels and gates: one channel at a time
    ([513], [(4, 0), (2, 1)], 2, (F.gelu, None)),
    ([77, 500], [(2047, 0)], 23, F.silu),                               # wide, no multiple of anything
    ([600], [(5, 0), (3, 2)], 1, None),
    ([50, 900], [(7, 0), (1, 1), (2, 3), (3, 0)], 1, GATE),                       # fields of order l > 0 without gates
    ([129, 64], [(3, 1), (3, 0)], 3, (None, torch.sigmoid)),            # no scalars but the gates
    ([2000], [(1, 0)], 1, F.gelu),
    ([40, 60], [(510, 0)], 2, F.relu),
    ([3, 4], [(2048, 0)], 4, None),
    ([900] * 33, [(16, 0)], 4, F.silu),                                 # more samples than lanes
    ([20000, 7], [(24, 0)], 2, torch.sigmoid),
    ([70, 70], [(500, 0), (1, 1), (1, 0)], 1, GATE),                    # wide rows, one gate
    ([9, 30], [(4, 0), (300, 1), (300, 0)], 4, (F.silu, torch.sigmoid)),    # more gates than 256
    ([1] * 700, [(6, 0)], 3, None),
    ([1, 500000], [(40, 0)], 5, F.silu),                                # rings that go round several times
    ([150000, 2, 150001], [(8, 0), (4, 1), (4, 0)], 2, GATE),
    ([3] * 40 + [0] * 40 + [500], [(5, 0), (1, 2), (1, 0)], 1, GATE),   # many pieces to a block, rows of no multiple of anything
    ([9000, 3000], [(80, 0)], 80, F.silu),                              # more groups than lanes, each in many pieces
    ([6000], [(33, 0), (33, 1), (33, 0)], 33, GATE),
    ([2500, 2500], [(5, 0), (5, 1), (5, 0)], 1, GATE),                  # three groups in many pieces
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_group_norm_and_gradients(cuda, case, dtype):
    from ss_conv.groupnorm import group_norm
    lengths, Rs, groups, act = CASES[case]
    g = torch.Generator().manual_seed(100 + case)
    c = sum(m * (2 * l + 1) for m, l in Rs)
    # off centre by a few spreads: the mean and the variance are not what sums of squares would give
    x = (torch.randn(sum(lengths), c, generator=g) * 0.7 + 2 * torch.randn(c, generator=g)).to(dtype)
    w = 1 + 0.3 * torch.randn(sum(m for m, _ in Rs), generator=g)
    b = 0.3 * torch.randn(sum(m for m, l in Rs if l == 0), generator=g)
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    xd, wd, bd = x.to(cuda).requires_grad_(True), w.to(cuda).requires_grad_(True), b.to(cuda).requires_grad_(True)
    y = group_norm(xd, torch.tensor(offsets, dtype=torch.int32, device=cuda), Rs, groups, wd, bd, 1e-3, act)
    x64, w64, b64 = (t.double().requires_grad_(True) for t in (x, w, b))
    y64 = reference(x64, offsets.tolist(), Rs, groups, w64, b64, 1e-3, act)
    assert y.dtype == dtype and y.shape == y64.shape
    # terms: |x| r |w| + |b| with r <= eps^-1/2, times a gate of at most one
    spread = x.double().abs().max() + 1
    r = min(1e-3 ** -0.5, 50.0) if min(lengths) < 3 else 4.0
    size = float(spread * r * w.abs().max() + b.abs().max())
    close(y, y64, size * (1 if act is None else 3), dtype, "result")
    gy = torch.randn(y64.shape, generator=g).to(dtype)
    grads = torch.autograd.grad(y, [xd, wd, bd], gy.to(cuda))
    want = torch.autograd.grad(y64, [x64, w64, b64], gy.double())
    # dx: r (a - s1 - xhat s2), each of them at most |dz| |w| xhat^2; slopes within 1.13; gates add a product for each channel of a field
    top = float(gy.abs().max()) * 1.13 * 7 * float(w.abs().max()) * max(1.0, float(y64.detach().abs().max())) ** 2
    close(grads[0], want[0], 8 * r * r * top * float(spread), dtype, "gx")
    # (a sum over all rows: the chain is longer, the terms add up)
    rows = sum(lengths)
    close(grads[1], want[1], 8 * r * top * float(spread) * max(1, rows ** 0.5), torch.float32, "weight")
    close(grads[2], want[2], 8 * top * max(1, rows ** 0.5), torch.float32, "bias")


def test_group_norm_against_differences(cuda):
    """The gradient against central differences of the operator itself, on float32 rows."""
    from ss_conv.groupnorm import group_norm
    Rs = [(4, 0), (2, 1), (2, 0)]
    g = torch.Generator().manual_seed(3)
    x = torch.randn(60, 12, generator=g).to(cuda)
    offsets = torch.tensor([0, 25, 60], dtype=torch.int32, device=cuda)
    act = (F.silu, torch.sigmoid)
    coef = torch.randn(60, 10, generator=g).to(cuda)
    xr = x.clone().requires_grad_(True)
    (group_norm(xr, offsets, Rs, 2, activation=act) * coef).sum().backward()
    for row, ch in ((0, 0), (24, 5), (25, 9), (59, 11), (40, 3)):
        h = 2.0 ** -6
        d = torch.zeros_like(x)
        d[row, ch] = h
        up, down = (((group_norm(x + s * d, offsets, Rs, 2, activation=act) * coef).double()).sum() for s in (1, -1))
        # third derivatives of order one times h^2 / 6, and rounding of 600 terms over 2 h
        assert abs(((up - down) / (2 * h)).item() - xr.grad[row, ch].item()) < 5e-3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_far_from_zero_and_rows_of_no_sample(cuda, dtype):
    """A mean a thousand spreads from zero keeps its variance; rows outside the offsets are zeros, offsets beyond the rows are cut."""
    from ss_conv.groupnorm import group_norm
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(4000, 32, generator=g) + (1000 if dtype == torch.float32 else 4)).to(dtype)
    off = [100, 1000, 1000, 3900]
    y = group_norm(x.to(cuda), torch.tensor(off, dtype=torch.int32, device=cuda), [(32, 0)], 4, activation=None)
    want = reference(x.double(), off, [(32, 0)], 4, None, None, 1e-5, None)
    # the mean is off by a few steps of 1000: 2^-24 * 1000 * 8 of a spread of one
    room = 1000 * 8 * 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8 * 6 + CHAIN * 40
    assert (y.cpu().double() - want).abs().max() < room
    assert not y[:100].any() and not y[3900:].any()
    xr = x.to(cuda).requires_grad_(True)
    z = group_norm(xr, torch.tensor([100, 1000, 9000], dtype=torch.int32, device=cuda), [(32, 0)], 4)
    gx, = torch.autograd.grad(z, [xr], torch.ones_like(z))
    assert not gx[:100].any() and torch.isfinite(z.float()).all() and z[3999].any()


def test_nan_and_infinity_stay_in_their_sample(cuda):
    from ss_conv.groupnorm import group_norm
    x = torch.randn(300, 16, generator=torch.Generator().manual_seed(1)).to(cuda)
    off = torch.tensor([0, 100, 200, 300], dtype=torch.int32, device=cuda)
    clean = group_norm(x, off, [(16, 0)], 4, activation=F.silu)
    x[150, 2] = float("inf")
    x[160, 9] = float("nan")
    y = group_norm(x, off, [(16, 0)], 4, activation=F.silu)
    assert torch.equal(y[:100], clean[:100]) and torch.equal(y[200:], clean[200:])
    assert torch.equal(y[100:200, 4:8], clean[100:200, 4:8])            # the other groups of the sample as well
    assert torch.isnan(y[100:200, 8:12]).all() and torch.isnan(y[150, 2])


def test_same_bits_every_time_and_in_any_batch(cuda):
    """No atomics: two passes are equal, gradients too."""
    from ss_conv.groupnorm import group_norm
    g = torch.Generator().manual_seed(8)
    x = torch.randn(30000, 76, generator=g).to(cuda)
    Rs = [(4, 0), (4, 1), (4, 2), (4, 3), (12, 0)]
    off = torch.tensor([0, 10000, 30000], dtype=torch.int32, device=cuda)
    gy = torch.randn(30000, 64, generator=g).to(cuda)
    runs = []
    for _ in range(2):
        xr, w = x.clone().requires_grad_(True), torch.ones(28, device=cuda, requires_grad=True)
        y = group_norm(xr, off, Rs, 2, w, None, activation=GATE)
        runs.append((y,) + torch.autograd.grad(y, [xr, w], gy))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_parameters_one_by_one(cuda):
    """Without weight or bias, with either frozen: each gradient is its own parameter's; parameters in 16 bits."""
    from ss_conv.groupnorm import group_norm
    g = torch.Generator().manual_seed(2)
    x = torch.randn(50, 12, generator=g).to(cuda)
    off = torch.tensor([0, 20, 50], dtype=torch.int32, device=cuda)
    w, b = (torch.randn(12, generator=g).to(cuda).requires_grad_(True) for _ in range(2))
    gy = torch.randn(50, 12, generator=g).to(cuda)
    call = lambda w, b: group_norm(x, off, [(12, 0)], 3, w, b, activation=F.silu)  # noqa: E731
    gw, gb = torch.autograd.grad(call(w, b), [w, b], gy)
    assert torch.equal(torch.autograd.grad(call(w.detach(), b), [b], gy)[0], gb)
    assert torch.equal(torch.autograd.grad(call(w, b.detach()), [w], gy)[0], gw)
    ones, zeros = torch.ones(12, device=cuda).requires_grad_(True), torch.zeros(12, device=cuda).requires_grad_(True)
    assert torch.equal(torch.autograd.grad(call(None, b), [b], gy)[0], torch.autograd.grad(call(ones, b), [b], gy)[0])
    assert torch.equal(torch.autograd.grad(call(w, None), [w], gy)[0], torch.autograd.grad(call(w, zeros), [w], gy)[0])
    half = w.detach().half().requires_grad_(True)
    assert torch.autograd.grad(call(half, b), [half], gy)[0].dtype == torch.float16
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(call(w, b).sum(), [w], create_graph=True)


def test_strided_rows_a_side_stream_and_a_graph(cuda):
    from ss_conv.groupnorm import group_norm
    g = torch.Generator().manual_seed(9)
    wide = torch.randn(2000, 65, generator=g).to(cuda)
    off = torch.tensor([0, 999, 2000], dtype=torch.int32, device=cuda)
    rows = wide[:, 1:]                                                   # a view, off by four bytes
    want = group_norm(rows.contiguous(), off, [(64, 0)], 8, activation=F.silu)
    assert torch.equal(group_norm(rows, off, [(64, 0)], 8, activation=F.silu), want)
    shifted = torch.empty(2000 * 64 + 1, device=cuda)[1:].view(2000, 64).copy_(rows)   # contiguous, no vector alignment
    assert (group_norm(shifted, off, [(64, 0)], 8, activation=F.silu) - want).abs().max() < CHAIN * 16
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = wide[:, :64].contiguous()
        graph = torch.cuda.CUDAGraph()
        group_norm(x, off, [(64, 0)], 8, activation=F.silu)
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        y = group_norm(x, off, [(64, 0)], 8, activation=F.silu)
    x.copy_(rows)
    off.copy_(torch.tensor([0, 500, 2000], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, group_norm(x, off, [(64, 0)], 8, activation=F.silu))


def test_block_with_group_norm_and_pending_rows(cuda):
    """SS_Conv with norm_groups: fused with the gate, its rows still pending behind a strided layer, the same as layer by layer on
    exact rows; state survives a capacity that was too small."""
    from ss_conv import _ext
    from ss_conv.sp_ops.tensor import SparseTensor
    from ss_conv.utils import synthetic as S
    from ss_conv_modules import SS_Conv
    torch.manual_seed(0)
    ind = torch.from_numpy(S.surface_voxels(range(3), 24, 1024, base_seed=3)).to(cuda)
    feats = torch.randn(ind.shape[0], 8, device=cuda)
    block = SS_Conv((2, 2), (2, 2), 3, stride=2, padding=1, activation=GATE, norm_groups=2).to(cuda)
    with torch.no_grad():
        block.bn.weight.uniform_(0.5, 1.5)
        block.bn.bias.normal_()

    def run(fused):
        x = SparseTensor(feats, ind, [24] * 3, 3)
        if fused:
            return block(x).features
        return block.activation(block.bn(block.conv(x))).features

    for mode in (False, True):
        block.train(mode)
        with torch.no_grad():
            a, b = run(True), run(False)
        assert a.shape == b.shape and (a - b).abs().max() < CHAIN * 16
        c = run(True)
        assert c.requires_grad and (a - c).abs().max() < CHAIN * 16
    before = _ext.kernel_launches()
    (run(True) ** 2).sum().backward()
    assert block.bn.weight.grad.abs().sum() > 0 and _ext.kernel_launches() > before + 6


def test_refusals(cuda):
    from ss_conv.groupnorm import group_norm
    x = torch.zeros(4, 6, device=cuda)
    off = torch.tensor([0, 4], dtype=torch.int32, device=cuda)
    Rs = [(6, 0)]
    with pytest.raises(ValueError, match="features must be"):
        group_norm(x[:, :5], off, Rs)
    with pytest.raises(TypeError, match="float32"):
        group_norm(x.double(), off, Rs)
    with pytest.raises(ValueError, match="offsets"):
        group_norm(x, off.long(), Rs)
    with pytest.raises(ValueError, match="offsets"):
        group_norm(x, off.cpu(), Rs)
    with pytest.raises(ValueError, match="weight"):
        group_norm(x, off, Rs, weight=torch.ones(5, device=cuda))
    with pytest.raises(ValueError, match="at most 2048"):
        group_norm(torch.zeros(4, 2049, device=cuda), off, [(2049, 0)])
    with pytest.raises(ValueError, match="513 gates"):
        group_norm(torch.zeros(4, 2052, device=cuda), off, [(513, 1), (513, 0)], activation=(None, torch.sigmoid))
    assert group_norm(x[:0], torch.zeros(2, dtype=torch.int32, device=cuda), Rs).shape == (0, 6)
    e = x[:0].requires_grad_(True)
    w = torch.ones(6, device=cuda, requires_grad=True)
    y = group_norm(e, torch.zeros(2, dtype=torch.int32, device=cuda), Rs, weight=w)
    ge, gw = torch.autograd.grad(y, [e, w], torch.zeros_like(y))
    assert ge.shape == (0, 6) and not gw.any()
