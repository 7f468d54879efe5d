"""Gated feed-forward block: forward and gradients against the formula in 64 bits, at the sizes where tiles, planes and shares of
the rows end.

Tolerances.  The products of float32 rows are exact to 2^-24 of |a| |b| a term; sums of K terms run in float32 inside tensor memory,
where an addition may cut instead of round: at most one step (2^-23) of the running sum each 8 or 16 terms, K / 8 of them for each of six
products of planes, which is what STEPS counts.  16-bit rows: h is rounded once (half a step of |h| a term), dg and du too."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def inputs(n, c, h, o, dtype, bias, residual, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return dict(x=r(n, c).to(dtype), w_in=(r(2, h, c) / c ** 0.5).to(dtype), w_out=(r(o, h) / h ** 0.5).to(dtype),
                b_in=(0.3 * r(2, h)).to(dtype) if bias else None, b_out=(0.3 * r(o)).to(dtype) if bias else None,
                residual=r(n, o).to(dtype) if residual else None), r(n, o).to(dtype)


def reference(t, act):
    g = F.linear(t["x"], t["w_in"][0], None if t["b_in"] is None else t["b_in"][0])
    u = F.linear(t["x"], t["w_in"][1], None if t["b_in"] is None else t["b_in"][1])
    y = F.linear((act(g) if act is not None else g) * u, t["w_out"], t["b_out"])
    return y if t["residual"] is None else y + t["residual"]


def bound(dtype, k, amount):
    """Of a sum over k terms whose absolute values add up to about `amount`: STEPS of float32, and in 16 bits one rounding of each term."""
    steps = (6 * k / 8 + 16) * 2.0 ** -23
    return amount * (steps + (0 if dtype == torch.float32 else 3 * torch.finfo(dtype).eps / 2))


def near(got, want, room, dtype, what):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, what
    if dtype != torch.float32:
        room = room + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal
    d = (got - want).abs()
    assert bool((d <= room).all()), (what, d.max().item(), want.abs().max().item())


SIZES = [
    # n, c, hidden, out, bias, residual, activation
    (1, 256, 1024, 256, False, True, F.silu),
    (1, 1, 1, 1, True, True, F.gelu),
    (3, 17, 33, 5, True, False, F.relu),
    (16, 64, 64, 64, False, False, F.silu),
    (17, 64, 64, 64, True, True, torch.sigmoid),
    (64, 256, 512, 128, True, False, F.gelu),
    (65, 100, 300, 76, True, True, F.silu),
    (127, 8, 72, 24, False, False, None),
    (128, 128, 128, 256, False, True, F.silu),
    (129, 65, 129, 257, True, False, F.silu),
    (1000, 512, 96, 320, False, True, F.gelu),
    (2500, 40, 200, 40, True, True, F.silu),
    (20011, 64, 160, 64, False, False, F.silu),
]


# More of them: rows on plain lanes in ones, twos, fours and eights with sums that end inside a piece, a warp or a share; tiles of more than 256 rows.
SIZES += [
    (2, 9, 65, 7, True, True, F.silu),
    (4, 257, 5, 258, False, False, F.gelu),
    (5, 40, 2050, 3, True, False, None),
    (8, 4100, 24, 8, False, True, F.silu),
    (9, 1025, 130, 31, True, True, torch.sigmoid),
    (31, 128, 512, 66, False, False, F.silu),
    (250, 33, 70, 12, True, True, F.relu),
    (256, 64, 128, 64, False, True, F.silu),
    (257, 65, 129, 257, True, False, F.silu),
    (300, 17, 33, 5, True, True, F.gelu),
    (383, 8, 72, 24, False, False, None),
    (511, 100, 300, 76, True, True, torch.sigmoid),
    (260, 600, 200, 64, False, True, F.silu),
    (40, 2048, 2048, 512, True, False, F.gelu),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", range(len(SIZES)))
def test_block_and_gradients(cuda, size, dtype):
    from ss_conv.feedforward import gated_feedforward
    n, c, h, o, bias, residual, act = SIZES[size]
    t, gy = inputs(n, c, h, o, dtype, bias, residual, 50 + size)
    names = [k for k in t if t[k] is not None]
    dev = {k: None if v is None else v.to(cuda).requires_grad_(True) for k, v in t.items()}
    t64 = {k: None if v is None else v.double().requires_grad_(True) for k, v in t.items()}
    with torch.no_grad():
        plain = gated_feedforward(dev["x"], dev["w_in"], dev["w_out"], dev["b_in"], dev["b_out"], act, dev["residual"])
    y = gated_feedforward(dev["x"], dev["w_in"], dev["w_out"], dev["b_in"], dev["b_out"], act, dev["residual"])
    assert torch.equal(plain, y) and y.dtype == dtype
    want = reference(t64, act)
    # every row of x, w_in[.] and w_out has a norm near 1 (x: sqrt c): sums of absolute values by Cauchy-Schwarz
    a64 = {k: None if v is None else v.detach().abs() for k, v in t64.items()}
    g_abs, u_abs = (F.linear(a64["x"], a64["w_in"][i], None if a64["b_in"] is None else a64["b_in"][i]) for i in (0, 1))
    h_abs = (g_abs + 1) * u_abs
    y_abs = F.linear(h_abs, a64["w_out"], a64["b_out"]) + (0 if a64["residual"] is None else a64["residual"])
    near(y, want, bound(dtype, c + h, y_abs), dtype, "y")
    grads = dict(zip(names, torch.autograd.grad(y, [dev[k] for k in names], gy.to(cuda))))
    exact = dict(zip(names, torch.autograd.grad(want, [t64[k] for k in names], gy.double())))
    gy_abs = gy.double().abs()
    dh = gy_abs @ a64["w_out"]
    dg, du = dh * u_abs * 1.13, dh * (g_abs + 1)
    near(grads["x"], exact["x"], bound(dtype, c + o + 2 * h, dg @ a64["w_in"][0] + du @ a64["w_in"][1]), dtype, "gx")
    near(grads["w_in"], exact["w_in"], bound(dtype, c + o + n, torch.stack([dg.t() @ a64["x"], du.t() @ a64["x"]])), dtype, "gw_in")
    near(grads["w_out"], exact["w_out"], bound(dtype, c + n, gy_abs.t() @ h_abs), dtype, "gw_out")
    if bias:
        near(grads["b_in"], exact["b_in"], bound(dtype, c + o + n, torch.stack([dg.sum(0), du.sum(0)])), dtype, "gb_in")
        near(grads["b_out"], exact["b_out"], bound(dtype, n, gy_abs.sum(0)), dtype, "gb_out")
    if residual:
        assert torch.equal(grads["residual"].cpu(), gy)


@pytest.mark.parametrize("dtype,most", [(torch.float32, 1e-6), (torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
def test_norm_of_the_error(cuda, dtype, most):
    """Over all values: float32 to a few steps of 2^-24, 16 bits to the roundings of h, its gradients and the result (each a step's root
    mean square, eps / sqrt(12) or less of a value, two of them in a row)."""
    from ss_conv.feedforward import gated_feedforward
    t, gy = inputs(4000, 256, 512, 192, dtype, True, False, 3)
    dev = {k: None if v is None else v.to(cuda).requires_grad_(True) for k, v in t.items()}
    t64 = {k: None if v is None else v.double().to(cuda).requires_grad_(True) for k, v in t.items()}
    y = gated_feedforward(dev["x"], dev["w_in"], dev["w_out"], dev["b_in"], dev["b_out"])
    want = reference(t64, F.silu)
    names = ["x", "w_in", "w_out", "b_in", "b_out"]
    got = [y, *torch.autograd.grad(y, [dev[k] for k in names], gy.to(cuda))]
    exact = [want, *torch.autograd.grad(want, [t64[k] for k in names], gy.double().to(cuda))]
    for name, a, b in zip(["y"] + names, got, exact):
        assert ((a.double() - b).norm() / b.norm()).item() < most, name


def test_some_gradients_alone_and_differences(cuda):
    from ss_conv.feedforward import gated_feedforward
    t, gy = inputs(200, 24, 40, 16, torch.float32, True, True, 4)
    dev = {k: v.to(cuda) for k, v in t.items()}
    gy = gy.to(cuda)

    def loss(**swap):
        a = {**dev, **swap}
        return (gated_feedforward(a["x"], a["w_in"], a["w_out"], a["b_in"], a["b_out"], F.silu, a["residual"]).double() * gy).sum()

    for name in dev:
        leaf = dev[name].clone().requires_grad_(True)
        g, = torch.autograd.grad(loss(**{name: leaf}), [leaf])
        flat = g.reshape(-1)
        at = int(flat.abs().argmax())
        h = 2.0 ** -6
        d = torch.zeros_like(dev[name]).reshape(-1)
        d[at] = h
        d = d.view_as(dev[name])
        num = (loss(**{name: dev[name] + d}) - loss(**{name: dev[name] - d})) / (2 * h)
        # third derivatives times h^2 / 6 (4e-5), and the rounding of 3200 terms over 2 h
        assert abs(num.item() - flat[at].item()) <= 1e-2 * max(1.0, abs(flat[at].item())), name


def test_rows_taken_in_turns(cuda):
    """More rows than one turn's scratch holds: the rows of all turns, the gradients of the weights over all of them, and the same bits
    twice.  float32, so the errors are those of the norm test below."""
    from ss_conv.feedforward import gated_feedforward
    from ss_conv import _ext
    n, c, h = 70001, 16, 2048
    one, all_ = (int(_ext.lib().ssc_gated_ff_scratch_bytes(0, k, c, h, c, 1)) for k in (20000, n))
    assert all_ < 3 * one                                       # (three turns or more)
    t, gy = inputs(n, c, h, c, torch.float32, True, False, 12)
    names = ["x", "w_in", "w_out", "b_in", "b_out"]
    dev = {k: t[k].to(cuda).requires_grad_(True) for k in names}
    d64 = {k: t[k].double().to(cuda).requires_grad_(True) for k in names}
    runs = []
    for _ in range(2):
        y = gated_feedforward(*(dev[k] for k in names))
        runs.append([y.detach(), *torch.autograd.grad(y, [dev[k] for k in names], gy.to(cuda))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    want = reference({**d64, "residual": None}, F.silu)
    exact = [want.detach(), *torch.autograd.grad(want, [d64[k] for k in names], gy.double().to(cuda))]
    for name, a, b in zip(["y"] + names, runs[0], exact):
        assert ((a.double() - b).norm() / b.norm()).item() < 2e-6, name
    assert (runs[0][0][-1].double() - exact[0][-1]).abs().max() < 1e-4 and (runs[0][1][-1].double() - exact[1][-1]).abs().max() < 1e-4


def test_every_choice_of_gradients(cuda):
    """Arguments that are absent, and those that ask for no gradient, in all combinations: each gradient is its own argument's."""
    import itertools
    from ss_conv.feedforward import gated_feedforward
    t, gy = inputs(70, 16, 24, 8, torch.float32, True, True, 9)
    names = list(t)
    full = {k: v.to(cuda).requires_grad_(True) for k, v in t.items()}
    for there in itertools.product((False, True), repeat=3):
        absent = [n for n, on in zip(("b_in", "b_out", "residual"), there) if not on]
        use = {k: (None if k in absent else v) for k, v in full.items()}
        y = gated_feedforward(use["x"], use["w_in"], use["w_out"], use["b_in"], use["b_out"], F.silu, use["residual"])
        have = [k for k in names if use[k] is not None]
        want = dict(zip(have, torch.autograd.grad(y, [use[k] for k in have], gy.to(cuda))))
        for asks in itertools.product((False, True), repeat=len(have)):
            if not any(asks):
                continue
            ask = [k for k, on in zip(have, asks) if on]
            leaf = {k: None if use[k] is None else use[k].detach().requires_grad_(k in ask) for k in names}
            y = gated_feedforward(leaf["x"], leaf["w_in"], leaf["w_out"], leaf["b_in"], leaf["b_out"], F.silu, leaf["residual"])
            for k, g in zip(ask, torch.autograd.grad(y, [leaf[k] for k in ask], gy.to(cuda))):
                assert torch.equal(g, want[k]), (absent, ask, k)
    y = gated_feedforward(full["x"], full["w_in"], full["w_out"])
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(y.sum(), [full["x"]], create_graph=True)


def test_not_finite_rows_stay_their_own(cuda):
    from ss_conv.feedforward import gated_feedforward
    for n in (8, 300):
        for dtype in (torch.float32, torch.bfloat16):
            t, _ = inputs(n, 32, 64, 32, dtype, False, False, 6)
            dev = {k: None if v is None else v.to(cuda) for k, v in t.items()}
            clean = gated_feedforward(dev["x"], dev["w_in"], dev["w_out"])
            dev["x"][5, 3] = float("nan")
            dev["x"][2, 0] = float("inf")
            y = gated_feedforward(dev["x"], dev["w_in"], dev["w_out"])
            keep = [i for i in range(n) if i not in (2, 5)]
            assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[5]).all() and not torch.isfinite(y[2]).any()


def test_views_streams_and_graphs(cuda):
    from ss_conv import _ext
    from ss_conv.feedforward import gated_feedforward
    t, gy = inputs(700, 48, 96, 48, torch.bfloat16, False, True, 7)
    dev = {k: None if v is None else v.to(cuda) for k, v in t.items()}
    want = gated_feedforward(dev["x"], dev["w_in"], dev["w_out"], residual=dev["residual"])
    wide = torch.zeros(700, 49, dtype=torch.bfloat16, device=cuda)
    wide[:, 1:] = dev["x"]
    assert torch.equal(gated_feedforward(wide[:, 1:], dev["w_in"], dev["w_out"], residual=dev["residual"]), want)
    off = torch.empty(700 * 48 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(700, 48).copy_(dev["x"])     # rows TMA cannot read in place
    assert torch.equal(gated_feedforward(off, dev["w_in"], dev["w_out"], residual=dev["residual"]), want)
    wt = dev["w_out"].t().contiguous().t()
    assert torch.equal(gated_feedforward(dev["x"], dev["w_in"], wt, residual=dev["residual"]), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    x = dev["x"].clone().requires_grad_(True)
    w = dev["w_in"].clone().requires_grad_(True)
    g = gy.to(cuda)
    with torch.cuda.stream(side):
        torch.autograd.grad(gated_feedforward(x, w, dev["w_out"]), [x, w], g)
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        y = gated_feedforward(x, w, dev["w_out"])
        gx, gw = torch.autograd.grad(y, [x, w], g)
    with torch.no_grad():
        x.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    y2 = gated_feedforward(x, w, dev["w_out"])
    gx2, gw2 = torch.autograd.grad(y2, [x, w], g)
    assert torch.equal(y, y2) and torch.equal(gx, gx2) and torch.equal(gw, gw2)
    _ext.check_status(cuda)


def test_modules_and_refusals(cuda):
    from ss_conv.feedforward import GatedFeedForward, gated_feedforward
    from ss_conv.sp_ops.tensor import SparseTensor
    torch.manual_seed(0)
    m = GatedFeedForward(24, 64, bias=True).to(cuda)
    x = torch.randn(90, 24, device=cuda)
    ind = torch.zeros(90, 4, dtype=torch.int32, device=cuda)
    y = m(x, x)
    assert torch.equal(m(SparseTensor(x, ind, [4] * 3, 1), x).features, y)
    with torch.no_grad():
        assert torch.equal(m(SparseTensor(x, ind, [4] * 3, 1)).features, m(x))
    m(x.bfloat16()).float().sum().backward()                # rows of another type than the parameters
    assert all(p.grad is not None and p.grad.dtype == torch.float32 for p in m.parameters())
    assert m(x[:0]).shape == (0, 24)
    e = x[:0].clone().requires_grad_(True)
    m.zero_grad()
    m(e).sum().backward()
    assert e.grad.shape == (0, 24) and not m.weight_in.grad.any()
    w_in, w_out = m.weight_in, m.weight_out
    for bad in ((x[:, :23], w_in, w_out), (x, w_in[:1], w_out), (x, w_in, w_out[:, 1:]), (x, w_in, w_out, torch.zeros(64, device=cuda)),
                (x, w_in, w_out, None, torch.zeros(23, device=cuda)), (x.half(), w_in, w_out), (x, w_in.cpu(), w_out)):
        with pytest.raises(ValueError):
            gated_feedforward(*bad)
    with pytest.raises(ValueError, match="residual"):
        gated_feedforward(x, w_in, w_out, residual=x[:1])
    with pytest.raises(TypeError):
        gated_feedforward(x.double(), w_in.double(), w_out.double())
    with pytest.raises(ValueError, match="activation"):
        gated_feedforward(x, w_in, w_out, activation=torch.tanh)
