"""Group norm and feed-forward together, as a network uses them: behind sparse convolutions, in training, in a recorded graph, on row
counts that are still on the device."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
GATE = (torch.relu, torch.sigmoid)


def voxels(cuda, batch=3, grid=24, seed=3):
    from ss_conv.utils import synthetic as S
    return torch.from_numpy(S.surface_voxels(range(batch), grid, 1024, base_seed=seed)).to(cuda)


def block64(block, x, offsets):
    """x + ff(norm(x)) in 64 bits by torch's own operations."""
    norm, ff = block.norm, block.ff
    y = torch.cat([F.group_norm(x[lo:hi].t()[None], norm.num_groups, norm.weight, norm.bias, norm.eps)[0].t()
                   for lo, hi in zip(offsets[:-1], offsets[1:])])
    b_in = ff.bias_in if ff.bias_in is not None else (None, None)
    h = F.silu(F.linear(y, ff.weight_in[0], b_in[0])) * F.linear(y, ff.weight_in[1], b_in[1])
    return x + F.linear(h, ff.weight_out, ff.bias_out)


@pytest.mark.parametrize("rows", [700, 40])
def test_residual_block_in_training(cuda, rows):
    """Results and all gradients of two blocks in a row and a step on them, against 64 bits; float32 sums throughout, so the errors are
    steps of 2^-24 times the lengths of the chains (some hundred) and the growth through the blocks."""
    import copy
    from ss_conv.sp_ops.tensor import SparseTensor
    from ss_conv_modules import SS_FeedForward
    torch.manual_seed(1)
    net = torch.nn.Sequential(SS_FeedForward(48, 96, 6, bias=True), SS_FeedForward(48, 80, 3)).to(cuda)
    with torch.no_grad():
        for m in net:
            m.norm.weight.uniform_(0.5, 1.5)
            m.norm.bias.normal_(0, 0.3)
    net64 = copy.deepcopy(net).double()
    ind = torch.zeros(rows, 4, dtype=torch.int32, device=cuda)
    cut = rows // 3
    ind[cut:, 0] = 1
    x = torch.randn(rows, 48, device=cuda).requires_grad_(True)
    x64 = x.detach().double().requires_grad_(True)
    gy = torch.randn(rows, 48, device=cuda)
    y = net(SparseTensor(x, ind, [8] * 3, 2)).features
    y64 = block64(net64[1], block64(net64[0], x64, [0, cut, rows]), [0, cut, rows])
    (y * gy).sum().backward()
    (y64 * gy.double()).sum().backward()

    def far(a, b):
        return ((a.double() - b).norm() / b.norm()).item()

    limit = 256 * 2.0 ** -24
    assert far(y.detach(), y64.detach()) < limit and far(x.grad, x64.grad) < limit
    for (name, p), q in zip(net.named_parameters(), net64.parameters()):
        assert far(p.grad, q.grad) < limit, name
    before = y.detach().clone()
    opt = torch.optim.SGD(net.parameters(), lr=1e-2)
    opt.step()
    opt.zero_grad()
    assert not torch.equal(net(SparseTensor(x.detach(), ind, [8] * 3, 2)).features, before)


@pytest.mark.parametrize("storage", [None, "bf16"])
def test_network_layer_by_layer_and_recorded(cuda, storage):
    """Convolution, group norm and gate, feed-forward on its scalars, pool: the recorded graph gives what the layers give one by one, on
    another batch than it was recorded with; so do layers on pending rows whose capacity was too small."""
    from ss_conv import _ext
    from ss_conv.graph import GraphedChain
    from ss_conv.pool import GlobalAvgPool
    from ss_conv.sp_ops.tensor import SparseTensor
    from ss_conv_modules import SS_Conv, SS_FeedForward
    torch.manual_seed(2)
    one = SS_Conv((4, 2), (16,), 3, stride=2, padding=1, activation=(torch.relu, None), norm_groups=4).to(cuda).eval()
    two, pool = SS_FeedForward(16, 48, 4).to(cuda).eval(), GlobalAvgPool()
    _ext.set_feature_storage(storage)
    try:
        with torch.no_grad():
            chain = GraphedChain(lambda t: pool(two(one(t))), [24] * 3, 3, 10, 6000, "cuda")
            for seed in (3, 4):
                ind = voxels(cuda, seed=seed)
                f = torch.randn(ind.shape[0], 10, device=cuda)
                want = pool(two(one(SparseTensor(f, ind, [24] * 3, 3))))
                got = chain(f, ind)
                room = 1e-5 if storage is None else 2.0 ** -6            # (atomics nowhere; the pool adds rows in another order at most)
                assert (got - want).abs().max() <= room * want.abs().max()
    finally:
        _ext.set_feature_storage(None)


def test_two_streams_and_two_graphs_at_once(cuda):
    """Calls on two streams, and two recorded passes replayed side by side, share nothing."""
    from ss_conv.feedforward import gated_feedforward
    from ss_conv.groupnorm import group_norm
    off = torch.tensor([0, 3000, 7000], dtype=torch.int32, device=cuda)
    data = []
    for k in range(2):
        g = torch.Generator("cuda").manual_seed(k)
        r = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
        data.append((r(7000, 64), r(2, 128, 64) / 8, r(64, 128) / 11))

    def step(x, w_in, w_out):
        return gated_feedforward(group_norm(x, off, [(64, 0)], 8, activation=F.silu), w_in, w_out, residual=x)

    want = [step(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for s, d in zip(streams, data):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(step(*d))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for s, d in zip(streams, data):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(step(*d))
        graphs.append(g)
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("converted", [False, True])
def test_a_training_pass_is_recorded_without_results_from_before(cuda, converted):
    """With an eager result of the same parameters alive (on the default stream) a recording is refused; without it, it replays."""
    from ss_conv.feedforward import gated_feedforward
    from ss_conv.groupnorm import group_norm
    off = torch.tensor([0, 300, 700], dtype=torch.int32, device=cuda)
    g = torch.Generator("cuda").manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    dtype = torch.bfloat16 if converted else torch.float32
    x, gy = r(700, 32).to(dtype), r(700, 32).to(dtype)
    params = [p.requires_grad_() for p in (r(32), r(32), r(2, 48, 32) / 6, r(32, 48) / 7)]

    def norm():
        return group_norm(x, off, [(32, 0)], 8, params[0], params[1], activation=F.silu)

    def ff():
        return gated_feedforward(x, params[2].to(dtype), params[3].to(dtype), residual=x)

    for step, mine in ((norm, params[:2]), (ff, params[2:])):
        want = torch.autograd.grad(step(), mine, gy)
        alive = step()
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            torch.zeros(8, device=cuda)
            with pytest.raises(RuntimeError, match="before this recording"):
                step()
        del alive, graph
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = torch.autograd.grad(step(), mine, gy)
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
