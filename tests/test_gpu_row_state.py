"""Row operators on the GPU against what surrounds a call: recordings, inference mode, the status word, forward-mode derivatives."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def offsets(cuda, *ends):
    return torch.tensor([0, *ends], dtype=torch.int32, device=cuda)


def test_new_layout_inside_a_recording(cuda):
    """It is refused, the recording goes on; after a call outside it can be recorded."""
    from ss_conv.groupnorm import group_norm
    x, off = torch.randn(90, 33, device=cuda), offsets(cuda, 40, 90)
    call = lambda: group_norm(x, off, [(33, 0)], 11, activation=F.silu)  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="call it once before"):
            call()
        twice = x * 2
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(twice, x * 2)
    want = call()
    again = torch.cuda.CUDAGraph()
    with torch.cuda.graph(again):
        y = call()
    y.zero_()
    again.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_training_after_a_first_call_in_inference_mode(cuda, monkeypatch):
    from ss_conv import _ext
    from ss_conv.feedforward import gated_feedforward
    from ss_conv.groupnorm import group_norm
    monkeypatch.setattr(_ext, "_status", {})
    g = torch.Generator("cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    x, off, w_in, w_out = r(90, 34), offsets(cuda, 40, 90), r(2, 16, 34), r(34, 16)

    def step(x):
        return gated_feedforward(group_norm(x, off, [(34, 0)], 17, activation=F.silu), w_in, w_out)

    with torch.inference_mode():
        want = step(x)
    leaf = x.clone().requires_grad_(True)
    y = step(leaf)
    assert torch.equal(y.detach(), want) and torch.autograd.grad(y.sum(), [leaf])[0].any()
    _ext.check_status(cuda)


def test_status_cleared_between_a_result_and_its_gradients(cuda):
    """A problem of one batch is raised and cleared; the passes of the others go on."""
    from ss_conv import _ext
    from ss_conv.feedforward import gated_feedforward
    from ss_conv.groupnorm import group_norm
    g = torch.Generator("cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    x, off, w_in, w_out = r(90, 32).requires_grad_(True), offsets(cuda, 40, 90), r(2, 16, 32), r(32, 16)
    passes = (lambda: group_norm(x, off, [(32, 0)], 4), lambda: gated_feedforward(x, w_in, w_out))
    want = [torch.autograd.grad(p().sum(), [x])[0] for p in passes]
    for p, w in zip(passes, want):
        y = p().sum()
        _ext.status_word(cuda).fill_(1)
        with pytest.raises(RuntimeError, match="kernel status 0x1"):
            _ext.check_status(cuda)
        assert torch.equal(torch.autograd.grad(y, [x])[0], w)


def test_tangents_are_refused(cuda):
    """Each argument of either operator, recorded by autograd or not: a derivative of zero would be wrong."""
    import torch.autograd.forward_ad as fa
    from ss_conv.feedforward import gated_feedforward
    from ss_conv.groupnorm import group_norm
    off = offsets(cuda, 40, 90)
    z = lambda *s: torch.ones(*s, device=cuda)  # noqa: E731
    norm = dict(features=z(90, 16), weight=z(16), bias=z(16))
    ff = dict(features=z(90, 16), weight_in=z(2, 8, 16), weight_out=z(16, 8), bias_in=z(2, 8), bias_out=z(16), residual=z(90, 16))
    for call, args in ((lambda **k: group_norm(offsets=off, Rs=[(16, 0)], **k), norm), (gated_feedforward, ff)):
        call(**args)
        for name, v in args.items():
            for leaf in (False, True):
                with fa.dual_level():
                    dual = fa.make_dual(v.clone().requires_grad_(leaf), torch.ones_like(v))
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        call(**{**args, name: dual})
                    with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                        call(**{**args, name: dual})
                call(**args)


@pytest.mark.parametrize("between", ["two operations", "a layer"])
def test_recordings_look_for_earlier_graphs_behind_the_arguments(cuda, between):
    """The leaf that an eager result still holds lies several operations behind the operator's arguments: refused as well (its backward pass
    could not be recorded); with the result gone it is recorded and replays."""
    from ss_conv.feedforward import gated_feedforward
    from ss_conv.groupnorm import group_norm
    g = torch.Generator("cuda").manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    x, gy, off = r(500, 32), r(500, 32).bfloat16(), offsets(cuda, 200, 500)
    w, scale = (r(2, 48, 32) / 6).requires_grad_(True), r(32).requires_grad_(True)
    w_out = (r(32, 48) / 7).bfloat16()
    if between == "two operations":
        mine = [w]
        step = lambda: gated_feedforward(x.bfloat16(), (w * 2).exp().to(torch.bfloat16) / 8, w_out)  # noqa: E731
    else:
        mine = [scale]
        step = lambda: group_norm(torch.relu(x * scale).bfloat16() * 3, off, [(32, 0)], 8)  # noqa: E731
    want = torch.autograd.grad(step(), mine, gy)
    alive = step()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
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
