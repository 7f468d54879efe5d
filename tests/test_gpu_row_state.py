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
