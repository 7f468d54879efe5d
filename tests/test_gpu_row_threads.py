"""Row operators called from threads that have not touched the GPU before, as autograd's are before their first backward pass."""
import ctypes
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def in_new_thread(fn):
    out = []
    t = threading.Thread(target=lambda: out.append(fn()))
    t.start()
    t.join()
    return out[0]


@pytest.mark.parametrize("kind,dtype", [(2, torch.float16), (3, torch.bfloat16), (0, torch.float32)])
@pytest.mark.parametrize("rows", [5, 400])
def test_first_call_of_a_thread(cuda, kind, dtype, rows):
    """All memory is there, so that the operator's own calls are the thread's first ones."""
    from ss_conv import _ext
    L = _ext.lib()
    g = torch.Generator("cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda).to(dtype)  # noqa: E731
    c, h = 64, 128
    x, gy, w_in, w_out = r(rows, c), r(rows, c), r(2, h, c) / 8, r(c, h) / 11
    y, gx, gw_in, gw_out = (torch.zeros_like(t) for t in (x, x, w_in, w_out))
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    need = max(int(L.ssc_gated_ff_scratch_bytes(kind, rows, c, h, c, back)) for back in (0, 1))
    scratch = torch.empty(need, dtype=torch.uint8, device=cuda)
    torch.cuda.synchronize()

    def forward():
        return L.ssc_gated_ff_fwd(p(x), kind, rows, c, h, c, p(w_in), p(w_out), None, None, None, 3, p(y), None, p(scratch), need, None), L.ssc_last_error()

    def backward():
        return L.ssc_gated_ff_bwd(p(x), p(gy), kind, rows, c, h, c, p(w_in), p(w_out), None, 3, p(gx), p(gw_in), p(gw_out), None, None, None, p(scratch), need,
                                  None), L.ssc_last_error()

    for call in (forward, backward):
        rc, what = in_new_thread(call)
        assert rc == 0, what
    torch.cuda.synchronize()
    got = [t.clone() for t in (y, gx, gw_in, gw_out)]
    assert forward()[0] == 0 and backward()[0] == 0
    torch.cuda.synchronize()
    assert all(t.any() and torch.equal(t, k) for t, k in zip((y, gx, gw_in, gw_out), got))


def test_operators_in_a_new_thread(cuda):
    """The Python functions, their memory from the allocator's store."""
    from ss_conv.feedforward import gated_feedforward
    from ss_conv.groupnorm import group_norm
    off = torch.tensor([0, 150, 400], dtype=torch.int32, device=cuda)
    g = torch.Generator("cuda").manual_seed(3)
    x, w_in, w_out = (torch.randn(*s, generator=g, device=cuda).bfloat16() for s in ((400, 64), (2, 128, 64), (64, 128)))
    call = lambda: gated_feedforward(group_norm(x, off, [(64, 0)], 8), w_in, w_out, residual=x)  # noqa: E731
    with torch.no_grad():
        want = call()
    torch.cuda.synchronize()

    def run():
        with torch.no_grad():
            y = call()
            torch.cuda.synchronize()
            return y

    assert torch.equal(in_new_thread(run), want)
    assert torch.equal(in_new_thread(lambda: gated_feedforward(x, w_in, w_out)), gated_feedforward(x, w_in, w_out))
