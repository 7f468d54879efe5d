"""Arguments of the row operators that are refused before anything reaches a GPU."""
import pytest
import torch
import torch.nn.functional as F


def test_group_norm_layouts():
    from ss_conv.groupnorm import GroupNorm, _layout, act_code, group_norm
    lay = _layout(((4, 0), (2, 1), (2, 0)), 2, True, True)
    assert (lay.c, lay.c_out, lay.n_gate, lay.n_group, lay.n_field, lay.n_scalar) == (12, 10, 2, 6, 8, 6)
    c, f, g = 12, 8, 6
    at = lay.rows
    assert at[:c] == [0, 0, 1, 1, 2, 2, 2, 3, 3, 3, 4, 5]
    assert at[c:2 * c] == [0, 1, 2, 3, 4, 4, 4, 5, 5, 5, 6, 7]
    assert at[2 * c:3 * c] == [0, 1, 2, 3] + [-1] * 6 + [4, 5]
    assert at[3 * c:3 * c + 10] == [-1] * 4 + [0] * 3 + [1] * 3
    rest = at[3 * c + 10:]
    assert rest[:f] == [0, 1, 2, 3, 4, 7, 10, 11] and rest[f:2 * f] == [1, 1, 1, 1, 3, 3, 1, 1]
    assert rest[2 * f:3 * f] == [0, 1, 2, 3, -1, -1, 4, 5] and rest[3 * f:3 * f + 2] == [4, 5]
    assert rest[3 * f + 2:] == [0, 2, 4, 7, 10, 11] + [2, 2, 3, 3, 1, 1] + [2, 2, 1, 1, 1, 1] and len(rest) == 3 * f + 2 + 3 * g
    for Rs, groups, act in (([(6, 0)], 4, None), ([(6, 0)], 0, None), ([], 1, None), ([(-1, 0)], 1, None), ([(0, 0)], 1, None),
                            ([(2, 0), (2, 1), (3, 0)], 1, (F.relu, torch.sigmoid)), ([(2, 0), (2, 1)], 1, (F.relu, torch.sigmoid))):
        with pytest.raises(ValueError):
            GroupNorm(Rs, groups, activation=act)
    with pytest.raises(ValueError, match="activation must be"):
        act_code(torch.tanh)
    assert [act_code(a) for a in (None, F.relu, torch.sigmoid, F.silu, F.gelu, torch.nn.SiLU(), torch.nn.GELU())] == [0, 1, 2, 3, 4, 3, 4]
    with pytest.raises(ValueError):
        act_code(torch.nn.GELU(approximate="tanh"))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        group_norm(torch.zeros(3, 6), torch.tensor([0, 3], dtype=torch.int32), [(6, 0)])
    with pytest.raises(ValueError, match="eps"):
        group_norm(torch.zeros(3, 6), torch.tensor([0, 3], dtype=torch.int32), [(6, 0)], eps=0)


def test_library_refuses_bad_arguments_of_the_norm():
    from ss_conv import _ext
    L = _ext.lib()

    def forward(type=0, out_type=0, n=0, c=8, batch=1, fields=8, scalars=8, groups=2, gates=0, act=0, eps=1e-5, table=64):
        # (addresses that nothing reads: the call ends before its first launch)
        return L.ssc_group_norm_fwd(64, type, n, c, 64, batch, table, fields, scalars, groups, gates, None, None, eps, act, 0, 64, out_type, 64,
                                    None, None, 0, None)

    assert forward() == 0                                               # no rows: nothing to do
    for bad in (dict(type=1), dict(type=2, out_type=0), dict(n=-1), dict(n=2 ** 30 + 1), dict(c=0), dict(batch=0), dict(fields=9), dict(scalars=9), dict(groups=0),
                dict(gates=8), dict(act=5), dict(eps=0.0), dict(table=None)):
        assert forward(**bad) == 1, bad
    assert forward(n=5) == 3 and b"scratch" in L.ssc_last_error()
    assert L.ssc_group_norm_scratch_bytes(0, 2, 8, 8) == 0


def test_feedforward_refusals():
    from ss_conv import _ext
    from ss_conv.feedforward import GatedFeedForward, gated_feedforward
    L = _ext.lib()

    def forward(type=0, n=0, c=8, hidden=8, out=8, act=3, w=64):
        return L.ssc_gated_ff_fwd(64, type, n, c, hidden, out, w, 64, None, None, None, act, 64, None, None, 0, None)

    assert forward() == 0
    for bad in (dict(type=1), dict(type=4), dict(n=-1), dict(n=2 ** 30 + 1), dict(c=0), dict(hidden=0), dict(out=0), dict(hidden=65537), dict(act=5), dict(act=-1), dict(w=None)):
        assert forward(**bad) == 1, bad
    assert forward(n=5) == 3 and b"scratch" in L.ssc_last_error()
    assert L.ssc_gated_ff_bwd(64, 64, 0, 5, 8, 8, 8, 64, 64, None, 3, 64, None, None, None, None, None, None, 0, None) == 3
    assert L.ssc_gated_ff_scratch_bytes(0, 5, 0, 8, 8, 0) == 0
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        gated_feedforward(torch.zeros(2, 4), torch.zeros(2, 8, 4), torch.zeros(4, 8))
    with pytest.raises(ValueError):
        GatedFeedForward(4, 8, activation=torch.tanh)


def test_feedforward_scratch_is_bounded_and_covers_its_pieces():
    """A million wide rows are taken in turns."""
    from ss_conv import _ext
    L = _ext.lib()
    for kind in (0, 2, 3):
        for back in (0, 1):
            sizes = [int(L.ssc_gated_ff_scratch_bytes(kind, n, 512, 2048, 512, back)) for n in (0, 1, 16, 17, 64, 65, 1000, 100000, 1000000, 2 ** 30)]
            assert max(sizes) < 3 * 2 ** 30 and all(s > 0 for s in sizes)
