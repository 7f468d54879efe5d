"""What the row operators keep from one call for the next: channel tables on the device and the status word."""
import gc
import weakref

import pytest
import torch

CPU = torch.device("cpu")


def test_channel_tables_outlive_any_number_of_layouts():
    """A recorded graph holds a table's address and nothing else: tables stay for the life of the process."""
    from ss_conv.groupnorm import GroupNorm, _layout, _plan
    norm = GroupNorm([(777, 0)], 7)
    table = _plan(tuple(norm.Rs), 7, None)[0].table(CPU)
    where, alive = table.data_ptr(), weakref.ref(table)
    del table
    for m in range(1, 600):
        _plan(((m, 1),), 1, None)[0].table(CPU)
        _layout(((m, 2),), 1, False, False)
    gc.collect()
    assert alive() is not None
    again = _plan(tuple(norm.Rs), 7, None)[0].table(CPU)
    assert again is alive() and again.data_ptr() == where


def test_plans_do_not_keep_modules():
    """What is kept for good are tables, not the activation modules that calls were made with."""
    from ss_conv.groupnorm import _plan
    act = torch.nn.SiLU()
    alive = weakref.ref(act)
    _plan(((8, 0),), 2, act)
    del act
    for m in range(1, 300):
        _plan(((m, 1),), 1, None)
    gc.collect()
    assert alive() is None


def test_first_call_of_a_layout_inside_a_recording_is_refused(monkeypatch):
    """Before anything reaches the device: the upload would void the recording.  A table that is there is handed out."""
    from ss_conv.groupnorm import _layout
    device = torch.device("cuda", 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    lay = _layout(((13, 0),), 13, False, False)
    with pytest.raises(RuntimeError, match="call it once before"):
        lay.table(device)
    assert not lay.tables
    lay.tables[device] = "there"
    assert lay.table(device) == "there"
    assert lay.table(CPU).dtype == torch.int32
    lay.tables.clear()


def test_what_is_kept_is_no_inference_tensor(monkeypatch):
    """The first call may be an evaluation under inference_mode; training passes use the same tensors afterwards."""
    from ss_conv import _ext
    from ss_conv.groupnorm import _layout
    monkeypatch.setattr(_ext, "_status", {})
    monkeypatch.setattr(_ext, "_open_alarm", lambda: None)
    with torch.inference_mode():
        assert not _layout(((14, 0),), 14, False, False).table(CPU).is_inference()
        assert not _ext.status_word(CPU).is_inference()
    _ext.status_word(CPU).zero_()


def test_rows_stay_pending_when_their_recomputation_fails():
    """An operation behind a row count that did not fit raises: no half of the new rows is left behind, and the next look tries again."""
    from ss_conv.sp_ops.tensor import PendingRows, SparseTensor
    old, new = torch.zeros(4, 3), torch.arange(21.0).view(7, 3)
    old_inds, new_inds = torch.zeros(4, 4, dtype=torch.int32), torch.ones(7, 4, dtype=torch.int32)
    t = SparseTensor(old, old_inds, [8] * 3, 2)
    t._rows = PendingRows(torch.tensor([7], dtype=torch.int32), 4, None, lambda: (new, new_inds))
    t._rows.count.value = 7
    fails, seen = [True, True], []

    def rowwise(f):
        seen.append(t.get_offsets().tolist())       # (sample by sample: of the new rows)
        if fails and fails.pop():
            raise RuntimeError("no room")
        return f + 1

    t._rows.post.append(rowwise)
    for look in (lambda: t.features, lambda: t.indices):
        with pytest.raises(RuntimeError, match="no room"):
            look()
        assert t.pending() and t._features is old and t._indices is old_inds
    assert torch.equal(t.features, new + 1) and t.indices is new_inds and not t.pending()
    assert seen == [[0, 0, 7]] * 3
