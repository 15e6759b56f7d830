"""Refusals of the ragged operators, before any CUDA call (CPU; no kernel is launched)."""

import ctypes

import pytest
import torch

import razorkv_b200 as R
from razorkv_b200 import _lib


def _tables(**changes):
    a = dict(lengths=torch.tensor([3, 0]), new_lengths=torch.tensor([4, 2]),
             page_table=torch.zeros(2, 5, dtype=torch.int64), free_ring=torch.arange(9),
             free_state=torch.tensor([0, 9, 0]), page_size=4, max_new_tokens=8)
    a.update(changes)
    return R.ragged_page_tables(**a)


def _append(**changes):
    a = dict(key=torch.zeros(3, 2, 8), value=torch.zeros(3, 2, 8), key_pool=torch.zeros(5, 2, 4, 8),
             value_pool=torch.zeros(5, 2, 4, 8), slot_map=torch.tensor([0, 5, -1]))
    a.update(changes)
    return R.ragged_append(**a)


def _attend(**changes):
    a = dict(query=torch.zeros(2, 4, 1, 8), key_pool=torch.zeros(5, 2, 4, 8),
             value_pool=torch.zeros(5, 2, 4, 8), page_table=torch.zeros(2, 3, dtype=torch.int64),
             lengths=torch.tensor([1, 7]))
    a.update(changes)
    return R.ragged_decode_attention(**a)


def test_valid_calls_end_at_the_device():
    """Nothing but the device is wrong with these (tensors on the CPU: it is looked at last)."""
    for call in (_tables, _append, _attend, lambda: _tables(inplace=True),
                 lambda: _attend(starts=torch.tensor([0, 3]), scale=0.5, return_lse=True,
                                 out=torch.zeros(2, 4, 1, 8)),
                 lambda: _attend(starts=torch.tensor([0, 3]), scale=2, validate=True)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("changes,error", [
    (dict(lengths=torch.tensor([3, 0], dtype=torch.int32)), TypeError),
    (dict(page_table=torch.zeros(2, 5, dtype=torch.int32)), TypeError),
    (dict(free_state=torch.zeros(3)), TypeError),
    (dict(lengths=torch.tensor([[3, 0]])), ValueError),
    (dict(new_lengths=torch.tensor([1, 2, 3])), ValueError),
    (dict(free_state=torch.tensor([0, 9])), ValueError),
    (dict(free_ring=torch.zeros(0, dtype=torch.int64)), ValueError),
    (dict(page_size=0), ValueError),
    (dict(page_size=1.5), TypeError),
    (dict(page_size=1 << 70), TypeError),
    (dict(free_ring=None), TypeError),
    (dict(max_new_tokens=-1), ValueError),
    (dict(page_table=torch.zeros(5, 2, dtype=torch.int64).t()), ValueError),
    (dict(page_table=torch.zeros(1, 5, dtype=torch.int64).expand(2, 5)), ValueError),
    (dict(free_ring=torch.arange(18)[::2]), ValueError),
    (dict(lengths=torch.tensor([3, 9, 0, 9])[::2], inplace=True), ValueError),
])
def test_tables_refusals(changes, error):
    with pytest.raises(error):
        _tables(**changes)


@pytest.mark.parametrize("changes,error", [
    (dict(key=torch.zeros(2, 2, 8)), ValueError),
    (dict(value=torch.zeros(3, 2, 4)), ValueError),
    (dict(key=torch.zeros(3, 2, 8, dtype=torch.float16)), TypeError),
    (dict(value_pool=torch.zeros(5, 2, 4, 8, dtype=torch.float16)), TypeError),
    (dict(slot_map=torch.tensor([0, 5, -1], dtype=torch.int32)), TypeError),
    (dict(slot_map=torch.tensor([[0, 5, -1]])), ValueError),
    (dict(value_pool=torch.zeros(5, 2, 4, 4)), ValueError),
    (dict(value_pool=torch.zeros(5, 4, 2, 8).transpose(1, 2)), ValueError),
    (dict(key_pool=torch.zeros(5, 2, 8, 4).transpose(2, 3),
          value_pool=torch.zeros(5, 2, 8, 4).transpose(2, 3)), ValueError),
    (dict(key_pool=torch.zeros(0, 2, 4, 8), value_pool=torch.zeros(0, 2, 4, 8)), ValueError),
    (dict(key=torch.zeros(3, 2, 8, dtype=torch.float64),
          value=torch.zeros(3, 2, 8, dtype=torch.float64),
          key_pool=torch.zeros(5, 2, 4, 8, dtype=torch.float64),
          value_pool=torch.zeros(5, 2, 4, 8, dtype=torch.float64)), TypeError),
])
def test_append_refusals(changes, error):
    with pytest.raises(error):
        _append(**changes)


@pytest.mark.parametrize("changes,error", [
    (dict(query=torch.zeros(2, 4, 2, 8)), AssertionError),
    (dict(query=torch.zeros(2, 4, 8)), ValueError),
    (dict(query=torch.zeros(2, 3, 1, 8)), ValueError),
    (dict(query=torch.zeros(2, 4, 1, 16)), ValueError),
    (dict(query=torch.zeros(2, 4, 1, 8, dtype=torch.bfloat16)), TypeError),
    (dict(lengths=torch.tensor([1, 7], dtype=torch.int32)), TypeError),
    (dict(lengths=torch.tensor([1])), ValueError),
    (dict(page_table=torch.zeros(3, 3, dtype=torch.int64)), ValueError),
    (dict(page_table=torch.zeros(2, 3)), TypeError),
    (dict(starts=torch.tensor([1])), ValueError),
    (dict(starts=torch.tensor([1., 2.])), TypeError),
    (dict(scale=0.0), ValueError),
    (dict(scale=1e-60), ValueError),
    (dict(scale=1e60), ValueError),
    (dict(scale="x"), TypeError),
    (dict(query=None), TypeError),
    (dict(scale=-1.0), ValueError),
    (dict(scale=float("nan")), ValueError),
    (dict(scale=float("inf")), ValueError),
    (dict(out=torch.zeros(2, 4, 8)), ValueError),
    (dict(out=torch.zeros(2, 4, 1, 8, dtype=torch.float16)), ValueError),
    (dict(value_pool=torch.zeros(5, 2, 8, 8)), ValueError),
])
def test_attend_refusals(changes, error):
    with pytest.raises(error):
        _attend(**changes)


def test_attend_refuses_its_query_as_output():
    q = torch.zeros(2, 4, 1, 8)
    with pytest.raises(ValueError, match="query"):
        _attend(query=q, out=q)


def test_validation_names_bad_lengths_and_pages():
    with pytest.raises(IndexError, match="lengths"):
        _attend(lengths=torch.tensor([1, 13]), validate=True)
    with pytest.raises(IndexError, match="lengths"):
        _attend(lengths=torch.tensor([-1, 3]), validate=True)
    bad = torch.tensor([[0, 9, 9], [4, 5, 0]])
    with pytest.raises(IndexError, match="page_table"):
        _attend(page_table=bad, lengths=torch.tensor([4, 7]), validate=True)
    with pytest.raises(RuntimeError, match="CUDA"):   # entries past a request's tokens are not looked at
        _attend(page_table=bad, lengths=torch.tensor([4, 4]), validate=True)


def test_c_entries_refuse_bad_arguments():
    """Every refusal comes before a CUDA call: this host has no device."""
    lib = _lib.load()
    t = lib.rkv_ragged_page_tables
    ok = [16, 16, 2, 4, 16, 5, 5, 16, 9, 16, 16, 16, 16, 16, 8, 16, None]
    for at, value in ((0, None), (1, None), (2, -1), (3, 0), (4, None), (5, 4), (6, -1), (7, None),
                      (8, 0), (9, None), (10, None), (11, None), (12, None), (13, None), (14, -1),
                      (15, None), (3, 1 << 62), (8, 1 << 62)):
        args = list(ok)
        args[at] = value
        assert t(*args) == 1, (at, value)
    lay, q, o = _lib.KVLayout(), _lib.Query(), _lib.Output()
    assert lib.rkv_ragged_append(lay, None, None, 0, 0, 1, None, None) == 1
    assert lib.rkv_ragged_decode_attention_workspace_size(q, lay) == 0
    assert lib.rkv_ragged_decode_attention(q, lay, None, None, 0.0, o, None, None, 0, None) == 1

    def layout(**changes):
        a = dict(k=16, v=16, dtype=2, head_dim=128, batch=2, num_kv_heads=2, stride_h=2048,
                 stride_p=4096, stride_t=128, page_size=16, num_slots=7, page_table=16,
                 pt_stride_b=3, num_tokens=48)
        a.update(changes)
        return _lib.KVLayout(**a)

    for changes, status in ((dict(k=None), 1), (dict(dtype=3), 2), (dict(head_dim=257), 2),
                            (dict(head_dim=0), 2), (dict(num_kv_heads=0), 1),
                            (dict(page_size=0), 1), (dict(num_slots=0), 1), (dict(row_map=16), 2)):
        assert lib.rkv_ragged_append(layout(**changes), 16, 16, 256, 128, 3, 16, None) == status
    assert lib.rkv_ragged_append(layout(), 16, 16, 256, 128, -3, 16, None) == 1
    assert lib.rkv_ragged_append(layout(), 16, 16, 256, 128, 3, None, None) == 1
    assert lib.rkv_ragged_append(layout(), None, None, 256, 128, 0, None, None) == 0

    def attend(lay=None, lengths=16, scale=0.0, ws=16, nbytes=None, q_changes=(), o_changes=()):
        lay = lay or layout()
        q = _lib.Query(16, 2, 8, 1, 1024, 128, 128)
        o = _lib.Output(16, 2, 0, 1024, 128, 128)
        for name, v in q_changes:
            setattr(q, name, v)
        for name, v in o_changes:
            setattr(o, name, v)
        if nbytes is None:
            nbytes = lib.rkv_ragged_decode_attention_workspace_size(q, lay)
        return lib.rkv_ragged_decode_attention(q, lay, lengths, None, scale, o, None, ws, nbytes, None)

    assert attend(lengths=None) == 1
    assert attend(scale=-1.0) == 1 and attend(scale=float("nan")) == 1
    assert attend(scale=float("inf")) == 1
    assert attend(ws=None) == 3 and attend(nbytes=64) == 3
    assert attend(q_changes=[("q_len", 2)]) == 2 and attend(q_changes=[("dtype", 1)]) == 2
    assert attend(q_changes=[("num_heads", 3)]) == 1 and attend(q_changes=[("q", None)]) == 1
    assert attend(o_changes=[("out", None)]) == 1 and attend(o_changes=[("dtype", 0)]) == 2
    assert attend(lay=layout(num_tokens=47)) == 1
    assert attend(lay=layout(page_table=None)) == 1
    assert attend(lay=layout(batch=-1)) == 1
    assert attend(lay=layout(batch=0)) == 0
    assert lib.rkv_ragged_error(0, ctypes.POINTER(_lib.c_i32)()) == 1


def test_error_codes_have_a_text():
    assert set(_lib.DEVICE_ERRORS) >= {1, 2, 3, 4}
    assert "refused" in str(_lib.DeviceError(4))


def test_check_reads_only_devices_that_ran_a_ragged_operator(monkeypatch):
    from razorkv_b200.kernels import Workspace, check_device_errors
    seen = []
    monkeypatch.setattr(Workspace, "_pool", {})
    monkeypatch.setattr(Workspace, "_retired", {})
    monkeypatch.setattr(_lib, "ragged_devices", lambda: [1])
    monkeypatch.setattr(_lib, "ragged_error", lambda dev, clear: seen.append((dev, clear)) or 3)
    with pytest.raises(_lib.DeviceError) as e:
        check_device_errors()
    assert e.value.code == 3 and seen == [(1, True)]
    check_device_errors(torch.device("cuda", 0))
    assert len(seen) == 1
