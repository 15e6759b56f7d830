"""Limits of the ragged operators: inconsistent rings, and what calls share (GPU)."""

import pytest
import torch

import razorkv_b200 as R
from razorkv_b200._lib import DeviceError
from razorkv_b200.kernels import check_device_errors

pytestmark = pytest.mark.gpu


def ints(*values):
    return torch.tensor(values, dtype=torch.int64, device="cuda")


def refused(code):
    with pytest.raises(DeviceError) as e:
        check_device_errors()
    assert e.value.code == code


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("most", [8, 5000])
def test_a_ring_without_room_for_what_comes_back(inplace, most):
    """Pages given back go behind the free ones, while pages are being taken from the front: the ring
    has to have room for them beside all that were free before the call."""
    check_device_errors()

    def call(count, n, m):
        ring, table = torch.arange(10, device="cuda"), torch.full((2, 4), 9, dtype=torch.int64, device="cuda")
        table[1, :3] = ints(6, 7, 8)
        n, state = ints(*n), ints(0, count, 0)
        before = ring.clone(), table.clone(), n.clone(), state.clone()
        t = R.ragged_page_tables(n, ints(*m), table, ring, state, 4, most, inplace=inplace)
        same = torch.equal(ring, before[0]) and torch.equal(table, before[1])
        kept = torch.equal(t.lengths, before[2]) and torch.equal(t.free_state, before[3])
        return t, ring, table, same and kept

    # 9 free, 2 taken, 3 back: entries 9, 0 and 1 would be written while 0 and 1 are read
    t, _, _, unchanged = call(9, (0, 12), (8, 0))
    refused(4)
    assert unchanged and t.slot_map.tolist() == [-1] * most and t.token_starts.tolist() == [0, 0, 0]
    # 8 free, 2 taken, 2 back: exactly as many as there is room for
    t, ring, table, _ = call(8, (0, 12), (8, 4))
    check_device_errors()
    assert t.free_state.tolist() == [2, 8, 0] and table.tolist() == [[0, 1, 9, 9], [6, 7, 8, 9]]
    assert ring.tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 7, 8]
    assert t.slot_map.tolist() == list(range(8)) + [-1] * (most - 8)


def test_requests_that_share_pages_and_both_leave():
    """Two rows with the same pages would bring each back twice: refused where the ring shows it."""
    check_device_errors()
    ring, state = R.ragged_free_ring(6, "cuda")
    table = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    t = R.ragged_page_tables(ints(0, 0), ints(12, 0), table, ring, state, 4, 12)
    table[1] = table[0]
    t = R.ragged_page_tables(ints(12, 12), ints(0, 0), table, ring, t.free_state, 4, 0)
    refused(4)
    assert t.lengths.tolist() == [12, 12] and t.free_state.tolist() == [3, 3, 0]


def test_a_page_outside_the_pool_comes_back():
    """It is reported by the call that gives it back, not only by the one that takes it again."""
    check_device_errors()
    ring, table = torch.arange(6, device="cuda"), ints(2, 6, 3, -1).reshape(2, 2)
    t = R.ragged_page_tables(ints(8, 4), ints(4, 4), table, ring, ints(0, 2, 0), 4, 0)
    refused(2)
    assert t.lengths.tolist() == [4, 4] and t.free_state.tolist() == [0, 3, 0]
    R.ragged_page_tables(ints(4, 4), ints(0, 0), table, ring, t.free_state, 4, 0)
    check_device_errors()       # (an entry behind a request's pages is not looked at)
