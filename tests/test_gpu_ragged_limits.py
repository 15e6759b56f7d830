"""Limits of the ragged operators: inconsistent rings, and what calls share (GPU)."""

from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

import razorkv_b200 as R
from razorkv_b200 import _lib
from razorkv_b200._lib import DeviceError
from razorkv_b200.kernels import check_device_errors
from tests.test_gpu_ragged import _pool_case

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


def test_one_workspace_for_dense_and_ragged_calls():
    """Every call of the library keeps to a workspace's header: zero at first, and zero after it."""
    lib = _lib.load()
    g = torch.Generator(device="cuda").manual_seed(1)
    B, Hq, Hkv, P, W, D = 2, 8, 2, 16, 40, 128
    kp, vp = (torch.randn(B * W, Hkv, P, D, generator=g, device="cuda").bfloat16() for _ in "kv")
    q = torch.randn(B, Hq, 1, D, generator=g, device="cuda").bfloat16()
    table, n = torch.arange(B * W, device="cuda").reshape(B, W), ints(W * P, 77)
    want = R.ragged_decode_attention(q, kp, vp, table, n)
    # the same rows as a dense cache [B, Hkv, T, D]
    k, v = (t.reshape(B, W, Hkv, P, D).transpose(1, 2).reshape(B, Hkv, W * P, D).contiguous() for t in (kp, vp))
    dense = _lib.KVLayout(k=k.data_ptr(), v=v.data_ptr(), dtype=_lib.dtype_code(q.dtype), head_dim=D, batch=B,
                          num_kv_heads=Hkv, stride_b=Hkv * W * P * D, stride_h=W * P * D, stride_t=D,
                          num_tokens=W * P)
    pool = _lib.KVLayout(k=kp.data_ptr(), v=vp.data_ptr(), dtype=_lib.dtype_code(q.dtype), head_dim=D, batch=B,
                         num_kv_heads=Hkv, stride_h=P * D, stride_p=Hkv * P * D, stride_t=D, page_size=P,
                         num_slots=B * W, page_table=table.data_ptr(), pt_stride_b=W, num_tokens=W * P)
    out, again = torch.empty_like(q), torch.empty_like(q)
    qs = _lib.Query(q.data_ptr(), _lib.dtype_code(q.dtype), Hq, 1, Hq * D, D, D)
    size = max(lib.rkv_decode_attention_workspace_size(qs, dense),
               lib.rkv_ragged_decode_attention_workspace_size(qs, pool))
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    first = None
    for _ in range(3):
        o = _lib.Output(out.data_ptr(), _lib.dtype_code(q.dtype), 0, Hq * D, D, D)
        assert lib.rkv_ragged_decode_attention(qs, pool, n.data_ptr(), None, 0.0, o, None, ws.data_ptr(), size,
                                               stream) == 0
        assert torch.equal(out, want)
        assert int(ws[:65536].count_nonzero()) == 0
        o = _lib.Output(again.data_ptr(), _lib.dtype_code(q.dtype), 0, Hq * D, D, D)
        assert lib.rkv_decode_attention(qs, dense, 0.0, 0, o, ws.data_ptr(), size, stream) == 0
        assert int(ws[:65536].count_nonzero()) == 0
        first = again.clone() if first is None else first
        assert torch.equal(again, first)
    # request 0 has all its tokens in both
    assert torch.allclose(first[0].float(), want[0].float(), atol=2e-2, rtol=1e-2)
    check_device_errors()


def test_the_check_waits_for_its_own_stream_only():
    """Work of another stream (half a second of it) goes on while the errors are read."""
    check_device_errors()
    R.ragged_append(torch.ones(1, 1, 8, device="cuda"), torch.ones(1, 1, 8, device="cuda"),
                    torch.zeros(1, 1, 4, 8, device="cuda"), torch.zeros(1, 1, 4, 8, device="cuda"), ints(4))
    other, done = torch.cuda.Stream(), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        torch.cuda._sleep(1_000_000_000)
        done.record()
    refused(2)
    check_device_errors()       # read and cleared
    busy = not done.query()
    torch.cuda.synchronize()
    assert busy


@pytest.mark.parametrize("mode", [torch.inference_mode, torch.no_grad, torch.enable_grad])
def test_results_are_ordinary_tensors(mode):
    """The step's five results lie on two allocations: each can be written, viewed and kept alone."""
    with mode():
        ring, state = R.ragged_free_ring(8, "cuda")
        table = torch.zeros(2, 4, dtype=torch.int64, device="cuda")
        t = R.ragged_page_tables(ints(0, 0), ints(5, 3), table, ring, state, 4, 10)
        want = [x.clone() for x in t]
        for i, x in enumerate(t):
            assert x.is_contiguous() and not x.requires_grad and x.is_inference() == (mode is torch.inference_mode)
            x.add_(1000 + i)
            assert all(torch.equal(y, w if j != i else w + 1000 + i) for j, (y, w) in enumerate(zip(t, want)))
            x.copy_(want[i])
        kp, vp = torch.zeros(2, 8, 2, 4, 8, device="cuda").unbind(0)
        rows = torch.ones(10, 2, 8, device="cuda", requires_grad=mode is torch.enable_grad)
        R.ragged_append(rows, rows, kp, vp, t.slot_map)
        q = torch.zeros(2, 4, 1, 8, device="cuda", requires_grad=mode is torch.enable_grad)
        out, lse = R.ragged_decode_attention(q, kp, vp, table, t.lengths, return_lse=True)
        assert not out.requires_grad and bool((out == 1).all())
        assert lse.exp().round().tolist() == [[5.0] * 4, [3.0] * 4]
    check_device_errors()


def test_calls_from_several_host_threads():
    """Threads that never made a CUDA call, each on a stream of its own, all at the same time."""
    cases = [_pool_case([n, 1, n // 3], 8, 2, 128, 16, torch.bfloat16, seed=n) for n in (300, 2000, 9000, 40)]
    want = [R.ragged_decode_attention(*c[:5], return_lse=True) for c in cases]
    torch.cuda.synchronize()

    def work(case):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [R.ragged_decode_attention(*case[:5], return_lse=True) for _ in range(50)]
            torch.cuda.current_stream().synchronize()
        return got

    with ThreadPoolExecutor(len(cases)) as pool:
        for got, (out, lse) in zip(pool.map(work, cases), want):
            assert all(torch.equal(a, out) and torch.equal(b, lse) for a, b in got)
