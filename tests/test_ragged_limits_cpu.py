"""Limits of the ragged operators that are found before any CUDA call (CPU)."""

import pytest
import torch

import razorkv_b200 as R
from razorkv_b200 import _lib


def test_workspace_alignment():
    lib = _lib.load()
    pool = _lib.KVLayout(k=16, v=16, dtype=2, head_dim=128, batch=2, num_kv_heads=2, stride_h=2048,
                         stride_p=4096, stride_t=128, page_size=16, num_slots=7, page_table=16,
                         pt_stride_b=3, num_tokens=48)
    q, o = _lib.Query(16, 2, 8, 1, 1024, 128, 128), _lib.Output(16, 2, 0, 1024, 128, 128)
    size = lib.rkv_ragged_decode_attention_workspace_size(q, pool)
    for at in (8, 24, 1):
        assert lib.rkv_ragged_decode_attention(q, pool, 16, None, 0.0, o, None, at, size, None) == 5


def _attend(lengths, starts, table, **changes):
    """A call that ends at the device (its tensors are on the CPU), unless its values are refused."""
    return R.ragged_decode_attention(
        torch.zeros(len(lengths), 4, 1, 8), torch.zeros(5, 2, 4, 8), torch.zeros(5, 2, 4, 8),
        torch.tensor(table), torch.tensor(lengths), starts=torch.tensor(starts), validate=True, **changes)


def test_validation_looks_at_the_pages_of_the_window():
    # pages in front of the window were given back; requests without a token in their window use none
    for lengths, starts, table in (([12, 5], [4, 0], [[-1, 1, 2], [3, 4, 9]]),
                                   ([12, 5], [8, 4], [[-1, -1, 2], [9, 4, 9]]),
                                   ([12, 5], [11, 5], [[9, 9, 0], [9, 9, 9]]),
                                   ([12, 5], [1 << 40, 7], [[9, 9, 9], [9, 9, 9]])):
        with pytest.raises(RuntimeError, match="CUDA"):
            _attend(lengths, starts, table)
    for starts, table in (([3, 0], [[-1, 1, 2], [3, 4, 9]]), ([4, 0], [[-1, 1, 5], [3, 4, 9]]),
                          ([4, 4], [[-1, 1, 2], [3, 9, 9]])):
        with pytest.raises(IndexError, match="page_table"):
            _attend([12, 5], starts, table)


def test_validation_refuses_negative_starts():
    with pytest.raises(IndexError, match="starts"):
        _attend([12, 5], [4, -1], [[0, 1, 2], [3, 4, 0]])
    with pytest.raises(RuntimeError, match="CUDA"):
        _attend([12, 5], [4, 0], [[0, 1, 2], [3, 4, 0]])


def test_the_binding_is_the_one_of_this_torch(monkeypatch):
    """A binary of another torch version, whose C++ interface may differ, is not loaded."""
    monkeypatch.setattr(_lib, "_ragged", None)
    monkeypatch.setattr(torch, "__version__", "1.0.0+other")
    with pytest.raises(ImportError, match="razorkv_b200.build"):
        _lib.ragged()
    monkeypatch.undo()
    assert _lib.ragged().devices() == 0 or torch.cuda.is_available()


def test_token_counts_beyond_64_bits_are_refused():
    """The step's sums are 64-bit numbers: all requests' tables together have room for fewer tokens."""
    lib = _lib.load()

    def call(requests, width, page):
        return lib.rkv_ragged_page_tables(16, 16, requests, page, 16, width, width, 16, 1, 16, 16, 16, 16, 16, 8,
                                          16, None)

    for requests, width, page in ((4, 2, 1 << 61), (3, 1, 1 << 62), (1 << 22, 5, 1 << 40)):
        assert call(requests, width, page) == 1


def test_scales_whose_exponent_overflows_are_refused():
    """Weights are powers of two of scale * log2 e, which has to be a number too."""
    q, pool, table = torch.zeros(2, 4, 1, 8), torch.zeros(5, 2, 4, 8), torch.zeros(2, 3, dtype=torch.int64)
    call = lambda scale: R.ragged_decode_attention(q, pool, pool, table, torch.tensor([1, 7]), scale)  # noqa: E731
    for scale in (2.4e38, 3.4e38):
        with pytest.raises(ValueError, match="scale"):
            call(scale)
    with pytest.raises(RuntimeError, match="CUDA"):
        call(2.3e38)
    lib = _lib.load()
    lay = _lib.KVLayout(k=16, v=16, dtype=2, head_dim=128, batch=2, num_kv_heads=2, stride_h=2048,
                        stride_p=4096, stride_t=128, page_size=16, num_slots=7, page_table=16,
                        pt_stride_b=3, num_tokens=48)
    qs, o = _lib.Query(16, 2, 8, 1, 1024, 128, 128), _lib.Output(16, 2, 0, 1024, 128, 128)
    assert lib.rkv_ragged_decode_attention(qs, lay, 16, None, 3e38, o, None, None, 0, None) == 1


def test_buffers_that_are_written_must_not_overlap():
    """Rows that lie on one another, or on what the call reads, would be written in any order."""
    table, n = torch.zeros(2, 3, dtype=torch.int64), torch.tensor([1, 7])
    pool, q = torch.zeros(5, 2, 4, 8), torch.zeros(2, 4, 1, 8)
    both = torch.zeros(2 * 4 * 8 + 8)
    joint = torch.zeros(2, 12, 1, 8)       # queries and outputs in columns of one tensor: apart
    for query, out, ok in ((q, torch.zeros(1, 4, 1, 8).expand(2, 4, 1, 8), False),
                           (q, torch.zeros(2, 1, 1, 8).expand(2, 4, 1, 8), False),
                           (both[:64].view(2, 4, 1, 8), both[8:].view(2, 4, 1, 8), False),
                           (q, pool.view(-1)[:64].view(2, 4, 1, 8), False),
                           (joint[:, :4], joint[:, 8:], True)):
        with pytest.raises(RuntimeError if ok else ValueError, match="CUDA" if ok else "out"):
            R.ragged_decode_attention(query, pool, pool, table, n, out=out)
    rows, slots = torch.zeros(3, 2, 8), torch.tensor([0, 5, -1])
    pair = torch.zeros(5, 2, 2, 4, 8)      # K and V of a page side by side: apart
    for kp, vp, ok in ((pool, pool, False), (torch.zeros(1, 2, 4, 8).expand(5, 2, 4, 8),
                                             torch.zeros(1, 2, 4, 8).expand(5, 2, 4, 8), False),
                       (pair[:, 0], pair[:, 1], True), (pool, torch.zeros_like(pool), True)):
        with pytest.raises(RuntimeError if ok else ValueError, match="CUDA" if ok else "pool"):
            R.ragged_append(rows, rows, kp, vp, slots)


def test_meta_shapes_of_the_torch_ops():
    i = lambda *shape: torch.empty(*shape, dtype=torch.int64, device="meta")  # noqa: E731
    got = torch.ops.razorkv.ragged_page_tables(i(3), i(3), i(3, 7), i(20), i(3), 16, 40)
    assert [tuple(t.shape) for t in got] == [(3,), (40,), (40,), (4,), (3,)]
    assert all(t.dtype == torch.int64 and t.device.type == "meta" for t in got)
    x = lambda *shape: torch.empty(*shape, dtype=torch.bfloat16, device="meta")  # noqa: E731
    assert torch.ops.razorkv.ragged_append(x(4, 2, 8), x(4, 2, 8), x(9, 2, 16, 8), x(9, 2, 16, 8), i(4)) is None
    out, lse = torch.ops.razorkv.ragged_decode_attention(x(3, 4, 1, 8), x(9, 2, 16, 8), x(9, 2, 16, 8), i(3, 7), i(3))
    assert out.shape == (3, 4, 1, 8) and out.dtype == torch.bfloat16
    assert lse.shape == (3, 4) and lse.dtype == torch.float32
