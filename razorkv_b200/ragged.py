"""Operators for requests of different lengths that share one page pool.

The cache (``PagedRazorKVCache``) and ``paged_sparse_attention`` hold one length for the whole
batch.  A server admits and retires requests one by one: each has its own length, the lengths
live on the GPU, and all of them take pages of one pool.  Per step and model,

* ``ragged_page_tables`` turns the requests' lengths into page tables and a slot map, taking
  pages from a ring of free pages and giving them back;

and per layer, over that layer's pools ``[num_slots, Hkv, P, D]``,

* ``ragged_append`` writes the new tokens' K/V rows through the slot map, and
* ``ragged_decode_attention`` attends one new token per request over its pages.

None of them reads anything back or needs a length on the host, so a step can be captured into
a CUDA graph; none differentiates.  What they find wrong on the device is raised by
``check_device_errors`` at the caller's next sync point.  They are registered as
``torch.ops.razorkv.ragged_*`` too.
"""

import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib
from ._lib import KVLayout, Output, Query, check, dtype_code, require_cuda

__all__ = [
    "RaggedTables",
    "ragged_append",
    "ragged_decode_attention",
    "ragged_free_ring",
    "ragged_page_tables",
]


class RaggedTables(NamedTuple):
    """What ``ragged_page_tables`` returns (int64 device tensors)."""

    lengths: torch.Tensor        # [R] tokens of each request after the step
    slot_map: torch.Tensor       # [max_new_tokens] pool slot of each new token, -1 past the last
    positions: torch.Tensor      # [max_new_tokens] its position in its request
    token_starts: torch.Tensor   # [R + 1] first new token of each request
    free_state: torch.Tensor     # [3] state of the ring of free pages


def _device_of(*tensors) -> int:
    """Index of the CUDA device that all tensors (None aside) are on."""
    index = tensors[0].get_device()     # -1 on the CPU
    for t in tensors:
        if t is not None and (t.get_device() != index or index < 0):
            require_cuda(*tensors)
            raise ValueError("tensors on different devices: "
                             + ", ".join(sorted({str(t.device) for t in tensors if t is not None})))
    return index


def _launch(index: int, what: str, entry, *args):
    """Calls a C entry with the current stream of device `index`, which is made current."""
    _lib.ragged_devices.add(index)
    if index == torch.cuda.current_device():
        st = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            st = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    check(st, what)


def _int64(name: str, t: torch.Tensor, dim: int):
    if t.dtype != torch.int64:
        raise TypeError(f"{name} must be int64, got {t.dtype}")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimension(s), got {tuple(t.shape)}")


def _written(name: str, t: torch.Tensor):
    """A tensor that is updated in place cannot be copied into shape first."""
    if t.numel() and not t.is_contiguous():
        raise ValueError(f"{name} is updated in place and must be contiguous")


def ragged_free_ring(num_slots: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
    """(ring, state) of a pool whose ``num_slots`` pages are all free, for
    ``ragged_page_tables``."""
    if num_slots < 1:
        raise ValueError(f"num_slots must be positive, got {num_slots}")
    ring = torch.arange(num_slots, dtype=torch.int64, device=device)
    return ring, torch.tensor([0, num_slots, 0], dtype=torch.int64, device=device)


def ragged_page_tables(
    lengths: torch.Tensor,
    new_lengths: torch.Tensor,
    page_table: torch.Tensor,
    free_ring: torch.Tensor,
    free_state: torch.Tensor,
    page_size: int,
    max_new_tokens: int,
    inplace: bool = False,
) -> RaggedTables:
    """Page tables and slot map of a step in which request r goes from ``lengths[r]`` to
    ``new_lengths[r]`` tokens.

    lengths, new_lengths [R]; page_table [R, W]; free_ring [num_slots] and free_state [3] as
    ``ragged_free_ring`` makes them; all int64.  A request that grows takes the pages it lacks
    from the ring, in request order, and has them entered in its row of ``page_table``; one
    that shrinks gives the pages behind its new end back (``new_lengths[r] == 0``: it leaves),
    to be taken from the next call on.  Entries past a request's pages stay as they are.  The
    new tokens' slots come request by request in ``slot_map``, which holds ``max_new_tokens``
    entries, so that a captured step can serve any number of new tokens up to that.

    The step is granted as a whole or refused as a whole (pages missing, more than
    ``max_new_tokens`` new tokens, a length outside [0, W * page_size]): refused, the returned
    lengths are ``lengths``, every slot is -1 and ``check_device_errors`` raises.

    ``page_table`` and ``free_ring`` are updated in place.  ``lengths`` and ``free_state`` are
    not unless ``inplace`` is set: the returned ones then ARE those tensors, updated.  Two
    calls on one ring must not overlap."""
    index = _device_of(lengths, new_lengths, page_table, free_ring, free_state)
    _int64("lengths", lengths, 1)
    _int64("new_lengths", new_lengths, 1)
    _int64("page_table", page_table, 2)
    _int64("free_ring", free_ring, 1)
    _int64("free_state", free_state, 1)
    R, W = page_table.shape
    if lengths.shape[0] != R or new_lengths.shape[0] != R:
        raise ValueError(f"lengths and new_lengths must be [{R}] like page_table's rows, got "
                         f"{tuple(lengths.shape)} and {tuple(new_lengths.shape)}")
    slots = free_ring.shape[0]
    if free_state.shape[0] != 3 or slots < 1:
        raise ValueError("free_state must be [3] and free_ring [num_slots], as ragged_free_ring makes them")
    if page_size < 1 or max_new_tokens < 0:
        raise ValueError(f"page_size {page_size} and max_new_tokens {max_new_tokens} must be positive")
    _written("page_table", page_table)
    _written("free_ring", free_ring)
    _written("free_state", free_state)
    if inplace:
        _written("lengths", lengths)
    n, m = lengths.contiguous(), new_lengths.contiguous()
    slot_map, positions = n.new_empty(max_new_tokens), n.new_empty(max_new_tokens)
    starts = n.new_empty(R + 1)
    after, state = (lengths, free_state) if inplace else (n.new_empty(R), n.new_empty(3))
    _launch(index, "rkv_ragged_page_tables", _lib.load().rkv_ragged_page_tables,
            n.data_ptr(), m.data_ptr(), R, page_size, page_table.data_ptr(), W, W,
            free_ring.data_ptr(), slots, free_state.data_ptr(), after.data_ptr(),
            state.data_ptr(), slot_map.data_ptr(), positions.data_ptr(), max_new_tokens,
            starts.data_ptr())
    return RaggedTables(after, slot_map, positions, starts, state)


def _pool_layout(key_pool, value_pool, batch, table, capacity) -> KVLayout:
    if key_pool.dim() != 4 or value_pool.shape != key_pool.shape:
        raise ValueError("key_pool and value_pool must both be [num_slots, Hkv, P, D], got "
                         f"{tuple(key_pool.shape)} and {tuple(value_pool.shape)}")
    if key_pool.dtype != value_pool.dtype:
        raise TypeError("key_pool and value_pool must share a dtype")
    stride = key_pool.stride()
    if value_pool.stride() != stride or stride[3] != 1:
        raise ValueError("key_pool and value_pool must share their strides, with contiguous rows")
    slots, heads, page, dim = key_pool.shape
    if not (slots and heads and page and dim):
        raise ValueError(f"the pool has an empty dimension: {tuple(key_pool.shape)}")
    return KVLayout(key_pool.data_ptr(), value_pool.data_ptr(), dtype_code(key_pool.dtype), dim,
                    batch, heads, 0, stride[1], stride[0], stride[2], page, slots,
                    table.data_ptr() if table is not None else None,
                    table.stride(0) if table is not None else 0, capacity, None)


def ragged_append(
    key: torch.Tensor,
    value: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    slot_map: torch.Tensor,
) -> None:
    """Writes row t of key / value [T, Hkv, D] to slot ``slot_map[t]`` (int64 [T]) of the pools
    [num_slots, Hkv, P, D]: row ``slot % P`` of page ``slot // P``.

    Negative slots are skipped (a padded tail); one past the pool is skipped and raised by
    ``check_device_errors``.  Rows of one slot must not repeat: either may be the one left."""
    index = _device_of(key, value, key_pool, value_pool, slot_map)
    _int64("slot_map", slot_map, 1)
    lay = _pool_layout(key_pool, value_pool, 0, None, 0)
    T = slot_map.shape[0]
    if key.shape != (T, lay.num_kv_heads, lay.head_dim) or value.shape != key.shape:
        raise ValueError(f"key and value must be [{T}, {lay.num_kv_heads}, {lay.head_dim}], got "
                         f"{tuple(key.shape)} and {tuple(value.shape)}")
    if key.dtype != key_pool.dtype or value.dtype != key_pool.dtype:
        raise TypeError(f"key and value must have the pool's dtype {key_pool.dtype}")
    if T == 0:
        return
    k = key if key.stride(2) == 1 else key.contiguous()
    v = value if value.stride(2) == 1 else value.contiguous()
    if k.stride() != v.stride():
        k, v = k.contiguous(), v.contiguous()
    slots = slot_map.contiguous()
    _launch(index, "rkv_ragged_append", _lib.load().rkv_ragged_append, lay, k.data_ptr(),
            v.data_ptr(), k.stride(0), k.stride(1), T, slots.data_ptr())


def ragged_decode_attention(
    query: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    scale: Optional[float] = None,
    starts: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    out: Optional[torch.Tensor] = None,
    validate: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of one new token per request over its pages.

    query [B, H, 1, D]; key_pool / value_pool [num_slots, Hkv, P, D]; page_table [B, W] and
    lengths [B] int64: request b attends its tokens ``starts[b] <= t < lengths[b]`` (from the
    first where ``starts`` is None; a sliding window or left padding otherwise), token t in
    row ``t % P`` of page ``page_table[b, t // P]``.  Returns [B, H, 1, D] in the query's dtype
    (in ``out`` where given), and with ``return_lse`` also log sum exp(scale * q . k) as fp32
    [B, H].  A request without such a token (a padded batch) gives zeros and -inf, and what the
    pool holds elsewhere has no effect.  ``scale`` defaults to 1 / sqrt(D).

    Lengths outside [0, W * P] and page ids outside the pool are kept inside them and raised by
    ``check_device_errors``; ``validate`` checks them on the host first (one device sync)."""
    index = _device_of(query, key_pool, value_pool, page_table, lengths, starts, out)
    if query.dim() != 4:
        raise ValueError(f"query must be [B, H, 1, D], got {tuple(query.shape)}")
    B, H, q_len, D = query.shape
    assert q_len == 1, "ragged decode attention is defined for single-token decoding (q_len == 1)."
    _int64("page_table", page_table, 2)
    _int64("lengths", lengths, 1)
    if starts is not None:
        _int64("starts", starts, 1)
    table = page_table if page_table.stride(1) == 1 else page_table.contiguous()
    rows, W = table.shape
    lay = _pool_layout(key_pool, value_pool, B, table, W * key_pool.shape[2])
    if lay.head_dim != D:
        raise ValueError(f"the pool's head_dim {lay.head_dim} is not the query's {D}")
    if H < 1 or H % lay.num_kv_heads:
        raise ValueError(f"num_heads {H} is not a multiple of num_kv_heads {lay.num_kv_heads}")
    if query.dtype != key_pool.dtype:
        raise TypeError(f"query {query.dtype} and pool {key_pool.dtype} must share a dtype")
    if rows != B or lengths.shape[0] != B or (starts is not None and starts.shape[0] != B):
        raise ValueError(f"page_table, lengths and starts must have one row per request ({B})")
    if scale is not None and not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if out is None:
        out = query.new_empty((B, H, 1, D))
    elif out.shape != query.shape or out.dtype != query.dtype or out.stride(3) != 1:
        raise ValueError("out must have the query's shape and dtype, with contiguous rows")
    elif B and out.data_ptr() == query.data_ptr():
        raise ValueError("out must not be the query")
    lse = query.new_empty((B, H), dtype=torch.float32) if return_lse else None
    if B == 0:
        return (out, lse) if return_lse else out
    # rows of 16-byte steps, as the vector kernels read them
    q, (sb, sh, st, sd), step = query, query.stride(), 16 // query.element_size()
    if sd != 1 or sb % step or sh % step or q.data_ptr() & 15:
        q = query.new_empty((B, H, 1, D)).copy_(query)
        sb, sh, st, _ = q.stride()
    n = lengths.contiguous()
    first = starts.contiguous() if starts is not None else None
    if validate:
        _validate(table, n, lay)
    qs = Query(q.data_ptr(), lay.dtype, H, 1, sb, sh, st)
    sb, sh, st, _ = out.stride()
    os_ = Output(out.data_ptr(), lay.dtype, 0, sb, sh, st)
    lib = _lib.load()
    nbytes = lib.rkv_ragged_decode_attention_workspace_size(qs, lay)
    # of the caching allocator, so that each call and each captured graph has its own
    ws = query.new_empty(nbytes, dtype=torch.uint8)
    _launch(index, "rkv_ragged_decode_attention", lib.rkv_ragged_decode_attention, qs, lay,
            n.data_ptr(), first.data_ptr() if first is not None else None,
            scale if scale is not None else 0.0, os_, lse.data_ptr() if lse is not None else None,
            ws.data_ptr(), nbytes)
    return (out, lse) if return_lse else out


def _validate(table: torch.Tensor, lengths: torch.Tensor, lay: KVLayout):
    P, capacity = lay.page_size, lay.num_tokens
    lo, hi = int(lengths.min()), int(lengths.max())
    if lo < 0 or hi > capacity:
        raise IndexError(f"lengths must lie in [0, {capacity}], got [{lo}, {hi}]")
    used = torch.arange(table.shape[1], device=table.device)[None] * P < lengths[:, None]
    if bool((used & ((table < 0) | (table >= lay.num_slots))).any()):
        raise IndexError(f"page_table entries must lie in [0, {lay.num_slots})")


# ---- torch.ops.razorkv registration ---------------------------------------------------------
def _register_ops():
    lib = torch.library.Library("razorkv", "FRAGMENT")
    lib.define("ragged_page_tables(Tensor lengths, Tensor new_lengths, Tensor(a!) page_table, "
               "Tensor(b!) free_ring, Tensor free_state, int page_size, int max_new_tokens) -> "
               "(Tensor lengths, Tensor slot_map, Tensor positions, Tensor token_starts, "
               "Tensor free_state)")
    lib.define("ragged_append(Tensor key, Tensor value, Tensor(a!) key_pool, "
               "Tensor(b!) value_pool, Tensor slot_map) -> ()")
    lib.define("ragged_decode_attention(Tensor query, Tensor key_pool, Tensor value_pool, "
               "Tensor page_table, Tensor lengths, float scale=0.0, Tensor? starts=None) -> "
               "(Tensor out, Tensor lse)")

    def _tables(lengths, new_lengths, page_table, free_ring, free_state, page_size, max_new_tokens):
        return tuple(ragged_page_tables(lengths, new_lengths, page_table, free_ring, free_state,
                                        page_size, max_new_tokens))

    def _tables_meta(lengths, new_lengths, page_table, free_ring, free_state, page_size,
                     max_new_tokens):
        e = lengths.new_empty
        return (e(lengths.shape[0]), e(max_new_tokens), e(max_new_tokens),
                e(lengths.shape[0] + 1), e(3))

    def _decode(query, key_pool, value_pool, page_table, lengths, scale=0.0, starts=None):
        return ragged_decode_attention(query, key_pool, value_pool, page_table, lengths,
                                       scale or None, starts, return_lse=True)

    def _decode_meta(query, key_pool, value_pool, page_table, lengths, scale=0.0, starts=None):
        return (query.new_empty(query.shape),
                query.new_empty(query.shape[:2], dtype=torch.float32))

    lib.impl("ragged_page_tables", _tables, "CUDA")
    lib.impl("ragged_append", ragged_append, "CUDA")
    lib.impl("ragged_decode_attention", _decode, "CUDA")
    lib.impl("ragged_page_tables", _tables_meta, "Meta")
    lib.impl("ragged_append", lambda *args: None, "Meta")
    lib.impl("ragged_decode_attention", _decode_meta, "Meta")
    return lib


try:
    _TORCH_LIBRARY = _register_ops()
except RuntimeError:   # already registered in this process
    _TORCH_LIBRARY = None
