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

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib

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
    ``max_new_tokens`` new tokens, a length outside [0, W * page_size], more pages coming back
    than the ring has room for beside its free ones): refused, the returned lengths are
    ``lengths``, every slot is -1 and ``check_device_errors`` raises.  Every page must belong to
    one request here; rows that share pages, which the attention takes, would each give them back.

    ``page_table`` and ``free_ring`` are updated in place.  ``lengths`` and ``free_state`` are
    not unless ``inplace`` is set: the returned ones then ARE those tensors, updated.  Two
    calls on one ring must not overlap."""
    return RaggedTables(*_lib.ragged().tables(lengths, new_lengths, page_table, free_ring,
                                              free_state, page_size, max_new_tokens, inplace))


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
    ``check_device_errors``.  A slot must not repeat: what is left there may be pieces of both rows."""
    _lib.ragged().append(key, value, key_pool, value_pool, slot_map)


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
    (in ``out`` where given, which must not overlap what is read), and with ``return_lse`` also
    log sum exp(scale * q . k) as fp32 [B, H].  A request without such a token (a padded batch) gives zeros and -inf, and what the
    pool holds elsewhere has no effect; infinities and NaN in attended rows take the formula's
    way into the output (an infinite element of V makes its column infinite, or NaN where both
    signs meet).  ``scale`` defaults to 1 / sqrt(D).

    Lengths outside [0, W * P], negative starts and page ids of attended tokens outside the pool
    are kept inside and raised by ``check_device_errors``; ``validate`` checks them on the host
    first (a few device syncs)."""
    return _lib.ragged().decode(query, key_pool, value_pool, page_table, lengths, scale, starts,
                                return_lse, out, validate)


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
