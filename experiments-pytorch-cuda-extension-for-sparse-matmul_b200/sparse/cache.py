"""Paged key / value cache: writing, reading, and the places of tokens.

The reference has no cached inference.  A cache is two tensors ``keys`` and
``values`` ``[pages, heads, page, head_dim]`` (page 16, 32, 64 or 128 -- the block
sizes of this package; head dimension 64 or 128).  It holds the tokens' own
16-bit type, or ``float8_e4m3fn`` codes with two float32 tensors
``key_scales`` and ``value_scales`` ``[pages, heads, page]``:

    a = max(max_d |x_d|, 2^-100)    scale = a / 448    code_d = e4m3(x_d * (448 / a))

so a stored value is ``code * scale``, within 2^-4 of itself or 2^-10 / 448 of the row's
largest magnitude.  A row that holds an infinity or a NaN reads back as NaN.  Scales that another program made may be any
finite number; those of a new cache are 0, so a place that was never written holds zeros.

A token lives at ``slot = page_id * page + place``.  A sequence's pages are a
row of a page table; ``cache_slots`` turns positions of sequences into slots.
A negative slot is skipped (written nowhere, read as zeros); one behind the
cache's end is skipped too and reported through ``check_device_status``.  The
non-negative slots of one write must differ: two tokens written to one slot
leave a row that mixes both (``kernel.debug_checks`` raises instead).

Serving only: no derivative passes through a cache.  Tokens that require grad may be
written (their numbers are kept, as those of a detached tensor); a cache that requires
grad is not read, and forward-mode derivatives are refused.
"""
from typing import NamedTuple, Optional, Tuple

import torch

from . import kernel


class Cache(NamedTuple):
    """The tensors of one layer's cache, in the order the cache operators take them."""
    keys: torch.Tensor
    values: torch.Tensor
    key_scales: Optional[torch.Tensor] = None
    value_scales: Optional[torch.Tensor] = None


def refuse_gradient(op: str, *tensors: Optional[torch.Tensor]) -> None:
    """Serving operators compute no gradient: asking for one is refused, not ignored."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("%s has no gradient: call it under torch.no_grad()" % op)


def make_cache(pages: int, page: int, heads: int, head_dim: int, dtype: torch.dtype, device=None) -> Cache:
    """An empty cache; ``dtype`` float16, bfloat16 or float8_e4m3fn."""
    if dtype not in (torch.float16, torch.bfloat16, torch.float8_e4m3fn):
        raise ValueError("a cache holds float16, bfloat16 or float8_e4m3fn, not %s" % (dtype,))
    if page not in (16, 32, 64, 128) or head_dim not in (64, 128):
        raise ValueError("page must be 16, 32, 64 or 128 and head_dim 64 or 128, got %r and %r" % (page, head_dim))
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    keys, values = (torch.zeros(pages, heads, page, head_dim, dtype=torch.uint8 if dtype == torch.float8_e4m3fn else dtype,
                                device=device) for _ in range(2))
    if dtype != torch.float8_e4m3fn:
        return Cache(keys, values)
    key_scales, value_scales = (torch.zeros(pages, heads, page, dtype=torch.float32, device=device) for _ in range(2))
    return Cache(keys.view(dtype), values.view(dtype), key_scales, value_scales)


def cache_slots(table: torch.Tensor, sequences: torch.Tensor, positions: torch.Tensor, page: int) -> torch.Tensor:
    """Slots (int64) of ``positions`` of ``sequences`` (broadcast together, flattened): sequence ``s`` has its pages in
    row ``s`` of ``table`` ``[sequences, pages]``.  -1 where the sequence is none of the table's, the position is negative
    or behind the table's end, or the table holds a negative page."""
    sequences, positions = torch.broadcast_tensors(sequences, positions)
    sequences, positions = sequences.reshape(-1).long(), positions.reshape(-1).long()
    inside = (sequences >= 0) & (sequences < table.size(0)) & (positions >= 0) & (positions < table.size(1) * page)
    if table.numel() == 0:
        return torch.full_like(positions, -1)
    held = table.long()[torch.where(inside, sequences, 0), torch.where(inside, positions, 0) // page]
    return torch.where(inside & (held >= 0), held * page + positions % page, -1)


def cache_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                key_scales: Optional[torch.Tensor] = None, value_scales: Optional[torch.Tensor] = None) -> None:
    """Keys and values ``[tokens, heads, head_dim]`` of new tokens into ``slots`` ``[tokens]`` of the cache, in place."""
    if kernel.debug_checks:
        real = slots[slots >= 0]
        if real.unique().numel() != real.numel():
            raise ValueError("the slots of one write must differ")
    kernel.sparse_ops.cache_write(k, v, slots, keys, values, key_scales, value_scales)
    kernel.check(keys)


def cache_read(slots: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, key_scales: Optional[torch.Tensor] = None,
               value_scales: Optional[torch.Tensor] = None,
               dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values ``[tokens, heads, head_dim]`` at ``slots`` ``[tokens]``.  ``dtype``: type of the result,
    float16 or bfloat16 (a 16-bit cache's own by default, bfloat16 for float8_e4m3fn)."""
    refuse_gradient("cache_read", keys, values, key_scales, value_scales)
    if dtype is None:
        dtype = torch.bfloat16 if keys.dtype == torch.float8_e4m3fn else keys.dtype
    k, v = kernel.sparse_ops.cache_read(slots, keys, values, key_scales, value_scales, dtype)
    kernel.check(k)
    return k, v
