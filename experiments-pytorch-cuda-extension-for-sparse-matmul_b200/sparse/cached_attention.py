"""Attention of new tokens over a paged key / value cache.

    o_i = sum_j p_ij v_j      p_ij = exp(scale q_i k_j - lse_i) over the keys j that draft i sees

A sequence has its tokens in the pages its row of ``table`` names (see
``cache``); the last ``counts[b]`` of its ``lengths[b]`` tokens are its drafts,
the tokens whose queries are given.  A draft sees every token before the
drafts, and among the drafts those of ``tree``: bit j of word i says that
draft i sees draft j (``tree_words`` makes the words of a tree from its
parents; without a tree the drafts are a chain, draft i sees drafts 0 .. i).
One draft is the ordinary decoding step; several are a chain of tokens or a
tree of guesses checked at once.

``layout`` restricts the keys as ``attention`` does for whole sequences: the
key at position j is seen from position i only where the layout has the block
(i // block, j // block).  A draft's position is the number of tokens before
the drafts plus the number of its ancestors.

Serving only: there is no gradient.  A NaN or an infinity among the values of a
sequence's drafts, or of a place that one of them sees, may reach all of that
sequence's rows, never another sequence's.  What lies behind a sequence's length,
and what the layout hides from all of its drafts, is never used.
"""
from typing import Optional, Sequence

import torch

from . import kernel
from .cache import refuse_gradient
from .layout import SparseLayout


def tree_words(parents: Sequence[Sequence[int]], device=None) -> torch.Tensor:
    """int64 words ``[sequences, drafts]`` of trees given by their parents: ``parents[b][i]`` is the draft that draft
    ``i`` of sequence ``b`` follows (smaller than ``i``), -1 where it follows the sequence itself."""
    rows = []
    for tree in parents:
        if len(tree) > 64:
            raise ValueError("at most 64 drafts per sequence, got %d" % len(tree))
        words = []
        for i, parent in enumerate(tree):
            if not -1 <= parent < i:
                raise ValueError("the parent of draft %d must be -1 or an earlier draft, got %r" % (i, parent))
            words.append((words[parent] if parent >= 0 else 0) | 1 << i)
        rows.append([w - (1 << 64) if w >> 63 else w for w in words])
    if len({len(row) for row in rows}) > 1:
        raise ValueError("all sequences need the same number of drafts (give `counts` for fewer)")
    return torch.tensor(rows, dtype=torch.int64, device=device)


def _pattern(layout: SparseLayout, device: torch.device) -> torch.Tensor:
    """The layout's block flags as the kernel reads them, made once per layout object and device: the first call waits for
    them, since later ones may come on other streams.  Under capture they are made in the graph, at each replay, and not
    kept."""
    held = getattr(layout, "_cached_pattern", None)
    if held is None or held.device != device:
        capturing = device.type == "cuda" and torch.cuda.is_current_stream_capturing()
        if capturing and layout.pattern.device != device:
            raise RuntimeError("cached_attention: the layout's pattern is on another device; call once with this layout before "
                               "the capture")
        held = (layout.pattern != 0).to(device=device, dtype=torch.uint8).contiguous()
        if capturing:
            return held
        if held.is_cuda:
            torch.cuda.current_stream(device).synchronize()
        layout._cached_pattern = held
    return held


def cached_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, key_scales: Optional[torch.Tensor],
                     value_scales: Optional[torch.Tensor], table: torch.Tensor, lengths: torch.Tensor,
                     counts: Optional[torch.Tensor] = None, tree: Optional[torch.Tensor] = None, scale: float = 1.0,
                     layout: Optional[SparseLayout] = None) -> torch.Tensor:
    """Attention of ``q [batch, drafts, heads, head_dim]`` (float16 or bfloat16, at most 65536 sequences and 64 drafts;
    ``heads`` a multiple of the cache's) over the cache ``keys, values, key_scales, value_scales``; returns q's shape.

    ``table`` int32 ``[batch, pages]``, ``lengths`` int32 ``[batch]``, ``counts`` int32 ``[batch]`` (default: every
    sequence has all drafts), ``tree`` int64 ``[batch, drafts]``.  Drafts from ``counts[b]`` on, and drafts that see
    nothing, give zeros.  Only table entries before a sequence's length are read; a page that is none of the cache's
    and a length behind the table's end leave those keys out and are reported by ``check_device_status``."""
    refuse_gradient("cached_attention", q, keys, values, key_scales, value_scales)
    pattern, block = (None, 0) if layout is None else (_pattern(layout, q.device), layout.block)
    return kernel.check(kernel.sparse_ops.cached_attention(q, keys, values, key_scales, value_scales, table, lengths,
                                                           counts, tree, float(scale), pattern, block))
