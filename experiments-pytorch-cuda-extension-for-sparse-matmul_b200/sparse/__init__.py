"""Block-sparse attention primitives for NVIDIA B200 (sm_100a).

Same public surface as the reference package (sparse/__init__.py:1-2):
``SparseLayout`` and ``matmul``; ``softmax`` is the op the reference left
unbound (sparse_softmax.cu:208-236); ``attention`` fuses the three steps of
block-sparse attention into one kernel; ``packed_attention`` is attention inside
the sequences of a packed batch.  ``cached_attention`` and the ``cache_*``
functions serve a model of these layers with a paged key / value cache.
"""
from .layout import SparseLayout
from .matmul import matmul, SparseMatMul
from .softmax import softmax, SparseSoftmax
from .attention import attention, SparseAttention
from .module import BlockSparseSelfAttention
from .packed import packed_attention
from .cache import Cache, cache_read, cache_slots, cache_write, make_cache
from .cached_attention import cached_attention, tree_words
from .batched import BatchedSparseLayout, batched_matmul, batched_softmax, batched_attention

__all__ = ["SparseLayout", "matmul", "SparseMatMul", "softmax", "SparseSoftmax", "attention", "SparseAttention", "BlockSparseSelfAttention",
           "packed_attention", "Cache", "cache_read", "cache_slots", "cache_write", "make_cache", "cached_attention", "tree_words",
           "BatchedSparseLayout", "batched_matmul", "batched_softmax", "batched_attention"]
