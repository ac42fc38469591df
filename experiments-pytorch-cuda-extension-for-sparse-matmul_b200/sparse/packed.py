"""Attention inside the sequences of a packed batch, forward and backward.

    o_i = sum_j p_ij v_j      p_ij = exp(scale q_i k_j - lse_i),  j in the sequence of i (and j <= i if causal)

``attention`` takes sequences of the one length its layout covers.  Here
sequences of any lengths lie one after the other in ``[rows, heads, head_dim]``
tensors, as prompts of a serving step or documents of a training batch do, and
groups of query heads may share a key head.  The reference has no such op.

Nothing about the lengths is read on the host: a captured CUDA graph follows
``offsets`` that change in place, as long as the number of rows stays.

The forward keeps the output, what its rounding to 16 bits took (so that
rowsum(dO o O) is exact to fp32) and the rows' log-sum-exp; the backward recomputes
the probabilities on chip, by key tiles for dK and dV (summed over the heads
that share a key head) and by query tiles for dQ, without atomics: gradients
repeat bit for bit.  There is no second derivative and no forward-mode one: both
are refused.  A backward pass may be captured; it is refused while a graph recorded
on the default stream still holds some of its leaves.
"""
import torch

from . import kernel


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, scale: float = 1.0,
                     causal: bool = True) -> torch.Tensor:
    """Attention of ``q [rows, heads, head_dim]`` over ``k, v [rows, kv_heads, head_dim]`` (float16 or bfloat16, head
    dimension 64 or 128, ``heads`` a multiple of ``kv_heads``; views of one projection are read in place).

    ``offsets`` int32 ``[sequences + 1]`` on q's device: sequence ``b`` is the rows ``offsets[b] .. offsets[b + 1] - 1``
    (it may be empty; at most 65536 sequences); ``offsets[0]`` is 0.  Rows behind the last sequence give zeros, and zero
    gradients.  Offsets that decrease or pass the last row are reported by ``check_device_status``.  A NaN or an infinity
    reaches rows of its own sequence only."""
    return kernel.sparse_ops.packed_attention(q, k, v, offsets, float(scale), bool(causal), kernel.debug_checks)
