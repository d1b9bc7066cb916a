"""
Paged attention with modified scores (no counterpart in MemForge): scores capped by a
tanh, a bias that grows with distance, a sliding window, a prefix that every row sees.

For the row at position p and key position k, in this order:

* ``s = scale * q.k``
* ``softcap``:       ``s = softcap * tanh(s / softcap)``
* ``alibi_slopes``:  ``s = s - alibi_slopes[head] * (p - k)``
* visible iff ``k < kv_len`` and (``k < prefix_lens[seq]`` or
  (``k <= p`` and (``window == 0`` or ``p - k < window``)))

``prefix_lens`` alone is a prefix mask (the prompt's first tokens see each other in both
directions); with ``window`` it keeps a sequence's first tokens visible behind it.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _kernels as K


def paged_attention_scored(q: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor,
                           layer_idx: int, block_tables: torch.Tensor, kv_lens: torch.Tensor, *,
                           cu_seqlens_q: Optional[torch.Tensor] = None, q_per_seq: int = 1,
                           max_q_len: Optional[int] = None, scale: Optional[float] = None,
                           causal: bool = True, row_map: Optional[torch.Tensor] = None,
                           softcap: float = 0.0, window: int = 0,
                           alibi_slopes: Optional[torch.Tensor] = None,
                           prefix_lens: Optional[torch.Tensor] = None,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    Attention of ``q`` ``(rows, heads, head_dim)`` over a layer of the pool
    ``(layers, blocks, block_size, kv_heads, head_dim)``.

    ``block_tables`` int32 ``[num_seqs, width]``, ``kv_lens`` int32 ``[num_seqs]``.  Rows
    are sequence-major: ``q_per_seq`` for each sequence, or ``cu_seqlens_q`` int32
    ``[num_seqs + 1]`` with ``max_q_len``; row i of a sequence is at position
    ``kv_len - q_len + i``.  ``alibi_slopes`` fp32 ``[heads]``, ``prefix_lens`` int32
    ``[num_seqs]``; a zero or None modifier is left out, and without any this is plain paged
    attention.  Returns ``out`` (q's shape and dtype).
    """
    if q.dim() != 3:
        raise ValueError(f"q must be (rows, heads, head_dim), got {tuple(q.shape)}")
    if cu_seqlens_q is not None and max_q_len is None:
        raise ValueError("cu_seqlens_q needs max_q_len")
    if cu_seqlens_q is None and q_per_seq * kv_lens.numel() != q.shape[0]:
        raise ValueError(f"{kv_lens.numel()} sequences of {q_per_seq} rows but {q.shape[0]} "
                         f"query rows")
    if q.stride(-1) != 1:
        q = q.contiguous()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if q.shape[0] == 0:
        return out
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    return K.paged_attention(q, out, key_pool[layer_idx], value_pool[layer_idx], block_tables,
                             kv_lens, cu_seqlens_q=cu_seqlens_q, q_per_seq=q_per_seq,
                             max_q_len=max_q_len, scale=scale, causal=causal, row_map=row_map,
                             softcap=softcap, window=window, alibi_slopes=alibi_slopes,
                             prefix_lens=prefix_lens)
