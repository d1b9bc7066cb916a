"""
The 4-bit paged KV cache: a pool, its quantising write, its dequantising read and
attention over it (sm_100a kernels; no counterpart in MemForge, whose pools hold the
model's dtype).

A cached row of ``head_dim`` values takes ``head_dim / 2`` bytes of codes and two
fp16 numbers: ``x ~ code * scale + base`` with one (scale, base) per token, kv head and
K or V.  ``include/memforge_sm100.h`` states the quantiser and the record layout exactly.
At head_dim 128 a token costs 136 bytes per kv head where bf16 costs 512.

``Q4KVPool`` has ``PagedKVPool``'s interface, so ``PagedCache``, ``VarlenPackedCache``,
``GraphedPagedDecoder`` and the ``memforge_paged`` attention function run on it
unchanged.  The functions below are the same operators on a bare pool tensor
``uint8 (layers, blocks, kv_heads, 16 * D + 128)``.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _kernels as K
from . import paged_gather
from .kv_pool import ModelKVSpec, PagedKVPool

BLOCK_SIZE = K.Q4_BLOCK


def record_bytes(head_dim: int) -> int:
    """Bytes of one record: 16 tokens of one kv head, K and V."""
    if head_dim not in (64, 128, 256):
        raise ValueError(f"the 4-bit cache holds head_dim 64, 128 or 256, got {head_dim}")
    return 16 * head_dim + 128


def scatter_kv_q4(pool: torch.Tensor, layer_idx: int, flat_index: torch.Tensor,
                  keys: torch.Tensor, values: torch.Tensor) -> None:
    """
    Quantise ``(1, heads, tokens, head_dim)`` K/V into layer ``layer_idx`` at slots
    ``flat_index`` (-1 skips a token), in place: ``paged_gather.scatter_kv`` for a
    4-bit pool.  Sources are fp32, fp16 or bf16, of any strides.
    """
    K.q4_reshape_and_cache(keys, values, pool, flat_index, layer=layer_idx, heads_first=True)


def gather_kv_q4(pool: torch.Tensor, layer_idx: int, flat_index: torch.Tensor,
                 dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    """
    The slots ``flat_index`` of a layer as dequantised ``(1, heads, tokens,
    head_dim)`` K/V of ``dtype``: ``paged_gather.gather_kv`` for a 4-bit pool.
    """
    return K.q4_gather_kv(pool, flat_index, dtype, layer=layer_idx)


def paged_attention_q4(q: torch.Tensor, pool: torch.Tensor, layer_idx: int,
                       block_tables: torch.Tensor, kv_lens: torch.Tensor, *,
                       cu_seqlens_q: Optional[torch.Tensor] = None, q_per_seq: int = 1,
                       max_q_len: Optional[int] = None, scale: Optional[float] = None,
                       causal: bool = True, row_map: Optional[torch.Tensor] = None,
                       softcap: float = 0.0, window: int = 0,
                       alibi_slopes: Optional[torch.Tensor] = None,
                       prefix_lens: Optional[torch.Tensor] = None,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    Attention of ``q`` ``(rows, heads, head_dim)`` over a layer of a 4-bit pool.

    ``block_tables`` int32 ``[num_seqs, width]``, ``kv_lens`` int32 ``[num_seqs]``
    (tokens in the cache, this step's included).  Rows are sequence-major:
    ``q_per_seq`` for each sequence, or ``cu_seqlens_q`` int32 ``[num_seqs + 1]`` with
    ``max_q_len``; row i of a sequence is at position ``kv_len - q_len + i``.  The
    score modifiers are those of ``scored_attention.paged_attention_scored``.  A row
    without a visible key comes out as zeros.  Returns ``out`` (q's shape and dtype).
    """
    if q.stride(-1) != 1:
        q = q.contiguous()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    return K.q4_paged_attention(q, out, pool, block_tables, kv_lens, layer=layer_idx,
                                cu_seqlens_q=cu_seqlens_q, q_per_seq=q_per_seq,
                                max_q_len=max_q_len, scale=scale, causal=causal, row_map=row_map,
                                softcap=softcap, window=window, alibi_slopes=alibi_slopes,
                                prefix_lens=prefix_lens)


class Q4KVPool(PagedKVPool):
    """
    ``PagedKVPool`` holding 4-bit rows.  ``spec.dtype`` is the dtype the model writes
    and reads back; ``pool`` is ``uint8 (layers, blocks, kv_heads, record)``.
    """

    def __init__(self, spec: ModelKVSpec, num_blocks: int, block_size: int = BLOCK_SIZE):
        if block_size != BLOCK_SIZE:
            raise ValueError(f"the 4-bit cache has blocks of {BLOCK_SIZE} tokens, got {block_size}")
        if spec.dtype not in K.DTYPES:
            raise TypeError(f"unsupported dtype {spec.dtype}; expected float32, float16 or bfloat16")
        self.spec = spec
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.pool = torch.zeros((spec.num_layers, num_blocks, spec.num_kv_heads,
                                 record_bytes(spec.head_dim)), dtype=torch.uint8,
                                device=spec.device)

    @property
    def device(self) -> torch.device:
        return self.pool.device

    @property
    def bytes_per_block(self) -> int:
        return self.spec.num_layers * self.spec.num_kv_heads * record_bytes(self.spec.head_dim)

    @staticmethod
    def blocks_for_budget(spec: ModelKVSpec, block_size: int, budget_mb: float) -> int:
        per_block = spec.num_layers * spec.num_kv_heads * record_bytes(spec.head_dim)
        return max(1, int((budget_mb * 1024 * 1024) // per_block))

    def write(self, layer_idx: int, physical: torch.Tensor, slots: torch.Tensor,
              keys: torch.Tensor, values: torch.Tensor) -> None:
        self.write_flat(layer_idx, paged_gather.flat_slot_index(physical, slots, self.block_size),
                        keys, values)

    def write_flat(self, layer_idx: int, flat_index: torch.Tensor, keys: torch.Tensor,
                   values: torch.Tensor) -> None:
        scatter_kv_q4(self.pool, layer_idx, flat_index, keys, values)

    def gather_flat(self, layer_idx: int, flat_index: torch.Tensor):
        return gather_kv_q4(self.pool, layer_idx, flat_index, self.spec.dtype)

    def write_rows(self, layer_idx: int, keys: torch.Tensor, values: torch.Tensor,
                   slots: torch.Tensor) -> None:
        K.q4_reshape_and_cache(keys, values, self.pool, slots, layer=layer_idx)

    def attend(self, layer_idx: int, q: torch.Tensor, out: torch.Tensor,
               block_tables: torch.Tensor, kv_lens: torch.Tensor, **how) -> torch.Tensor:
        return K.q4_paged_attention(q, out, self.pool, block_tables, kv_lens, layer=layer_idx,
                                    **how)

    def copy_blocks(self, pairs: torch.Tensor) -> None:
        """Copy block src -> dst in every layer; ``pairs`` int32 ``[n, 2]`` on the device."""
        K.copy_blocks(self.pool, self.pool, pairs)   # K and V share a record

    def zero_(self) -> None:
        self.pool.zero_()

    def describe(self) -> dict:
        per_token = self.bytes_per_block // self.block_size
        return {
            "num_blocks": self.num_blocks, "block_size": self.block_size,
            "capacity_tokens": self.capacity_tokens,
            "bytes_per_token": per_token, "bytes_per_block": self.bytes_per_block,
            "total_mb": round(self.total_bytes / (1024 * 1024), 2),
            "num_layers": self.spec.num_layers, "num_kv_heads": self.spec.num_kv_heads,
            "head_dim": self.spec.head_dim, "dtype": "4-bit (" + str(self.spec.dtype) + ")",
            "device": self.spec.device,
        }
