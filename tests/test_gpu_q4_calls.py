"""Calls of 4-bit attention at the edges of what is allowed: after a refused call, without rows."""

import math

import pytest
import torch

from memforge_b200.quant_cache import paged_attention_q4
from tests.gpu_util import TORCH_DT
from tests.test_gpu_q4 import Case

pytestmark = pytest.mark.gpu

K = pytest.importorskip("memforge_b200._kernels")


def test_a_refused_call_leaves_later_ones_as_they_were():
    """A refused call says nothing about the workspace that a valid one of its sizes needs."""
    for seed, hq, bad in ((200, 12, dict(scale=0.0)), (201, 20, dict(scale=math.nan))):
        c = Case(seed, "bf16", hq, 4, 128, [333, 41, 97], [1] * 3)  # (sizes of no other test)
        with pytest.raises(RuntimeError, match="scale"):
            c.run(**bad)
        c.check()
    c = Case(202, "bf16", 28, 4, 128, [333, 41, 98], [1] * 3)
    tables = torch.from_numpy(c.tables).cuda()
    kv = torch.tensor(c.kv_lens, dtype=torch.int32).cuda()
    room = torch.zeros(c.pool.size + 8, dtype=torch.uint8, device="cuda")
    with pytest.raises(RuntimeError, match="16 bytes"):
        K.q4_paged_attention(c.q_dev, torch.empty_like(c.q_dev), room[8:].view(c.pool.shape), tables,
                             kv, scale=c.scale)
    c.check()


def test_a_batch_without_rows_is_nothing_to_do():
    pool = torch.zeros((2, 4, 2, 2176), dtype=torch.uint8, device="cuda")
    q = torch.empty((0, 8, 128), dtype=torch.bfloat16, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    tables = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    kv, cu = tables[:, 0].contiguous(), torch.zeros(4, dtype=torch.int32, device="cuda")
    assert paged_attention_q4(q, pool, 1, tables[:0], none).shape == (0, 8, 128)
    assert paged_attention_q4(q, pool, 1, tables, kv, cu_seqlens_q=cu, max_q_len=0).shape == (0, 8, 128)
    assert paged_attention_q4(q, pool, 1, tables, kv, cu_seqlens_q=cu, max_q_len=5).shape == (0, 8, 128)
    with pytest.raises(ValueError, match="num_seqs"):
        paged_attention_q4(q, pool, 1, tables[:2], kv, cu_seqlens_q=cu, max_q_len=0)


@pytest.mark.parametrize("dtype,ql", [("bf16", 1), ("bf16", 300), ("f32", 3)])
def test_tables_without_entries_are_contexts_without_keys(dtype, ql):
    """No block for any sequence: every row is zeros; a length that would need one is reported."""
    q = torch.ones((2 * ql, 16, 128), dtype=TORCH_DT[dtype], device="cuda")
    pool = torch.zeros((4, 4, 2176), dtype=torch.uint8, device="cuda")
    tables = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    kv = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    K.q4_paged_attention(q, out, pool, tables, kv, q_per_seq=ql, scale=0.1)
    K.check_device_errors()
    assert not out.any()
    K.q4_paged_attention(q, out, pool, tables, kv + 1, q_per_seq=ql, scale=0.1)
    with pytest.raises(IndexError, match="block table"):
        K.check_device_errors()
