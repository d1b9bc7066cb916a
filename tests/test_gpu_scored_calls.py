"""Calls of attention with modified scores at the edges of what is allowed."""

import pytest
import torch

from memforge_b200.scored_attention import paged_attention_scored

pytestmark = pytest.mark.gpu


def test_a_batch_without_rows_is_nothing_to_do():
    pool = torch.zeros((2, 4, 16, 2, 128), dtype=torch.bfloat16, device="cuda")
    q = torch.empty((0, 8, 128), dtype=torch.bfloat16, device="cuda")
    tables = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    kv, cu = tables[:, 0].contiguous(), torch.zeros(4, dtype=torch.int32, device="cuda")
    for how in (dict(window=5), dict(softcap=3.0), dict()):
        out = paged_attention_scored(q, pool, pool, 1, tables, kv, cu_seqlens_q=cu, max_q_len=4, **how)
        assert out.shape == (0, 8, 128)
