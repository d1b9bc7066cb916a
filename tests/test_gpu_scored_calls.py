"""Calls of attention with modified scores at the edges of what is allowed."""

import math

import numpy as np
import pytest
import torch

from memforge_b200.scored_attention import paged_attention_scored
from tests.test_gpu_q4 import Case as Q4Case
from tests.test_gpu_scored import Case

pytestmark = pytest.mark.gpu

K = pytest.importorskip("memforge_b200._kernels")


def test_a_batch_without_rows_is_nothing_to_do():
    pool = torch.zeros((2, 4, 16, 2, 128), dtype=torch.bfloat16, device="cuda")
    q = torch.empty((0, 8, 128), dtype=torch.bfloat16, device="cuda")
    tables = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    kv, cu = tables[:, 0].contiguous(), torch.zeros(4, dtype=torch.int32, device="cuda")
    for how in (dict(window=5), dict(softcap=3.0), dict()):
        out = paged_attention_scored(q, pool, pool, 1, tables, kv, cu_seqlens_q=cu, max_q_len=4, **how)
        assert out.shape == (0, 8, 128)


@pytest.mark.parametrize("dtype,hq,d,ql,block", [("f32", 4, 80, 1, 16), ("f32", 4, 128, 3, 8),
                                                 ("bf16", 4, 256, 40, 16), ("f32", 4, 64, 20, 4),
                                                 ("bf16", 4, 128, 1, 16), ("bf16", 4, 128, 90, 16)])
@pytest.mark.parametrize("prefix", [0, 5, 36])
def test_blocks_behind_a_window_may_be_freed(dtype, hq, d, ql, block, prefix):
    """Table entries of blocks that no row sees are not read: -1 there is no error."""
    c = Case(240, dtype, hq, 2, d, [ql + 150, ql + 39, ql + 77], [ql] * 3, window=13, block=block,
             prefix=[prefix] * 3 if prefix else None)
    freed = 0
    for s, n in enumerate(c.kv_lens):
        low = n - ql - 13 + 1
        for b in range(low // block):
            if b * block >= prefix:
                c.tables[s, b] = -1
                freed += 1
    assert freed > 3
    # (the reference below reads block -1, the last one: its rows are hidden)
    c.check()


@pytest.mark.parametrize("softcap", [1e-30, 1e-20, 1e-12, 1e-6, 50.0, 1e30])
@pytest.mark.parametrize("dtype,hq,d,ql", [("bf16", 16, 128, 200), ("f16", 8, 128, 1),
                                           ("bf16", 8, 128, 20), ("f32", 4, 80, 3)])
def test_scores_of_zero_under_any_cap(softcap, dtype, hq, d, ql):
    """A zero query weighs its keys alike, however small the cap is."""
    c = Case(241, dtype, hq, 4, d, [ql + 60, ql + 200], [ql] * 2, softcap=softcap, q_scale=0.0)
    c.check()
    if d == 128:
        Q4Case(242, dtype, hq, 4, d, [ql + 60, ql + 200], [ql] * 2, softcap=softcap, q_scale=0.0).check()


@pytest.mark.parametrize("dtype,hq,d,ql", [("bf16", 8, 128, 1), ("f16", 8, 64, 1), ("bf16", 8, 128, 5),
                                           ("bf16", 16, 128, 40), ("f32", 4, 80, 3),
                                           ("bf16", 4, 256, 2)])
def test_a_row_that_sees_only_nan_keys_is_nan(dtype, hq, d, ql):
    c = Case(243, dtype, hq, 4, d, [ql, ql + 40], [ql] * 2, window=1)
    slots = c.tables[0, np.arange(ql) // 16] * 16 + np.arange(ql) % 16
    c.k_dev.view(-1, 4, d)[torch.from_numpy(slots).cuda().long()] = math.nan
    got = c.run().double().cpu().numpy()
    want, tol = c.want()
    assert np.isnan(got[:ql]).all()
    assert (np.abs(got - want)[ql:] <= tol[ql:]).all()


def test_tensors_that_do_not_fit_the_call_are_refused():
    """Before any launch: the kernels would read or write past them."""
    c = Case(244, "bf16", 8, 2, 128, [50, 20, 33], [1] * 3, window=9)
    tables = torch.from_numpy(c.tables).cuda()
    kv = torch.tensor(c.kv_lens, dtype=torch.int32).cuda()
    cu = torch.arange(4, dtype=torch.int32, device="cuda")

    def call(out=None, v=None, t=None, **how):
        out = torch.empty_like(c.q_dev) if out is None else out
        return K.paged_attention(c.q_dev, out, c.k_dev, c.v_dev if v is None else v,
                                 tables if t is None else t, kv, scale=c.scale, window=9, **how)

    call(cu_seqlens_q=cu, max_q_len=1, row_map=cu[:3])
    short = torch.empty_like(c.q_dev)
    for bad in (dict(out=short[:2]), dict(out=short[:, :4]), dict(v=c.v_dev[:-1]), dict(t=tables[:2]),
                dict(t=tables[0]), dict(cu_seqlens_q=cu[:3], max_q_len=1), dict(cu_seqlens_q=cu),
                dict(cu_seqlens_q=torch.arange(8, dtype=torch.int32, device="cuda")[::2], max_q_len=1),
                dict(row_map=cu[:2]), dict(row_map=torch.zeros(6, dtype=torch.int32, device="cuda")[::2])):
        with pytest.raises(ValueError):
            call(**bad)
    K.check_device_errors()
