"""Argument checks of the 4-bit cache and modified-score entry points (no GPU)."""

import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from memforge_b200 import _kernels as K
from memforge_b200 import _lib as L
from memforge_b200 import quant_cache as Q
from memforge_b200.kv_pool import ModelKVSpec
from memforge_b200.scored_attention import paged_attention_scored
from tests.conftest import ROOT


@pytest.mark.parametrize("cname,struct", [("mf_score_mods", L.ScoreMods),
                                          ("mf_q4_attention_args", L.Q4AttentionArgs)])
def test_struct_layout_matches_the_header(cname, struct):
    fields = [f for f, _ in struct._fields_]
    src = ["#include <stdio.h>", "#include <stddef.h>", '#include "memforge_sm100.h"',
           "int main(void){", f'printf("%zu\\n", sizeof({cname}));']
    src += [f'printf("%zu\\n", offsetof({cname}, {f}));' for f in fields] + ["return 0;}"]
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(c, "w").write("\n".join(src))
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        vals = [int(x) for x in subprocess.run([exe], capture_output=True, text=True,
                                               check=True).stdout.split()]
    assert vals[0] == ctypes.sizeof(struct)
    for f, off in zip(fields, vals[1:]):
        assert getattr(struct, f).offset == off, f


def test_record_bytes():
    assert [Q.record_bytes(d) for d in (64, 128, 256)] == [1152, 2176, 4224]
    assert [L.lib().mf_q4_record_bytes(d) for d in (64, 128, 256)] == [1152, 2176, 4224]
    assert L.lib().mf_q4_record_bytes(80) == L.MF_EUNSUPPORTED
    with pytest.raises(ValueError, match="head_dim"):
        Q.record_bytes(96)


def args(**kw):
    a = L.Q4AttentionArgs()
    a.struct_size = ctypes.sizeof(a)
    a.q = a.out = a.pool = a.block_tables = a.kv_lens = 0x1000
    a.q_stride_row = a.out_stride_row = 512
    a.q_stride_head = a.out_stride_head = 128
    a.pool_stride_block, a.pool_stride_head = 2 * 2176, 2176
    a.num_blocks, a.table_stride, a.table_width = 4, 4, 4
    a.q_per_seq, a.num_seqs, a.total_q, a.max_q_len = 1, 2, 2, 1
    a.num_q_heads, a.num_kv_heads, a.head_dim = 4, 2, 128
    a.scale, a.causal, a.dtype = 0.1, 1, L.MF_BF16
    for k, v in kw.items():
        if k in ("softcap", "window"):
            setattr(a.mods, k, v)
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad,code", [
    (dict(struct_size=8), L.MF_EINVAL), (dict(num_seqs=-1), L.MF_EINVAL),
    (dict(num_q_heads=3), L.MF_EINVAL), (dict(num_kv_heads=0), L.MF_EINVAL),
    (dict(head_dim=80), L.MF_EUNSUPPORTED), (dict(num_blocks=0), L.MF_EINVAL),
    (dict(dtype=7), L.MF_EINVAL), (dict(q_per_seq=0), L.MF_EINVAL),
    (dict(pool=0x1008), L.MF_EINVAL), (dict(pool_stride_head=2177), L.MF_EINVAL),
    (dict(num_seqs=70000, total_q=70000), L.MF_EUNSUPPORTED), (dict(kv_lens=None), L.MF_EINVAL),
    (dict(softcap=-1.0), L.MF_EINVAL), (dict(softcap=float("nan")), L.MF_EINVAL),
    (dict(window=-3), L.MF_EINVAL), (dict(table_width=-1), L.MF_EINVAL),
    (dict(), L.MF_EWORKSPACE)])
def test_attention_arguments_are_checked_before_any_launch(bad, code):
    assert L.lib().mf_q4_paged_attention(args(**bad), None, 0, None, None) == code
    assert L.lib().mf_last_error().startswith(b"q4 attention")


def test_attention_without_rows_is_nothing_to_do():
    assert L.lib().mf_q4_paged_attention(args(num_seqs=0), None, 0, None, None) == L.MF_OK
    assert L.lib().mf_q4_paged_attention(args(total_q=0), None, 0, None, None) == L.MF_OK


@pytest.mark.parametrize("bad,code", [
    (dict(pool=0x1004), L.MF_EINVAL), (dict(d=32), L.MF_EINVAL), (dict(tokens=-1), L.MF_EINVAL),
    (dict(blocks=0), L.MF_EINVAL), (dict(key=None), L.MF_EINVAL), (dict(dtype=9), L.MF_EINVAL)])
def test_write_and_read_arguments_are_checked(bad, code):
    v = dict(key=0x1000, pool=0x1000, d=128, tokens=3, blocks=2, dtype=L.MF_BF16)
    v.update(bad)
    lib = L.lib()
    assert lib.mf_q4_reshape_and_cache(v["key"], 0x1000, v["dtype"], 256, 128, 256, 128, v["pool"],
                                       4352, 2176, v["blocks"], 0x1000, 0, v["tokens"], 2, v["d"],
                                       None, None) == code
    assert lib.mf_q4_gather_kv(v["pool"], 4352, 2176, v["blocks"], 0x1000, 0, v["tokens"], 2,
                               v["d"], v["key"], 0x1000, v["dtype"], 384, 128, None, None) == code


def test_scored_arguments_are_checked():
    a = L.AttentionArgs()
    a.struct_size = ctypes.sizeof(a)
    a.q = a.out = a.k_pool = a.v_pool = a.block_tables = a.kv_lens = 0x1000
    a.num_blocks, a.block_size, a.table_stride = 4, 16, 4
    a.q_per_seq, a.num_seqs, a.total_q, a.max_q_len = 1, 1, 1, 1
    a.num_q_heads, a.num_kv_heads, a.head_dim, a.dtype = 2, 2, 128, L.MF_BF16
    call = L.lib().mf_paged_attention_scored
    assert call(a, None, None, 0, None, None) == L.MF_EINVAL
    assert call(a, L.ScoreMods(-1.0, 0, None, None), None, 0, None, None) == L.MF_EINVAL
    assert call(a, L.ScoreMods(0.0, -1, None, None), None, 0, None, None) == L.MF_EINVAL
    a.win_k = a.win_v = 0x1000
    assert call(a, L.ScoreMods(1.0, 0, None, None), None, 0, None, None) == L.MF_EUNSUPPORTED


def test_cpu_tensors_are_refused():
    pool = torch.zeros((1, 2, 2, 2176), dtype=torch.uint8)
    kv = torch.zeros((1, 2, 3, 128))
    with pytest.raises(RuntimeError, match="CUDA"):
        Q.scatter_kv_q4(pool, 0, torch.arange(3), kv, kv)
    with pytest.raises(RuntimeError, match="CUDA"):
        Q.gather_kv_q4(pool, 0, torch.arange(3), torch.float32)
    one = torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        Q.paged_attention_q4(torch.zeros((1, 4, 128)), pool, 0, one.view(1, 1), one)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_attention_scored(torch.zeros((1, 4, 128)), torch.zeros((1, 2, 16, 2, 128)),
                               torch.zeros((1, 2, 16, 2, 128)), 0, one.view(1, 1), one, window=4)


def test_modifier_values_are_refused():
    cpu = torch.device("cpu")
    assert K.score_mods(cpu, 4, 2, 0.0, 0, None, None) is None
    for bad in (dict(softcap=-1.0), dict(softcap=float("nan")), dict(window=-1),
                dict(alibi_slopes=torch.ones(3)), dict(alibi_slopes=torch.ones(4).double()),
                dict(alibi_slopes=torch.ones(8)[::2]), dict(prefix_lens=torch.ones(2)),
                dict(prefix_lens=torch.ones(1, dtype=torch.int32))):
        v = dict(softcap=0.0, window=0, alibi_slopes=None, prefix_lens=None)
        v.update(bad)
        with pytest.raises(ValueError):
            K.score_mods(cpu, 4, 2, **v)


@pytest.mark.parametrize("cap", [1e-38, 1e31, float("inf")])
def test_caps_outside_the_range_are_refused(cap):
    with pytest.raises(ValueError, match="softcap"):
        K.score_mods(torch.device("cpu"), 4, 2, cap, 0, None, None)
    assert L.lib().mf_q4_paged_attention(args(softcap=cap), None, 0, None, None) == L.MF_EINVAL


@pytest.mark.parametrize("scale", [0.0, -0.1, float("nan"), float("inf")])
def test_scales_that_order_nothing_are_refused(scale):
    assert L.lib().mf_q4_paged_attention(args(scale=scale), None, 0, None, None) == L.MF_EINVAL
    a = L.AttentionArgs()
    a.struct_size = ctypes.sizeof(a)
    a.q = a.out = a.k_pool = a.v_pool = a.block_tables = a.kv_lens = 0x1000
    a.num_blocks, a.block_size, a.table_stride = 4, 16, 4
    a.q_per_seq, a.num_seqs, a.total_q, a.max_q_len = 1, 1, 1, 1
    a.num_q_heads, a.num_kv_heads, a.head_dim, a.dtype = 2, 2, 128, L.MF_BF16
    a.scale = scale
    assert L.lib().mf_paged_attention_scored(a, L.ScoreMods(9.0, 0, None, None), None, 0, None,
                                             None) == L.MF_EINVAL


def test_fewer_rows_than_the_sequences_have_are_refused():
    bad = args(q_per_seq=3, total_q=5)
    assert L.lib().mf_q4_paged_attention(bad, None, 0, None, None) == L.MF_EINVAL
    a = L.AttentionArgs()
    a.struct_size = ctypes.sizeof(a)
    a.q = a.out = a.k_pool = a.v_pool = a.block_tables = a.kv_lens = 0x1000
    a.num_blocks, a.block_size, a.table_stride = 4, 16, 4
    a.q_per_seq, a.num_seqs, a.total_q, a.max_q_len = 2, 2, 3, 2
    a.num_q_heads, a.num_kv_heads, a.head_dim, a.dtype, a.scale = 2, 2, 128, L.MF_BF16, 0.1
    assert L.lib().mf_paged_attention_scored(a, L.ScoreMods(9.0, 0, None, None), None, 0, None,
                                             None) == L.MF_EINVAL


def test_a_window_past_32_bits_is_no_narrow_one():
    cpu = torch.device("cpu")
    assert K.score_mods(cpu, 4, 2, 0.0, 2 ** 32 + 5, None, None).window == 2 ** 31 - 1


def test_pool_shapes_are_refused():
    for t in (torch.zeros((2, 2, 2176)), torch.zeros((2, 2, 2000), dtype=torch.uint8),
              torch.zeros((2, 2, 1408), dtype=torch.uint8), torch.zeros((2, 2176), dtype=torch.uint8),
              torch.zeros((2, 2176, 2), dtype=torch.uint8).transpose(1, 2)):
        with pytest.raises(ValueError):
            K.q4_head_dim(t)


def test_pool_accounting():
    spec = ModelKVSpec(3, 2, 128, torch.bfloat16, "cpu")
    pool = Q.Q4KVPool(spec, 5)
    assert pool.pool.shape == (3, 5, 2, 2176) and pool.capacity_tokens == 80
    assert pool.bytes_per_block == 3 * 2 * 2176 and pool.total_bytes == pool.pool.numel()
    assert Q.Q4KVPool.blocks_for_budget(spec, 16, 1.0) == (1 << 20) // pool.bytes_per_block
    assert pool.describe()["bytes_per_token"] == 3 * 2 * 136
    with pytest.raises(ValueError, match="16 tokens"):
        Q.Q4KVPool(spec, 5, block_size=32)


def test_a_mask_handed_to_the_attention_function_decides_about_its_window():
    from memforge_b200 import attention_backend as AB
    p, k = torch.arange(3)[:, None] + 4, torch.arange(7)[None]
    causal, near = k <= p, p - k < 3
    as_bias = torch.where(causal & near, 0.0, float("-inf"))
    assert AB._require_plain(causal, 3, 7, True) == 0
    assert AB._require_plain(causal, 3, 7, True, 3) == 0      # the mask has no window
    assert AB._require_plain(causal & near, 3, 7, True, 3) == 3
    assert AB._require_plain(as_bias[None, None], 3, 7, True, 3) == 3
    assert AB._require_plain(near, 3, 7, False, 3) == 3
    for window, mask in ((0, causal & near), (2, causal & near), (3, causal & (k != 2))):
        with pytest.raises(NotImplementedError):
            AB._require_plain(mask, 3, 7, True, window)
