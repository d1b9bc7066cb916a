"""
Pools of other classes: an object with ``key_pool``, ``value_pool`` and ``block_size`` (as
MemForge's own pool is) serves the bindings, the packed cache and the graphed decoder.
"""

from types import SimpleNamespace

import pytest
import torch

from memforge_b200 import _kernels as K
from memforge_b200 import attention_backend as AB
from memforge_b200 import kv_pool as KP
from memforge_b200.varlen_attention import paged_attention_varlen_materialised

transformers = pytest.importorskip("transformers")

from memforge_b200.paged_cache import VarlenPackedCache  # noqa: E402


def plain_pool(device="cpu", layers=2, blocks=6, heads=2, d=64, dtype=torch.float32):
    k = torch.randn((layers, blocks, 16, heads, d), device=device).to(dtype)
    return SimpleNamespace(key_pool=k, value_pool=k.clone(), block_size=16)


@pytest.fixture
def calls(monkeypatch):
    """The calls that reach the kernels' wrappers, which need a GPU."""
    seen = []

    def attention(q, out, key_pool, value_pool, tables, kv, **how):
        out.zero_()
        seen.append((key_pool, value_pool, tables.tolist(), kv.tolist(), how))
        return out

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(K, "paged_attention", attention)
    monkeypatch.setattr(K, "reshape_and_cache", lambda *a: seen.append(a))
    return seen


def test_the_packed_cache_and_its_binding(calls):
    pool = plain_pool()
    tables = [torch.tensor([4, 1]), torch.tensor([2])]
    seq_ids, positions = [0, 0, 1], [16, 17, 3]
    cache = VarlenPackedCache(pool, 2, tables, seq_ids, positions)
    assert cache.write_index.tolist() == [16, 17, 35]
    q = torch.zeros((1, 4, 3, 64))
    with AB.varlen_attention_context(pool, tables, seq_ids, positions) as b:
        out, _ = AB.paged_attention_forward(SimpleNamespace(layer_idx=1), q, None, None, softcap=5.0)
    assert out.shape == (1, 3, 4, 64) and b.used == 1
    k, v, _, kv, how = calls[-1]
    assert torch.equal(k, pool.key_pool[1]) and torch.equal(v, pool.value_pool[1])
    assert sorted(kv) == [4, 18] and how["softcap"] == 5.0


def test_one_sequence_and_a_graphed_step(calls):
    pool = plain_pool()
    cache = SimpleNamespace(position=20, block_table_tensor_cached=lambda: torch.tensor([5, 0]))
    with AB.paged_attention_context(pool, cache):
        AB.paged_attention_forward(SimpleNamespace(layer_idx=0), torch.zeros((1, 4, 2, 64)), None, None)
    assert torch.equal(calls[-1][0], pool.key_pool[0]) and calls[-1][2:4] == ([[5, 0]], [20])
    tables, ctx = torch.tensor([[1], [3]], dtype=torch.int32), torch.tensor([4, 5], dtype=torch.int32)
    with AB.graph_attention_context(pool, tables, ctx):
        AB.paged_attention_forward(SimpleNamespace(layer_idx=1), torch.zeros((2, 4, 1, 64)), None, None,
                                   sliding_window=9)
    assert torch.equal(calls[-1][0], pool.key_pool[1]) and calls[-1][4]["window"] == 9
    rows = torch.zeros((2, 2, 64))
    KP.pool_write_rows(pool, 1, rows, rows, torch.tensor([3, 4]))
    assert torch.equal(calls[-1][2], pool.key_pool[1]) and KP.pool_device(pool).type == "cpu"


def test_the_materialised_seam(calls, monkeypatch):
    monkeypatch.setattr(K, "require_cuda", lambda *a: None)
    pool = plain_pool()
    out = paged_attention_varlen_materialised(torch.zeros((1, 4, 2, 64)), pool, 1,
                                              [torch.tensor([4, 1])], [0, 0], [16, 17])
    assert out.shape == (1, 4, 2, 64) and torch.equal(calls[-1][1], pool.value_pool[1])


@pytest.mark.gpu
@torch.no_grad()
def test_the_graphed_decoder_on_a_plain_pool():
    from memforge_b200.graphed_decode import GraphedPagedDecoder
    from memforge_b200.kv_pool import ModelKVSpec, PagedKVPool
    from tests.test_gpu_engine import tiny_llama
    model = tiny_llama(128, torch.bfloat16)
    spec = ModelKVSpec.from_config(model.config, torch.bfloat16, "cuda")
    own = PagedKVPool(spec, 16)
    plain = SimpleNamespace(key_pool=own.key_pool.clone(), value_pool=own.value_pool.clone(),
                            block_size=16, spec=spec)
    tables = [torch.tensor([3, 9], device="cuda"), torch.tensor([1, 8], device="cuda")]
    got = []
    for pool in (own, plain):
        dec = GraphedPagedDecoder(model, pool, max_batch=2, max_model_len=30)
        got.append([dec.step([11 + i, 12 + i], [i, i], tables) for i in range(3)])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert torch.equal(own.key_pool, plain.key_pool) and own.key_pool.any()
