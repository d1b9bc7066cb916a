"""
Models on the paths that the small ones of test_gpu_q4_engine do not reach: a prompt long
enough for the tensor-core kernel over the 4-bit cache, and a model with capped scores and a
sliding window in the graphed decoder.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

transformers = pytest.importorskip("transformers")

from memforge_b200 import _kernels as K  # noqa: E402
from memforge_b200 import attention_backend as AB  # noqa: E402
from memforge_b200.graphed_decode import GraphedPagedDecoder  # noqa: E402
from memforge_b200.kv_pool import ModelKVSpec, PagedKVPool  # noqa: E402
from memforge_b200.paged_cache import PagedCache  # noqa: E402
from memforge_b200.quant_cache import Q4KVPool  # noqa: E402
from tests.test_gpu_engine import tiny_llama  # noqa: E402
from tests.test_gpu_q4_chunks import form  # noqa: E402
from tests.test_gpu_q4_engine import tiny_gemma2  # noqa: E402


@torch.no_grad()
def test_a_long_prompt_on_the_4_bit_cache(monkeypatch):
    """1500 tokens, then 200 more behind them: logits as of sdpa over the dequantised rows."""
    model, tokens = tiny_llama(128, torch.bfloat16), 1500
    spec = ModelKVSpec.from_config(model.config, torch.bfloat16, "cuda")
    g = torch.Generator().manual_seed(5)
    table = torch.randperm(120, generator=g).tolist()[:108]
    ids = torch.randint(2, 250, (1, tokens + 200), generator=g).cuda()
    forms, real = [], K.q4_paged_attention

    def seen(q, out, pool, tables, kv, **how):
        forms.append(form(kv.numel(), how["q_per_seq"], q.shape[1], pool.shape[2], tables.shape[1],
                          q.shape[0]))
        return real(q, out, pool, tables, kv, **how)

    monkeypatch.setattr(K, "q4_paged_attention", seen)

    def run(lazy):
        pool = Q4KVPool(spec, 120)
        cache = PagedCache(pool, table, lazy_read=lazy)
        out = []
        for a, b in ((0, tokens), (tokens, tokens + 200)):
            cache.begin_step(table)
            kw = dict(input_ids=ids[:, a:b], past_key_values=cache, use_cache=True,
                      position_ids=torch.arange(a, b, device="cuda")[None])
            if lazy:
                with AB.backend_enabled_on(model), AB.paged_attention_context(pool, cache):
                    out.append(model(**kw).logits[0])
            else:
                out.append(model(**kw).logits[0])
        return torch.cat(out).float()

    want, got = run(False), run(True)
    K.check_device_errors()
    assert forms[:2] == ["expanded"] * 2 and len(forms) == 4
    assert (got - want).abs().max() <= 5e-2 * max(1.0, float(want.abs().max()))
    assert (got - want).square().mean().sqrt() <= 1e-2 * want.square().mean().sqrt()


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("dtype,atol", [(torch.float32, 1e-4), (torch.bfloat16, 5e-2)])
@torch.no_grad()
def test_a_capped_and_windowed_model_in_the_graphed_decoder(dtype, atol, four_bit):
    """Steps through graphs equal eager ones over the same rows, on contexts past the window."""
    model = tiny_gemma2(dtype)
    spec = ModelKVSpec.from_config(model.config, dtype, "cuda")
    pool = (Q4KVPool if four_bit else PagedKVPool)(spec, 32)
    tables = [torch.tensor(t, device="cuda") for t in ([3, 9, 17], [1, 8, 2], [4, 6, 30])]
    lens = [30, 5, 18]
    for t, n in zip(tables, lens):   # prompts
        c = PagedCache(pool, t.tolist(), lazy_read=True)
        with AB.backend_enabled_on(model), AB.paged_attention_context(pool, c):
            model(input_ids=torch.arange(3, 3 + n, device="cuda")[None], past_key_values=c, use_cache=True,
                  position_ids=torch.arange(n, device="cuda")[None])
    state = [t.clone() for t in ([pool.pool] if four_bit else [pool.key_pool, pool.value_pool])]
    dec = GraphedPagedDecoder(model, pool, max_batch=4, max_model_len=47)
    toks = [[11, 12, 13], [90, 91, 92], [50, 7, 200]]
    graphed = [dec.step(t, [n + i for n in lens], tables).float() for i, t in enumerate(toks)]
    for t, s in zip([pool.pool] if four_bit else [pool.key_pool, pool.value_pool], state):
        t.copy_(s)
    for i, t in enumerate(toks):
        for s in range(3):
            c = PagedCache(pool, tables[s].tolist(), lazy_read=True)
            c.seed_position(lens[s] + i)
            with AB.backend_enabled_on(model), AB.paged_attention_context(pool, c):
                eager = model(input_ids=torch.tensor([[t[s]]], device="cuda"), past_key_values=c,
                              use_cache=True, position_ids=torch.tensor([[lens[s] + i]], device="cuda"))
            eager = eager.logits[0, -1].float()
            assert (graphed[i][s] - eager).abs().max() <= atol * max(1.0, float(eager.abs().max()))
    K.check_device_errors()
