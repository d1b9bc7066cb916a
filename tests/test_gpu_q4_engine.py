"""
Models served with the 4-bit cache and with modified scores: a tiny randomly initialised
Llama on ``Q4KVPool`` (cache, attention function, packed pass, graphed decoder), and a tiny
Gemma-2 (capped scores, a sliding window on alternate layers) on the 16-bit pool, each against
transformers' own attention over the same cached rows.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

transformers = pytest.importorskip("transformers")

from memforge_b200 import _kernels as K  # noqa: E402
from memforge_b200 import attention_backend as AB  # noqa: E402
from memforge_b200.graphed_decode import GraphedPagedDecoder  # noqa: E402
from memforge_b200.kv_pool import ModelKVSpec, PagedKVPool  # noqa: E402
from memforge_b200.paged_cache import PagedCache, VarlenPackedCache  # noqa: E402
from memforge_b200.quant_cache import Q4KVPool  # noqa: E402
from memforge_b200.varlen_attention import paged_attention_varlen_materialised  # noqa: E402
from tests.test_gpu_engine import PROMPT, TABLE, tiny_llama  # noqa: E402


def q4_pool(model, dtype, blocks=64):
    return Q4KVPool(ModelKVSpec.from_config(model.config, dtype, "cuda"), num_blocks=blocks)


@torch.no_grad()
def run(model, pool, lazy, steps=6):
    """Logits of the prompt and of greedy steps through ``PagedCache`` on `pool`."""
    cache = PagedCache(pool, TABLE, lazy_read=lazy)
    ids, out = torch.tensor([PROMPT], device="cuda"), []
    for i in range(steps + 1):
        pos = torch.arange(cache.position, cache.position + ids.shape[1], device="cuda")[None]
        cache.begin_step(TABLE)
        kw = dict(input_ids=ids, position_ids=pos, past_key_values=cache, use_cache=True)
        if lazy:
            with AB.backend_enabled_on(model), AB.paged_attention_context(pool, cache) as b:
                logits = model(**kw).logits
            assert b.used == model.config.num_hidden_layers
        else:
            logits = model(**kw).logits
        out.append(logits[0, -1].float())
        ids = torch.tensor([[PROMPT[i]]], device="cuda")  # the same inputs on every path
    return torch.stack(out)


@pytest.mark.parametrize("dtype,head_dim,atol", [(torch.float32, 64, 1e-4), (torch.float32, 128, 1e-4),
                                                 (torch.bfloat16, 128, 5e-2)])
def test_llama_on_the_4_bit_cache(dtype, head_dim, atol):
    """Attention read from 4-bit pages equals sdpa over the dequantised rows of the same pool
    (fp32: to 1e-4, as the 32-bit pool's lazy mode is held; bf16: bf16 noise)."""
    model = tiny_llama(head_dim, dtype)
    # sdpa reads prompts' dequantised rows back too, so both paths see the same keys
    want = run(model, q4_pool(model, dtype), lazy=False)
    got = run(model, q4_pool(model, dtype), lazy=True)
    K.check_device_errors()
    assert torch.isfinite(got).all()
    assert (got - want).abs().max() <= atol * max(1.0, float(want.abs().max()))


@torch.no_grad()
def test_packed_pass_and_graphed_decoder_on_the_4_bit_cache():
    model = tiny_llama(128, torch.bfloat16)
    pool = q4_pool(model, torch.bfloat16)
    tables = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([3, 9, 17, 5], [1, 8, 2])]
    lens = [37, 20]
    seq_ids = [0] * lens[0] + [1] * lens[1]
    positions = list(range(lens[0])) + list(range(lens[1]))
    ids = torch.tensor([[(7 * p + 3 * s) % 250 for s, p in zip(seq_ids, positions)]], device="cuda")
    cache = VarlenPackedCache(pool, model.config.num_hidden_layers, tables, seq_ids, positions)
    with AB.backend_enabled_on(model), AB.varlen_attention_context(pool, tables, seq_ids, positions):
        packed = model(input_ids=ids, position_ids=torch.tensor([positions], device="cuda"),
                       past_key_values=cache, use_cache=True).logits[0]
    # each sequence alone, on a pool of its own
    at = 0
    for t, n in zip(tables, lens):
        p2 = q4_pool(model, torch.bfloat16)
        c2 = PagedCache(p2, t.tolist(), lazy_read=True)
        with AB.backend_enabled_on(model), AB.paged_attention_context(p2, c2):
            alone = model(input_ids=ids[:, at:at + n], past_key_values=c2, use_cache=True,
                          position_ids=torch.arange(n, device="cuda")[None]).logits[0]
        assert (packed[at:at + n].float() - alone.float()).abs().max() <= 5e-2 * float(alone.abs().max())
        at += n
    # the graphed step equals the eager one on the same pool
    state = pool.pool.clone()
    dec = GraphedPagedDecoder(model, pool, max_batch=2, max_model_len=60)
    graphed = [dec.step([11, 12], lens, tables).float()]
    graphed.append(dec.step([13, 14], [n + 1 for n in lens], tables).float())
    pool.pool.copy_(state)
    for i, toks in enumerate(([11, 12], [13, 14])):
        for s in range(2):
            c = PagedCache(pool, tables[s].tolist(), lazy_read=True)
            c.seed_position(lens[s] + i)
            with AB.backend_enabled_on(model), AB.paged_attention_context(pool, c):
                eager = model(input_ids=torch.tensor([[toks[s]]], device="cuda"), use_cache=True,
                              past_key_values=c,
                              position_ids=torch.tensor([[lens[s] + i]], device="cuda")).logits[0, -1]
            assert (graphed[i][s] - eager.float()).abs().max() <= 5e-2 * float(eager.abs().max())
    K.check_device_errors()


def test_materialised_seam_and_block_copy():
    spec = ModelKVSpec(2, 2, 128, torch.float32, "cuda")
    pool = Q4KVPool(spec, 8)
    g = torch.Generator(device="cuda").manual_seed(1)
    kv = [torch.randn((1, 2, 20, 128), generator=g, device="cuda") for _ in range(2)]
    table = torch.tensor([5, 2], device="cuda")
    for layer in range(2):
        pool.write(layer, *pool.slot_indices(table, 0, 20), *kv)
    q = torch.randn((1, 4, 3, 128), generator=g, device="cuda")
    out = paged_attention_varlen_materialised(q, pool, 1, [table], [0, 0, 0], [17, 18, 19])
    k, v = pool.gather(1, *pool.slot_indices(table, 0, 20))
    s = torch.einsum("hqd,hkd->hqk", q[0].double(), k[0].double().repeat_interleave(2, 0)) / 128 ** 0.5
    s = s.masked_fill(torch.arange(20, device="cuda") > torch.tensor([[17], [18], [19]], device="cuda"),
                      float("-inf"))
    want = torch.softmax(s, -1) @ v[0].double().repeat_interleave(2, 0)
    assert (out[0].double() - want).abs().max() <= 1e-5
    pool.copy_blocks(torch.tensor([[5, 0], [2, 7]], dtype=torch.int32, device="cuda"))
    assert torch.equal(pool.pool[:, 0], pool.pool[:, 5]) and torch.equal(pool.pool[:, 7], pool.pool[:, 2])


def tiny_gemma2(dtype, seed=3):
    from transformers import Gemma2Config, Gemma2ForCausalLM
    torch.manual_seed(seed)
    cfg = Gemma2Config(vocab_size=256, hidden_size=256, intermediate_size=256, num_hidden_layers=2,
                       num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                       query_pre_attn_scalar=4, sliding_window=9, attn_logit_softcapping=5.0,
                       final_logit_softcapping=None, max_position_embeddings=512, eos_token_id=1,
                       bos_token_id=0, pad_token_id=0, attn_implementation="eager")
    return Gemma2ForCausalLM(cfg).to(device="cuda", dtype=dtype).eval()


@pytest.mark.parametrize("dtype,atol", [(torch.float32, 1e-4), (torch.bfloat16, 6e-2)])
@pytest.mark.parametrize("four_bit", [False, True])
@torch.no_grad()
def test_gemma2_scores_are_capped_and_windowed(dtype, atol, four_bit):
    """Prompt and steps equal transformers' eager attention (which caps and masks) over the same
    rows; without the cap or the window they would not."""
    model = tiny_gemma2(dtype)
    spec = ModelKVSpec.from_config(model.config, dtype, "cuda")

    def pool():
        return Q4KVPool(spec, 64) if four_bit else PagedKVPool(spec, 64)

    want = run(model, pool(), lazy=False)
    got = run(model, pool(), lazy=True)
    size = max(1.0, float(want.abs().max()))
    assert (got - want).abs().max() <= atol * size
    saved = AB._score_mods
    AB._score_mods = lambda kw: {}
    try:
        plain = run(model, pool(), lazy=True)
    finally:
        AB._score_mods = saved
    if dtype == torch.float32:  # (in bf16 the noise is of the modifiers' size here)
        assert (plain - want).abs().max() > 4 * atol * size
