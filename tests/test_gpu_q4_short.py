"""
Short runs and 32-bit ones over the 4-bit cache (mma.sync, exact codes), held to bounds by type:
elementwise and in the mean (tests/q4_bounds.py).  fp32 in fp16's precision would not pass.
"""

import math

import numpy as np
import pytest
import torch

from tests import q4_bounds as B
from tests import q4_reference as R
from tests.gpu_util import TORCH_DT
from tests.test_gpu_q4 import as_dtype, rng, tables_for

pytestmark = pytest.mark.gpu

K = pytest.importorskip("memforge_b200._kernels")


def parameters(pool, d, par, tables, pos):
    """(scale, base) of the rows at positions pos of one sequence, (N, H) each."""
    both = np.ascontiguousarray(pool[:, :, par:par + 64]).view(np.float16)
    both = both.reshape(pool.shape[0], pool.shape[1], 16, 2)[tables[pos // 16], :, pos % 16]
    return both[..., 0].astype(np.float64), both[..., 1].astype(np.float64)


def check(seed, dtype, hq, hkv, d, kv, ql, k_size=1.0, v_size=1.0, **mods):
    g = rng(seed)
    tables, blocks = tables_for(g, kv)
    pool = B.sized_pool(g, blocks, hkv, d, k_size, v_size)
    q_size = min(1 / k_size, 1e4) if dtype == "f16" else 1 / k_size   # (1e5 passes fp16's range)
    q, q_dev = as_dtype(g.standard_normal((len(kv) * ql, hq, d)) * q_size, dtype)
    slopes = (2.0 ** -(8.0 * np.arange(1, hq + 1) / hq)).astype(np.float32) if mods.pop("slopes", 0) else None
    prefix = mods.pop("prefix", None)
    scale, out = 1 / math.sqrt(d), torch.full_like(q_dev, 7.0)
    K.q4_paged_attention(
        q_dev, out, torch.from_numpy(pool).cuda(), torch.from_numpy(tables).cuda(),
        torch.tensor(kv, dtype=torch.int32).cuda(), q_per_seq=ql, scale=scale,
        alibi_slopes=None if slopes is None else torch.from_numpy(slopes).cuda(),
        prefix_lens=None if prefix is None else torch.tensor(prefix, dtype=torch.int32).cuda(), **mods)
    K.check_device_errors()
    got, want = out.double().cpu().numpy(), []
    for s, n in enumerate(kv):
        rows = slice(s * ql, (s + 1) * ql)
        pos = np.arange(n)
        k, v = R.read_rows(pool, d, tables[s, pos // 16] * 16 + pos % 16)
        see = R.visible(ql, n, True, mods.get("window", 0), prefix[s] if prefix else 0)
        how = (scale, see, mods.get("softcap", 0.0), slopes)
        o, _, _ = B.attention(q[rows], k, v, *how)
        (ks, kb), (vs, vb) = (parameters(pool, d, par, tables[s], pos) for par in (16 * d, 16 * d + 64))
        code = [np.where(p[0][..., None] > 0, np.rint((x - p[1][..., None]) /
                np.where(p[0] > 0, p[0], 1.0)[..., None]), 0) for x, p in ((k, (ks, kb)), (v, (vs, vb)))]
        _, _, size = B.attention(q[rows], B.parts(code[0], ks, kb, dtype == "f32"), v, *how)
        _, mag, _ = B.attention(q[rows], k, B.parts(code[1], vs, vb, dtype != "bf16"), *how)
        tol = B.exact_code_bound(dtype, o, size, mag, n, d, mods.get("softcap", 0.0), slopes)
        err = np.abs(got[rows] - o)
        assert (err <= tol).all(), f"{(err / tol).max():.2f} times the bound"
        want.append(o)
    want = np.concatenate(want)
    assert B.rms(got - want) <= B.RMS[dtype] * B.rms(want)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hq,hkv,d,ql", [(8, 2, 128, 1), (40, 8, 128, 5), (4, 1, 64, 9), (4, 2, 256, 2),
                                         (6, 2, 64, 40), (2, 1, 256, 1)])
def test_types(dtype, hq, hkv, d, ql):
    check(300, dtype, hq, hkv, d, [ql + 30, ql + 300, ql + 700], ql)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", [1e-2, 1e-4, 1e-5])
def test_rows_of_any_size(dtype, size):
    # (an fp16 output of size 1e-5 is subnormal itself: larger values there)
    check(301, dtype, 8, 2, 128, [100, 400], 3, k_size=size, v_size=1.0 if dtype == "f16" else size)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("mods", [dict(softcap=5.0), dict(window=20), dict(slopes=True),
                                  dict(window=16, prefix=[5, 33])])
def test_modified_scores(dtype, mods):
    check(302, dtype, 8, 2, 128, [300, 500], 4, **mods)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_long_runs_of_the_types_that_stay(dtype):
    check(303, dtype, 8, 2, 128, [420, 260], 150)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hq,hkv,d,ql,tokens", [(16, 8, 128, 1, 131072), (16, 8, 128, 5, 60000),
                                                (8, 8, 64, 1, 131072), (8, 8, 256, 1, 40000)])
def test_sums_over_long_contexts(dtype, hq, hkv, d, ql, tokens):
    """Flat weights (q = 0) over many keys: the output is the values' mean, far smaller than they
    are, so a sum that loses a little of itself with each key would show.  Enough sequences (of
    the same pages) that a thread block takes whole contexts."""
    g = torch.Generator(device="cuda").manual_seed(7)
    seqs, blocks = 72, tokens // 16
    pool = torch.zeros((blocks, hkv, R.record_bytes(d)), dtype=torch.uint8, device="cuda")
    rows = torch.randn((2, tokens, hkv, d), generator=g, device="cuda")
    index = torch.arange(tokens, device="cuda")
    K.q4_reshape_and_cache(rows[0], rows[1], pool, index)
    values = K.q4_gather_kv(pool, index, torch.float32)[1][0].double()     # (H, tokens, d)
    q = torch.zeros((seqs * ql, hq, d), device="cuda").to(TORCH_DT[dtype])
    out = torch.full_like(q, 7.0)
    tables = torch.arange(blocks, dtype=torch.int32, device="cuda").expand(seqs, -1).contiguous()
    kv = torch.full((seqs,), tokens, dtype=torch.int32, device="cuda")
    K.q4_paged_attention(q, out, pool, tables, kv, q_per_seq=ql, scale=1 / math.sqrt(d))
    K.check_device_errors()
    sums = values.sum(1) - torch.stack([values[:, tokens - ql + 1 + i:].sum(1) for i in range(ql)])
    count = tokens - ql + 1 + torch.arange(ql, device="cuda").view(-1, 1, 1)
    want = (sums / count).repeat_interleave(hq // hkv, 1)                   # (ql, hq, d)
    got = out.view(seqs, ql, hq, d).double()
    off = (got - want).square().mean().sqrt()
    assert off <= B.RMS[dtype] * want.square().mean().sqrt()
