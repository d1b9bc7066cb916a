"""
The 4-bit KV cache on the GPU against its definition in 64 bits: write and read
bit-exact, attention within bounds derived in tests/q4_reference.py.
"""

import math

import numpy as np
import pytest
import torch

from tests import q4_reference as R
from tests.gpu_util import TORCH_DT

pytestmark = pytest.mark.gpu

K = pytest.importorskip("memforge_b200._kernels")


def rng(seed):
    return np.random.default_rng(seed)


def as_dtype(x, dtype):
    """fp64 values rounded to `dtype`, and the CUDA tensor that holds them."""
    t = torch.from_numpy(np.ascontiguousarray(x)).to(TORCH_DT[dtype])
    return t.double().numpy(), t.cuda()


def random_pool(g, blocks, heads, d, spread=1.0):
    """A packed pool of random codes and parameters (uint8 numpy)."""
    pool = g.integers(0, 256, (blocks, heads, R.record_bytes(d)), dtype=np.uint8)
    scale = (0.05 + 0.4 * g.random((blocks, heads, 2, 16))) * spread
    base = -7.5 * scale + 0.3 * g.standard_normal(scale.shape) * spread
    par = np.stack([scale, base], -1).astype(np.float16)
    pool[:, :, 16 * d:] = par.reshape(blocks, heads, -1).view(np.uint8)
    return pool


def tables_for(g, kv_lens, spare=3, width=None):
    need = [(n + 15) // 16 for n in kv_lens]
    blocks = sum(need) + spare
    perm = g.permutation(blocks)
    width = max(need + [1]) if width is None else width
    t = np.zeros((len(kv_lens), width), np.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = perm[at:at + n]
        at += n
    return t, blocks


class Case:
    def __init__(self, seed, dtype, hq, hkv, d, kv_lens, q_lens, causal=True, softcap=0.0,
                 window=0, slopes=False, prefix=None, spread=1.0, poison=True, q_scale=1.0):
        g = rng(seed)
        self.dtype, self.hq, self.hkv, self.d = dtype, hq, hkv, d
        self.kv_lens, self.q_lens, self.causal = list(kv_lens), list(q_lens), causal
        self.softcap, self.window = softcap, window
        self.tables, blocks = tables_for(g, kv_lens)
        self.pool = random_pool(g, blocks, hkv, d, spread)
        if poison:  # slots behind the last token hold NaN parameters
            for i, n in enumerate(kv_lens):
                if n % 16:
                    par = self.pool[self.tables[i, n // 16]][:, 16 * d:].reshape(hkv, 2, 16, 4)
                    par[:, :, n % 16:] = 0xFF
                    self.pool[self.tables[i, n // 16]][:, 16 * d:] = par.reshape(hkv, -1)
        rows = sum(q_lens)
        self.q, self.q_dev = as_dtype(g.standard_normal((rows, hq, d)) * q_scale, dtype)
        self.slopes = (2.0 ** -(8.0 * np.arange(1, hq + 1) / hq)).astype(np.float32) if slopes else None
        self.prefix = None if prefix is None else np.asarray(prefix, np.int32)
        self.scale = 1 / math.sqrt(d)

    def mods(self):
        return dict(softcap=self.softcap, window=self.window,
                    alibi_slopes=None if self.slopes is None else torch.from_numpy(self.slopes).cuda(),
                    prefix_lens=None if self.prefix is None else torch.from_numpy(self.prefix).cuda())

    def rows(self):
        if len(set(self.q_lens)) == 1:
            return dict(q_per_seq=self.q_lens[0])
        cu = torch.tensor(np.concatenate([[0], np.cumsum(self.q_lens)]), dtype=torch.int32).cuda()
        return dict(cu_seqlens_q=cu, max_q_len=max(self.q_lens))

    def run(self, q=None, out=None, **kw):
        q = self.q_dev if q is None else q
        out = torch.full_like(q, 7.0) if out is None else out
        args = dict(scale=self.scale, causal=self.causal, **self.rows(), **self.mods())
        args.update(kw)
        K.q4_paged_attention(q, out, torch.from_numpy(self.pool).cuda(),
                             torch.from_numpy(self.tables).cuda(),
                             torch.tensor(self.kv_lens, dtype=torch.int32).cuda(), **args)
        torch.cuda.synchronize()
        return out

    def want(self):
        outs, tols, at = [], [], 0
        for s, (n, ql) in enumerate(zip(self.kv_lens, self.q_lens)):
            q = self.q[at:at + ql]
            at += ql
            pos = np.arange(n)
            k, v = R.read_rows(self.pool, self.d, self.tables[s, pos // 16] * 16 + pos % 16) \
                if n else (np.zeros((0, self.hkv, self.d)),) * 2
            see = R.visible(ql, n, self.causal, self.window,
                            0 if self.prefix is None else int(self.prefix[s]))
            o, _ = R.attention(q, k, v, self.scale, see, self.softcap, self.slopes)
            size = np.nanmax(np.abs(np.concatenate([k, v])), initial=0.0)
            # |n * scale| and |base| of a row are at most its largest value plus its
            # span; three times the largest magnitude bounds their sum
            outs.append(o)
            chunk = self.d == 128 and self.dtype != "f32" and ql * self.hq // self.hkv > 32
            tols.append(R.q4_tolerance(self.dtype, o, q, 3 * size, 3 * size, self.scale, chunk))
        return np.concatenate(outs), np.concatenate(tols)

    def check(self, **kw):
        got = self.run(**kw).double().cpu().numpy()
        want, tol = self.want()
        K.check_device_errors()
        assert np.isfinite(got).all()
        err = np.abs(got - want)
        assert (err <= tol).all(), f"{(err - tol).max():.3e} beyond the bound, err {err.max():.3e}"
        return got


# ------------------------------------------------------------- write and read

@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d,heads,tokens", [(64, 1, 1), (128, 8, 33), (256, 3, 50), (128, 2, 17)])
def test_write_then_read_is_the_definition(dtype, d, heads, tokens):
    g = rng(tokens + d)
    kx, k = as_dtype(g.standard_normal((tokens, heads, d)) * 2 + 0.5, dtype)
    vx, v = as_dtype(g.standard_normal((tokens, heads, d)) * 0.01 - 3, dtype)
    blocks = tokens // 16 + 4
    pool = torch.from_numpy(random_pool(g, blocks, heads, d)).cuda()
    before = pool.cpu().numpy()
    slots = g.permutation(blocks * 16)[:tokens]
    K.q4_reshape_and_cache(k, v, pool, torch.from_numpy(slots).cuda())
    after = pool.cpu().numpy()
    want = before.copy()
    for t, s in enumerate(slots):
        for h in range(heads):
            R.write_token(want, d, s // 16, s % 16, h, kx[t, h], vx[t, h])
    assert np.array_equal(after, want)  # written slots exactly, the others untouched
    for index in (slots.astype(np.int64), slots.astype(np.int32)):
        kr, vr = K.q4_gather_kv(pool, torch.from_numpy(index).cuda(), TORCH_DT[dtype])
        for got, x in ((kr, kx), (vr, vx)):
            code, scale, base = R.quantise(x)
            exact = torch.from_numpy((code * scale[..., None] + base[..., None]).astype(np.float32))
            assert torch.equal(got[0].cpu(), exact.to(TORCH_DT[dtype]).transpose(0, 1))
    K.check_device_errors()


def test_write_of_special_rows():
    """Ties, constants, zeros, denormals, the largest magnitudes, NaN and infinities."""
    d = 64
    rows = [np.zeros(d), np.full(d, 3.3), np.full(d, -1e-30), np.full(d, 65504.0),
            np.concatenate([np.arange(16) + 0.5, np.arange(16), [0, 15], np.full(30, 7.5)]),
            np.concatenate([[0.0, 15.0], np.tile(np.arange(15) + 0.5, 4), [1, 2]]),
            np.concatenate([[-65504.0, 65504.0], np.linspace(-6e4, 6e4, 62)]),
            np.linspace(0, 6e-8, d), np.linspace(-1e-6, 1e-6, d), np.linspace(0, 1e-38, d),
            np.concatenate([[65505.0], np.zeros(63)]), np.concatenate([[np.nan], np.ones(63)]),
            np.concatenate([np.ones(63), [np.inf]]), np.concatenate([[-np.inf], np.ones(63)]),
            np.concatenate([[-0.0, 0.0], np.full(62, 1e-3)])]
    x = np.stack(rows)[:, None].astype(np.float32).astype(np.float64)
    T = len(rows)
    k = torch.from_numpy(x).float().cuda()
    pool = torch.zeros((T // 16 + 1, 1, R.record_bytes(d)), dtype=torch.uint8, device="cuda")
    want = pool.cpu().numpy()
    K.q4_reshape_and_cache(k, k, pool, torch.arange(T, device="cuda"))
    got = pool.cpu().numpy()
    good = [t for t in range(T) if (np.abs(x[t]) <= 65504).all()]
    for t in good:
        R.write_token(want, d, t // 16, t % 16, 0, x[t, 0], x[t, 0])
    kg, vg = R.read_rows(got, d, np.arange(T))
    kw, vw = R.read_rows(want, d, np.arange(T))
    assert np.array_equal(kg[good], kw[good]) and np.array_equal(vg[good], vw[good])
    bad = [t for t in range(T) if t not in good]
    assert len(bad) == 4 and np.isnan(kg[bad]).all() and np.isnan(vg[bad]).all()


def test_random_borders_are_decided_exactly():
    """fp32 rows whose elements lie on, just above and just below half codes."""
    g = rng(5)
    d, T = 128, 64
    scale = 2.0 ** g.integers(-8, 4, (T, 1)) * (1 + g.integers(0, 1024, (T, 1)) / 1024)
    x = scale * (g.integers(0, 15, (T, d)) + 0.5)
    x[:, 0], x[:, 1] = 0.0, 15 * scale[:, 0]
    near = np.float32(x)
    near[:, 2::3] = np.nextafter(near[:, 2::3], np.float32(np.inf))
    near[:, 3::3] = np.nextafter(near[:, 3::3], np.float32(-np.inf))
    xs = near.astype(np.float64)[:, None]
    k = torch.from_numpy(near[:, None]).cuda()
    pool = torch.zeros((T // 16, 1, R.record_bytes(d)), dtype=torch.uint8, device="cuda")
    K.q4_reshape_and_cache(k, k, pool, torch.arange(T, device="cuda"))
    kr, vr = R.read_rows(pool.cpu().numpy(), d, np.arange(T))
    want = R.dequantised(xs)
    assert np.array_equal(kr, want) and np.array_equal(vr, want)


def test_write_reads_any_strides_and_skips():
    g = rng(6)
    T, H, d = 21, 3, 128
    wide = torch.from_numpy(g.standard_normal((T, 2 * H + 1, d + 5))).to(torch.bfloat16).cuda()
    k, v = wide[:, 1:2 * H:2, 3:3 + d], wide[:, 0:2 * H:2, 1:1 + d]  # odd offsets: scalar loads
    slots = torch.from_numpy(g.permutation(48)[:T]).cuda()
    slots[[2, 7]] = -1
    a = torch.zeros((3, H, R.record_bytes(d)), dtype=torch.uint8, device="cuda")
    # records of a wider pool: strides of their own
    big = torch.zeros((3, 2 * H, R.record_bytes(d)), dtype=torch.uint8, device="cuda")
    K.q4_reshape_and_cache(k, v, big[:, ::2], slots)
    K.q4_reshape_and_cache(k.contiguous(), v.contiguous(), a, slots.int())
    assert torch.equal(a, big[:, ::2].contiguous()) and not big[:, 1::2].any()
    live = slots >= 0
    for s in range(48):
        if s not in slots[live].tolist():
            assert not a[s // 16, :, 16 * d + 4 * (s % 16):16 * d + 4 * (s % 16) + 4].any()
    K.check_device_errors()


def test_slots_outside_the_pool_are_reported_and_skipped():
    d = 64
    k = torch.ones((3, 1, d), device="cuda")
    pool = torch.zeros((2, 1, R.record_bytes(d)), dtype=torch.uint8, device="cuda")
    K.q4_reshape_and_cache(k, k, pool, torch.tensor([32, -2, 5], device="cuda"))
    with pytest.raises(IndexError, match="slot_mapping"):
        K.check_device_errors()
    kr, _ = K.q4_gather_kv(pool, torch.tensor([5, 32, -1], device="cuda"), torch.float32)
    with pytest.raises(IndexError, match="slot_mapping"):
        K.check_device_errors()
    assert torch.equal(kr[0, 0, 0], torch.ones(d, device="cuda")) and not kr[0, 0, 1:].any()


def test_offsets_past_32_bits():
    """A pool of more than 4 GiB, written and read at its end."""
    d, H = 128, 8
    blocks = (1 << 32) // (H * R.record_bytes(d)) + 50
    pool = torch.empty((blocks, H, R.record_bytes(d)), dtype=torch.uint8, device="cuda")
    g = rng(8)
    x, k = as_dtype(g.standard_normal((20, H, d)), "bf16")
    slots = torch.arange(blocks * 16 - 20, blocks * 16, device="cuda")
    K.q4_reshape_and_cache(k, k, pool, slots)
    kr, vr = K.q4_gather_kv(pool, slots, torch.float32)
    want = torch.from_numpy(R.dequantised(x).astype(np.float32)).transpose(0, 1)
    assert torch.equal(kr[0].cpu(), want) and torch.equal(vr[0].cpu(), want)
    q = torch.from_numpy(g.standard_normal((1, 8, d))).to(torch.bfloat16).cuda()
    tables = torch.tensor([[blocks - 2, blocks - 1]], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    # 20 tokens from slot 12 of the last block but one: read the 4 + 16 live ones by
    # writing the first 12 too
    first = torch.arange(blocks * 16 - 32, blocks * 16 - 20, device="cuda")
    K.q4_reshape_and_cache(k[:12], k[:12], pool, first)
    K.q4_paged_attention(q, out, pool, tables, torch.tensor([32], dtype=torch.int32).cuda(),
                         scale=0.1)
    rows = np.concatenate([R.dequantised(x[:12]), R.dequantised(x)])
    o, _ = R.attention(q.double().cpu().numpy(), rows, rows, 0.1, np.ones((1, 32), bool))
    tol = R.q4_tolerance("bf16", o, q.double().cpu().numpy(), 15.0, 15.0, 0.1)
    assert (np.abs(out.double().cpu().numpy() - o) <= tol).all()


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 1, 128), (4, 4, 64), (14, 2, 128), (32, 8, 128),
                                      (6, 3, 256), (16, 1, 64), (40, 2, 128)])
def test_decode(dtype, hq, hkv, d):
    Case(hq + d, dtype, hq, hkv, d, [1, 77, 300, 16, 17], [1] * 5).check()


@pytest.mark.parametrize("kv", [[1], [15, 16, 17], [63, 64, 65], [2048, 5], [129, 128, 127, 16]])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_lengths_around_pages(kv, d):
    Case(7, "bf16", 8, 2, d, kv, [1] * len(kv)).check()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hq,hkv,d,ql", [(8, 8, 128, 2), (40, 8, 128, 5), (4, 1, 64, 9),
                                         (8, 2, 256, 7), (5, 1, 128, 40), (2, 2, 64, 100)])
def test_several_rows_per_sequence(dtype, hq, hkv, d, ql):
    Case(ql, dtype, hq, hkv, d, [ql, ql + 33, ql + 150], [ql] * 3).check()


def test_ragged_runs_and_empty_ones():
    Case(11, "bf16", 8, 2, 128, [50, 200, 33, 9, 70], [3, 60, 0, 9, 1]).check()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,ql", [(8, 2, 33), (4, 4, 129), (28, 4, 50), (40, 1, 7),
                                       (48, 2, 11), (128, 1, 3)])
def test_long_runs(dtype, hq, hkv, ql):
    """Row tiles of 128 with every GQA size, odd ones included; contexts around key tiles."""
    Case(50 + ql, dtype, hq, hkv, 128, [ql, ql + 127, ql + 128, 700], [ql] * 4).check()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("mods", [dict(), dict(softcap=4.0), dict(window=130, prefix=[20, 300, 0]),
                                  dict(slopes=True)])
def test_runs_of_many_row_tiles(dtype, wide, mods):
    """Runs of four row tiles and more read an expanded copy of the cache, unless the tables'
    width would let it grow past its limit (then they convert as they go): both agree with the
    definition, beside a short run and one without rows."""
    c = Case(60, dtype, 8, 2, 128, [420, 300, 700], [200, 131, 512], **mods)
    if wide:
        t = np.full((3, 30000), -1, np.int32)
        t[:, :c.tables.shape[1]] = c.tables
        c.tables = t
    c.check()
    c = Case(61, dtype, 8, 2, 128, [420, 33, 50, 700], [300, 3, 0, 129])
    c.check()


def test_many_row_tiles_row_map_and_strides():
    c = Case(62, "bf16", 8, 1, 128, [190, 220], [140, 133])
    rows = 273
    wide_q = torch.zeros((rows, 8, 131), dtype=torch.bfloat16, device="cuda")
    perm = torch.from_numpy(rng(62).permutation(rows).astype(np.int32)).cuda()
    wide_q[perm.long(), :, 1:129] = c.q_dev
    wide_o = torch.full((rows, 8, 133), 5.0, dtype=torch.bfloat16, device="cuda")
    c.run(q=wide_q[:, :, 1:129], out=wide_o[:, :, 2:130], row_map=perm)
    want, tol = c.want()
    got = wide_o[perm.long(), :, 2:130].double().cpu().numpy()
    assert (np.abs(got - want) <= tol).all() and (wide_o[:, :, :2] == 5.0).all()


def test_long_runs_non_causal_and_without_keys():
    Case(51, "bf16", 4, 2, 128, [150, 9], [70] * 2, causal=False).check()
    got = Case(52, "bf16", 4, 1, 128, [0, 20, 300], [60] * 3).check()
    assert not got[:60].any() and not got[60:100].any() and got[100:120].any()


def test_long_runs_many_items_per_sm():
    """More (tile, head) items than SMs, ragged: every CTA walks several."""
    g = rng(53)
    ql = g.integers(40, 200, 40).tolist()
    Case(53, "bf16", 16, 8, 128, [q + int(g.integers(0, 300)) for q in ql], ql).check()


def test_long_runs_of_large_values_and_offsets():
    """Rows near fp16's largest number, rows on a large offset, and tiny rows."""
    c = Case(54, "bf16", 4, 2, 128, [200], [50], q_scale=1e-6)
    par = c.pool[:, :, 16 * 128:].view(np.float16).reshape(-1, 2, 2, 16, 2)
    scale = np.zeros_like(par[..., 0])
    base = np.zeros_like(scale)
    scale[..., 0::3], base[..., 0::3] = 8728.0, -65504.0   # codes reach 65416
    scale[..., 1::3], base[..., 1::3] = 0.5, 60000.0
    scale[..., 2::3], base[..., 2::3] = 2.0 ** -24, -2.0 ** -20
    par[..., 0], par[..., 1] = scale, base
    c.check()


def test_long_runs_row_map_and_strides():
    c = Case(55, "bf16", 4, 1, 128, [90, 120], [40, 33])
    rows = 73
    wide_q = torch.zeros((rows + 2, 4, 131), dtype=torch.bfloat16, device="cuda")
    perm = torch.from_numpy(rng(55).permutation(rows).astype(np.int32)).cuda()
    wide_q[perm.long(), :, 1:129] = c.q_dev
    wide_o = torch.full((rows + 2, 4, 133), 5.0, dtype=torch.bfloat16, device="cuda")
    c.run(q=wide_q[:, :, 1:129], out=wide_o[:, :, 2:130],
          row_map=torch.cat([perm, torch.tensor([73, 74], dtype=torch.int32, device="cuda")]))
    want, tol = c.want()
    got = wide_o[perm.long(), :, 2:130].double().cpu().numpy()
    assert (np.abs(got - want) <= tol).all()
    assert (wide_o[rows:] == 5.0).all() and (wide_o[:, :, :2] == 5.0).all()


@pytest.mark.parametrize("window", [1, 16, 127, 128, 129, 300])
def test_long_runs_windows_around_tiles(window):
    Case(56, "bf16", 4, 1, 128, [500, 217, 640], [200] * 3, window=window).check()
    Case(57, "f16", 4, 1, 128, [500, 217, 640], [200] * 3, window=window, prefix=[130, 1, 600]).check()


def test_many_ranges_join():
    """Two long sequences: each unit is cut into many ranges, the joined result repeats."""
    c = Case(12, "bf16", 32, 8, 128, [3000, 1999, 1], [1] * 3)
    first = c.check()
    assert np.array_equal(c.run().double().cpu().numpy(), first)


def test_many_short_sequences():
    g = rng(13)
    kv = g.integers(0, 60, 300).tolist()
    Case(13, "bf16", 4, 2, 64, kv, [1] * 300).check()


@pytest.mark.parametrize("mods", [dict(softcap=5.0), dict(window=20), dict(slopes=True),
                                  dict(prefix=[40, 0, 7, 200]), dict(window=16, prefix=[5, 17, 0, 33]),
                                  dict(softcap=2.0, window=33, slopes=True, prefix=[3, 64, 16, 1]),
                                  dict(window=1)])
@pytest.mark.parametrize("dtype,ql", [("bf16", 1), ("f16", 6), ("f32", 3), ("bf16", 37)])
def test_modified_scores(mods, dtype, ql):
    Case(14, dtype, 8, 2, 128, [ql, 100, 257, 400], [ql] * 4, **mods).check()


@pytest.mark.parametrize("d", [64, 256])
def test_modified_scores_other_head_dims(d):
    Case(15, "bf16", 4, 2, d, [90, 300], [5] * 2, softcap=3.0, window=50, prefix=[10, 20]).check()


def test_rows_that_see_nothing_are_zeros():
    """kv_len 0, and rows before the first key (kv_len < q_len)."""
    c = Case(16, "bf16", 4, 2, 128, [0, 2, 40, 0], [4] * 4)
    got = c.check()
    assert not got[0:4].any() and not got[4:6].any() and not got[12:].any() and got[6:8].any()


def test_non_causal():
    Case(17, "bf16", 8, 2, 128, [50, 9], [7] * 2, causal=False).check()


def test_scales_of_very_different_sizes():
    """Pages whose scales differ by factors of 2^16, in both orders; tiny and large q."""
    for flip in (False, True):
        for q_scale in (1e-3, 30.0):
            c = Case(18, "bf16", 8, 2, 128, [160], [1], q_scale=q_scale)
            par = c.pool[:, :, 16 * 128:].view(np.float16).reshape(-1, 2, 2, 16, 2)
            order = np.arange(10)[::-1] if flip else np.arange(10)
            for i, blk in enumerate(c.tables[0, order]):
                par[blk, :, 1] = par[blk, :, 1] * np.float16(2.0 ** (i - 8) * 4 ** (i // 5))
            c.check()


def test_a_row_of_nan_keys_spoils_only_rows_that_see_it():
    c = Case(19, "bf16", 4, 2, 128, [40], [8])
    blk, t = c.tables[0, 2], 36 % 16  # position 36: rows at 32 .. 35 do not see it
    for par in (16 * 128, 16 * 128 + 64):
        c.pool[blk, :, par + 4 * t:par + 4 * t + 4] = 0xFF
    got = c.run().double().cpu().numpy()
    want, tol = c.want()
    assert (np.abs(got - want)[:4] <= tol[:4]).all() and np.isfinite(got[:4]).all()
    assert np.isnan(got[4:]).all()


def test_a_nan_query_spoils_only_its_row():
    c = Case(20, "bf16", 8, 2, 128, [100, 30], [1, 1])
    q = c.q_dev.clone()
    q[0, 1, 5] = math.nan
    q[1, 6, 0] = math.inf
    got = c.run(q=q).double().cpu().numpy()
    want, tol = c.want()
    ok = np.ones((2, 8), bool)
    ok[0, 1] = ok[1, 6] = False
    assert np.isnan(got[0, 1]).all() and np.isnan(got[1, 6]).all()
    assert (np.abs(got - want)[ok] <= tol[ok]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides_row_map_and_untouched_rows(dtype):
    """Odd strides of q and out, packed rows in another order, rows behind the last sequence."""
    c = Case(21, dtype, 6, 2, 128, [50, 20], [3, 2])
    wide_q = torch.zeros((7, 6, 131), dtype=TORCH_DT[dtype], device="cuda")
    perm = torch.tensor([3, 0, 4, 1, 2], dtype=torch.int32, device="cuda")
    wide_q[perm.long(), :, 1:129] = c.q_dev
    wide_o = torch.full((7, 6, 133), 5.0, dtype=TORCH_DT[dtype], device="cuda")
    c.run(q=wide_q[:, :, 1:129], out=wide_o[:, :, 2:130],
          row_map=torch.cat([perm, torch.tensor([5, 6], dtype=torch.int32, device="cuda")]))
    want, tol = c.want()
    got = wide_o[perm.long(), :, 2:130].double().cpu().numpy()
    assert (np.abs(got - want) <= tol).all()
    assert (wide_o[5:] == 5.0).all() and (wide_o[:, :, :2] == 5.0).all() and (wide_o[:, :, 130:] == 5.0).all()


def test_table_with_row_stride_and_short_table():
    c = Case(22, "bf16", 4, 2, 64, [100, 60], [1, 1])
    want, tol = c.want()
    wide = np.full((2, 20), -1, np.int32)
    wide[:, :c.tables.shape[1]] = c.tables
    view = torch.from_numpy(wide).cuda()[:, :c.tables.shape[1]]
    out = torch.empty_like(c.q_dev)
    pool, kv = torch.from_numpy(c.pool).cuda(), torch.tensor([100, 60], dtype=torch.int32).cuda()
    K.q4_paged_attention(c.q_dev, out, pool, view, kv, scale=c.scale)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
    K.check_device_errors()
    K.q4_paged_attention(c.q_dev, out, pool, view[:, :5], kv, scale=c.scale)  # 100 needs 7
    with pytest.raises(IndexError, match="block table"):
        K.check_device_errors()
    assert (np.abs(out.double().cpu().numpy() - want)[1] <= tol[1]).all()


def test_bad_block_id_is_reported():
    c = Case(23, "bf16", 4, 2, 64, [100], [1], poison=False)
    c.tables[0, 2] = c.pool.shape[0]
    c.run()
    with pytest.raises(IndexError, match="block table entry"):
        K.check_device_errors()


def test_run_longer_than_declared_is_reported():
    c = Case(24, "bf16", 4, 2, 64, [100, 50], [6, 2])
    c.run(max_q_len=4)
    with pytest.raises(IndexError, match="length"):
        K.check_device_errors()


def test_graph_replay_reads_new_lengths_and_two_graphs_do_not_share():
    c = Case(25, "bf16", 32, 8, 128, [900, 400, 33], [1] * 3)
    pool, tables = torch.from_numpy(c.pool).cuda(), torch.from_numpy(c.tables).cuda()
    kv = torch.tensor(c.kv_lens, dtype=torch.int32).cuda()
    outs, graphs = [], []
    K.q4_paged_attention(c.q_dev, torch.empty_like(c.q_dev), pool, tables, kv, scale=c.scale)
    for _ in range(2):
        g, out = torch.cuda.CUDAGraph(), torch.empty_like(c.q_dev)
        with torch.cuda.graph(g):
            K.q4_paged_attention(c.q_dev, out, pool, tables, kv, scale=c.scale)
        graphs.append(g)
        outs.append(out)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    want, tol = c.want()
    for out in outs:
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
    c.kv_lens = [100, 401, 0]
    kv.copy_(torch.tensor(c.kv_lens, dtype=torch.int32))
    # the poison of the old lengths lies behind these
    graphs[0].replay()
    torch.cuda.synchronize()
    want, tol = c.want()
    assert (np.abs(outs[0].double().cpu().numpy() - want)[[0, 2]] <= tol[[0, 2]]).all()


def test_write_then_attend_on_another_stream():
    c = Case(26, "bf16", 8, 2, 128, [64], [1], poison=False)
    g = rng(26)
    x, k = as_dtype(g.standard_normal((64, 2, 128)), "bf16")
    pool = torch.from_numpy(c.pool).cuda()
    flat = torch.from_numpy(c.tables[0, np.arange(64) // 16] * 16 + np.arange(64) % 16).cuda()
    tables, kv = torch.from_numpy(c.tables).cuda(), torch.tensor([64], dtype=torch.int32).cuda()
    out = torch.empty_like(c.q_dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        K.q4_reshape_and_cache(k, k, pool, flat)
        K.q4_paged_attention(c.q_dev, out, pool, tables, kv, scale=c.scale)
    s.synchronize()
    rows = R.dequantised(x)
    o, _ = R.attention(c.q, rows, rows, c.scale, np.ones((1, 64), bool))
    tol = R.q4_tolerance("bf16", o, c.q, 15.0, 15.0, c.scale)
    assert (np.abs(out.double().cpu().numpy() - o) <= tol).all()


@pytest.mark.parametrize("window", [1, 16, 127, 128, 129, 300])
@pytest.mark.parametrize("wide", [False, True])
def test_many_row_tiles_windows_around_tiles(window, wide):
    """Enough heads that the tensor-core kernels take the runs, expanded and converting."""
    for mods in (dict(), dict(prefix=[130, 1, 600])):
        c = Case(63, "bf16", 16, 4, 128, [500, 217, 640], [200] * 3, window=window, **mods)
        if wide:
            t = np.full((3, 15000), -1, np.int32)
            t[:, :c.tables.shape[1]] = c.tables
            c.tables = t
        c.check()


@pytest.mark.parametrize("wide", [False, True])
def test_many_row_tiles_non_causal_without_keys_and_extremes(wide):
    def run(c):
        if wide:
            t = np.full((len(c.kv_lens), 15000), -1, np.int32)
            t[:, :c.tables.shape[1]] = c.tables
            c.tables = t
        return c.check()
    run(Case(64, "bf16", 16, 4, 128, [150, 9, 400], [130] * 3, causal=False))
    got = run(Case(65, "bf16", 16, 4, 128, [0, 20, 300], [160] * 3))
    assert not got[:160].any() and not got[160:300].any() and got[300:320].any()
    c = Case(66, "bf16", 16, 4, 128, [200, 200, 200], [140] * 3, q_scale=1e-6)
    par = c.pool[:, :, 16 * 128:].view(np.float16).reshape(-1, 4, 2, 16, 2)
    par[:, :, :, 0::3] = (8728.0, -65504.0)   # codes reach 65416
    par[:, :, :, 1::3] = (0.5, 60000.0)
    par[:, :, :, 2::3] = (2.0 ** -24, -2.0 ** -20)
    run(c)


def test_many_row_tiles_of_every_group_size():
    for hq, hkv, ql in ((4, 4, 700), (28, 4, 100), (8, 4, 300), (80, 5, 40), (96, 2, 60)):
        Case(67 + hq, "bf16", hq, hkv, 128, [ql + 5, ql + 300, ql], [ql] * 3).check()


@pytest.mark.parametrize("hq,hkv,kv,ql", [(8, 2, [3, 90], 6), (32, 8, [100, 700], 300),
                                          (32, 8, [20, 400], 60)])
def test_the_widest_window_hides_nothing(hq, hkv, kv, ql):
    c = Case(60, "bf16", hq, hkv, 128, kv, [ql] * 2, window=2 ** 31 - 1)
    got = c.check()
    assert (c.run(window=1 << 20).double().cpu().numpy() == got).all()


@pytest.mark.parametrize("softcap", [1e-30, 1e-3, 1e5, 1e7, 1e30])
@pytest.mark.parametrize("dtype,ql", [("bf16", 1), ("f32", 3)])
def test_caps_far_from_the_scores(softcap, dtype, ql):
    # Beyond the scores a cap leaves them as they are: its error scales with the scores
    # (at most 4 * 2^-21 of the largest), not with the cap.
    c = Case(61, dtype, 8, 2, 128, [90, 300], [ql] * 2, softcap=softcap)
    want, tol = c.want()
    slots = (c.tables[..., None] * 16 + np.arange(16)).reshape(-1)
    k, v = R.read_rows(c.pool, 128, slots[slots >= 0])
    size = c.scale * np.abs(c.q).sum(-1, keepdims=True) * np.nanmax(np.abs(k))
    tol = tol + 4 * 4 * 2.0 ** -21 * np.minimum(size, softcap) * np.nanmax(np.abs(v))
    got = c.run().double().cpu().numpy()
    K.check_device_errors()
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("hq,hkv,ql", [(4, 4, 800), (28, 4, 120), (8, 4, 400), (80, 5, 56),
                                       (9, 3, 300)])
def test_runs_of_six_row_tiles_of_every_group_size(hq, hkv, ql):
    Case(70 + hq, "bf16", hq, hkv, 128, [ql + 5, ql + 300, ql], [ql] * 3).check()


def test_runs_of_six_row_tiles_non_causal_without_keys_and_extremes():
    Case(71, "bf16", 16, 4, 128, [250, 9, 400], [220] * 3, causal=False).check()
    got = Case(72, "bf16", 16, 4, 128, [0, 20, 300], [200] * 3).check()
    assert not got[:200].any() and not got[200:380].any() and got[380:400].any()
    c = Case(73, "bf16", 16, 4, 128, [250, 200, 230], [200] * 3, q_scale=1e-6)
    par = c.pool[:, :, 16 * 128:].view(np.float16).reshape(-1, 4, 2, 16, 2)
    par[:, :, :, 0::3] = (8728.0, -65504.0)   # codes reach 65416
    par[:, :, :, 1::3] = (0.5, 60000.0)
    par[:, :, :, 2::3] = (2.0 ** -24, -2.0 ** -20)
    c.check()
