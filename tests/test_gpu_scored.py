"""
Attention with modified scores (cap, distance bias, window, prefix) over 16- and 32-bit
pools, against its definition in 64 bits.
"""

import math

import numpy as np
import pytest
import torch

from tests import q4_reference as R
from tests.gpu_util import TORCH_DT
from tests.test_gpu_q4 import as_dtype, rng, tables_for

pytestmark = pytest.mark.gpu

K = pytest.importorskip("memforge_b200._kernels")

MODS = [dict(softcap=5.0), dict(window=20), dict(slopes=True), dict(prefix=[40, 0, 7, 200]),
        dict(window=16, prefix=[5, 17, 0, 33]), dict(window=1),
        dict(softcap=2.0, window=33, slopes=True, prefix=[3, 64, 16, 1])]


class Case:
    def __init__(self, seed, dtype, hq, hkv, d, kv_lens, q_lens, causal=True, softcap=0.0,
                 window=0, slopes=False, prefix=None, block=16, q_scale=1.0):
        g = rng(seed)
        self.dtype, self.hq, self.hkv, self.d, self.block = dtype, hq, hkv, d, block
        self.kv_lens, self.q_lens, self.causal = list(kv_lens), list(q_lens), causal
        self.softcap, self.window = softcap, window
        self.tables, blocks = tables_for(g, kv_lens) if block == 16 else (None, 0)
        if block != 16:
            need = max((n + block - 1) // block for n in kv_lens)
            blocks = need * len(kv_lens) + 2
            self.tables = g.permutation(blocks)[:need * len(kv_lens)].reshape(-1, need).astype(np.int32)
        pools = []
        for _ in range(2):
            x, t = as_dtype(g.standard_normal((blocks, block, hkv, d)), dtype)
            for i, n in enumerate(kv_lens):  # slots behind the last token: NaN
                if n % block:
                    t[self.tables[i, n // block], n % block:] = math.nan
            pools.append((x, t))
        (self.k, self.k_dev), (self.v, self.v_dev) = pools
        self.q, self.q_dev = as_dtype(g.standard_normal((sum(q_lens), hq, d)) * q_scale, dtype)
        self.slopes = (2.0 ** -(8.0 * np.arange(1, hq + 1) / hq)).astype(np.float32) if slopes else None
        self.prefix = None if prefix is None else np.asarray(prefix, np.int32)
        self.scale = 1 / math.sqrt(d)

    def run(self, q=None, out=None, **kw):
        q = self.q_dev if q is None else q
        out = torch.full_like(q, 7.0) if out is None else out
        args = dict(scale=self.scale, causal=self.causal, softcap=self.softcap, window=self.window,
                    alibi_slopes=None if self.slopes is None else torch.from_numpy(self.slopes).cuda(),
                    prefix_lens=None if self.prefix is None else torch.from_numpy(self.prefix).cuda())
        if len(set(self.q_lens)) == 1:
            args["q_per_seq"] = self.q_lens[0]
        else:
            args["cu_seqlens_q"] = torch.tensor(np.concatenate([[0], np.cumsum(self.q_lens)]),
                                                dtype=torch.int32).cuda()
            args["max_q_len"] = max(self.q_lens)
        args.update(kw)
        K.paged_attention(q, out, self.k_dev, self.v_dev, torch.from_numpy(self.tables).cuda(),
                          torch.tensor(self.kv_lens, dtype=torch.int32).cuda(), **args)
        torch.cuda.synchronize()
        return out

    def want(self):
        """Exact output, and the bound of the kernel's distance from it.

        Bound, elementwise: the output's own rounding (eps / 2 of |out|); P rounded to the
        pool's 16-bit type (eps / 2 of each weight: times sum w |v|); a score off by delta
        moves each weight by at most 4 delta of sum w |v| (top and bottom of the quotient),
        delta = D 2^-24 scale sum|q| max|k| for the fp32 sums, plus 2^-21 for the
        exponential and 2^-21 cap for the cap's.
        """
        outs, tols, at = [], [], 0
        fin = torch.finfo(TORCH_DT[self.dtype])
        for s, (n, ql) in enumerate(zip(self.kv_lens, self.q_lens)):
            q = self.q[at:at + ql]
            at += ql
            pos = np.arange(n)
            slots = self.tables[s, pos // self.block] * self.block + pos % self.block
            k = self.k.reshape(-1, self.hkv, self.d)[slots]
            v = self.v.reshape(-1, self.hkv, self.d)[slots]
            see = R.visible(ql, n, self.causal, self.window,
                            0 if self.prefix is None else int(self.prefix[s]))
            o, mag = R.attention(q, k, v, self.scale, see, self.softcap, self.slopes)
            size = self.scale * np.abs(q).sum(-1, keepdims=True) * np.abs(k).max(initial=0.0)
            delta = self.d * 2.0 ** -24 * size + 2.0 ** -21 * (1 + self.softcap)
            p = fin.eps / 2 if self.dtype != "f32" else 2.0 ** -22
            outs.append(o)
            tols.append(fin.eps / 2 * np.abs(o) + (p + 4 * delta) * mag + 1e-30)
        return np.concatenate(outs), np.concatenate(tols)

    def check(self, **kw):
        got = self.run(**kw).double().cpu().numpy()
        want, tol = self.want()
        K.check_device_errors()
        assert np.isfinite(got).all()
        err = np.abs(got - want)
        assert (err <= tol).all(), f"{(err - tol).max():.3e} beyond the bound, err {err.max():.3e}"
        return got


@pytest.mark.parametrize("mods", MODS)
@pytest.mark.parametrize("dtype,hq,hkv,d,ql", [
    ("bf16", 8, 2, 128, 1), ("f16", 4, 4, 64, 1), ("f32", 4, 2, 80, 3), ("bf16", 8, 1, 128, 1),
    ("bf16", 8, 2, 128, 2), ("bf16", 8, 2, 64, 13), ("bf16", 8, 2, 128, 37), ("f16", 16, 1, 128, 5),
    ("f16", 6, 2, 128, 150), ("bf16", 2, 1, 256, 9)])
def test_modified_scores(mods, dtype, hq, hkv, d, ql):
    Case(31, dtype, hq, hkv, d, [ql, 100 + ql, 257, 400], [ql] * 4, **mods).check()


@pytest.mark.parametrize("mods", [dict(softcap=3.0), dict(window=40, prefix=[9, 70, 0, 300, 1]),
                                  dict(slopes=True)])
def test_ragged_runs_short_and_long(mods):
    """One-row runs beside long ones: the decode and the chunk kernel in one call."""
    Case(32, "bf16", 8, 2, 128, [300, 500, 40, 700, 33], [1, 140, 2, 300, 0], **mods).check()


def test_long_sequences_split_over_many_ranges():
    c = Case(33, "bf16", 16, 8, 128, [5000, 2600, 17], [1] * 3, softcap=30.0, window=2000,
             prefix=[100, 0, 17])
    assert np.array_equal(c.check(), c.run().double().cpu().numpy())


@pytest.mark.parametrize("window", [1, 15, 16, 17, 127, 128, 129, 1000])
@pytest.mark.parametrize("ql", [1, 200])
def test_windows_around_page_and_tile_borders(window, ql):
    Case(34, "bf16", 4, 1, 128, [ql + 300, ql + 17, 640], [ql] * 3, window=window).check()


@pytest.mark.parametrize("prefix", [[1, 16], [127, 128], [129, 511], [600, 10000]])
def test_prefixes_around_page_and_tile_borders(prefix):
    """A prefix longer than the sequence is the whole of it; rows inside it see ahead."""
    Case(35, "bf16", 4, 1, 128, [400, 600], [250] * 2, prefix=prefix).check()
    Case(36, "bf16", 4, 1, 128, [400, 600], [250] * 2, prefix=prefix, window=60).check()


def test_many_sequences():
    g = rng(37)
    kv = g.integers(1, 90, 260).tolist()
    Case(37, "bf16", 4, 2, 128, kv, [1] * 260, window=23, softcap=4.0).check()


def test_rows_that_see_nothing_are_zeros():
    """kv_len 0 and rows before the first key come out as zeros, with no error."""
    for ql, dtype, d in ((1, "bf16", 128), (4, "bf16", 128), (40, "bf16", 128), (4, "f32", 80)):
        c = Case(38, dtype, 4, 2, d, [0, 2, 50, 0], [ql] * 4, softcap=9.0)
        got = c.check()
        assert not got[:ql].any() and not got[3 * ql:].any()


def test_non_causal():
    Case(39, "bf16", 8, 2, 128, [50, 9], [7] * 2, causal=False, softcap=3.0).check()
    Case(40, "bf16", 8, 2, 128, [150, 90], [1] * 2, causal=False, window=20).check()


def test_other_block_sizes_and_large_scores():
    Case(41, "f32", 4, 2, 64, [50, 9], [2] * 2, block=8, softcap=3.0).check()
    # scores of a hundred and more, far above the cap
    Case(42, "bf16", 4, 2, 128, [200, 90], [1] * 2, softcap=50.0, q_scale=30.0).check()
    Case(43, "bf16", 4, 2, 128, [200, 90], [40] * 2, softcap=50.0, q_scale=30.0).check()


def test_strides_and_row_map():
    c = Case(44, "bf16", 6, 2, 128, [50, 20], [3, 2], window=9)
    wide_q = torch.zeros((7, 6, 131), dtype=torch.bfloat16, device="cuda")
    perm = torch.tensor([3, 0, 4, 1, 2], dtype=torch.int32, device="cuda")
    wide_q[perm.long(), :, 1:129] = c.q_dev
    wide_o = torch.full((7, 6, 133), 5.0, dtype=torch.bfloat16, device="cuda")
    c.run(q=wide_q[:, :, 1:129], out=wide_o[:, :, 2:130],
          row_map=torch.cat([perm, torch.tensor([5, 6], dtype=torch.int32, device="cuda")]))
    want, tol = c.want()
    got = wide_o[perm.long(), :, 2:130].double().cpu().numpy()
    assert (np.abs(got - want) <= tol).all()
    assert (wide_o[5:] == 5.0).all() and (wide_o[:, :, :2] == 5.0).all()


def test_no_modifier_is_plain_attention():
    from memforge_b200.scored_attention import paged_attention_scored
    c = Case(45, "bf16", 8, 2, 128, [300, 77], [1, 1])
    out = paged_attention_scored(c.q_dev, c.k_dev[None], c.v_dev[None], 0,
                                 torch.from_numpy(c.tables).cuda(),
                                 torch.tensor(c.kv_lens, dtype=torch.int32).cuda())
    assert torch.equal(out, c.run())


def test_graph_replays_on_two_streams_and_new_lengths():
    c = Case(46, "bf16", 16, 8, 128, [900, 400, 33], [1] * 3, window=300, softcap=20.0)
    tables, kv = torch.from_numpy(c.tables).cuda(), torch.tensor(c.kv_lens, dtype=torch.int32).cuda()
    how = dict(scale=c.scale, softcap=20.0, window=300)
    K.paged_attention(c.q_dev, torch.empty_like(c.q_dev), c.k_dev, c.v_dev, tables, kv, **how)
    graphs, outs = [], []
    for _ in range(2):
        g, out = torch.cuda.CUDAGraph(), torch.empty_like(c.q_dev)
        with torch.cuda.graph(g):
            K.paged_attention(c.q_dev, out, c.k_dev, c.v_dev, tables, kv, **how)
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
    c.kv_lens = [33, 16, 32]
    kv.copy_(torch.tensor(c.kv_lens, dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    want, tol = c.want()
    assert (np.abs(outs[0].double().cpu().numpy() - want) <= tol).all()


def test_bad_tables_are_reported():
    c = Case(47, "bf16", 4, 2, 128, [100, 60], [1, 1], window=1000)
    c.tables[1, 1] = 10 ** 6
    c.run()
    with pytest.raises(IndexError, match="block table entry"):
        K.check_device_errors()


@pytest.mark.parametrize("dtype,d,ql", [("bf16", 128, 2), ("bf16", 128, 200), ("f32", 80, 6)])
def test_the_widest_window_hides_nothing(dtype, d, ql):
    c = Case(40, dtype, 8, 2, d, [max(ql // 2, 1), 3 * ql + 40], [ql] * 2, window=2 ** 31 - 1)
    got = c.check()
    assert (c.run(window=1 << 20) == torch.from_numpy(got).cuda().to(TORCH_DT[dtype])).all()


@pytest.mark.parametrize("softcap", [1e-30, 1e-3, 1e5, 1e7, 1e30])
@pytest.mark.parametrize("dtype,d,ql", [("bf16", 128, 1), ("bf16", 128, 60), ("f32", 80, 2)])
def test_caps_far_from_the_scores(softcap, dtype, d, ql):
    # Beyond the scores a cap leaves them as they are: its error scales with the scores
    # (at most 4 * 2^-21 of the largest), not with the cap; below them, with the cap.
    c = Case(41, dtype, 8, 2, d, [90, 300], [ql] * 2, softcap=softcap)
    want, tol = c.want()
    if softcap > 1:
        c.softcap = 0.0
        tol = c.want()[1]
        size = c.scale * np.abs(c.q).sum(-1, keepdims=True) * np.abs(c.k).max()
        tol = tol + 4 * 4 * 2.0 ** -21 * size * np.abs(c.v).max()
        c.softcap = softcap
    got = c.run().double().cpu().numpy()
    K.check_device_errors()
    assert (np.abs(got - want) <= tol).all()


def test_an_aborted_launch_leaves_no_counters_behind():
    c = Case(42, "bf16", 8, 2, 128, [4000, 33], [1, 1], window=500)
    c.check()
    ws = K._stream_workspaces[(0, torch.cuda.current_stream().cuda_stream)]
    ws[:64] = 7   # as a launch that gave up in mid-way would leave them
    K.err_word(torch.device("cuda", 0)).fill_(1)
    with pytest.raises(IndexError):
        K.check_device_errors()
    c.check()
