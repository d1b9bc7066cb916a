"""
Long runs over the 4-bit cache on the tensor-core kernels (converting and expanded), held to
bounds of a few percent of the output (tests/q4_bounds.py).  Every case states which of the
two kernels it is meant for and checks that the call's plan says so.
"""

import ctypes
import math

import numpy as np
import pytest
import torch

from tests import q4_bounds as B
from tests import q4_reference as R
from tests.test_gpu_q4 import as_dtype, random_pool, rng, tables_for

pytestmark = pytest.mark.gpu

K = pytest.importorskip("memforge_b200._kernels")
L = pytest.importorskip("memforge_b200._lib")

D = 128


def form(num_seqs, q_per_seq, hq, hkv, width, rows):
    """Which kernel a call of equal runs takes: the workspace tells.  The mma.sync kernel needs
    some, converting none, and an expanded copy is what it may do without."""
    a = L.Q4AttentionArgs()
    a.struct_size = ctypes.sizeof(a)
    a.q = a.out = a.pool = a.block_tables = a.kv_lens = 0x1000
    a.q_stride_row = a.out_stride_row = hq * D
    a.q_stride_head = a.out_stride_head = D
    a.pool_stride_block, a.pool_stride_head = hkv * 2176, 2176
    a.num_blocks, a.table_stride, a.table_width = 4, width, width
    a.q_per_seq, a.num_seqs, a.total_q, a.max_q_len = q_per_seq, num_seqs, rows, q_per_seq
    a.num_q_heads, a.num_kv_heads, a.head_dim = hq, hkv, D
    a.scale, a.causal, a.dtype = 0.1, 1, L.MF_BF16
    need, least = (f(a, 0) for f in (L.lib().mf_q4_paged_attention_workspace_size,
                                     L.lib().mf_q4_paged_attention_min_workspace_size))
    return "expanded" if need > least else "converting" if need == 0 else "mma.sync"


CONVERTING = dict(hq=16, hkv=4, kv=[200, 527, 640], ql=125)   # 32 row tiles of 16 a head, 4 of 128
EXPANDED = dict(hq=16, hkv=4, kv=[200, 527, 640], ql=200)     # 7 of 128


class Case:
    def __init__(self, seed, hq, hkv, kv, ql, k_size=1.0, v_size=1.0, q_size=None, causal=True,
                 softcap=0.0, window=0, slopes=False, prefix=None):
        g = rng(seed)
        self.hq, self.hkv, self.kv, self.ql = hq, hkv, list(kv), ql
        self.causal, self.softcap, self.window = causal, softcap, window
        self.tables, blocks = tables_for(g, kv)
        self.pool = B.sized_pool(g, blocks, hkv, D, k_size, v_size)
        for i, n in enumerate(kv):  # slots behind the last token: NaN parameters
            if n % 16:
                par = self.pool[self.tables[i, n // 16]][:, 16 * D:].reshape(hkv, 2, 16, 4)
                par[:, :, n % 16:] = 0xFF
                self.pool[self.tables[i, n // 16]][:, 16 * D:] = par.reshape(hkv, -1)
        size = 1 / k_size if q_size is None else q_size
        self.q, self.q_dev = as_dtype(g.standard_normal((len(kv) * ql, hq, D)) * size, "bf16")
        self.slopes = (2.0 ** -(8.0 * np.arange(1, hq + 1) / hq)).astype(np.float32) if slopes else None
        self.prefix = None if prefix is None else np.asarray(prefix, np.int32)
        self.scale = 1 / math.sqrt(D)

    def form(self):
        return form(len(self.kv), self.ql, self.hq, self.hkv, self.tables.shape[1],
                    len(self.kv) * self.ql)

    def args(self, **kw):
        how = dict(q_per_seq=self.ql, scale=self.scale, causal=self.causal, softcap=self.softcap,
                   window=self.window,
                   alibi_slopes=None if self.slopes is None else torch.from_numpy(self.slopes).cuda(),
                   prefix_lens=None if self.prefix is None else torch.from_numpy(self.prefix).cuda())
        how.update(kw)
        return how

    def device(self):
        return (torch.from_numpy(self.pool).cuda(), torch.from_numpy(self.tables).cuda(),
                torch.tensor(self.kv, dtype=torch.int32).cuda())

    def run(self, q=None, out=None, **kw):
        q = self.q_dev if q is None else q
        out = torch.full_like(q, 7.0) if out is None else out
        K.q4_paged_attention(q, out, *self.device(), **self.args(**kw))
        torch.cuda.synchronize()
        return out

    def rows(self, s):
        pos = np.arange(self.kv[s])
        return R.read_rows(self.pool, D, self.tables[s, pos // 16] * 16 + pos % 16)

    def want(self):
        """Outputs over the operands' roundings and their bound, and by the definition."""
        outs, tols, exact = [], [], []
        for s, n in enumerate(self.kv):
            q = self.q[s * self.ql:(s + 1) * self.ql]
            k, v = self.rows(s)
            see = R.visible(self.ql, n, self.causal, self.window,
                            0 if self.prefix is None else int(self.prefix[s]))
            how = (self.scale, see, self.softcap, self.slopes)
            o, mag, size = B.attention(q, B.operand(k), B.operand(v), *how)
            outs.append(o)
            tols.append(B.chunk_bound("bf16", o, mag, size, n, D, self.softcap, self.slopes,
                                      np.abs(v).max(initial=0.0)))
            exact.append(B.attention(q, k, v, *how)[0])
        return np.concatenate(outs), np.concatenate(tols), np.concatenate(exact)

    def hold(self, got):
        want, tol, exact = self.want()
        assert np.isfinite(got).all()
        err = np.abs(got - want)
        assert (err <= tol).all(), (f"{(err > tol).mean():.2%} beyond the bound, worst "
                                    f"{(err / tol).max():.2f} times it")
        assert B.rms(got - exact) <= B.RMS["bf16"] * B.rms(exact)

    def check(self, **kw):
        got = self.run(**kw).double().cpu().numpy()
        K.check_device_errors()
        self.hold(got)
        return got


FORMS = [("converting", CONVERTING), ("expanded", EXPANDED)]


@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4, 3e-5, 1e-5, 1e-6])
@pytest.mark.parametrize("kind,shape", FORMS)
def test_rows_of_any_size(kind, shape, size):
    """Keys and values of one size alone in the pool; q makes up for the keys'."""
    c = Case(80, **shape, k_size=size, v_size=size)
    assert c.form() == kind
    c.check()


@pytest.mark.parametrize("kind,shape", FORMS)
def test_rows_that_reach_the_largest_fp16(kind, shape):
    """Their largest code may stand for up to 120 more, which the kernels hold to 65504."""
    c = Case(82, **shape, k_size=5e4, v_size=5e4)
    assert c.form() == kind
    k, v = c.rows(1)
    assert (k > 65520).any() and (v > 65520).any()
    c.check()


@pytest.mark.parametrize("kind,shape", FORMS)
@pytest.mark.parametrize("which", ["key", "value", "both"])
def test_a_nan_row_spoils_only_rows_that_see_it(kind, shape, which):
    """Late in a run's own rows, where the rows of one tile differ in what they see; and behind
    the window of some of them."""
    for mods in (dict(), dict(window=40), dict(softcap=5.0, prefix=[3, 0, 70])):
        c = Case(81, **shape, **mods)
        assert c.form() == kind
        hit = [(s, n - 37) for s, n in enumerate(c.kv)]
        clean = c.pool.copy()
        for s, at in hit:
            for par in {"key": [0], "value": [64], "both": [0, 64]}[which]:
                first = 16 * D + par + 4 * (at % 16)
                c.pool[c.tables[s, at // 16], 1, first:first + 4] = 0xFF
        got = c.run().double().cpu().numpy()
        K.check_device_errors()
        c.pool = clean
        want, tol, _ = c.want()
        sees = np.concatenate([R.visible(c.ql, n, True, c.window, 0 if c.prefix is None else c.prefix[s])
                               [:, at] for (s, at), n in zip(hit, c.kv)])
        assert sees.any() and not sees.all()
        group = np.arange(c.hq) // (c.hq // c.hkv) == 1   # the head whose row is NaN
        assert np.isnan(got[sees][:, group]).all()
        fine = ~(sees[:, None] & group)
        assert np.isfinite(got[fine]).all() and (np.abs(got - want) <= tol)[fine].all()


@pytest.mark.parametrize("kind,shape", FORMS)
@pytest.mark.parametrize("pad", [-1, 10 ** 6])
def test_entries_of_row_map_behind_the_last_sequence_are_not_followed(kind, shape, pad):
    """A padded batch: rows behind the last sequence, whose entries name no row of q."""
    c = Case(83, **shape)
    rows, spare = len(c.kv) * c.ql, 37
    perm = torch.from_numpy(rng(83).permutation(rows).astype(np.int32)).cuda()
    q = torch.full((rows + spare, c.hq, D), math.nan, dtype=torch.bfloat16, device="cuda")
    q[perm.long()] = c.q_dev
    out = torch.full_like(q, 5.0)
    row_map = torch.cat([perm, torch.full((spare,), pad, dtype=torch.int32, device="cuda")])
    cu = torch.arange(len(c.kv) + 1, dtype=torch.int32, device="cuda") * c.ql
    for how in (dict(), dict(cu_seqlens_q=cu, max_q_len=c.ql)):
        if how:
            c.run(q=q, out=out, row_map=row_map, **how)
        else:   # (without offsets every row belongs to a sequence)
            c.run(q=q[:rows], out=out[:rows], row_map=perm)
        K.check_device_errors()
        c.hold(out[perm.long()].double().cpu().numpy())
        assert (out[rows:] == 5.0).all()
        out.fill_(5.0)


@pytest.mark.parametrize("ragged", [False, True])
def test_without_room_for_the_expanded_copy_runs_convert(ragged, monkeypatch):
    c = Case(84, **EXPANDED)
    assert c.form() == "expanded"
    how = dict(cu_seqlens_q=torch.arange(4, dtype=torch.int32, device="cuda") * c.ql,
               max_q_len=c.ql) if ragged else dict()
    real, refused = torch.empty, []

    def empty(*size, **kw):
        if kw.get("dtype") == torch.uint8 and size[0] > 4 << 20:
            refused.append(size[0])
            raise torch.OutOfMemoryError("no room")
        return real(*size, **kw)

    room = c.run(**how)
    monkeypatch.setattr(torch, "empty", empty)
    got = c.run(**how)
    assert len(refused) == 1
    monkeypatch.undo()
    K.check_device_errors()
    c.hold(got.double().cpu().numpy())
    assert torch.equal(c.run(**how), room)   # with room again: as before
    if not ragged:   # a given workspace that is too small for the copy
        assert torch.equal(c.run(workspace_tensor=torch.empty(64, dtype=torch.uint8, device="cuda")), got)


MODS = [dict(softcap=4.0), dict(slopes=True), dict(window=130, prefix=[20, 300, 0]), dict(window=1),
        dict(softcap=2.0, window=33, slopes=True, prefix=[3, 64, 16])]


@pytest.mark.parametrize("kind,shape", FORMS)
@pytest.mark.parametrize("mods", MODS)
def test_modified_scores(kind, shape, mods):
    c = Case(85, **shape, **mods)
    assert c.form() == kind
    c.check()


@pytest.mark.parametrize("kind,shape", FORMS)
@pytest.mark.parametrize("window", [1, 16, 17, 127, 128, 129, 300])
def test_windows_and_prefixes_around_pages_and_tiles(kind, shape, window):
    Case(86, **shape, window=window).check()
    Case(87, **shape, window=window, prefix=[128, 1, 600]).check()


@pytest.mark.parametrize("kind,shape", FORMS)
def test_non_causal_and_contexts_shorter_than_their_rows(kind, shape):
    shape = dict(shape, kv=[0, 100, 400])
    c = Case(88, **shape)
    assert c.form() == kind
    got = c.check()
    ql = shape["ql"]
    assert not got[:ql].any() and not got[ql:2 * ql - 100].any() and got[2 * ql - 100].any()
    Case(89, **shape, causal=False).check()


@pytest.mark.parametrize("kind,hq,hkv,ql", [
    ("converting", 8, 8, 400), ("converting", 35, 5, 70), ("converting", 40, 5, 60),
    ("converting", 96, 3, 60), ("converting", 128, 4, 23), ("converting", 84, 4, 40),
    ("expanded", 4, 4, 800), ("expanded", 28, 4, 120), ("expanded", 80, 5, 56),
    ("expanded", 27, 3, 300)])
def test_every_group_size(kind, hq, hkv, ql):
    c = Case(90, hq, hkv, [ql + 5, ql + 300, ql], ql)
    assert c.form() == kind
    c.check()


@pytest.mark.parametrize("shape", [CONVERTING, EXPANDED])
@pytest.mark.parametrize("mods", [dict(), dict(softcap=3.0, window=70)])
def test_rows_without_alignment(shape, mods):
    """Odd strides of q and out, rows in another order and rows of no sequence: element by
    element, which only the converting form does."""
    c = Case(91, **shape, **mods)
    rows = len(c.kv) * c.ql
    perm = torch.from_numpy(rng(91).permutation(rows).astype(np.int32)).cuda()
    q = torch.full((rows + 9, c.hq, 131), math.nan, dtype=torch.bfloat16, device="cuda")
    q[perm.long(), :, 1:129] = c.q_dev
    out = torch.full((rows + 9, c.hq, 133), 5.0, dtype=torch.bfloat16, device="cuda")
    row_map = torch.cat([perm, torch.full((9,), -1, dtype=torch.int32, device="cuda")])
    cu = torch.arange(len(c.kv) + 1, dtype=torch.int32, device="cuda") * c.ql
    c.run(q=q[:, :, 1:129], out=out[:, :, 2:130], row_map=row_map, cu_seqlens_q=cu, max_q_len=c.ql)
    K.check_device_errors()
    c.hold(out[perm.long(), :, 2:130].double().cpu().numpy())
    assert (out[rows:] == 5.0).all() and (out[:, :, :2] == 5.0).all() and (out[:, :, 130:] == 5.0).all()


@pytest.mark.parametrize("kind,shape", FORMS)
def test_ragged_runs_beside_short_and_empty_ones(kind, shape):
    """One call's long runs take the chunk kernel, its short ones mma.sync."""
    c = Case(92, **shape)
    lens = [c.ql, 3, 0, c.ql - 50]
    kv = [c.kv[2], 90, 40, c.kv[1]]
    part = Case(92, c.hq, c.hkv, kv, c.ql)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32).cuda()
    rows = sum(lens)
    out = torch.full((rows + 2, c.hq, D), 5.0, dtype=torch.bfloat16, device="cuda")
    q = part.q_dev[:rows + 2]
    part.run(q=q, out=out, cu_seqlens_q=cu, max_q_len=c.ql)
    K.check_device_errors()
    got, at = out.double().cpu().numpy(), 0
    for s, n in enumerate(lens):
        k, v = part.rows(s)
        see = R.visible(n, kv[s])
        o, mag, size = B.attention(part.q[at:at + n], B.operand(k), B.operand(v), part.scale, see)
        if n > 8:
            tol = B.chunk_bound("bf16", o, mag, size, kv[s], D, v_top=np.abs(v).max())
            assert (np.abs(got[at:at + n] - o) <= tol).all()
        elif n:
            assert B.rms(got[at:at + n] - o) <= B.RMS["bf16"] * B.rms(o)
        at += n
    assert (out[rows:] == 5.0).all()


@pytest.mark.parametrize("kind,shape", FORMS)
def test_graphs_on_two_streams_and_new_lengths(kind, shape):
    c = Case(93, **shape)
    pool, tables, kv = c.device()
    how, graphs, outs = c.args(), [], []
    K.q4_paged_attention(c.q_dev, torch.empty_like(c.q_dev), pool, tables, kv, **how)
    for _ in range(2):
        g, out = torch.cuda.CUDAGraph(), torch.empty_like(c.q_dev)
        with torch.cuda.graph(g):
            K.q4_paged_attention(c.q_dev, out, pool, tables, kv, **how)
        graphs.append(g)
        outs.append(out)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    c.hold(outs[0].double().cpu().numpy())
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], c.run())
    kv.copy_(torch.tensor([160, 512, 0], dtype=torch.int32))   # (the poison lies behind these)
    graphs[1].replay()
    torch.cuda.synchronize()
    c.kv = [160, 512, 0]
    c.hold(outs[1].double().cpu().numpy())
    K.check_device_errors()


@pytest.mark.parametrize("kind,shape", FORMS)
def test_reports(kind, shape):
    """A block id outside the pool, a table too short for the length, a run longer than declared,
    a negative length: reported, and the other sequences' rows as they are."""
    c = Case(94, **shape)
    want = c.run()
    ql, keep = c.ql, c.tables.copy()

    def others(out):
        return torch.equal(out[:ql], want[:ql]) and torch.equal(out[2 * ql:], want[2 * ql:])

    for bad in (-5, c.pool.shape[0]):
        c.tables[1, 3] = bad
        out = c.run()
        with pytest.raises(IndexError, match="block table entry"):
            K.check_device_errors()
        assert others(out)
    c.tables = keep
    out = torch.full_like(c.q_dev, 5.0)
    K.q4_paged_attention(c.q_dev, out, c.device()[0], torch.from_numpy(keep[:, :34]).cuda(),
                         torch.tensor(c.kv, dtype=torch.int32).cuda(), **c.args())
    with pytest.raises(IndexError, match="block table"):
        K.check_device_errors()
    assert torch.equal(out[:2 * ql], want[:2 * ql])   # (640 tokens need 40 entries)
    cu = torch.tensor([0, ql, 2 * ql + 20, 3 * ql], dtype=torch.int32, device="cuda")
    out = c.run(cu_seqlens_q=cu, max_q_len=ql, out=torch.full_like(c.q_dev, 5.0))
    with pytest.raises(IndexError, match="length"):
        K.check_device_errors()
    assert torch.equal(out[:ql], want[:ql]) and (out[2 * ql:2 * ql + 20] == 5.0).all()
    c.kv[1] = -3
    out = c.run()
    with pytest.raises(IndexError, match="length"):
        K.check_device_errors()
    assert others(out) and not out[ql:2 * ql].any()


@pytest.mark.parametrize("kind,shape", FORMS)
def test_results_repeat(kind, shape):
    c = Case(95, **shape, softcap=9.0)
    first = c.run()
    assert all(torch.equal(c.run(), first) for _ in range(5))
