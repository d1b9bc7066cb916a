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


CONVERTING = dict(hq=16, hkv=4, kv=[200, 527, 640], ql=150)   # 60 row tiles of 16 a head, 5 of 128
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
