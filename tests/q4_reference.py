"""
The 4-bit cache and modified-score attention in 64 bits, from their definitions
(numpy, no code of the package): the checker of the q4 and scored kernels.
"""

from __future__ import annotations

import math

import numpy as np

BLOCK = 16
HALVES = np.arange(0, 31744, dtype=np.uint16).view(np.float16).astype(np.float64)
HALVES = np.concatenate([-HALVES[:0:-1], HALVES])


def quantise(x):
    """codes, scale, base of the rows of x (fp64): see include/memforge_sm100.h."""
    x = np.asarray(x, np.float64)
    bad = ~(np.abs(x) <= 65504).all(-1)
    y = np.where(bad[..., None], 0.0, x)
    base = HALVES[np.searchsorted(HALVES, y.min(-1), side="right") - 1]
    scale = HALVES[np.searchsorted(HALVES * 15, y.max(-1) - base, side="left")]
    with np.errstate(all="ignore"):
        code = np.where(scale[..., None] > 0, np.rint((y - base[..., None]) / scale[..., None]), 0)
    return code, np.where(bad, np.nan, scale), np.where(bad, np.nan, base)


def dequantised(x):
    code, scale, base = quantise(x)
    return code * scale[..., None] + base[..., None]


def record_bytes(d):
    return 16 * d + 128


def v_byte(t, dim, d):
    """Byte and shift of V code (token t, dim) inside a record."""
    w_ = min(4, d // 32)
    c, i = divmod(dim, 128)
    g, w, n = i // (4 * w_), (i // 4) % w_, dim % 4
    at = 8 * d + ((((c * 2 + t // 8) * 8 + g) * 4 + (t // 2) % 4) * w_ + w) * 4 + (t % 2) * 2
    return at + n // 2, 4 * (n % 2)


def k_byte(t, dim, d):
    return t * (d // 2) + dim // 2, 4 * (dim % 2)


def write_token(pool, d, blk, t, head, krow, vrow):
    """Pack one token's quantised K and V rows into a uint8 pool (blocks, H, record)."""
    rec = pool[blk, head]
    for row, place, par in ((krow, k_byte, 16 * d), (vrow, v_byte, 16 * d + 64)):
        code, scale, base = quantise(row)
        for dim in range(d):
            at, sh = place(t, dim, d)
            rec[at] = (int(rec[at]) & ~(15 << sh)) | (int(code[dim]) << sh)
        rec[par + 4 * t:par + 4 * t + 4] = np.array([scale, base], np.float16).view(np.uint8)


def read_rows(pool, d, slots):
    """(K, V) rows (T, H, D) in fp64 of a uint8 pool at flat slots."""
    slots = np.asarray(slots)
    blk, tok = slots // BLOCK, slots % BLOCK
    out = []
    for place, par in ((k_byte, 16 * d), (v_byte, 16 * d + 64)):
        at = np.array([[place(t, i, d) for i in range(d)] for t in range(BLOCK)])
        byte = pool[blk[:, None], :, at[tok, :, 0]]             # (T, D, H)
        code = (byte >> at[tok, :, 1][..., None]) & 15
        pars = np.ascontiguousarray(pool[:, :, par:par + 64]).view(np.float16)
        pars = pars.reshape(pool.shape[0], pool.shape[1], BLOCK, 2)[blk, :, tok].astype(np.float64)
        out.append(np.transpose(code, (0, 2, 1)) * pars[..., :1] + pars[..., 1:])
    return out


def visible(q_len, kv_len, causal=True, window=0, prefix=0):
    """(q_len, kv_len) truth values."""
    p = kv_len - q_len + np.arange(q_len)[:, None]
    k = np.arange(kv_len)[None]
    see = np.ones((q_len, kv_len), bool)
    if causal:
        see &= k <= p
    if window:
        see &= p - k < window
    return see | (k < prefix)


def attention(q, k, v, scale, see, softcap=0.0, slopes=None, kv_len=None):
    """
    q (Q, Hq, D), k / v (N, H, D) in fp64 -> out, and sum_k w_k |v_k| (the size its
    rounding errors scale with).  Values a row does not see take no part (NaN included).
    """
    Q, Hq, D = q.shape
    H = k.shape[1]
    G = Hq // H
    out = np.zeros((Q, Hq, D))
    mag = np.zeros((Q, Hq, D))
    for h in range(Hq):
        for i in range(Q):
            idx = np.nonzero(see[i])[0]
            if idx.size == 0:
                continue
            kk, vv = k[idx, h // G], v[idx, h // G]
            s = kk @ q[i, h] * scale
            if softcap:
                s = softcap * np.tanh(s / softcap)
            if slopes is not None:
                s = s - slopes[h] * (k.shape[0] - Q + i - idx)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ vv
            mag[i, h] = w @ np.abs(vv)
    return out, mag


HALF_ULP = {"bf16": 2.0 ** -9, "f16": 2.0 ** -12, "f32": 2.0 ** -25}


def q4_tolerance(dtype, out, q, codes_size, key_size, scale, chunk=False):
    """
    Bound of |kernel - exact| for attention over 4-bit rows, elementwise.

    * the output's rounding: half a unit, |out| * eps / 2 (eps / 2 taken from
      torch.finfo; HALF_ULP * 2 bounds it for any mantissa);
    * P rounded to fp16 (2^-12 relative, twice for fp32: 2^-23): times codes_size = the
      largest 15 * scale + |base| of a V row, which bounds every |n * scale|, |base|;
    * a score's error delta moves a weight by exp(delta) - 1, at most 2 delta, on top and
      bottom of the quotient (4 delta in all): fp32 sums of D products and of their
      pieces, D * 2^-24 of scale * sum|q| * key_size, and 2^-21 for the exponential;
    * chunk: long runs read keys and values rounded to fp16 (2^-12 relative each): the
      values add 2^-12 of their size, the keys 2^-12 of scale * sum|q| * key_size to delta.
    """
    p = 2.0 ** -23 if dtype == "f32" else 2.0 ** -12
    D = q.shape[-1]
    size = scale * np.abs(q).sum(-1, keepdims=True) * key_size
    delta = D * 2.0 ** -24 * size + 2.0 ** -21
    if chunk:
        p += 2.0 ** -12
        delta = delta + 2.0 ** -12 * size
    return 2 * HALF_ULP[dtype] * np.abs(out) + (p + 4 * delta) * codes_size + 1e-30
