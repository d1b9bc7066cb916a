"""
Long runs over the 4-bit cache in 64 bits, with the roundings that the tensor-core kernels
make: keys and values are fp16 numbers there (code * scale + base rounded once), so the
reference takes the same numbers and what is left to bound is small beside the output.
"""

from __future__ import annotations

import numpy as np

from tests import q4_reference as R

EPS_HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}  # torch.finfo(t).eps / 2


def operand(x):
    """fp16 nearest to x (64 bits), past the largest one that one; NaN stays."""
    with np.errstate(over="ignore"):
        return np.clip(np.asarray(x, np.float64).astype(np.float16).astype(np.float64), -65504.0, 65504.0)


def attention(q, k, v, scale, see, softcap=0.0, slopes=None):
    """
    q (Q, Hq, D), k / v (N, H, D) in 64 bits -> out, sum_k w_k |v_k|, and the largest
    scale * sum_d |q_d k_d| of a row's keys (the size that its scores' errors scale with).
    Keys that a row does not see take no part; a row without one is zeros.
    """
    Q, Hq, D = q.shape
    N, H = k.shape[:2]
    G = Hq // H
    if N == 0:
        return np.zeros((Q, Hq, D)), np.zeros((Q, Hq, D)), np.zeros((Q, Hq, 1))
    out, mag = np.zeros((Q, Hq, D)), np.zeros((Q, Hq, D))
    size = np.zeros((Q, Hq, 1))
    back = (N - Q + np.arange(Q)[:, None]) - np.arange(N)[None]
    any_seen = see.any(1)
    for h in range(Hq):
        kk, vv = k[:, h // G], v[:, h // G]
        s = q[:, h] @ kk.T * scale
        size[:, h, 0] = np.where(see, np.abs(q[:, h]) @ np.abs(kk).T * scale, 0.0).max(1)
        if softcap:
            s = softcap * np.tanh(s / softcap)
        if slopes is not None:
            s = s - float(slopes[h]) * back
        s = np.where(see, s, -np.inf)
        w = np.exp(s - np.where(any_seen, s.max(1), 0.0)[:, None])
        w /= np.where(any_seen, w.sum(1), 1.0)[:, None]
        out[:, h], mag[:, h] = w @ vv, w @ np.abs(vv)
    return out, mag, size


def chunk_bound(dtype, out, mag, size, n_keys, d, softcap=0.0, slopes=None, v_top=0.0):
    """
    Elementwise bound of |kernel - attention() over the same fp16 operands|, for P in fp16:

    * the output's rounding, eps / 2 of |out|;
    * P's rounding, 2^-11 of each weight (the row sum adds unrounded weights), and 2^-25
      absolute where it is subnormal: weights are taken relative to a maximum that lies at most
      2^8 below the row's own and never above it, so the row sum is at least 1;
    * a score's error delta, on top and bottom of the quotient (a weight moves by at most
      2 delta each): the fp32 sum of D products, D * 2^-23 of its size; the scaling, the
      difference to the maximum and the exponential, 2^-22 of (2 + size); 2^-21 of the cap for
      its tanh; 2^-20 of the largest bias for its steps;
    * fp32 sums over the keys: of P V and of the weights, 2^-23 of sum w |v| a key each.
    """
    delta = d * 2.0 ** -23 * size + 2.0 ** -22 * (2 + size) + 2.0 ** -21 * softcap
    if slopes is not None:
        delta = delta + 2.0 ** -20 * np.asarray(slopes, np.float64)[None, :, None] * n_keys
    weight = 2.0 ** -11 + 4 * delta + 2 * n_keys * 2.0 ** -23
    return EPS_HALF[dtype] * np.abs(out) + 1.01 * weight * mag + n_keys * 2.0 ** -25 * v_top + 1e-30


def parts(code, scale, base, centred):
    """Largest sums that a value's code and parameters take in the products: the codes are
    multiplied as they are, or less 8, and the rest of the value enters apart."""
    if centred:
        return np.abs(code - 8) * scale[..., None] + np.abs(8 * scale + base)[..., None]
    return code * scale[..., None] + np.abs(base)[..., None]


def exact_code_bound(dtype, out, k_size, v_mag, n_keys, d, softcap=0.0, slopes=None):
    """
    The same for kernels that multiply the codes themselves (short runs, fp32), against the
    record's own values.  k_size and v_mag are attention()'s size and mag over parts(): sums are
    as large as those.  P is fp16 (2^-11), for fp32 two fp16 numbers as q is (2^-21 each).
    """
    p = 2.0 ** -21 if dtype == "f32" else 2.0 ** -11
    delta = d * 2.0 ** -23 * k_size + 2.0 ** -22 * (2 + k_size) + 2.0 ** -21 * softcap
    if dtype == "f32":
        delta = delta + 2.0 ** -21 * k_size
    if slopes is not None:
        delta = delta + 2.0 ** -22 * np.asarray(slopes, np.float64)[None, :, None] * n_keys
    weight = p + 4 * delta + 2 * n_keys * 2.0 ** -23
    return EPS_HALF[dtype] * np.abs(out) + 1.01 * weight * v_mag + 1e-30


# RMS error over RMS output, where single errors average out: the output's rounding (eps / 2 over
# sqrt 3 at most) and P's (2^-11 over sqrt 3, up to threefold where codes are not centred); for
# fp32 sums of D random errors of 2^-24, sqrt(D) 2^-24 of a score, a few of them.
RMS = {"bf16": 2.0 ** -8, "f16": 2.0 ** -10, "f32": 2.0 ** -14}


def rms(x):
    return float(np.sqrt(np.mean(np.square(x))))


def sized_pool(g, blocks, heads, d, k_size, v_size):
    """A packed pool (uint8) of quantised normal rows of the given sizes, held to +-65504."""
    rows = [np.clip(g.standard_normal((blocks, 16, heads, d)) * s, -65504, 65504)
            for s in (k_size, v_size)]
    pool = np.zeros((blocks, heads, R.record_bytes(d)), np.uint8)
    at = {kv: [place(t, i, d) for t in range(16) for i in range(d)]
          for kv, place in (("k", R.k_byte), ("v", R.v_byte))}
    for x, kv, par in ((rows[0], "k", 16 * d), (rows[1], "v", 16 * d + 64)):
        code, scale, base = R.quantise(x)
        code = code.astype(np.uint8).transpose(0, 2, 1, 3).reshape(blocks, heads, 16 * d)
        for i, (byte, shift) in enumerate(at[kv]):
            pool[:, :, byte] |= code[:, :, i] << shift
        both = np.stack([scale, base], -1).astype(np.float16).transpose(0, 2, 1, 3)
        pool[:, :, par:par + 64] = np.ascontiguousarray(both).reshape(blocks, heads, 32).view(np.uint8)
    return pool
