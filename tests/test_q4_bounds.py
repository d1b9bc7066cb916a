"""The bounds of tests/q4_bounds.py reject what is wrong and hold what is right (no GPU)."""

import math

import numpy as np
import pytest

from tests import q4_bounds as B
from tests import q4_reference as R

D, SEED = 128, 3


def case(size, n=300, rows=40):
    g = np.random.default_rng(SEED)
    pool = B.sized_pool(g, (n + 15) // 16, 2, D, size, size)
    k, v = R.read_rows(pool, D, np.arange(n))
    q = g.standard_normal((rows, 4, D)) / size
    return q, k, v, 1 / math.sqrt(D), R.visible(rows, n)


def bound_of(q, k, v, scale, see):
    out, mag, size = B.attention(q, B.operand(k), B.operand(v), scale, see)
    return out, B.chunk_bound("bf16", out, mag, size, k.shape[0], D, v_top=np.abs(v).max())


def beyond(got, want, tol):
    return float((np.abs(got - want) > tol).mean())


@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4, 1e-5, 1e-6])
def test_the_chunk_bound_is_a_few_percent_and_rejects_wrong_outputs(size):
    q, k, v, scale, see = case(size)
    want, tol = bound_of(q, k, v, scale, see)
    assert np.median(tol) < 0.05 * B.rms(want)
    assert beyond(np.zeros_like(want), want, tol) > 0.8
    one_less = R.visible(*see.shape, window=see.shape[1] - 1)   # the last row loses a key
    got, _, _ = B.attention(q, k, v, scale, see & one_less)
    assert beyond(got[-1], want[-1], tol[-1]) > 0.1
    # values of rows one page off
    got, _, _ = B.attention(q, k, np.roll(v, 16, 0), scale, see)
    assert beyond(got, want, tol) > 0.5


@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-6])
def test_rounded_operands_agree_with_the_definition(size):
    """Any code * scale + base is a multiple of 2^-24, so its rounding to fp16 is off by at most
    2^-11 of it, small rows included; the attention over them then stays within the output's
    rounding of a bf16 (in the mean, where the single errors average out)."""
    q, k, v, scale, see = case(size)
    for x in (k, v):
        assert (np.abs(B.operand(x) - x) <= 2.0 ** -11 * np.abs(x)).all()
    exact, _, _ = B.attention(q, k, v, scale, see)
    near, _, _ = B.attention(q, B.operand(k), B.operand(v), scale, see)
    assert B.rms(near - exact) < 0.2 * B.RMS["bf16"] * B.rms(exact)


def test_halved_subnormals_are_rejected():
    """Scale and base halved in fp16 lose their last bit: rows of size 1e-6 are off by more than
    their size, rows of 1e-5 by percents."""
    def halved(code, scale, base):
        s, b = (np.float16(x * 0.5).astype(np.float64)[..., None] for x in (scale, base))
        return 2 * np.float16(code * s + b).astype(np.float64)

    g = np.random.default_rng(SEED)
    for size, wrong in ((1e-5, 0.02), (1e-6, 0.3)):
        x = g.standard_normal((300, 2, D)) * size
        code, scale, base = R.quantise(x)
        v = code * scale[..., None] + base[..., None]
        q, k, _, sc, see = case(1.0)
        want, tol = bound_of(q, k, v, sc, see)
        got, _, _ = B.attention(q, B.operand(k), halved(code, scale, base), sc, see)
        assert beyond(got, want, tol) > wrong


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_the_bounds_of_short_runs_tell_the_types_apart(dtype):
    import torch
    g = np.random.default_rng(SEED)
    x = [g.standard_normal((300, 2, D)) for _ in range(2)]
    q, scale, see = g.standard_normal((3, 4, D)), 1 / math.sqrt(D), R.visible(3, 300)
    (k, kp), (v, vp) = ((R.dequantised(t), B.parts(*R.quantise(t), centred=dtype != "bf16")) for t in x)
    want, _, _ = B.attention(q, k, v, scale, see)
    _, _, size = B.attention(q, kp, v, scale, see)
    _, mag, _ = B.attention(q, k, vp, scale, see)
    tol = B.exact_code_bound(dtype, want, size, mag, 300, D)
    assert np.median(tol) < (0.35 if dtype == "bf16" else 0.07) * B.rms(want)
    assert beyond(np.zeros_like(want), want, tol) > 0.7
    coarse = {"bf16": torch.float8_e4m3fn, "f16": torch.bfloat16, "f32": torch.float16}[dtype]
    rounded = torch.from_numpy(want).to(coarse).double().numpy()
    assert B.rms(rounded - want) > B.RMS[dtype] * B.rms(want)


def test_the_pool_of_the_bounds_holds_its_rows():
    g = np.random.default_rng(1)
    pool = B.sized_pool(g, 2, 3, 64, 1.0, 1e-5)
    g = np.random.default_rng(1)
    rows = [g.standard_normal((2, 16, 3, 64)) * s for s in (1.0, 1e-5)]
    k, v = R.read_rows(pool, 64, np.arange(32))
    assert np.array_equal(k, R.dequantised(rows[0]).reshape(32, 3, 64))
    assert np.array_equal(v, R.dequantised(rows[1]).reshape(32, 3, 64))
