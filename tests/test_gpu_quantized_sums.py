"""The norm's mean of squares of rows of any length, with bounds that count the roundings of the kernels' own sums.

A row in registers (4096 pieces of 16 bytes at most): a thread adds up 32 squares at most, a wavefront's 64 threads 6 deep, a block's 16 wavefronts one after another: 54 roundings of
2^-24.  A longer one, or one whose elements lie apart: in 64 bits, rounded once.  Then the division by the length (1, the length itself 1), the sum with eps (1), the root (half of all that and 1)
and its reciprocal (1): 30.5 at most.  Each value of the norm has two products and its type's rounding more; a scale one product of the value (1), its product with the root (1) and a division (1)."""
import numpy as np
import pytest

import tannic_amd as ta
from quantized_support import HALF, TINY, assert_stands_for, integers_of, rounded
from tannic_amd import ops

pytestmark = pytest.mark.gpu

EPS = float(np.float32(1e-5))
ROOT = 30.5 * 2.0 ** -24


def check(dx, dr, dg, total, gain, dtype):
    """The norm of `total` (fp32, as it is kept) in the type and in 8 bits, by its definition in 64 bits."""
    wide = total.astype(np.float64)
    want = wide / np.sqrt((wide * wide).mean(-1, keepdims=True) + EPS) * gain.astype(np.float64)
    normed, sums = ops.add_rms_norm(dx, dr, dg, EPS)
    if dr is not None:
        np.testing.assert_array_equal(sums.numpy().astype(np.float32), total)
    error = np.abs(normed.numpy().astype(np.float64) - want)
    assert (error <= (HALF[dtype] * (1 + 2.0 ** -10) + ROOT + 2 * 2.0 ** -24) * np.abs(want) + TINY[dtype]).all(), float((error / np.abs(want)).max())
    values, scales, _ = ops.add_rms_norm_quantized(dx, dr, dg, EPS)
    integers, largest, _ = integers_of(total * gain)
    np.testing.assert_array_equal(values.numpy(), integers)
    factor = 1 / np.sqrt((wide * wide).mean(-1) + EPS)
    assert (np.abs(scales.numpy() * 127.0 / (largest * factor) - 1) <= ROOT + 3 * 2.0 ** -24).all()
    assert_stands_for(values.numpy(), scales.numpy(), want, ROOT + 3 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float16, ta.float32], ids=str)
@pytest.mark.parametrize("length", [1, 64, 513, 2048, 4096, 8192, 14336, 16384, 32768, 32769, 140001])
def test_rows_of_nearly_equal_values(length, dtype, device):
    """Nothing averages out: all squares are of one size, their sums' roundings fall one way."""
    rng = np.random.default_rng(51)
    x = rounded(np.stack([np.full(length, 1.0078125), np.full(length, -0.7), rng.uniform(0.99, 1.01, length)]), dtype)
    gain = rounded(rng.uniform(0.9, 1.1, length), dtype)
    check(ta.tensor(x, dtype, device), None, ta.tensor(gain, dtype, device), x, gain, dtype)
    residual = rounded(np.full(x.shape, 0.25), dtype)
    check(ta.tensor(x, dtype, device), ta.tensor(residual, dtype, device), ta.tensor(gain, dtype, device), rounded(x + residual, dtype), gain, dtype)
    apart = ta.tensor(np.repeat(x, 2, -1), dtype, device)[:, ::2]
    check(apart, None, ta.tensor(gain, dtype, device), x, gain, dtype)


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float32], ids=str)
def test_a_row_of_millions(dtype, device):
    """65536 squares of a thread one after another."""
    length = (1 << 24) + 5
    x = rounded(np.stack([np.full(length, 1.0078125), np.full(length, 0.7)]), dtype)
    gain = rounded(np.resize([0.75, 1.0, 1.5], length), dtype)
    check(ta.tensor(x, dtype, device), None, ta.tensor(gain, dtype, device), x, gain, dtype)


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float32], ids=str)
@pytest.mark.parametrize("length", [64, 4096, 16384, 40000])
def test_squares_beyond_the_floats(length, dtype, device):
    """A mean of squares that is no float: the norm is 0, as ``rms_norm``'s is, in either form; below that bound it is what it should be."""
    rng = np.random.default_rng(52)
    x = rounded(rng.uniform(1, 2, (2, length)) * [[3e19], [2.0 ** 60 / length ** 0.5]], dtype)
    gain = rounded(np.ones(length), dtype)
    dx, dg = ta.tensor(x, dtype, device), ta.tensor(gain, dtype, device)
    normed, _ = ops.add_rms_norm(dx, None, dg, EPS)
    values, scales, _ = ops.add_rms_norm_quantized(dx, None, dg, EPS)
    assert not normed.numpy()[0].any() and scales.numpy()[0] == 0
    assert not ops.rms_norm(dx, dg, EPS).numpy()[0].any()
    wide = x[1].astype(np.float64)
    want = wide / np.sqrt((wide * wide).mean() + EPS)
    assert (np.abs(normed.numpy()[1].astype(np.float64) - want) <= (HALF[dtype] * (1 + 2.0 ** -10) + ROOT + 2 * 2.0 ** -24) * np.abs(want)).all()
    assert_stands_for(values.numpy()[1:], scales.numpy()[1:], want[None], ROOT + 3 * 2.0 ** -24)
