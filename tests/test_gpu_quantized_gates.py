"""``swiglu_quantized`` where the gates alone make a row small: gates so far below zero that exp(-gate), its reciprocal or the quotient is beyond the normal floats while ``up`` is as large
as the type has it, and gates that are not finite."""
import numpy as np
import pytest

import tannic_amd as ta
from quantized_support import assert_stands_for, rounded
from tannic_amd import ops

pytestmark = pytest.mark.gpu

# a wavefront of a row, an element more than a piece, blocks of a row, rows beyond the registers
LENGTHS = [40, 41, 2048, 5000, 14336, 40000, 70001]


def exactly(gate, up):
    gate, up = gate.astype(np.float64), up.astype(np.float64)
    return gate / (1 + np.exp(np.minimum(-gate, 700))) * up


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float32], ids=str)
@pytest.mark.parametrize("length", LENGTHS)
def test_rows_of_gates_far_below_zero_only(length, dtype, device):
    """u is off by 8 * 2^-24 at most as everywhere (5 below -64), or by 2^-150, which is 2^-31 of the least largest value: the bounds of every gated row."""
    rng = np.random.default_rng(41)
    ranges = [(-95, -85), (-87.4, -87.3), (-130, -88), (-176, -100), (-66, -62), (-174, -160), (-300, -90), (-88.8, -88.6)]
    gate = rounded(np.stack([rng.uniform(low, high, length) for low, high in ranges] + [np.full(length, -90.0), np.full(length, -87.5)]), dtype)
    up = rounded(rng.uniform(1e38, 3e38, gate.shape) * rng.choice([-1, 1], gate.shape), dtype)
    values, scales = ops.swiglu_quantized(ta.tensor(gate, dtype, device), ta.tensor(up, dtype, device))
    v = values.numpy()
    assert (np.abs(v).max(-1) == 127).all()
    assert_stands_for(v, scales.numpy(), exactly(gate, up), 6 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float16, ta.float32], ids=str)
@pytest.mark.parametrize("length", LENGTHS)
def test_far_gates_among_others(length, dtype, device):
    """One gate of a row is far below zero and its up the largest of the type: what stands beside it is as without it."""
    rng = np.random.default_rng(42)
    gate, up = (rounded(rng.standard_normal((4, length)) * 3, dtype) for _ in range(2))
    largest = 6e4 if dtype is ta.float16 else 3e38
    for row, far in enumerate((-89.0, -200.0, -3e4, -largest)):
        gate[row, length // 3], up[row, length // 3] = rounded([far, largest], dtype)
    values, scales = ops.swiglu_quantized(ta.tensor(gate, dtype, device), ta.tensor(up, dtype, device))
    assert_stands_for(values.numpy(), scales.numpy(), exactly(gate, up), 6 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float16, ta.float32], ids=str)
@pytest.mark.parametrize("length", LENGTHS)
def test_gates_that_are_not_finite(length, dtype, device):
    rng = np.random.default_rng(43)
    gate, up = (rounded(rng.standard_normal((6, length)), dtype) for _ in range(2))
    gate[0, length - 1], gate[1, 0], gate[2, length // 2], gate[4, 3] = np.inf, -np.inf, np.nan, -np.nan
    up[1, 0] = 0.0
    gate[5, 7], up[5, 7] = -100.0, np.inf
    values, scales = ops.swiglu_quantized(ta.tensor(gate, dtype, device), ta.tensor(up, dtype, device))
    s = scales.numpy()
    assert np.isnan(s[[0, 1, 2, 4, 5]]).all() and np.isfinite(s[3]) and not values.numpy()[[0, 1, 2, 4, 5]].any()
