"""Rows in 8-bit integers with a scale each: of any values, of a gated activation, of a norm with the residual's addition; and back.  The integers have to be those of the
same steps in fp32, which are single roundings, and what they stand for the definition in 64 bits."""
import numpy as np
import pytest

import tannic_amd as ta
from quantized_support import HALF, LEAST, TINY, assert_stands_for, integers_of, rounded
from tannic_amd import ops

pytestmark = pytest.mark.gpu

TYPES = [ta.bfloat16, ta.float16, ta.float32]
# rows and their length: single elements, pieces of 16 bytes and one element more or less, what a wavefront, a block and its registers hold and one more, many rows
SHAPES = [(1, 1), (3, 7), (1, 8), (5, 64), (2, 255), (3, 512), (4, 513), (1, 2048), (3, 4096), (2, 4097), (1, 14336), (2, 16384), (3, 16392), (1, 40000), (2, 66000), (1, 140001),
          (1030, 64), (2000, 33), (4097, 16), (1500, 1024), (300, 5120), (70000, 8)]


def spread(rng, shape, dtype):
    """Values over some powers of two, a few of them large."""
    return rounded(rng.standard_normal(shape) * np.exp2(rng.integers(-6, 3, shape)), dtype)


def check_integers(values, scales, u, one=None):
    want, largest, finite = integers_of(u)
    assert finite.all()
    np.testing.assert_array_equal(values, want)
    if one is None:
        np.testing.assert_array_equal(scales, largest / np.float32(127))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_quantize_and_back(shape, dtype, device):
    x = spread(np.random.default_rng(1), shape, dtype)
    values, scales = ops.quantize(ta.tensor(x, dtype, device))
    assert values.dtype is ta.int8 and scales.dtype is ta.float32 and values.shape == shape and scales.shape == shape[:-1]
    v, s = values.numpy(), scales.numpy()
    check_integers(v, s, x)
    assert_stands_for(v, s, x.astype(np.float64), 0.0)
    for to in TYPES:
        np.testing.assert_array_equal(ops.dequantize(values, scales, to).numpy(), rounded(v.astype(np.float32) * s[..., None], to))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_swiglu(shape, dtype, device):
    """u is off by 8 * 2^-24 at most: 3 of the exponential (its instruction 2, the correction 1), 1 of its sum with 1, 2 of the reciprocal, 1 of each product.  The scale is off by these
    and 1 of its division, within the 6 + 4 asked for here; an element by 8 of u, 3 of the factor and its product and 9 of the scale, within 12 + 8."""
    rng = np.random.default_rng(2)
    rows, length = shape
    both = rounded(rng.standard_normal((rows, 2 * length)) * 3, dtype)
    on_device = ta.tensor(both, dtype, device)
    gate, up = both[:, :length].astype(np.float64), both[:, length:].astype(np.float64)
    want = gate / (1 + np.exp(-gate)) * up
    values, scales = ops.swiglu_quantized(on_device[:, 0:length], on_device[:, length:2 * length])
    assert_stands_for(values.numpy(), scales.numpy(), want, 6 * 2.0 ** -24)


def check_norm(x, residual, gain, eps, dtype, device, make=lambda x, dtype, device: ta.tensor(x, dtype, device)):
    rows = x.reshape(-1, x.shape[-1]).shape[0]
    length = x.shape[-1]
    dx, dr, dg = make(x, dtype, device), None if residual is None else make(residual, dtype, device), ta.tensor(gain, dtype, device)
    with np.errstate(over="ignore"):
        total = x if residual is None else rounded(x + residual, dtype)
    size = total.astype(np.float64)
    want = size / np.sqrt((size * size).mean(-1, keepdims=True) + eps) * gain.astype(np.float64)
    # the mean of squares: a thread adds up some of them one after another (256 threads at least, or 64 of them where a row is at most 64 pieces), then a tree; its root takes half of that
    slack = (length / 64 / 2 + 12) * 2.0 ** -24
    normed, sums = ops.add_rms_norm(dx, dr, dg, eps)
    if residual is None:
        assert sums is dx
    else:
        np.testing.assert_array_equal(sums.numpy().astype(np.float32), total)
    assert (np.abs(normed.numpy().astype(np.float64) - want) <= (HALF[dtype] + slack + 2.0 ** -22) * np.abs(want) + TINY[dtype]).all(), (rows, length)
    values, scales, sums = ops.add_rms_norm_quantized(dx, dr, dg, eps)
    if residual is not None:
        np.testing.assert_array_equal(sums.numpy().astype(np.float32), total)
    check_integers(values.numpy(), scales.numpy(), total * gain, one=True)
    assert_stands_for(values.numpy(), scales.numpy(), want, slack + 2.0 ** -22)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("with_residual", [True, False])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_add_rms_norm(shape, with_residual, dtype, device):
    rng = np.random.default_rng(3)
    x, gain = spread(rng, shape, dtype), rounded(1 + 0.2 * rng.standard_normal(shape[-1]), dtype)
    residual = spread(rng, shape, dtype) if with_residual else None
    check_norm(x, residual, gain, float(np.float32(1e-5)), dtype, device)


def test_add_rms_norm_of_float64(device):
    rng = np.random.default_rng(4)
    x, residual, gain = rng.standard_normal((5, 333)), rng.standard_normal((5, 333)), rng.standard_normal(333)
    normed, total = ops.add_rms_norm(*(ta.tensor(t, ta.float64, device) for t in (x, residual, gain)), 1e-5)
    np.testing.assert_array_equal(total.numpy(), x + residual)
    want = (x + residual) / np.sqrt(((x + residual) ** 2).mean(-1, keepdims=True) + float(np.float32(1e-5))) * gain
    assert (np.abs(normed.numpy() - want) <= 350 * 2.0 ** -53 * np.abs(want)).all()


# how a tensor of a shape lies: a view of a larger one that starts anywhere, rows of another length, dims in another order, elements apart, one row for all
LAYOUTS = {
    "columns": ((3, 5, 72), lambda t: t[:, :, 8:48]),
    "odd_columns": ((3, 5, 73), lambda t: t[:, :, 3:44]),
    "dims_turned": ((5, 3, 40), lambda t: t.transpose(0, 1)),
    "apart": ((3, 5, 82), lambda t: t[:, :, 1:82:2]),
    "last_dim_first": ((41, 3, 5), lambda t: t.permute(1, 2, 0)),
    "rows_apart": ((6, 10, 40), lambda t: t[::2, 1::2]),
    "one_row": ((1, 1, 40), lambda t: t.expand(3, 5, 40)),
    "five_dims": ((2, 3, 2, 3, 16), lambda t: t.permute(2, 1, 3, 0, 4)),
    "long_odd": ((2, 3, 9000), lambda t: t[:, 1:3, 1:8192]),
}


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_operands_in_other_orders(layout, dtype, device):
    rng = np.random.default_rng(5)
    shape, view = LAYOUTS[layout]

    def operand():
        whole = ta.tensor(spread(rng, shape, dtype), dtype, device)
        return view(whole)

    x, y = operand(), operand()
    n = x.numpy().astype(np.float32)
    values, scales = ops.quantize(x)
    assert values.shape == x.shape and scales.shape == x.shape[:-1]
    check_integers(values.numpy(), scales.numpy(), n)
    gate, up = n.astype(np.float64), y.numpy().astype(np.float64)
    v, s = ops.swiglu_quantized(x, y)
    assert_stands_for(v.numpy(), s.numpy(), gate / (1 + np.exp(-gate)) * up, 6 * 2.0 ** -24)
    gain = rounded(1 + 0.2 * rng.standard_normal(x.shape[-1]), dtype)
    operands = iter((x, y))
    check_norm(n, y.numpy().astype(np.float32), gain, float(np.float32(1e-5)), dtype, device, make=lambda *_: next(operands))
    # the integers themselves, seen through the same view
    whole = ta.tensor(rng.integers(-127, 128, shape), ta.int8, device)
    seen = view(whole)
    each = ta.tensor(rng.uniform(0.01, 1, seen.shape[:-1]), ta.float32, device)
    np.testing.assert_array_equal(ops.dequantize(seen, each, dtype).numpy(), rounded(seen.numpy().astype(np.float32) * each.numpy()[..., None], dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("length", [40, 41, 4096, 5001])
def test_rows_of_zeros_and_of_what_is_not_finite(length, dtype, device):
    rng = np.random.default_rng(6)
    x = spread(rng, (6, length), dtype)
    x[1] = 0.0
    x[2, length // 2] = np.inf
    x[3, length - 1] = np.nan
    x[4, 0] = -np.inf
    ones = np.ones(length)
    gain = ta.tensor(ones, dtype, device)
    least = float(LEAST) / 127
    d = ta.tensor(x, dtype, device)
    zero = ta.tensor(np.zeros((6, length)), dtype, device)
    some = ta.tensor(np.ones((6, length)), dtype, device)
    for values, scales in (ops.quantize(d), ops.add_rms_norm_quantized(d, zero, gain)[:2], ops.add_rms_norm_quantized(d, None, gain)[:2], ops.swiglu_quantized(some, d)):
        v, s = values.numpy(), scales.numpy()
        assert np.isnan(s[[2, 3, 4]]).all() and not v[[1, 2, 3, 4]].any()
        assert np.isfinite(s[[0, 1, 5]]).all() and (np.abs(v[[0, 5]]).max(-1) == 127).all()
        back = ops.dequantize(values, scales, dtype).numpy()
        assert np.isnan(back[[2, 3, 4]]).all() and not back[1].any()
    assert ops.quantize(d)[1].numpy()[1] == np.float32(least)
    normed = ops.add_rms_norm(d, zero, gain)[0].numpy()
    np.testing.assert_array_equal(np.isnan(normed), np.isnan(ops.rms_norm(d, gain).numpy()))


def test_the_smallest_and_the_largest_rows(device):
    """fp32 rows around the least largest value, of subnormal numbers, and up to the largest number."""
    x = np.zeros((6, 16), np.float32)
    x[0, 3], x[0, 4] = 2.0 ** -119, -2.0 ** -120
    x[1, 3], x[1, 4] = 2.0 ** -118, 2.0 ** -125
    x[2, 3] = 2.0 ** -130
    x[3, 3], x[3, 5] = 2.0 ** -149, -2.0 ** -149
    x[4, 3], x[4, 7] = np.finfo(np.float32).max, -1e38
    x[5] = 1.0
    values, scales = ops.quantize(ta.tensor(x, ta.float32, device))
    check_integers(values.numpy(), scales.numpy(), x)
    assert_stands_for(values.numpy(), scales.numpy(), x.astype(np.float64), 0.0)


def test_ties_go_to_even(device):
    x = np.zeros((1, 64), np.float32)
    x[0, 0] = 127.0
    x[0, 1:33] = np.arange(32) - 15.5
    values, scales = ops.quantize(ta.tensor(x, ta.float32, device))
    assert scales.numpy()[0] == 1.0
    np.testing.assert_array_equal(values.numpy()[0, 1:33], np.rint(np.arange(32) - 15.5))


@pytest.mark.parametrize("shape", [(0, 8), (3, 0, 8), (2, 0), (0, 0)], ids=str)
def test_nothing_there(shape, device):
    x = ta.Tensor(ta.float32, shape).initialize(device)
    gain = ta.Tensor(ta.float32, shape[-1:]).initialize(device)
    values, scales = ops.quantize(x)
    assert values.shape == shape and scales.shape == shape[:-1]
    # (rows of no elements have the scale of rows of zeros)
    assert (scales.numpy() == LEAST / np.float32(127)).all()
    assert ops.swiglu_quantized(x, x)[0].shape == shape
    assert ops.add_rms_norm(x, x, gain)[0].shape == shape and ops.add_rms_norm_quantized(x, None, gain)[0].shape == shape
    assert ops.dequantize(values, scales, ta.float16).shape == shape


def test_a_single_row_of_rank_one(device):
    x = spread(np.random.default_rng(7), (100,), ta.float32)
    values, scales = ops.quantize(ta.tensor(x, ta.float32, device))
    assert scales.shape == ()
    check_integers(values.numpy(), scales.numpy(), x)
    np.testing.assert_array_equal(ops.dequantize(values, scales, ta.float32).numpy(), values.numpy().astype(np.float32) * scales.numpy())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("length", [256, 257, 30000])
@pytest.mark.parametrize("onto", ["x", "residual"])
def test_the_sum_may_be_an_operand(onto, length, dtype, device):
    """Through the C ABI: the sum is written over x or over the residual."""
    import ctypes as C
    rng = np.random.default_rng(8)
    x, residual = spread(rng, (9, length), dtype), spread(rng, (9, length), dtype)
    gain = ta.tensor(rounded(1 + 0.1 * rng.standard_normal(length), dtype), dtype, device)
    want = [t.numpy() for t in ops.add_rms_norm_quantized(ta.tensor(x, dtype, device), ta.tensor(residual, dtype, device), gain)]
    dx, dr = ta.tensor(x, dtype, device), ta.tensor(residual, dtype, device)
    total = dx if onto == "x" else dr
    values, scales = ta.Tensor(ta.int8, (9, length)).initialize(device), ta.Tensor(ta.float32, (9,)).initialize(device)
    status = ta.library().kernels["add_rms_norm"](*(C.byref(t.descriptor()) for t in (dx, dr, gain, total, values, scales)), device.stream(), 1e-5)
    assert status == 0
    for t, w in zip((values, scales, total), want):
        np.testing.assert_array_equal(t.numpy(), w)
