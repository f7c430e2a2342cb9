"""Products of 8-bit integers with a scale for each row and column: the sums are exact and everything after them is a single rounding, so results have to be those of the
same steps in fp32, bit for bit, whatever kernel forms them; and within their roundings of the definition in 64 bits."""
import numpy as np
import pytest

import tannic_amd as ta
from quantized_support import HALF, TINY, product, rounded
from tannic_amd import ops

pytestmark = pytest.mark.gpu

TYPES = [ta.bfloat16, ta.float16, ta.float32]
# M, N, K: single tokens, what a wavefront's rows hold and one more, tiles and one more or less, K of one window and of many, no whole pieces, the pieces of few tiles under a long K
SIZES = [(1, 1, 1), (1, 16, 64), (1, 17, 33), (2, 5, 1000), (1, 1000, 128), (1, 4096, 4096), (3, 129, 256), (16, 512, 384), (17, 500, 640), (32, 4096, 1024), (31, 33, 14336), (33, 96, 2048),
         (48, 1000, 512), (64, 640, 4096), (65, 130, 128), (100, 2049, 1030), (127, 255, 272), (128, 128, 128), (129, 257, 144), (200, 4096, 512), (256, 256, 2048), (257, 300, 4096),
         (300, 1536, 1024), (512, 6144, 256), (700, 1000, 999), (1025, 1280, 640), (77, 2049, 1030), (5, 3, 131071)]


def operands(rng, m, n, k, batch_a=(), batch_b=()):
    a, b = rng.integers(-127, 128, batch_a + (m, k)), rng.integers(-127, 128, batch_b + (k, n))
    # (a scale of about 1 / (127 sqrt K): results of some units in every type)
    each = 1.0 / (70.0 * max(k, 1) ** 0.5)
    return a, rng.uniform(0.5, 1.5, batch_a + (m,)).astype(np.float32) * np.float32(each), b, rng.uniform(0.005, 0.02, batch_b + (n,)).astype(np.float32)


def check(got, a, a_scales, b, b_scales, dtype):
    in_fp32 = product(a, a_scales, b, b_scales)
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(got, rounded(in_fp32, dtype))
    want = (a.astype(np.float64) @ b.astype(np.float64)) * a_scales.astype(np.float64)[..., :, None] * b_scales.astype(np.float64)[..., None, :]
    assert (np.abs(got.astype(np.float64) - want) <= (HALF[dtype] + 4 * 2.0 ** -24) * np.abs(want) + TINY[dtype]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_weights_as_they_are_kept(size, dtype, device):
    m, n, k = size
    a, sa, b, sb = operands(np.random.default_rng(11), m, n, k)
    w = ta.tensor(np.ascontiguousarray(b.T), ta.int8, device).transpose()
    got = ops.matmul_quantized(ta.tensor(a, ta.int8, device), ta.tensor(sa, ta.float32, device), w, ta.tensor(sb, ta.float32, device), dtype)
    assert got.dtype is dtype and got.shape == (m, n)
    check(got.numpy(), a, sa, b, sb, dtype)


# how an operand lies: (what it is cut out of, its view) from rows and K
def slack(shape, rows, columns):
    return tuple(shape[:-2]) + (shape[-2] + rows, shape[-1] + columns)


LAYOUTS = {
    "whole": (lambda s: s, lambda t, s: t),
    "other_order": (lambda s: s[:-2] + (s[-1], s[-2]), lambda t, s: t.transpose()),
    "columns_of_more": (lambda s: slack(s, 0, 32), lambda t, s: t[..., 16:16 + s[-1]]),
    "odd_columns_of_more": (lambda s: slack(s, 1, 7), lambda t, s: t[..., 1:, 3:3 + s[-1]]),
    "other_order_of_more": (lambda s: s[:-2] + (s[-1] + 3, s[-2] + 5), lambda t, s: t[..., 2:2 + s[-1], 1:1 + s[-2]].transpose()),
    "every_other": (lambda s: s[:-2] + (2 * s[-2], 2 * s[-1]), lambda t, s: t[..., ::2, 1::2]),
}


@pytest.mark.parametrize("of_b", LAYOUTS)
@pytest.mark.parametrize("of_a", LAYOUTS)
@pytest.mark.parametrize("size", [(1, 300, 256), (20, 200, 384), (150, 260, 512), (40, 70, 90)], ids=str)
def test_operands_in_other_orders(size, of_a, of_b, device):
    m, n, k = size
    rng = np.random.default_rng(12)
    seen = []
    for shape, layout in (((m, k), LAYOUTS[of_a]), ((k, n), LAYOUTS[of_b])):
        whole = ta.tensor(rng.integers(-127, 128, layout[0](shape)), ta.int8, device)
        seen.append(layout[1](whole, shape))
        assert seen[-1].shape == shape
    sa, sb = rng.uniform(0.001, 0.002, 2 * m + 1).astype(np.float32), rng.uniform(0.005, 0.02, 3 * n).astype(np.float32)
    dsa, dsb = ta.tensor(sa, ta.float32, device)[1::2], ta.tensor(sb, ta.float32, device)[::3]
    got = ops.matmul_quantized(seen[0], dsa, seen[1], dsb, ta.bfloat16)
    check(got.numpy(), seen[0].numpy().astype(np.int64), sa[1::2], seen[1].numpy().astype(np.int64), sb[::3], ta.bfloat16)


# batch dims of a and b, M, N, K: tokens of several sequences over one matrix, a matrix each, one set of tokens over several matrices, both broadcast
BATCHES = [((3,), (), 40, 200, 256), ((3,), (), 1, 200, 256), ((2, 3), (), 64, 100, 128), ((4,), (4,), 17, 130, 384), ((), (3,), 20, 64, 256), ((2, 1), (3,), 33, 70, 130),
           ((5,), (5,), 150, 140, 128), ((1,), (), 70, 300, 512), ((2, 3), (2, 3), 1, 48, 64), ((3,), (1,), 300, 200, 256), ((0,), (), 4, 5, 6), ((3, 1), (1, 4), 129, 65, 256)]


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float32], ids=str)
@pytest.mark.parametrize("case", BATCHES, ids=str)
def test_batches(case, dtype, device):
    batch_a, batch_b, m, n, k = case
    a, sa, b, sb = operands(np.random.default_rng(13), m, n, k, batch_a, batch_b)
    w = ta.tensor(np.ascontiguousarray(np.swapaxes(b, -1, -2)), ta.int8, device).transpose()
    got = ops.matmul_quantized(ta.tensor(a, ta.int8, device), ta.tensor(sa, ta.float32, device), w, ta.tensor(sb, ta.float32, device), dtype)
    assert got.shape == np.broadcast_shapes(batch_a, batch_b) + (m, n)
    check(got.numpy(), a, sa, b, sb, dtype)


@pytest.mark.parametrize("rows", [9, 150])
def test_sequences_cut_out_of_longer_ones(rows, device):
    """A batch whose sequences do not lie one behind the other, and one whose rows lie turned round."""
    rng = np.random.default_rng(14)
    a, sa, b, sb = operands(rng, rows + 3, 192, 256, (4,))
    w = ta.tensor(np.ascontiguousarray(b.T), ta.int8, device).transpose()
    da, dsa, dsb = ta.tensor(a, ta.int8, device), ta.tensor(sa, ta.float32, device), ta.tensor(sb, ta.float32, device)
    got = ops.matmul_quantized(da[:, 1:rows + 1], dsa[:, 1:rows + 1], w, dsb, ta.float32)
    check(got.numpy(), a[:, 1:rows + 1], sa[:, 1:rows + 1], b, sb, ta.float32)
    got = ops.matmul_quantized(da.transpose(0, 1), dsa.transpose(0, 1), w, dsb, ta.float32)
    check(got.numpy(), np.swapaxes(a, 0, 1), np.swapaxes(sa, 0, 1), b, sb, ta.float32)


@pytest.mark.parametrize("m", [1, 20, 40, 200])
def test_the_largest_sums(m, device):
    """-128 throughout, as few bits as a sum may lose: 2^14 K."""
    k, n = 131071 if m <= 20 else 65536, 24
    a, b = np.full((m, k), -128), np.full((n, k), -128)
    b[1::2] = 127
    ones = ta.tensor(np.ones(max(m, n)), ta.float32, device)
    got = ops.matmul_quantized(ta.tensor(a, ta.int8, device), ones[0:m], ta.tensor(b, ta.int8, device).transpose(), ones[0:n], ta.float32).numpy()
    want = np.where(np.arange(n) % 2 == 0, 16384.0 * k, -16256.0 * k)
    np.testing.assert_array_equal(got, np.broadcast_to(want.astype(np.float32), (m, n)))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 40, 256), (40, 200, 128), (300, 520, 512), (7, 9, 10)])
def test_rows_that_are_not_finite_stay_among_themselves(m, n, k, dtype, device):
    rng = np.random.default_rng(15)
    a, sa, b, sb = operands(rng, m, n, k)
    sa[m // 2], sb[n - 1] = np.nan, np.inf
    w = ta.tensor(np.ascontiguousarray(b.T), ta.int8, device).transpose()
    got = ops.matmul_quantized(ta.tensor(a, ta.int8, device), ta.tensor(sa, ta.float32, device), w, ta.tensor(sb, ta.float32, device), dtype).numpy()
    with np.errstate(invalid="ignore"):
        want = rounded(product(a, sa, b, sb), dtype)
    np.testing.assert_array_equal(got, want)
    assert np.isnan(got[m // 2]).all()


@pytest.mark.parametrize("shape", [((0, 16), (16, 8)), ((4, 16), (16, 0)), ((4, 0), (0, 8)), ((2, 0, 16), (16, 8))], ids=str)
def test_nothing_there(shape, device):
    a, b = (ta.Tensor(ta.int8, s).initialize(device) for s in shape)
    sa, sb = ta.tensor(np.ones(shape[0][:-1]), ta.float32, device), ta.tensor(np.ones(shape[1][-1:]), ta.float32, device)
    got = ops.matmul_quantized(a, sa, b, sb, ta.float16)
    assert got.shape == shape[0][:-1] + shape[1][-1:]
    assert not got.numpy().any()


def test_the_same_bits_every_time(device):
    """Parts of a sum that meet in any order give the same whole number."""
    rng = np.random.default_rng(16)
    for m, n, k in ((33, 256, 8192), (128, 512, 4096), (64, 4096, 2048)):
        a, sa, b, sb = operands(rng, m, n, k)
        on_device = ta.tensor(a, ta.int8, device), ta.tensor(sa, ta.float32, device), ta.tensor(np.ascontiguousarray(b.T), ta.int8, device).transpose(), ta.tensor(sb, ta.float32, device)
        want = rounded(product(a, sa, b, sb), ta.float16)
        for _ in range(5):
            np.testing.assert_array_equal(ops.matmul_quantized(*on_device, ta.float16).numpy(), want)
