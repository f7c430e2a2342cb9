"""Large products of 8-bit integers whose operands lie along K but not as the direct loads want them, and which are not copied into aligned rows first: batches of several dims, rows far apart
or in reverse order, more bytes than are copied.  ``test_quantized_plan`` says that these are the kernel for rows from anywhere; here are their results."""
import numpy as np
import pytest

import tannic_amd as ta
from quantized_support import product, rounded
from tannic_amd import ops

pytestmark = pytest.mark.gpu

# batch dims, M, N, K, the pitch of a matrix's rows in elements of the weights (None: K) and of the tokens
PRODUCTS = {
    "two_dims": ((2, 3), 1024, 1024, 1030, None, None),
    "two_dims_ragged": ((3, 2), 700, 1111, 1001, None, None),
    "two_dims_many": ((2, 4), 1024, 1024, 4095, None, None),
    "weights_far_apart": ((), 512, 4096, 4096, 1 << 22, None),
    "tokens_far_apart": ((), 1024, 2048, 2048, None, 1 << 22),
    "weights_far_apart_odd": ((), 512, 2048, 4001, (1 << 22) + 5, None),
}


def shapes(name):
    batch, m, n, k, weights, tokens = PRODUCTS[name]
    return batch + (m, k), batch + (n, k), batch + (m, n), weights, tokens


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float32], ids=str)
@pytest.mark.parametrize("name", list(PRODUCTS))
def test_products(name, dtype, device):
    a_shape, w_shape, _, weights, tokens = shapes(name)
    rng = np.random.default_rng(61)
    a, w = rng.integers(-127, 128, a_shape), rng.integers(-127, 128, w_shape)
    sa, sw = rng.uniform(0.0001, 0.0002, a_shape[:-1]).astype(np.float32), rng.uniform(0.005, 0.02, w_shape[:-1]).astype(np.float32)

    def placed(values, pitch):
        if pitch is None:
            return ta.tensor(values, ta.int8, device)
        # (what lies between the rows is whatever the memory held)
        view = ta.Tensor(ta.int8, (len(values), pitch)).initialize(device)[:, :values.shape[1]]
        ops.copy_into(view, ta.tensor(values, ta.int8, device))
        return view

    got = ops.matmul_quantized(placed(a, tokens), ta.tensor(sa, ta.float32, device), placed(w, weights).transpose(), ta.tensor(sw, ta.float32, device), dtype)
    np.testing.assert_array_equal(got.numpy(), rounded(product(a, sa, np.swapaxes(w, -1, -2), sw), dtype))


def test_rows_in_reverse_order(device):
    """Negative pitches, which Python's views do not have: the descriptors of the C ABI do."""
    import ctypes as C
    rng = np.random.default_rng(62)
    m, n, k = 512, 2048, 2048
    a, w = rng.integers(-127, 128, (m, k)), rng.integers(-127, 128, (n, k))
    sa, sw = np.full(m, 0.0001, np.float32), np.full(n, 0.01, np.float32)
    da, dw, dsa, dsw = ta.tensor(a, ta.int8, device), ta.tensor(w, ta.int8, device), ta.tensor(sa, ta.float32, device), ta.tensor(sw, ta.float32, device)
    out = ta.Tensor(ta.float32, (m, n)).initialize(device)
    turned = [t.descriptor() for t in (da, dsa, dw.transpose(), dsw, out)]
    turned[0].address += (m - 1) * k
    turned[0].strides.sizes[0] = -k
    turned[2].address += (n - 1) * k
    turned[2].strides.sizes[1] = -k
    plan = (C.c_uint32 * 2)()
    assert ta.library().gemm_quantized_plan(*(C.byref(t) for t in turned), plan) == 0 and tuple(plan) == (3, 0)
    assert ta.library().kernels["gemm_quantized"](*(C.byref(t) for t in turned), device.stream()) == 0
    np.testing.assert_array_equal(out.numpy(), product(a[::-1], sa, w[::-1].T, sw))
