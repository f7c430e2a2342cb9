"""Which kernel a product of 8-bit integers runs, asked of the library without a GPU (``tannic_hip_gemm_quantized_plan``): operands along K never end in the kernel for any operands because
copies were counted on that are not made."""
import ctypes as C

import pytest

import tannic_amd as ta
import test_gpu_quantized_routes as routes
from tannic_amd import abi, types
from tannic_amd.tensor import contiguous_strides

ANY, FEW, TILES, ANYWHERE = 0, 1, 2, 3


def descriptor(dtype, shape):
    """A contiguous tensor of that shape at an address that is never read."""
    t = abi.tensor_t()
    t.address, t.rank, t.dtype, t.size = 0x10000, len(shape), types.BY_NAME[dtype].code, 1
    t.shape.sizes[:len(shape)] = shape
    t.strides.sizes[:len(shape)] = contiguous_strides(shape)
    return t


def plan(a_shape, w_shape, dst_shape, weights=None, tokens=None, start=0, order=None):
    a, w, dst, sa, sw = descriptor("int8", a_shape), descriptor("int8", w_shape), descriptor("bfloat16", dst_shape), descriptor("float32", a_shape[:-1]), descriptor("float32", w_shape[:-1])
    for t, pitch in ((a, tokens), (w, weights)):
        if pitch:
            t.strides.sizes[t.rank - 2] = pitch
    a.address += start
    if order == "weights":      # [K, N] one row after the other
        w.strides.sizes[w.rank - 2], w.strides.sizes[w.rank - 1] = 1, w_shape[-2]
    r = w.rank      # the matrix [out, in] is the second operand as [in, out]
    w.shape.sizes[r - 2], w.shape.sizes[r - 1] = w.shape.sizes[r - 1], w.shape.sizes[r - 2]
    w.strides.sizes[r - 2], w.strides.sizes[r - 1] = w.strides.sizes[r - 1], w.strides.sizes[r - 2]
    out = (C.c_uint32 * 2)()
    assert ta.library().gemm_quantized_plan(*(C.byref(t) for t in (a, sa, w, sw, dst)), out) == abi.SUCCESS
    return tuple(out)


def matrices(m, n, k, batch=()):
    return batch + (m, k), batch + (n, k), batch + (m, n)


@pytest.mark.parametrize("name", list(routes.PRODUCTS))
def test_the_products_of_the_gpu_tests(name):
    a, w, dst, weights, tokens = routes.shapes(name)
    assert plan(a, w, dst, weights, tokens) == (ANYWHERE, 0)


# M, N, K, batch dims -> the kernel, and what is copied first
PRODUCTS = [((1, 4096, 4096), (FEW, 0)), ((32, 6144, 4096), (FEW, 0)), ((32, 4096, 14336), (TILES, 0)), ((1, 28672, 4096), (TILES, 0)), ((512, 6144, 4096), (TILES, 0)),
            ((77, 2049, 1030), (ANYWHERE, 0)), ((1, 28672, 4095), (ANYWHERE, 0)), ((2048, 4096, 4095), (TILES, 3)), ((1024, 1024, 4095, (8,)), (TILES, 3)),
            ((1024, 1024, 4095, (2, 4)), (ANYWHERE, 0)), ((1024, 1024, 4096, (2, 4)), (TILES, 0)), ((300, 300, 10), (TILES, 3)), ((30, 30, 10), (ANY, 0)),
            # more bytes than are copied
            ((8192, 28672, 100001), (ANYWHERE, 0)), ((8192, 28672, 4095), (TILES, 3))]


@pytest.mark.parametrize("problem,want", PRODUCTS, ids=str)
def test_products(problem, want):
    assert plan(*matrices(*problem)) == want


def test_tokens_of_a_batch_over_one_matrix_are_rows_of_one_product():
    assert plan((2, 4, 300, 4095), (4096, 4095), (2, 4, 300, 4096)) == plan(*matrices(2400, 4096, 4095)) == (TILES, 3)


def test_copies_are_not_made_in_vain():
    """Tokens that would be copied beside weights that lie too far apart for the tiles, whatever is copied."""
    assert plan(*matrices(512, 4096, 4096), weights=1 << 22, start=1) == (ANYWHERE, 0)
    assert plan(*matrices(512, 4096, 4096), start=1) == (TILES, 1)
    assert plan(*matrices(512, 4096, 4096), weights=4097) == (TILES, 2)
    assert plan(*matrices(512, 4096, 4096), order="weights") == (TILES, 2)
    assert plan(*matrices(512, 4096, 4096, (2, 2)), order="weights") == (ANY, 0)


def test_what_the_product_refuses():
    a, w, dst, sa, sw = (descriptor(t, s) for t, s in (("int8", (4, 8)), ("int8", (8, 5)), ("bfloat16", (4, 6)), ("float32", (4,)), ("float32", (5,))))
    out = (C.c_uint32 * 2)()
    assert ta.library().gemm_quantized_plan(*(C.byref(t) for t in (a, sa, w, sw, dst)), out) == abi.ERROR
    assert ta.library().gemm_quantized_plan(C.byref(a), None, C.byref(w), C.byref(sw), C.byref(dst), out) == abi.ERROR
    dst.dtype = a.dtype
    assert ta.library().gemm_quantized_plan(*(C.byref(t) for t in (a, sa, w, sw, dst)), out) == abi.UNSUPPORTED_DTYPE
