"""What the operators on rows of 8-bit integers and their product refuse, before anything is launched: no GPU is needed."""
import ctypes as C

import pytest

import tannic_amd as ta
from tannic_amd import abi, ops


def zeros(shape, dtype=ta.float32):
    return ta.Tensor(dtype, shape).initialize()


def named(shape, dtype=ta.float32, strides=None):
    """A tensor of any size as a descriptor only: nothing may read it."""
    t = ta.Tensor(dtype, shape, strides)
    t.buffer = zeros((16,)).buffer
    return t


def call(name, operands, *extra):
    lib = ta.library()
    stream = abi.stream_t(0)
    operands = [None if t is None else C.byref(t.descriptor()) for t in operands]
    return lib.kernels[name](*operands, stream, *extra), lib.error_message()


def ids(other):
    return "-".join(f"{k}{None if v is None else v.shape}{'' if v is None else v.dtype}" for k, v in other.items())


def quantize(**other):
    t = {"x": zeros((3, 8)), "dst": zeros((3, 8), ta.int8), "scales": zeros((3,))}
    t.update(other)
    return call("quantize", list(t.values()))


def swiglu(**other):
    t = {"gate": zeros((3, 8)), "up": zeros((3, 8)), "dst": zeros((3, 8), ta.int8), "scales": zeros((3,))}
    t.update(other)
    return call("swiglu_quantize", list(t.values()))


def norm(**other):
    t = {"x": zeros((3, 8)), "residual": zeros((3, 8)), "gain": zeros((8,)), "total": zeros((3, 8)), "dst": zeros((3, 8), ta.int8), "scales": zeros((3,))}
    t.update(other)
    return call("add_rms_norm", list(t.values()), 1e-5)


def dequantize(**other):
    t = {"values": zeros((3, 8), ta.int8), "scales": zeros((3,)), "dst": zeros((3, 8))}
    t.update(other)
    return call("dequantize", list(t.values()))


def gemm(**other):
    t = {"a": zeros((3, 8), ta.int8), "a_scales": zeros((3,)), "b": zeros((8, 5), ta.int8), "b_scales": zeros((5,)), "dst": zeros((3, 5))}
    t.update(other)
    return call("gemm_quantized", list(t.values()))


@pytest.mark.parametrize("other", [{"x": None}, {"dst": None}, {"scales": None}, {"x": zeros((3, 9))}, {"x": zeros((24,))}, {"dst": zeros((8, 3), ta.int8).transpose()}, {"scales": zeros((3, 1))},
                                   {"scales": zeros((4,))}, {"scales": zeros((6,))[::2]}, {"x": zeros(()), "dst": zeros((), ta.int8), "scales": zeros(())},
                                   {"x": named((1 << 31, 2)), "dst": named((1 << 31, 2), ta.int8), "scales": named((1 << 31,))},
                                   {"x": named((1 << 20, 1 << 11, 2)), "dst": named((1 << 20, 1 << 11, 2), ta.int8), "scales": named((1 << 20, 1 << 11))},
                                   {"x": named((1, 1 << 31)), "dst": named((1, 1 << 31), ta.int8), "scales": zeros((1,))}], ids=ids)
def test_quantize_shapes(other):
    status, message = quantize(**other)
    assert status == abi.ERROR and "quantize" in message, message


@pytest.mark.parametrize("other", [{"up": None}, {"scales": None}, {"up": zeros((3, 9))}, {"up": zeros((1, 8))}, {"dst": zeros((3, 9), ta.int8)}, {"scales": zeros((8,))},
                                   {"gate": zeros(()), "up": zeros(()), "dst": zeros((), ta.int8), "scales": zeros(())}], ids=ids)
def test_swiglu_shapes(other):
    status, message = swiglu(**other)
    assert status == abi.ERROR and "swiglu_quantize" in message, message


@pytest.mark.parametrize("other", [{"x": None}, {"gain": None}, {"dst": None}, {"residual": None}, {"total": None}, {"residual": zeros((1, 8))}, {"total": zeros((8, 3)).transpose()},
                                   {"dst": zeros((3, 7), ta.int8)}, {"gain": zeros((7,))}, {"gain": zeros((1, 8))}, {"gain": zeros((16,))[::2]}, {"scales": zeros((3, 1))}, {"scales": zeros((6,))[::2]},
                                   {"x": zeros(()), "residual": None, "total": None, "dst": zeros((), ta.int8), "scales": zeros(())}], ids=ids)
def test_add_rms_norm_shapes(other):
    status, message = norm(**other)
    assert status == abi.ERROR and "add_rms_norm" in message, message


@pytest.mark.parametrize("other", [{"values": None}, {"dst": None}, {"scales": None}, {"scales": zeros((8,))}, {"dst": zeros((3, 7))}, {"dst": zeros((8, 3)).transpose()},
                                   {"values": zeros((), ta.int8), "dst": zeros(()), "scales": zeros(())}], ids=ids)
def test_dequantize_shapes(other):
    status, message = dequantize(**other)
    assert status == abi.ERROR and "dequantize" in message, message


@pytest.mark.parametrize("other", [{"a": None}, {"a_scales": None}, {"b_scales": None}, {"dst": None}, {"a": zeros((3, 9), ta.int8)}, {"a": zeros((8,), ta.int8)}, {"b": zeros((8, 6), ta.int8)},
                                   {"a_scales": zeros((8,))}, {"a_scales": zeros((3, 1))}, {"a_scales": zeros(())}, {"b_scales": zeros((8,))}, {"b_scales": zeros((1, 5))},
                                   {"dst": zeros((5, 3)).transpose()}, {"dst": zeros((3, 5, 1))},
                                   {"a": zeros((2, 3, 8), ta.int8), "a_scales": zeros((3,)), "dst": zeros((2, 3, 5))},
                                   {"b": zeros((2, 8, 5), ta.int8), "b_scales": zeros((3, 5)), "dst": zeros((2, 3, 5))},
                                   {"b": zeros((2, 8, 5), ta.int8), "b_scales": zeros((2, 5)), "dst": zeros((3, 3, 5))},
                                   {"a": named((3, 1 << 17), ta.int8), "b": named((1 << 17, 5), ta.int8)}], ids=ids)
def test_gemm_quantized_shapes(other):
    status, message = gemm(**other)
    assert status == abi.ERROR and "gemm" in message, message


@pytest.mark.parametrize("call_of,other", [
    (quantize, {"x": zeros((3, 8), ta.float64)}), (quantize, {"x": zeros((3, 8), ta.int32)}), (quantize, {"dst": zeros((3, 8), ta.int16)}), (quantize, {"scales": zeros((3,), ta.float16)}),
    (swiglu, {"up": zeros((3, 8), ta.float16)}), (swiglu, {"gate": zeros((3, 8), ta.float64), "up": zeros((3, 8), ta.float64)}), (swiglu, {"dst": zeros((3, 8))}),
    (norm, {"gain": zeros((8,), ta.float16)}), (norm, {"residual": zeros((3, 8), ta.bfloat16)}), (norm, {"total": zeros((3, 8), ta.bfloat16)}), (norm, {"scales": None}),
    (norm, {"dst": zeros((3, 8))}), (norm, {n: zeros((8,) if n == "gain" else (3, 8), ta.float64) for n in ("x", "residual", "gain", "total")}),
    (dequantize, {"values": zeros((3, 8), ta.int16)}), (dequantize, {"dst": zeros((3, 8), ta.float64)}), (dequantize, {"scales": zeros((3,), ta.bfloat16)}),
    (gemm, {"a": zeros((3, 8), ta.int16)}), (gemm, {"b": zeros((8, 5), ta.float32)}), (gemm, {"a_scales": zeros((3,), ta.float64)}), (gemm, {"b_scales": zeros((5,), ta.float16)}),
    (gemm, {"dst": zeros((3, 5), ta.int32)}), (gemm, {"dst": zeros((3, 5), ta.float64)}),
], ids=lambda v: v.__name__ if callable(v) else ids(v))
def test_types(call_of, other):
    assert call_of(**other)[0] == abi.UNSUPPORTED_DTYPE


@pytest.mark.parametrize("call_of", [quantize, swiglu, norm, dequantize, gemm], ids=lambda f: f.__name__)
def test_host_operands_are_refused(call_of):
    status, message = call_of()
    assert status == abi.ERROR and "device" in message


def test_no_storage():
    for call_of, name in ((quantize, "x"), (swiglu, "up"), (norm, "gain"), (dequantize, "scales"), (gemm, "b")):
        t = ta.Tensor(ta.int8 if call_of is gemm else ta.float32, {"gain": (8,), "scales": (3,), "b": (8, 5)}.get(name, (3, 8)))
        t.buffer = zeros((16,)).buffer
        d = t.descriptor()
        d.address = None
        t.descriptor = lambda d=d: d
        status, message = call_of(**{name: t})
        assert status == abi.ERROR and "storage" in message


def test_the_operators_on_the_host():
    x, values, scales = zeros((3, 8)), zeros((3, 8), ta.int8), zeros((3,))
    for refused in (lambda: ops.quantize(x), lambda: ops.swiglu_quantized(x, x), lambda: ops.add_rms_norm(x, x, zeros((8,))), lambda: ops.add_rms_norm_quantized(x, None, zeros((8,))),
                    lambda: ops.dequantize(values, scales, ta.float32), lambda: ops.matmul_quantized(values, scales, values.transpose(), scales, ta.float32)):
        with pytest.raises(ta.BackendError):
            refused()


def test_the_operators_ask_for_rows():
    for refused in (lambda: ops.quantize(zeros(())), lambda: ops.swiglu_quantized(zeros(()), zeros(())), lambda: ops.add_rms_norm(zeros(()), None, zeros((1,))),
                    lambda: ops.matmul_quantized(zeros((8,), ta.int8), zeros(()), zeros((8, 5), ta.int8), zeros((5,)), ta.float32),
                    lambda: ops.matmul_quantized(zeros((3, 8), ta.int8), zeros((3,)), zeros((7, 5), ta.int8), zeros((5,)), ta.float32),
                    lambda: ops.matmul_quantized(zeros((2, 3, 8), ta.int8), zeros((2, 3)), zeros((3, 8, 5), ta.int8), zeros((3, 5)), ta.float32)):
        with pytest.raises(ta.TannicError):
            refused()
