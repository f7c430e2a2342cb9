"""What the operators on a paged cache and the attention refuse, before anything is launched: no GPU is needed."""
import ctypes as C

import numpy as np
import pytest

import tannic_amd as ta
from tannic_amd import abi, ops


def zeros(shape, dtype=ta.float32):
    return ta.Tensor(dtype, shape).initialize()


def call(name, operands, *extra):
    lib = ta.library()
    stream = abi.stream_t(0)
    operands = [None if t is None else C.byref(t.descriptor()) for t in operands]
    return lib.kernels[name](*operands, stream, *extra), lib.error_message()


def attend_pages(**other):
    t = {"q": zeros((5, 4, 8)), "keys": zeros((6, 2, 4, 8)), "values": zeros((6, 2, 4, 8)), "table": zeros((3, 2), ta.int32), "starts": zeros((4,), ta.int32),
         "context": zeros((3,), ta.int32), "dst": zeros((5, 4, 8))}
    t.update(other)
    return call("attend_pages", list(t.values()), 1.0)


@pytest.mark.parametrize("other", [
    {"q": None}, {"dst": None}, {"table": None},
    {"q": zeros((5, 4, 9))}, {"q": zeros((5, 32))}, {"dst": zeros((5, 4, 7))}, {"dst": zeros((4, 5, 8)).transpose(0, 1)},
    {"q": zeros((5, 3, 8)), "dst": zeros((5, 3, 8))}, {"q": zeros((5, 8, 4)).transpose(1, 2)[:, :, 0:8]},
    {"keys": zeros((6, 2, 4, 9))}, {"values": zeros((6, 2, 5, 8))}, {"keys": zeros((6, 2, 8, 4)).transpose(2, 3), "values": zeros((6, 2, 8, 4)).transpose(2, 3)},
    {"keys": zeros((6, 2, 0, 8)), "values": zeros((6, 2, 0, 8))}, {"keys": zeros((6, 0, 4, 8)), "values": zeros((6, 0, 4, 8))},
    {"table": zeros((4, 2), ta.int32)}, {"table": zeros((6,), ta.int32)}, {"table": zeros((2, 3), ta.int32).transpose(0, 1)}, {"starts": zeros((3,), ta.int32)},
    {"context": zeros((3, 1), ta.int32)}, {"context": zeros((6,), ta.int32)[::2]}, {"q": zeros((5, 4, 257)), "dst": zeros((5, 4, 257)), "keys": zeros((6, 2, 4, 257)), "values": zeros((6, 2, 4, 257))},
], ids=lambda o: "-".join(f"{k}{None if v is None else v.shape}" for k, v in o.items()))
def test_attend_pages_shapes(other):
    status, message = attend_pages(**other)
    assert status == abi.ERROR and ("attend_pages" in message or "paged cache" in message), message


@pytest.mark.parametrize("other", [{"q": zeros((5, 4, 8), ta.float16)}, {"keys": zeros((6, 2, 4, 8), ta.bfloat16)}, {"table": zeros((3, 2), ta.int64)}, {"starts": zeros((4,), ta.float32)},
                                   {"context": zeros((3,), ta.int16)}, {"dst": zeros((5, 4, 8), ta.float64)}], ids=lambda o: str(list(o)))
def test_attend_pages_types(other):
    assert attend_pages(**other)[0] == abi.UNSUPPORTED_DTYPE


def test_host_operands_are_refused():
    status, message = attend_pages()
    assert status == abi.ERROR and "device" in message
    with pytest.raises(ta.BackendError):
        ops.attend_pages(zeros((5, 4, 8)), zeros((6, 2, 4, 8)), zeros((6, 2, 4, 8)), zeros((3, 2), ta.int32), zeros((4,), ta.int32), zeros((3,), ta.int32))
    with pytest.raises(ta.BackendError):
        ops.attend(zeros((2, 5, 4, 8)), zeros((2, 6, 2, 8)), zeros((2, 6, 2, 8)))
    with pytest.raises(ta.BackendError):
        ops.copy_pages(zeros((4, 2, 4, 8)), [0], [1])
    with pytest.raises(ta.BackendError):
        ops.append_pages(zeros((5, 2, 8)), zeros((5, 2, 8)), zeros((6, 2, 4, 8)), zeros((6, 2, 4, 8)), zeros((3, 2), ta.int32), zeros((4,), ta.int32), zeros((3,), ta.int32))


def test_nothing_to_do_is_no_error():
    assert attend_pages(q=zeros((0, 4, 8)), dst=zeros((0, 4, 8)))[0] == abi.SUCCESS
    assert attend_pages(table=zeros((0, 2), ta.int32), starts=zeros((1,), ta.int32), context=zeros((0,), ta.int32))[0] == abi.SUCCESS
    assert call("attend", [zeros((0, 5, 4, 8)), zeros((0, 6, 2, 8)), zeros((0, 6, 2, 8)), None, zeros((0, 5, 4, 8))], 1.0)[0] == abi.SUCCESS
    assert call("copy_pages", [zeros((4, 2, 4, 8))], None, None, 0)[0] == abi.SUCCESS


def attend(**other):
    t = {"q": zeros((2, 5, 4, 8)), "k": zeros((2, 6, 2, 8)), "v": zeros((2, 6, 2, 8)), "lengths": zeros((2,), ta.int32), "dst": zeros((2, 5, 4, 8))}
    t.update(other)
    return call("attend", list(t.values()), 1.0)


@pytest.mark.parametrize("other", [
    {"k": None}, {"q": zeros((5, 4, 8))}, {"k": zeros((2, 6, 2, 9))}, {"v": zeros((2, 7, 2, 8))}, {"k": zeros((3, 6, 2, 8)), "v": zeros((3, 6, 2, 8))},
    {"k": zeros((2, 6, 3, 8)), "v": zeros((2, 6, 3, 8))}, {"k": zeros((2, 6, 0, 8)), "v": zeros((2, 6, 0, 8))}, {"dst": zeros((2, 4, 5, 8)).transpose(1, 2)}, {"lengths": zeros((3,), ta.int32)},
    {"lengths": zeros((2, 1), ta.int32)}, {"lengths": zeros((4,), ta.int32)[::2]}, {"k": zeros((2, 6, 8, 2)).transpose(2, 3), "v": zeros((2, 6, 8, 2)).transpose(2, 3)},
    {"q": zeros((2, 5, 4, 300)), "dst": zeros((2, 5, 4, 300)), "k": zeros((2, 6, 2, 300)), "v": zeros((2, 6, 2, 300))},
], ids=lambda o: "-".join(f"{k}{None if v is None else v.shape}" for k, v in o.items()))
def test_attend_shapes(other):
    status, message = attend(**other)
    assert status == abi.ERROR and "attend" in message, message


def test_attend_types():
    assert attend(q=zeros((2, 5, 4, 8), ta.int32), dst=zeros((2, 5, 4, 8), ta.int32))[0] == abi.UNSUPPORTED_DTYPE
    assert attend(k=zeros((2, 6, 2, 8), ta.float16))[0] == abi.UNSUPPORTED_DTYPE
    assert attend(lengths=zeros((2,), ta.int64))[0] == abi.UNSUPPORTED_DTYPE


def append(**other):
    t = {"k": zeros((5, 2, 8)), "v": zeros((5, 2, 8)), "table": zeros((3, 2), ta.int32), "starts": zeros((4,), ta.int32), "context": zeros((3,), ta.int32), "cos": zeros((9, 4)),
         "sin": zeros((9, 4)), "q": zeros((5, 4, 8)), "keys": zeros((6, 2, 4, 8)), "values": zeros((6, 2, 4, 8)), "turned": zeros((5, 4, 8))}
    t.update(other)
    return call("append_pages", list(t.values()))


@pytest.mark.parametrize("other", [
    {"k": None}, {"keys": None}, {"cos": None}, {"sin": None}, {"q": None}, {"turned": None}, {"cos": None, "sin": None}, {"k": zeros((5, 3, 8)), "v": zeros((5, 3, 8))}, {"v": zeros((4, 2, 8))},
    {"k": zeros((5, 2, 6)), "v": zeros((5, 2, 6))}, {"q": zeros((4, 4, 8)), "turned": zeros((4, 4, 8))}, {"turned": zeros((5, 4, 9))}, {"turned": zeros((4, 5, 8)).transpose(0, 1)},
    {"cos": zeros((9, 8)), "sin": zeros((9, 8))}, {"cos": zeros((8, 4))}, {"cos": zeros((0, 4)), "sin": zeros((0, 4))}, {"cos": zeros((4, 9)).transpose(0, 1), "sin": zeros((4, 9)).transpose(0, 1)},
    {"k": zeros((5, 8, 2)).transpose(1, 2), "v": zeros((5, 8, 2)).transpose(1, 2)}, {"starts": zeros((3,), ta.int32)},
    {n: zeros(s) for n, s in (("k", (5, 2, 7)), ("v", (5, 2, 7)), ("q", (5, 4, 7)), ("turned", (5, 4, 7)), ("keys", (6, 2, 4, 7)), ("values", (6, 2, 4, 7)), ("cos", (9, 3)), ("sin", (9, 3)))},
], ids=lambda o: "-".join(f"{k}{None if v is None else v.shape}" for k, v in o.items()))
def test_append_pages_shapes(other):
    status, message = append(**other)
    assert status == abi.ERROR and ("append_pages" in message or "paged cache" in message), message


def test_append_pages_types():
    assert append(k=zeros((5, 2, 8), ta.float16))[0] == abi.UNSUPPORTED_DTYPE
    assert append(cos=zeros((9, 4), ta.float16), sin=zeros((9, 4), ta.float16))[0] == abi.UNSUPPORTED_DTYPE
    assert append(cos=zeros((9, 4), ta.float64))[0] == abi.UNSUPPORTED_DTYPE
    assert append(context=zeros((3,), ta.int64))[0] == abi.UNSUPPORTED_DTYPE
    status, message = append()
    assert status == abi.ERROR and "device" in message


def numbers(*n):
    return (C.c_int32 * len(n))(*n)


@pytest.mark.parametrize("pool,sources,targets", [
    (None, (0,), (1,)), (zeros((4, 2, 8)), (0,), (1,)), (zeros((4, 2, 4, 8)), (4,), (0,)), (zeros((4, 2, 4, 8)), (0,), (4,)), (zeros((4, 2, 4, 8)), (-1,), (0,)), (zeros((4, 2, 4, 8)), (0,), (-(1 << 31),)),
    (zeros((4, 4, 2, 8)).transpose(1, 2), (0,), (1,)), (zeros((1, 2, 4, 8)).expand(4, 2, 4, 8), (0,), (1,)), (zeros((0, 2, 4, 8)), (0,), (0,)),
], ids=str)
def test_copy_pages(pool, sources, targets):
    lib = ta.library()
    status = lib.kernels["copy_pages"](None if pool is None else C.byref(pool.descriptor()), abi.stream_t(0), numbers(*sources), numbers(*targets), len(sources))
    assert status == abi.ERROR and "copy_pages" in lib.error_message()


def test_copy_pages_lists():
    pool = zeros((4, 2, 4, 8))
    for sources, targets in (([0, 1], [2]), ([0.5], [1]), ([1 << 31], [0]), ([-1], [0]), ([(1 << 32) + 1], [0])):
        with pytest.raises(ta.TannicError):
            ops.copy_pages(pool, sources, targets)
    lib = ta.library()
    assert lib.kernels["copy_pages"](C.byref(zeros((4, 2, 4, 8), ta.boolean).descriptor()), abi.stream_t(0), numbers(0), numbers(1), 1) == abi.UNSUPPORTED_DTYPE
    assert lib.kernels["copy_pages"](C.byref(pool.descriptor()), abi.stream_t(0), None, None, 1) == abi.ERROR


def test_more_tokens_than_a_launch_has_blocks():
    many, one = zeros((1 << 24, 1, 1), ta.float16), zeros((1, 1, 1, 1), ta.float16)
    table, starts, context = zeros((1, 1), ta.int32), zeros((2,), ta.int32), zeros((1,), ta.int32)
    for status, message in (call("attend_pages", [many, one, one, table, starts, context, many], 1.0), call("append_pages", [many, many, table, starts, context, None, None, None, one, one, None]),
                            call("attend", [zeros((1, 1 << 24, 1, 1), ta.float16), one, one, None, zeros((1, 1 << 24, 1, 1), ta.float16)], 1.0)):
        assert status == abi.ERROR and "2^24" in message, message
