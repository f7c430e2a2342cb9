"""Several Python threads on one device: what a thread reads is what was computed, whoever computed it, and the streams that memory and copies follow stay those of the calls."""
import ctypes as C
import threading

import numpy as np
import pytest

import tannic_amd as ta
from quantized_support import product, rounded
from tannic_amd import ops
from tannic_amd.tensor import Buffer

pytestmark = pytest.mark.gpu


def together(*works):
    """Runs the functions in threads; what any of them raised."""
    raised = []

    def run(work):
        try:
            work()
        except BaseException as e:      # (an assertion as well: a thread's is lost otherwise)
            raised.append(e)

    threads = [threading.Thread(target=run, args=(work,)) for work in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if raised:
        raise raised[0]


def handed_out(device):
    lib = ta.library()
    dvc = device.structure()
    stream = lib.pop_stream(C.byref(dvc))
    lib.put_stream(C.byref(dvc), stream)
    return stream.address


def test_memory_and_copies_leave_the_pool_as_it_is(device):
    """Whatever threads allocate, release and copy at the same time, the stream that is handed out next is the one that the device's calls run on."""
    before = handed_out(device)
    assert before == device.stream_number()
    host = np.arange(1000, dtype=np.float32)

    def work():
        held = ta.tensor(host, ta.float32, device)
        for _ in range(1500):
            Buffer(4096, device)
            assert held.storage()[7] == 7.0

    together(work, work, work)
    after = handed_out(device)
    # (a pool that was turned round is put right before anything is said: the tests after this one take it as it is)
    lib, dvc, above = ta.library(), device.structure(), []
    while handed_out(device) != before and len(above) < 16:
        above.append(lib.pop_stream(C.byref(dvc)))
    mine = lib.pop_stream(C.byref(dvc))
    for stream in (*above, mine):
        lib.put_stream(C.byref(dvc), stream)
    assert after == before


# M, N, K: blocks that share K, joined by the last of them and by a second kernel, and one that shares nothing
SIZES = [(40, 128, 8192), (128, 384, 8192), (128, 4096, 14336), (30, 90, 500)]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_each_thread_reads_its_own(size, device):
    """Rows are quantised and multiplied by two threads on the device's stream, each of which reads its results right away, and releases them."""
    m, n, k = size
    rng = np.random.default_rng(91)
    w, sw = rng.integers(-127, 128, (n, k)), np.full(n, 0.01, np.float32)
    weights, channels = ta.tensor(w, ta.int8, device).transpose(), ta.tensor(sw, ta.float32, device)
    rows = [ta.tensor(rounded(rng.standard_normal((m, k)), ta.bfloat16), ta.bfloat16, device) for _ in range(2)]
    want = []
    for x in rows:
        values, scales = ops.quantize(x)
        want.append(rounded(product(values.numpy(), scales.numpy(), w.T, sw), ta.float32))

    def work(x, right):
        def run():
            for _ in range(40):
                np.testing.assert_array_equal(ops.matmul_quantized(*ops.quantize(x), weights, channels, ta.float32).numpy(), right)
        return run

    together(*(work(x, right) for x, right in zip(rows, want)))
    # and what one of them left is read by this one
    left = []
    together(lambda: left.extend(ops.matmul_quantized(*ops.quantize(rows[0]), weights, channels, ta.float32) for _ in range(20)),
             lambda: [ops.quantize(rows[1])[0].numpy() for _ in range(20)])
    for got in left:
        np.testing.assert_array_equal(got.numpy(), want[0])


def test_a_stream_is_of_the_device_that_it_is_asked_for(device):
    """A device that is not there has no streams (the current one's were handed out for it), and asking leaves no error behind."""
    from tannic_amd import abi
    lib = ta.library()
    nowhere = abi.device_t(lib.get_device_count())
    assert not lib.pop_stream(C.byref(nowhere)).address
    assert ops.add(ta.tensor(np.ones(5), ta.float32, device), ta.tensor(np.ones(5), ta.float32, device)).numpy().tolist() == [2.0] * 5


def test_the_other_calls_of_two_threads(device):
    """Operators that had taken a stream of the pool for themselves: softmax, allclose and copies between tensors."""
    rng = np.random.default_rng(92)
    x = rng.standard_normal((64, 3000)).astype(np.float32)
    d = ta.tensor(x, ta.float32, device)
    want = ops.softmax(d).storage()

    def work():
        for _ in range(60):
            y = ops.softmax(ops.add(d, d), None, 0.5)
            assert ops.allclose(y, y)
            np.testing.assert_array_equal(y.to(device).to(ta.Host()).storage(), want)

    together(work, work)
    assert handed_out(device) == device.stream_number()
