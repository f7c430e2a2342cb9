"""Where products and rows of 8-bit integers could go wrong beside the usual sizes: offsets beyond 32 bits, one row or column seen as many, steps without tokens, rows that no sequence
owns, and a process whose first calls are recorded."""
import subprocess
import sys

import numpy as np
import pytest

import support
import tannic_amd as ta
from quantized_support import assert_stands_for, integers_of, product, rounded
from tannic_amd import decoder_layer as dl, ops
from tannic_amd.paged_cache import PagedCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 20, 40, 300])
def test_weights_beyond_32_bits(m, device):
    """A matrix of 4.6 GB of which only the last and some first channels are looked at (the others hold whatever the memory held)."""
    n, k = 140000, 32768
    rng = np.random.default_rng(21)
    w = ta.Tensor(ta.int8, (n, k)).initialize(device)
    known = {0: 40, n - 70: 70}
    values = {}
    for first, count in known.items():
        values[first] = rng.integers(-127, 128, (count, k))
        ops.copy_into(w[first:first + count], ta.tensor(values[first], ta.int8, device))
    a, sa = rng.integers(-127, 128, (m, k)), rng.uniform(0.001, 0.002, m).astype(np.float32)
    sb = rng.uniform(0.005, 0.02, n).astype(np.float32)
    got = ops.matmul_quantized(ta.tensor(a, ta.int8, device), ta.tensor(sa, ta.float32, device), w.transpose(), ta.tensor(sb, ta.float32, device), ta.float32)
    for first, count in known.items():
        np.testing.assert_array_equal(ops.repack(got[:, first:first + count]).numpy(), product(a, sa, values[first].T, sb[first:first + count]))


@pytest.mark.parametrize("pitch", [4096, 4097, 1 << 23])
def test_rows_far_apart(pitch, device):
    """Rows of a cache of other things: pitches that no tile's 32-bit offsets hold are another kernel's."""
    rng = np.random.default_rng(22)
    rows, k = 300, 512
    w = ta.Tensor(ta.int8, (rows, pitch)).initialize(device)[:, 32:32 + k]
    values = rng.integers(-127, 128, (rows, k))
    ops.copy_into(w, ta.tensor(values, ta.int8, device))
    one = ta.tensor(np.ones(rows), ta.float32, device)
    for m in (3, 40, 300):
        a = rng.integers(-127, 128, (m, k))
        got = ops.matmul_quantized(ta.tensor(a, ta.int8, device), one[0:m], w.transpose(), one, ta.float32)
        np.testing.assert_array_equal(got.numpy(), (a @ values.T).astype(np.float32))
        got = ops.matmul_quantized(w[0:m], one[0:m], ta.tensor(values, ta.int8, device).transpose(), one, ta.float32)
        np.testing.assert_array_equal(got.numpy(), (values[:m] @ values.T).astype(np.float32))


def test_rows_beyond_32_bits(device):
    """5.2 GB of rows, the last of them looked at (the others hold whatever the memory held): values, sums, integers and the way back."""
    rows, length = 130000, 20008
    rng = np.random.default_rng(23)
    x = ta.Tensor(ta.bfloat16, (rows, length)).initialize(device)
    some = rounded(rng.standard_normal((3, length)), ta.bfloat16)
    ops.copy_into(x[rows - 3:], ta.tensor(some, ta.bfloat16, device))
    values, scales = ops.quantize(x)
    want, largest, _ = integers_of(some)

    def last(t):
        return ops.repack(t[rows - 3:]).numpy()

    np.testing.assert_array_equal(last(values), want)
    np.testing.assert_array_equal(scales.numpy()[rows - 3:], largest / np.float32(127))
    np.testing.assert_array_equal(last(ops.dequantize(values, scales, ta.bfloat16)), rounded(want * (largest / np.float32(127))[:, None], ta.bfloat16))
    del values, scales
    gain = ta.tensor(np.ones(length), ta.bfloat16, device)
    values, _, total = ops.add_rms_norm_quantized(x, x, gain)
    np.testing.assert_array_equal(last(total), 2 * some)
    np.testing.assert_array_equal(last(values), want)


def test_more_blocks_than_a_launch_has(device):
    """17.6 GB of short rows times one channel: as many of the smallest tiles as no launch holds, the first and the last rows looked at."""
    m, k = 1100000000, 16
    rng = np.random.default_rng(27)
    a = ta.Tensor(ta.int8, (m, k)).initialize(device)
    known = {0: 300, m - 300: 300}
    values = {first: rng.integers(-127, 128, (count, k)) for first, count in known.items()}
    for first, count in known.items():
        ops.copy_into(a[first:first + count], ta.tensor(values[first], ta.int8, device))
    b = rng.integers(-127, 128, (1, k))
    one = ta.tensor(np.ones(1), ta.float32, device)
    got = ops.matmul_quantized(a, one.expand(m), ta.tensor(b, ta.int8, device).transpose(), one, ta.float32)
    for first, count in known.items():
        np.testing.assert_array_equal(ops.repack(got[first:first + count]).numpy(), values[first] @ b.T)


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float16, ta.float32], ids=str)
@pytest.mark.parametrize("m,n,k", [(64, 64, 16), (70, 90, 17), (1, 1, 31), (5, 100, 127), (33, 65, 129), (40, 70, 255), (65, 60, 385), (1, 100, 4097), (33, 1000, 14335), (64, 300, 8191), (100, 70, 40001),
                                   (20, 64, 131071)])
def test_rows_of_any_length_from_anywhere(m, n, k, dtype, device):
    """K of no whole pieces, of a piece and a little, short and shared between blocks; rows one after the other, and from a byte that no load is aligned to."""
    rng = np.random.default_rng(28)
    a, b = rng.integers(-128, 128, (m, k)), rng.integers(-128, 128, (n, k))
    each = 1.0 / (70.0 * k ** 0.5)
    sa, sb = rng.uniform(0.5 * each, 1.5 * each, m).astype(np.float32), rng.uniform(0.005, 0.02, n).astype(np.float32)
    want = rounded(product(a, sa, b.T, sb), dtype)
    scales = ta.tensor(sa, ta.float32, device), ta.tensor(sb, ta.float32, device)

    def cut(values, pitch, first):
        whole = ta.tensor(rng.integers(-128, 128, (len(values), pitch)), ta.int8, device)[:, first:first + values.shape[1]]
        ops.copy_into(whole, ta.tensor(values, ta.int8, device))
        return whole
    for da, db in ((ta.tensor(a, ta.int8, device), ta.tensor(b, ta.int8, device)), (cut(a, k + 5, 3), cut(b, k + 18, 7))):
        np.testing.assert_array_equal(ops.matmul_quantized(da, scales[0], db.transpose(), scales[1], dtype).numpy(), want)


def test_recordings_of_rows_from_anywhere(device):
    """Two recordings whose products share K between blocks, replayed in turn with eager products between."""
    rng = np.random.default_rng(29)
    made = []
    for m, n, k in ((40, 128, 8191), (20, 64, 4097), (64, 500, 4099)):
        a, b = (rng.integers(-127, 128, s) for s in ((m, k), (n, k)))
        operands = (ta.tensor(a, ta.int8, device), ta.tensor(np.full(m, 0.001), ta.float32, device), ta.tensor(b, ta.int8, device).transpose(), ta.tensor(np.full(n, 0.01), ta.float32, device))
        made.append((operands, product(a, np.full(m, 0.001, np.float32), b.T, np.full(n, 0.01, np.float32))))
    with ta.Graph(device) as first:
        ones = [ops.matmul_quantized(*operands, ta.float32) for operands, _ in made]
    with ta.Graph(device) as second:
        twos = [ops.matmul_quantized(*operands, ta.float32) for operands, _ in reversed(made)]
    for _ in range(4):
        first.launch()
        second.launch()
        for operands, want in made:
            np.testing.assert_array_equal(ops.matmul_quantized(*operands, ta.float32).numpy(), want)
        first.launch()
        for (_, want), one, two in zip(made, ones, reversed(twos)):
            np.testing.assert_array_equal(one.numpy(), want)
            np.testing.assert_array_equal(two.numpy(), want)


@pytest.mark.parametrize("m,n,k", [(5, 40, 256), (40, 300, 128), (300, 64, 1000), (40, 70, 333)])
def test_one_row_and_one_column_seen_as_many(m, n, k, device):
    rng = np.random.default_rng(24)
    a, b = rng.integers(-127, 128, (1, k)), rng.integers(-127, 128, (1, k))
    da, db = ta.tensor(a, ta.int8, device), ta.tensor(b, ta.int8, device)
    sa, sb = ta.tensor(rng.uniform(0.001, 0.002, 1), ta.float32, device).expand(m), ta.tensor(rng.uniform(0.01, 0.02, 1), ta.float32, device).expand(n)
    got = ops.matmul_quantized(da.expand(m, k), sa, db.expand(n, k).transpose(), sb, ta.float32).numpy()
    np.testing.assert_array_equal(got, product(np.repeat(a, m, 0), sa.numpy(), np.repeat(b, n, 0).T, sb.numpy()))


@pytest.mark.parametrize("length", [40, 41, 5000, 70000])
@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float32], ids=str)
def test_gates_at_the_ends_of_the_type(dtype, length, device):
    """A gate beyond 2^127 / log2 e is itself, or 0 below 0: a row of nothing else, and beside small ones (the same bounds as everywhere: the steps are the same)."""
    largest = 3e38
    rng = np.random.default_rng(30)
    gate = rounded(np.stack([np.full(length, largest), rng.choice([largest, -largest, 0.5], length), rng.choice([-largest, 1.0], length), rng.choice([-150.0, 150.0, 88.0, -88.0], length)]), dtype)
    up = rounded(rng.uniform(0.25, 0.75, (4, length)), dtype)
    values, scales = ops.swiglu_quantized(ta.tensor(gate, dtype, device), ta.tensor(up, dtype, device))
    wide = gate.astype(np.float64)
    want = np.where(wide > -700, wide / (1 + np.exp(np.minimum(-wide, 700))), 0) * up
    assert_stands_for(values.numpy(), scales.numpy(), want, 6 * 2.0 ** -24)


SHAPE = dl.LayerShape(hidden=128, heads=4, kv_heads=2, head_dim=32, ffn=320)


def model(device, dtype=ta.bfloat16):
    w = dl.quantize_weights({name: ta.tensor(np.ones(size) if name.startswith("g") else support.normal(91, 10 + i, size, 0.05), dtype, device)
                             for i, (name, size) in enumerate(dl.weight_shapes(SHAPE).items())})
    return w, w["g1"], *dl.rotary_tables(SHAPE, 64, dtype, device), PagedCache(1, 16, 8, SHAPE.kv_heads, SHAPE.head_dim, dtype, device)


def test_a_step_without_tokens(device):
    w, gain, cos, sin, cache = model(device)
    a = cache.add()
    step = cache.plan([a], [0])
    out = dl.stack_paged_quantized(SHAPE, [w], gain, ta.Tensor(ta.bfloat16, (1, 0, SHAPE.hidden)).initialize(device), cos, sin, cache, step)
    assert out.shape == (1, 0, SHAPE.hidden)


@pytest.mark.parametrize("rest", [0.0, np.nan, 3e38])
def test_rows_of_no_sequence_stay_among_themselves(rest, device):
    """A batch padded with rows of anything: the others come out as without them, bit for bit."""
    rng = np.random.default_rng(25)
    w, gain, cos, sin, cache = model(device)
    a, b = cache.add(), cache.add()
    x = rng.standard_normal((7, SHAPE.hidden))
    step = cache.plan([a, b], [4, 3])
    want = dl.stack_paged_quantized(SHAPE, [w], gain, ta.tensor(x[None], ta.bfloat16, device), cos, sin, cache, step).numpy()
    padded = np.full((12, SHAPE.hidden), rest)
    padded[:7] = x
    got = dl.stack_paged_quantized(SHAPE, [w], gain, ta.tensor(padded[None], ta.bfloat16, device), cos, sin, cache, step).numpy()
    np.testing.assert_array_equal(got[:, :7], want)


def test_a_first_call_that_is_recorded(tmp_path):
    """A process whose first product that shares K is inside a recording: scratch and counts are there at every replay, and for eager calls after it."""
    program = tmp_path / "first.py"
    program.write_text('''
import sys
sys.path.insert(0, sys.argv[1])
import numpy as np
import tannic_amd as ta
from tannic_amd import ops
device = ta.Device(0)
rng = np.random.default_rng(26)
x = ta.tensor(rng.standard_normal((40, 8192)), ta.float16, device)
w = ta.tensor(rng.integers(-127, 128, (128, 8192)), ta.int8, device).transpose()
each = ta.tensor(np.full(128, 0.01), ta.float32, device)
gain = ta.tensor(np.ones(8192), ta.float16, device)
def chain():
    values, scales, total = ops.add_rms_norm_quantized(x, x, gain)
    return ops.matmul_quantized(values, scales, w, each, ta.float16)
with ta.Graph(device) as g:
    held = chain()
for i in range(4):
    g.launch()
    got = held.storage()
    eager = chain().storage()
    assert np.array_equal(got, eager), i
assert held.numpy().any()
print("same")
''')
    import os
    done = subprocess.run([sys.executable, str(program), os.path.dirname(os.path.dirname(os.path.abspath(__file__)))], capture_output=True, text=True, timeout=110)
    assert done.returncode == 0 and done.stdout.strip() == "same", done.stdout + done.stderr
