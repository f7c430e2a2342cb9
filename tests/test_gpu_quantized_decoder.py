"""The operators of 8-bit integers together, as a serving program uses them: prompts and single tokens of several sequences through layers with quantised parameters over a paged
cache, eager and recorded, on the default device and several times at once."""
import threading

import numpy as np
import pytest

import support
import tannic_amd as ta
from attention_support import assert_within, head_attention
from quantized_support import HALF, TINY, integers_of, rounded
from tannic_amd import decoder_layer as dl, ops
from tannic_amd.paged_cache import PagedCache

pytestmark = pytest.mark.gpu

SHAPE = dl.LayerShape(hidden=256, heads=8, kv_heads=2, head_dim=64, ffn=704)
POSITIONS = 128


def parameters(dtype, device, seed, packed):
    w = {name: ta.tensor(1 + 0.1 * support.normal(seed, 10 + i, size, 1.0) if name.startswith("g") else support.normal(seed, 10 + i, size, 0.05), dtype, device)
         for i, (name, size) in enumerate(dl.weight_shapes(SHAPE).items())}
    return dl.pack_weights(w) if packed else w


class Model:
    def __init__(self, dtype, device, layers=2, packed=True):
        self.dtype, self.device = dtype, device
        self.kept = [parameters(dtype, device, 70 + i, packed) for i in range(layers)]
        self.w = [dl.quantize_weights(w) for w in self.kept]
        self.gain = ta.tensor(1 + 0.1 * support.normal(80, 1, (SHAPE.hidden,), 1.0), dtype, device)
        self.cos, self.sin = dl.rotary_tables(SHAPE, POSITIONS, dtype, device)
        self.cache = PagedCache(layers, 48, 16, SHAPE.kv_heads, SHAPE.head_dim, dtype, device)

    def step(self, ids, rows):
        step = self.cache.plan(ids, [len(r) for r in rows])
        x = ta.tensor(np.concatenate(rows)[None], self.dtype, self.device)
        out = dl.stack_paged_quantized(SHAPE, self.w, self.gain, x, self.cos, self.sin, self.cache, step)
        self.cache.advance(step)
        return out.numpy()[0]


def test_the_parameters(device):
    for packed in (True, False):
        kept = parameters(ta.bfloat16, device, 90, packed)
        w = dl.quantize_weights(kept)
        names = {"wqkv", "w13", "wo", "w2"} if packed else {"wq", "wk", "wv", "w1", "w3", "wo", "w2"}
        assert set(w) == names | {n + "_scales" for n in names} | {"g1", "g2"}
        for name in names:
            values, largest, _ = integers_of(kept[name].numpy())
            assert w[name].dtype is ta.int8 and w[name].shape == kept[name].shape
            np.testing.assert_array_equal(w[name].numpy(), values)
            np.testing.assert_array_equal(w[name + "_scales"].numpy(), largest / np.float32(127))


def product(trace_values, trace_scales, w, name):
    sums = trace_values.astype(np.float64) @ w[name].numpy().astype(np.float64).T
    return sums.astype(np.float32) * trace_scales[..., None] * w[name + "_scales"].numpy()


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float16, ta.float32], ids=str)
@pytest.mark.parametrize("packed", [True, False])
def test_every_stage_of_a_layer(dtype, packed, device):
    """Each stage from what the one before it left: sums, integers and products bit for bit, attention within its own bound."""
    rng = np.random.default_rng(71)
    m = Model(dtype, device, layers=1, packed=packed)
    w = m.w[0]
    a, b = m.cache.add(), m.cache.add()
    for new in ([37, 5], [1, 1], [1, 33]):
        step = m.cache.plan([a, b], new)
        tokens = sum(new)
        x, more = (rounded(rng.standard_normal((1, tokens, SHAPE.hidden)), dtype) for _ in range(2))
        trace = {}
        h, y = dl.forward_paged_quantized(SHAPE, w, ta.tensor(x, dtype, device), ta.tensor(more, dtype, device), m.cos, m.sin, m.cache, 0, step, trace)
        assert h is trace["h"] and y is trace["y"] and y.dtype is dtype
        t = {name: value.numpy() for name, value in trace.items()}
        np.testing.assert_array_equal(t["x"], rounded(x + more, dtype))
        np.testing.assert_array_equal(t["xn"], integers_of(t["x"].astype(np.float32) * w["g1"].numpy().astype(np.float32))[0])
        qkv = product(t["xn"], t["xn_scales"], w, "wqkv") if packed else np.concatenate([product(t["xn"], t["xn_scales"], w, n) for n in ("wq", "wk", "wv")], -1)
        np.testing.assert_array_equal(np.concatenate([t[n].reshape(tokens, -1) for n in "qkv"], -1), rounded(qkv[0], dtype))
        lengths, first = [m.cache.length(s) for s in (a, b)], 0
        keys, values = m.cache.keys(0).numpy().astype(np.float64), m.cache.values(0).numpy().astype(np.float64)
        for s, n, have in zip((a, b), new, lengths):
            at = [(m.cache.pages_of(s)[j // 16], j % 16) for j in range(have + n)]
            for head in (0, 7):
                mine_k, mine_v = (np.stack([pool[page, head // 4, row] for page, row in at]) for pool in (keys, values))
                want, slack, size = head_attention(t["q_rot"][first:first + n, head].astype(np.float64), mine_k, mine_v, float(np.float32(0.125)), have + 1 + np.arange(n))
                assert_within(t["o"][first:first + n, head].astype(np.float64), want, slack, size, dtype, np.abs(mine_v).sum(0))
            first += n
        o8, largest, _ = integers_of(t["o"].reshape(1, tokens, -1))
        np.testing.assert_array_equal(t["o8"], o8)
        np.testing.assert_array_equal(t["o_scales"], largest / np.float32(127))
        np.testing.assert_array_equal(t["attended"], rounded(product(t["o8"], t["o_scales"], w, "wo"), dtype))
        np.testing.assert_array_equal(t["h"], rounded(t["attended"].astype(np.float32) + t["x"].astype(np.float32), dtype))
        np.testing.assert_array_equal(t["hn"], integers_of(t["h"].astype(np.float32) * w["g2"].numpy().astype(np.float32))[0])
        both = product(t["hn"], t["hn_scales"], w, "w13") if packed else np.concatenate([product(t["hn"], t["hn_scales"], w, n) for n in ("w1", "w3")], -1)
        np.testing.assert_array_equal(np.concatenate([t["gate"], t["up"]], -1), rounded(both, dtype))
        gate, up = t["gate"].astype(np.float64), t["up"].astype(np.float64)
        act = gate / (1 + np.exp(-gate)) * up
        # (half a step, and what u and the scale are off by: 20 units of 2^-24 of the row's largest, see test_swiglu)
        assert (np.abs(t["act"] * t["act_scales"].astype(np.float64)[..., None] - act) <= 0.5 * t["act_scales"][..., None] + 20 * 2.0 ** -24 * np.abs(act).max(-1, keepdims=True)).all()
        np.testing.assert_array_equal(t["y"], rounded(product(t["act"], t["act_scales"], w, "w2"), dtype))
        m.cache.advance(step)


def test_chunks_and_tokens_give_what_the_whole_prompt_gives(device):
    """Rows are quantised, multiplied and normed by themselves: the first token of a prompt is the same bits in any company of rows (its attention sees itself only, whose weight is 1)."""
    rng = np.random.default_rng(72)
    m = Model(ta.float32, device)
    x = rng.standard_normal((40, SHAPE.hidden))
    alone = m.step([m.cache.add()], [x[:1]])
    for n in (2, 20, 40):
        np.testing.assert_array_equal(m.step([m.cache.add()], [x[:n]])[:1], alone)
    others = [m.cache.add() for _ in range(3)]
    np.testing.assert_array_equal(m.step(others, [x[5:9], x[:1], x[7:8]])[4:5], alone)


def test_a_recorded_step_follows_the_tables(device):
    """Replays with the program's own work between them give the eager steps' bits."""
    rng = np.random.default_rng(73)
    m, other = Model(ta.bfloat16, device), Model(ta.bfloat16, device)
    rows = [rng.standard_normal((n, SHAPE.hidden)) for n in (20, 30)]
    ids, others = [m.cache.add(), m.cache.add()], [other.cache.add(), other.cache.add()]
    m.step(ids, rows), other.step(others, rows)
    step = m.cache.plan(ids, [1, 1], columns=6)
    held = ta.tensor(np.zeros((1, 2, SHAPE.hidden)), ta.bfloat16, device)
    with ta.Graph(device) as g:
        out = dl.stack_paged_quantized(SHAPE, m.w, m.gain, held, m.cos, m.sin, m.cache, step)
    for token in range(12):
        row = rng.standard_normal((2, SHAPE.hidden))
        m.cache.plan(ids, [1, 1], into=step)
        ops.copy_into(held, ta.tensor(row[None], ta.bfloat16, device))
        g.launch()
        m.cache.advance(step)
        np.testing.assert_array_equal(out.numpy()[0], other.step(others, [row[:1], row[1:]]), err_msg=f"token {token}")


# M, N, K of products whose blocks share K: joined by the last block, and by a second kernel
SHARED = [(40, 128, 8192), (20, 64, 8192), (128, 384, 8192), (128, 4096, 14336)]


def test_two_recordings_and_eager_calls_of_products_that_share_k(device):
    """Two recordings made on one stream, replayed in turn with eager products between: each gives its own results every time."""
    rng = np.random.default_rng(74)
    made = []
    for m, n, k in SHARED:
        a, b = (rng.integers(-127, 128, s) for s in ((m, k), (n, k)))
        sa, sb = rng.uniform(0.001, 0.002, m).astype(np.float32), rng.uniform(0.005, 0.02, n).astype(np.float32)
        operands = [ta.tensor(a, ta.int8, device), ta.tensor(sa, ta.float32, device), ta.tensor(b, ta.int8, device).transpose(), ta.tensor(sb, ta.float32, device)]
        made.append((operands, ops.matmul_quantized(*operands, ta.bfloat16).storage()))
    with ta.Graph(device) as first:
        ones = [ops.matmul_quantized(*operands, ta.bfloat16) for operands, _ in made]
    with ta.Graph(device) as second:
        twos = [ops.matmul_quantized(*operands, ta.bfloat16) for operands, _ in reversed(made)]
    for _ in range(4):
        first.launch()
        second.launch()
        for operands, want in made:
            np.testing.assert_array_equal(ops.matmul_quantized(*operands, ta.bfloat16).storage(), want)
        second.launch()
        first.launch()
        for got, (_, want) in zip(ones, made):
            np.testing.assert_array_equal(got.storage(), want)
        for got, (_, want) in zip(twos, reversed(made)):
            np.testing.assert_array_equal(got.storage(), want)


def test_two_streams_at_once(device):
    """Products that share K on two streams: parts and counts are a stream's own.  (What is compared with comes first: a copy to the host is ordered with the stream of the pool.)"""
    import ctypes as C
    rng = np.random.default_rng(75)
    lib = ta.library()
    made = []
    for m, n, k in SHARED[:3]:
        a, b = (rng.integers(-127, 128, s) for s in ((m, k), (n, k)))
        operands = [ta.tensor(a, ta.int8, device), ta.tensor(np.full(m, 0.001), ta.float32, device), ta.tensor(b, ta.int8, device).transpose(), ta.tensor(np.full(n, 0.01), ta.float32, device)]
        made.append((operands, [[ta.Tensor(ta.bfloat16, (m, n)).initialize(device) for _ in range(8)] for _ in range(2)], ops.matmul_quantized(*operands, ta.bfloat16).storage()))
    lib.device_synchronize()
    dvc = device.structure()
    streams = [lib.pop_stream(C.byref(dvc)) for _ in range(2)]
    try:
        for operands, results, _ in made:
            for i in range(8):
                for stream, into in zip(streams, results):
                    assert lib.kernels["gemm_quantized"](*(C.byref(t.descriptor()) for t in (*operands, into[i])), stream) == 0
        for stream in streams:
            assert lib.stream_synchronize(stream) == 0
    finally:
        for stream in reversed(streams):      # (the pool hands out the last one: the device's has to be it again)
            lib.put_stream(C.byref(dvc), stream)
    for _, results, want in made:
        for into in results:
            for t in into:
                np.testing.assert_array_equal(t.storage(), want)


def test_two_threads(device):
    rng = np.random.default_rng(76)
    x = rounded(rng.standard_normal((30, 500)), ta.float32)
    w = ta.tensor(rng.integers(-127, 128, (90, 500)), ta.int8, device).transpose()
    sw = ta.tensor(np.full(90, 0.01), ta.float32, device)
    d = ta.tensor(x, ta.float32, device)
    want = ops.matmul_quantized(*ops.quantize(d), w, sw, ta.float32).numpy()
    results = [[], []]

    def work(mine):
        for _ in range(30):
            mine.append(ops.matmul_quantized(*ops.quantize(d), w, sw, ta.float32))

    threads = [threading.Thread(target=work, args=(mine,)) for mine in results]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    # (read by one thread: copies to the host take streams from the pool, which hands two threads two of them)
    for mine in results:
        assert len(mine) == 30
        for got in mine:
            np.testing.assert_array_equal(got.numpy(), want)


def test_results_that_share_an_allocation(device):
    """values, scales and a small sum lie in one buffer, which lives as long as one of them does."""
    rng = np.random.default_rng(77)
    x, residual = (rounded(rng.standard_normal((7, 300)), ta.float16) for _ in range(2))
    gain = ta.tensor(np.ones(300), ta.float16, device)
    values, scales, total = ops.add_rms_norm_quantized(ta.tensor(x, ta.float16, device), ta.tensor(residual, ta.float16, device), gain)
    assert values.buffer is scales.buffer and values.buffer is total.buffer
    want = [t.numpy() for t in (values, scales, total)]
    del values, total
    for _ in range(20):      # (memory that would be given out again)
        ops.quantize(ta.tensor(rng.standard_normal((7, 300)), ta.float16, device))
    np.testing.assert_array_equal(scales.numpy(), want[1])
    np.testing.assert_array_equal(want[0], integers_of(rounded(x + residual, ta.float16))[0])
    # a large sum has memory of its own
    big = ta.tensor(np.ones((600, 1000)), ta.float16, device)
    values, scales, total = ops.add_rms_norm_quantized(big, big, ta.tensor(np.ones(1000), ta.float16, device))
    assert values.buffer is scales.buffer and values.buffer is not total.buffer
    for normed, total in (ops.add_rms_norm(big, big, ta.tensor(np.ones(1000), ta.float16, device)), ops.add_rms_norm(big[0:3], big[0:3], ta.tensor(np.ones(1000), ta.float16, device))):
        np.testing.assert_array_equal(total.numpy(), 2.0)
        assert (np.abs(normed.numpy() - 1.0) <= HALF[ta.float16] + 2.0 ** -16 + TINY[ta.float16]).all()
