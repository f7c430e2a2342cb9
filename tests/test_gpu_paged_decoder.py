"""The operators of a serving program together: prompts in chunks and single tokens of several sequences over a paged cache, forks, a compaction, a
recorded step, and the attention to an encoder's states behind it."""
import subprocess
import sys
import os

import numpy as np
import pytest

import support
import tannic_amd as ta
from attention_support import HALF, assert_within, head_attention
from tannic_amd import decoder_layer as dl, ops
from tannic_amd.paged_cache import PagedCache

pytestmark = pytest.mark.gpu

SHAPE = dl.LayerShape(hidden=256, heads=8, kv_heads=2, head_dim=64, ffn=512)
POSITIONS = 256


def weights(dtype, device, seed, shapes):
    return {name: ta.tensor(np.ones(size) if name.startswith("g") else support.normal(seed, 10 + i, size, 0.05), dtype, device) for i, (name, size) in enumerate(shapes.items())}


class Model:
    def __init__(self, dtype, device, layers=2, packed=True, pages=64, page=16):
        self.dtype, self.device = dtype, device
        w = [weights(dtype, device, 40 + i, dl.weight_shapes(SHAPE)) for i in range(layers)]
        self.w = [dl.pack_weights(x) for x in w] if packed else w
        self.cos, self.sin = dl.rotary_tables(SHAPE, POSITIONS, dtype, device)
        self.cache = PagedCache(layers, pages, page, SHAPE.kv_heads, SHAPE.head_dim, dtype, device)

    def step(self, ids, rows, check=False, step=None):
        """One step of the sequences with their rows of x; what every layer gives, as float64."""
        step = self.cache.plan(ids, [len(r) for r in rows]) if step is None else step
        x = ta.tensor(np.concatenate(rows)[None], self.dtype, self.device)
        for layer, w in enumerate(self.w):
            trace = {}
            x = dl.forward_paged(SHAPE, w, x, self.cos, self.sin, self.cache, layer, step, trace)
            if check:
                self.check(layer, step, trace)
        self.cache.advance(step)
        return np.split(x.numpy()[0], np.cumsum(step.new)[:-1])

    def check(self, layer, step, trace):
        """The new keys are the rotated ones, and every row attends to what its sequence's pages hold."""
        with np.errstate(invalid="ignore"):      # (what no token wrote)
            keys, values = self.cache.keys(layer).numpy().astype(np.float64), self.cache.values(layer).numpy().astype(np.float64)
        cos, sin = self.cos.numpy().astype(np.float64), self.sin.numpy().astype(np.float64)
        got, q, k, v = (trace[n].numpy().astype(np.float64) for n in ("o", "q_rot", "k", "v"))
        first = 0
        for i, (s, n) in enumerate(zip(step.ids, step.new)):
            have, page = self.cache.length(s), self.cache.page
            at = [(self.cache.pages_of(s)[j // page], j % page) for j in range(have + n)]
            mine_k, mine_v = (np.stack([pool[a, :, b] for a, b in at]) if at else np.zeros((0, 2, 64)) for pool in (keys, values))
            np.testing.assert_array_equal(mine_v[have:], v[first:first + n])
            c, sn, x = cos[have:have + n][:, None], sin[have:have + n][:, None], k[first:first + n]
            turned = np.empty_like(x)
            turned[..., 0::2], turned[..., 1::2] = x[..., 0::2] * c - x[..., 1::2] * sn, x[..., 0::2] * sn + x[..., 1::2] * c
            # (a rounding of the result, two units of fp32 of its two terms)
            assert (np.abs(mine_k[have:] - turned) <= HALF[self.dtype] * np.abs(turned) + 2.0 ** -22 * np.abs(x).max(initial=0.0) + 2.0 ** -25).all()
            for h in range(SHAPE.heads):
                kv = h // (SHAPE.heads // SHAPE.kv_heads)
                want, slack, size = head_attention(q[first:first + n, h], mine_k[:, kv], mine_v[:, kv], float(np.float32(0.125)), have + 1 + np.arange(n))
                assert_within(got[first:first + n, h], want, slack, size, self.dtype, np.abs(mine_v[:, kv]).sum(0), f"layer {layer} sequence {s} head {h}")
            first += n


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float16, ta.float32], ids=str)
@pytest.mark.parametrize("packed", [True, False])
def test_a_serving_run(dtype, packed, device):
    rng = np.random.default_rng(51)
    m = Model(dtype, device, packed=packed)
    rows = lambda n: rng.standard_normal((n, SHAPE.hidden))   # noqa: E731
    a, b = m.cache.add(), m.cache.add()
    m.step([a, b], [rows(37), rows(5)], True)              # two prompts
    m.step([a, b], [rows(1), rows(70)], True)              # one decodes, the other's next chunk
    c = m.cache.fork(a)
    m.step([c, a, b], [rows(1), rows(1), rows(1)], True)   # the fork writes its own copy of the page
    m.cache.free(b)
    assert m.cache.compact() > 0
    m.step([a, c], [rows(1), rows(3)], True)
    m.cache.truncate(c, 38)
    m.step([c, a], [rows(2), rows(0)], True)


@pytest.mark.parametrize("page", [16, 5])
def test_chunks_and_tokens_give_what_the_whole_prompt_gives(page, device):
    """fp32: the layer over the whole prompt at once (scores in memory) against chunks and single tokens over the cache.  Every value is a chain of eight products of at most 512
    terms in fp32: 512 units each of the sums of magnitudes, which here are below some 20 times the results: 8 * 512 * 20 * 2^-24 < 5e-3 of the largest."""
    rng = np.random.default_rng(52)
    m = Model(ta.float32, device, layers=1, page=page)
    x = rng.standard_normal((100, SHAPE.hidden))
    cos, sin = dl.rotary_tables(SHAPE, 100, ta.float32, device)
    want = dl.forward_fused(SHAPE, m.w[0], ta.tensor(x[None], ta.float32, device), cos, sin, dl.causal_mask(100, ta.float32, device)).numpy()[0]
    a = m.cache.add()
    got, at = [], 0
    for n in (33, 1, 1, 50, 1, 14):
        got.append(m.step([a], [x[at:at + n]])[0])
        at += n
    assert np.abs(np.concatenate(got) - want).max() <= 5e-3 * np.abs(want).max()
    # in the same pieces of another order of sequences: the same bits
    b, c = m.cache.add(), m.cache.add()
    first = m.step([b, c], [x[:33], x[:1]])[0]
    np.testing.assert_array_equal(first, got[0])


def test_a_recorded_step_follows_the_tables(device):
    rng = np.random.default_rng(53)
    m, other = Model(ta.bfloat16, device), Model(ta.bfloat16, device)
    x = [rng.standard_normal((n, SHAPE.hidden)) for n in (20, 30)]
    ids = [m.cache.add(), m.cache.add()]
    others = [other.cache.add(), other.cache.add()]
    m.step(ids, x), other.step(others, x)
    step = m.cache.plan(ids, [1, 1], columns=8)
    held = ta.tensor(np.zeros((1, 2, SHAPE.hidden)), ta.bfloat16, device)
    with ta.Graph(device) as g:
        y = held
        for layer, w in enumerate(m.w):
            y = dl.forward_paged(SHAPE, w, y, m.cos, m.sin, m.cache, layer, step)
    for token in range(15):      # (over the end of a page)
        row = rng.standard_normal((2, SHAPE.hidden))
        m.cache.plan(ids, [1, 1], into=step)
        ops.copy_into(held, ta.tensor(row[None], ta.bfloat16, device))
        g.launch()
        m.cache.advance(step)
        want = np.concatenate(other.step(others, [row[:1], row[1:]]))
        np.testing.assert_array_equal(y.numpy()[0], want, err_msg=f"token {token}")


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float32], ids=str)
@pytest.mark.parametrize("tokens", [1, 40])
def test_attention_to_an_encoder(dtype, tokens, device):
    rng = np.random.default_rng(54)
    w = weights(dtype, device, 60, dl.cross_weight_shapes(SHAPE))
    states = ta.tensor(rng.standard_normal((3, 90, SHAPE.hidden)), dtype, device)
    x = ta.tensor(rng.standard_normal((3, tokens, SHAPE.hidden)), dtype, device)
    lengths = np.array([90, 0, 33])
    k, v = dl.encoder_keys(SHAPE, w, states)
    out = dl.cross_attention(SHAPE, w, x, k, v, ta.tensor(lengths, ta.int32, device))
    assert out.shape == x.shape
    # a sequence without states keeps its rows
    np.testing.assert_array_equal(out.numpy()[1], x.numpy()[1])
    q = ops.matmul(ops.rms_norm(x, w["g3"], SHAPE.eps), w["cq"].transpose()).view(3, tokens, 8, 64)
    got = ops.attend(q, k, v, ta.tensor(lengths, ta.int32, device))
    qn, kn, vn, on = (t.numpy().astype(np.float64) for t in (q, k, v, got))
    for b in (0, 2):
        for h in range(8):
            want, slack, size = head_attention(qn[b, :, h], kn[b, :, h // 4], vn[b, :, h // 4], float(np.float32(0.125)), [lengths[b]] * tokens)
            assert_within(on[b, :, h], want, slack, size, dtype, np.abs(vn[b, :, h // 4]).sum(0))
    # the rest are operators that were there
    np.testing.assert_array_equal(out.storage(), ops.add(x, ops.matmul(got.view(3, tokens, 512), w["co"].transpose())).storage())


def test_a_first_call_that_is_recorded(tmp_path):
    """A process whose first attention is inside a recording: the library's counts of arrivals are there and 0 at every replay, and for eager calls after it."""
    program = tmp_path / "first.py"
    program.write_text('''
import sys
sys.path[:0] = [%r, %r]
import numpy as np
import tannic_amd as ta
from attention_support import Cache
from tannic_amd import ops
device = ta.Device(0)
rng = np.random.default_rng(55)
for heads, new in (((8, 2, 64), [1, 1]), ((4, 2, 128), [200])):
    c = Cache(rng, ta.bfloat16, device, *heads, 16, new, [3000] * len(new))
    q = ta.tensor(c.q, ta.bfloat16, device)
    with ta.Graph(device) as g:
        out = ops.attend_pages(q, c.keys, c.values, c.table, c.starts, c.lengths)
    g.launch()
    first = out.storage()
    for _ in range(3):
        eager = ops.attend_pages(q, c.keys, c.values, c.table, c.starts, c.lengths).storage()
        np.testing.assert_array_equal(eager, first)
        g.launch()
        np.testing.assert_array_equal(out.storage(), first)
    g.close()      # (destroying a recording waits for the stream, which the next one records)
print("the same")
''' % (os.path.dirname(os.path.dirname(os.path.abspath(__file__))), os.path.dirname(os.path.abspath(__file__))))
    done = subprocess.run([sys.executable, str(program)], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "the same" in done.stdout, done.stdout + done.stderr
