"""Attention over a paged cache and over dense states of another length, against the definition in 64 bits."""
import ctypes as C
import threading

import numpy as np
import pytest

import tannic_amd as ta
from attention_support import Cache, assert_within, head_attention, rounded
from tannic_amd import abi, ops

pytestmark = pytest.mark.gpu

TYPES = [ta.float16, ta.bfloat16, ta.float32, ta.float64]


def check(c, device, scale=None, q=None):
    scale = 1.0 / np.sqrt(c.d) if scale is None else scale
    q = ta.tensor(c.q, c.dtype, device) if q is None else q
    got = ops.attend_pages(q, c.keys, c.values, c.table, c.starts, c.lengths, scale).numpy()
    want, slack, size, total = c.expected(np.float32(scale).astype(np.float64))
    assert_within(got, want, slack, size, c.dtype, total)
    return got


# heads, kv heads, head size
HEADS = [(4, 1, 64), (8, 2, 128), (5, 5, 40), (32, 2, 16), (6, 2, 256), (3, 1, 80), (8, 8, 96), (4, 2, 8), (2, 2, 200)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_single_tokens(heads, dtype, device):
    """One token of every sequence, contexts around the sizes where tiles, wavefronts and shares of blocks end."""
    rng = np.random.default_rng(1)
    context = [0, 1, 14, 15, 16, 30, 31, 32, 33, 62, 63, 64, 65, 127, 128, 255, 300]
    check(Cache(rng, dtype, device, *heads, 16, [1] * len(context), context), device)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("page", [1, 3, 16, 20, 64, 100])
def test_pages_of_any_size(page, dtype, device):
    rng = np.random.default_rng(2)
    check(Cache(rng, dtype, device, 4, 2, 64, page, [1, 1, 7, 40], [77, 200, 130, 0]), device)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads", [(4, 1, 64), (4, 4, 128), (2, 1, 256), (3, 3, 40), (12, 2, 32)], ids=str)
@pytest.mark.parametrize("new,context", [([2, 3, 5], [9, 0, 60]), ([33, 1, 16, 0, 64], [31, 100, 0, 5, 65]), ([130], [70]), ([65, 127], [1, 129])], ids=str)
def test_chunks(new, context, heads, dtype, device):
    """Chunks of several tokens behind what is there, single tokens and sequences without new ones among them."""
    rng = np.random.default_rng(3)
    check(Cache(rng, dtype, device, *heads, 16, new, context), device)


@pytest.mark.parametrize("dtype", [ta.float16, ta.bfloat16, ta.float32], ids=str)
@pytest.mark.parametrize("new,context,heads", [([1], [5000], (8, 2, 128)), ([1, 1], [2047, 4100], (16, 2, 64)), ([3], [3001], (4, 1, 128)), ([300], [1700], (2, 1, 128)), ([257], [0], (4, 2, 64))], ids=str)
def test_long_contexts(new, context, heads, dtype, device):
    rng = np.random.default_rng(4)
    check(Cache(rng, dtype, device, *heads, 16, new, context), device)


@pytest.mark.parametrize("dtype", [ta.float16, ta.bfloat16, ta.float32], ids=str)
@pytest.mark.parametrize("d,slip", [(7, 0), (33, 0), (64, 1), (128, 3)])
def test_head_sizes_and_starts_that_no_vector_fits(d, slip, dtype, device):
    """Odd head sizes, and queries whose rows start anywhere: columns of a wider tensor."""
    rng = np.random.default_rng(5)
    c = Cache(rng, dtype, device, 4, 2, d, 5, [1, 6], [20, 33])
    wide = np.full((c.q.shape[0], 4, d + slip + 2), np.inf)
    wide[:, :, slip:slip + d] = c.q
    check(c, device, q=ta.tensor(wide, dtype, device)[:, :, slip:slip + d])


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float32], ids=str)
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 70]], ids=str)
def test_other_layouts(new, dtype, device):
    """Tokens before heads in the pages, and queries that are columns of one projection's result."""
    rng = np.random.default_rng(6)
    c = Cache(rng, dtype, device, 4, 2, 64, 16, new, [100, 17, 3], token_major=True)
    qkv = np.full((sum(new), 8, 64), np.nan)
    qkv[:, 2:6] = c.q
    check(c, device, q=ta.tensor(qkv, dtype, device)[:, 2:6])


@pytest.mark.parametrize("dtype", [ta.float16, ta.bfloat16, ta.float32], ids=str)
@pytest.mark.parametrize("new", [[1, 1, 1], [9, 70, 2]], ids=str)
def test_pages_that_do_not_exist(new, dtype, device):
    """Keys of missing pages are left out; a sequence that has none at all gives zeros."""
    rng = np.random.default_rng(7)
    c = Cache(rng, dtype, device, 4, 2, 64, 16, new, [100, 64, 10])
    missing = [(0, 0), (0, 3), (1, 2)] + [(2, i) for i in range(c.host_table.shape[1])]
    for s, column in missing:
        c.host_table[s, column] = [-1, 1 << 30][column % 2]
    got = ops.attend_pages(ta.tensor(c.q, dtype, device), c.keys, c.values, ta.tensor(c.host_table, ta.int32, device), c.starts, c.lengths).numpy()
    want, slack, size, total = c.expected(0.125, missing)
    assert_within(got, want, slack, size, dtype, total)
    assert (got[sum(new[:2]):] == 0).all()


@pytest.mark.parametrize("dtype", [ta.float16, ta.bfloat16, ta.float32], ids=str)
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_scales(scale, dtype, device):
    rng = np.random.default_rng(8)
    check(Cache(rng, dtype, device, 4, 2, 64, 16, [1, 50], [200, 60]), device, scale)


def call(name, operands, device, extra=()):
    lib = ta.library()
    descriptors = [None if t is None else C.byref(t.descriptor()) for t in operands]
    status = lib.kernels[name](*descriptors, device.stream(), *extra)
    return status, lib.error_message()


@pytest.mark.parametrize("dtype", [ta.float16, ta.float32], ids=str)
@pytest.mark.parametrize("most", [1, 60])
def test_rows_of_no_sequence_stay_as_they_were(most, dtype, device):
    """A padded batch: rows in front of the first sequence and behind the last, and lengths no batch can have."""
    rng = np.random.default_rng(9)
    new = [most, 1, 0]
    c = Cache(rng, dtype, device, 4, 2, 64, 16, new, [33, 40, 8])
    n = sum(new)
    q = np.full((n + 7, 4, 64), np.nan)
    q[2:2 + n] = c.q
    starts = ta.tensor(np.array([2, 2 + most, 2 + n, 2 + n]), ta.int32, device)
    out = ta.tensor(np.full((n + 7, 4, 64), 7.0), dtype, device)
    status, message = call("attend_pages", [ta.tensor(q, dtype, device), c.keys, c.values, c.table, starts, c.lengths, out], device, (0.125,))
    assert status == abi.SUCCESS, message
    got = out.numpy()
    want, slack, size, total = c.expected(0.125)
    assert_within(got[2:2 + n], want, slack, size, dtype, total)
    assert (got[:2] == 7).all() and (got[2 + n:] == 7).all()
    # whatever the lengths hold, nothing outside the tensors is touched
    for bad in ([-5, 2, 1 << 30, -1], [(1 << 31) - 1] * 4, [-(1 << 31)] * 4, [5, 4, 3, 2]):
        for context in ([-3, (1 << 31) - 1, 7], [1 << 30, 0, -(1 << 31)]):
            status, message = call("attend_pages", [ta.tensor(q, dtype, device), c.keys, c.values, c.table, ta.tensor(np.array(bad), ta.int32, device),
                                                    ta.tensor(np.array(context), ta.int32, device), out], device, (0.125,))
            assert status == abi.SUCCESS, message
    ta.library().device_synchronize()


@pytest.mark.parametrize("dtype", [ta.float16, ta.bfloat16, ta.float32], ids=str)
@pytest.mark.parametrize("new", [[1, 1], [37, 80]], ids=str)
def test_what_later_tokens_hold_does_not_reach_earlier_ones(new, dtype, device):
    """Keys and values behind a token's position are infinite or NaN: the token before them gives the same bits as without them."""
    rng = np.random.default_rng(10)
    c = Cache(rng, dtype, device, 4, 2, 64, 16, new, [60, 20])
    q = ta.tensor(c.q, dtype, device)
    want = ops.attend_pages(q, c.keys, c.values, c.table, c.starts, c.lengths).numpy()
    keys, values = c.keys.numpy().copy(), c.values.numpy().copy()
    for s in range(2):
        j = c.new[s] + c.context[s] - 1      # the last token's key and value
        keys[c.host_table[s, j // 16], :, j % 16], values[c.host_table[s, j // 16], :, j % 16] = np.nan, [np.inf, np.nan][s]
    got = ops.attend_pages(q, ta.tensor(keys, dtype, device), ta.tensor(values, dtype, device), c.table, c.starts, c.lengths).numpy()
    ends = np.cumsum(new)
    rows = np.setdiff1d(np.arange(sum(new)), ends - 1)
    np.testing.assert_array_equal(got[rows], want[rows])
    assert not np.isfinite(got[ends - 1]).any()


@pytest.mark.parametrize("dtype", [ta.float16, ta.bfloat16, ta.float32], ids=str)
def test_scores_that_differ_by_much(dtype, device):
    """Scores of some hundreds apart: the largest decides, whatever order the keys are met in; scores of -inf weigh nothing."""
    rng = np.random.default_rng(11)
    c = Cache(rng, dtype, device, 2, 1, 64, 16, [1, 40], [500, 300])
    c.q = rounded(c.q * 16, dtype)
    check(c, device, 1.0)
    check(c, device, -1.0)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads", [(4, 4, 64), (8, 2, 128), (3, 1, 80), (4, 2, 256), (5, 5, 33)], ids=str)
@pytest.mark.parametrize("tokens,states", [(1, 130), (5, 77), (70, 200), (130, 64), (33, 1)])
def test_other_lengths(tokens, states, heads, dtype, device):
    """Queries over states of another length, as many of them as the sequence has: none, one, some, all; the padding is NaN."""
    h, kv, d = heads
    rng = np.random.default_rng(12)
    lengths = np.array([states, 0, 1, (states + 1) // 2])
    q = rounded(rng.standard_normal((4, tokens, h, d)), dtype)
    k, v = (rounded(rng.standard_normal((4, states, kv, d)), dtype) for _ in range(2))
    scale = float(np.float32(1.0 / np.sqrt(d)))
    want, slack, size, total = (np.zeros(q.shape) for _ in range(4))
    for b in range(4):
        for i in range(h):
            kb, vb = k[b, :, i * kv // h], v[b, :, i * kv // h]
            want[b, :, i], slack[b, :, i], size[b, :, i] = head_attention(q[b, :, i], kb, vb, scale, [lengths[b]] * tokens)
            total[b, :, i] = np.abs(vb).sum(0)
        k[b, lengths[b]:], v[b, lengths[b]:] = np.nan, np.nan
    got = ops.attend(*(ta.tensor(x, dtype, device) for x in (q, k, v)), ta.tensor(lengths, ta.int32, device)).numpy()
    assert_within(got, want, slack, size, dtype, total)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("dtype", [ta.float16, ta.float32], ids=str)
@pytest.mark.parametrize("tokens", [1, 50])
def test_other_lengths_in_other_layouts(tokens, dtype, device):
    """Heads before tokens, seen through a transposed view, keys and values as columns of one product, lengths not given."""
    rng = np.random.default_rng(13)
    q = rounded(rng.standard_normal((2, 4, tokens, 64)), dtype)
    kv = rounded(rng.standard_normal((2, 90, 2, 2, 64)), dtype)
    got = ops.attend(ta.tensor(q, dtype, device).transpose(1, 2), *(ta.tensor(kv, dtype, device)[:, :, i] for i in (0, 1)), None, 0.125).numpy()
    for b in range(2):
        for h in range(4):
            want, slack, size = head_attention(q[b, h], kv[b, :, 0, h // 2], kv[b, :, 1, h // 2], 0.125, [90] * tokens)
            assert_within(got[b, :, h], want, slack, size, dtype, np.abs(kv[b, :, 1, h // 2]).sum(0))


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float32], ids=str)
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 9]], ids=str)
def test_a_recorded_call_follows_the_lengths(new, dtype, device):
    """Replays with other queries, lengths and pages in the same tensors, two recordings in turn, eager work in between."""
    rng = np.random.default_rng(14)
    first, second = (Cache(rng, dtype, device, 8, 2, 64, 16, new, context, room=64, width=24) for context in ([300, 0, 17], [5, 299, 64]))
    q = [ta.tensor(c.q, dtype, device) for c in (first, second)]
    want = [ops.attend_pages(x, c.keys, c.values, c.table, c.starts, c.lengths).storage() for x, c in zip(q, (first, second))]
    recorded = []
    for _ in range(2):
        held = [ta.Tensor(t.dtype, t.shape).initialize(device) for t in (q[0], first.keys, first.values, first.table, first.starts, first.lengths)]
        for t, x in zip(held, (q[0], first.keys, first.values, first.table, first.starts, first.lengths)):
            ops.copy_into(t, x)
        with ta.Graph(device) as g:
            out = ops.attend_pages(*held)
        recorded.append((g, held, out))
    for turn in range(3):
        for g, held, out in recorded:
            for x, c, w in zip(q, (first, second), want):
                for t, y in zip(held, (x, c.keys, c.values, c.table, c.starts, c.lengths)):
                    ops.copy_into(t, y)
                g.launch()
                ops.attend_pages(q[0], first.keys, first.values, first.table, first.starts, first.lengths)
                np.testing.assert_array_equal(out.storage(), w)


def test_offsets_past_32_bits(device):
    """A cache of more than 2^32 bytes and 2^31 elements: the pages a sequence uses lie at both ends."""
    pages, kv, page, d = 9000, 8, 256, 128
    keys = ta.Tensor(ta.float16, (pages, kv, page, d)).initialize(device)
    rng = np.random.default_rng(15)
    ids = [pages - 1, 0, pages - 2, 8300]
    k, v = (rounded(rng.standard_normal((4 * page, kv, d)), ta.float16) for _ in range(2))
    values = ta.Tensor(ta.float16, (pages, kv, page, d)).initialize(device)
    assert keys.nelements > 1 << 31
    for i, at in enumerate(ids):
        for pool, x in ((keys, k), (values, v)):
            ops.copy_into(pool[at:at + 1], ta.tensor(x[i * page:(i + 1) * page].transpose(1, 0, 2)[None], ta.float16, device))
    for n in (1, 70):
        q = rounded(rng.standard_normal((n, 16, d)), ta.float16)
        got = ops.attend_pages(ta.tensor(q, ta.float16, device), keys, values, ta.tensor(np.array([ids]), ta.int32, device), ta.tensor(np.array([0, n]), ta.int32, device),
                               ta.tensor(np.array([1000 - n]), ta.int32, device)).numpy()
        for h in (0, 15):
            want, slack, size = head_attention(q[:, h], k[:, h // 2], v[:, h // 2], float(np.float32(1 / np.sqrt(d))), 1001 - n + np.arange(n))
            assert_within(got[:, h], want, slack, size, ta.float16, np.abs(v[:, h // 2]).sum(0))


@pytest.mark.parametrize("dtype", [ta.float16, ta.bfloat16, ta.float32], ids=str)
@pytest.mark.parametrize("new,context,heads", [([8], [2200], (4, 1, 64)), ([5], [5000], (4, 1, 128)), ([9], [33500], (4, 1, 64)), ([4, 30], [3000, 1500], (6, 1, 256))], ids=str)
def test_few_rows_over_many_parts(new, context, heads, dtype, device):
    """A few rows of one group over keys that many blocks share, so that parts are put together more than once."""
    rng = np.random.default_rng(hash((tuple(new), heads)) & 0xFFFF)
    check(Cache(rng, dtype, device, *heads, 16, new, context), device)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens", [1, 40, 200])
def test_one_state_that_is_not_finite(tokens, dtype, device):
    """Nothing stands behind a single key: its value is the result, the infinite one too."""
    rng = np.random.default_rng(tokens)
    k, v = rounded(rng.standard_normal((2, 2, 1, 3, 64)), dtype)
    q = rounded(rng.standard_normal((2, tokens, 6, 64)), dtype)
    v[0, 0, 1, 5], v[1, 0, 2, 60], v[1, 0, 0, 8] = np.inf, -np.inf, np.nan
    got = ops.attend(*(ta.tensor(x, dtype, device) for x in (q, k, v)), None, 0.125).numpy()
    want = np.broadcast_to(np.repeat(v, 2, axis=2), q.shape)
    assert np.array_equal(np.asarray(got, np.float64), want, equal_nan=True)


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float32], ids=str)
def test_sequences_that_overlap_leave_nothing_behind(dtype, device):
    """Starts that descend are against what they may hold: no row outside q is written, and the next call's results are right."""
    rng = np.random.default_rng(17)
    c = Cache(rng, dtype, device, 4, 1, 64, 16, [1300], [700])
    n = 16
    table = ta.tensor(np.repeat(c.host_table, n, axis=0), ta.int32, device)
    starts = ta.tensor(np.array([0, 1300] * (n // 2) + [0]), ta.int32, device)
    q = ta.tensor(c.q, dtype, device)
    ops.attend_pages(q, c.keys, c.values, table, starts, ta.tensor(np.full(n, 700), ta.int32, device), 0.125)
    check(c, device)
    check(Cache(rng, dtype, device, 4, 1, 64, 16, [30], [2500]), device)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens", [1, 40])
def test_no_states_at_all(tokens, dtype, device):
    q = ta.tensor(np.ones((2, tokens, 4, 64)), dtype, device)
    empty = ta.Tensor(dtype, (2, 0, 2, 64)).initialize(device)
    assert (ops.attend(q, empty, empty).numpy() == 0).all()


def test_calls_of_two_threads(device):
    """Each thread's calls share keys between blocks, on whatever streams they get: no counts and no partial results are mixed up."""
    rng = np.random.default_rng(18)
    shapes = [((8, 2, 128), [1, 1], [3000, 1700]), ((4, 1, 64), [30], [4000])]
    caches = [Cache(rng, ta.bfloat16, device, *heads, 16, new, context) for heads, new, context in shapes]
    q = [ta.tensor(c.q, ta.bfloat16, device) for c in caches]
    want = [ops.attend_pages(x, c.keys, c.values, c.table, c.starts, c.lengths, 0.1).storage() for x, c in zip(q, caches)]
    results = [[], []]

    def work(i):
        c = caches[i]
        for _ in range(40):
            results[i].append(ops.attend_pages(q[i], c.keys, c.values, c.table, c.starts, c.lengths, 0.1))

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    ta.library().device_synchronize()
    for w, got in zip(want, results):
        assert len(got) == 40
        for g in got:
            np.testing.assert_array_equal(g.storage(), w)


@pytest.mark.parametrize("dtype", [ta.float16, ta.bfloat16], ids=str)
@pytest.mark.parametrize("page,d", [(7, 64), (20, 128), (33, 256), (24, 64)])
def test_chunks_over_pages_that_end_inside_a_step(page, d, dtype, device):
    """What later tokens hold is infinite or NaN, pages are missing in the middle, and one of them ends with the last key."""
    rng = np.random.default_rng(page)
    context, n = 2 * page + 150, 3 * page - 2 * page % 5 + 40
    c = Cache(rng, dtype, device, 6, 1, d, page, [n], [context])
    keys, values = c.keys.numpy(), c.values.numpy()
    for j, bad in ((context + n - 1, np.inf), (context + n - 2, np.nan), (context + n // 2, -np.inf)):
        values[c.host_table[0, j // page], 0, j % page, 3] = bad
        c.v[0][j, 0, 3] = bad
    c.table = ta.tensor(np.where(np.arange(c.host_table.shape[1]) == 1, -1, c.host_table), ta.int32, device)
    got = ops.attend_pages(ta.tensor(c.q, dtype, device), ta.tensor(keys, dtype, device), ta.tensor(values, dtype, device), c.table, c.starts, c.lengths, 0.125).numpy()
    with np.errstate(all="ignore"):
        want, slack, size, total = c.expected(0.125, missing=[(0, 1)])
    first = n // 2      # the first row that sees one of them; column 3 is no number, or infinite, from there on
    assert np.isneginf(got[first:n - 2, :, 3]).all() and np.isnan(got[n - 2:, :, 3]).all()
    total[...] = np.abs(np.where(np.isfinite(c.v[0]), c.v[0], 0)).sum(0)
    keep = np.ones(got.shape, bool)
    keep[first:, :, 3] = False
    for x in (got, want, slack, size):
        x[~keep] = 0
    assert_within(got, want, slack, size, dtype, total)


@pytest.mark.parametrize("dtype", [ta.float16, ta.bfloat16], ids=str)
@pytest.mark.parametrize("heads", [(48, 8, 64), (34, 2, 256)], ids=str)
def test_a_long_sequence_among_many(heads, dtype, device):
    """More groups than blocks run at a time, and one sequence that is much longer than a block's share of all keys."""
    rng = np.random.default_rng(19)
    n = 600 // heads[1] if heads[1] == 8 else 140
    context = rng.integers(0, 40, n)
    context[n // 3], context[n - 1] = 4000, 1500
    check(Cache(rng, dtype, device, *heads, 16, [3] * n, context.tolist()), device)


@pytest.mark.parametrize("dtype", [ta.float16, ta.float32, ta.float64], ids=str)
@pytest.mark.parametrize("most", [1, 40])
@pytest.mark.parametrize("n", [64, 65, 130, 300])
def test_many_sequences(n, most, dtype, device):
    """More sequences than a wavefront has lanes, some without new tokens."""
    rng = np.random.default_rng(n)
    new = rng.integers(0, most + 1, n) if most == 1 else np.where(rng.random(n) < 0.1, rng.integers(20, most, n), rng.integers(0, 3, n))
    check(Cache(rng, dtype, device, 8, 1, 16, 16, new.tolist(), rng.integers(0, 70, n).tolist()), device)


def test_more_sequences_than_lanes_squared(device):
    """Each lane looks after more than 64 sequences."""
    rng = np.random.default_rng(20)
    n = 64 * 65 + 3
    for new in (rng.integers(0, 2, n), np.where(np.arange(n) % 50 == 7, 30, 0)):
        check(Cache(rng, ta.bfloat16, device, 32, 1, 16, 16, new.tolist(), rng.integers(0, 5, n).tolist()), device)
