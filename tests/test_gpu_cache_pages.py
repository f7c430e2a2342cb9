"""Writing into a paged cache and copying its pages."""
import ctypes as C

import numpy as np
import pytest

import tannic_amd as ta
from attention_support import HALF, rounded
from tannic_amd import abi, ops

pytestmark = pytest.mark.gpu

TYPES = [ta.float16, ta.bfloat16, ta.float32, ta.float64]


def turned(x, cos, sin):
    """The pairs (2i, 2i+1) by the angles; and what fp32 products and their sum may be off by."""
    even, odd = x[..., 0::2], x[..., 1::2]
    out, size = np.empty_like(x), np.empty_like(x)
    out[..., 0::2], out[..., 1::2] = even * cos - odd * sin, even * sin + odd * cos
    size[..., 0::2], size[..., 1::2] = np.abs(even * cos) + np.abs(odd * sin), np.abs(even * sin) + np.abs(odd * cos)
    return out, size


def near(got, want, size, dtype, what):
    unit = 2.0 ** -53 if dtype is ta.float64 else 2.0 ** -24
    b = HALF[dtype] * np.abs(want) + 2 * unit * size * (1 + HALF[dtype]) + (2.0 ** -25 if dtype is ta.float16 else 0.0)
    assert (np.abs(got - want) <= b).all(), what


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads,kv,d,page", [(4, 2, 64, 16), (6, 1, 80, 7), (2, 2, 6, 1), (32, 8, 128, 16)])
@pytest.mark.parametrize("wide", [False, True])
def test_append_turns_and_writes(heads, kv, d, page, wide, dtype, device):
    """New tokens at, in front of and behind the ends of pages, sequences without new ones among them; everything else keeps its bits."""
    rng = np.random.default_rng(21)
    new, context = [1, 0, 17, 2, 1], [page - 1, 5, 0, 3 * page, 2 * page + 1]
    have = [-(-(a + b) // page) for a, b in zip(new, context)]
    room = sum(have) + 2
    table = np.full((5, max(have) + 1), -1)
    order, at = rng.permutation(room), 0
    for s, n in enumerate(have):
        table[s, :n] = order[at:at + n]
        at += n
    angle_type = ta.float32 if wide else dtype
    positions = max(a + b for a, b in zip(new, context))
    angles = rng.uniform(0, 6.28, (positions, d // 2))
    cos, sin = rounded(np.cos(angles), angle_type), rounded(np.sin(angles), angle_type)
    total = sum(new)
    qkv = rounded(rng.standard_normal((total, heads + 2 * kv, d)), dtype)
    keys, values = (rounded(rng.standard_normal((room, kv, page, d)), dtype) for _ in range(2))
    dk, dv, dqkv = ta.tensor(keys, dtype, device), ta.tensor(values, dtype, device), ta.tensor(qkv, dtype, device)
    got = ops.append_pages(dqkv[:, heads:heads + kv], dqkv[:, heads + kv:], dk, dv, ta.tensor(table, ta.int32, device),
                           ta.tensor(np.concatenate([[0], np.cumsum(new)]), ta.int32, device), ta.tensor(np.array(context), ta.int32, device),
                           ta.tensor(cos, angle_type, device), ta.tensor(sin, angle_type, device), dqkv[:, :heads])
    place = [(s, context[s] + i) for s in range(5) for i in range(new[s])]
    at = np.array([p for _, p in place])
    want, size = turned(qkv, cos[at][:, None], sin[at][:, None])
    near(got.numpy(), want[:, :heads], size[:, :heads], dtype, "q")
    written = np.zeros((room, page), bool)
    k, v = dk.numpy(), dv.numpy()
    for t, (s, p) in enumerate(place):
        where = table[s, p // page], slice(None), p % page
        near(k[where], want[t, heads:heads + kv], size[t, heads:heads + kv], dtype, "k")
        np.testing.assert_array_equal(v[where], qkv[t, heads + kv:])
        written[table[s, p // page], p % page] = True
    np.testing.assert_array_equal(np.moveaxis(k, 2, 1)[~written], np.moveaxis(keys, 2, 1)[~written])
    np.testing.assert_array_equal(np.moveaxis(v, 2, 1)[~written], np.moveaxis(values, 2, 1)[~written])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d,slip", [(64, 0), (64, 1), (6, 2), (5, 0)])
def test_append_without_angles_copies_bits(d, slip, dtype, device):
    """Rows that start anywhere (columns of a wider tensor), a cache with tokens before heads, no rotation: NaN and infinities travel too."""
    rng = np.random.default_rng(22)
    x = rounded(rng.standard_normal((9, 4, d + slip + 1)), dtype)
    x[0, 0], x[3, 1, 1], x[5, 2, 2] = np.nan, np.inf, -np.inf
    dx = ta.tensor(x, dtype, device)
    k, v = dx[:, 0:2, slip:slip + d], dx[:, 2:4, slip:slip + d]
    pools = [ta.tensor(np.zeros((6, 4, 2, d)), dtype, device).transpose(1, 2) for _ in range(2)]
    table = np.array([[4, 1, 0], [2, 5, 3]])
    assert ops.append_pages(k, v, *pools, ta.tensor(table, ta.int32, device), ta.tensor(np.array([0, 4, 9]), ta.int32, device), ta.tensor(np.array([3, 7]), ta.int32, device)) is None
    for pool, first in zip(pools, (0, 2)):
        want = np.zeros((6, 2, 4, d))
        for t in range(9):
            s, p = (0, 3 + t) if t < 4 else (1, 7 + t - 4)
            want[table[s, p // 4], :, p % 4] = x[t, first:first + 2, slip:slip + d]
        np.testing.assert_array_equal(pool.numpy(), want)


def test_append_where_there_is_no_page(device):
    """Missing pages, positions behind the table, padding rows: nothing is written, the queries turn all the same (padding rows stay)."""
    rng = np.random.default_rng(23)
    kv, d, page, dtype = 2, 8, 4, ta.float32
    x = rounded(rng.standard_normal((10, 3 * kv, d)), dtype)
    dx = ta.tensor(x, dtype, device)
    dk, dv = (ta.tensor(np.zeros((3, kv, page, d)), dtype, device) for _ in range(2))
    table = np.array([[2, -1], [1 << 30, 0]])
    cos, sin = np.cos(np.arange(6)[:, None] + np.zeros(d // 2)), np.sin(np.arange(6)[:, None] + np.zeros(d // 2))
    out = ta.tensor(np.full((10, kv, d), 7.0), dtype, device)
    operands = [dx[:, kv:2 * kv], dx[:, 2 * kv:], ta.tensor(table, ta.int32, device), ta.tensor(np.array([1, 4, 8]), ta.int32, device), ta.tensor(np.array([2, 3]), ta.int32, device),
                ta.tensor(cos, dtype, device), ta.tensor(sin, dtype, device), dx[:, :kv], dk, dv, out]
    lib = ta.library()
    assert lib.kernels["append_pages"](*[C.byref(t.descriptor()) for t in operands], device.stream()) == abi.SUCCESS
    k, got = dk.numpy(), out.numpy()
    assert (got[0] == 7).all() and (got[8:] == 7).all()
    positions = [2, 3, 4, 3, 4, 5, 6]                  # (6 is behind the angles: their last row)
    at = np.minimum(positions, 5)
    want, size = turned(x[1:8], rounded(cos, dtype)[at][:, None], rounded(sin, dtype)[at][:, None])
    near(got[1:8], want[:, :kv], size[:, :kv], dtype, "q")
    near(k[2, :, 2:4].transpose(1, 0, 2), want[:2, kv:2 * kv], size[:2, kv:2 * kv], dtype, "k of page 2")
    near(k[0, :, 0:3].transpose(1, 0, 2), want[4:7, kv:2 * kv], size[4:7, kv:2 * kv], dtype, "k of page 0")
    assert (k[1] == 0).all() and (k[2, :, :2] == 0).all() and (k[0, :, 3] == 0).all()


def test_append_writes_past_32_bits(device):
    pages, kv, page, d = 9000, 8, 256, 128
    keys, values = (ta.Tensor(ta.float16, (pages, kv, page, d)).initialize(device) for _ in range(2))
    assert keys.nelements > 1 << 31
    rng = np.random.default_rng(24)
    x = rounded(rng.standard_normal((3, 2 * kv, d)), ta.float16)
    dx = ta.tensor(x, ta.float16, device)
    ops.append_pages(dx[:, :kv], dx[:, kv:], keys, values, ta.tensor(np.array([[pages - 1, 8400]]), ta.int32, device), ta.tensor(np.array([0, 3]), ta.int32, device),
                     ta.tensor(np.array([254]), ta.int32, device))
    for pool, first in ((keys, 0), (values, kv)):
        np.testing.assert_array_equal(ops.repack(pool[pages - 1, :, 254:256]).numpy(), x[:2, first:first + kv].transpose(1, 0, 2))
        np.testing.assert_array_equal(ops.repack(pool[8400, :, 0]).numpy(), x[2, first:first + kv])


@pytest.mark.parametrize("dtype", [ta.int8, ta.bfloat16, ta.float32, ta.float64], ids=str)
@pytest.mark.parametrize("lead,page", [((), (2, 16, 64)), ((3, 2), (2, 16, 64)), ((2,), (1, 5, 7)), ((2, 1, 2, 2), (1, 1, 2))])
def test_copies_one_after_another(lead, page, dtype, device):
    """Chains, swaps through a third page, the same source and the same target twice, a page onto itself; more copies than one launch takes."""
    rng = np.random.default_rng(25)
    pages = 1200
    pool = rng.integers(-100, 100, lead + (pages,) + page)
    sources = [3, 4, 5, 3, 3, 9, 9, 7, 8, 1, 2, 1199] + list(rng.integers(0, pages, 1500))
    targets = [4, 5, 6, 3, 9, 10, 10, 8, 7, 2, 1, 0] + list(rng.integers(0, pages, 1500))
    for count in (1, 5, 12, 40, len(sources)):
        got = ta.tensor(pool, dtype, device)
        want = np.moveaxis(got.numpy().copy(), len(lead), 0)
        assert ops.copy_pages(got, sources[:count], targets[:count]) is got
        for a, b in zip(sources[:count], targets[:count]):
            want[b] = want[a]
        np.testing.assert_array_equal(got.numpy(), np.moveaxis(want, 0, len(lead)))


def test_copies_of_views_and_recorded_copies(device):
    """Layers that lie apart (keys of every layer in a tensor of keys and values), a recording replayed with other contents."""
    rng = np.random.default_rng(26)
    first, second = (rng.standard_normal((4, 2, 10, 2, 4, 8)).astype(np.float32) for _ in range(2))
    whole = ta.tensor(first, ta.float32, device)
    with ta.Graph(device) as g:
        ops.copy_pages(whole[:, 1], [1, 2], [2, 7])
    for x in (first, second, first):
        ops.copy_into(whole, ta.tensor(x, ta.float32, device))
        g.launch()
        want = x.copy()
        want[:, 1, 2] = x[:, 1, 1]
        want[:, 1, 7] = x[:, 1, 1]
        np.testing.assert_array_equal(whole.numpy(), want)


def test_copies_past_32_bits(device):
    pool = ta.Tensor(ta.float16, (9000, 8, 256, 128)).initialize(device)
    x = np.random.default_rng(27).standard_normal((1, 8, 256, 128)).astype(np.float16)
    ops.copy_into(pool[8999:9000], ta.tensor(x, ta.float16, device))
    ops.copy_pages(pool, [8999], [8300])
    np.testing.assert_array_equal(ops.repack(pool[8300:8301]).numpy(), x)


@pytest.mark.parametrize("n", [63, 64, 65, 300, 4163])
def test_append_to_many_sequences(n, device):
    """More sequences than a wavefront has lanes, empty ones in front, behind and in between, tokens of no sequence at both ends."""
    rng = np.random.default_rng(n)
    new = rng.integers(0, 3, n)
    new[[0, 1, n - 1]] = 0
    total, first = int(new.sum()), 2
    context = rng.integers(0, 4, n)
    table = rng.permutation(2 * n).reshape(n, 2)                  # pages of 4, at most 5 tokens
    k = rounded(rng.standard_normal((total + 5, 1, 8)), ta.bfloat16)
    keys, values = (ta.tensor(np.zeros((2 * n, 1, 4, 8)), ta.bfloat16, device) for _ in range(2))
    starts = first + np.concatenate([[0], np.cumsum(new)])
    dk = ta.tensor(k, ta.bfloat16, device)
    ops.append_pages(dk, dk, keys, values, *(ta.tensor(x, ta.int32, device) for x in (table, starts, context)))
    want = np.zeros((2 * n, 1, 4, 8))
    for s in range(n):
        for i in range(new[s]):
            at = context[s] + i
            want[table[s, at // 4], 0, at % 4] = k[starts[s] + i, 0]
    np.testing.assert_array_equal(keys.numpy(), want)
    np.testing.assert_array_equal(values.numpy(), want)
