"""Operands of the attention that lie otherwise than a cache's own: keys and values in different orders, every other page of a pool, columns of a wider table, one
sequence's states for all, and lengths that go beyond the table."""
import numpy as np
import pytest

import tannic_amd as ta
from attention_support import Cache, assert_within, head_attention, rounded
from tannic_amd import ops

pytestmark = pytest.mark.gpu

TYPES = [ta.float16, ta.bfloat16, ta.float32, ta.float64]
NEW = [[1, 1, 1], [40, 3, 70]]


def check(c, device, keys=None, values=None, table=None, lengths=None):
    got = ops.attend_pages(ta.tensor(c.q, c.dtype, device), keys or c.keys, values or c.values, table or c.table, c.starts, lengths or c.lengths, 0.125).numpy()
    want, slack, size, total = c.expected(0.125)
    assert_within(got, want, slack, size, c.dtype, total)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new", NEW, ids=str)
@pytest.mark.parametrize("page,d", [(16, 64), (16, 128), (5, 128), (64, 256)])
def test_keys_and_values_in_different_orders(page, d, new, dtype, device):
    rng = np.random.default_rng(page + d)
    c = Cache(rng, dtype, device, 4, 2, d, page, new, [100, 17, 3])
    with np.errstate(invalid="ignore"):
        values = np.asarray(c.values.numpy(), np.float64)
    # values with the tokens of a page before its heads, every other page of a pool; the table is columns of a wider one
    pool = np.full((2 * values.shape[0], page, 2, d), np.nan)
    pool[::2] = values.transpose(0, 2, 1, 3)
    wide = np.full((3, c.host_table.shape[1] + 5), 7)
    wide[:, 2:2 + c.host_table.shape[1]] = c.host_table
    check(c, device, values=ta.tensor(pool, dtype, device)[::2].transpose(1, 2), table=ta.tensor(wide, ta.int32, device)[:, 2:2 + c.host_table.shape[1]])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens", [1, 50])
def test_one_encoder_for_all(tokens, dtype, device):
    rng = np.random.default_rng(tokens)
    q = rounded(rng.standard_normal((3, tokens, 4, 64)), dtype)
    k, v = (rounded(rng.standard_normal((1, 90, 2, 64)), dtype) for _ in range(2))
    lengths = [90, 0, 33]
    got = ops.attend(ta.tensor(q, dtype, device), *(ta.tensor(x, dtype, device).expand(3, 90, 2, 64) for x in (k, v)), ta.tensor(np.array(lengths), ta.int32, device), 0.125).numpy()
    for b in range(3):
        for h in range(4):
            want, slack, size = head_attention(q[b, :, h], k[0, :, h // 2], v[0, :, h // 2], 0.125, [lengths[b]] * tokens)
            assert_within(got[b, :, h], want, slack, size, dtype, np.abs(v[0, :, h // 2]).sum(0))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new", [[1, 1], [20, 45]], ids=str)
def test_lengths_beyond_the_table(new, dtype, device):
    """Positions that no column is for have no keys: the rows see what the table has."""
    rng = np.random.default_rng(5)
    c = Cache(rng, dtype, device, 4, 2, 64, 16, new, [64 - n for n in new], columns=0, width=4)
    lengths = ta.tensor(np.array([500, (1 << 31) - 1]), ta.int32, device)
    got = ops.attend_pages(ta.tensor(c.q, dtype, device), c.keys, c.values, c.table, c.starts, lengths, 0.125).numpy()
    first = 0
    for s, n in enumerate(new):
        for h in range(4):
            want, slack, size = head_attention(c.q[first:first + n, h], c.k[s][:, h // 2], c.v[s][:, h // 2], 0.125, [64] * n)
            assert_within(got[first:first + n, h], want, slack, size, dtype, np.abs(c.v[s][:, h // 2]).sum(0))
        first += n


@pytest.mark.parametrize("dtype", [ta.bfloat16, ta.float32], ids=str)
def test_a_chunk_among_single_tokens(dtype, device):
    """Most sequences have one new token, one has a chunk: which kernel takes the call goes by the average."""
    rng = np.random.default_rng(6)
    for tokens, chunk in ((30, 40), (9, 200)):
        context = rng.integers(0, 300, tokens + 1).tolist()
        new = [1] * tokens + [chunk]
        check(Cache(rng, dtype, device, 8, 2, 64, 16, new, context), device)
