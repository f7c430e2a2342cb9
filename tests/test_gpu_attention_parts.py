"""Attention of one group of rows over so many keys that its parts meet in five turns, against the definition in 64 bits."""
import numpy as np
import pytest

import tannic_amd as ta
from attention_support import Cache, assert_within, head_attention, rounded
from tannic_amd import ops

pytestmark = pytest.mark.gpu

SCALE = float(np.float32(1.0 / np.sqrt(128)))


@pytest.mark.parametrize("dtype", [ta.float16, ta.bfloat16], ids=str)
@pytest.mark.parametrize("missing", [False, True])
def test_one_kv_head_behind_70000_keys(missing, dtype, device):
    """17 rows of one kv head, 274 parts; with the last pages missing the last parts come first.  Every call gives the same bits, and the next one of other sizes is right."""
    rng = np.random.default_rng(70)
    c = Cache(rng, dtype, device, 17, 1, 128, 64, [1], [70000])
    gone = [(0, column) for column in range(65600 // 64, 1094)] if missing else []
    for s, column in gone:
        c.host_table[s, column] = -1
    table, q = ta.tensor(c.host_table, ta.int32, device), ta.tensor(c.q, dtype, device)
    results = [ops.attend_pages(q, c.keys, c.values, table, c.starts, c.lengths, SCALE) for _ in range(20)]
    first = results[0].storage()
    for r in results[1:]:
        np.testing.assert_array_equal(r.storage(), first)
    want, slack, size, total = c.expected(SCALE, gone)
    assert_within(results[0].numpy(), want, slack, size, dtype, total)
    c = Cache(rng, dtype, device, 4, 1, 128, 16, [30], [2500])
    got = ops.attend_pages(ta.tensor(c.q, dtype, device), c.keys, c.values, c.table, c.starts, c.lengths, SCALE).numpy()
    want, slack, size, total = c.expected(SCALE)
    assert_within(got, want, slack, size, dtype, total)


def test_one_kv_head_over_66000_states(device):
    rng = np.random.default_rng(71)
    q = rounded(rng.standard_normal((1, 2, 10, 128)), ta.bfloat16)
    k, v = (rounded(rng.standard_normal((1, 66000, 1, 128)), ta.bfloat16) for _ in range(2))
    got = ops.attend(*(ta.tensor(x, ta.bfloat16, device) for x in (q, k, v)), None, SCALE).numpy()
    for h in range(10):
        want, slack, size = head_attention(q[0, :, h], k[0, :, 0], v[0, :, 0], SCALE, [66000] * 2)
        assert_within(got[0, :, h], want, slack, size, ta.bfloat16)
