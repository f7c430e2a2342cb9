"""Attention of queries and keys that are not finite, whichever kernel takes them: 0 times them is no number."""
import numpy as np
import pytest

import tannic_amd as ta
from attention_support import Cache, assert_within
from tannic_amd import ops

pytestmark = pytest.mark.gpu

TYPES = [ta.float16, ta.bfloat16, ta.float32, ta.float64]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 128, 256, 33])
@pytest.mark.parametrize("scale", [0.0, -0.0])
@pytest.mark.parametrize("new,context", [([1, 1, 1], [40, 3, 200]), ([50, 1, 20], [100, 0, 30])], ids=str)
def test_a_scale_of_zero(new, context, scale, d, dtype, device):
    """Every key weighs the same; a row whose query has an infinite or no number in it, or that sees such a key, is no number."""
    rng = np.random.default_rng(80)
    c = Cache(rng, dtype, device, 4, 2, d, 16, new, context)
    want, slack, size, total = c.expected(0.0)
    n = sum(new)
    q, keys, odd = c.q.copy(), c.keys.numpy().astype(np.float64), np.zeros((n, 4), bool)
    q[0, 1, 5], odd[0, 1] = np.nan, True
    q[n - 1, 0, d - 1], odd[n - 1, 0] = np.inf, True
    q[n - 2, 3, 0], odd[n - 2, 3] = -np.inf, True
    j = context[0] + new[0] - 1      # the last key of the first sequence, which its last token sees
    keys[c.host_table[0, j // 16], 1, j % 16, 2] = np.inf
    odd[new[0] - 1, 2:] = True
    got = ops.attend_pages(ta.tensor(q, dtype, device), ta.tensor(keys, dtype, device), c.values, c.table, c.starts, c.lengths, scale).numpy()
    assert np.isnan(got[odd]).all()
    assert_within(got[~odd], want[~odd], slack[~odd], size[~odd], dtype, total[~odd])
