"""What a paged cache does on the host is not recorded: inside a recording it is refused, and nothing has changed."""
import numpy as np
import pytest

import tannic_amd as ta
from tannic_amd import ops
from tannic_amd.paged_cache import PagedCache

pytestmark = pytest.mark.gpu


def test_nothing_is_planned_or_moved_inside_a_recording(device):
    cache = PagedCache(1, 8, 4, 1, 8, ta.float32, device)
    ops.copy_into(cache.storage, ta.tensor(np.arange(2 * 8 * 4 * 8, dtype=np.float32).reshape(1, 2, 8, 1, 4, 8), ta.float32, device))
    a = cache.add()
    cache.advance(cache.plan([a], [6]))
    b = cache.fork(a)
    cache.advance(cache.plan([b], [0]))
    gone = cache.add()
    cache.advance(cache.plan([gone], [1]))
    late = cache.add()
    cache.advance(cache.plan([late], [1]))
    cache.free(gone)
    x = ta.tensor(np.ones(4), ta.float32, device)
    before = {i: cache.pages_of(i) for i in (a, b, late)}, cache.free_pages, list(cache._users), cache.storage.numpy().copy()
    with ta.Graph(device) as g:
        y = ops.add(x, x)
        for call in (lambda: cache.plan([b], [1]), lambda: cache.plan([b, a], [1, 0], columns=4), cache.compact):
            with pytest.raises(ta.TannicError, match="record"):
                call()
    for _ in range(2):
        g.launch()
        assert (y.numpy() == 2).all()
    after = {i: cache.pages_of(i) for i in (a, b, late)}, cache.free_pages, list(cache._users), cache.storage.numpy()
    assert before[:3] == after[:3]
    np.testing.assert_array_equal(after[3], before[3])
    # afterwards all of it works
    step = cache.plan([b], [1])
    assert cache.pages_of(b)[1] != cache.pages_of(a)[1]
    cache.advance(step)
    assert cache.compact() in (0, 1)
